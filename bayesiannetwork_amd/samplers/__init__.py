from .abstractions import IBayesianNetworkSampler
from .batched_sampler import BatchedBayesianNetworkSampler
from .hip_sampler import HipBayesianNetworkSampler
from .state_draws import draw_states

__all__ = ["IBayesianNetworkSampler", "BatchedBayesianNetworkSampler", "HipBayesianNetworkSampler", "draw_states"]
