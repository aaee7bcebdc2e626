from .common import BatchEvaluator, Evaluator, OptimizerLogger
from .em_batch_optimizer import EmBatchOptimizer, EmBatchOptimizerSettings
from .em_optimizer import EmOptimizer, EmOptimizerSettings
from .gradient_clipper import HipGradientClipper
from .states_likelihood import states_log_likelihood, states_log_likelihood_and_gradient

__all__ = [
    "BatchEvaluator", "Evaluator", "OptimizerLogger",
    "EmBatchOptimizer", "EmBatchOptimizerSettings", "EmOptimizer", "EmOptimizerSettings",
    "HipGradientClipper", "states_log_likelihood", "states_log_likelihood_and_gradient",
]
