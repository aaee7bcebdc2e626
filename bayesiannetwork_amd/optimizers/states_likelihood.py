"""Log-likelihood of observed states under rows of logits, with its gradient.

EM learns CPTs from expected counts.  A distribution whose logits come from somewhere else - a CPT row
as the softmax of free parameters, a network that maps features to a node's states, the class posterior
of a discriminatively trained model - is learned by the gradient of this log-likelihood instead
(``bn_states_log_likelihood`` and ``bn_states_log_likelihood_gradient`` of ``include/bn_hip.h``).
``HipGradientClipper`` bounds the step.  There is no CPU path.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from .. import rows as _rows
from ..inference_machines.hip_spa import _native

_STATE_BYTES = {torch.uint8: 1, torch.int32: 4, torch.int64: 8}


def _ll_dtype(logits: torch.Tensor) -> torch.dtype:
    return torch.float64 if logits.dtype == torch.float64 else torch.float32


def _row_arguments(logits, counts, states):
    return (_native.DTYPE_CODES[logits.dtype], logits.data_ptr(), logits.size(0), logits.size(1), logits.stride(0),
            _native.pointer(counts), states.data_ptr(), _STATE_BYTES[states.dtype])


def _forward(logits, states, counts, with_totals):
    rows, device = logits.size(0), logits.device
    ll = torch.empty((rows,), device=device, dtype=_ll_dtype(logits))
    totals = torch.empty((rows, 2), device=device, dtype=torch.float64) if with_totals else None
    _native.launch(device, _native.load().bn_states_log_likelihood, *_row_arguments(logits, counts, states),
                   ll.data_ptr(), _native.pointer(totals))
    return ll, totals


def _gradient(logits, states, counts, totals, weights, ll, out):
    _native.launch(logits.device, _native.load().bn_states_log_likelihood_gradient,
                   *_row_arguments(logits, counts, states), _native.pointer(totals), _native.pointer(weights),
                   0 if weights is None else weights.stride(0), _native.pointer(ll), out.data_ptr(), out.stride(0))


class _StatesLogLikelihood(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, states, counts):
        ll, totals = _forward(logits, states, counts, True)
        ctx.save_for_backward(logits, states, totals, *(() if counts is None else (counts,)))
        return ll

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, weights):
        logits, states, totals, *counts = ctx.saved_tensors
        out = torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)
        _gradient(logits, states, counts[0] if counts else None, totals, weights, None, out)
        return out, None, None


def _check(logits, states, num_states):
    _rows.check_logits(logits)
    _rows.check_per_row(states, logits, tuple(_STATE_BYTES), "states")
    return states.contiguous(), _rows.row_states(num_states, logits)


def states_log_likelihood(logits: torch.Tensor, states: torch.Tensor, *,
                          num_states: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``log softmax(logits[r])[states[r]]`` for every row: float32 ``[rows]`` (float64 for float64
    logits), differentiable in ``logits``.

    ``logits``: ``[rows, states]``, float32, float64, float16 or bfloat16, rows any distance apart.
    ``states``: uint8, int32 or int64 ``[rows]``; one that is none of its row's states (negative or too
    large) means the row was not observed: log-likelihood 0, gradient 0.  ``num_states`` (int32 /
    int64 ``[rows]``): how many states each row has, the rest being padding that is not read and gets
    gradient 0.  Logits of ``-inf`` are impossible states; a row with NaN or ``+inf`` gives NaN.
    Derivatives are of first order and reverse mode: logits with a tangent (``forward_ad``) are refused.
    """
    states, counts = _check(logits, states, num_states)
    # (a dual tensor requires no gradient, and its address is that of its values alone)
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(logits).tangent is not None:
        raise NotImplementedError("states_log_likelihood has no forward-mode derivative: the logits carry a tangent")
    if torch.is_grad_enabled() and logits.requires_grad:
        return _StatesLogLikelihood.apply(logits, states, counts)
    return _forward(logits, states, counts, False)[0]


def states_log_likelihood_and_gradient(logits: torch.Tensor, states: torch.Tensor,
                                       weights: Optional[torch.Tensor] = None, *,
                                       num_states: Optional[torch.Tensor] = None,
                                       out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The log-likelihoods ``ll`` of ``states_log_likelihood`` and the gradient of
    ``(weights * ll).sum()`` (no weights: 1 each) in the logits, in one call that reads the logits
    once where a row fits a block's registers.  Nothing is recorded for autograd.

    ``weights``: ``[rows]`` of ll's type.  ``out``: where the gradient goes, of the logits' shape
    and type; it may be ``logits`` itself, whose values the gradient then replaces.  As after any
    operation in place, a backward pass that needs what ``out`` held before raises.
    """
    states, counts = _check(logits, states, num_states)
    if weights is not None:
        _rows.check_per_row(weights, logits, (_ll_dtype(logits),), "weights")
    given = out is not None
    if not given:
        out = torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)
    else:
        _rows.check_logits(out, "out")
        if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
            raise ValueError("out must have the logits' shape, type and device")
        if out.requires_grad:
            raise ValueError("out must not require a gradient (pass its .detach())")
    ll = torch.empty((logits.shape[0],), device=logits.device, dtype=_ll_dtype(logits))
    _gradient(logits, states, counts, None, weights, ll, out)
    if given:
        torch.autograd.graph.increment_version(out)  # autograd does not see what a kernel writes
    return ll, out
