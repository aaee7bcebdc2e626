"""Draws from rows of logits: one state per row, at uniform numbers the caller gives.

``HipBayesianNetworkSampler`` draws from a network's CPTs; ``draw_states`` draws from distributions
that no CPT holds: posteriors (``infer_single_nodes(...)[0].log()``) or logits a model computes, with
the usual restrictions of the tail (``bn_draw_states`` of ``include/bn_hip.h``).  There is no CPU path.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Union

import torch

from .. import rows as _rows
from ..inference_machines.hip_spa import _native

Setting = Union[float, torch.Tensor, None]


def draw_states(logits: torch.Tensor, uniforms: torch.Tensor, *, temperature: Setting = None,
                top_k: Union[int, torch.Tensor, None] = None, top_p: Setting = None, min_p: Setting = None,
                num_states: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One state per row of ``logits`` as an ``int32`` tensor ``[rows]``.

    ``logits``: ``[rows, states]``, float32, float64, float16 or bfloat16; rows may lie any distance
    apart (``expand`` for many draws from one row), up to 2^24 states.  ``uniforms``: float32 or
    float64 ``[rows]`` in [0, 1].

    With weights ``exp((x - max x) / temperature)``, ``top_k`` keeps the most probable states, ``top_p``
    the shortest prefix of those (most probable first, ties by index) that holds that share of their
    weight, ``min_p`` those of at least that share of the largest weight.  The state is the first kept one,
    in ascending index, at which the cumulative weight exceeds ``uniform`` times the kept total.
    ``temperature=0`` takes the largest logit (lowest index).  A setting is a number, or a tensor
    ``[rows]`` with one per row (float32 / float64; int32 / int64 for ``top_k``), in which 0 switches
    ``top_k`` and ``min_p`` off and 1 switches ``top_p`` off.

    ``num_states`` (int32 / int64 ``[rows]``): how many states each row has; the rest is padding
    and not read.  Sums are taken in double: a border within 1e-11 of a row's weight may be decided either way.
    A row without anything to draw from gives -1: no states, all ``-inf``, a NaN or
    ``+inf`` among its states, a uniform number outside [0, 1], a bad temperature of its own.
    """
    _rows.check_logits(logits)
    _rows.check_per_row(uniforms, logits, (torch.float32, torch.float64), "uniforms")
    filters = _native.DrawFilters(1.0, 0, 1.0, 0.0)
    keep = []  # tensors the call reads, alive until it is enqueued

    def per_row(value, name, dtypes, dtype):
        _rows.check_per_row(value, logits, dtypes, name)
        value = value.to(dtype).contiguous()
        keep.append(value)
        setattr(filters, name + "_dev", value.data_ptr())

    for name, value in (("temperature", temperature), ("top_p", top_p), ("min_p", min_p)):
        if isinstance(value, torch.Tensor):
            per_row(value, name, (torch.float32, torch.float64), torch.float64)
        elif value is not None:
            setattr(filters, name, float(value))
    if isinstance(top_k, torch.Tensor):
        per_row(top_k, "top_k", (torch.int64, torch.int32), torch.int64)
    elif top_k is not None:
        if not 0 <= top_k < 2**63 or int(top_k) != top_k:
            raise ValueError(f"top_k must be a whole number that is not negative, not {top_k}")
        filters.top_k = int(top_k)
    if not 0.0 <= filters.temperature < float("inf"):
        raise ValueError(f"temperature must be finite and not negative, not {temperature}")
    if not 0.0 < filters.top_p <= 1.0:
        raise ValueError(f"top_p must be in (0, 1], not {top_p}")
    if not 0.0 <= filters.min_p <= 1.0:
        raise ValueError(f"min_p must be in [0, 1], not {min_p}")

    uniforms = uniforms.contiguous()
    counts = _rows.row_states(num_states, logits)
    lib = _native.load()
    rows, states = logits.shape
    dtype = _native.DTYPE_CODES[logits.dtype]
    device = logits.device
    out = torch.empty((rows,), device=device, dtype=torch.int32)
    if rows == 0:
        return out
    need = lib.bn_draw_states_workspace_bytes(dtype, rows, states)
    if need < 0:
        raise ValueError(f"draw_states takes at most 2^24 states per row, not {states}")
    workspace = torch.empty((need,), device=device, dtype=torch.uint8) if need else None
    _native.launch(device, lib.bn_draw_states, dtype, logits.data_ptr(), rows, states, logits.stride(0),
                   _native.pointer(counts), _native.DTYPE_CODES[uniforms.dtype], uniforms.data_ptr(),
                   ctypes.byref(filters), _native.pointer(workspace), out.data_ptr())
    return out
