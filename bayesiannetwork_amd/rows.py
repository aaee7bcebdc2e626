"""Argument checks shared by the operators on rows of logits (``samplers.draw_states``,
``optimizers.states_log_likelihood``): a row is one categorical distribution over its states."""

from __future__ import annotations

from typing import Optional

import torch

from .inference_machines.hip_spa import _native


def check_logits(logits: torch.Tensor, name: str = "logits") -> None:
    if not isinstance(logits, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if logits.dtype not in _native.DTYPE_CODES:
        raise TypeError(f"{name} must be float32, float64, float16 or bfloat16, not {logits.dtype}")
    if logits.dim() != 2:
        raise ValueError(f"{name} must be [rows, states], not of shape {tuple(logits.shape)}")
    width = logits.size(1)
    if width < 1:
        raise ValueError(f"{name} must have at least one state per row")
    if not logits.is_cuda:
        raise ValueError(f"{name} must be on an AMD GPU (there is no CPU path)")
    if width > 1 and logits.stride(1) != 1:
        raise ValueError(f"the states of a row of {name} must lie side by side (call .contiguous())")


def check_per_row(tensor: torch.Tensor, logits: torch.Tensor, dtypes, name: str) -> None:
    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if tensor.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, not {tensor.dtype}")
    if tensor.dim() != 1 or tensor.size(0) != logits.size(0):
        raise ValueError(f"{name} must have one entry per row: shape {(logits.size(0),)}, not {tuple(tensor.shape)}")
    if tensor.device != logits.device:
        raise ValueError(f"{name} is on {tensor.device}, the logits are on {logits.device}")


def row_states(num_states: Optional[torch.Tensor], logits: torch.Tensor) -> Optional[torch.Tensor]:
    """States of each row as the library takes them: contiguous int64."""
    if num_states is None:
        return None
    check_per_row(num_states, logits, (torch.int64, torch.int32), "num_states")
    return num_states.to(torch.int64).contiguous()
