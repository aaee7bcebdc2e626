"""The global norm of many gradients, and clipping by it.

A network's parameters are many small tables (785 of them in the 784-leaf model); a clipper lists their
gradients once and then needs two kernel launches per step, however many there are
(``bn_gradient_set_*`` of ``include/bn_hip.h``).  There is no CPU path.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from ..inference_machines.hip_spa import _native


def _check(tensors, name):
    for i, t in enumerate(tensors):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name}[{i}] must be a tensor")
        if t.dtype not in _native.DTYPE_CODES:
            raise TypeError(f"{name}[{i}] must be float32, float64, float16 or bfloat16, not {t.dtype}")
        if t.device.type != "cuda":
            raise ValueError(f"{name}[{i}] must be on an AMD GPU (there is no CPU path)")
        if t.device != tensors[0].device:
            raise ValueError(f"{name}[{i}] is on {t.device}, {name}[0] on {tensors[0].device}")
        if not t.is_contiguous():
            raise ValueError(f"{name}[{i}] must be contiguous")


class HipGradientClipper:
    """``clip(max_norm)`` scales the gradients it was built for so that their global norm
    ``sqrt(sum of all squares)`` is at most ``max_norm``, and returns the norm they had.

    ``gradients``: tensors on one GPU, each float32, float64, float16 or bfloat16 and contiguous, any sizes.  They
    are read where they lie at every call: keep them (fill them in place rather than
    replacing them: ``zero_grad(set_to_none=False)``; after its default, which drops ``.grad``, the clipper would
    scale the dropped tensors).  ``out``: tensors of the same shapes and types for the clipped copies; without it the
    gradients themselves are scaled.  Listing one tensor twice in place, or an output over
    another tensor, is an error.  Build a clipper outside of graph capture; its calls may be captured, and
    the clipper is kept as long as their graph is replayed.

    The norm is summed in float64, in an order that depends on the list alone.  With a NaN among the
    gradients the norm and everything scaled by it is NaN; with an infinite norm the factor is 0.
    """

    def __init__(self, gradients: Sequence[torch.Tensor], out: Optional[Sequence[torch.Tensor]] = None):
        gradients = list(gradients)
        outputs = gradients if out is None else list(out)
        if not gradients:
            raise ValueError("no gradients given")
        _check(gradients, "gradients")
        if out is not None:
            if len(outputs) != len(gradients):
                raise ValueError(f"{len(outputs)} outputs for {len(gradients)} gradients")
            _check(outputs, "out")
            for i, (g, o) in enumerate(zip(gradients, outputs)):
                if g.shape != o.shape or g.dtype != o.dtype or g.device != o.device:
                    raise ValueError(f"out[{i}] must have the shape, type and device of gradients[{i}]")
        # one tensor for each version counter among the outputs: views share their base's
        written = (o if o._base is None else o._base for o in outputs)
        self._written = list({id(t): t for t in written}.values())
        self._device = gradients[0].device
        self._gradients, self._outputs = gradients, outputs  # the set holds their addresses
        self._lib = _native.load()
        count = len(gradients)
        handle = ctypes.c_void_p()
        with torch.cuda.device(self._device):
            _native.check(self._lib.bn_gradient_set_create(
                count, _native.i32_array([_native.DTYPE_CODES[g.dtype] for g in gradients]),
                (ctypes.c_int64 * count)(*[g.numel() for g in gradients]),
                (ctypes.c_void_p * count)(*[g.data_ptr() for g in gradients]),
                (ctypes.c_void_p * count)(*[o.data_ptr() for o in outputs]), ctypes.byref(handle)))
        self._handle = handle
        self._workspace_bytes = self._lib.bn_gradient_set_workspace_bytes(handle)

    def __del__(self):
        handle = getattr(self, "_handle", None)
        if handle:
            try:
                self._lib.bn_gradient_set_destroy(handle)
            except Exception:
                pass
            self._handle = None

    def _call(self, entry, *args) -> torch.Tensor:
        norm = torch.empty((), device=self._device, dtype=torch.float64)
        workspace = torch.empty((self._workspace_bytes,), device=self._device, dtype=torch.uint8)
        _native.launch(self._device, entry, self._handle, *args, workspace.data_ptr(), norm.data_ptr())
        return norm

    def norm(self) -> torch.Tensor:
        """The gradients' global norm, a float64 scalar on the device."""
        return self._call(self._lib.bn_gradient_set_norm)

    def clip(self, max_norm: float) -> torch.Tensor:
        """Writes the gradients, scaled by ``max_norm / norm`` where the norm exceeds ``max_norm``, to
        their outputs; returns the norm before scaling (float64 scalar on the device).  As after any
        operation in place, a backward pass that needs what the outputs held before raises."""
        max_norm = float(max_norm)
        if not 0.0 < max_norm < float("inf"):
            raise ValueError(f"max_norm must be positive and finite, not {max_norm}")
        norm = self._call(self._lib.bn_gradient_set_clip, max_norm)
        torch.autograd.graph.increment_version(self._written)  # autograd does not see what a kernel writes
        return norm
