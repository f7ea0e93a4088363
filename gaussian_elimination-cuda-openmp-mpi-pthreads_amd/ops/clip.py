"""2-norm over many tensors and clipping by it (csrc/hip/clip.hip)."""
from __future__ import annotations

import math
from array import array
from typing import Sequence

import torch
from torch.autograd.graph import increment_version

from .. import _native
from ..utils.tensors import has_tangent, stream_handle
from .adapter import TYPES


def _dense(t: torch.Tensor) -> bool:
    """Whether t fills its memory without gaps, in any order of its dimensions."""
    if t.is_contiguous():
        return True
    size = 1
    for n, s in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n != 1), key=lambda d: d[1]):
        if s != size:
            return False
        size *= n
    return True


_PTR, _NUMEL, _SAME_SIZE = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.is_same_size
_DTYPE = torch.Tensor.dtype.__get__


def _types(tensors: list[torch.Tensor]) -> bytes:
    try:
        return bytes(map(TYPES.__getitem__, map(_DTYPE, tensors)))
    except KeyError as e:
        raise TypeError(f"clip_global_norm takes float32, bfloat16 and float16, not {e.args[0]}") from None


def _check_memory(tensors: list[torch.Tensor], dev: torch.device) -> bool:
    """Whether all are contiguous; an error where one is elsewhere or not dense."""
    if set(map(torch.Tensor.get_device, tensors)) != {dev.index}:
        raise ValueError("all tensors must be on one device")
    if all(map(torch.Tensor.is_contiguous, tensors)):
        return True
    if not all(map(_dense, tensors)):
        raise ValueError("a tensor has gaps in memory, or overlaps itself")
    return False


def clip_global_norm(tensors: Sequence[torch.Tensor], max_norm: float,
                     out: Sequence[torch.Tensor] | None = None) -> torch.Tensor:
    """Scales all tensors by min(1, max_norm / (norm + 1e-6)), norm the 2-norm of
    all their elements together, and returns that norm (a float32 scalar on
    the device, infinite where it leaves that type; nothing waits for it).

    tensors: float32, bfloat16 and float16 in any mixture, on one device, each
    without gaps in memory (any order of dimensions).
    out: tensors of the same types and shapes (and strides, if they are not
    contiguous) that get the scaled copies, the inputs staying as they are;
    None: in place.  What is written must not overlap anything else in the call.
    max_norm = math.inf only measures.  As the factor comes from the norm, a NaN anywhere
    makes all of them NaN, and an infinity makes the finite elements zero.
    Squares and their sum are held in float64, in an order that does not change
    from run to run.  Autograd records nothing, as under torch.no_grad(), and
    sees that what is written has changed; tensors with forward-mode tangents
    are refused.  May be captured into a graph."""
    tensors = list(tensors)
    max_norm = float(max_norm)
    if math.isnan(max_norm) or max_norm < 0:
        raise ValueError("max_norm must be a number and not negative")
    if not tensors:
        raise ValueError("no tensors")
    dev = tensors[0].device
    if dev.type != "cuda":
        raise ValueError("clip_global_norm needs CUDA tensors")
    types = _types(tensors)
    sizes = array("q", map(_NUMEL, tensors))
    contiguous = _check_memory(tensors, dev)
    src = array("Q", map(_PTR, tensors))
    if out is None:
        dst = src
    else:
        out = list(out)
        if len(out) != len(tensors) or _types(out) != types or not all(map(_SAME_SIZE, out, tensors)):
            raise ValueError("out must have one tensor of the same type and shape per input")
        if not (_check_memory(out, dev) and contiguous):
            if any(o.stride() != t.stride() for t, o in zip(tensors, out)):
                raise ValueError("each out must have the strides of its input")
        dst = array("Q", map(_PTR, out))
    if has_tangent(tensors if out is None else [*tensors, *out]):
        raise ValueError("clip_global_norm is not followed by forward-mode differentiation: it would drop the tangents")
    norm = torch.empty((), dtype=torch.float32, device=dev)
    lib = _native.lib()
    ws = torch.empty(lib.gelim_clip_workspace(), dtype=torch.uint8, device=dev)

    def call():
        _native.check(lib.gelim_clip_norm(src.buffer_info()[0], dst.buffer_info()[0], sizes.buffer_info()[0], types,
                                          len(tensors), max_norm, norm.data_ptr(), ws.data_ptr(), ws.numel(),
                                          stream_handle(dev)), "clip_global_norm")

    if torch.cuda.current_device() == dev.index:
        call()
    else:
        with torch.cuda.device(dev):
            call()
    if out is not None or max_norm != math.inf:
        increment_version(tensors if out is None else out)  # they may have been saved for a backward pass
    return norm
