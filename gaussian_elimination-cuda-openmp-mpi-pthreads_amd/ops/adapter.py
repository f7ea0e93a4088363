"""Low-rank adapters of many requests beside a shared projection, and their gradients.

Row t of X with the adapter i = index[t]:

    Y[t] = X[t] @ W + scale[i] * (X[t] @ A[i]) @ B[i]

W (K, N) is shared by all rows, A (n, K, r) and B (n, r, N) hold the factors
of n adapters.  One call serves prompts, single tokens and any mixture of
requests; the gradient call is its backward pass for training the adapters
(W stays as it is).  fp32, bf16 and fp16; sums are held in fp32, and X @ A[i]
enters the second product with all of its bits (csrc/hip/adapter.hip).
"""
from __future__ import annotations

import struct
from functools import lru_cache

import torch
from torch.autograd.graph import increment_version

from .. import _native
from ..utils.tensors import has_tangent, stream_handle

MAX_RANK = 256
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
# gelim_adapter_args (csrc/include/gelim/gelim.h): 64-bit words, one of them a double
_ARGS = struct.Struct("=21qd8q")


def _stored(t: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """(t, distance of two rows as stored, 1 if stored transposed) of the last
    two dimensions; a copy where neither of them has unit stride."""
    if t.is_contiguous():
        return t, t.shape[-1], 0
    rs, cs = t.stride(-2), t.stride(-1)
    rows, cols = t.shape[-2:]
    if cs == 1 or cols == 1:
        return t, rs, 0
    if rs == 1 or rows == 1:
        return t, cs, 1
    t = t.contiguous()
    return t, t.stride(-2), 0


def _span(t: torch.Tensor) -> tuple[int, int]:
    """First and one past the last byte that t may touch."""
    if t.numel() == 0:
        return 0, 0
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a0 < b1 and b0 < a1


def _check(X, W, A, B, index, scale, more=()):
    # called for single tokens as well, so short of anything that takes a microsecond
    dtype = X.dtype
    if dtype not in TYPES:
        raise TypeError(f"adapter_matmul takes float32, bfloat16 and float16, not {dtype}")
    if not (W.dtype == A.dtype == B.dtype == dtype):
        raise TypeError("X, W, A and B must have one type")
    at = X.get_device()
    if not X.is_cuda or not (W.get_device() == A.get_device() == B.get_device() == at):
        raise ValueError("adapter_matmul needs CUDA tensors on one device")
    dev = X.device
    xs, ws, as_, bs = X.shape, W.shape, A.shape, B.shape
    if len(xs) != 2 or len(ws) != 2 or len(as_) != 3 or len(bs) != 3:
        raise ValueError("X and W must be 2-D, A and B 3-D")
    (T, K), (KW, N), (n, KA, r) = xs, ws, as_
    if KW != K or KA != K or bs != (n, r, N):
        raise ValueError(f"shape mismatch: X {tuple(xs)}, W {tuple(ws)}, A {tuple(as_)}, B {tuple(bs)}")
    if K < 1 or N < 1 or n < 1 or r < 1:
        raise ValueError("K, N, the rank and the number of adapters must be at least 1")
    if r > MAX_RANK:
        raise ValueError(f"rank {r} is above {MAX_RANK}")
    if index is None:
        if n != 1:
            raise ValueError("index may be left out with one adapter only")
    elif index.dtype != torch.int32:
        raise TypeError("index must be int32")
    elif index.shape != (T,) or index.get_device() != at:
        raise ValueError("index must have one entry per row of X, on its device")
    if isinstance(scale, torch.Tensor):
        if scale.dtype != torch.float32:
            raise TypeError("scale must be a number or float32")
        if scale.shape != (n,) or scale.get_device() != at:
            raise ValueError("scale must have one entry per adapter, on the device of X")
    if torch.is_grad_enabled() and (X.requires_grad or W.requires_grad or A.requires_grad or B.requires_grad or
                                    isinstance(scale, torch.Tensor) and scale.requires_grad):
        raise ValueError("adapter_matmul is not recorded by autograd: call it under torch.no_grad() and take the "
                         "gradients from adapter_matmul_grad")
    if has_tangent(t for t in (X, W, A, B, scale, *more) if isinstance(t, torch.Tensor)):
        raise ValueError("adapter_matmul is not followed by forward-mode differentiation: it would drop the tangents")
    return dev, T, K, N, n, r


@lru_cache(maxsize=4096)
def _workspace_bytes(grad: bool | tuple[bool, bool, bool], *layout) -> int:
    """What a call of these sizes and layouts needs; grad: whether it is the gradient, or which of its results."""
    dtype, T, K, N, r, n, ldx, ldw, wt, lda, at, ldb, bt, ldy, x, w, y, indexed = layout
    dX, dA, dB = grad if isinstance(grad, tuple) else (grad,) * 3
    # an address's low bits choose between reading in place and copying, so they take the place of the addresses
    args = _ARGS.pack(dtype, T, K, N, r, n, x, ldx, w, ldw, wt, 0, 0, lda, at, 0, 0, ldb, bt, indexed, 0, 0.0,
                      y, ldy, dX, K, dA, dB, 0, 0)
    need = _native.lib().gelim_adapter_workspace(args, bool(grad))
    if need < 0:
        _native.check(need, "adapter_matmul")
    return need


def _call(grad, dev, T, K, N, n, r, X, W, A, B, index, scale, Y, dX=None, dA=None, dB=None):
    """One native call; Y is the product's output, or the dY that the gradient reads."""
    X, ldx, turned = _stored(X)
    if turned:
        X = X.contiguous()
        ldx = K
    W, ldw, wt = _stored(W)
    A, lda, at = _stored(A)
    B, ldb, bt = _stored(B)
    ldy = Y.stride(0)
    factors, value = (scale.contiguous(), 0.0) if isinstance(scale, torch.Tensor) else (None, float(scale))
    if index is not None:
        index = index.contiguous()
    dtype = TYPES[X.dtype]
    xp, wp, yp = X.data_ptr(), W.data_ptr(), Y.data_ptr()
    wanted = (dX is not None, dA is not None, dB is not None) if grad else False
    ws_bytes = _workspace_bytes(wanted, dtype, T, K, N, r, n, ldx, ldw, wt, lda, at, ldb, bt, ldy,
                                xp & 15, wp & 15, yp & 15, index is not None)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    args = _ARGS.pack(dtype, T, K, N, r, n, xp, ldx, wp, ldw, wt, A.data_ptr(), A.stride(0), lda, at, B.data_ptr(),
                      B.stride(0), ldb, bt, 0 if index is None else index.data_ptr(),
                      0 if factors is None else factors.data_ptr(), value, yp, ldy,
                      0 if dX is None else dX.data_ptr(), K, 0 if dA is None else dA.data_ptr(),
                      0 if dB is None else dB.data_ptr(), ws.data_ptr(), ws_bytes)
    lib = _native.lib()
    fn, what = ((lib.gelim_adapter_matmul_grad, "adapter_matmul_grad") if grad else
                (lib.gelim_adapter_matmul, "adapter_matmul"))
    if torch.cuda.current_device() == dev.index:
        _native.check(fn(args, stream_handle(dev)), what)
    else:
        with torch.cuda.device(dev):
            _native.check(fn(args, stream_handle(dev)), what)


def adapter_matmul(X: torch.Tensor, W: torch.Tensor, A: torch.Tensor, B: torch.Tensor,
                   index: torch.Tensor | None = None, scale: float | torch.Tensor = 1.0,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """Y = X W + scale_i (X A_i) B_i with the adapter i = index[t] of each row.

    X (T, K), W (K, N), A (n, K, r), B (n, r, N): float32, bfloat16 or float16,
    all of one type.  Any strides; W, A and B are read in place if one of their
    last two dimensions has unit stride, so weights kept as (out, in) are
    passed as transposed views.  T may be 0; r is at most 256, n at most 65535.
    index (T,) int32: the adapter of each row, in any order; -1: the row has
    none; any other value outside [0, n) makes the row NaN.  None: n is 1 and
    every row has that adapter.
    scale: a number, or (n,) float32 on the device.
    out: (T, N) with unit column stride; no input begins or ends between its
    first and last element.
    Runs on the current stream; may be captured into a graph."""
    dev, T, K, N, n, r = _check(X, W, A, B, index, scale, (out,))
    fresh = out is None
    if fresh:
        out = X.new_empty((T, N))
    else:
        if out.dtype != X.dtype or out.device != dev:
            raise ValueError("out must have the type and device of X")
        if out.shape != (T, N) or (N > 1 and out.stride(1) != 1) or (T > 1 and out.stride(0) < N):
            raise ValueError("out must be a (T, N) tensor with unit column stride")
        if torch.is_grad_enabled() and out.requires_grad:
            raise ValueError("out is not recorded by autograd: call under torch.no_grad()")
        if any(_overlap(out, t) for t in (X, W, A, B, index, scale) if isinstance(t, torch.Tensor)):
            raise ValueError("out overlaps an input")
    if T:
        _call(False, dev, T, K, N, n, r, X, W, A, B, index, scale, out)
        if not fresh:
            increment_version(out)  # it may have been saved for a backward pass
    return out


def adapter_matmul_grad(dY: torch.Tensor, X: torch.Tensor, W: torch.Tensor, A: torch.Tensor, B: torch.Tensor,
                        index: torch.Tensor | None = None, scale: float | torch.Tensor = 1.0,
                        need: tuple[bool, bool, bool] = (True, True, True)
                        ) -> tuple[torch.Tensor | None, torch.Tensor | None, torch.Tensor | None]:
    """(dX, dA, dB) of `adapter_matmul` for the gradient dY (T, N) of its result.

    W is shared and frozen: it gets no gradient.  `need` says which of the
    three are wanted; the others are None and cost nothing.  dA and dB have
    the shapes of A and B, stored as those are (row-major, or transposed);
    an adapter without rows gets zeros.  Rows without an adapter (-1) add
    nothing to dA and dB; rows with an index outside [-1, n) have a NaN dX."""
    dev, T, K, N, n, r = _check(X, W, A, B, index, scale, (dY,))
    if dY.dtype != X.dtype:
        raise TypeError("dY must have the type of X")
    if dY.shape != (T, N) or dY.device != dev:
        raise ValueError("dY must be (T, N) on the device of X")
    if torch.is_grad_enabled() and dY.requires_grad:
        raise ValueError("adapter_matmul_grad has no gradient of its own: call it under torch.no_grad()")
    if N > 1 and dY.stride(1) != 1:
        dY = dY.contiguous()

    def like(F):
        rows, cols = F.shape[1:]
        if _stored(F)[2]:
            return torch.empty((n, cols, rows), dtype=F.dtype, device=dev).transpose(1, 2)
        return torch.empty(F.shape, dtype=F.dtype, device=dev)

    dX = torch.empty((T, K), dtype=X.dtype, device=dev) if need[0] else None
    dA = like(A) if need[1] else None
    dB = like(B) if need[2] else None
    if any(need):
        _call(True, dev, T, K, N, n, r, X, W, A, B, index, scale, dY, dX, dA, dB)
    return dX, dA, dB
