"""Adapter products and gradients where single bits, infinities and unused adapters decide."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def long_value(dtype):
    """Three values whose sum of products with `ones` needs 21 (bf16) or 24 bits, more than two values of the type hold:
    v . ones = 1 + a + b, v . less = 1 + a, exact in fp32 in any order."""
    small, least = (2.0 ** -9, 2.0 ** -20) if dtype == torch.bfloat16 else (2.0 ** -12, 2.0 ** -23)
    half = math.sqrt(least) if dtype == torch.bfloat16 else 2.0 ** -11
    return (1.0, small, half), (1.0, 1.0, least / half), least


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("r", [2, 8, 16, 40, 256])
@pytest.mark.parametrize("T", [64, 65, 300, 2050])
def test_low_rank_sums_are_held_in_32_bits(gelim, cuda, T, r, dtype):
    """Y = 1024 (S_0 - S_last) with S_0 = 1 + a + b, S_last = 1 + a: exactly 1024 b, as every sum on the way is a
    multiple of b that 24 bits hold.  The same for dX, whose factors change places."""
    K = N = 72
    v, ones, least = long_value(dtype)
    at = [0, 17, 70]
    U, F, G = torch.zeros(T, K), torch.zeros(1, K, r), torch.zeros(1, r, N)
    U[:, at] = torch.tensor(v)
    F[0, at, 0] = torch.tensor(ones)
    F[0, at, r - 1] = torch.tensor(ones[:2] + (0.0,))
    G[0, 0], G[0, r - 1] = 1024.0, -1024.0
    U, F, G, W = (x.to(dtype).to(cuda) for x in (U, F, G, torch.zeros(K, N)))
    assert (gelim.ops.adapter_matmul(U, W, F, G) == 1024 * least).all()
    FT, GT = F.transpose(1, 2), G.transpose(1, 2)
    dX = gelim.ops.adapter_matmul_grad(U, torch.zeros_like(U), W, GT, FT, need=(True, False, False))[0]
    assert (dX == 1024 * least).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("r", [1, 16, 40, 256])
@pytest.mark.parametrize("T", [2, 128, 129, 700])
def test_factor_gradients_of_32_bit_sums(gelim, cuda, T, r, dtype):
    """Two rows of opposite sign whose D (or S) differ by their last bit: the gradient is 1024 times that bit."""
    K = N = 72
    v, ones, least = long_value(dtype)
    at = [0, 17, 70]
    low, other, factor = torch.zeros(T, K), torch.zeros(T, N), torch.zeros(1, K, r)
    low[0, at], low[1, at] = torch.tensor(v), torch.tensor(v[:2] + (0.0,))
    other[0], other[1] = 1024.0, -1024.0
    factor[0, at] = torch.tensor(ones)[:, None]
    low, other, factor, W = (x.to(dtype).to(cuda) for x in (low, other, factor, torch.zeros(K, N)))
    zero = torch.zeros_like(factor)
    dB = gelim.ops.adapter_matmul_grad(other, low, W, factor, zero.transpose(1, 2))[2]
    assert (dB == 1024 * least).all()
    dA = gelim.ops.adapter_matmul_grad(low, other, W, zero, factor.transpose(1, 2))[1]
    assert (dA == 1024 * least).all()


def same_kind(got, ref):
    """Infinities of the same sign and NaN in the same places, finite values elsewhere."""
    got, ref = got.detach().cpu().double(), ref
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    where = torch.isinf(ref)
    assert torch.equal(torch.isinf(got), where) and torch.equal(got[where], ref[where])


def mm(a, b):
    """a @ b with each sum's terms as they are: no zeros of a padded tile beside an infinity."""
    return (a.unsqueeze(-1) * b.unsqueeze(-3)).sum(-2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("r", [1, 3, 16, 17])
@pytest.mark.parametrize("T", [7, 64, 65, 130, 300])
def test_infinities_are_what_the_formula_makes_of_them(gelim, cuda, T, r, dtype):
    """An infinite weight, factor or input, on either side of the sizes at which other kernels take over.  Small whole
    numbers, so that sums of a few bits (one part of the type holds them, the others are zero) stand beside infinities."""
    K, N = 24, 40
    g = torch.Generator().manual_seed(100 * T + r)

    def whole(*shape):
        v = torch.randint(1, 3, shape, generator=g) * (torch.randint(0, 2, shape, generator=g) * 2 - 1)
        return v.double()

    for k in range(5):
        X, W, A, B, dY = whole(T, K), whole(K, N), whole(2, K, r), whole(2, r, N), whole(T, N)
        index = torch.randint(-1, 2, (T,), generator=g)
        index[T - 1] = 0
        inf = float("inf") if k % 2 else -float("inf")
        if k == 0:
            B[0, r - 1, 5] = inf
        elif k == 1:
            A[0, 3, 0] = inf
        elif k == 2:
            X[T - 1, 7] = inf
        elif k == 3:
            dY[T - 1, 9] = inf
        else:
            W[3, 5] = inf
        args = [v.to(dtype).to(cuda) for v in (X, W, A, B)] + [index.int().to(cuda), 2.0]
        Y, dX = mm(X, W), mm(dY, W.t())
        dA, dB = torch.zeros_like(A), torch.zeros_like(B)
        for i in range(2):
            t = index == i
            S, D = mm(X[t], A[i]), mm(dY[t], B[i].t())
            Y[t] += 2 * mm(S, B[i])
            dX[t] += 2 * mm(D, A[i].t())
            dA[i], dB[i] = 2 * mm(X[t].t(), D), 2 * mm(S.t(), dY[t])
        same_kind(gelim.ops.adapter_matmul(*args), Y)
        for got, ref in zip(gelim.ops.adapter_matmul_grad(dY.to(dtype).to(cuda), *args), (dX, dA, dB)):
            same_kind(got, ref)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [40, 128, 129, 700, 9000])
@pytest.mark.parametrize("n", [5, 30])
def test_scales_of_adapters_without_rows(gelim, cuda, T, n, dtype):
    """An adapter that no row has gets zeros whatever its scale is: a slot not filled yet, or alpha / 0."""
    K, N, r = 72, 136, 12
    g = torch.Generator().manual_seed(T + n)
    X, W, A, B, dY = (torch.randn(s, generator=g).to(dtype).to(cuda) for s in
                      ((T, K), (K, N), (n, K, r), (n, r, N), (T, N)))
    index = (torch.arange(T) % 3 * 2 - 1).clamp(max=n - 1).int().to(cuda)  # -1, 1 and 3
    scale = torch.full((n,), 0.5, device=cuda)
    want = gelim.ops.adapter_matmul_grad(dY, X, W, A, B, index, scale)
    wantY = gelim.ops.adapter_matmul(X, W, A, B, index, scale)
    for bad in (math.nan, math.inf, -math.inf):
        scale[[0, 2, 4]] = bad
        scale[5:] = bad
        assert torch.equal(gelim.ops.adapter_matmul(X, W, A, B, index, scale), wantY)
        got = gelim.ops.adapter_matmul_grad(dY, X, W, A, B, index, scale)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert not got[1][0].any() and not got[2][4].any() and not got[1][5:].any()
        norm = gelim.ops.clip_global_norm([got[1], got[2]], 1.0)
        assert torch.isfinite(norm)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T, n, used", [(129, 500, 129), (200, 3000, 7), (400, 401, 400), (700, 900, 3), (1500, 40, 40)])
def test_pieces_of_many_adapters(gelim, cuda, T, n, used, dtype):
    """More adapters than rows, most with one row or none, a few with several pieces."""
    from test_gpu_adapter import check, make, ref_grad, ref_product

    K, N, r = 72, 40, 5
    X, W, A, B, index, scale = make(cuda, T, K, N, r, n, dtype)
    g = torch.Generator().manual_seed(T + n)
    some = torch.randperm(n, generator=g)[:used]
    which = torch.cat([some, some[torch.randint(0, min(3, used), (T,), generator=g)]])[:T]
    index = which[torch.randperm(T, generator=g)].int().to(cuda)
    index[T // 3] = -1
    args = X, W, A, B, index, scale
    check(gelim.ops.adapter_matmul(*args), *ref_product(*args, device=cuda))
    dY = torch.randn(T, N, generator=g).to(dtype).to(cuda)
    for v, t in zip(gelim.ops.adapter_matmul_grad(dY, *args), ref_grad(dY, *args, device=cuda)):
        check(v, *t)


def test_a_scale_that_requires_gradients_is_refused(gelim, cuda):
    X, W, A, B = (torch.randn(s, device=cuda).bfloat16() for s in ((6, 32), (32, 40), (2, 32, 4), (2, 4, 40)))
    index, scale = torch.zeros(6, dtype=torch.int32, device=cuda), torch.ones(2, device=cuda, requires_grad=True)
    with pytest.raises(ValueError, match="autograd"):
        gelim.ops.adapter_matmul(X, W, A, B, index, scale)
    with pytest.raises(ValueError, match="autograd"):
        gelim.ops.adapter_matmul_grad(torch.zeros(6, 40, device=cuda).bfloat16(), X, W, A, B, index, scale)
    with torch.no_grad():
        Y = gelim.ops.adapter_matmul(X, W, A, B, index, scale)
    assert torch.equal(Y, gelim.ops.adapter_matmul(X, W, A, B, index, scale.detach()))


def test_forward_mode_tangents_are_refused(gelim, cuda):
    from torch.autograd import forward_ad

    X, W, A, B = (torch.randn(s, device=cuda).bfloat16() for s in ((6, 32), (32, 40), (1, 32, 4), (1, 4, 40)))
    dY, scale = torch.zeros(6, 40, device=cuda).bfloat16(), torch.ones(1, device=cuda)
    want = gelim.ops.adapter_matmul(X, W, A, B, scale=scale)
    with forward_ad.dual_level(), torch.no_grad():
        for k in range(5):
            args = [X, W, A, B, None, scale]
            k += k == 4
            args[k] = forward_ad.make_dual(args[k], torch.ones_like(args[k]))
            with pytest.raises(ValueError, match="forward-mode"):
                gelim.ops.adapter_matmul(*args)
            with pytest.raises(ValueError, match="forward-mode"):
                gelim.ops.adapter_matmul_grad(dY, *args)
            with pytest.raises(ValueError, match="forward-mode"):
                gelim.ops.clip_global_norm([A.clone(), args[k]], 1.0)
        dual = forward_ad.make_dual(dY, torch.ones_like(dY))
        with pytest.raises(ValueError, match="forward-mode"):
            gelim.ops.adapter_matmul_grad(dual, X, W, A, B)
        with pytest.raises(ValueError, match="forward-mode"):
            gelim.ops.adapter_matmul(X, W, A, B, out=dual)
        with pytest.raises(ValueError, match="forward-mode"):
            gelim.ops.clip_global_norm([A], 1.0, out=[forward_ad.make_dual(A.clone(), A.clone())])
        assert torch.equal(gelim.ops.adapter_matmul(X, W, A, B, scale=scale), want)  # others may be duals meanwhile


def test_autograd_sees_what_is_written(gelim, cuda):
    """A tensor saved for a backward pass and then written by a call: the backward pass must not go on with the new
    values, as after any in-place operation."""
    X, W, A, B = (torch.randn(s, device=cuda) for s in ((70, 32), (32, 40), (1, 32, 4), (1, 4, 40)))

    def saved():
        y = torch.randn(70, 40, device=cuda)
        p = torch.ones(70, 40, device=cuda, requires_grad=True)
        return y, (p * y).sum()

    y, loss = saved()
    gelim.ops.adapter_matmul(X, W, A, B, out=y)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    for apart in (False, True):
        y, loss = saved()
        gelim.ops.clip_global_norm([X.clone(), W.clone() if apart else y], 1e-3,
                                   out=[torch.empty_like(X), y[:32]] if apart else None)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    y, loss = saved()
    gelim.ops.clip_global_norm([y], math.inf)  # only measures
    gelim.ops.clip_global_norm([y], 1.0, out=[torch.empty_like(y)])
    gelim.ops.adapter_matmul(X, W, A, B)
    loss.backward()
    with torch.inference_mode():  # such tensors have no version
        y = torch.randn(70, 40, device=cuda)
        gelim.ops.clip_global_norm([y], 1.0)
        gelim.ops.adapter_matmul(X, W, A, B, out=y)


def test_clipped_copies_have_their_inputs_shapes(gelim, cuda):
    a, b = torch.ones(2, 3, device=cuda), torch.ones(4, device=cuda)
    for out in ([torch.empty(3, 2, device=cuda), torch.empty_like(b)], [torch.empty(6, device=cuda), torch.empty_like(b)],
                [torch.empty_like(a), torch.empty(2, 2, device=cuda)], [torch.empty_like(b), torch.empty_like(a)]):
        with pytest.raises(ValueError, match="same type and shape"):
            gelim.ops.clip_global_norm([a, b], 1.0, out=out)
    out = [torch.empty_like(a), torch.empty_like(b)]
    gelim.ops.clip_global_norm([a, b], 1.0, out=out)
    assert torch.equal(out[0].flatten()[:4], out[1])


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("max_norm", [26.69, 19.71, 21.25, 39.42, 30.23, 36.77])
@pytest.mark.parametrize("dtype", DTYPES)
def test_clipping_rounds_alike_at_every_place(gelim, cuda, dtype, max_norm, apart):
    """Equal values have equal results, whether they stand in a whole pack of 16 bytes or at a tensor's end.  These norms
    have factors for which 8 to 12 of the products in fp16 depend on whether they are rounded to fp32 before."""
    v = torch.randn(4096, generator=torch.Generator().manual_seed(3)).to(dtype).to(cuda)
    small = [torch.cat([v[:8], v[k:k + 1]]) for k in range(v.numel())]
    tensors = [v.clone()] + small
    out = [torch.empty_like(t) for t in tensors] if apart else tensors
    gelim.ops.clip_global_norm(tensors, max_norm, out=out if apart else None)
    assert torch.equal(torch.stack([o[8] for o in out[1:]]), out[0])


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_factor_below_the_normal_numbers(gelim, cuda, dtype, apart):
    """Norms so large that max_norm / norm is subnormal in fp32: the results are normal all the same and have the
    accuracy that the others have.  Tolerance: the rounding of the factor and of the product to fp32 and of the result to
    its type (2^-24 each and eps / 2), and half a step of the subnormal numbers of fp32, 2^-150, and of the type."""
    g = torch.Generator().manual_seed(7)
    for size, max_norm in ((1e38, 1e-3), (3e37, 1e-7), (1e30, 1e-14), (1e38, 1e-12)):
        a = (torch.rand(4000, generator=g) + 0.5).mul(size).to(dtype).to(cuda)
        a[1], a[2] = 2.0 ** -3 * a[1], 1.0
        norm = math.sqrt(math.fsum(a.double().square().tolist()))
        f = max_norm / (norm + 1e-6)
        assert f < 2.0 ** -126
        out = torch.empty_like(a) if apart else a.clone()
        src = a if apart else out
        gelim.ops.clip_global_norm([src], max_norm, out=[out] if apart else None)
        want = a.double() * f
        tol = (torch.finfo(dtype).eps / 2 + 2.0 ** -23) * want.abs() + 2.0 ** -150
        tol += torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
        assert ((out.double() - want).abs() <= tol).all()
