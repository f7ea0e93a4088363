"""Low-rank adapters beside a shared projection and their gradients, against the formulas in 64 bits.

Tolerance of an element: one rounding of the result (eps / 2 of its type), the
fp32 sums (each of the terms + 16 roundings counted with a full 2^-23 of the
sum of absolute values), and X A_i entering the second product with 16 bits
(2^-16 of that product's absolute values; exact in fp32)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
# T, K, N, r, n: one token to several tiles, odd sizes, tails in every dimension
SHAPES = [(1, 1, 1, 1, 1), (1, 17, 33, 3, 2), (1, 2048, 512, 8, 1), (5, 64, 128, 8, 3), (13, 255, 301, 12, 5),
          (16, 520, 1032, 16, 9), (33, 1000, 72, 5, 40), (64, 256, 512, 16, 64), (65, 128, 96, 4, 7),
          (100, 1024, 1024, 8, 1), (130, 520, 264, 12, 5), (256, 264, 256, 32, 3), (300, 1000, 777, 9, 6),
          (513, 136, 520, 64, 2), (257, 512, 2048, 100, 4), (70, 96, 160, 256, 2), (700, 2050, 1030, 17, 3)]


def make(dev, T, K, N, r, n, dtype, layout="kn", rows="mixed", seed=0):
    g = torch.Generator().manual_seed(seed * 1000 + T * 7 + K * 5 + N * 3 + r + n)

    def t(*shape, size=1.0):
        if layout == "nk":
            return (torch.randn(*shape[:-2], shape[-1], shape[-2], generator=g) * size).to(dtype).to(dev).transpose(-1, -2)
        return (torch.randn(*shape, generator=g) * size).to(dtype).to(dev)

    X = (torch.randn(T, K, generator=g)).to(dtype).to(dev)
    W, A, B = t(K, N, size=K ** -0.5), t(n, K, r, size=K ** -0.5), t(n, r, N, size=r ** -0.5)
    if rows == "mixed":
        index = torch.randint(-1, n, (T,), generator=g)
    elif rows == "runs":
        index = torch.sort(torch.randint(-1, n, (T,), generator=g))[0].flip(0)
    elif rows == "none":
        index = torch.full((T,), -1)
    else:
        index = torch.zeros(T)
    scale = torch.linspace(0.5, 2.0, n).to(dev)
    return X, W, A, B, index.int().to(dev), scale


def ref_product(X, W, A, B, index, scale, device="cpu"):
    """(result, tolerance) in 64 bits."""
    dtype = X.dtype
    X, W, A, B, index = (v.detach().to(device) for v in (X, W, A, B, index))
    X, W, A, B = (v.double() for v in (X, W, A, B))
    scale = torch.full((len(A),), float(scale), dtype=torch.float64) if not isinstance(scale, torch.Tensor) \
        else scale.to(device).double()
    Y, total = X @ W, X.abs() @ W.abs()
    low = torch.zeros_like(Y)
    for i in range(len(A)):
        rows = index == i
        Y[rows] += scale[i] * (X[rows] @ A[i]) @ B[i]
        low[rows] = scale[i].abs() * ((X[rows].abs() @ A[i].abs()) @ B[i].abs())
    split = 0.0 if dtype == torch.float32 else 2.0 ** -16
    terms = X.shape[1] + A.shape[2]
    tol = torch.finfo(dtype).eps / 2 * Y.abs() + (terms + 16) * 2.0 ** -23 * (total + low) + split * low
    return Y, tol + torch.finfo(dtype).smallest_normal


def check(got, ref, tol, scale=1.0):
    got = got.detach().to(ref.device).double()
    assert got.shape == ref.shape
    assert torch.isfinite(got).all()
    off = ((got - ref).abs() / tol).max().item() if got.numel() else 0.0
    assert off <= scale, f"off by {off} times the tolerance"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("shape", SHAPES)
def test_product(gelim, cuda, shape, layout, dtype):
    args = make(cuda, *shape, dtype, layout)
    check(gelim.ops.adapter_matmul(*args), *ref_product(*args))


# sizes for which each tile shape is chosen, whole and with the sum cut, with tails in every dimension; a sum of fewer
# tiles than are kept in LDS, and of a number of them that is no multiple of that
TILES = [(2050, 72, 4104, 40, 3), (2050, 264, 4104, 16, 9), (2303, 520, 4104, 8, 1), (2050, 72, 2056, 33, 5),
         (1030, 136, 4104, 16, 4), (1500, 200, 4104, 64, 2), (2050, 4104, 1032, 16, 3), (1030, 4104, 2056, 24, 7),
         (513, 72, 4104, 16, 3), (1030, 392, 2056, 9, 5), (513, 4104, 2056, 64, 3), (257, 4104, 4104, 16, 20),
         (130, 1032, 264, 128, 4), (70, 2056, 520, 256, 3)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("rows", ["mixed", "runs"])
@pytest.mark.parametrize("shape", TILES)
def test_tiles(gelim, cuda, shape, rows, layout, dtype):
    args = make(cuda, *shape, dtype, layout, rows)
    check(gelim.ops.adapter_matmul(*args), *ref_product(*args, device=cuda))
    T, K, N, r, n = shape
    dY = torch.randn(T, N, generator=torch.Generator().manual_seed(2)).to(dtype).to(cuda)
    for v, t in zip(gelim.ops.adapter_matmul_grad(dY, *args), ref_grad(dY, *args, device=cuda)):
        check(v, *t)


def shifted(v):
    """v one element behind a multiple of 16 bytes."""
    return torch.cat([v.new_zeros(1), v.reshape(-1)])[1:].view(v.shape)


# one operand of three at another address than the others: the tile is chosen by what is copied, and so is the workspace
@pytest.mark.parametrize("grad, which, T, K, N, layout", [
    (False, "W", 2973, 852, 680, "kn"), (False, "W", 943, 1120, 732, "kn"), (False, "Y", 630, 1092, 1136, "kn"),
    (False, "Y", 1013, 1112, 664, "kn"), (True, "X", 2983, 448, 852, "nk"), (True, "X", 1551, 796, 856, "nk"),
    (True, "W", 2099, 1200, 852, "nk"), (True, "Y", 2686, 860, 832, "nk")])
def test_addresses(gelim, cuda, grad, which, T, K, N, layout):
    X, W, A, B, index, scale = make(cuda, T, K, N, 16, 2, torch.float32, layout)
    X = shifted(X) if which == "X" else X
    if which == "W":
        W = shifted(W) if layout == "kn" else shifted(W.t()).t()
    args = X, W, A, B, index, scale
    if not grad:
        out = shifted(X.new_zeros(T, N)) if which == "Y" else None
        check(gelim.ops.adapter_matmul(*args, out=out), *ref_product(*args, device=cuda))
        return
    dY = torch.randn(T, N, generator=torch.Generator().manual_seed(2)).to(cuda)
    dY = shifted(dY) if which == "Y" else dY
    for v, t in zip(gelim.ops.adapter_matmul_grad(dY, *args), ref_grad(dY, *args, device=cuda)):
        check(v, *t)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 17, 40, 64])
@pytest.mark.parametrize("K, N", [(1, 1), (3, 7), (7, 3), (8, 8), (31, 9), (33, 127), (511, 129), (4097, 130)])
@pytest.mark.parametrize("layout", ["kn", "nk"])
def test_few_rows_of_odd_sizes(gelim, cuda, T, K, N, layout, dtype):
    args = make(cuda, T, K, N, 5, 3, dtype, layout)
    check(gelim.ops.adapter_matmul(*args), *ref_product(*args))


@pytest.mark.parametrize("rows", ["runs", "none", "all"])
@pytest.mark.parametrize("T", [7, 64, 65, 600])
def test_product_rows(gelim, cuda, T, rows):
    args = make(cuda, T, 256, 384, 16, 5, torch.bfloat16, rows=rows)
    check(gelim.ops.adapter_matmul(*args), *ref_product(*args))


@pytest.mark.parametrize("T", [3, 200])
def test_number_as_scale_and_no_index(gelim, cuda, T):
    X, W, A, B, index, _ = make(cuda, T, 128, 136, 8, 1, torch.float16, rows="all")
    Y = gelim.ops.adapter_matmul(X, W, A, B, scale=-0.75)
    check(Y, *ref_product(X, W, A, B, index, -0.75))
    assert torch.equal(Y, gelim.ops.adapter_matmul(X, W, A, B, index, torch.full((1,), -0.75, device=cuda)))


@pytest.mark.parametrize("T", [9, 300])
@pytest.mark.parametrize("dtype", DTYPES)
def test_row_outside_the_adapters_is_nan(gelim, cuda, T, dtype):
    args = list(make(cuda, T, 72, 100, 4, 3, dtype))
    args[4] = args[4].clone()
    args[4][1], args[4][5], args[4][7] = 3, -2, 2 ** 31 - 1
    Y = gelim.ops.adapter_matmul(*args)
    bad = torch.zeros(T, dtype=torch.bool)
    bad[[1, 5, 7]] = True
    assert torch.isnan(Y[bad.to(cuda)]).all()
    ref, tol = ref_product(*args)
    check(Y.cpu()[~bad], ref[~bad], tol[~bad])
    dX, dA, dB = gelim.ops.adapter_matmul_grad(Y.nan_to_num(0.0), *args)
    assert torch.isnan(dX[bad.to(cuda)]).all() and torch.isfinite(dX[~bad.to(cuda)]).all()
    assert torch.isfinite(dA).all() and torch.isfinite(dB).all()


@pytest.mark.parametrize("T", [16, 128, 520])
@pytest.mark.parametrize("dtype", DTYPES)
def test_what_a_row_does_not_use_does_not_reach_it(gelim, cuda, T, dtype):
    """Infinities and NaN in another adapter, or in another row, stay there."""
    X, W, A, B, index, scale = make(cuda, T, 136, 264, 16, 4, dtype)
    A[1], B[1] = float("nan"), float("inf")
    B[2, 3, 5] = float("-inf")
    X[3] = float("nan")
    X[4, 7] = float("inf")
    index[3], index[4], index[5:9] = 0, 3, torch.tensor([0, 1, 2, 3], dtype=torch.int32)
    Y = gelim.ops.adapter_matmul(X, W, A, B, index, scale).cpu()
    clean = (index != 1).cpu()
    clean[3] = clean[4] = False
    only = clean & (index != 2).cpu()
    fine = [v.clone() for v in (X, W, A, B)]
    fine[0][3] = fine[0][4] = 0
    fine[2][1] = fine[3][1] = 0
    fine[3][2, 3, 5] = 0
    ref, tol = ref_product(*fine, index, scale)
    check(Y[only], ref[only], tol[only])
    two = (index == 2).cpu() & clean
    keep = torch.arange(264) != 5
    check(Y[two][:, keep], ref[two][:, keep], tol[two][:, keep])
    assert not torch.isfinite(Y[two][:, 5]).any()
    assert torch.isnan(Y[3]).all() and torch.isnan(Y[(index == 1).cpu()]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T, K, N", [(2050, 264, 4104), (1030, 136, 4104), (513, 72, 4104), (257, 4104, 1032)])
def test_rows_of_large_tiles_stay_apart(gelim, cuda, T, K, N, dtype):
    """NaN and infinities in a row or in an adapter, where a wave's rows have one adapter, several, and none."""
    X, W, A, B, index, scale = make(cuda, T, K, N, 16, 4, dtype, rows="runs")
    index[40:70] = torch.arange(30, device=cuda).int() % 4
    want = gelim.ops.adapter_matmul(X, W, A, B, index, scale)
    dY = torch.randn(T, N, generator=torch.Generator().manual_seed(5)).to(dtype).to(cuda)
    grads = gelim.ops.adapter_matmul_grad(dY, X, W, A, B, index, scale)
    rows = torch.tensor([0, 41, 63, 64, T // 2, T - 1], device=cuda)
    clean = torch.ones(T, dtype=torch.bool, device=cuda)
    clean[rows] = False
    X2, dY2 = X.clone(), dY.clone()
    X2[rows[::2]], X2[rows[1::2], 3] = float("nan"), float("inf")
    dY2[rows] = float("nan")
    Y = gelim.ops.adapter_matmul(X2, W, A, B, index, scale)
    assert torch.equal(Y[clean], want[clean]) and not torch.isfinite(Y[rows]).any()
    dX = gelim.ops.adapter_matmul_grad(dY2, X, W, A, B, index, scale)[0]
    assert torch.equal(dX[clean], grads[0][clean]) and torch.isnan(dX[rows]).all()
    A2, B2 = A.clone(), B.clone()
    A2[2], B2[2] = float("nan"), float("inf")
    Y = gelim.ops.adapter_matmul(X, W, A2, B2, index, scale)
    other = index != 2
    assert torch.equal(Y[other], want[other]) and torch.isnan(Y[~other]).all()
    got = gelim.ops.adapter_matmul_grad(dY, X, W, A2, B2, index, scale)
    assert torch.equal(got[0][other], grads[0][other])
    for a, b in zip(got[1:], grads[1:]):
        assert torch.equal(a[[0, 1, 3]], b[[0, 1, 3]]) and torch.isnan(a[2]).all()
    # rows with no adapter, whatever they hold, add nothing to the gradients
    index[rows] = -1
    fine = gelim.ops.adapter_matmul_grad(torch.where(clean[:, None], dY, 0), X, W, A, B, index, scale)
    got = gelim.ops.adapter_matmul_grad(dY2, X2, W, A, B, index, scale)
    for a, b in zip(got[1:], fine[1:]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [6, 150])
def test_strides(gelim, cuda, T, dtype):
    """Slices of larger matrices, transposed X, a repeated row, adapters picked with a step, a strided index."""
    K, N, r, n = 200, 184, 8, 3
    g = torch.Generator().manual_seed(T)
    big = torch.randn(400, 500, generator=g).to(dtype).to(cuda)
    fac = (torch.randn(6, 260, 260, generator=g) * 0.1).to(dtype).to(cuda)
    W = big[100:100 + K, 33:33 + N]
    A, B = fac[::2, 3:3 + K, 5:5 + r], fac[1::2, 7:7 + r, 1:1 + N]
    index = torch.randint(-1, n, (2 * T,), generator=g).int().to(cuda)[::2]
    scale = torch.rand(6, generator=g).to(cuda)[::2]
    for X in (big[5:5 + T, 9:9 + K], big[:K, 7:7 + T].t(), big[3, 50:50 + K].expand(T, K)):
        for W_ in (W, big[20:20 + N, 8:8 + K].t(), big.as_strided((K, N), (2 * N, 2))):
            args = (X, W_, A, B, index, scale)
            check(gelim.ops.adapter_matmul(*args), *ref_product(*args))
    # the factors stored transposed, and a result inside a larger matrix
    A2, B2 = fac[::2, 3:3 + r, 5:5 + K].transpose(1, 2), fac[1::2, 7:7 + N, 1:1 + r].transpose(1, 2)
    room = torch.full((T + 2, N + 9), 7.0, dtype=dtype, device=cuda)
    args = (big[5:5 + T, 9:9 + K], W, A2, B2, index, scale)
    Y = gelim.ops.adapter_matmul(*args, out=room[1:1 + T, 4:4 + N])
    check(Y, *ref_product(*args))
    room[1:1 + T, 4:4 + N] = 7.0
    assert (room == 7.0).all()


def test_no_rows(gelim, cuda):
    X, W, A, B, index, scale = make(cuda, 4, 64, 48, 4, 2, torch.bfloat16)
    Y = gelim.ops.adapter_matmul(X[:0], W, A, B, index[:0], scale)
    assert Y.shape == (0, 48)
    dX, dA, dB = gelim.ops.adapter_matmul_grad(Y, X[:0], W, A, B, index[:0], scale)
    assert dX.shape == (0, 64) and not dA.any() and not dB.any()


@pytest.mark.parametrize("T", [1, 20, 64, 400])
@pytest.mark.parametrize("dtype", DTYPES)
def test_same_bits_every_time(gelim, cuda, T, dtype):
    args = make(cuda, T, 520, 392, 16, 7, dtype)
    Y = gelim.ops.adapter_matmul(*args)
    grads = gelim.ops.adapter_matmul_grad(Y, *args)
    for _ in range(3):
        assert torch.equal(Y, gelim.ops.adapter_matmul(*args))
        for a, b in zip(grads, gelim.ops.adapter_matmul_grad(Y, *args)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T", [12, 200])
def test_large_and_small_low_rank_parts(gelim, cuda, T, dtype):
    """X A_i beyond the range of fp16, and far below its smallest normal number."""
    X, W, A, B, index, _ = make(cuda, T, 256, 128, 8, 2, dtype, rows="all")
    index[1::2] = 1
    big = A.clone()
    big[0] *= 2.0 ** 13
    big[1] *= 2.0 ** -8
    X16 = X * 16
    Bs = B * 2.0 ** -12
    args = (X16, W, big, Bs, index, 1.0)
    ref, tol = ref_product(*args)
    # beside the rule at the top: B itself has subnormal entries in fp16, exact all the same
    check(gelim.ops.adapter_matmul(*args), ref, tol)
    small = A * 2.0 ** -12
    args = (X * 2.0 ** -6, W * 2.0 ** -8, small, B, index, 1.0)
    ref, tol = ref_product(*args)
    check(gelim.ops.adapter_matmul(*args), ref, tol + 2.0 ** -25)  # half a step of fp16's subnormal numbers


def ref_grad(dY, X, W, A, B, index, scale, device="cpu"):
    dtype = X.dtype
    dY, X, W, A, B, index = (v.detach().to(device) for v in (dY, X, W, A, B, index))
    dY, X, W, A, B = (v.double() for v in (dY, X, W, A, B))
    T, K = X.shape
    n, _, r = A.shape
    N = W.shape[1]
    scale = torch.full((n,), float(scale), dtype=torch.float64) if not isinstance(scale, torch.Tensor) \
        else scale.to(device).double()
    eps, u = torch.finfo(dtype).eps / 2, 2.0 ** -23
    split = 0.0 if dtype == torch.float32 else 2.0 ** -16
    tiny = torch.finfo(dtype).smallest_normal
    dX, tX = dY @ W.t(), dY.abs() @ W.abs().t()
    lX = torch.zeros_like(dX)
    dA, dB = torch.zeros_like(A), torch.zeros_like(B)
    tA, tB = torch.zeros_like(A), torch.zeros_like(B)
    for i in range(n):
        rows = index == i
        x, y = X[rows], dY[rows]
        D, S = y @ B[i].t(), x @ A[i]
        aD, aS = y.abs() @ B[i].abs().t(), x.abs() @ A[i].abs()
        dX[rows] += scale[i] * D @ A[i].t()
        lX[rows] = scale[i].abs() * aD @ A[i].abs().t()
        dA[i] = scale[i] * x.t() @ D
        dB[i] = scale[i] * S.t() @ y
        m = int(rows.sum())
        tA[i] = scale[i].abs() * (x.abs().t() @ aD) * ((m + N + 16) * u + split)
        tB[i] = scale[i].abs() * (aS.t() @ y.abs()) * ((m + K + 16) * u + split)
    tX = eps * dX.abs() + (N + r + 16) * u * (tX + lX) + split * lX + tiny
    return (dX, tX), (dA, eps * dA.abs() + tA + tiny), (dB, eps * dB.abs() + tB + tiny)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("shape", SHAPES)
def test_gradient(gelim, cuda, shape, layout, dtype):
    args = make(cuda, *shape, dtype, layout)
    g = torch.Generator().manual_seed(1)
    dY = torch.randn(shape[0], shape[2], generator=g).to(dtype).to(cuda)
    got = gelim.ops.adapter_matmul_grad(dY, *args)
    for v, t, like in zip(got, ref_grad(dY, *args), (args[0], args[2], args[3])):
        check(v, *t)
        assert like is args[0] or v.stride() == like.stride() or 1 in like.shape
        assert v.shape == like.shape and v.dtype == dtype


@pytest.mark.parametrize("rows", ["runs", "none", "all"])
@pytest.mark.parametrize("T", [7, 64, 65, 1200])
def test_gradient_rows(gelim, cuda, T, rows):
    args = make(cuda, T, 256, 384, 16, 5, torch.bfloat16, rows=rows)
    dY = torch.randn(T, 384, device=cuda).bfloat16()
    for v, t in zip(gelim.ops.adapter_matmul_grad(dY, *args), ref_grad(dY, *args)):
        check(v, *t)


def test_gradient_parts_alone(gelim, cuda):
    args = make(cuda, 90, 128, 200, 8, 3, torch.bfloat16)
    dY = torch.randn(90, 200, device=cuda).bfloat16()
    whole = gelim.ops.adapter_matmul_grad(dY, *args)
    for need in [(True, False, False), (False, True, False), (False, False, True), (False, True, True),
                 (False, False, False)]:
        part = gelim.ops.adapter_matmul_grad(dY, *args, need=need)
        for a, b, wanted in zip(part, whole, need):
            assert torch.equal(a, b) if wanted else a is None


@pytest.mark.parametrize("T", [24, 300])
def test_gradient_against_differences(gelim, cuda, T):
    """The product is linear in X, in A and in B, so a central difference of any step has no error but rounding:
    with values of size 1 the sum <dY, Y> has T N terms and each Y the rounding that the product's tolerance counts."""
    X, W, A, B, index, scale = make(cuda, T, 96, 80, 8, 3, torch.float32)
    g = torch.Generator().manual_seed(5)
    dY = torch.randn(T, 80, generator=g).to(cuda)
    dX, dA, dB = gelim.ops.adapter_matmul_grad(dY, X, W, A, B, index, scale)
    for k, grad in ((0, dX), (2, dA), (3, dB)):
        V = torch.randn(grad.shape, generator=g).to(cuda)
        up, down = [X, W, A, B], [X, W, A, B]
        up[k], down[k] = up[k] + V, down[k] - V
        ups, downs = (gelim.ops.adapter_matmul(*v, index, scale).cpu().double() for v in (up, down))
        diff = (dY.cpu().double() * (ups - downs)).sum() / 2
        tol = (dY.cpu().double().abs() * (ref_product(*up, index, scale)[1] + ref_product(*down, index, scale)[1])).sum() / 2
        # up and down themselves are rounded to fp32: 2^-24 of every entry of the moved operand, on both sides
        slack = 2.0 ** -24 * ((up[k].abs() + down[k].abs()).cpu().double() * grad.abs().cpu().double()).sum() / 2
        slack += 2.0 ** -23 * (grad.abs() * V.abs()).double().sum().item() * 128  # the gradient's own rounding
        assert abs(diff - (grad.double() * V.double()).sum().item()) <= tol + slack


@pytest.mark.parametrize("T", [8, 64, 300])
def test_captured_and_replayed(gelim, cuda, T):
    """Two captured graphs with eager calls between their replays; new inputs in the same tensors."""
    sets = [make(cuda, T, 256, 200, 8, 4, torch.bfloat16, seed=s) for s in range(4)]
    dYs = [torch.randn(T, 200, device=cuda).bfloat16() for _ in range(4)]
    held = [[v.clone() for v in sets[0]] + [dYs[0].clone()] for _ in range(2)]
    graphs, outs = [], []

    def step(h):
        Y = gelim.ops.adapter_matmul(*h[:6])
        grads = list(gelim.ops.adapter_matmul_grad(h[6], *h[:6]))
        copies = [torch.empty_like(v) for v in grads]
        norm = gelim.ops.clip_global_norm(grads, 0.5, out=copies)
        return [Y, *grads, norm, *copies]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(held[0])
    torch.cuda.current_stream().wait_stream(side)
    for h in held:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(h))
        graphs.append(graph)
    for k in range(4):
        for j in (0, 1):
            new = sets[(k + j) % 4] + (dYs[(k + j) % 4],)
            for h, v in zip(held[j], new):
                h.copy_(v)
            graphs[j].replay()
        for j in (0, 1):
            new = sets[(k + j) % 4] + (dYs[(k + j) % 4],)
            for a, b in zip(outs[j], step(list(new))):
                assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_other_stream(gelim, cuda):
    args = make(cuda, 80, 512, 512, 16, 4, torch.bfloat16)
    want = gelim.ops.adapter_matmul(*args)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = [gelim.ops.adapter_matmul(*args) for _ in range(5)]
    s.synchronize()
    for v in got:
        assert torch.equal(v, want)


@pytest.mark.parametrize("seed", range(60))
def test_any_sizes_and_places(gelim, cuda, seed):
    """Sizes, layouts and wanted gradients as they come; operands between NaN, or at an address of their type's size only."""
    import math
    import random

    rng = random.Random(seed)

    def size(most, step=1):
        return max(1, int(round(math.exp(rng.uniform(0.0, math.log(most))))) // step * step)

    def put(v):
        v, how = v.contiguous(), rng.randrange(3)
        if how == 1:
            first = rng.choice([1, 2, 3, 4, 8])
            return torch.cat([v.new_zeros(first), v.reshape(-1)])[first:].view(v.shape)
        if how == 2:
            more = rng.choice([1, 4, 8, 13])
            at = rng.randint(0, more)
            room = v.new_full((*v.shape[:-2], v.shape[-2] + 2, v.shape[-1] + more), float("nan"))
            room[..., 1:1 + v.shape[-2], at:at + v.shape[-1]] = v
            return room[..., 1:1 + v.shape[-2], at:at + v.shape[-1]]
        return v

    dtype, layout = rng.choice(DTYPES), rng.choice(["kn", "nk"])
    step = rng.choice([1, 8, 64])
    T, K, N, n = size(3000), size(2000, step), size(2000, step), size(40)
    r = rng.choice([1, 2, 7, 8, 16, 17, 33, 64, 100, 129, 256])
    X, W, A, B, index, scale = make(cuda, T, K, N, r, n, dtype, layout, rng.choice(["mixed", "runs", "none", "all"]), seed)
    W, A, B = (put(v) if layout == "kn" else put(v.transpose(-1, -2)).transpose(-1, -2) for v in (W, A, B))
    args = (put(X), W, A, B, index, scale)
    out = put(X.new_zeros(T, N))
    gelim.ops.adapter_matmul(*args, out=out)
    check(out, *ref_product(*args, device=cuda))
    dY = put(torch.randn(T, N, generator=torch.Generator().manual_seed(seed)).to(dtype).to(cuda))
    need = rng.choice([(True, True, True), (True, False, False), (False, True, False), (False, False, True)])
    for v, t, wanted in zip(gelim.ops.adapter_matmul_grad(dY, *args, need=need), ref_grad(dY, *args, device=cuda), need):
        assert (v is not None) == wanted
        if wanted:
            check(v, *t)


def test_two_at_a_time(gelim, cuda):
    """Calls and replays on two streams, from two threads: sums cut over workgroups that wait for each other's parts."""
    from threading import Thread

    sizes = [(70, 2056, 520, 64, 3), (20, 1024, 512, 8, 2), (257, 4104, 1032, 16, 5)]
    sets = [[make(cuda, *z, torch.bfloat16, seed=s) for z in sizes] for s in range(2)]

    def work(args):
        Y = gelim.ops.adapter_matmul(*args)
        return [Y, *gelim.ops.adapter_matmul_grad(Y, *args)]

    want = [[work(a) for a in mine] for mine in sets]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for mine in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append([work(a) for a in mine])
        graphs.append(graph)
    got, failed = [[], []], []

    def thread(k):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(10):
                    got[k].append([work(a) for a in sets[k]])
                    graphs[k].replay()
                    got[k].append([[v.clone() for v in vs] for vs in outs[k]])
            s.synchronize()
        except Exception as e:
            failed.append(e)

    threads = [Thread(target=thread, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for k in range(2):
        for once in got[k]:
            for a, b in zip(once, want[k]):
                for v, w in zip(a, b):
                    assert torch.equal(v, w)


@pytest.mark.parametrize("T", [2, 70])
def test_offsets_past_32_bits(gelim, cuda, T):
    """Rows of X, W and Y, and adapters, that begin more than 2^31 elements into their tensors."""
    K, N, r = 64, 48, 8
    ld = (2 ** 31 + 4096) // (T - 1) if T > 2 else 2 ** 31 + 4096
    ld = ld // 8 * 8
    room = torch.empty((T - 1) * ld + K, dtype=torch.bfloat16, device=cuda)
    X = room.as_strided((T, K), (ld, 1))
    g = torch.Generator().manual_seed(T)
    X.copy_(torch.randn(T, K, generator=g))
    W = (torch.randn(K, N, generator=g) * 0.1).bfloat16().to(cuda)
    fac = torch.empty(2 ** 31 + 8192, dtype=torch.bfloat16, device=cuda)
    A = fac.as_strided((2, K, r), (2 ** 31 + 64, r, 1))
    B = fac.as_strided((2, r, N), (2 ** 31 + 64, N, 1), 4096)
    A.copy_(torch.randn(2, K, r, generator=g))
    B.copy_(torch.randn(2, r, N, generator=g))
    index = (torch.arange(T) % 2).int().to(cuda)
    out = torch.empty((T - 1) * ld + N, dtype=torch.bfloat16, device=cuda).as_strided((T, N), (ld, 1))
    args = (X, W, A, B, index, 0.5)
    check(gelim.ops.adapter_matmul(*args, out=out), *ref_product(*args))
    dY = torch.randn(T, N, generator=g).bfloat16().to(cuda)
    for v, t in zip(gelim.ops.adapter_matmul_grad(dY, *args), ref_grad(dY, *args)):
        check(v, *t)


def test_many_rows(gelim, cuda):
    """A batch whose rows are past the largest grid of one dimension, and past a sort's first blocks."""
    T, K, N, r, n = 70001, 32, 40, 4, 37
    args = make(cuda, T, K, N, r, n, torch.bfloat16)
    check(gelim.ops.adapter_matmul(*args), *ref_product(*args))
    dY = torch.randn(T, N, device=cuda).bfloat16()
    for v, t in zip(gelim.ops.adapter_matmul_grad(dY, *args), ref_grad(dY, *args)):
        check(v, *t)


def test_more_adapters_than_rows(gelim, cuda):
    for T in (5, 90):
        args = make(cuda, T, 64, 64, 4, 1500, torch.float16)
        check(gelim.ops.adapter_matmul(*args), *ref_product(*args))
        dY = torch.randn(T, 64, device=cuda).half()
        for v, t in zip(gelim.ops.adapter_matmul_grad(dY, *args), ref_grad(dY, *args)):
            check(v, *t)


@pytest.mark.parametrize("T", [66, 257, 5000, 9000])
def test_many_resident_adapters_of_which_few_are_used(gelim, cuda, T):
    """What the adapters that no row has hold does not matter, and their gradients are zeros."""
    X, W, A, B, index, scale = make(cuda, T, 136, 72, 12, 30, torch.bfloat16)
    index = torch.where(index % 7 == 3, index, -1)
    index[T - 1] = 29
    unused = torch.ones(30, dtype=torch.bool, device=cuda)
    unused[index[index >= 0].long()] = False
    ref = ref_product(X, W, A, B, index, scale)
    dY = torch.randn(T, 72, generator=torch.Generator().manual_seed(T)).bfloat16().to(cuda)
    grads = ref_grad(dY, X, W, A, B, index, scale)
    A[unused], B[unused] = float("nan"), float("inf")
    check(gelim.ops.adapter_matmul(X, W, A, B, index, scale), *ref)
    for v, t in zip(gelim.ops.adapter_matmul_grad(dY, X, W, A, B, index, scale), grads):
        check(v, *t)


def test_refusals(gelim, cuda):
    X, W, A, B, index, scale = make(cuda, 6, 32, 40, 4, 3, torch.bfloat16)
    f = gelim.ops.adapter_matmul
    bad = [(TypeError, (X.double(), W, A, B, index)), (TypeError, (X, W.float(), A, B, index)),
           (TypeError, (X, W, A, B, index.long())), (ValueError, (X, W, A, B)), (ValueError, (X, W, A, B, index[:5])),
           (ValueError, (X[:, :31], W, A, B, index)), (ValueError, (X, W, A[:2], B, index)),
           (ValueError, (X, W, A, B[:, :3], index)), (ValueError, (X, W, A[0], B, index)),
           (ValueError, (X, W, A[:, :, :0], B[:, :0], index)), (ValueError, (X, W, A[:0], B[:0], index)),
           (ValueError, (X, W, A, B, index.cpu())), (ValueError, (X.cpu(), W, A, B, index)),
           (TypeError, (X, W, A, B, index, scale.double())), (ValueError, (X, W, A, B, index, scale[:2]))]
    for error, args in bad:
        with pytest.raises(error):
            f(*args)
    wide = torch.zeros(1, 32, 257, device=cuda).bfloat16()
    with pytest.raises(ValueError, match="256"):
        f(X, W, wide, torch.zeros(1, 257, 40, device=cuda).bfloat16())
    for out in (torch.empty(6, 41, device=cuda).bfloat16(), torch.empty(6, 40, device=cuda),
                torch.empty(40, 6, device=cuda).bfloat16().t(), X.new_empty(1, 40).expand(6, 40)):
        with pytest.raises(ValueError):
            f(X, W, A, B, index, out=out)
    square = torch.zeros(6, 32, device=cuda).bfloat16()
    with pytest.raises(ValueError, match="overlaps"):
        f(square, torch.zeros(32, 32, device=cuda).bfloat16(), A, torch.zeros(3, 4, 32, device=cuda).bfloat16(), index,
          out=square)
    with pytest.raises(ValueError, match="autograd"):
        f(X, W, A.clone().requires_grad_(), B, index)
    with torch.no_grad():
        f(X, W, A.clone().requires_grad_(), B, index)
    Y = f(X, W, A, B, index, scale)
    with pytest.raises(ValueError):
        gelim.ops.adapter_matmul_grad(Y[:, :39], X, W, A, B, index, scale)
    with pytest.raises(TypeError):
        gelim.ops.adapter_matmul_grad(Y.float(), X, W, A, B, index, scale)


def test_tune_clip_and_serve(gelim, cuda):
    """Two adapters tuned together for three steps, then served beside others: prompts and single tokens agree."""
    T, K, N, r, n = 192, 256, 320, 8, 2
    X, W, A, B, index, _ = make(cuda, T, K, N, r, n, torch.float32, rows="runs")
    target = torch.randn(T, N, device=cuda)
    A, B = A.clone(), B.clone()
    for _ in range(3):
        Y = gelim.ops.adapter_matmul(X, W, A, B, index, 2.0)
        dY = (Y - target) / T
        _, dA, dB = gelim.ops.adapter_matmul_grad(dY, X, W, A, B, index, 2.0, need=(False, True, True))
        (_, _), (rA, tA), (rB, tB) = ref_grad(dY, X, W, A, B, index, 2.0)
        norm = gelim.ops.clip_global_norm([dA, dB], 0.01)
        size = (rA.square().sum() + rB.square().sum()).sqrt()
        off = (tA.square().sum() + tB.square().sum()).sqrt()
        assert abs(norm.item() - size) <= off + 2.0 ** -23 * size
        f = min(1.0, 0.01 / (size.item() + 1e-6))
        rel = (off / size).item() + 2.0 ** -22
        for got, ref, tol in ((dA, rA, tA), (dB, rB, tB)):
            assert ((got.cpu().double() - f * ref).abs() <= f * (tol + rel * ref.abs()) + 1e-30).all()
        A -= 0.1 * dA
        B -= 0.1 * dB
    stack_a = torch.cat([A, torch.randn(5, K, r, device=cuda)]).bfloat16()
    stack_b = torch.cat([B, torch.randn(5, r, N, device=cuda)]).bfloat16()
    X16, W16 = X.bfloat16(), W.bfloat16()
    which = torch.randint(-1, 7, (T,), device=cuda, dtype=torch.int32)
    whole = gelim.ops.adapter_matmul(X16, W16, stack_a, stack_b, which, 2.0)
    ref, tol = ref_product(X16, W16, stack_a, stack_b, which, 2.0)
    check(whole, ref, tol)
    for t0, t1 in ((0, 1), (1, 33), (33, 97)):
        part = gelim.ops.adapter_matmul(X16[t0:t1], W16, stack_a, stack_b, which[t0:t1], 2.0)
        check(part, ref[t0:t1], tol[t0:t1])
