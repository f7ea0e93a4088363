"""The 2-norm over many tensors and clipping, against 64 bits.

The sum of squares is held in 64 bits, so the norm is off by its one rounding
to fp32 (2^-24) and the 64-bit sum's (below 2^-40); a scaled element by the
rounding of the factor and of the product to fp32 and of the result to its type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def reference(tensors, max_norm):
    norm = math.sqrt(math.fsum(t.double().square().sum().item() for t in tensors))
    return norm, min(1.0, max_norm / (norm + 1e-6))


def check(tensors, before, norm, max_norm):
    ref, f = reference(before, max_norm)
    assert norm.dtype == torch.float32 and norm.shape == ()
    assert abs(norm.item() - ref) <= (2.0 ** -24 + 2.0 ** -40) * ref
    for t, b in zip(tensors, before):
        info = torch.finfo(t.dtype)
        want = b.double() * f
        tol = (info.eps / 2 + 2.0 ** -22) * want.abs() + info.smallest_normal * info.eps
        assert t.shape == b.shape and ((t.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", [[1], [7], [0, 3, 0], [255, 256, 257], [16384], [16385, 5, 32768], [100000, 1, 99999],
                                   [9] * 127, [9] * 128, [10] * 129, [33] * 400, [1 << 22]])
@pytest.mark.parametrize("max_norm", [0.25, 1e9])
def test_in_place_and_apart(gelim, cuda, sizes, dtype, max_norm):
    g = torch.Generator().manual_seed(len(sizes))
    before = [torch.randn(n, generator=g).to(dtype).to(cuda) for n in sizes]
    tensors = [t.clone() for t in before]
    out = [torch.full_like(t, 9.0) for t in before]
    check(out, before, gelim.ops.clip_global_norm(tensors, max_norm, out=out), max_norm)
    for t, b in zip(tensors, before):
        assert torch.equal(t, b)
    norm = gelim.ops.clip_global_norm(tensors, max_norm)
    check(tensors, before, norm, max_norm)
    for t, o in zip(tensors, out):
        assert torch.equal(t, o)


def test_mixed_types_packed_without_gaps(gelim, cuda):
    """Tensors that begin at odd addresses, next to each other; what lies around them stays as it was."""
    flat = [torch.randn(60001, device=cuda).to(t) for t in DTYPES]
    before = [f.clone() for f in flat]
    cuts = [1, 4, 5, 1003, 1010, 20001, 59999]
    views, olds = [], []
    for f, b in zip(flat, before):
        for lo, hi in zip(cuts, cuts[1:]):
            views.append(f[lo:hi])
            olds.append(b[lo:hi])
    order = torch.randperm(len(views), generator=torch.Generator().manual_seed(3)).tolist()
    views, olds = [views[i] for i in order], [olds[i] for i in order]
    check(views, olds, gelim.ops.clip_global_norm(views, 2.0), 2.0)
    for f, b in zip(flat, before):
        assert f[0] == b[0] and torch.equal(f[59999:], b[59999:])


def test_any_dense_order_of_dimensions(gelim, cuda):
    a = torch.randn(5, 6, 7, device=cuda).permute(2, 0, 1)
    b = torch.randn(33, 65, device=cuda).bfloat16().t()
    c = torch.randn((), device=cuda)
    before = [a.clone(), b.clone(), c.clone()]
    check([a, b, c], before, gelim.ops.clip_global_norm([a, b, c], 1.5), 1.5)


def test_measures_only(gelim, cuda):
    a = torch.randn(70000, device=cuda)
    a[5] = float("inf")
    b = a.clone()
    assert gelim.ops.clip_global_norm([a], math.inf).item() == math.inf
    assert torch.equal(a, b)


def test_values_whose_squares_leave_fp32(gelim, cuda):
    for size in (1e30, 1e-30):
        t = [torch.full((1000,), size, device=cuda), torch.full((24,), size, device=cuda).bfloat16()]
        check(t, [v.clone() for v in t], gelim.ops.clip_global_norm(t, 1.0), 1.0)


def test_nan_infinity_and_zeros(gelim, cuda):
    a, b = torch.ones(100, device=cuda), torch.ones(50, device=cuda)
    b[3] = float("nan")
    assert math.isnan(gelim.ops.clip_global_norm([a, b], 1.0).item())
    assert torch.isnan(a).all() and torch.isnan(b).all()
    a, b = torch.ones(100, device=cuda), torch.ones(50, device=cuda)
    b[3] = float("inf")
    assert gelim.ops.clip_global_norm([a, b], 1.0).item() == math.inf
    assert not a.any() and torch.isnan(b[3]) and not b[:3].any()
    z = torch.zeros(1000, device=cuda)
    assert gelim.ops.clip_global_norm([z], 1.0).item() == 0 and not z.any()
    a = torch.ones(10, device=cuda)
    gelim.ops.clip_global_norm([a], 0.0)
    assert not a.any()


def test_same_bits_every_time(gelim, cuda):
    t = [torch.randn(n, device=cuda) for n in (300001, 17, 40000)]
    first = gelim.ops.clip_global_norm(t, math.inf)
    for _ in range(5):
        assert torch.equal(first, gelim.ops.clip_global_norm(t, math.inf))


def test_past_32_bits(gelim, cuda):
    n = 2 ** 31 + 77
    t = torch.ones(n, device=cuda, dtype=torch.bfloat16)
    t[-1] = 3.0
    norm = gelim.ops.clip_global_norm([t], 2.0 ** -2)
    assert abs(norm.item() - math.sqrt(n + 8)) <= 2.0 ** -23 * math.sqrt(n)
    f = 0.25 / (math.sqrt(n + 8) + 1e-6)
    for i in (0, 2 ** 31 - 1, 2 ** 31 + 1, n - 2, n - 1):
        want = f * (3 if i == n - 1 else 1)
        assert abs(t[i].item() - want) <= 2.0 ** -7 * want


def test_refusals(gelim, cuda):
    f = gelim.ops.clip_global_norm
    a, b = torch.ones(8, device=cuda), torch.ones(8, device=cuda)
    for error, args, kw in [(ValueError, ([], 1.0), {}), (ValueError, ([a], -1.0), {}), (ValueError, ([a], math.nan), {}),
                            (TypeError, ([a.double()], 1.0), {}), (ValueError, ([a.cpu()], 1.0), {}),
                            (ValueError, ([a, b.cpu()], 1.0), {}), (ValueError, ([a[::2]], 1.0), {}),
                            (ValueError, ([a[:1].expand(4)], 1.0), {}), (ValueError, ([a], 1.0), {"out": []}),
                            (ValueError, ([a], 1.0), {"out": [b[:7]]}), (ValueError, ([a], 1.0), {"out": [b.half()]}),
                            (ValueError, ([a.view(2, 4).t()], 1.0), {"out": [b.view(4, 2)]}),
                            (gelim.GelimError, ([a, a], 1.0), {}), (gelim.GelimError, ([a, a[4:]], 1.0), {}),
                            (gelim.GelimError, ([a[:4], b[:4]], 1.0), {"out": [b[2:6], a[4:8]]}),
                            (gelim.GelimError, ([a[:4], b[:4]], 1.0), {"out": [b[4:], b[4:]]})]:
        with pytest.raises(error):
            f(*args, **kw)
    assert (a == 1).all() and (b == 1).all()
    f([a, a], math.inf, out=[torch.empty_like(a), torch.empty_like(a)])
