"""Workloads of the adapter products and of the gradient clipping: what is timed, and what the results have to be.

Three operators:

  product   Y = X W + scale_i (X A_i) B_i, row t of X with the adapter i = index[t] (none where it is -1)
  gradient  dX, dA, dB of that product for a given dY (W is shared and frozen)
  clip      the 2-norm over many tensors and their copies scaled by min(1, max_norm / (norm + 1e-6))

`own` false computes them from elementary torch operations in 32 bits, `own` true calls this package.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one token of one conversation with one adapter: nothing but latency
        dict(name="product_1_token", op="product", T=1, K=2048, N=2048, r=8, n=1, dtype="bf16", layout="kn", rows="mixed"),
        # a decoding step: a token of each of 32 requests, 64 adapters resident
        dict(name="product_32_requests", op="product", T=32, K=4096, N=4096, r=16, n=64, dtype="bf16", layout="kn", rows="mixed"),
        # a small decoding step with odd sizes, weights stored as (out, in)
        dict(name="product_13_odd_fp16", op="product", T=13, K=2055, N=5001, r=12, n=5, dtype="fp16", layout="nk", rows="mixed"),
        # prompts of several requests in one batch, one after the other
        dict(name="product_prompts_2048", op="product", T=2048, K=4096, N=4096, r=16, n=8, dtype="bf16", layout="kn", rows="runs"),
        # prompts in 32 bits at this framework's headline matrix size, ragged in rows and rank
        dict(name="product_1000_fp32", op="product", T=1000, K=2048, N=2048, r=10, n=3, dtype="fp32", layout="kn", rows="runs"),
        # the largest batch of prompts
        dict(name="product_prompts_8192", op="product", T=8192, K=8192, N=8192, r=64, n=4, dtype="bf16", layout="nk", rows="runs"),
        # one short sequence of a fine-tuning run: latency
        dict(name="gradient_100", op="gradient", T=100, K=1024, N=1024, r=8, n=1, dtype="bf16", layout="kn", rows="all"),
        # a fine-tuning batch of one adapter
        dict(name="gradient_4096", op="gradient", T=4096, K=4096, N=4096, r=16, n=1, dtype="bf16", layout="kn", rows="all"),
        # six adapters tuned together on ragged sequences, odd sizes, weights stored as (out, in)
        dict(name="gradient_1777_odd_fp16", op="gradient", T=1777, K=2050, N=1030, r=9, n=6, dtype="fp16", layout="nk", rows="runs"),
        # the gradients of the adapters of four products: latency
        dict(name="clip_8_small", op="clip", count=8, total=8 * 2048 * 8, dtype="bf16", align=128, max_norm=1.0),
        # the gradients of every adapter of a model, in one buffer without gaps, so that most begin at odd places
        dict(name="clip_448_packed_fp32", op="clip", count=448, total=29_000_003, dtype="fp32", align=1, max_norm=1.0),
        # the gradients of whole layers
        dict(name="clip_290_large", op="clip", count=290, total=1_000_000_007, dtype="bf16", align=128, max_norm=0.5),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["product", "product", "product", "gradient", "gradient", "clip"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "clip":
        total = _log(rng, 20_000, 500_000_000)
        return dict(op=op, count=min(_log(rng, 1, 512), total // 16), total=total, dtype=dtype, align=rng.choice([1, 8, 128]),
                    max_norm=rng.choice([0.1, 1.0, 1e9]))
    few = op == "product" and rng.random() < 0.5  # tokens of a decoding step, or prompts
    T = _log(rng, 1, 64) if few else _log(rng, 65, 8192 if op == "product" else 4096)
    K, N, step = _log(rng, 256, 7168), _log(rng, 256, 7168), rng.choice([1, 8, 64])
    K, N = max(step, K // step * step), max(step, N // step * step)
    if dtype == "fp32":  # 32 bits take about ten times as long
        T, K, N = min(T, 4096), min(K, 4096), min(N, 4096)
    return dict(op=op, T=T, K=K, N=N, r=rng.choice([1, 4, 8, 16, 16, 32, 64, rng.randint(2, 64)]), n=_log(rng, 1, 64 if few else 16),
                dtype=dtype, layout=rng.choice(["kn", "nk"]), rows=rng.choice(["mixed", "runs"]) if few else "runs")


def _index(case, seed):
    """The adapter of each row: runs of rows of one request after another, or each row another request's; about one in eight has none."""
    g = torch.Generator().manual_seed(seed)
    T, n = case["T"], case["n"]
    if case["rows"] == "all":
        return torch.zeros(T, dtype=torch.int32)
    many = T if case["rows"] == "mixed" else min(T, n + 3)
    which = torch.randint(0, n, (many,), generator=g)
    which[torch.rand(many, generator=g) < 0.125] = -1
    if case["rows"] == "mixed":
        return which.int()
    ends = torch.sort(torch.randint(0, T + 1, (many - 1,), generator=g))[0]
    return which[torch.searchsorted(ends, torch.arange(T), right=True)].int()


def _sizes(case):
    """`count` sizes that add up to at most `total`, spread over a factor of 64."""
    g = torch.Generator().manual_seed(case["count"])
    part = torch.exp(torch.rand(case["count"], generator=g, dtype=torch.float64) * math.log(64.0))
    return (part / part.sum() * case["total"]).long().clamp_min(1).tolist()


def _scale(case):
    return torch.linspace(0.5, 2.0, case["n"], dtype=torch.float32)


def prepare(case, seed):
    t, g = TYPES[case["dtype"]], torch.Generator("cuda").manual_seed(seed)
    if case["op"] == "clip":
        sizes, align = _sizes(case), case["align"]
        room = torch.tensor([-(-s // align) * align for s in sizes])
        starts = (torch.cumsum(room, 0) - room).tolist()
        flat = torch.randn(int(room.sum()), generator=g, device="cuda", dtype=t).mul_(0.03)
        views = [(s, s + z) for s, z in zip(starts, sizes)]
        keep = torch.zeros(flat.numel(), device="cuda", dtype=t)
        grads = [flat[a:b].mul_(0.1 + (7 * i) % 5) for i, (a, b) in enumerate(views)]
        return dict(op="clip", grads=grads, max_norm=case["max_norm"], flat_out=keep, out=[keep[a:b] for a, b in views])
    T, K, N, r, n = (case[k] for k in "TKNrn")
    kn = case["layout"] == "kn"

    def random(*shape, turned=False, size=1.0):
        if turned:
            return random(*shape[:-2], shape[-1], shape[-2], size=size).transpose(-1, -2)
        return torch.randn(shape, generator=g, device="cuda", dtype=t).mul_(size)

    state = dict(op=case["op"], X=random(T, K), W=random(K, N, turned=not kn, size=K ** -0.5), A=random(n, K, r, turned=not kn, size=K ** -0.5),
                 B=random(n, r, N, turned=not kn, size=0.5 * r ** -0.5), index=_index(case, seed).cuda(), scale=_scale(case).cuda())
    if case["op"] == "gradient":
        state["dY"] = random(T, N, size=0.01)
    return state


def _plain_low(U, F, chosen):
    """U times the adapters' factors side by side, each row's own ones kept and scaled."""
    return ((U @ F).view(U.shape[0], chosen.shape[1], -1) * chosen[:, :, None]).view(U.shape[0], -1)


def _plain_chosen(state):
    n = state["A"].shape[0]
    hit = state["index"][:, None] == torch.arange(n, device="cuda", dtype=torch.int32)
    return torch.where(hit, state["scale"], torch.zeros_like(state["scale"]))


def _plain_product(state):
    X, W, A, B = (state[k].float() for k in "XWAB")
    n, K, r = A.shape
    low = _plain_low(X, A.permute(1, 0, 2).reshape(K, n * r), _plain_chosen(state))
    return (X @ W + low @ B.reshape(n * r, -1)).to(state["X"].dtype)


def _plain_gradient(state):
    X, W, A, B, dY = (state[k].float() for k in ("X", "W", "A", "B", "dY"))
    n, K, r = A.shape
    chosen, flat_a, flat_b = _plain_chosen(state), A.permute(1, 0, 2).reshape(K, n * r), B.reshape(n * r, -1)
    back = _plain_low(dY, flat_b.t(), chosen)
    dX = dY @ W.t() + back @ flat_a.t()
    dA = (X.t() @ back).view(K, n, r).permute(1, 0, 2)
    dB = (_plain_low(X, flat_a, chosen).t() @ dY).view(B.shape)
    return [v.to(state["X"].dtype) for v in (dX, dA, dB)]


def _plain_clip(state):
    squares = torch.stack([g.float().square().sum(dtype=torch.float64) for g in state["grads"]])
    norm = squares.sum().sqrt()
    factor = (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    [o.copy_(g.float() * factor) for g, o in zip(state["grads"], state["out"])]
    return norm.float()


def run(state):
    if own:
        import gelim

        if state["op"] == "clip":
            norm = gelim.ops.clip_global_norm(state["grads"], state["max_norm"], out=state["out"])
            return [norm, state["flat_out"]]
        args = [state[k] for k in ("X", "W", "A", "B", "index", "scale")]
        if state["op"] == "product":
            return gelim.ops.adapter_matmul(*args)
        return list(gelim.ops.adapter_matmul_grad(state["dY"], *args))
    if state["op"] == "clip":
        return [_plain_clip(state), state["flat_out"]]
    return _plain_product(state) if state["op"] == "product" else _plain_gradient(state)


def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "clip":
        return {"bytes": 2 * size * case["total"], "flops": 3 * case["total"]}
    T, K, N, r, n = (case[k] for k in "TKNrn")
    used = min(n, T)
    adapters, rows = used * r * (K + N) * size, T * (K + N) * size
    if case["op"] == "product":
        return {"bytes": rows + K * N * size + adapters + 4 * T, "flops": 2 * T * (K * N + r * (K + N))}
    # reads X, dY, W and the adapters, writes dX and the adapters' gradients
    return {"bytes": rows + T * K * size + K * N * size + adapters + n * r * (K + N) * size + 4 * T, "flops": 2 * T * (K * N + r * (3 * K + 2 * N))}


def exact(case, seed):
    """From the definitions, one adapter after the other, in 64 bits."""
    state = prepare(case, seed)
    if case["op"] == "clip":
        norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(g, dtype=torch.float64)) ** 2 for g in state["grads"]))
        factor = min(1.0, case["max_norm"] / (norm + 1e-6))
        out = torch.zeros(state["flat_out"].numel(), dtype=torch.float64, device="cuda")
        at = 0
        for g in state["grads"]:
            out[at:at + g.numel()] = g.double() * factor
            at += -(-g.numel() // case["align"]) * case["align"]
        return [torch.tensor(norm, dtype=torch.float64), out]
    X, W, A, B = (state[k].double() for k in "XWAB")
    index = state["index"].long()
    scale = state["scale"].double().tolist()
    if case["op"] == "product":
        Y = torch.mm(X, W)
        for i in range(case["n"]):
            rows = torch.nonzero(index == i)[:, 0]
            Y[rows] += scale[i] * torch.mm(torch.mm(X[rows], A[i]), B[i])
        return Y
    dY = state["dY"].double()
    dX, dA, dB = torch.mm(dY, W.T), torch.zeros_like(A), torch.zeros_like(B)
    for i in range(case["n"]):
        rows = torch.nonzero(index == i)[:, 0]
        x, y = X[rows], dY[rows]
        dX[rows] += scale[i] * torch.mm(torch.mm(y, B[i].T), A[i].T)
        dA[i] = scale[i] * torch.mm(x.T, torch.mm(y, B[i].T))
        dB[i] = scale[i] * torch.mm(torch.mm(x, A[i]).T, y)
    return [dX, dA, dB]
