"""Cases of the operators that train and serve many low-rank adapters at once: the adapter linear (`ops.adapter_linear`), the
LayerNorm with its weight gradients (`ops.layernorm_train`) and the 8-bit activation checkpoint (`ops.act8_pack`).

`run` computes them in plain 32-bit torch operations, or through the framework's own calls when `own` is true; `exact` computes
the same definitions in 64 bits, request by request and row by row.

Definitions.  Row m of the adapter linear belongs to one request and so to one adapter g (or to none):
    t_m = s_g A_g x_m,   y_m = W x_m + b + B_g t_m (+ residual_m)
    dt_m = s_g B_g^T dy_m,   dx_m = W^T dy_m + A_g^T dt_m,   dA_g = sum_m dt_m x_m^T,   dB_g = sum_m dy_m t_m^T
The 8-bit checkpoint of a row: blocks of 32 columns, one power of two 2^e per block (the smallest that brings the block's largest
magnitude to 127.5 or less), codes round(x 2^-e) to the nearest even integer within +-127.  A backward pass with a checkpoint sees the
values of the codes in place of x (dA and dB of the adapter linear, dx and dgamma of the LayerNorm); the forward pass sees x itself.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------------------------ cases
def listed():
    lin = dict(op="linear", train=False, ckpt8=False, residual=False, ragged=False)
    norm = dict(op="norm", ckpt8=False)
    return [
        # the timestep rows of a batch: one row per request, every request with its owner's adapter -- latency
        dict(lin, name="linear_single_rows", requests=8, rows=8, K=1280, N=1280, adapters=8, rank=32),
        # one row per request, many owners, small ranks of several sizes
        dict(lin, name="linear_many_adapters", requests=193, rows=193, K=320, N=1280, adapters=48, rank=16),
        # the text states of 13 prompts of 77 tokens through a key projection, some requests without an adapter
        dict(lin, name="linear_text", requests=13, rows=1001, K=768, N=640, adapters=5, rank=64),
        # an attention projection with its residual over the tokens of 8 images
        dict(lin, name="linear_images", requests=8, rows=32768, K=320, N=320, adapters=8, rank=32, residual=True),
        # the wide feed-forward projection of 16 images: bound by the matrix cores
        dict(lin, name="linear_feed_forward", requests=16, rows=4096, K=1280, N=10240, adapters=16, rank=32),
        # a training step of the large rank, forward and backward
        dict(lin, name="linear_train_rank320", train=True, requests=4, rows=4096, K=640, N=640, adapters=3, rank=320),
        # a training step over requests of very different lengths that keeps its input in 8 bits
        dict(lin, name="linear_train_ragged_8bit", train=True, ckpt8=True, ragged=True, requests=21, rows=9001, K=1280, N=1280,
             adapters=7, rank=64),
        # the token rows of 8 images, forward and backward
        dict(norm, name="norm_images", rows=32768, C=320, dtype="bf16"),
        # full-precision rows of an odd width
        dict(norm, name="norm_odd_fp32", rows=2005, C=1001, dtype="fp32"),
        # the widest level, input kept in 8 bits
        dict(norm, name="norm_8bit", rows=16384, C=1280, dtype="bf16", ckpt8=True),
        # 8-bit checkpoint of a small odd full-precision activation
        dict(op="act8", name="act8_odd_fp32", rows=77, C=1001, dtype="fp32"),
        # 8-bit checkpoint of the token rows of 16 images
        dict(op="act8", name="act8_images", rows=65536, C=640, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["serve", "serve", "single", "train", "train", "norm", "norm", "act8"])
    if kind == "norm":
        C = _log(rng, 16, 4096)
        return dict(op="norm", rows=_log(rng, 1, min(60000, 20_000_000 // C)), C=C, dtype=rng.choice(["bf16", "bf16", "fp32"]),
                    ckpt8=rng.random() < 0.5)
    if kind == "act8":
        C = _log(rng, 16, 4096)
        return dict(op="act8", rows=_log(rng, 1, min(60000, 40_000_000 // C)), C=C, dtype=rng.choice(["bf16", "bf16", "fp32"]))
    train = kind == "train"
    rank = rng.choice([4, 8, 16, 24, 32, 32, 64, 100, 320])
    adapters = rng.randint(1, max(1, min(40, 1024 // rank)))
    K, N = 8 * _log(rng, 8, 320), 8 * _log(rng, 8, 640)
    if kind == "single":
        requests = rows = _log(rng, 1, 256)
    else:
        requests = rng.randint(1, 24)
        rows = max(requests, _log(rng, 16, min(40000, (12_000_000_000 if train else 36_000_000_000) // (K * N))))
    return dict(op="linear", train=train, ckpt8=train and rng.random() < 0.5, residual=rng.random() < 0.4,
                ragged=kind != "single" and rng.random() < 0.6, requests=requests,
                rows=rows if kind == "single" else max(requests, rows), K=K, N=N, adapters=adapters, rank=rank)


def _requests(case):
    """(rows of each request, adapter of each request or -1, rank of each adapter): goes by the case alone."""
    r = random.Random("%(requests)d %(rows)d %(adapters)d %(rank)d" % case)
    n, rows, G = case["requests"], case["rows"], case["adapters"]
    if case["ragged"]:
        w = [math.exp(r.gauss(0.0, 1.3)) for _ in range(n)]
        lengths = [1 + int(x / sum(w) * (rows - n)) for x in w]
        lengths[0] += rows - sum(lengths)
    else:
        lengths = [rows // n] * n
        lengths[-1] += rows - sum(lengths)
    ids = [r.randrange(G) if r.random() > 0.1 or n < 10 else -1 for _ in range(n)]
    ranks = [max(1, case["rank"] >> (g % 3)) if G > 4 else case["rank"] for g in range(G)]
    return lengths, ids, ranks


# ------------------------------------------------------------------------------------------------------------------ inputs
def _activation(shape, dtype, gen):
    x = torch.randn(shape, generator=gen, device=DEV)
    x *= torch.exp(0.7 * torch.randn(shape[1], generator=gen, device=DEV))      # channels of unlike size
    return (x + 0.1 * torch.randn(shape[1], generator=gen, device=DEV)).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(DEV).manual_seed(seed)
    randn = lambda *s: torch.randn(s, generator=gen, device=DEV)  # noqa: E731
    st = {"case": case}
    if case["op"] != "linear":
        st["x"] = _activation((case["rows"], case["C"]), DT[case["dtype"]], gen)
        if case["op"] == "norm":
            st["dy"] = randn(case["rows"], case["C"]).to(DT[case["dtype"]])
            st["gamma"], st["beta"] = 1.0 + 0.2 * randn(case["C"]), 0.2 * randn(case["C"])
            if own:
                for k in ("x", "gamma", "beta"):
                    st[k].requires_grad_(True)
        return st
    M, K, N, G, R = (case[k] for k in ("rows", "K", "N", "adapters", "rank"))
    lengths, ids, ranks = _requests(case)
    bf = torch.bfloat16
    st["x"] = _activation((M, K), bf, gen)
    st["w"], st["bias"] = (randn(N, K) / math.sqrt(K)).to(bf), (0.1 * randn(N)).to(bf)
    live = (torch.arange(R, device=DEV)[None] < torch.tensor(ranks, device=DEV)[:, None]).float()     # [G, R]
    st["down"] = (randn(G, R, K) / R * live[:, :, None]).to(bf)
    st["up"] = (0.03 * randn(G, N, R) * live[:, None, :]).to(bf)
    scales = [1.03 if g % 2 else 0.75 for g in range(G)]
    st["residual"] = randn(M, N).to(bf) if case["residual"] else None
    st["dy"] = randn(M, N).to(bf) if case["train"] else None
    if own:
        from aqualora_amd import adapters, ops
        st["packed"] = ops.PackedLinear(st["w"], st["bias"])
        st["bank"] = adapters.AdapterBank(st["down"], st["up"], ranks=ranks, scales=scales, trainable=case["train"])
        st["plan"] = adapters.RequestPlan(ids, lengths)
        if case["train"]:
            st["x"].requires_grad_(True)
            if st["residual"] is not None:
                st["residual"].requires_grad_(True)
    else:
        st["adapter_of_row"] = torch.tensor(ids, device=DEV).repeat_interleave(torch.tensor(lengths, device=DEV))
        st["scales"] = torch.tensor(scales, device=DEV)
    return st


# ------------------------------------------------------------------------------------------------------------------ one pass
def run(st):
    return {"linear": _linear, "norm": _norm, "act8": _act8}[st["case"]["op"]](st)


def _codes(x):
    """The values that a row's 8-bit codes stand for, in 32 bits: powers of two are put together from their exponents' bits, so that
    every step is exact but the rounding that defines the code."""
    rows, C = x.shape
    pad = -C % 32
    b = torch.cat([x.float(), x.new_zeros(rows, pad, dtype=torch.float32)], 1).view(rows, -1, 32)
    m, e = torch.frexp(b.abs().amax(2, keepdim=True))             # amax = m 2^e with m in [0.5, 1)
    e = torch.clamp(e - 7 + (m > 127.5 / 128.0).int(), -126, 121)
    q = torch.clamp(torch.round(b * ((127 - e) << 23).view(torch.float32)), -127.0, 127.0)
    return (q * ((127 + e) << 23).view(torch.float32)).view(rows, C + pad)[:, :C].contiguous()


def _act8(st):
    x = st["x"]
    if own:
        from aqualora_amd import ops
        return ops.act8_pack(x).unpack()
    return _codes(x).to(x.dtype)


def _norm(st):
    x, gamma, beta, dy, eps = st["x"], st["gamma"], st["beta"], st["dy"], 1e-5
    if own:
        from aqualora_amd import ops
        y = ops.layernorm_train(x, gamma, beta, eps, ckpt8=st["case"]["ckpt8"])
        return (y.detach(),) + torch.autograd.grad(y, (x, gamma, beta), dy)
    xf, dyf = x.float(), dy.float()
    mean = xf.mean(1, keepdim=True)
    rstd = torch.rsqrt((xf - mean).square().mean(1, keepdim=True) + eps)
    y = (xf - mean) * rstd * gamma + beta
    xh = ((_codes(x) if st["case"]["ckpt8"] else xf) - mean) * rstd
    g = dyf * gamma
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return y.to(x.dtype), dx.to(x.dtype), (dyf * xh).sum(0), dyf.sum(0)


def _linear(st):
    case = st["case"]
    x, res, dy = st["x"], st["residual"], st["dy"]
    if own:
        from aqualora_amd import ops
        y = ops.adapter_linear(x, st["packed"], st["bank"], st["plan"], residual=res, ckpt8=case["ckpt8"])
        if not case["train"]:
            return y
        wrt = (x, st["bank"].down, st["bank"].up) + (() if res is None else (res,))
        return (y.detach(),) + torch.autograd.grad(y, wrt, dy)
    M, K = x.shape
    G, R, N = st["down"].shape[0], st["down"].shape[1], st["w"].shape[0]
    xf, w = x.float(), st["w"].float()
    A, B = st["down"].float().view(G * R, K), st["up"].float().permute(0, 2, 1).reshape(G * R, N)
    pick = ((st["adapter_of_row"][:, None] == torch.arange(G, device=x.device)) * st["scales"])[:, :, None]      # [M, G, 1]
    low = lambda v, S: ((v @ S.t()).view(M, G, R) * pick).view(M, G * R)  # noqa: E731
    t = low(xf, A)
    y = xf @ w.t() + st["bias"].float() + t @ B
    if res is not None:
        y = y + res.float()
    y = y.to(x.dtype)
    if not case["train"]:
        return y
    dyf = dy.float()
    if case["ckpt8"]:
        xf = _codes(x)
        t = low(xf, A)
    dt = low(dyf, B)
    dx = (dyf @ w + dt @ A).to(x.dtype)
    dA = (dt.t() @ xf).view(G, R, K)
    dB = (t.t() @ dyf).view(G, R, N).permute(0, 2, 1).contiguous()
    return (y, dx, dA, dB) + (() if res is None else (dy,))


# ------------------------------------------------------------------------------------------------------------------ accounts
def work(case):
    if case["op"] != "linear":
        n, s = case["rows"] * case["C"], 2 if case["dtype"] == "bf16" else 4
        code = n * 33.0 / 32.0
        if case["op"] == "act8":                       # read x, write the codes; read the codes, write the values
            return {"bytes": 2 * n * s + 2 * code, "flops": 4.0 * n}
        if case["ckpt8"]:                              # x -> y and codes; codes, dy -> dx
            return {"bytes": 4 * n * s + 2 * code + 16 * case["C"], "flops": 22.0 * n}
        return {"bytes": 5 * n * s + 16 * case["C"], "flops": 20.0 * n}      # x -> y; x, dy -> dx
    M, K, N = case["rows"], case["K"], case["N"]
    lengths, ids, ranks = _requests(case)
    low = sum(2.0 * n * ranks[g] * (K + N) for n, g in zip(lengths, ids) if g >= 0)
    stack = sum(2.0 * ranks[g] * (K + N) for g in set(ids) if g >= 0)
    flops, nbytes = 2.0 * M * K * N + low, 2.0 * (M * K + N * K + N + M * N) + stack
    if case["residual"]:
        nbytes += 2.0 * M * N
    if case["train"]:
        flops += 2.0 * M * K * N + 2 * low
        nbytes += 2.0 * (M * N + M * K) + 4.0 * case["adapters"] * case["rank"] * (K + N)          # dy, dx, dA, dB
        nbytes += 2.0 * M * K * 33.0 / 32.0 if case["ckpt8"] else 2.0 * M * K                       # x again for dA
    return {"bytes": nbytes, "flops": flops}


# ------------------------------------------------------------------------------------------------------------------ 64 bits
def _pow2(e):
    return ((e + 1023) << 52).view(torch.float64)


def _values64(x):
    """The checkpoint's values from its definition: e is counted up from below until the block's largest magnitude fits."""
    rows, C = x.shape
    out = torch.empty(rows, C, dtype=torch.float64, device=x.device)
    for c in range(0, C, 32):
        b = x[:, c:c + 32].double()
        top = b.abs().amax(1, keepdim=True)
        e = torch.floor(torch.log2(torch.clamp(top, min=2.0 ** -160))).long() - 8
        for _ in range(4):
            e = torch.where(top > 127.5 * _pow2(e), e + 1, e)
        step = _pow2(torch.clamp(e, -126, 121))
        out[:, c:c + 32] = torch.clamp(torch.round(b / step), -127, 127) * step
    return out


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = kept
    x = st["x"].double()
    if case["op"] == "act8":
        return _values64(st["x"])
    if case["op"] == "norm":
        dy, gamma, beta = st["dy"].double(), st["gamma"].double(), st["beta"].double()
        C = case["C"]
        mean = x.sum(1, keepdim=True) / C
        sd = torch.sqrt(((x - mean) ** 2).sum(1, keepdim=True) / C + 1e-5)
        xh = ((_values64(st["x"]) if case["ckpt8"] else x) - mean) / sd
        h = dy * gamma
        dx = (h - h.sum(1, keepdim=True) / C - xh * ((h * xh).sum(1, keepdim=True) / C)) / sd
        return (x - mean) / sd * gamma + beta, dx, (dy * xh).sum(0), dy.sum(0)
    lengths, ids, _ = _requests(case)
    w, A, B = st["w"].double(), st["down"].double(), st["up"].double()
    y = torch.addmm(st["bias"].double(), x, w.t())
    at, spans = 0, []
    for n, g in zip(lengths, ids):
        spans.append((slice(at, at + n), g, float(st["scales"][g]) if g >= 0 else 0.0))
        at += n
    for rows, g, s in spans:
        if g >= 0:
            y[rows] += s * ((x[rows] @ A[g].t()) @ B[g].t())
    if st["residual"] is not None:
        y += st["residual"].double()
    if not case["train"]:
        return y
    dy = st["dy"].double()
    xs = _values64(st["x"]) if case["ckpt8"] else x
    dx, dA, dB = dy @ w, torch.zeros_like(A), torch.zeros_like(B)
    for rows, g, s in spans:
        if g >= 0:
            dt = s * (dy[rows] @ B[g])
            dx[rows] += dt @ A[g]
            dA[g] += dt.t() @ xs[rows]
            dB[g] += s * (dy[rows].t() @ (xs[rows] @ A[g].t()))
    return (y, dx, dA, dB) + (() if st["residual"] is None else (dy,))
