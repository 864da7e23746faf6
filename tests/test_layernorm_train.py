"""LayerNorm with weight gradients and the 8-bit activation checkpoint against their definitions in 64 bits.

Tolerances.  u = 2^-24 is half a step of fp32, h = finfo(dtype).eps / 2 half a step of the stored type.  A sum whose longest chain of fp32
additions has L links is off by at most L u sum|terms|; a row sum has at most 8 * 4 + 9 links in a thread and its reductions (L = 64 covers
it with the roundings of the terms), a column sum at most rows / groups + 512 / 16 + 48 (LR below).  The rest is first-order propagation,
written out in `bounds`."""
import pytest
import torch

from aqualora_amd import _lib, ops

DEV = "cuda"
U = 2.0 ** -24
L = 64
SHAPES = [(1, 1), (1, 8), (3, 7), (5, 16), (17, 33), (64, 128), (33, 129), (7, 256), (9, 257), (130, 320), (4099, 320), (65, 1001),
          (12, 1280), (3, 2048), (5, 2049), (3, 4096), (2, 4097), (2, 8192)]
gpu = pytest.mark.gpu


def codes64(x):
    """The values of the codes by the format's definition, block by block, in 64 bits."""
    x = x.double().cpu()
    out = torch.empty_like(x)
    for c in range(0, x.shape[1], 32):
        b = x[:, c:c + 32]
        top = b.abs().amax(1, keepdim=True)
        e = torch.full(top.shape, -126, dtype=torch.int64)
        for k in range(-125, 122):
            e = torch.where(top > 127.5 * 2.0 ** (k - 1), torch.full_like(e, k), e)
        step = ((e + 1023) << 52).view(torch.float64)
        q = torch.clamp(torch.round(b / step), -127, 127) * step
        out[:, c:c + 32] = torch.where(torch.isfinite(top), q, torch.full_like(q, float("nan")))
    return out


def reference(x, x_seen, gamma, beta, dy, dres, eps):
    """y, dx, dgamma, dbeta in 64 bits and how far fp32 sums may be from them before the last rounding."""
    x, xs, g, dy = (t.double().cpu() for t in (x, x_seen, gamma, dy))
    b = torch.zeros_like(g) if beta is None else beta.double().cpu()
    M, C = x.shape
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    y = (x - mean) * rstd * g + b
    xh = (xs - mean) * rstd
    h = dy * g
    m1, m2 = h.mean(1, keepdim=True), (h * xh).mean(1, keepdim=True)
    dx = rstd * (h - m1 - xh * m2) + (0 if dres is None else dres.double().cpu())
    dmean = L * U * x.abs().mean(1, keepdim=True)                       # |error of the mean|
    # relative error of rstd: the chain of the variance, its 1 / sqrt, and the mean's own error (its first order cancels)
    drstd = (L + 8) * U + (dmean * rstd) ** 2
    dy_ = (g.abs() * rstd * dmean + (y - b).abs() * (drstd + 4 * U) + 2 * U * y.abs())
    dxh = rstd * (dmean + 2 * U * (xs - mean).abs()) + xh.abs() * drstd
    dm2 = (h.abs() * dxh).mean(1, keepdim=True) + L * U * (h * xh).abs().mean(1, keepdim=True)
    ddx = rstd * (2 * U * h.abs() + L * U * h.abs().mean(1, keepdim=True) + xh.abs() * dm2 + dxh * m2.abs() + 4 * U * (h.abs() + m1.abs() + (xh * m2).abs()))
    ddx = ddx + (drstd + 4 * U) * (rstd * (h - m1 - xh * m2)).abs() + 2 * U * dx.abs()
    LR = M // 2 + 100 if M < 200 else M // 8 + 100
    dg = (dy * xh).sum(0)
    ddg = (dy.abs() * (dxh + LR * U * xh.abs())).sum(0)
    return (y, dx, dg, dy.sum(0)), (dy_, ddx, ddg, LR * U * dy.abs().sum(0))


def inputs(M, C, dtype, seed, offset=0.3):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    x = (r(M, C) * torch.exp(r(C)) + offset).to(dtype)
    return x, 1 + 0.3 * r(C), 0.3 * r(C), r(M, C).to(dtype), r(M, C).to(dtype)


def check(name, got, ref, slack, dtype):
    half = torch.finfo(dtype).eps / 2
    got = got.double().cpu()
    assert got.shape == ref.shape and torch.isfinite(got).all(), name
    over = ((got - ref).abs() - (half * ref.abs() + slack * (1 + half))).max()
    assert over <= 0, f"{name}: {over.item():.3e} over its bound"


@gpu
@pytest.mark.parametrize("ckpt8", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,C", SHAPES)
def test_layernorm_train_vs_64_bits(M, C, dtype, ckpt8):
    x, g, b, dy, dres = inputs(M, C, dtype, M * 10007 + C)
    seen = codes64(x) if ckpt8 else x
    for residual in (False, True):
        xd, gd, bd = (t.to(DEV).requires_grad_(True) for t in (x, g, b))
        f = ops.layernorm_train_res if residual else ops.layernorm_train
        out = f(xd, gd, bd, 1e-5, ckpt8=ckpt8)
        y, seeds = (out[0], (dy.to(DEV), dres.to(DEV))) if residual else (out, dy.to(DEV))
        grads = torch.autograd.grad(out, (xd, gd, bd), seeds)
        ref, slack = reference(x, seen, g, b, dy, dres if residual else None, 1e-5)
        check("y", y, ref[0], slack[0], dtype)
        for n, a, r, s, t in zip(("dx", "dgamma", "dbeta"), grads, ref[1:], slack[1:], (dtype, torch.float32, torch.float32)):
            check(n, a, r, s, t)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layernorm_train_strides_types_and_absent_parts(dtype):
    M, C = 37, 203
    x, g, b, dy, _ = inputs(M, C, dtype, 5)
    wide = torch.zeros(M, C + 9, dtype=dtype, device=DEV)
    wide[:, 5:5 + C] = x.to(DEV)
    xd = wide[:, 5:5 + C].detach().requires_grad_(True)
    assert xd.stride(0) == C + 9
    g16 = g.to(torch.bfloat16).to(DEV).requires_grad_(True)
    y = ops.layernorm_train(xd, g16, None)                                       # bf16 weights, no beta, strided rows
    dyt = dy.to(DEV).t().contiguous().t()                                        # column-major gradient
    dx, dg = torch.autograd.grad(y, (xd, g16), dyt)
    ref, slack = reference(x, x, g16.detach(), None, dy, None, 1e-5)
    check("y", y, ref[0], slack[0], dtype)
    check("dx", dx, ref[1], slack[1], dtype)
    assert dg.dtype == torch.bfloat16
    check("dgamma", dg, ref[2], slack[2], torch.bfloat16)
    # a broadcast gradient (y.sum()): stride 0 in both directions
    y = ops.layernorm_train(xd, g16, None, ckpt8=True)
    dx, = torch.autograd.grad(y.sum(), xd)
    ref, slack = reference(x, codes64(x), g16.detach(), None, torch.ones(M, C), None, 1e-5)
    check("dx of a sum", dx, ref[1], slack[1], dtype)
    # frozen weights: only dx; a frozen x: only the weights
    gd = g.to(DEV)
    assert ops.layernorm_train(xd, gd, None).grad_fn is not None
    y = ops.layernorm_train(xd.detach(), gd.requires_grad_(True), None)
    y.sum().backward()
    assert gd.grad is not None and xd.grad is None


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layernorm_train_rows_without_variation_and_non_finite_rows(dtype):
    x = torch.ones(6, 96, dtype=dtype, device=DEV)
    x[1] = 0
    x[2] = torch.linspace(-3, 3, 96)
    x[3, 40] = float("inf")
    x[4, 95] = float("nan")
    x[5] = torch.linspace(1, 2, 96)
    for ckpt8 in (False, True):
        xd = x.clone().requires_grad_(True)
        y = ops.layernorm_train(xd, torch.ones(96, device=DEV), None, 1e-5, ckpt8=ckpt8)
        dx, = torch.autograd.grad(y, xd, torch.ones_like(y))
        assert (y[:2] == 0).all() and torch.isfinite(dx[:3]).all() and torch.isfinite(dx[5]).all()
        assert torch.isnan(y[4]).all() and torch.isnan(y[3]).any() and torch.isfinite(y[5]).all() and torch.isfinite(y[2]).all()


@gpu
def test_layernorm_train_empty():
    x = torch.empty(0, 48, device=DEV, requires_grad=True)
    g, b = torch.ones(48, device=DEV, requires_grad=True), torch.zeros(48, device=DEV, requires_grad=True)
    for ckpt8 in (False, True):
        y = ops.layernorm_train(x, g, b, ckpt8=ckpt8)
        dx, dg, db = torch.autograd.grad(y.sum(), (x, g, b))
        assert y.shape == dx.shape == (0, 48) and (dg == 0).all() and (db == 0).all()


def test_gradient_formula_against_differences():
    """The formula that the kernel is held to, against central differences of the 64-bit forward pass (h = 1e-5: truncation and rounding
    both stay under 1e-7 of the gradient's size)."""
    x, g, b, dy, _ = inputs(3, 40, torch.float32, 11)
    (y, dx, dg, db), _ = reference(x, x, g, b, dy, None, 1e-5)
    loss = lambda x, g, b: (reference(x, x, g, b, dy, None, 1e-5)[0][0] * dy.double()).sum()  # noqa: E731
    gen = torch.Generator().manual_seed(3)
    for k, grad in enumerate((dx, dg, db)):
        a = [x.double(), g.double(), b.double()]
        v = torch.randn(a[k].shape, generator=gen, dtype=torch.float64)
        hi, lo = list(a), list(a)
        hi[k], lo[k] = a[k] + 1e-5 * v, a[k] - 1e-5 * v
        num = (loss(*hi) - loss(*lo)) / 2e-5
        assert abs(num - (grad * v).sum()) <= 1e-6 * (grad.abs() * v.abs()).sum()


@gpu
def test_layernorm_train_same_bits_streams_and_graph():
    M, C = 3000, 640
    x, g, b, dy, _ = (t.to(DEV) for t in inputs(M, C, torch.bfloat16, 21))

    def step(x, ckpt8):
        xd, gd, bd = (t.detach().requires_grad_(True) for t in (x, g, b))
        y = ops.layernorm_train(xd, gd, bd, ckpt8=ckpt8)
        return (y.detach(),) + torch.autograd.grad(y, (xd, gd, bd), dy)

    for ckpt8 in (False, True):
        want = step(x, ckpt8)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step(x, ckpt8)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, c) for a, c in zip(want, other))
        buf = x.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(buf, ckpt8)
        for k in range(4):
            xk = torch.roll(x, k, 0) * (1 + k)
            buf.copy_(xk)
            graph.replay()
            eager = step(xk, ckpt8)
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(eager, out)), (ckpt8, k)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,C", [(1, 1), (1, 31), (2, 32), (3, 33), (77, 1001), (5, 8193), (0, 40), (257, 640)])
def test_act8_is_its_definition(M, C, dtype):
    gen = torch.Generator().manual_seed(M + C)
    x = torch.randn(M, C, generator=gen) * torch.exp(8 * torch.randn(M, C, generator=gen))
    if M:
        x[0] = 127.5 * 2.0 ** torch.arange(C).remainder(7)      # largest codes and ties
        x[-1, : C // 2] = 0.0
    if M > 4:
        x[1] = 2.0 ** -130                                       # below the smallest step
        x[2, 0] = 2.0 ** 127
        x[3, 0], x[4, C - 1] = float("inf"), float("nan")
    x = x.to(dtype)
    a = ops.act8_pack(x.to(DEV))
    want = codes64(x)
    for t in (dtype, torch.float32):
        got = a.unpack(t).double().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
    # half a step of the block
    for c in range(0, C, 32):
        blk, val = x[:, c:c + 32].double(), want[:, c:c + 32]
        top = blk.abs().amax(1, keepdim=True)
        ok = torch.isfinite(top[:, 0]) & (top[:, 0] > 2.0 ** -119) & (top[:, 0] <= 127.5 * 2.0 ** 121)
        assert ((blk - val).abs() <= top / 127.5 * 1.0)[ok].all()
    assert a.codes.shape == (M, (C + 31) // 32 * 32) and (a.codes[:, C:] == 0).all()


@gpu
def test_act8_strided_and_many_dimensions():
    gen = torch.Generator().manual_seed(1)
    big = torch.randn(4, 6, 70, generator=gen).to(torch.bfloat16).to(DEV)
    x = big[..., 3:60]
    a = ops.act8_pack(x)
    assert a.shape == (4, 6, 57)
    assert torch.equal(a.unpack().double().cpu().reshape(24, 57), codes64(x.reshape(24, 57)))
    assert torch.equal(ops.act8_pack(big.transpose(1, 2)).unpack().double().cpu().reshape(-1, 6), codes64(big.transpose(1, 2).reshape(-1, 6)))
    v = ops.act8_pack(big[0, 0])
    assert torch.equal(v.unpack().double().cpu()[None], codes64(big[0, 0][None]))


@gpu
def test_rows_past_31_bit_offsets():
    """More than 2^31 elements: the last rows of the codes, of y and of dx against the definition."""
    C, last = 1280, 50
    M = (1 << 31) // C + 3000
    gen = torch.Generator("cuda").manual_seed(13)
    x = torch.empty(M, C, device="cuda", dtype=torch.bfloat16)
    for part in x.split(100000):
        part.copy_(torch.randn(part.shape, generator=gen, device="cuda"))
    packed = ops.act8_pack(x)
    tail = x[-last:].cpu()
    assert torch.equal(packed.unpack()[-last:].double().cpu(), codes64(tail))
    del packed
    gamma, beta = torch.randn(C, generator=gen, device="cuda"), torch.randn(C, generator=gen, device="cuda")
    for ckpt8 in (False, True):
        xg = x.detach().requires_grad_(True)
        y = ops.layernorm_train(xg, gamma, beta, ckpt8=ckpt8)
        dx, = torch.autograd.grad(y, (xg,), x)
        ref, slack = reference(tail, codes64(tail) if ckpt8 else tail, gamma.cpu(), beta.cpu(), tail, None, 1e-5)
        for name, got, k in (("y", y[-last:], 0), ("dx", dx[-last:], 1)):
            check(name, got, ref[k], slack[k], torch.bfloat16)


@gpu
def test_double_backward_is_refused():
    x = torch.randn(4, 32, device=DEV, requires_grad=True)
    g = torch.ones(32, device=DEV, requires_grad=True)
    d, = torch.autograd.grad(ops.layernorm_train(x, g, None).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()


def test_refusals():
    g = torch.ones(32)
    with pytest.raises(_lib.AqlError):
        ops.layernorm_train(torch.zeros(4, 32), g, None)
    with pytest.raises(_lib.AqlError):
        ops.act8_pack(torch.zeros(4, 32))
    for x, gamma in ((torch.zeros(4, 32, dtype=torch.float16), g), (torch.zeros(2, 4, 32), g), (torch.zeros(4, 31), g),
                     (torch.zeros(4, 32), g.double()), (torch.zeros(4, 32), torch.ones(64)[::2]), (torch.zeros(4, 9000), torch.ones(9000))):
        with pytest.raises(ValueError):
            ops.layernorm_train(x, gamma, None)
    with pytest.raises(ValueError):
        ops.layernorm_train(torch.zeros(4, 32), g, g.to(torch.bfloat16))
    for x in (torch.zeros(4, 32, dtype=torch.float16), torch.zeros(4, 0), torch.tensor(1.0)):
        with pytest.raises(ValueError):
            ops.act8_pack(x)


def test_act8_of_parts_that_do_not_fit_is_refused():
    codes, exps, f = torch.zeros(6, 64, dtype=torch.uint8), torch.zeros(6, 2, dtype=torch.uint8), torch.float32
    for c, e, shape in ((codes[:5], exps, (6, 64)), (codes, exps[:, :1], (6, 64)), (codes, exps, (6, 65)), (codes, exps, (7, 64)), (codes, exps, (2, 4, 64)),
                        (codes.float(), exps, (6, 64)), (codes.t().contiguous().t(), exps, (6, 64)), (codes[0], exps[0], (64,)), (codes, exps, ()), (codes, exps, (6, 0))):
        with pytest.raises(ValueError):
            ops.Act8(c, e, shape, f).unpack()
    with pytest.raises(_lib.AqlError):
        ops.Act8(codes, exps, (2, 3, 40), f).unpack()      # all fits: only the GPU is missing


@gpu
def test_captured_backward_next_to_a_live_eager_graph_is_refused():
    gen = torch.Generator().manual_seed(21)
    x, dy = torch.randn(40, 320, generator=gen).to("cuda"), torch.randn(40, 320, generator=gen).to("cuda")
    gamma = torch.ones(320, device="cuda", requires_grad=True)
    step = lambda: torch.autograd.grad(ops.layernorm_train(x, gamma, None), (gamma,), dy)  # noqa: E731
    want = step()
    alive = ops.layernorm_train(x, gamma, None)
    with pytest.raises(RuntimeError, match="still lives"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    torch.cuda.synchronize()
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(want[0], got[0])


def test_c_entries_refuse_bad_arguments():
    lib = _lib.load()
    p = _lib.c_p(4096)     # never dereferenced: every call below is refused on the host
    assert lib.aql_layernorm_train_fwd(p, 0, 4, 9000, 9000, p, p, 1, 1e-5, p, 9000, p, None, None, None) != 0
    assert lib.aql_layernorm_train_fwd(p, 0, 4, 64, 63, p, p, 1, 1e-5, p, 64, p, None, None, None) != 0
    assert lib.aql_layernorm_train_fwd(p, 0, 4, 64, 64, p, p, 1, 1e-5, p, 64, p, p, None, None) != 0
    assert lib.aql_layernorm_train_fwd(None, 0, 4, 64, 64, p, p, 1, 1e-5, p, 64, p, None, None, None) != 0
    need = lib.aql_layernorm_train_scratch_floats(4, 64)
    assert need == 2 * 64
    args = lambda x, codes, n: (x, codes, codes, p, None, 0, 4, 64, 64, 64, 0, p, 1, p, p, 64, p, p, p, n, None)  # noqa: E731
    assert lib.aql_layernorm_train_bwd(*args(p, p, need)) != 0        # both x and codes
    assert lib.aql_layernorm_train_bwd(*args(None, None, need)) != 0  # neither
    assert lib.aql_layernorm_train_bwd(*args(p, None, need - 1)) != 0
    assert b"workspace" in lib.aql_last_error()
    assert lib.aql_act8_pack(p, 2, 4, 64, 64, p, p, None) != 0
    assert lib.aql_act8_pack(p, 0, 4, 64, 60, p, p, None) != 0
    assert lib.aql_act8_unpack(None, p, 4, 64, p, 0, 64, None) != 0
    assert lib.aql_act8_pack(None, 0, 0, 64, 64, None, None, None) == 0   # no rows: nothing to do


def test_act8_of_rows_beyond_the_format_is_refused():
    """More columns than the kernels' 2^24, also where the count's low 32 bits would pass (a broadcast row: no memory)."""
    for columns in ((1 << 24) + 1, (1 << 31) + 8, (1 << 32) + 5):
        with pytest.raises(ValueError, match="columns"):
            ops.act8_pack(torch.zeros(1, 1).expand(1, columns))
        with pytest.raises(ValueError):
            ops.Act8(torch.zeros(0, 1, dtype=torch.uint8).expand(0, (columns + 31) // 32 * 32), torch.zeros(0, 1, dtype=torch.uint8).expand(0, (columns + 31) // 32),
                     (0, columns), torch.float32).unpack()
