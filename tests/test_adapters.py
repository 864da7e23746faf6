"""Adapters of many requests beside one projection (ops.adapter_linear), against the definition in 64 bits, request by request.

Tolerances.  u = 2^-24.  A dot product of n terms in fp32, in whatever order, is off by at most n u sum|terms|.  T (and dT) enters the product with
B (A) as bf16: half a step, 2^-8 relative.  The output is rounded to bf16 once: 2^-8 of its value.  dA and dB are fp32 sums of products with
T (dT) split into three bf16 parts that hold 24 bits (u relative)."""
import copy
import os
import pickle
import shutil
import subprocess
import sys
import threading

import pytest
import torch

from aqualora_amd import _lib, adapters, lora, ops
from tests.test_layernorm_train import codes64

DEV = "cuda"
U, HALF = 2.0 ** -24, 2.0 ** -8
gpu = pytest.mark.gpu

# lengths (a number: that many equal requests, plan without lengths), adapters, K, N, rank
CASES = {
    "one_row": ([1], [0], 8, 8, 1),
    "one_row_no_adapter": ([1], [-1], 16, 8, 4),
    "single_rows": ([1] * 40, [(7 * i) % 5 - 1 for i in range(40)], 48, 56, 16),
    "single_rows_equal_plan": ((19, 19), [(3 * i) % 4 for i in range(19)], 1280, 320, 32),
    "ragged": ([5, 0, 1, 130, 64, 3, 17, 0], [2, 1, 0, 2, -1, 1, 2, 3], 320, 328, 20),
    "ragged_more_rows": ([200, 1, 1, 1, 37, 300, 2], [0, 1, 2, 0, -1, 3, 1], 72, 136, 33),
    "equal_77": ((5, 385), [0, 3, 1, 3, -1], 768, 640, 64),
    "tiles_of_128": ([1030, 1, 2000, 1169], [1, 0, 2, 1], 72, 1032, 8),
    "large_rank": ([130, 70, 200], [1, 0, 1], 200, 320, 320),
    "whole_rows_in_one_launch": ([9000, 130, 5, 15500], [1, 0, -1, 2], 200, 264, 40),
    "wide_tiles": ([7000, 3000, 6400], [0, 1, 0], 72, 1600, 16),
    "whole_wide_tiles": ((8, 16384), [1, 0, -1, 2, 2, 0, 1, -1], 72, 1280, 24),
    "columns_of_160": ([13000, 8700], [1, 0], 64, 480, 72),
    "columns_of_320": ([20000, 12700], [1, 0], 64, 320, 72),
    "columns_of_192": ([4000, 1, 3500, 1500], [1, 0, 2, 1], 72, 1280, 24),
    "two_rounds": ([20000, 13000], [1, 0], 64, 320, 72),
    "neighbours_of_one_adapter": ([16, 16, 16, 300], [1, 1, 0, 0], 64, 64, 12),
    "many_rows_many_adapters": ([1] * 300, [(7 * i) % 40 for i in range(300)], 320, 640, 16),
    "wide_few_rows": ([60, 4], [1, 0], 72, 10240, 24),
    "few_tiles": ([200, 1, 99], [1, 2, 0], 200, 1280, 24),
    "few_tiles_of_t": ([3000, 1001, 677], [1, 0, 2], 136, 160, 64),
    "no_adapters": ([3, 270], [-1, -1], 64, 72, 8),
}


def make(name, seed=0):
    lengths, ids, K, N, r = CASES[name]
    equal = isinstance(lengths, tuple)
    M = lengths[1] if equal else sum(lengths)
    rows = [M // lengths[0]] * lengths[0] if equal else lengths
    G = max(max(ids) + 1, 1) + 1                        # the last adapter has no request
    gen = torch.Generator().manual_seed(len(name) * 31 + seed)
    rn = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    ranks = [max(1, r - 3 * g) for g in range(G)]
    live = torch.arange(r)[None] < torch.tensor(ranks)[:, None]
    bf = lambda t: t.to(torch.bfloat16)  # noqa: E731
    d = dict(x=bf(rn(M, K) * torch.exp(0.5 * rn(K))), w=bf(rn(N, K) / K ** 0.5), bias=bf(rn(N)), res=bf(rn(M, N)), dy=bf(rn(M, N)),
             down=bf(rn(G, r, K) / r), up=bf(0.2 * rn(G, N, r)), scales=[1.25 - 0.5 * g for g in range(G)], ranks=ranks, live=live)
    return d, lengths, rows, ids, equal


def handles(d, lengths, ids, equal, trainable):
    packed = ops.PackedLinear(d["w"].to(DEV), d["bias"].to(DEV))
    bank = adapters.AdapterBank(d["down"], d["up"], ranks=d["ranks"], scales=d["scales"], trainable=trainable)
    return packed, bank, adapters.RequestPlan(ids, None if equal else lengths)


def reference(d, rows, ids, residual, seen):
    x, w, b, dy = (d[k].double() for k in ("x", "w", "bias", "dy"))
    xs = seen.double()
    A, B = d["down"].double() * d["live"][:, :, None], d["up"].double() * d["live"][:, None, :]
    M, K = x.shape
    N = w.shape[0]
    R = A.shape[1]
    y, dx = x @ w.t() + b, dy @ w
    ey, edx = (K + 4) * U * (x.abs() @ w.t().abs()) + 4 * U * b.abs(), (N + 4) * U * (dy.abs() @ w.abs())
    dA, dB, eA, eB = (torch.zeros_like(t) for t in (A, B, A, B))
    at = 0
    for n, g in zip(rows, ids):
        s = slice(at, at + n)
        at += n
        if g < 0 or n == 0:
            continue
        sc = d["scales"][g]
        t, dt = sc * (x[s] @ A[g].t()), sc * (dy[s] @ B[g])
        et, edt = (K + 4) * U * abs(sc) * (x[s].abs() @ A[g].t().abs()), (N + 4) * U * abs(sc) * (dy[s].abs() @ B[g].abs())
        y[s] += t @ B[g].t()
        dx[s] += dt @ A[g]
        ey[s] += (et + HALF * (t.abs() + et)) @ B[g].t().abs() + (K + R) * U * (t.abs() @ B[g].t().abs())
        edx[s] += (edt + HALF * (dt.abs() + edt)) @ A[g].abs() + (N + R) * U * (dt.abs() @ A[g].abs())
        ts = sc * (xs[s] @ A[g].t())
        ets = (K + 4) * U * abs(sc) * (xs[s].abs() @ A[g].t().abs())
        dA[g] += dt.t() @ xs[s]
        dB[g] += dy[s].t() @ ts
        eA[g] += edt.t() @ xs[s].abs() + (M + 8) * U * (dt.abs().t() @ xs[s].abs())
        eB[g] += dy[s].abs().t() @ ets + (M + 8) * U * (dy[s].abs().t() @ ts.abs())
    if residual:
        y = y + d["res"].double()
        ey = ey + 4 * U * d["res"].double().abs()
    ey, edx = ey + 4 * U * y.abs(), edx + 4 * U * dx.abs()
    return (y, dx, dA, dB), (ey, edx, eA, eB)


def check(name, got, ref, slack, half):
    got = got.double().cpu()
    assert got.shape == ref.shape and torch.isfinite(got).all(), name
    if got.numel():
        over = ((got - ref).abs() - (half * ref.abs() + slack * (1 + half))).max()
        assert over <= 0, f"{name}: {over.item():.3e} over its bound"


@gpu
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("name", list(CASES))
def test_forward_vs_64_bits(name, residual):
    d, lengths, rows, ids, equal = make(name)
    packed, bank, plan = handles(d, lengths, ids, equal, False)
    y = ops.adapter_linear(d["x"].to(DEV), packed, bank, plan, residual=d["res"].to(DEV) if residual else None)
    ref, slack = reference(d, rows, ids, residual, d["x"])
    check("y", y, ref[0], slack[0], HALF)


@gpu
@pytest.mark.parametrize("ckpt8", [False, True])
@pytest.mark.parametrize("name", list(CASES))
def test_training_vs_64_bits(name, ckpt8):
    d, lengths, rows, ids, equal = make(name, 1)
    packed, bank, plan = handles(d, lengths, ids, equal, True)
    x, res = d["x"].to(DEV).requires_grad_(True), d["res"].to(DEV).requires_grad_(True)
    y = ops.adapter_linear(x, packed, bank, plan, residual=res, ckpt8=ckpt8)
    dx, dA, dB, dres = torch.autograd.grad(y, (x, bank.down, bank.up, res), d["dy"].to(DEV))
    ref, slack = reference(d, rows, ids, True, codes64(d["x"]) if ckpt8 else d["x"])
    check("y", y, ref[0], slack[0], HALF)
    check("dx", dx, ref[1], slack[1], HALF)
    assert dA.dtype == dB.dtype == torch.float32
    check("dA", dA, ref[2], slack[2], U)
    check("dB", dB, ref[3], slack[3], U)
    assert torch.equal(dres.cpu(), d["dy"])
    # an adapter without rows and the part past a rank have gradients of exactly zero
    assert (dA[-1] == 0).all() and (dB[-1] == 0).all()
    dead = ~d["live"].to(DEV)
    assert (dA[dead] == 0).all() and (dB.transpose(1, 2)[dead] == 0).all()


@gpu
def test_frozen_input_or_frozen_adapters():
    d, lengths, rows, ids, equal = make("ragged", 2)
    packed, bank, plan = handles(d, lengths, ids, equal, True)
    dy = d["dy"].to(DEV)
    ref, slack = reference(d, rows, ids, False, d["x"])
    y = ops.adapter_linear(d["x"].to(DEV), packed, bank, plan)                     # only the adapters learn
    dA, dB = torch.autograd.grad(y, (bank.down, bank.up), dy)
    check("dA", dA, ref[2], slack[2], U)
    check("dB", dB, ref[3], slack[3], U)
    packed, bank, plan = handles(d, lengths, ids, equal, False)                    # only the input
    x = d["x"].to(DEV).requires_grad_(True)
    dx, = torch.autograd.grad(ops.adapter_linear(x, packed, bank, plan), x, dy)
    check("dx", dx, ref[1], slack[1], HALF)
    y = ops.adapter_linear(x, packed, handles(d, lengths, ids, equal, True)[1], plan)
    g, = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)       # no second derivative: refused, not dropped
    with pytest.raises(RuntimeError):
        g.sum().backward()
    with torch.no_grad():
        assert not ops.adapter_linear(x, packed, bank, plan).requires_grad


@gpu
def test_strides_and_alignments():
    d, lengths, rows, ids, equal = make("ragged", 3)
    packed, bank, plan = handles(d, lengths, ids, equal, True)
    M, K = d["x"].shape
    want = ops.adapter_linear(d["x"].to(DEV), packed, bank, plan, residual=d["res"].to(DEV))
    for pad, at in ((16, 8), (9, 3), (8, 1)):
        wide = torch.full((M, K + pad), float("nan"), dtype=torch.bfloat16, device=DEV)
        wide[:, at:at + K] = d["x"].to(DEV)
        rw = torch.full((M, packed.N + pad), float("nan"), dtype=torch.bfloat16, device=DEV)
        rw[:, at:at + packed.N] = d["res"].to(DEV)
        x = wide[:, at:at + K].detach().requires_grad_(True)
        y = ops.adapter_linear(x, packed, bank, plan, residual=rw[:, at:at + packed.N])
        assert torch.equal(y, want)
        dyt = d["dy"].to(DEV).t().contiguous().t()
        g = torch.autograd.grad(y, (x, bank.down, bank.up), dyt)
        x2 = d["x"].to(DEV).requires_grad_(True)
        g2 = torch.autograd.grad(ops.adapter_linear(x2, packed, bank, plan), (x2, bank.down, bank.up), d["dy"].to(DEV))
        assert all(torch.equal(a, b) for a, b in zip(g, g2))
    xt = d["x"].to(DEV).t().contiguous().t()
    assert torch.equal(ops.adapter_linear(xt, packed, bank, plan, residual=d["res"].to(DEV)), want)
    x = d["x"].to(DEV).requires_grad_(True)                                       # a broadcast gradient
    g = torch.autograd.grad(ops.adapter_linear(x, packed, bank, plan).sum(), (x, bank.down, bank.up))
    d1 = dict(d, dy=torch.ones_like(d["dy"]))
    ref, slack = reference(d1, rows, ids, False, d["x"])
    for n, a, k, h in (("dx", g[0], 1, HALF), ("dA", g[1], 2, U), ("dB", g[2], 3, U)):
        check(n, a, ref[k], slack[k], h)


@gpu
@pytest.mark.parametrize("name", ["single_rows", "ragged", "ragged_more_rows", "tiles_of_128"])
def test_requests_do_not_reach_each_other(name):
    """Infinities and NaN in one request's rows, in an unused adapter and past an adapter's rank stay where they are."""
    d, lengths, rows, ids, equal = make(name, 4)
    packed, bank, plan = handles(d, lengths, ids, equal, True)
    victim = next(i for i, (n, g) in enumerate(zip(rows, ids)) if g >= 0 and n > 0)
    a0 = sum(rows[:victim])
    hit = torch.zeros(len(d["x"]), dtype=torch.bool)
    hit[a0:a0 + rows[victim]] = True
    dy = d["dy"].to(DEV)

    def step(d, packed, bank, plan, ckpt8):
        x = d["x"].to(DEV).requires_grad_(True)
        y = ops.adapter_linear(x, packed, bank, plan, ckpt8=ckpt8)
        return (y.detach(),) + torch.autograd.grad(y, (x, bank.down, bank.up), dy)

    for ckpt8 in (False, True):
        want = step(d, packed, bank, plan, ckpt8)
        bad = {k: (v.clone() if torch.is_tensor(v) else v) for k, v in d.items()}
        bad["x"][hit] = float("nan")
        bad["x"][a0, 0] = float("inf")
        bad["down"][~d["live"]] = float("nan")
        bad["up"].transpose(1, 2)[~d["live"]] = float("inf")
        bad["down"][-1] = float("nan")
        _, bank2, _ = handles(bad, lengths, ids, equal, True)
        got = step(bad, packed, bank2, plan, ckpt8)
        keep = ~hit.to(DEV)
        assert torch.equal(got[0][keep], want[0][keep]) and torch.equal(got[1][keep], want[1][keep])
        assert not torch.isfinite(got[0][~keep]).any()
        other = [g for g in range(bank.G) if g != ids[victim]]
        assert torch.equal(got[2][other], want[2][other]) and torch.equal(got[3][other], want[3][other])


@gpu
@pytest.mark.parametrize("name", [n for n, c in CASES.items() if len(set(c[1]) - {-1}) > 1])
def test_adapters_do_not_reach_each_other(name):
    """An adapter in use whose weights hold infinities and NaN: the rows and gradients of all the others keep their bits."""
    d, lengths, rows, ids, equal = make(name, 9)
    packed, bank, plan = handles(d, lengths, ids, equal, True)
    victim = next(g for n, g in zip(rows, ids) if g >= 0 and n > 0)
    of = torch.repeat_interleave(torch.tensor(ids), torch.tensor(rows))
    dy = d["dy"].to(DEV)

    def step(bank):
        x = d["x"].to(DEV).requires_grad_(True)
        y = ops.adapter_linear(x, packed, bank, plan)
        return (y.detach(),) + torch.autograd.grad(y, (x, bank.down, bank.up), dy)
    want = step(bank)
    keep = (of != victim).to(DEV)
    others = [g for g in range(bank.G) if g != victim]
    for key, value in (("down", float("nan")), ("up", float("nan")), ("up", float("inf"))):
        bad = dict(d, **{key: d[key].clone()})
        bad[key][victim, -1 if key == "up" else 0, 0] = value
        _, bank2, _ = handles(bad, lengths, ids, equal, True)
        got = step(bank2)
        assert not torch.isfinite(got[0][~keep]).all()
        for a, b in zip(got[:2], want[:2]):
            assert torch.equal(a[keep], b[keep]), (key, value)
        for a, b in zip(got[2:], want[2:]):
            assert torch.equal(a[others], b[others]), (key, value)
        if key == "up":      # ... and of the adapter itself the columns that it does not touch
            assert torch.equal(got[0][:, :-1], want[0][:, :-1])


@gpu
@pytest.mark.parametrize("ckpt8", [False, True])
def test_rows_past_31_bit_offsets(ckpt8):
    """More than 2^31 elements in x and dx: the last request, which alone uses its adapter, against the definition."""
    K, N, r, last = 1280, 64, 16, 700
    M = (1 << 31) // K + 3000
    gen = torch.Generator(DEV).manual_seed(11)
    cpu = torch.Generator().manual_seed(12)
    rn = lambda *s: torch.randn(s, generator=cpu)  # noqa: E731
    bf = lambda t: t.to(torch.bfloat16)  # noqa: E731
    x = torch.empty(M, K, device=DEV, dtype=torch.bfloat16)
    dy = torch.empty(M, N, device=DEV, dtype=torch.bfloat16)
    for t in (x, dy):
        for part in t.split(100000):
            part.copy_(torch.randn(part.shape, generator=gen, device=DEV))
    d = dict(x=x[-last:].cpu(), dy=dy[-last:].cpu(), w=bf(rn(N, K) / K ** 0.5), bias=bf(rn(N)), down=bf(rn(2, r, K) / r), up=bf(0.2 * rn(2, N, r)),
             scales=[1.0, 0.5], ranks=[r, r - 3], live=torch.arange(r)[None] < torch.tensor([[r], [r - 3]]))
    packed, bank, _ = handles(d, [1], [0], False, True)
    x.requires_grad_(True)
    y = ops.adapter_linear(x, packed, bank, adapters.RequestPlan([0, 1], [M - last, last]), ckpt8=ckpt8)
    dx, dA, dB = torch.autograd.grad(y, (x, bank.down, bank.up), dy)
    ref, slack = reference(d, [last], [1], False, codes64(d["x"]) if ckpt8 else d["x"])
    check("y", y[-last:], ref[0], slack[0], HALF)
    check("dx", dx[-last:], ref[1], slack[1], HALF)
    check("dA", dA[1], ref[2][1], slack[2][1], 2.0 ** -24)
    check("dB", dB[1], ref[3][1], slack[3][1], 2.0 ** -24)


@gpu
def test_empty_call():
    d, *_ = make("one_row")
    packed = ops.PackedLinear(d["w"].to(DEV), d["bias"].to(DEV))
    bank = adapters.AdapterBank(d["down"], d["up"], trainable=True)
    for plan in (adapters.RequestPlan([]), adapters.RequestPlan([], []), adapters.RequestPlan([0, 1], [0, 0])):
        x = torch.empty(0, 8, dtype=torch.bfloat16, device=DEV, requires_grad=True)
        y = ops.adapter_linear(x, packed, bank, plan)
        assert y.shape == (0, 8)
        g = torch.autograd.grad(y.sum(), (x, bank.down, bank.up))
        assert g[0].shape == (0, 8) and (g[1] == 0).all() and (g[2] == 0).all()


@gpu
def test_same_bits_streams_and_graphs():
    d, lengths, rows, ids, equal = make("ragged_more_rows", 5)
    packed, bank, plan = handles(d, lengths, ids, equal, True)
    x0, dy = d["x"].to(DEV), d["dy"].to(DEV)

    def step(x, ckpt8):
        x = x.detach().requires_grad_(True)
        y = ops.adapter_linear(x, packed, bank, plan, ckpt8=ckpt8)
        return (y.detach(),) + torch.autograd.grad(y, (x, bank.down, bank.up), dy)

    for ckpt8 in (False, True):
        want = step(x0, ckpt8)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step(x0, ckpt8)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(want, other))
        bufs, graphs, outs = [], [], []
        for _ in range(2):                              # two graphs alive together: no workspace is shared
            buf = x0.clone()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step(buf, ckpt8)
            bufs.append(buf), graphs.append(graph), outs.append(out)
        for k in range(4):
            xs = [torch.roll(x0, k + 1, 0), torch.roll(x0, 2 * k, 1) * 0.5]
            for b, x in zip(bufs, xs):
                b.copy_(x)
            torch.cuda.synchronize()
            streams = [torch.cuda.Stream(), torch.cuda.Stream()]
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
            torch.cuda.synchronize()
            for x, out in zip(xs, outs):
                eager = step(x, ckpt8)
                assert all(torch.equal(a, b) for a, b in zip(eager, out)), (ckpt8, k)


@gpu
def test_bank_follows_its_parameters():
    d, lengths, rows, ids, equal = make("ragged", 6)
    packed, bank, plan = handles(d, lengths, ids, equal, True)
    x = d["x"].to(DEV).requires_grad_(True)
    y = ops.adapter_linear(x, packed, bank, plan)
    with torch.no_grad():
        bank.up.mul_(0.5)
    half = dict(d, up=(d["up"].float() * 0.5).to(torch.bfloat16))
    ref, slack = reference(half, rows, ids, False, d["x"])
    check("y", ops.adapter_linear(x, packed, bank, plan), ref[0], slack[0], HALF)
    with pytest.raises(RuntimeError):
        y.sum().backward()                              # the weights changed after that forward pass
    opt = torch.optim.SGD(bank.parameters(), lr=0.25)
    ops.adapter_linear(x, packed, bank, plan).backward(d["dy"].to(DEV))
    new_up = bank.up.detach() - 0.25 * bank.up.grad
    opt.step()
    assert torch.equal(bank.up.detach(), new_up)
    ops.adapter_linear(x, packed, bank, plan)
    assert torch.equal(bank.handle.b[:, :, :bank.rank][:-1], (new_up * d["live"].to(DEV)[:, None, :]).to(torch.bfloat16)[:-1])
    assert torch.equal(bank.handle.bt, bank.handle.b.transpose(1, 2)) and torch.equal(bank.handle.at, bank.handle.a.transpose(1, 2))


@gpu
@pytest.mark.parametrize("rows_per", [1, 77, 256])
def test_agrees_with_the_single_adapter_linear(rows_per):
    """One adapter for every request is what ops.lora_linear computes with a scale of one (both round T and the output to bf16)."""
    gen = torch.Generator().manual_seed(9)
    K, N, r, nb = 320, 640, 32, 4
    host = lora.LoRACompatibleLinear(K, N).to(DEV, torch.bfloat16)
    layer = lora.LoRALinearLayer(K, N, r).to(DEV)
    with torch.no_grad():
        layer.down.weight.copy_((torch.randn(r, K, generator=gen) / r).to(torch.bfloat16))
        layer.up.weight.copy_((0.1 * torch.randn(N, r, generator=gen)).to(torch.bfloat16))
    host.set_lora_layer(layer)
    x = torch.randn(nb, rows_per, K, generator=gen).to(torch.bfloat16).to(DEV)
    with torch.no_grad():
        want = host(x, 1.0).reshape(-1, N).float()
        bank = adapters.AdapterBank.from_layers([layer, layer])
        got = ops.adapter_linear(x.reshape(-1, K), ops.PackedLinear(host.weight, host.bias), bank, adapters.RequestPlan([0, 1, 1, 0])).float()
    # both are within (2^-8 of the value + 2^-8 sum|B||T|) of the 64-bit value; the sum of the two bounds
    t = x.reshape(-1, K).double() @ layer.down.weight.double().t()
    # (the single-adapter linear rounds T twice: T and T * scale)
    bound = 2 * HALF * want.double().abs() + 3.1 * HALF * (t.abs() @ layer.up.weight.double().abs().t()) + 1e-3
    assert ((got - want).double().abs() <= bound).all()


def test_gradient_formula_against_differences():
    """The 64-bit formulas that the kernels are held to, against central differences (the map is linear in each argument: exact up to rounding)."""
    d, lengths, rows, ids, equal = make("ragged", 7)
    (y, dx, dA, dB), _ = reference(d, rows, ids, True, d["x"])
    gen = torch.Generator().manual_seed(2)
    for key, grad in (("x", dx), ("down", dA), ("up", dB)):
        v = torch.randn(d[key].shape, generator=gen, dtype=torch.float64)
        hi, lo = dict(d), dict(d)
        hi[key], lo[key] = d[key].double() + 0.5 * v, d[key].double() - 0.5 * v
        num = sum(s * (reference(a, rows, ids, True, a["x"])[0][0] * d["dy"].double()).sum() for s, a in ((1, hi), (-1, lo)))
        assert abs(num - (grad * v).sum()) <= 1e-10 * (grad.abs() * v.abs()).sum()


@gpu
def test_two_threads_with_one_bank_and_one_plan():
    """Calls with different row counts on threads and streams of their own, against the same calls one after the other."""
    d, lengths, rows, ids, equal = make("equal_77", 6)
    packed, bank, plan = handles(d, lengths, ids, equal, True)
    n = plan.requests
    xs = [torch.randn(n * k, d["x"].shape[1], generator=torch.Generator().manual_seed(k)).to(DEV, torch.bfloat16) for k in (1, 3, 7, 20)]

    def step(x):
        x = x.detach().requires_grad_(True)
        y = ops.adapter_linear(x, packed, bank, plan)
        return (y.detach(),) + torch.autograd.grad(y, (x, bank.down, bank.up), torch.ones_like(y))
    fresh = adapters.RequestPlan(plan.adapters)
    want = [step(x) for x in xs]
    plan = fresh
    got, errors = [None] * len(xs), []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i] = step(xs[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(xs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(want, got):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


@gpu
@pytest.mark.parametrize("trainable", [False, True])
def test_banks_and_plans_are_copied_and_pickled(trainable):
    d, lengths, rows, ids, equal = make("ragged", 12)
    packed, bank, plan = handles(d, lengths, ids, equal, trainable)
    x = d["x"].to(DEV)
    with torch.no_grad():
        want = ops.adapter_linear(x, packed, bank, plan)
        for b, p in ((copy.deepcopy(bank), copy.deepcopy(plan)), (pickle.loads(pickle.dumps(bank)), pickle.loads(pickle.dumps(plan)))):
            assert b.down is not bank.down and b.down.data_ptr() != bank.down.data_ptr() and len(b.parameters()) == len(bank.parameters())
            assert torch.equal(ops.adapter_linear(x, packed, b, p), want)


@gpu
def test_inference_mode():
    d, lengths, rows, ids, equal = make("ragged", 13)
    packed, bank, plan = handles(d, lengths, ids, equal, False)
    x = d["x"].to(DEV)
    gamma = torch.ones(x.shape[1], device=DEV, requires_grad=True)
    with torch.no_grad():
        want, norm = ops.adapter_linear(x, packed, bank, plan), ops.layernorm_train(x, gamma)
    for trainable in (False, True):
        with torch.inference_mode():
            xi = d["x"].to(DEV)
            _, bank, plan = handles({k: v.clone() if torch.is_tensor(v) else v for k, v in d.items()}, lengths, ids, equal, trainable)
            moved = adapters.AdapterBank(d["down"].to(DEV), d["up"].to(DEV), ranks=d["ranks"], scales=d["scales"])
            for b in (bank, moved):
                assert torch.equal(ops.adapter_linear(xi, packed, b, plan), want)
            for ckpt8 in (False, True):
                y, skip = ops.layernorm_train_res(xi, gamma, ckpt8=ckpt8)
                assert torch.equal(y, norm) and torch.equal(skip, xi)
            assert torch.equal(ops.act8_pack(xi).unpack(), ops.act8_pack(x).unpack())
    y = ops.adapter_linear(x, packed, bank, plan)               # a bank made there trains outside
    torch.autograd.grad(y, bank.parameters(), d["dy"].to(DEV))


@gpu
def test_frozen_bank_captures_without_gradients():
    """An input that asks for a gradient is no reason to lay out the transposed stacks where gradients are off."""
    d, lengths, rows, ids, equal = make("ragged", 7)
    packed, bank, plan = handles(d, lengths, ids, equal, False)
    x = d["x"].to(DEV).requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad():
        want = ops.adapter_linear(x, packed, bank, plan)
        with torch.cuda.graph(graph):
            y = ops.adapter_linear(x, packed, bank, plan)
    for _ in range(2):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


@gpu
def test_captured_backward_next_to_a_live_eager_graph_is_refused():
    d, lengths, rows, ids, equal = make("ragged", 8)
    packed, bank, plan = handles(d, lengths, ids, equal, True)
    x, dy = d["x"].to(DEV), d["dy"].to(DEV)
    step = lambda: torch.autograd.grad(ops.adapter_linear(x, packed, bank, plan), (bank.down, bank.up), dy)  # noqa: E731
    want = step()
    alive = ops.adapter_linear(x, packed, bank, plan)
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
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_the_binding_uses_the_library_that_is_loaded(tmp_path):
    """AQL_LIB selects the kernel library for the operators bound in C++ as well."""
    other = tmp_path / "other.so"
    shutil.copy(_lib.LIB_PATH, other)
    code = ("import torch\nfrom aqualora_amd import _lib\n_lib.native()\n"
            "maps = {l.split()[-1] for l in open('/proc/self/maps') if l.strip().endswith('.so')}\n"
            "print(sorted(m for m in maps if m.endswith('other.so') or m.endswith('libaqualora_hip.so')))")
    out = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, AQL_LIB=str(other)), cwd=os.path.dirname(os.path.dirname(_lib.__file__)),
                         capture_output=True, text=True)
    assert out.returncode == 0, out.stderr
    assert out.stdout.strip() == str([str(other)])


def test_refusals_without_a_gpu():
    with pytest.raises(_lib.AqlError):
        adapters.RequestPlan([0], device="cpu")
    with pytest.raises(_lib.AqlError):
        adapters.AdapterBank(torch.zeros(1, 4, 8), torch.zeros(1, 8, 4), device="cpu")
    lib, p = _lib.load(), _lib.c_p(4096)               # p is never dereferenced: every call is refused on the host

    def linear(M=64, N=64, K=64, R=8, ldx=64, X=p, T=p, slots=2, nseg=1, unit=1, seg=p, parts=1):
        return lib.aql_adapter_linear(X, ldx, p, K, None, None, 0, p, N, M, N, K, p, p, p, p, R, seg, unit, nseg, slots, 1, T, parts, None)
    for kw in (dict(N=60), dict(K=60, ldx=64), dict(ldx=56), dict(R=4), dict(R=0), dict(X=None), dict(T=None), dict(slots=0), dict(slots=17), dict(unit=0),
               dict(seg=None), dict(nseg=-1), dict(X=_lib.c_p(4104)), dict(M=-1), dict(M=1 << 31), dict(ldx=1 << 21), dict(parts=2)):
        assert linear(**kw) != 0, kw
    assert linear(M=0) == 0
    assert lib.aql_adapter_down(p, 64, p, p, 64, 64, p, p, p, 8, p, 1, 1, 2, p, 3, None) != 0       # both sources
    assert lib.aql_adapter_down(None, 0, None, None, 64, 64, p, p, p, 8, p, 1, 1, 2, p, 3, None) != 0
    assert lib.aql_adapter_down(p, 1 << 21, None, None, 64, 64, p, p, p, 8, p, 1, 1, 2, p, 3, None) != 0     # past the copies' 32-bit offsets
    assert lib.aql_adapter_down(None, 0, p, p, 64, 1 << 21, p, p, p, 8, p, 1, 1, 2, p, 3, None) != 0
    need = lib.aql_adapter_wgrad_scratch_floats(64, 2, 64, 64, 8)
    assert need > 0 and lib.aql_adapter_wgrad_scratch_floats(1 << 30, 60000, 1 << 14, 1 << 14, 1024) == -1
    assert 0 < lib.aql_adapter_wgrad_scratch_floats(64, 2, 64, 0, 8) < need
    assert lib.aql_adapter_wgrad_scratch_floats(64, 2, -128, 64, 8) == lib.aql_adapter_wgrad_scratch_floats(64, 2, 0, 64, 8) > 0
    assert lib.aql_adapter_wgrad_scratch_floats(64, 2, -5, -1, 8) == 0 == lib.aql_adapter_wgrad_scratch_floats(0, 0, 64, 64, 8)

    def wgrad(X=p, codes=None, r=8, rows=64, n=need, G=3, K=64, unit=1, dA=p, dB=p, dY=p, dT=p):
        return lib.aql_adapter_wgrad(dT, X, 64, codes, codes, K, dA, p, dY, 64, 64, dB, 64, G, 8, r, p, p, p, p, 2, 3, unit, rows, p, n, None)
    for kw in (dict(codes=p), dict(X=None), dict(r=9), dict(rows=65), dict(n=need - 1), dict(G=0), dict(G=1 << 16), dict(K=60), dict(unit=0), dict(unit=3),
               dict(dA=None, dB=None), dict(dY=None), dict(dT=None)):
        assert wgrad(**kw) != 0, kw


@gpu
def test_refusals():
    d, lengths, rows, ids, equal = make("ragged", 8)
    packed, bank, plan = handles(d, lengths, ids, equal, True)
    x, res = d["x"].to(DEV), d["res"].to(DEV)
    M = len(x)
    bad = [(x.float(), bank, plan, None), (x[None], bank, plan, None), (x[:, :312], bank, plan, None), (x[:-1], bank, plan, None),
           (x, bank, plan, res.float()), (x, bank, plan, res[:, :-8]), (x, bank, adapters.RequestPlan([7], [M]), None),
           (x, bank, adapters.RequestPlan([0] * 7), None)]                     # 220 rows do not divide among 7
    for xx, b, p, r in bad:
        with pytest.raises(ValueError):
            ops.adapter_linear(xx, packed, b, p, residual=r)
    with pytest.raises(_lib.AqlError):
        ops.adapter_linear(x.cpu(), packed, bank, plan)
    other = adapters.AdapterBank(torch.zeros(1, 4, 64), torch.zeros(1, 328, 4))
    with pytest.raises(ValueError):
        ops.adapter_linear(x, packed, other, plan)
    for args in ((torch.zeros(2, 4, 8), torch.zeros(2, 8, 5)), (torch.zeros(2, 4, 8), torch.zeros(3, 8, 4)), (torch.zeros(4, 8), torch.zeros(8, 4)),
                 (torch.zeros(2, 4, 9), torch.zeros(2, 8, 4)), (torch.zeros(2, 4, 8).half(), torch.zeros(2, 8, 4).half()),
                 (torch.zeros(2, 1025, 8), torch.zeros(2, 8, 1025))):
        with pytest.raises(ValueError):
            adapters.AdapterBank(*args)
    for kw in (dict(ranks=[4]), dict(ranks=[4, 5]), dict(scales=[1.0])):
        with pytest.raises(ValueError):
            adapters.AdapterBank(torch.zeros(2, 4, 8), torch.zeros(2, 8, 4), **kw)
    for a in (([-2], [3]), ([0], [3, 4]), ([0], [-1])):
        with pytest.raises(ValueError):
            adapters.RequestPlan(*a)


@gpu
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(grad):
    """A tangent of any differentiable input is refused, not dropped, whether or not reverse gradients are asked for."""
    d, lengths, rows, ids, equal = make("ragged", 14)
    packed, bank, plan = handles(d, lengths, ids, equal, True)
    x, res = d["x"].to(DEV), d["res"].to(DEV)
    fw = torch.autograd.forward_ad
    with torch.set_grad_enabled(grad), fw.dual_level():
        for xd, rd in ((fw.make_dual(x, torch.ones_like(x)), res), (x, fw.make_dual(res, torch.ones_like(res)))):
            with pytest.raises(RuntimeError):
                ops.adapter_linear(xd, packed, bank, plan, residual=rd)
        ops.adapter_linear(x, packed, bank, plan, residual=res)


def test_plans_of_adapters_that_no_bank_holds_are_refused():
    """A bank has at most 65535 adapters; the tables are as long as the largest number, and 32 bits wide."""
    for ids in ([0, 65535], [1 << 31], [(1 << 32) + 3], [-2], [0, -(1 << 32)]):
        with pytest.raises(ValueError, match="numbered"):
            adapters.RequestPlan(ids)


@gpu
def test_projections_that_do_not_fit_together_are_refused():
    d, lengths, rows, ids, equal = make("ragged", 16)
    packed, bank, plan = handles(d, lengths, ids, equal, False)
    x = d["x"].to(DEV)
    for name, value in (("bias", packed.bias[:-8]), ("bias", packed.bias.float()), ("bias", packed.bias.cpu()), ("wt", packed.wt[:, :-8].contiguous()), ("wt", packed.w.t()),
                        ("w", packed.w.float()), ("w", packed.w[0])):
        bad = copy.copy(packed)
        setattr(bad, name, value)
        with pytest.raises(ValueError):
            ops.adapter_linear(x, bad, bank, plan)
    bad = copy.copy(packed)
    bad.bias = None
    ops.adapter_linear(x, bad, bank, plan)
