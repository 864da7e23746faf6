"""layernorm_train_res where one of its two outputs goes unused, against the definition."""
import pytest
import torch

from aqualora_amd import ops
from tests.test_layernorm_train import check, codes64, inputs, reference

DEV = "cuda"
gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("ckpt8", [False, True])
@pytest.mark.parametrize("weight", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_only_the_residual_output_is_used(dtype, weight, ckpt8):
    """Its gradient comes back bit for bit, also in rows whose statistics are NaN; the weights have none."""
    x, g, b, _, dres = inputs(40, 203, dtype, 31)
    x[3, 7], x[5, 0] = float("nan"), float("inf")
    xd, gd, bd = x.to(DEV).requires_grad_(True), g.to(DEV, weight).requires_grad_(True), b.to(DEV, weight).requires_grad_(True)
    _, skip = ops.layernorm_train_res(xd, gd, bd, ckpt8=ckpt8)
    dx, dg, db = torch.autograd.grad(skip, (xd, gd, bd), dres.to(DEV))
    assert torch.equal(dx.cpu(), dres)
    assert dg.dtype == db.dtype == weight and (dg == 0).all() and (db == 0).all()
    y, skip = ops.layernorm_train_res(xd, gd, bd, ckpt8=ckpt8)
    skip.backward(dres.to(DEV))
    assert torch.equal(xd.grad.cpu(), dres)


@gpu
@pytest.mark.parametrize("ckpt8", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_only_the_normalised_output_is_used(dtype, ckpt8):
    x, g, b, dy, _ = inputs(40, 203, dtype, 32)
    xd, gd, bd = (t.to(DEV).requires_grad_(True) for t in (x, g, b))
    y, _ = ops.layernorm_train_res(xd, gd, bd, ckpt8=ckpt8)
    grads = torch.autograd.grad(y, (xd, gd, bd), dy.to(DEV))
    ref, slack = reference(x, codes64(x) if ckpt8 else x, g, b, dy, None, 1e-5)
    for n, a, r, s, t in zip(("dx", "dgamma", "dbeta"), grads, ref[1:], slack[1:], (dtype, torch.float32, torch.float32)):
        check(n, a, r, s, t)
    want = torch.autograd.grad(ops.layernorm_train(xd, gd, bd, ckpt8=ckpt8), (xd, gd, bd), dy.to(DEV))
    assert all(torch.equal(a, c) for a, c in zip(grads, want))


@gpu
def test_neither_output_of_a_chain_is_lost():
    """Both used, one, the other: what autograd makes of the plain form in 64 bits, from the pattern of gradients alone."""
    x, g, b, dy, dres = inputs(17, 64, torch.float32, 33)
    for use in ((True, True), (True, False), (False, True)):
        xd, gd = x.to(DEV).requires_grad_(True), g.to(DEV).requires_grad_(True)
        y, skip = ops.layernorm_train_res(xd, gd, b.to(DEV))
        sum(((o * w.to(DEV)).sum() for o, w, u in zip((y, skip), (dy, dres), use) if u)).backward()
        zero = torch.zeros_like(dy)
        ref, slack = reference(x, x, g, b, dy if use[0] else zero, dres if use[1] else None, 1e-5)
        check("dx", xd.grad, ref[1], slack[1], torch.float32)
        check("dgamma", gd.grad, ref[2], slack[2], torch.float32)


@gpu
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(grad):
    x, g, b, dy, _ = (t.to(DEV) for t in inputs(5, 64, torch.float32, 34))
    fw = torch.autograd.forward_ad
    with torch.set_grad_enabled(grad), fw.dual_level():
        for args in ((fw.make_dual(x, dy), g, b), (x, fw.make_dual(g, b), b), (x, g, fw.make_dual(b, g))):
            with pytest.raises((RuntimeError, NotImplementedError)):
                ops.layernorm_train(*args)


@gpu
def test_a_node_behind_it_that_has_no_gradient():
    class Stop(torch.autograd.Function):
        @staticmethod
        def forward(ctx, y):
            return y * 2

        @staticmethod
        def backward(ctx, g):
            return None
    x, g, b, *_ = (t.to(DEV) for t in inputs(5, 64, torch.float32, 35))
    x, g = x.requires_grad_(True), g.requires_grad_(True)
    for f in (ops.layernorm_train, lambda *a: ops.layernorm_train_res(*a)[0]):
        (Stop.apply(f(x, g, b)).sum() + 0 * x.sum()).backward()
        assert (x.grad == 0).all() and g.grad is None
