"""Hooks of saved tensors around the training operators: what comes back as it was saved gives the same bits, wherever it was meanwhile; other things are refused."""
import pytest
import torch

from aqualora_amd import adapters, ops
from tests.test_adapters import handles, make

DEV = "cuda"
gpu = pytest.mark.gpu


def same(t):
    return t


def wide(t):
    """The same values with another row stride."""
    if t.dim() < 2:
        return t.clone()
    out = torch.zeros(t.shape[:-1] + (t.shape[-1] + 24,), dtype=t.dtype, device=t.device)
    out[..., 3:3 + t.shape[-1]] = t
    return out[..., 3:3 + t.shape[-1]]


def turned(t):
    return t.transpose(0, 1).contiguous().transpose(0, 1) if t.dim() >= 2 else t.clone()


def norm(dtype, ckpt8):
    gen = torch.Generator().manual_seed(3)
    rn = lambda *s: torch.randn(s, generator=gen).to(DEV)  # noqa: E731
    big, g, dy, dres = rn(37, 220).to(dtype), (1 + 0.2 * rn(203)).requires_grad_(True), rn(37, 203).to(dtype), rn(37, 203).to(dtype)
    x = big[:, 5:208].detach().requires_grad_(True)
    return (lambda: ops.layernorm_train_res(x, g, None, ckpt8=ckpt8)), (x, g), (dy, dres)


def linear(ckpt8):
    d, lengths, rows, ids, equal = make("ragged", 15)
    packed, bank, plan = handles(d, lengths, ids, equal, True)
    x = d["x"].to(DEV).requires_grad_(True)
    return (lambda: (ops.adapter_linear(x, packed, bank, plan, ckpt8=ckpt8),)), (x, bank.down, bank.up), (d["dy"].to(DEV),)


CALLS = {f"{n}{'_8bit' if c else ''}": (f, a + (c,)) for n, f, a in (("norm_bf16", norm, (torch.bfloat16,)), ("norm_fp32", norm, (torch.float32,)), ("linear", linear, ()))
         for c in (False, True)}


def grads(call, wrt, seeds, pack, unpack):
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        out = call()
    return torch.autograd.grad(out, wrt, seeds)


@gpu
@pytest.mark.parametrize("name", list(CALLS))
def test_tensors_that_come_back(name):
    f, args = CALLS[name]
    call, wrt, seeds = f(*args)
    want = torch.autograd.grad(call(), wrt, seeds)
    for pack, unpack in ((lambda t: t.cpu(), lambda t: t.to(DEV)), (same, wide), (same, turned)):
        got = grads(call, wrt, seeds, pack, unpack)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.autograd.graph.save_on_cpu():
        out = call()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, wrt, seeds), want))


@gpu
@pytest.mark.parametrize("name", list(CALLS))
def test_tensors_that_come_back_otherwise_are_refused(name):
    f, args = CALLS[name]
    call, wrt, seeds = f(*args)
    for unpack in (lambda t: t.cpu(), lambda t: t[:-1], lambda t: t.double(), lambda t: t.reshape(-1)[None], lambda t: t[..., :-1]):
        with pytest.raises(RuntimeError, match="came back"):
            grads(call, wrt, seeds, same, unpack)
