"""LayerNorm with weight gradients over more rows than its launches hold at once: every form's second and third turn of the row loop.

A row's result does not depend on where it stands, so y, dx and the codes have the bits of calls on few rows (held to 64 bits elsewhere).  dgamma and dbeta are
sums over all rows: off by at most LR u sum|terms| for the chain of LR = rows / 8 + 100 additions (a group walks over its share of the rows, the groups of a
workgroup and the workgroups follow) and by the error of each xh: relative (64 + 8) u of rstd, and rstd * 64 u mean|x| of the mean."""
import pytest
import torch

from aqualora_amd import ops

DEV = "cuda"
U = 2.0 ** -24
# (rows, columns): a form by its width, in whole chunks of 8 columns and with a tail; rows past its grid
SHAPES = [(33001, 128), (66003, 100), (21001, 256), (41003, 201), (33001, 320), (17003, 333), (9001, 512), (17003, 500), (6001, 1024), (11003, 1001),
          (4999, 1280), (9001, 1411), (2500, 2048), (5003, 2043), (1400, 4096), (2801, 3001), (1300, 8192), (2701, 4097)]
FEW = 500      # rows of a call that every form holds at once


def step(x, gamma, beta, dy, dres, ckpt8):
    xd, g, b = (t.detach().requires_grad_(True) for t in (x, gamma, beta))
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (kept.append(t), t)[1], lambda t: t):
        y, skip = ops.layernorm_train_res(xd, g, b, ckpt8=ckpt8)
    grads = torch.autograd.grad((y, skip), (xd, g, b), (dy, dres))
    return y.detach(), grads[0], [t for t in kept if t is not None and t.dtype == torch.uint8], grads[1:]


@pytest.mark.gpu
@pytest.mark.parametrize("ckpt8", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,C", SHAPES)
def test_rows_beyond_one_launch(M, C, dtype, ckpt8):
    gen = torch.Generator(DEV).manual_seed(M + C)
    rn = lambda *s: torch.randn(s, generator=gen, device=DEV)  # noqa: E731
    x, dy, dres = ((rn(M, C) * torch.exp(rn(C)) + 0.3).to(dtype), rn(M, C).to(dtype), rn(M, C).to(dtype))
    gamma, beta = 1 + 0.3 * rn(C), 0.3 * rn(C)
    y, dx, codes, (dg, db) = step(x, gamma, beta, dy, dres, ckpt8)
    packed = ops.act8_pack(x)
    if ckpt8:
        assert len(codes) == 2 and torch.equal(codes[0], packed.codes) and torch.equal(codes[1], packed.exps)
    for at in range(0, M, FEW):
        rows = slice(at, at + FEW)
        few = step(x[rows], gamma, beta, dy[rows], dres[rows], ckpt8)
        assert torch.equal(y[rows], few[0]) and torch.equal(dx[rows], few[1]), at
    xd, d = x.double(), dy.double()
    seen = packed.unpack(torch.float32).double() if ckpt8 else xd
    mean = xd.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((xd - mean) ** 2).mean(1, keepdim=True) + 1e-5)
    xh = (seen - mean) * rstd
    dmean = 64 * U * xd.abs().mean(1, keepdim=True)
    dxh = rstd * (dmean + 2 * U * (seen - mean).abs()) + xh.abs() * (72 * U + (dmean * rstd) ** 2)
    LR = M // 8 + 100
    for name, got, terms, off in (("dgamma", dg, d * xh, d.abs() * dxh), ("dbeta", db, d, 0 * d)):
        err = (got.double() - terms.sum(0)).abs()
        over = (err - (off.sum(0) + LR * U * terms.abs().sum(0) + U * terms.sum(0).abs())).max()
        assert over <= 0, f"{name}: {over.item():.3e} over its bound"
