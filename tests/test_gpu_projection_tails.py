"""The projection's activations and slopes over their whole range, with tolerances relative to the values themselves.

Forward: one rounding to bf16 (half a step, 2^-8) of a value whose fp32 arithmetic is off by less than 2^-15 of it: ex2's
2^-22, the division's and a polynomial's few 2^-24, and the exponent's own roundings, at most three of 2^-24 of 126, times
ln 2.  Results below the normal range (2^-126) may be any.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def act64(z, kind):
    """In 64 bits, without cancellation: 1 + erf, as which special.ndtr comes on the GPU, loses the tail below -7."""
    return 0.5 * z * torch.special.erfc(-z * 0.5 ** 0.5) if kind == "gelu" else z * torch.sigmoid(z)


def sweep():
    """Every bf16 value of both signs up to 16 but for the smallest, and far ones."""
    bits = torch.arange(0x3000, 0x4180, dtype=torch.int32)  # 4.7e-10 .. 16
    near = bits.to(torch.int16).view(torch.bfloat16)
    far = torch.tensor([0.0, 17.0, 40.0, 80.0, 85.0, 87.0, 88.0, 89.0, 100.0, 1e4, 1e19, 1e30]).bfloat16()
    v = torch.cat([near, far])
    return torch.cat([v, -v]).to(DEV)


@pytest.mark.parametrize("activation", ["gelu", "silu"])
@pytest.mark.parametrize("rows,k", [(1, 8), (3, 64), (8, 64), (100, 72), (40, 4096), (300, 64)])
def test_forward_over_the_range(pkg, activation, rows, k):
    """On the CUDA cores, on whole tiles and on tiles split along k."""
    z = sweep()
    x = torch.zeros(rows, k, device=DEV, dtype=torch.bfloat16)
    w = torch.zeros(z.numel(), k, device=DEV, dtype=torch.bfloat16)
    x[:, k // 2], w[:, k // 2] = 1.0, z
    y = pkg.projection.linear(x, w, activation=activation).double()
    want = act64(z.double(), activation)[None]
    tol = (2.0 ** -8 + 2.0 ** -15) * want.abs() + 2.0 ** -126
    ok = (y - want).abs() <= tol
    assert bool(ok.all()), (z.expand_as(y)[~ok][:8], y[~ok][:8], want.expand_as(y)[~ok][:8], int((~ok).sum()))


def slope64(z, kind):
    if kind == "gelu":
        return 0.5 * torch.special.erfc(-z * 0.5 ** 0.5) + z * torch.exp(-z * z / 2) * (2 * torch.pi) ** -0.5
    s = torch.sigmoid(z)
    return s + z * s * (1 - s)


def curvature64(z, kind):
    if kind == "gelu":
        return torch.exp(-z * z / 2) * (2 * torch.pi) ** -0.5 * (2 - z * z)
    s = torch.sigmoid(z)
    return s * (1 - s) * (2 + z * (1 - 2 * s))


@pytest.mark.parametrize("activation", ["gelu", "silu"])
@pytest.mark.parametrize("rows,k", [(1, 8), (8, 64), (100, 72), (40, 4096), (300, 64)])
def test_gradient_over_the_range(pkg, activation, rows, k):
    """Slopes of pre-activations that need fp32, from the saved fp16 ones: off by half a step of fp16 (2^-11 of z, or 2^-25
    below its normal range) times the curvature, a second order of at most its square, and the slope's own arithmetic; then
    dz's rounding to bf16 (exact once more as the product's result).  Around the slopes' zeros (-0.75, -1.28) a saved bf16
    would be off by eight times as much."""
    g = torch.Generator(device=DEV).manual_seed(rows)
    x0 = (torch.rand(2000, device=DEV, generator=g) * 12 - 8).bfloat16()
    x0[::4] = (torch.rand(500, device=DEV, generator=g) * 1.5 - 2).bfloat16()
    b = ((torch.rand(2000, device=DEV, generator=g) - 0.5) * 2.0 ** -6).bfloat16()
    x = torch.zeros(rows, k, device=DEV, dtype=torch.bfloat16)
    w = torch.zeros(2000, k, device=DEV, dtype=torch.bfloat16)
    x[:, k // 2], w[:, k // 2] = 1.0, x0
    z = x0.double() + b.double()
    dy = torch.randn(rows, 2000, device=DEV, generator=g).bfloat16()
    w.requires_grad_(True)
    bias = b.detach().requires_grad_(True)
    y = pkg.projection.linear(x, w, bias, activation=activation)
    dw, db = torch.autograd.grad(y, (w, bias), dy)
    d = dy.double() * slope64(z, activation)
    step = 2.0 ** -11 * z.abs() + 2.0 ** -25 + 2.0 ** -24  # and z's own rounding to fp32
    each = dy.double().abs() * (step * curvature64(z, activation).abs() + step * step + 2.0 ** -21)
    want, off = d.sum(0), each.sum(0) + 2.0 ** -20 * d.abs().sum(0)
    ok = (db.double() - want).abs() <= off * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs()
    assert bool(ok.all()), (z[~ok][:8], db[~ok][:8], want[~ok][:8], off[~ok][:8])
    rounded = (each + 2.0 ** -8 * (d.abs() + each)).sum(0)
    got = dw[:, k // 2].double()
    ok = (got - want).abs() <= (rounded + 2.0 ** -20 * d.abs().sum(0)) * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs()
    assert bool(ok.all()), (z[~ok][:8], got[~ok][:8], want[~ok][:8])
    assert not bool(dw[:, :k // 2].any()) and not bool(dw[:, k // 2 + 1:].any())
