"""Microscaled blocks at the edges of the formats, in rows of every length: borders of rounding at scales over the whole range,
blocks down to the smallest scale, NaN and infinities, for the kernels of short rows and those of long ones (aligned or not, few rows
a warp or many), and for the 8-bit blocks that the projection keeps.  Bit for bit against the rounding in 64 bits: 4-bit values
are two bits times 2^-128 at least, exact in bf16 and fp32.
"""

import pytest
import torch

from tests import _mx
from tests.test_gpu_projection import act64

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
SHAPES = [(7, 32), (7, 128), (9, 160), (300, 257), (12, 4096), (20_011, 257), (10_009, 520), (2500, 4096)]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def border_blocks(grid, top):
    """[blocks, 32]: the largest grid value's power of two first, then values at, above and below each border, either sign."""
    g = torch.tensor(grid, dtype=torch.float64)
    mids = torch.cat([(g[1:] + g[:-1]) / 2, g[1:], torch.tensor([2.0 ** (top + 1) - 2.0 ** (top - 2), 2.0 ** (top + 1) * 0.99])]).float()
    near = torch.cat([mids, torch.nextafter(mids, torch.tensor(0.0)), torch.nextafter(mids, torch.tensor(1e9))])
    near = near[near < 2.0 ** (top + 1)].double()
    rows = []
    for e in [*range(-127 - 3, 125 - top, 7), 127 - top]:
        for part in near.split(15):
            row = torch.zeros(32, dtype=torch.float64)
            row[0] = 2.0 ** top
            row[1:1 + len(part)], row[16:16 + len(part)] = part, -part
            rows.append(torch.ldexp(row, torch.tensor(e)))
    return torch.stack(rows).float().to(DEV)


def small_blocks():
    x = torch.randn(600, 32, device=DEV, generator=gen(2))
    return x * torch.exp2(torch.randint(-140, -112, (600, 1), device=DEV, generator=gen(3)).double()).float()


def laid_out(blocks, rows, k):
    """The blocks one after another, again and again, as [rows, k] (a row's last block cut)."""
    nb = -(-k // 32)
    at = torch.arange(rows * nb, device=DEV) % len(blocks)
    return blocks[at].view(rows, nb * 32)[:, :k].contiguous()


def as_type(x, dtype):
    return x.to(dtype).clamp(torch.finfo(dtype).min, torch.finfo(dtype).max)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,k", SHAPES)
@pytest.mark.parametrize("kind", ["borders", "small"])
def test_blocks(pkg, kind, rows, k, dtype):
    x = as_type(laid_out(border_blocks(_mx.E2M1, 2) if kind == "borders" else small_blocks(), rows, k), dtype)
    wide = torch.zeros(rows, k + 3, device=DEV, dtype=dtype)
    wide[:, 1:1 + k] = x
    want = _mx.four(x)
    for v in (x, wide[:, 1:1 + k]):
        q = pkg.mx.quantize(v)
        assert torch.equal(_mx.unpack(q.codes, q.scales, k), want)
    for out in (torch.float32, torch.bfloat16):
        assert torch.equal(pkg.mx.dequantize(q, dtype=out).double(), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,k", SHAPES)
def test_not_finite(pkg, rows, k, dtype):
    """A block with NaN or an infinity comes back as NaN throughout, its neighbours as they are."""
    x = (torch.randn(rows, k, device=DEV, generator=gen(k)) * 3).to(dtype)
    want = _mx.four(x)
    r = torch.arange(0, rows, 3, device=DEV)
    c = (r * 37 + 5) % k
    x[r, c] = torch.tensor([float("nan"), float("inf"), -float("inf")], device=DEV, dtype=dtype)[r // 3 % 3]
    bad = torch.zeros(rows, -(-k // 32), dtype=torch.bool, device=DEV)
    bad[r, c // 32] = True
    bad = bad.repeat_interleave(32, 1)[:, :k]
    q = pkg.mx.quantize(x)
    for out in (torch.float32, torch.bfloat16):
        y = pkg.mx.dequantize(q, dtype=out).double()
        assert bool(torch.isnan(y[bad]).all()) and torch.equal(y[~bad], want[~bad])


def eight_bits(codes, scales, n):
    return (codes.view(torch.float8_e4m3fn).double() * torch.exp2(scales.double() - 127).t().repeat_interleave(32, 1))[:, :n]


@pytest.mark.parametrize("kind", ["borders", "small"])
@pytest.mark.parametrize("n,k,m", [(5, 64, 288), (300, 64, 288), (300, 256, 1537), (40, 4096, 200), (16, 16384, 256)])
def test_kept_blocks(pkg, kind, n, k, m):
    """x and the pre-activation in 8 bits.  The weight is zero, so that the pre-activation is the bias, exactly."""
    blocks = border_blocks(_mx.E4M3, 8) if kind == "borders" else small_blocks()
    x = as_type(laid_out(blocks, n, k), torch.bfloat16)
    for first in range(0, min(len(blocks), 4 * (-(-m // 32))), -(-m // 32)):
        b = as_type(laid_out(blocks.roll(-first, 0), 1, m), torch.bfloat16)[0]
        w = torch.zeros(m, k, device=DEV, dtype=torch.bfloat16)
        y, xc, xs, zc, zs = torch.ops.minicpmo_sampler.linear_kept(x, w, b, None, 0, True, True, None)
        assert torch.equal(y, b.expand(n, m))
        assert torch.equal(eight_bits(zc, zs, m), _mx.eight(b[None]).expand(n, m))
    assert torch.equal(eight_bits(xc, xs, k), _mx.eight(x))


@pytest.mark.parametrize("activation", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("n,k", [(1, 64), (3, 64), (40, 64), (300, 64), (40, 4096)])
def test_far_preactivations(pkg, n, k, activation):
    """Columns far out but finite, within half a step of the activation in 64 bits (the operands' products are exact there)."""
    g = gen(n)
    x = torch.randint(-12, 13, (n, k), device=DEV, generator=g).bfloat16() * 0.5
    w = torch.randint(-12, 13, (200, k), device=DEV, generator=g).bfloat16() * 0.0625
    b = torch.randint(-16, 17, (200,), device=DEV, generator=g).bfloat16() * 0.25
    b[5], b[60], b[61], b[130], b[199] = 1e4, -1e4, 3e4, -200.0, 150.0
    y = pkg.mx.linear(x, pkg.mx.quantize(w), b, activation=activation).double()
    z = _mx.four(x) @ _mx.four(w).t() + b.double()
    want = act64(z, activation)
    assert bool(((y - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * (1 + z.abs())).all())
