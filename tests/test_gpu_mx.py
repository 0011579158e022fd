"""Microscaled 4-bit matrices on the B200: quantisation bit for bit against a plain 64-bit rounding, and the product.

Operands' values are known exactly (a few bits each), so the product's only errors are the fp32 accumulation and the output's
one rounding.  With the scales of a matrix within a factor of 2^4 of each other every partial sum is a multiple of one
power of two and below 2^24 of it: exact in any order, and the output has to be equal bit for bit without a transcendental
activation.
"""

import pytest
import torch

from tests import _mx
from tests.test_gpu_projection import act64, slope64

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def spread(rows, k, seed, dtype, most=20):
    g = gen(seed)
    x = torch.randn(rows, k, device=DEV, generator=g)
    x *= torch.exp2(torch.randint(-most, most + 1, (rows, k), device=DEV, generator=g) * (torch.rand(rows, k, device=DEV, generator=g) < 0.1))
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 32), (2, 31), (3, 33), (127, 256), (129, 257), (300, 4095), (64, 4096),
                                    (1000, 100), (5, 70_001), (2000, 768)])
def test_quantize(pkg, rows, k, dtype):
    x = spread(rows, k, rows + k, dtype)
    q = pkg.mx.quantize(x)
    want, e = _mx.rounded(x, _mx.E2M1, 2)
    assert torch.equal(_mx.unpack(q.codes, q.scales, k), want)
    assert torch.equal(pkg.mx.dequantize(q, dtype=torch.float32).double(), want)
    assert torch.equal(pkg.mx.dequantize(q).double(), want)  # two bits: exact in bf16
    # what lies past the matrix: codes zero, scales zero
    flat = torch.stack((q.codes & 15, q.codes >> 4), -1).view(rows, -1)
    assert not bool(flat[:, k:].any())
    full = q.scales.view(*q.scales.shape[:2], 2, 32, 4, 4).permute(0, 4, 3, 1, 2, 5).reshape(q.scales.shape[0] * 128, -1)
    nb = -(-k // 32)
    assert torch.equal(full[:rows, :nb].int() - 127, e.int()) and not bool(full[rows:].any()) and not bool(full[:, nb:].any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 5, 129, 1000])
@pytest.mark.parametrize("k", [1, 8, 32, 40, 60, 64, 72, 96, 100, 120, 128, 136, 576, 768])
def test_short_rows(pkg, rows, k, dtype):
    """Several rows a warp, aligned or not, from strided rows too; the layout's padding is zero."""
    x = (torch.randn(rows, k + 8, device=DEV, generator=gen(rows + k)) * 3).to(dtype)
    for part in (x[:, :k], x[:, :k].contiguous(), x[:, 3:3 + k]):
        q = pkg.mx.quantize(part)
        want = _mx.four(part)
        assert torch.equal(_mx.unpack(q.codes, q.scales, k)[:, :k], want)
        for out in (torch.float32, torch.bfloat16):
            assert torch.equal(pkg.mx.dequantize(q, dtype=out).double(), want)
        blocks = -(-k // 32)
        tiles = q.scales.view(q.scales.shape[0], q.scales.shape[1], 2, 32, 4, 4).permute(0, 4, 3, 1, 2, 5).reshape(q.scales.shape[0] * 128, -1)
        assert int(tiles[rows:].sum()) == 0 and int(tiles[:, blocks:].sum()) == 0


def test_every_value_of_a_block(pkg):
    """Every fp32 magnitude near a rounding border of the grid, of either sign, at scales over the whole range."""
    grid = torch.tensor(_mx.E2M1, dtype=torch.float64)
    mids = torch.cat([(grid[1:] + grid[:-1]) / 2, grid[1:], torch.tensor([7.0, 7.999])])
    near = torch.cat([mids.float(), torch.nextafter(mids.float(), torch.tensor(0.0)), torch.nextafter(mids.float(), torch.tensor(9.0))])
    near = near[near < 8]
    rows = []
    for e in list(range(-130, 125, 5)) + [125]:
        block = torch.ldexp(near.double(), torch.tensor(e)).float()
        for part in block.split(15):
            row = torch.zeros(32)
            row[0] = torch.ldexp(torch.tensor(4.0, dtype=torch.float64), torch.tensor(e)).float()
            row[1:1 + len(part)] = part
            row[16:16 + len(part)] = -part
            rows.append(row)
    x = torch.stack(rows).to(DEV)
    assert bool(torch.isfinite(x).all())
    q = pkg.mx.quantize(x)
    assert torch.equal(_mx.unpack(q.codes, q.scales, 32), _mx.four(x))
    assert torch.equal(pkg.mx.dequantize(q, dtype=torch.float32).double(), _mx.four(x))


def test_small_bf16_blocks(pkg):
    """Blocks down to bf16's smallest numbers, whose scale is the smallest there is."""
    g = gen(2)
    x = torch.randn(300, 32, device=DEV, generator=g) * torch.exp2(torch.randint(-133, -115, (300, 1), device=DEV, generator=g).double()).float()
    for v in (x, x.bfloat16()):
        q = pkg.mx.quantize(v)
        want = _mx.four(v)
        assert torch.equal(_mx.unpack(q.codes, q.scales, 32), want)
        assert torch.equal(pkg.mx.dequantize(q, dtype=torch.float32).double(), want)
        assert torch.equal(pkg.mx.dequantize(q), want.float().bfloat16())


def test_not_finite_blocks(pkg):
    x = torch.randn(4, 96, device=DEV)
    x[0, 3], x[1, 40], x[2, 95] = float("nan"), float("inf"), -float("inf")
    for dtype in (torch.float32, torch.bfloat16):
        y = pkg.mx.dequantize(pkg.mx.quantize(x.to(dtype)), dtype=dtype)
        want = _mx.four(torch.nan_to_num(x.to(dtype), 0, 0, 0)).to(dtype)
        want[0, :32] = want[1, 32:64] = want[2, 64:] = float("nan")
        assert torch.equal(torch.nan_to_num(y, 9e9), torch.nan_to_num(want, 9e9))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_strides_and_shapes(pkg, dtype):
    x = spread(6, 200, 3, dtype)
    for shift, wide in ((0, 0), (1, 0), (0, 3), (5, 8)):
        buf = torch.full((6 * (200 + wide) + shift,), 55.0, device=DEV, dtype=dtype)
        v = buf[shift:].view(6, 200 + wide)[:, :200]
        v.copy_(x)
        assert torch.equal(pkg.mx.dequantize(pkg.mx.quantize(v), dtype=dtype).double(), _mx.four(x))
    q = pkg.mx.quantize(x.view(2, 3, 200))
    assert q.shape == (2, 3, 200) and torch.equal(pkg.mx.dequantize(q).double().view(6, 200), _mx.four(x))
    one = pkg.mx.quantize(x[0])
    assert one.shape == (200,) and torch.equal(pkg.mx.dequantize(one).double(), _mx.four(x[:1])[0])
    none = pkg.mx.quantize(x[:0])
    assert pkg.mx.dequantize(none).shape == (0, 200)
    assert torch.equal(pkg.mx.dequantize(pkg.mx.quantize(x.t().contiguous().t())).double(), _mx.four(x))


SIZES = [(1, 1, 1), (9, 1, 1), (130, 1, 300), (5, 32, 127), (1, 30, 7), (1, 4096, 768), (2, 768, 768), (3, 72, 5), (4, 2049, 100), (5, 64, 40), (16, 4096, 777), (17, 641, 333),
         (64, 768, 6562), (100, 200, 129), (128, 64, 256), (129, 1000, 257), (513, 768, 1537), (1000, 256, 4096),
         (2050, 80, 64), (31, 8192, 40), (1300, 2048, 1024), (300, 33, 4000), (257, 515, 513)]


def operands(pkg, n, k, m, seed):
    """Rows and weights whose products and sums are exact in fp32 in any order."""
    g = gen(seed)

    def small(rows):  # a few non-zero values, scales within 2^2
        v = torch.randint(-12, 13, (rows, k), device=DEV, generator=g).float() * 0.5
        v *= torch.exp2(torch.randint(0, 3, (rows, 1), device=DEV, generator=g))
        return torch.where(torch.rand(rows, k, device=DEV, generator=g) < min(1.0, 48.0 / k), v, torch.zeros_like(v)).bfloat16()

    x, w = small(n), small(m) * 0.125
    b = torch.randint(-16, 17, (m,), device=DEV, generator=g).bfloat16() * 0.25
    r = torch.randint(-40, 41, (n, m), device=DEV, generator=g).bfloat16() * 0.25
    dy = torch.randint(-4, 5, (n, m), device=DEV, generator=g).bfloat16() * 0.25
    return x, w, b, r, dy


@pytest.mark.parametrize("activation", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("n,k,m", SIZES)
def test_product(pkg, n, k, m, activation):
    x, w, b, r, _ = operands(pkg, n, k, m, n + k + m)
    q = pkg.mx.quantize(w)
    for bias, res in ((b, r), (None, None), (b, None), (None, r)):
        st = torch.zeros(1, dtype=torch.int32, device=DEV)
        y = pkg.mx.linear(x, q, bias, activation=activation, residual=res, status=st)
        z = _mx.four(x) @ _mx.four(w).t() + (0 if bias is None else bias.double())
        want = act64(z, activation) + (0 if res is None else res.double())
        assert y.dtype == torch.bfloat16 and y.shape == (n, m) and int(st) == 0
        if activation in (None, "relu"):
            assert torch.equal(y, want.float().bfloat16())
        else:
            tol = 2.0 ** -8 * want.abs() + 2.0 ** -20 * (1 + z.abs())
            assert bool(((y.double() - want).abs() <= tol).all())
    assert torch.equal(pkg.mx.linear(pkg.mx.quantize(x), q, None, activation=activation, residual=r), y)


@pytest.mark.parametrize("n,k,m", [(1, 4096, 300), (7, 1000, 257), (40, 4096, 513), (300, 4096, 300), (1100, 768, 1537)])
def test_product_of_any_values(pkg, n, k, m):
    """Sums that round: fp32 accumulation of k products is off by at most k 2^-23 of their magnitudes' sum (a truncation an
    addition), the output by half a step of bf16."""
    x, w = spread(n, k, n, torch.bfloat16, most=6), spread(m, k, m, torch.bfloat16, most=6)
    y = pkg.mx.linear(x, pkg.mx.quantize(w))
    xd, wd = _mx.four(x), _mx.four(w)
    want, size = xd @ wd.t(), xd.abs() @ wd.abs().t()
    assert bool(((y.double() - want).abs() <= k * 2.0 ** -23 * size + 2.0 ** -8 * want.abs()).all())


@pytest.mark.parametrize("n", [1, 3, 200, 700])
def test_not_finite_rows(pkg, n):
    """NaN or an infinity in x makes its row of the output NaN, in the weight its column; the others stay as they were."""
    x, w, b, _, _ = operands(pkg, n, 544, 300, 5)
    clean = pkg.mx.linear(x, pkg.mx.quantize(w), b)
    x2, w2 = x.clone(), w.clone()
    x2[n // 2, 100] = float("nan")
    w2[7, 540] = float("inf")
    y = pkg.mx.linear(x2, pkg.mx.quantize(w2), b)
    bad = torch.zeros(n, 300, dtype=torch.bool, device=DEV)
    bad[n // 2] = bad[:, 7] = True
    assert bool(torch.isnan(y[bad]).all()) and torch.equal(y[~bad], clean[~bad])


@pytest.mark.parametrize("n", [1, 40, 300])
@pytest.mark.parametrize("activation", [None, "relu", "gelu", "silu"])
def test_infinite_and_far_preactivations(pkg, n, activation):
    """Columns whose bias is far out: what the activation is there, NaN for NaN, the others as they were."""
    x, w, b, _, _ = operands(pkg, n, 64, 200, 3)
    q = pkg.mx.quantize(w)
    clean = pkg.mx.linear(x, q, b, activation=activation)
    far = b.clone()
    far[5], far[100], far[101], far[130], far[199] = float("inf"), 3e38, -3e38, float("nan"), 1e4
    y = pkg.mx.linear(x, q, far, activation=activation)
    keep = torch.ones(200, dtype=torch.bool, device=DEV)
    keep[[5, 100, 101, 130, 199]] = False
    assert torch.equal(y[:, keep], clean[:, keep])
    assert bool((y[:, 5] == float("inf")).all()) and bool(torch.isnan(y[:, 130]).all())
    assert torch.equal(y[:, 100], far[100].expand(n))  # the sums are far below a step of 3e38
    assert torch.equal(y[:, 101], far[101].expand(n) if activation is None else torch.zeros_like(y[:, 101]))
    assert bool(((y[:, 199].double() - 1e4).abs() <= 2.0 ** -8 * 1e4 + 64 * 12 * 12 * 2).all())


@pytest.mark.parametrize("n", [1, 3, 40, 300])
@pytest.mark.parametrize("far", [100, 120])
def test_scales_whose_product_passes_fp32(pkg, n, far):
    """Exact in any order: powers of two in one block, a small product in another."""
    def product(a, b):
        x, w = torch.zeros(n, 256, device="cuda", dtype=torch.bfloat16), torch.zeros(320, 256, device="cuda", dtype=torch.bfloat16)
        x[:, 0], x[:, 40], w[:, 40] = 2.0 ** a, 1.0, 3.0
        for at, value in b.items():
            w[:, at] = 2.0 ** value
        return pkg.mx.linear(x, pkg.mx.quantize(w)).float().unique().tolist()
    assert product(far, {1: far}) == [3.0]  # zeros met by 2^far on either side
    assert product(far, {0: -far}) == [4.0]
    assert product(far, {0: far}) == [float("inf")]
    assert product(-far, {0: -far}) == [3.0]


@pytest.mark.parametrize("activation", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("n,k,m", [(1, 30, 7), (3, 72, 5), (17, 641, 333), (129, 1000, 257), (513, 768, 1537), (64, 768, 6562)])
def test_gradient(pkg, n, k, m, activation):
    """As the projection's: the slope comes from a pre-activation in fp16 (2^-12 of z times the curvature) and dz is rounded to
    bf16; without a transcendental activation all is exact."""
    x, w, b, r, dy = operands(pkg, n, k, m, n + k + m)
    q = pkg.mx.quantize(w)
    leaves = [v.detach().requires_grad_(True) for v in (x, b, r)]
    y = pkg.mx.linear(leaves[0], q, leaves[1], activation=activation, residual=leaves[2])
    assert torch.equal(y, pkg.mx.linear(x, q, b, activation=activation, residual=r))
    dx, db, dr = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(dr, dy) and dx.shape == x.shape
    wd = _mx.four(w)
    z = _mx.four(x) @ wd.t() + b.double()
    dz = dy.double() * slope64(z, activation)
    curve = {None: 0.0, "relu": 0.0, "silu": 0.5, "gelu": 0.8}[activation]
    exact = activation in (None, "relu")
    tz = 0 if exact else dy.double().abs() * (2.0 ** -11 * curve * z.abs() + 2.0 ** -18)
    td = tz if exact else tz + 2.0 ** -8 * (dz.abs() + tz)
    for got, want, tol in ((dx, dz @ wd, 0 if exact else td @ wd.abs()),
                           (db, dz.sum(0), 0 if exact else tz.sum(0) + 2.0 ** -20 * dz.abs().sum(0))):
        if exact:
            assert torch.equal(got, want.float().bfloat16())
        else:
            assert bool(((got.double() - want).abs() <= tol * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs() + 2.0 ** -60).all())


def test_gradients_apart_and_of_other_forms(pkg):
    x, w, b, r, dy = operands(pkg, 20, 96, 50, 9)
    q = pkg.mx.quantize(w)
    for act in (None, "silu"):
        leaves = [v.detach().requires_grad_(True) for v in (x, b, r)]
        want = torch.autograd.grad(pkg.mx.linear(leaves[0], q, leaves[1], activation=act, residual=leaves[2]), leaves, dy)
        for i in range(3):
            only = [v.detach().requires_grad_(i == j) for j, v in enumerate((x, b, r))]
            got, = torch.autograd.grad(pkg.mx.linear(only[0], q, only[1], activation=act, residual=only[2]), only[i], dy)
            assert torch.equal(got, want[i])
        # without a bias the residual's edge is another; of a quantised x only bias and residual have gradients
        dr, = torch.autograd.grad(pkg.mx.linear(x, q, activation=act, residual=leaves[2]), leaves[2], dy)
        assert torch.equal(dr, dy)
        y = pkg.mx.linear(pkg.mx.quantize(x), q, leaves[1], activation=act, residual=leaves[2])
        db, dr = torch.autograd.grad(y, leaves[1:], dy)
        assert torch.equal(db, want[1]) and torch.equal(dr, dy)
    y3 = pkg.mx.linear(x.view(4, 5, 96), q, b, residual=r.view(4, 5, 50))
    assert y3.shape == (4, 5, 50) and torch.equal(y3.view(20, 50), pkg.mx.linear(x, q, b, residual=r))
    assert torch.equal(pkg.mx.linear(x[0], q, b), pkg.mx.linear(x[:1], q, b)[0])
    assert pkg.mx.linear(x[:0], q, b).shape == (0, 50)


@pytest.mark.parametrize("n", [1, 40, 300])
def test_strides_of_rows(pkg, n):
    x, w, b, r, _ = operands(pkg, n, 136, 200, 4)
    q = pkg.mx.quantize(w)
    want = pkg.mx.linear(x, q, b, activation="relu", residual=r)
    for shift, wide in ((1, 0), (0, 1), (3, 5), (8, 8)):
        def off(v):
            buf = torch.full((v.numel() + n * wide + shift,), 77.0, device=DEV, dtype=torch.bfloat16)
            return buf[shift:].view(n, v.shape[1] + wide)[:, :v.shape[1]].copy_(v)

        bias = torch.zeros(200 + shift, device=DEV, dtype=torch.bfloat16)[shift:].copy_(b)
        assert torch.equal(pkg.mx.linear(off(x), q, bias, activation="relu", residual=off(r)), want)


@pytest.mark.parametrize("n", [1, 16, 300])
def test_capture_replays_with_new_rows(pkg, n):
    x, w, b, r, dy = operands(pkg, n, 768, 600, 8)
    q = pkg.mx.quantize(w)
    xs, graph = x.clone().requires_grad_(True), torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(pkg.mx.linear(xs, q, b, activation="relu"), xs, dy)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        y = pkg.mx.linear(xs, q, b, activation="relu")
        d, = torch.autograd.grad(y, xs, dy)
    for seed in (1, 2):
        x2 = operands(pkg, n, 768, 600, seed)[0]
        with torch.no_grad():
            xs.copy_(x2)
        graph.replay()
        x3 = x2.clone().requires_grad_(True)
        y3 = pkg.mx.linear(x3, q, b, activation="relu")
        assert torch.equal(y, y3) and torch.equal(d, torch.autograd.grad(y3, x3, dy)[0])


def test_a_decode_loop_from_a_4_bit_table(pkg):
    """Token -> row -> 4-bit head -> greedy token, with the same table at both ends, against the loop in 64 bits; finished rows
    sample PAD and look up zeros."""
    g = gen(21)
    table = torch.randn(700, 512, device=DEV, generator=g).bfloat16()
    q, values = pkg.mx.quantize(table), _mx.four(table)
    token = torch.tensor([5, 600, -1, 31], device=DEV)
    for _ in range(4):
        h = pkg.embedding.lookup(token, q, scale=2.0)
        logits = pkg.mx.linear(h, q)
        rows = torch.where(token[:, None] >= 0, values[token.clamp_min(0)] * 2.0, 0.0)
        assert torch.equal(h.double(), rows)
        want = rows @ values.t()  # rows of 4-bit values keep them: their blocks' scales double
        assert bool(((logits.double() - want).abs() <= 512 * 2.0 ** -23 * (rows.abs() @ values.abs().t()) + 2.0 ** -8 * want.abs()).all())
        nxt = pkg.thinker_sampler.argmax(logits)
        lp = pkg.logprobs.token_logprobs(logits, nxt)
        assert torch.equal(lp.rank, torch.zeros_like(nxt))
        token = torch.where(token >= 0, (nxt * 7 + 3) % 700, token)
