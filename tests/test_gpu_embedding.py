"""``embedding.lookup`` on the B200 against a plain implementation in 64 bits.

A looked-up value is one product, rounded to fp32 and then to the table's type: off by half a step of each, 2^-24 and, for
bf16, 2^-8, relative.  A gradient is a sum of n_v terms in fp32 (error at most n_v 2^-24 of the sum of magnitudes, the
formula's worst case), times the scale, rounded; with small whole numbers it is exact.
"""

import pytest
import torch

from tests import _mx

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8}


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def want_rows(tokens, table, scale):
    v = table.shape[0]
    ok = (tokens >= 0) & (tokens < v)
    rows = table.double()[tokens.clamp(0, v - 1)] * scale
    return torch.where(ok[..., None], rows, torch.zeros_like(rows))


def want_grad(tokens, dy, vocab, scale):
    ok = (tokens >= 0) & (tokens < vocab)
    d = torch.zeros(vocab + 1, dy.shape[-1], dtype=torch.float64, device=DEV)
    d.index_add_(0, torch.where(ok, tokens, vocab), dy.double())
    return d[:-1] * scale


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,vocab,width", [(1, 1, 1), (1, 500, 4096), (3, 7, 33), (64, 1000, 768), (257, 333, 1030),
                                           (1000, 50, 8), (5000, 6562, 96), (31, 100, 20_001), (700, 2000, 1024)])
def test_lookup(pkg, n, vocab, width, dtype):
    g = gen(n + width)
    table = torch.randn(vocab, width, device=DEV, generator=g).to(dtype)
    tokens = torch.randint(-2, vocab, (n,), device=DEV, generator=g)
    for scale in (1.0, 12.0, -0.3):
        st = torch.zeros(1, dtype=torch.int32, device=DEV)
        y = pkg.embedding.lookup(tokens, table, scale=scale, status=st)
        want = want_rows(tokens, table, scale)
        assert y.dtype == dtype and y.shape == (n, width) and int(st) == 0
        assert bool(((y.double() - want).abs() <= want.abs() * (HALF[dtype] + 2.0 ** -23)).all())
        if scale == 1.0:
            assert torch.equal(y.double(), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift,wide", [(0, 0), (1, 0), (0, 1), (3, 8), (8, 24)])
def test_lookup_strides_shapes_and_ranges(pkg, dtype, shift, wide):
    """Tables off their alignment and inside wider ones, tokens of any shape, ids past the table."""
    vocab, width = 77, 264
    buf = torch.randn(vocab * (width + wide) + shift, device=DEV, generator=gen(1)).to(dtype)
    table = buf[shift:].view(vocab, width + wide)[:, :width]
    tokens = torch.tensor([[0, 76, -1], [77, 5, 2 ** 40]], device=DEV)
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    y = pkg.embedding.lookup(tokens, table, status=st)
    assert y.shape == (2, 3, width) and int(st) == 32
    assert torch.equal(y.double(), want_rows(tokens, table, 1.0))
    st.zero_()
    t32 = torch.tensor([3, -5, 76], dtype=torch.int32, device=DEV)
    assert torch.equal(pkg.embedding.lookup(t32, table, status=st).double(), want_rows(t32.long(), table, 1.0)) and int(st) == 0
    strided = torch.arange(20, device=DEV)[::3]
    assert torch.equal(pkg.embedding.lookup(strided, table).double(), want_rows(strided, table, 1.0))
    assert torch.equal(pkg.embedding.lookup(torch.tensor(4, device=DEV), table), table[4])
    t = table.t().contiguous().t()  # columns contiguous: taken as a copy
    assert torch.equal(pkg.embedding.lookup(tokens, t), y)


def test_lookup_of_nothing(pkg):
    table = torch.randn(5, 16, device=DEV, requires_grad=True)
    y = pkg.embedding.lookup(torch.zeros(0, dtype=torch.int64, device=DEV), table)
    assert y.shape == (0, 16)
    d, = torch.autograd.grad(y.sum(), table)
    assert torch.equal(d, torch.zeros_like(table))
    y = pkg.embedding.lookup(torch.full((40,), -1, device=DEV), table)
    d, = torch.autograd.grad(y, table, torch.full_like(y, float("nan")))
    assert torch.equal(y, torch.zeros_like(y)) and torch.equal(d, torch.zeros_like(table))


@pytest.mark.parametrize("width", [1, 31, 32, 33, 256, 257, 4096, 4099])
def test_lookup_of_a_4_bit_table(pkg, width):
    g = gen(width)
    table = torch.randn(300, width, device=DEV, generator=g) * torch.exp2(torch.randint(-20, 20, (300, 1), device=DEV, generator=g))
    q = pkg.mx.quantize(table)
    tokens = torch.randint(-1, 301, (123,), device=DEV, generator=g)
    for scale in (1.0, 12.0):
        st = torch.zeros(1, dtype=torch.int32, device=DEV)
        y = pkg.embedding.lookup(tokens, q, scale=scale, status=st)
        want = want_rows(tokens, _mx.four(table), scale)
        assert y.dtype == torch.bfloat16 and int(st) == (32 if bool((tokens == 300).any()) else 0)
        assert torch.equal(y.double(), want.bfloat16().double())  # 12 times two bits is exact before the rounding


@pytest.mark.parametrize("width", [8, 120, 128, 136, 248, 256, 264, 512, 520, 768, 1001, 1016, 1024, 1032, 2056])
def test_rows_of_every_length(pkg, width):
    """Rows that a warp takes at once or in pieces of each size, of every kind of table, and into outputs of 4-bit tables that are not
    aligned."""
    g = gen(width)
    tokens = torch.randint(-1, 90, (301,), device=DEV, generator=g)
    table = torch.randn(90, width, device=DEV, generator=g)
    for t in (table, table.bfloat16()):
        assert torch.equal(pkg.embedding.lookup(tokens, t, scale=2.0).double(), want_rows(tokens, t, 2.0))
    assert torch.equal(pkg.embedding.lookup(tokens, pkg.mx.quantize(table)).double(), want_rows(tokens, _mx.four(table), 1.0))


def cases():
    yield 1, 1, 8, "equal"
    yield 33, 5, 24, "equal"          # one id in two pieces
    yield 31, 40, 1030, "uniform"
    yield 1000, 10, 64, "uniform"     # every id past the short lists
    yield 4096, 6562, 96, "zipf"
    yield 5000, 100, 768, "zipf"
    yield 3000, 3, 40, "equal"
    yield 140_000, 50, 8, "uniform"   # positions past one bitmap
    yield 300_000, 2, 4, "equal"
    yield 2000, 20_000, 33, "zipf"


def draw_tokens(kind, n, vocab, g):
    if kind == "equal":
        t = torch.full((n,), vocab - 1, device=DEV)
        t[::7] = -1
        return t
    if kind == "uniform":
        return torch.randint(-1, vocab, (n,), device=DEV, generator=g)
    u = torch.rand(n, device=DEV, generator=g, dtype=torch.float64)
    return torch.exp(u * torch.log(torch.tensor(vocab + 1.0, device=DEV, dtype=torch.float64))).long() - 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,vocab,width,kind", list(cases()))
def test_gradient(pkg, n, vocab, width, kind, dtype):
    g = gen(n + vocab)
    tokens = draw_tokens(kind, n, vocab, g)
    table = torch.randn(vocab, width, device=DEV, generator=g).to(dtype).requires_grad_(True)
    dy = torch.randn(n, width, device=DEV, generator=g).to(dtype)
    for scale in (1.0, 12.0):
        y = pkg.embedding.lookup(tokens, table, scale=scale)
        d, = torch.autograd.grad(y, table, dy)
        assert d.dtype == dtype and d.shape == table.shape
        want, size = want_grad(tokens, dy, vocab, scale), want_grad(tokens, dy.abs(), vocab, scale)
        count = want_grad(tokens, torch.ones(n, 1, device=DEV), vocab, 1.0)
        assert bool(((d.double() - want).abs() <= (count + 2) * 2.0 ** -24 * size + HALF[dtype] * want.abs()).all())
        again, = torch.autograd.grad(pkg.embedding.lookup(tokens, table, scale=scale), table, dy)
        assert torch.equal(d, again)
    whole = torch.randint(-3, 4, (n, width), device=DEV, generator=g).to(dtype)  # sums below 2^24: exact, rounded once
    d, = torch.autograd.grad(pkg.embedding.lookup(tokens, table, scale=0.5), table, whole)
    assert torch.equal(d, want_grad(tokens, whole, vocab, 0.5).float().to(dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [2, 3, 7, 8, 9, 12, 13, 31, 47, 1021, 4094, 4096, 4097])
@pytest.mark.parametrize("vocab,width", [(1, 520), (5, 264), (900, 40), (3000, 7)])
def test_gradient_at_changes_of_path(pkg, n, vocab, width, dtype):
    """Whole numbers, exact in any order below 2^24 and rounded once: positions by rank or by counts, chunks that end in a row of an
    id or between two, absent ids in the last rows."""
    g = gen(n * 7 + vocab)
    tokens = torch.randint(-1, vocab, (n,), device=DEV, generator=g)
    tokens[tokens == vocab - 2] = -1
    table = torch.zeros(vocab, width, device=DEV, dtype=dtype, requires_grad=True)
    dy = torch.randint(-3, 4, (n, width), device=DEV, generator=g).to(dtype)
    d, = torch.autograd.grad(pkg.embedding.lookup(tokens, table), table, dy)
    assert torch.equal(d, want_grad(tokens, dy, vocab, 1.0).float().to(dtype))


@pytest.mark.parametrize("n,vocab,width,kind", [(65_535, 40_000, 5, "uniform"), (65_536, 40_000, 8, "uniform"), (65_537, 5_000_000, 4, "zipf"),
                                                (200_000, 3000, 16, "zipf"), (600_000, 9000, 8, "zipf"), (400_000, 3, 8, "uniform"),
                                                (131_073, 1, 8, "equal"), (300_000, 600, 1, "uniform")])
def test_gradient_of_many_positions(pkg, n, vocab, width, kind):
    """Whole numbers, exact in any order and rounded once: ids with a few positions, hundreds, thousands and most of them, on either
    side of a bitmap's end, joined over several levels."""
    g = gen(n + width)
    tokens = draw_tokens(kind, n, vocab, g)
    dy = torch.randint(-3, 4, (n, width), device=DEV, generator=g).bfloat16()
    table = torch.zeros(vocab, width, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    d, = torch.autograd.grad(pkg.embedding.lookup(tokens, table), table, dy)
    assert torch.equal(d, want_grad(tokens, dy, vocab, 1.0).float().bfloat16())
    loud = torch.randn(n, width, device=DEV, generator=g).bfloat16()  # the same bits each time
    first, = torch.autograd.grad(pkg.embedding.lookup(tokens, table), table, loud)
    again, = torch.autograd.grad(pkg.embedding.lookup(tokens, table), table, loud)
    assert torch.equal(first, again)


def test_gradient_ignores_what_padding_and_lost_ids_receive(pkg):
    tokens = torch.tensor([2, -1, 9, 2, 500, -7], device=DEV)
    table = torch.zeros(10, 16, device=DEV, requires_grad=True)
    dy = torch.ones(6, 16, device=DEV)
    dy[1] = dy[5] = float("nan")
    dy[4] = float("inf")
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    y = pkg.embedding.lookup(tokens, table, status=st)
    d, = torch.autograd.grad(y, table, dy)
    want = torch.zeros(10, 16, device=DEV)
    want[2], want[9] = 2.0, 1.0
    assert torch.equal(d, want) and int(st) == 32


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient_of_strided_and_broadcast_rows(pkg, dtype):
    g = gen(5)
    tokens = torch.randint(0, 30, (4, 25), device=DEV, generator=g)
    table = torch.randn(30, 136, device=DEV, generator=g).to(dtype).requires_grad_(True)
    wide = torch.randint(-3, 4, (4, 25, 141), device=DEV, generator=g).to(dtype)
    for dy in (wide[..., 3:139], wide[..., :1].expand(4, 25, 136), wide[:, :1, :136].expand(4, 25, 136)):
        d, = torch.autograd.grad(pkg.embedding.lookup(tokens, table), table, dy)
        assert torch.equal(d, want_grad(tokens.reshape(-1), dy.reshape(-1, 136), 30, 1.0).to(dtype))


def test_gradient_against_differences(pkg):
    """The formula's gradient is the slope of the lookup: a weighted sum of outputs along a direction, in fp32."""
    g = gen(7)
    tokens = torch.randint(-1, 12, (50,), device=DEV, generator=g)
    table = torch.randint(-8, 9, (12, 20), device=DEV, generator=g).float().requires_grad_(True)
    weight = torch.randint(-4, 5, (50, 20), device=DEV, generator=g).float()
    step = torch.randint(-2, 3, (12, 20), device=DEV, generator=g).float()
    f = lambda t: (pkg.embedding.lookup(tokens, t, scale=2.0) * weight).double().sum()  # noqa: E731  linear and exact in whole numbers
    d, = torch.autograd.grad(f(table), table)
    assert float((d.double() * step.double()).sum()) == float(f(table.detach() + step) - f(table.detach()))


def test_capture_and_streams(pkg):
    """Replayed with new tokens and gradients, forward and backward; two captures do not share a workspace."""
    g = gen(11)
    table = torch.randn(200, 64, device=DEV, generator=g).requires_grad_(True)
    tokens = [torch.zeros(300, dtype=torch.int64, device=DEV) for _ in range(2)]
    dys = [torch.zeros(300, 64, device=DEV) for _ in range(2)]
    graphs, outs = [], []
    for t, dy in zip(tokens, dys):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(pkg.embedding.lookup(t, table), table, dy)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = pkg.embedding.lookup(t, table, scale=3.0)
            d, = torch.autograd.grad(y, table, dy)
        graphs.append(graph)
        outs.append((y, d))
    for round_ in range(3):
        for t, dy in zip(tokens, dys):
            t.copy_(torch.randint(-1, 200, (300,), device=DEV, generator=g))
            dy.copy_(torch.randint(-3, 4, (300, 64), device=DEV, generator=g))
        streams = [torch.cuda.Stream() for _ in graphs]
        for s, graph in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for t, dy, (y, d) in zip(tokens, dys, outs):
            assert torch.equal(y, want_rows(t, table.detach(), 3.0).float())
            assert torch.equal(d, want_grad(t, dy, 200, 3.0).float())
