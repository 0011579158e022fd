"""The embedding, the microscaled product and the projection with kept activations inside what programs put around them:
recomputation, vmap, a traced graph, captures beside live graphs, streams, waits that give up, tensors past 2^31 elements."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from tests import _mx
from tests.test_wait_limit import limit

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def data(n=6, k=64, v=40):
    g = torch.Generator(device=DEV).manual_seed(3)
    table = (torch.randn(v, k, device=DEV, generator=g) / 4).bfloat16()
    w = (torch.randn(k, k, device=DEV, generator=g) / 8).bfloat16()
    return table, w, torch.randint(-1, v, (n,), device=DEV, generator=g)


def leaves(*v):
    return [u.detach().requires_grad_(True) for u in v]


def chain(pkg, table, w, t, q):
    """Token -> row -> kept projection -> frozen 4-bit head."""
    x = pkg.embedding.lookup(t, table, scale=2.0)
    y = pkg.projection.linear(x, w, activation="silu", residual=x, checkpoint="e4m3")
    return pkg.mx.linear(y, q, activation="gelu").float().square().sum()


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputation(pkg, reentrant):
    table, w, t = data()
    q = pkg.mx.quantize(table)
    a, b = leaves(table, w), leaves(table, w)
    chain(pkg, *a, t, q).backward()
    checkpoint(lambda *v: chain(pkg, *v, t, q), *b, use_reentrant=reentrant).backward()
    for u, v in zip(a, b):
        assert torch.equal(u.grad, v.grad) and bool(u.grad.any())


def test_vmap(pkg):
    table, w, t = data(12)
    q = pkg.mx.quantize(table)
    x = pkg.embedding.lookup(t, table).view(3, 4, 64)
    for f in (lambda v: pkg.mx.linear(v, q, activation="gelu"), lambda v: pkg.projection.linear(v, w, checkpoint="e4m3")):
        assert torch.equal(torch.func.vmap(f)(x), torch.stack([f(v) for v in x]))
    look = lambda i: pkg.embedding.lookup(i, table)  # noqa: E731
    assert torch.equal(torch.func.vmap(look)(t.view(3, 4)), torch.stack([look(i) for i in t.view(3, 4)]))


def test_traced(pkg):
    table, w, t = data()
    q = pkg.mx.quantize(table)
    a, b = leaves(table, w), leaves(table, w)
    ops = pkg._native.ops()

    def f(table, w, t):
        x = ops.embedding(t, table, 2.0, None)
        y = ops.linear_kept(x, w, None, x, 3, False, False, None)[0]
        return ops.mx_linear(y, None, q.codes, q.scales, 64, None, None, 2, False, None)[0].float().square().sum()

    want = f(*a, t)
    want.backward()
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(*b, t)
    got.backward()
    assert torch.equal(got, want)
    for u, v in zip(a, b):
        assert torch.equal(u.grad, v.grad)


def test_capture_beside_a_live_eager_graph_is_refused(pkg):
    """Refused with the reason while the eager graph lives, captured once it is gone."""
    table, w, t = data()
    q = pkg.mx.quantize(table)
    table.requires_grad_(True)
    x = torch.randn(6, 64, device=DEV).bfloat16().requires_grad_(True)
    for leaf, f in ((table, lambda: pkg.embedding.lookup(t, table)), (x, lambda: pkg.mx.linear(x, q, activation="silu")),
                    (x, lambda: pkg.projection.linear(x.view(2, 3, 64), w, activation="silu", checkpoint="e4m3"))):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            y = f()
            want = torch.autograd.grad(y, leaf, torch.ones_like(y))[0].clone()
        torch.cuda.current_stream().wait_stream(s)
        del y
        alive = f()
        one = torch.ones_like(alive)
        with pytest.raises(RuntimeError, match="eager graph"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), capture_error_mode="thread_local"):
                f()
        del alive
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, capture_error_mode="thread_local"):
            y = f()
            got = torch.autograd.grad(y, leaf, one)[0]
        g.replay()
        assert torch.equal(got, want)
        del g, y


def test_calls_on_two_streams(pkg):
    """No state between calls: the same operators at once on two streams, sizes that take every path."""
    g = torch.Generator(device=DEV).manual_seed(9)
    w = pkg.mx.quantize(torch.randn(1000, 768, device=DEV, generator=g).bfloat16())
    table = torch.randn(3000, 256, device=DEV, generator=g)
    jobs = []
    for n in (2, 100, 1500, 6000):
        x = torch.randn(n, 768, device=DEV, generator=g).bfloat16()
        t = torch.randint(-1, 3000, (n,), device=DEV, generator=g)
        dy = torch.randn(n, 256, device=DEV, generator=g)
        jobs.append((x, t, dy))

    def run(x, t, dy):
        leaf = table.clone().requires_grad_(True)
        d, = torch.autograd.grad(pkg.embedding.lookup(t, leaf), leaf, dy)
        return pkg.mx.linear(x, w), pkg.mx.dequantize(pkg.mx.quantize(x)), d

    want = [run(*j) for j in jobs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append([run(*j) for j in jobs])
    torch.cuda.synchronize()
    for batch in got:
        for a, b in zip(want, batch):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_a_weight_quantised_just_before_its_product(pkg):
    """The product may read its weight before the kernel in front of it is done: not before the weight is there."""
    g = torch.Generator(device=DEV).manual_seed(4)
    codes, scales = None, None
    x = torch.randn(300, 2048, device=DEV, generator=g).bfloat16()
    for i in range(20):
        v = torch.randn(4096, 2048, device=DEV, generator=g).bfloat16()
        q = pkg.mx.quantize(v)
        if codes is None:
            codes, scales = torch.empty_like(q.codes), torch.empty_like(q.scales)
        want = pkg.mx.linear(x, q)
        torch.cuda.synchronize()
        lib = pkg._native.capi()
        stream = torch.cuda.current_stream().cuda_stream
        torch.cuda._sleep(1_000_000)
        pkg._native.check(lib.b2s_mx_quantize(v.data_ptr(), 1, 4096, 2048, 2048, codes.data_ptr(), scales.data_ptr(), stream), "quantize")
        got = pkg.mx.linear(x, pkg.mx.MXTensor(codes, scales, (4096, 2048)))
        assert torch.equal(got, want)


@pytest.mark.parametrize("n,k,m", [(17, 64, 40), (200, 768, 1537), (700, 4096, 600), (16, 16_384, 256)])
def test_waits_that_give_up(pkg, n, k, m):
    """Tiles of one CTA and of a pair, whole and split along k: NaN and the status word, and the next call is sound."""
    g = torch.Generator(device=DEV).manual_seed(n)
    lib = pkg._native.capi()
    x, q = torch.randn(n, k, device=DEV, generator=g).bfloat16(), pkg.mx.quantize(torch.randn(m, k, device=DEV, generator=g))
    r = torch.randn(n, m, device=DEV, generator=g).bfloat16()
    want = pkg.mx.linear(x, q, activation="silu", residual=r)
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    leaf = x.clone().requires_grad_(True)
    with limit(lib, 0):
        y = pkg.mx.linear(leaf, q, activation="silu", residual=r, status=st)
        z = pkg.mx.linear(x, q, activation="silu", residual=r)
    d, = torch.autograd.grad(y, leaf, torch.ones_like(y))
    torch.cuda.synchronize()
    assert int(st) == 4 and bool(torch.isnan(y).all()) and bool(torch.isnan(z).all()) and bool(torch.isnan(d).all())
    assert torch.equal(pkg.mx.linear(x, q, activation="silu", residual=r, status=st), want)


@pytest.mark.parametrize("activation", [None, "gelu"])
def test_kept_waits_that_give_up(pkg, activation):
    g = torch.Generator(device=DEV).manual_seed(1)
    lib = pkg._native.capi()
    v = leaves(torch.randn(200, 64, device=DEV, generator=g).bfloat16(), torch.randn(96, 64, device=DEV, generator=g).bfloat16())
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    with limit(lib, 0):
        y = pkg.projection.linear(*v, activation=activation, status=st, checkpoint="e4m3")
    d = torch.autograd.grad(y, v, torch.ones_like(y))
    torch.cuda.synchronize()
    assert int(st) == 4 and bool(torch.isnan(y).all())
    assert not activation or all(bool(torch.isnan(u).all()) for u in d)  # the kept pre-activation is NaN too


def test_past_two_to_the_31_elements(pkg):
    """Offsets beyond 32 bits: a table's, a matrix's and a gradient's last rows."""
    vocab, width = 540_000, 4096  # 2.2 G elements
    table = torch.zeros(vocab, width, device=DEV, dtype=torch.bfloat16)
    table[-1], table[-2], table[7] = 3.0, -1.5, 0.5
    tokens = torch.tensor([vocab - 1, 7, vocab - 2, -1, vocab - 1], device=DEV)
    table.requires_grad_(True)
    y = pkg.embedding.lookup(tokens, table)
    assert [float(v) for v in y.detach()[:, -1]] == [3.0, 0.5, -1.5, 0.0, 3.0]
    d, = torch.autograd.grad(y, table, torch.ones_like(y))
    assert [float(d[v, -1]) for v in (vocab - 1, vocab - 2, 7, 8, 0)] == [2.0, 1.0, 1.0, 0.0, 0.0]
    assert float(d.sum(dtype=torch.float64)) == 4.0 * width
    del d, y
    table = table.detach()
    q = pkg.mx.quantize(table)
    assert torch.equal(pkg.embedding.lookup(tokens, q)[:, -1], torch.tensor([3.0, 0.5, -1.5, 0.0, 3.0], device=DEV).bfloat16())
    x = torch.ones(3, width, device=DEV, dtype=torch.bfloat16)
    for n in (1, 3, 40):
        z = pkg.mx.linear(x[:1].expand(n, width), q)
        assert [float(v) for v in z[-1, [vocab - 1, vocab - 2, 7, 8]]] == [3.0 * width, -1.5 * width, 0.5 * width, 0.0]
        assert float(z.sum(dtype=torch.float64)) == 2.0 * width * n
    back = pkg.mx.dequantize(q)
    assert torch.equal(back[-2:], table[-2:]) and float(back.sum(dtype=torch.float64)) == 2.0 * width
    rows = pkg.mx.linear(table[-1_000:], pkg.mx.quantize(torch.eye(width, device=DEV)[:600]))
    assert torch.equal(rows[-2:], table[-2:, :600])


def test_long_outputs(pkg):
    """A product whose output passes 2^31 elements, rows at its end."""
    w = pkg.mx.quantize(torch.ones(70_000, 32, device=DEV))
    x = torch.zeros(31_000, 32, device=DEV, dtype=torch.bfloat16)
    x[-1], x[5] = 2.0, -1.0
    y = pkg.mx.linear(x, w)
    assert bool((y[-1] == 64).all()) and bool((y[5] == -32).all()) and float(y[-2].abs().max()) == 0.0
    assert float(y.sum(dtype=torch.float64)) == 70_000 * 32.0
