"""``projection.linear(checkpoint="e4m3")`` on the B200: the output as without, the gradients from x and z in microscaled 8 bits.

The reference rounds x and the exact z to 8 bits itself (``_mx.eight``).  Operands are small multiples of a quarter, so that z is
exact in fp32 and rounds to the same 8 bits on both sides; dx, dw and db then differ as the projection's do: dz is rounded to
bf16 as the products' operand (2^-8), the slope's fp32 arithmetic is off by a few 2^-20, the outputs by half a step.
"""

import pytest
import torch

from tests import _mx
from tests.test_gpu_projection import SIZES, act64, operands, slope64

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("activation", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("n,k,m", SIZES)
def test_gradient(pkg, n, k, m, activation):
    x, w, b, r, dy = operands(n, k, m, n + k + m)
    leaves = [v.detach().requires_grad_(True) for v in (x, w, b, r)]
    y = pkg.projection.linear(leaves[0], leaves[1], leaves[2], activation=activation, residual=leaves[3], checkpoint="e4m3")
    z = x.double() @ w.double().t() + b.double()
    want = act64(z, activation) + r.double()
    if activation in (None, "relu"):
        assert torch.equal(y, want.float().bfloat16())
    else:
        assert bool(((y.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * (1 + z.abs())).all())
    with torch.no_grad():
        assert torch.equal(y, pkg.projection.linear(x, w, b, activation=activation, residual=r, checkpoint="e4m3"))
    dx, dw, db, dr = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(dr, dy)
    xh, zh = _mx.eight(x), _mx.eight(z)
    dz = dy.double() * (slope64(zh, activation) if activation else 1.0)
    exact = activation in (None, "relu")
    tz = 0 if exact else dy.double().abs() * 2.0 ** -18
    td = tz if exact else tz + 2.0 ** -8 * (dz.abs() + tz)
    for got, ref, tol in ((dx, dz @ w.double(), 0 if exact else td @ w.double().abs()),
                          (dw, dz.t() @ xh, 0 if exact else td.t() @ xh.abs()),
                          (db, dz.sum(0), 0 if exact else tz.sum(0) + 2.0 ** -20 * dz.abs().sum(0))):
        if exact:
            assert torch.equal(got, ref.float().bfloat16())
        else:
            assert bool(((got.double() - ref).abs() <= tol * (1 + 2.0 ** -8) + 2.0 ** -8 * ref.abs() + 2.0 ** -60).all())


@pytest.mark.parametrize("n,k,m", [(4099, 768, 1537), (2000, 8192, 200), (300, 4096, 64), (64, 768, 6562), (1, 8, 8)])
def test_what_is_kept_runs_beside_the_products(pkg, n, k, m):
    """x is quantised beside the product and brought back beside the rows' gradient: from an x that the kernel in front has just
    written, before the kernel behind writes it anew, every time the same, also with no other kernel in the call."""
    ops = torch.ops.minicpmo_sampler
    x, w, b, _, dy = operands(n, k, m, n + k)
    none = torch.empty(0, (m + 31) // 32 * 32, device=DEV, dtype=torch.uint8), torch.empty((m + 31) // 32, 0, device=DEV, dtype=torch.uint8)
    work = x.clone()

    def run(again):
        if again:
            work.fill_(float("nan"))
            work.copy_(x)
        kept = ops.linear_kept(work, w, b, None, 3, True, True, None)
        if again:
            work.fill_(0.5)
        plain = ops.linear_kept_grad(dy, w, *kept[1:3], *none, 0, False, True, False, None)[1]
        return (*kept, plain, *ops.linear_kept_grad(dy, w, *kept[1:], 3, True, True, True, None),
                ops.linear_kept_grad(dy, w, *kept[1:], 3, False, True, False, None)[1])
    want = run(False)
    torch.cuda.synchronize()
    assert torch.equal(_mx.eight(x), (want[1][:, :k].view(torch.float8_e4m3fn).double()
                                      * torch.exp2(want[2].double() - 127).t().repeat_interleave(32, 1)[:, :k]))
    for _ in range(10):
        assert all(torch.equal(p, q) for p, q in zip(run(True), want))


@pytest.mark.parametrize("activation", [None, "silu"])
def test_each_gradient_alone_and_twice(pkg, activation):
    x, w, b, r, dy = operands(70, 96, 130, 3)
    every = [v.detach().requires_grad_(True) for v in (x, w, b, r)]
    call = lambda v, **o: pkg.projection.linear(v[0], v[1], v[2], activation=activation, residual=v[3], checkpoint="e4m3", **o)  # noqa: E731
    want = torch.autograd.grad(call(every), every, dy)
    for again in torch.autograd.grad(call(every), every, dy), torch.autograd.grad(call(every, status=torch.zeros(1, dtype=torch.int32, device=DEV)), every, dy):
        assert all(torch.equal(p, q) for p, q in zip(want, again))
    for i in range(4):
        only = [v.detach().requires_grad_(i == j) for j, v in enumerate((x, w, b, r))]
        got, = torch.autograd.grad(call(only), only[i], dy)
        assert torch.equal(got, want[i])
    lone = [v.detach().requires_grad_(True) for v in (x, w)]
    got = torch.autograd.grad(pkg.projection.linear(*lone, activation=None, checkpoint="e4m3"), lone, dy)
    assert torch.equal(got[0], (dy.double() @ w.double()).float().bfloat16())


def test_memory_kept(pkg):
    """Between the passes 33/32 bytes an element of x and z stay, where without the checkpoint x and z stay at 2 each."""
    n, k, m = 2048, 1024, 1024
    g = torch.Generator(device=DEV).manual_seed(1)
    w = (torch.randn(m, k, device=DEV, generator=g) / 32).bfloat16().requires_grad_(True)

    def kept(**o):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        x = torch.randn(n, k, device=DEV, generator=g).bfloat16()
        y = pkg.projection.linear(x, w, activation="gelu", **o)
        del x
        after = torch.cuda.memory_allocated() - y.numel() * 2
        torch.autograd.grad(y, w, torch.ones_like(y))
        return after - before

    assert kept() == 2 * n * k + 2 * n * m
    assert kept(checkpoint="e4m3") == (n * k + n * m) * 33 // 32


def test_strides_and_shapes(pkg):
    n, k, m = 60, 72, 50
    x, w, b, r, dy = operands(n, k, m, 5)

    def off(v, shift, wide):
        buf = torch.full((v.shape[0] * (v.shape[1] + wide) + shift,), 77.0, device=DEV, dtype=torch.bfloat16)
        return buf[shift:].view(v.shape[0], v.shape[1] + wide)[:, :v.shape[1]].copy_(v)

    def grads(x, w, r, dy):
        v = [t.detach().requires_grad_(True) for t in (x, w, r)]
        y = pkg.projection.linear(v[0], v[1], b, activation="relu", residual=v[2], checkpoint="e4m3")
        return (y, *torch.autograd.grad(y, v, dy))

    want = grads(x, w, r, dy)
    for shift, wide in ((1, 0), (0, 3), (8, 8)):
        got = grads(off(x, shift, wide), off(w, shift, wide), off(r, shift, wide), off(dy, shift, wide))
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    y3, dx3, dw3, dr3 = grads(x.view(6, 10, k), w, r.view(6, 10, m), dy.view(6, 10, m))
    assert torch.equal(y3.view(n, m), want[0]) and torch.equal(dx3.view(n, k), want[1]) and torch.equal(dw3, want[2])
    none = grads(x[:0], w, r[:0], dy[:0])
    assert none[0].shape == (0, m) and torch.equal(none[2], torch.zeros_like(w))


def test_not_finite_blocks(pkg):
    """A row's NaN stays in its row of dx, and reaches the weight's gradient through x's block."""
    x, w, b, r, dy = operands(40, 64, 64, 7)
    x[3, 5] = float("nan")
    v = [t.detach().requires_grad_(True) for t in (x, w)]
    y = pkg.projection.linear(*v, activation="silu", checkpoint="e4m3")
    dx, dw = torch.autograd.grad(y, v, dy)
    assert bool(torch.isnan(y[3]).all()) and not bool(torch.isnan(y[4:]).any())
    assert bool(torch.isnan(dx[3]).all()) and not bool(torch.isnan(dx[4:]).any())
    assert bool(torch.isnan(dw).all())


def test_capture_replays_with_new_rows(pkg):
    x, w, b, r, dy = operands(200, 128, 96, 8)
    v = [t.clone().requires_grad_(True) for t in (x, w)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(pkg.projection.linear(*v, b, activation="gelu", checkpoint="e4m3"), v, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = pkg.projection.linear(*v, b, activation="gelu", checkpoint="e4m3")
        d = torch.autograd.grad(y, v, dy)
    for seed in (1, 2):
        with torch.no_grad():
            v[0].copy_(operands(200, 128, 96, seed)[0])
        graph.replay()
        u = [t.detach().clone().requires_grad_(True) for t in v]
        y2 = pkg.projection.linear(*u, b, activation="gelu", checkpoint="e4m3")
        assert torch.equal(y, y2) and all(torch.equal(p, q) for p, q in zip(d, torch.autograd.grad(y2, u, dy)))


def test_a_training_step(pkg):
    """Token -> embedding -> checkpointed projection -> the same table as a head -> log probabilities, and all gradients against
    the composition in 64 bits with the 8-bit roundings, at tolerances of the roundings between the parts: rows, hidden and
    gradients of either are bf16 (2^-8 each; sums of them in norm)."""
    g = torch.Generator(device=DEV).manual_seed(13)
    v, h, n = 500, 128, 300
    table = (torch.randn(v, h, device=DEV, generator=g) / 4).bfloat16().requires_grad_(True)
    w = (torch.randn(h, h, device=DEV, generator=g) / 11).bfloat16().requires_grad_(True)
    tokens = torch.randint(-1, v, (n,), device=DEV, generator=g)
    target = torch.randint(-1, v, (n,), device=DEV, generator=g)
    x = pkg.embedding.lookup(tokens, table, scale=2.0)
    y = pkg.projection.linear(x, w, activation="silu", residual=x, checkpoint="e4m3")
    loss = -pkg.logprobs.LMHeadLogprobs(table)(y, target).logprob.sum()
    d_table, d_w = torch.autograd.grad(loss, (table, w))

    t64, w64 = table.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    real = (tokens >= 0)[:, None]
    x64 = torch.where(real, t64[tokens.clamp_min(0)] * 2.0, 0.0)

    class Kept(torch.autograd.Function):
        @staticmethod
        def forward(ctx, a, m):
            z = a @ m.t()
            ctx.save_for_backward(_mx.eight(a), _mx.eight(z), m)
            return act64(z, "silu")

        @staticmethod
        def backward(ctx, gy):
            ah, zh, m = ctx.saved_tensors
            dz = gy * slope64(zh, "silu")
            return dz @ m, dz.t() @ ah

    y64 = Kept.apply(x64, w64) + x64
    lp = torch.log_softmax(y64 @ t64.t(), -1).gather(1, target.clamp_min(0)[:, None])[:, 0]
    loss64 = -torch.where(target >= 0, lp, 0.0).sum()
    e_table, e_w = torch.autograd.grad(loss64, (t64, w64))
    assert abs(float(loss.detach()) - float(loss64.detach())) <= 2.0 ** -8 * float(loss64.detach())
    for got, want in ((d_table, e_table), (d_w, e_w)):
        # y, dlogits, d hidden, dz, dx and the gradients: six roundings of at most 2^-8 each, a z on the other side of an 8-bit
        # border (2^-4 in one of a few hundred) left inside the last one's slack
        assert float((got.double() - want).norm()) <= 6 * 2.0 ** -8 * float(want.norm())
