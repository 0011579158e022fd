"""The projection ``projection.linear`` on the B200 against a plain implementation in 64 bits.

Operands are small multiples of 1/4 whose products and sums are exact in fp32, so that without a transcendental
activation the output is the exact value rounded once and has to be equal bit for bit; with one, the activation's fp32
error (a few 2^-24) can only move a value across a rounding border: half a step of bf16 (2^-8) and a little.  With an
activation the gradient's slope is taken from a pre-activation rounded to 16 bits (at most half a step of bf16 of z times
the curvature, below 0.5 for silu and 0.8 for gelu) and dz is rounded to bf16 as the products' operand.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
CURVATURE = {None: 0.0, "relu": 0.0, "silu": 0.5, "gelu": 0.8}


def act64(z, kind):
    if kind == "relu":
        return z.clamp_min(0)
    if kind == "gelu":
        return z * torch.special.ndtr(z)
    if kind == "silu":
        return z * torch.sigmoid(z)
    return z


def slope64(z, kind):
    if kind == "relu":
        return (z > 0).double()
    if kind == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) * (2 * torch.pi) ** -0.5
    if kind == "silu":
        s = torch.sigmoid(z)
        return s + z * s * (1 - s)
    return torch.ones_like(z)


def quarter(g, *shape, most=4):
    return torch.randint(-most, most + 1, shape, device=DEV, generator=g).to(torch.bfloat16) * 0.25


def operands(n, k, m, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x, w, b, r, dy = quarter(g, n, k), quarter(g, m, k), quarter(g, m, most=16), quarter(g, n, m, most=40), quarter(g, n, m)
    # few non-zero weights per output, so that pre-activations spread over the activations' bends
    w = torch.where(torch.rand(m, k, device=DEV, generator=g) < 24.0 / k, w, torch.zeros_like(w))
    return x, w, b, r, dy


SIZES = [(1, 8, 1), (1, 4096, 768), (2, 768, 768), (3, 72, 5), (16, 4096, 768), (17, 640, 333), (64, 768, 6562),
         (100, 200, 129), (128, 64, 256), (129, 1000, 257), (513, 768, 1537), (1000, 256, 4096), (2050, 80, 64),
         (31, 8192, 40), (1300, 2048, 4096)]


@pytest.mark.parametrize("activation", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("n,k,m", SIZES)
def test_forward(pkg, n, k, m, activation):
    x, w, b, r, _ = operands(n, k, m, n + k + m)
    for bias, res in ((b, r), (None, None), (b, None), (None, r)):
        st = torch.zeros(1, dtype=torch.int32, device=DEV)
        y = pkg.projection.linear(x, w, bias, activation=activation, residual=res, status=st)
        z = x.double() @ w.double().t() + (0 if bias is None else bias.double())
        want = act64(z, activation) + (0 if res is None else res.double())
        assert y.dtype == torch.bfloat16 and y.shape == (n, m) and int(st) == 0
        if activation in (None, "relu"):
            assert torch.equal(y, want.float().bfloat16())  # the sums are exact in fp32
        else:
            tol = 2.0 ** -8 * want.abs() + 2.0 ** -20 * (1 + z.abs())
            assert bool(((y.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("activation", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("n,k,m", SIZES)
def test_gradient(pkg, n, k, m, activation):
    x, w, b, r, dy = operands(n, k, m, n + k + m)
    leaves = [v.detach().requires_grad_(True) for v in (x, w, b, r)]
    y = pkg.projection.linear(leaves[0], leaves[1], leaves[2], activation=activation, residual=leaves[3])
    assert torch.equal(y, pkg.projection.linear(x, w, b, activation=activation, residual=r))
    dx, dw, db, dr = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(dr, dy)
    z = x.double() @ w.double().t() + b.double()
    dz = dy.double() * slope64(z, activation)
    exact = activation in (None, "relu")
    # pre-activation's rounding, the slope's own fp32 arithmetic
    tz = 0 if exact else dy.double().abs() * (2.0 ** -8 * CURVATURE[activation] * z.abs() + 2.0 ** -18)
    td = tz if exact else tz + 2.0 ** -8 * (dz.abs() + tz)
    for got, want, tol in ((dx, dz @ w.double(), 0 if exact else td @ w.double().abs()),
                           (dw, dz.t() @ x.double(), 0 if exact else td.t() @ x.double().abs()),
                           (db, dz.sum(0), 0 if exact else tz.sum(0) + 2.0 ** -20 * dz.abs().sum(0))):
        if exact:
            assert torch.equal(got, want.float().bfloat16())
        else:
            assert bool(((got.double() - want).abs() <= tol * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs() + 2.0 ** -60).all())


@pytest.mark.parametrize("activation", [None, "silu"])
@pytest.mark.parametrize("shift,wide", [(1, 0), (2, 0), (3, 1), (0, 1), (1, 8), (5, 3)])
def test_gradient_of_unaligned_rows(pkg, activation, shift, wide):
    """The output's gradient (and the residual) off their 16-byte alignment: every element as from aligned rows."""
    n, k, m = 301, 136, 520
    x, w, b, r, dy = operands(n, k, m, 4)

    def off(v):
        buf = torch.full((n * (m + wide) + shift,), 77.0, device=DEV, dtype=torch.bfloat16)
        view = buf[shift:].view(n, m + wide)[:, :m]
        return view.copy_(v)

    leaves = [v.detach().requires_grad_(True) for v in (x, w, b)]
    y = pkg.projection.linear(*leaves, activation=activation, residual=r)
    want = torch.autograd.grad(y, leaves, dy)
    z = pkg.projection.linear(*leaves, activation=activation, residual=off(r))
    assert torch.equal(y, z)
    for got, exact in zip(torch.autograd.grad(z, leaves, off(dy)), want):
        assert torch.equal(got, exact)


@pytest.mark.parametrize("activation", [None, "relu", "gelu", "silu"])
def test_each_gradient_alone_and_twice(pkg, activation):
    """Any subset of the inputs, the same bits each time."""
    x, w, b, r, dy = operands(300, 128, 200, 1)
    full = None
    for mask in (15, 15, 1, 2, 4, 8, 6, 5):
        leaves = [v.detach().requires_grad_(bool(mask >> i & 1)) for i, v in enumerate((x, w, b, r))]
        y = pkg.projection.linear(leaves[0], leaves[1], leaves[2], activation=activation, residual=leaves[3])
        got = torch.autograd.grad(y, [v for v in leaves if v.requires_grad], dy)
        if full is None:
            full = got
        for g, i in zip(got, [i for i in range(4) if mask >> i & 1]):
            assert torch.equal(g, full[i])


def test_gradient_against_differences(pkg):
    x, w, b, r, dy = operands(5, 64, 40, 3)
    for activation in ("gelu", "silu"):
        leaves = [v.detach().requires_grad_(True) for v in (x, w, b)]
        y = pkg.projection.linear(*leaves, activation=activation)
        grads = torch.autograd.grad(y, leaves, dy)

        def f(a, c, e):
            return float((act64(a @ c.t() + e, activation) * dy.double()).sum())

        base = [v.double() for v in (x, w, b)]
        for i, g in enumerate(grads):
            d = torch.randn(base[i].shape, device=DEV, dtype=torch.float64)
            s = 1e-5
            hi = f(*[v + s * d if j == i else v for j, v in enumerate(base)])
            lo = f(*[v - s * d if j == i else v for j, v in enumerate(base)])
            got = float((g.double() * d).sum())
            assert abs((hi - lo) / (2 * s) - got) <= 4 * 2.0 ** -7 * float((g.double() * d).abs().sum())


def test_shapes_and_strides(pkg):
    lin = pkg.projection.linear
    x, w, b, r, dy = operands(24, 64, 50, 2)
    want = lin(x, w, b, activation="relu", residual=r)
    assert torch.equal(lin(x.view(2, 3, 4, 64), w, b, activation="relu", residual=r.view(2, 3, 4, 50)).view(24, 50), want)
    assert torch.equal(lin(x[5], w, b, activation="relu", residual=r[5]), want[5])
    wide = torch.zeros(24, 100, dtype=torch.bfloat16, device=DEV)
    wide[:, 1:65] = x
    rw = torch.zeros(24, 61, dtype=torch.bfloat16, device=DEV)
    rw[:, 3:53] = r
    bb = torch.zeros(60, dtype=torch.bfloat16, device=DEV)
    bb[7:57] = b
    wt = w.t().contiguous().t()
    xl, wl = wide[:, 1:65].detach().requires_grad_(True), wt.detach().requires_grad_(True)
    y = lin(xl, wl, bb[7:57], activation="relu", residual=rw[:, 3:53])
    assert torch.equal(y, want)
    x2, w2 = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    for g, e in zip(torch.autograd.grad(y, (xl, wl), dy),
                    torch.autograd.grad(lin(x2, w2, b, activation="relu", residual=r), (x2, w2), dy)):
        assert torch.equal(g, e)
    # broadcast operands and an expanded gradient
    xe = x[:1].detach().requires_grad_(True)
    re = r[:, :1].detach().requires_grad_(True)
    y = lin(xe.expand(24, 64), w, residual=re.expand(24, 50))
    y.sum().backward()
    ones = torch.ones(24, 50, device=DEV, dtype=torch.float64)
    row = ones[:1] @ w.double()
    assert bool(((xe.grad.double() - 24 * row).abs() <= 2.0 ** -7 * 24 * row.abs()).all())
    assert bool((re.grad == 50).all())
    e = lin(x[:0], w, b)
    assert e.shape == (0, 50)
    wl = w.detach().requires_grad_(True)
    bl = b.detach().requires_grad_(True)
    for g in torch.autograd.grad(lin(x[:0], wl, bl, activation="silu").sum(), (wl, bl)):
        assert not bool(g.any())


def test_nan_and_infinity_stay_in_their_rows(pkg):
    x, w, b, r, _ = operands(140, 64, 70, 4)
    want = pkg.projection.linear(x, w, b, activation="relu", residual=r)
    x2 = x.clone()
    x2[9, 3] = float("nan")
    w2 = w.clone()
    w2[:, 3] = 0.25
    got = pkg.projection.linear(x2, w2, b, activation="relu")
    assert bool(torch.isnan(got[9]).all())
    keep = torch.arange(140, device=DEV) != 9
    assert bool(torch.isfinite(got[keep]).all())
    x3 = x.clone()
    x3[130, :] = float("inf")
    got = pkg.projection.linear(x3, w, b, activation="relu", residual=r)
    keep = torch.arange(140, device=DEV) != 130
    assert torch.equal(got[keep], want[keep])
    zl = torch.tensor([[-3.0e38, -1.0e5, -6.0e4, 0.0, 1.0e-9, 6.0e4, 1.0e5, 3.0e38]], device=DEV).bfloat16().requires_grad_(True)
    for act, low in (("gelu", 0.5), ("silu", 0.5), ("relu", 1.0)):  # slopes far out, and next to zero
        d, = torch.autograd.grad(pkg.projection.linear(zl, torch.eye(8, device=DEV, dtype=torch.bfloat16), activation=act),
                                 (zl,), torch.ones(1, 8, device=DEV, dtype=torch.bfloat16))
        assert d[0].tolist() == [0.0, 0.0, 0.0, 0.0 if act == "relu" else 0.5, low, 1.0, 1.0, 1.0], act
    for act in ("gelu", "silu"):  # the tails: act(-large) = 0, act(large) = large
        z = torch.tensor([[-200.0, 200.0, -30000.0, 30000.0, 0.0, -3.0e38, 3.0e38, 1.0]], device=DEV).bfloat16()
        y = pkg.projection.linear(z, torch.eye(8, device=DEV, dtype=torch.bfloat16), activation=act)
        assert torch.equal(y[0, [0, 2, 4, 5]].abs(), torch.zeros(4, device=DEV, dtype=torch.bfloat16))
        assert torch.equal(y[0, [1, 3, 6]], z[0, [1, 3, 6]])


def test_streams_and_graph(pkg):
    lin = pkg.projection.linear
    sets = [operands(150, 256, 300, 10 + i) for i in range(2)]
    want = [lin(x, w, b, activation="silu", residual=r) for x, w, b, r, _ in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                x, w, b, r, _ = sets[i]
                outs[i].append(lin(x, w, b, activation="silu", residual=r))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in outs[i])
    x, w, b, r, dy = (v.clone() for v in sets[0])
    leaves = [v.requires_grad_(True) for v in (x, w, b, r)]

    def step():
        y = lin(leaves[0], leaves[1], leaves[2], activation="silu", residual=leaves[3])
        return (y, *torch.autograd.grad(y, leaves[:3], dy))

    eager = []
    for s_ in sets:
        with torch.no_grad():
            for v, e in zip((*leaves, dy), s_):
                v.copy_(e)
        eager.append([v.detach().clone() for v in step()])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, capture_error_mode="thread_local"):
        out = step()
    for i in (1, 0):
        with torch.no_grad():
            for v, e in zip((*leaves, dy), sets[i]):
                v.copy_(e)
        g.replay()
        assert all(torch.equal(a, e) for a, e in zip(out, eager[i]))
    del g


def test_projection_into_a_head(pkg):
    """The operators together: rows projected with a residual, scored by a codec head, one loss, every gradient."""
    g = torch.Generator(device=DEV).manual_seed(1)
    n, k, m, V = 260, 512, 768, 6562
    x = torch.randn(n, k, device=DEV, generator=g).bfloat16()
    w = (torch.randn(m, k, device=DEV, generator=g) / k ** 0.5).bfloat16()
    b = (0.1 * torch.randn(m, device=DEV, generator=g)).bfloat16()
    r = torch.randn(n, m, device=DEV, generator=g).bfloat16()
    head = (torch.randn(V, m, device=DEV, generator=g) * (2 / m ** 0.5)).bfloat16()
    tok = torch.randint(0, V, (n,), device=DEV, generator=g)
    tok[::7] = -1
    adv = torch.randn(n, device=DEV, generator=g)
    leaves = [v.detach().requires_grad_(True) for v in (x, w, b, r, head)]
    h = pkg.projection.linear(leaves[0], leaves[1], leaves[2], activation="gelu", residual=leaves[3])
    s = pkg.logprobs.LMHeadLogprobs(leaves[4])(h, tok)
    loss = -(adv * s.logprob).sum() - 0.01 * s.entropy.sum()
    grads = torch.autograd.grad(loss, leaves)
    ref = [v.double().requires_grad_(True) for v in (x, w, b, r, head)]
    z = act64(ref[0] @ ref[1].t() + ref[2], "gelu") + ref[3]
    logp = torch.log_softmax(z @ ref[4].t(), 1)
    lp = torch.where(tok >= 0, logp.gather(1, tok.clamp_min(0)[:, None])[:, 0], 0.0)
    ent = -(logp.exp() * logp).sum(1)
    want = torch.autograd.grad(-(adv.double() * lp).sum() - 0.01 * ent.sum(), ref)
    # h is rounded to bf16 between the two (2^-8): logits move by up to 2^-8 of their terms' magnitudes, about 2^-8 of 1.6
    # sqrt(m) x 2 / sqrt(m), and gradients by the like; norms are compared
    assert float((s.logprob.double() - lp).abs().max()) <= 0.1
    for a, e in zip(grads, want):
        assert float((a.double() - e).norm()) <= 0.02 * float(e.norm())
