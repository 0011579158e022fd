"""Log probabilities of given tokens (``logprobs.token_logprobs``, ``logprobs.LMHeadLogprobs``) on the B200 against a
plain implementation in 64 bits.

Tolerances (eps = 2^-24, half a step of fp32).  The kernels' sum S of 2^y has at most V / 512 + 8 terms per thread and
about 20 pairwise merges, each one rounding; a term carries ex2.approx's 2^-22 = 4 eps and y's own roundings, 2 eps |y|
ln 2 weighted by p.  So log S is off by at most eps (V / 512 + 64) for rows whose p-weighted |y| is below 20, and the
log probability by 4 eps |logprob| more (y, c = log2(e) / T and the conversion to base e).  The entropy adds U / S, whose
relative error is twice that.  A gradient is p's relative error times its terms, then half a step of its own type.
Ranks and alternatives are whole numbers and equal.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
EPS = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def plain(x, tokens, temperature=1.0, top=0):
    """logprob, entropy, rank, top ids and their logprobs from the definition, in 64 bits."""
    x = x.double()
    V = x.shape[1]
    z = x / temperature
    bad = torch.isnan(x).any(1) | torch.isposinf(x).any(1)
    empty = torch.isneginf(x).all(1)
    # taken off first: beside a row of 1e38 the logarithm of its length is below half a step of 64 bits too
    z = z - torch.where(bad | empty, 0.0, z.amax(1))[:, None]
    lse = torch.logsumexp(z, 1)
    logp = z - torch.where(empty, 0.0, lse)[:, None]
    logp[bad] = float("nan")
    p = torch.exp(logp)
    H = torch.special.entr(p).sum(1)
    H[bad] = float("nan")
    has = (tokens >= 0) & (tokens < V)
    at = torch.where(has, tokens, 0)
    lp = torch.where(has, logp.gather(1, at[:, None])[:, 0], 0.0)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    place = torch.empty_like(order).scatter_(1, order, torch.arange(V, device=x.device).expand_as(order).contiguous())
    rank = torch.where(has, place.gather(1, at[:, None])[:, 0], -1)
    ids = order[:, :top]
    return lp, H, rank, ids, logp.gather(1, ids), p, logp


def plain_grad(x, tokens, g_lp, g_h, temperature):
    lp, H, _, _, _, p, logp = plain(x, tokens, temperature)
    V = x.shape[1]
    has = (tokens >= 0) & (tokens < V) & ~torch.isneginf(x).all(1)
    gl = torch.where(has, g_lp.double(), 0.0)
    hot = torch.zeros_like(p).scatter_(1, torch.where(has, tokens, 0)[:, None], has.double()[:, None])
    plogp = torch.where(p > 0, p * logp, 0.0)
    d = gl[:, None] * (hot - p) - g_h.double()[:, None] * (plogp + p * H[:, None])
    # the magnitudes that relative errors multiply; log p and H inside p (log p + H) are off by s and 2 s (2 + H)
    # (s = s_eps(V)) whatever their own size, which is 2 s times p (1 / 2 + 2 + H): a row of one id has log p = H = 0
    # and still y's rounding
    size = gl.abs()[:, None] * (hot + p) + g_h.double().abs()[:, None] * (plogp.abs() + p * (2.5 + 2 * H.abs()[:, None]))
    return d / temperature, size / temperature


def close(got, want, tol):
    got, want = got.double(), want.double()
    same = (torch.isnan(got) & torch.isnan(want)) | (got == want)
    ok = same | ((got - want).abs() <= tol)
    assert bool(ok.all()), (got[~ok][:8], want[~ok][:8], int((~ok).sum()))


def s_eps(V):
    return EPS * (V / 512 + 64)


def check(r, x, tokens, temperature=1.0, top=0):
    V = x.shape[1]
    lp, H, rank, ids, vals, _, _ = plain(x, tokens, temperature, top)
    assert r.logprob.dtype == r.entropy.dtype == torch.float32 and r.rank.dtype == torch.int64
    close(r.logprob, lp, s_eps(V) + 4 * EPS * lp.abs())
    close(r.entropy, H, 2 * s_eps(V) * (2 + H.abs()))
    assert torch.equal(r.rank, rank)
    if top:
        assert torch.equal(r.top_ids, ids)
        close(r.top_logprobs, vals, s_eps(V) + 4 * EPS * vals.abs())
    else:
        assert r.top_ids is None and r.top_logprobs is None


def rows_of(n, V, dtype, seed, pad=0, shift=0, scale=2.0):
    """[n, V] rows inside a wider buffer, `shift` elements off its alignment."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    buf = (torch.randn(n * (V + pad) + shift, device=DEV, generator=g) * scale).to(dtype)
    x = buf[shift:].view(n, V + pad)[:, :V]
    return x, torch.randint(0, V, (n,), device=DEV, generator=g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 31, 33, 511, 4096, 4097, 6561, 6562, 33_001])
@pytest.mark.parametrize("n", [1, 5, 130])
def test_sizes(pkg, n, V, dtype):
    for top, T, pad, shift in ((0, 1.0, 0, 0), (min(V, 20), 0.7, 3, 1), (min(V, 32), 1.3, 8, 3), (1, 1.0, 0, 1)):
        x, t = rows_of(n, V, dtype, V + n, pad, shift)
        check(pkg.logprobs.token_logprobs(x, t, top=top, temperature=T), x, t, T, top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 2, 9, 40, 64, 150, 400])
def test_thinker_rows(pkg, n, dtype):
    """Every split of a row over CTAs; one case of every length passes over each."""
    for top in (0, 20):
        x, t = rows_of(n, 151_936, dtype, n)
        check(pkg.logprobs.token_logprobs(x, t, top=top), x, t, 1.0, top)


def test_row_offsets_beyond_32_bits(pkg):
    """A batch whose last row starts past 2^31 elements (rows of a wide buffer, so that only a few are read)."""
    V, stride, n = 1000, 1_100_000_003, 3
    buf = torch.empty(2 * stride + V, dtype=torch.bfloat16, device=DEV)
    x = torch.as_strided(buf, (n, V), (stride, 1))
    x.copy_(torch.randn(n, V, device=DEV))
    t = torch.tensor([0, 999, 500], device=DEV)
    check(pkg.logprobs.token_logprobs(x, t, top=7), x, t, 1.0, 7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [9, 700, 6561, 151_936])
def test_masks_ties_and_special_values(pkg, V, dtype):
    top = min(V, 32)
    x, t = rows_of(20, V, dtype, 3)
    low = torch.finfo(dtype).min
    big = torch.finfo(dtype).max
    ninf, inf, nan = float("-inf"), float("inf"), float("nan")
    x[0] = ninf                              # nothing left
    x[1] = ninf
    x[1, V // 2] = 3.0                       # one id left
    x[2] = low                               # masked throughout with the type's lowest value: uniform
    x[3, : V - 4] = low                      # all but a few
    x[4] = 0.25                              # all equal
    x[5, V // 3] = nan
    x[6, V // 3] = inf
    x[7, ::2] = ninf
    x[8] = big                               # exponents' references that overflow
    x[9, :3] = big
    x[10] = torch.where(torch.arange(V, device=DEV) % 2 == 0, 0.0, -0.0).to(dtype)  # the zeros tie
    x[11] = torch.arange(V, device=DEV).to(dtype)                    # ascending
    x[12] = -torch.arange(V, device=DEV).to(dtype)                   # descending
    x[13] = (x[13] * 2).round()                                      # few distinct values
    x[14] = 10_000 + x[14]                                           # far from zero
    x[15, 5:] = ninf
    x[16] = torch.where(torch.arange(V, device=DEV) % 512 == 3, 50.0, -50.0).to(dtype)  # the largest in one thread
    x[17, V // 2:] = nan
    t[2::3] = x[2::3].float().argmax(1)
    t[10] = V - 1
    t[15] = V - 1                            # a masked token
    t[1] = V // 2
    r = pkg.logprobs.token_logprobs(x, t, top=top)
    lp, H, rank, ids, vals, _, _ = plain(x, t, 1.0, top)
    assert torch.equal(r.rank, rank)
    assert torch.equal(r.top_ids, ids)
    close(r.logprob, lp, s_eps(V) + 4 * EPS * lp.abs())
    close(r.entropy, H, 2 * s_eps(V) * (2 + H.abs()))
    close(r.top_logprobs, vals, s_eps(V) + 4 * EPS * vals.abs())
    # the NaN tokens' ranks: among the NaN entries
    t[5], t[17] = V // 3, V - 1
    r = pkg.logprobs.token_logprobs(x, t)
    assert torch.equal(r.rank, plain(x, t)[2])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,V", [(300, 6000), (300, 14_001), (310, 40_003), (160, 160_001), (3, 160_001)])
def test_rows_that_defeat_the_bound(pkg, n, V, dtype):
    """Many rows (one CTA each, of either size), where the first chunk's bound is no help: ascending values, ties beyond
    the list, a masked beginning, NaN by the hundred."""
    g = torch.Generator(device=DEV).manual_seed(V)
    x = (torch.randn(n, V, device=DEV, generator=g) * 2).to(dtype)
    i = torch.arange(V, device=DEV)
    ninf, nan = float("-inf"), float("nan")
    kinds = [i.to(dtype), -i.to(dtype), torch.full((V,), 0.5, device=DEV, dtype=dtype), (i % 7).to(dtype),
             torch.where(i < V - 100, ninf, 1.0).to(dtype), torch.where(i < V // 2, ninf, (i % 1000).float()).to(dtype),
             torch.where(i % 9 == 0, nan, 1.0).to(dtype), torch.where(i == V - 1, 3.0, ninf).to(dtype),
             torch.where(i % (V // 600 + 1) == 0, 9.0, -9.0).to(dtype), torch.full((V,), ninf, device=DEV, dtype=dtype)]
    for r in range(n):
        if r % 2 == 0 or n < 10:
            x[r] = kinds[(r // 2 if n >= 10 else r) % len(kinds)]
    t = torch.randint(0, V, (n,), device=DEV, generator=g)
    for top in (32, 1, 5):
        r = pkg.logprobs.token_logprobs(x, t, top=top)
        lp, H, rank, ids, vals, _, _ = plain(x, t, 1.0, top)
        assert torch.equal(r.rank, rank)
        assert torch.equal(r.top_ids, ids)
        close(r.logprob, lp, s_eps(V) + 4 * EPS * lp.abs())
        close(r.entropy, H, 2 * s_eps(V) * (2 + H.abs()))
        close(r.top_logprobs, vals, s_eps(V) + 4 * EPS * vals.abs())
    if n < 10:  # every kind in turn where rows are split over CTAs
        for k in range(len(kinds)):
            y = kinds[k][None].expand(2, V).contiguous()
            r = pkg.logprobs.token_logprobs(y, t[:2], top=32)
            assert torch.equal(r.top_ids, plain(y, t[:2], 1.0, 32)[3])


def warp_close(r, x, t, T):
    """A warp per row: 32 lanes with two sums each add a 64th of the row into each, then as `check`."""
    V = x.shape[1]
    s = EPS * (V / 64 + 64)
    lp, H, rank, _, _, _, _ = plain(x, t, T)
    assert torch.equal(r.rank, rank)
    close(r.logprob, lp, s + 4 * EPS * lp.abs())
    close(r.entropy, H, 2 * s * (2 + H.abs()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,V", [(300, 1), (301, 2), (303, 7), (307, 8), (299, 9), (300, 17), (300, 255), (300, 256),
                                 (300, 700), (2000, 33), (1801, 1023), (1777, 2049), (1776, 6562), (1783, 16_001)])
def test_many_short_rows(pkg, n, V, dtype):
    """Rows that take a warp each, with a last CTA that has rows left over; tokens in the ragged ends too."""
    for T, pad, shift in ((1.0, 0, 0), (0.7, 3, 1), (1.3, 8, 3), (1.0, 1, 0)):
        x, t = rows_of(n, V, dtype, V + n, pad, shift)
        t[::5] = torch.arange(t[::5].numel(), device=DEV) % min(V, 9)
        t[1::5] = V - 1 - torch.arange(t[1::5].numel(), device=DEV) % min(V, 9)
        t[2::50] = -1
        warp_close(pkg.logprobs.token_logprobs(x, t, temperature=T), x, t, T)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,V,shift", [(320, 9, 0), (320, 700, 1), (1800, 700, 0), (1800, 6561, 0), (1800, 16_000, 3)])
def test_many_short_rows_special_values(pkg, n, V, shift, dtype):
    x, t = rows_of(n, V, dtype, V, 0, shift)
    low, big = torch.finfo(dtype).min, torch.finfo(dtype).max
    ninf, inf, nan = float("-inf"), float("inf"), float("nan")
    i = torch.arange(V, device=DEV)

    def only(where, value, rest=ninf):
        return torch.where(where, value, rest).to(dtype)

    kinds = [only(i < 0, 0.0), only(i == V // 2, 3.0), only(i < 0, 0.0, low), only(i >= V - 4, 1.0, low),
             only(i >= 0, 0.25), only(i == V // 3, nan, 1.0), only(i == V // 3, inf, 1.0), only(i % 2 == 0, 0.5),
             only(i >= 0, big), only(i < 3, big, 0.0), only(i % 2 == 0, 0.0, -0.0), i.to(dtype), -i.to(dtype),
             (i % 7).to(dtype), only(i < 5, 2.0), only(i >= V // 2, nan, 1.0), only(i % 64 == 3, 50.0, -50.0)]
    for r in range(n):
        if r % 3:
            x[r] = kinds[r % len(kinds)]
    t[::4] = x[::4].float().argmax(1)
    t[1::8] = V - 1
    t[3::8] = V // 3
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    warp_close(pkg.logprobs.token_logprobs(x, t, status=st), x, t, 1.0)
    assert int(st) == 0
    t[n - 1] = V
    r = pkg.logprobs.token_logprobs(x, t, status=st)
    assert int(st) == 32 and float(r.logprob[n - 1]) == 0.0 and int(r.rank[n - 1]) == -1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,V,pad,shift", [(300, 33, 0, 0), (310, 700, 3, 1), (1800, 6562, 0, 0), (601, 1, 0, 0),
                                           (605, 2, 1, 0), (593, 700, 0, 0), (603, 1023, 0, 0), (607, 2041, 3, 1),
                                           (3553, 4000, 8, 5), (3555, 6562, 0, 0)])
def test_many_short_rows_gradient(pkg, n, V, pad, shift, dtype):
    x, t = rows_of(n, V, dtype, V, pad, shift)
    x[0, ::2] = float("-inf")
    t[0], t[1] = 1, -1
    x[2] = float("-inf")
    g = torch.Generator(device=DEV).manual_seed(7)
    gl, gh = torch.randn(n, device=DEV, generator=g), torch.randn(n, device=DEV, generator=g)
    leaf = x.detach().requires_grad_(True)
    r = pkg.logprobs.token_logprobs(leaf, t, temperature=0.6)
    d, = torch.autograd.grad((r.logprob, r.entropy), (leaf,), (gl, gh))
    want, size = plain_grad(x, t, gl, gh, 0.6)
    logp = plain(x, t, 0.6)[6]
    rel = EPS * (V / 64 + 64) + 4 * EPS * torch.where(torch.isfinite(logp), logp.abs(), 0.0)
    close(d, want, 2 * rel * size + HALF_STEP[dtype] * want.abs() + 2.0 ** -126)


def test_no_token_rows_and_status(pkg):
    x, t = rows_of(6, 501, torch.float32, 5)
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    t[1], t[2] = -1, -(1 << 40)
    check(pkg.logprobs.token_logprobs(x, t, top=3, status=st), x, t, 1.0, 3)
    assert int(st) == 0
    t[3], t[4] = 501, 1 << 40
    r = pkg.logprobs.token_logprobs(x, t, top=3, status=st)
    check(r, x, t, 1.0, 3)
    assert int(st) == 32 and r.logprob[1:5].tolist() == [0.0] * 4 and r.rank[1:5].tolist() == [-1] * 4
    e = pkg.logprobs.token_logprobs(x[:0], t[:0], top=3)
    assert e.logprob.shape == (0,) and e.top_ids.shape == (0, 3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,V,pad,shift", [(1, 1, 0, 0), (3, 9, 0, 0), (5, 6561, 0, 0), (4, 6562, 3, 1), (70, 4096, 8, 0),
                                           (2, 151_936, 0, 0), (3, 20_001, 0, 5)])
def test_gradient(pkg, n, V, pad, shift, dtype):
    for T in (1.0, 0.6):
        x, t = rows_of(n, V, dtype, V, pad, shift)
        t = t.clone()
        if n > 2:
            x[0, ::2] = float("-inf")
            t[0] = 1
            t[1] = -1
            x[2] = float("-inf")
        g = torch.Generator(device=DEV).manual_seed(7)
        gl, gh = torch.randn(n, device=DEV, generator=g), torch.randn(n, device=DEV, generator=g)
        leaf = x.detach().requires_grad_(True)
        for use in ((True, True), (True, False), (False, True)):
            r = pkg.logprobs.token_logprobs(leaf, t, temperature=T, top=1)
            check(r, x, t, T, 1)
            outs = [o for o, u in zip((r.logprob, r.entropy), use) if u]
            d, = torch.autograd.grad(outs, (leaf,), [o for o, u in zip((gl, gh), use) if u])
            assert d.dtype == dtype and d.shape == x.shape
            want, size = plain_grad(x, t, gl * use[0], gh * use[1], T)
            logp = plain(x, t, T)[6]
            rel = s_eps(V) + 4 * EPS * torch.where(torch.isfinite(logp), logp.abs(), 0.0)
            close(d, want, 2 * rel * size + HALF_STEP[dtype] * want.abs() + 2.0 ** -126)


def test_gradient_against_differences(pkg):
    x, t = rows_of(4, 300, torch.float32, 11)
    gl, gh = torch.tensor([1.0, -0.5, 0.0, 2.0], device=DEV), torch.tensor([0.3, 0.0, -1.0, 0.1], device=DEV)
    leaf = x.detach().requires_grad_(True)
    r = pkg.logprobs.token_logprobs(leaf, t, temperature=0.8)
    ((r.logprob * gl).sum() + (r.entropy * gh).sum()).backward()

    def f(v):
        lp, H = plain(v, t, 0.8)[:2]
        return (lp * gl.double()).sum() + (H * gh.double()).sum()

    g = torch.Generator(device=DEV).manual_seed(1)
    for _ in range(4):
        d = torch.randn(x.shape, device=DEV, generator=g, dtype=torch.float64)
        h = 1e-5
        diff = (f(x.double() + h * d) - f(x.double() - h * d)) / (2 * h)
        # central differences: h^2 / 6 of a third derivative of order 10; rounding 1e-16 / h; the kernel's 2^-18 of |d| |grad|
        assert abs(float(diff - (leaf.grad.double() * d).sum())) <= 1e-8 + 2.0 ** -18 * float((leaf.grad.double() * d).abs().sum())


def test_gradient_of_broadcast_and_repeated_use(pkg):
    """An expanded gradient, a row used twice, and logits reached through a view."""
    base = torch.randn(1, 400, device=DEV, requires_grad=True)
    t = torch.tensor([3, 3, 399], device=DEV)
    r = pkg.logprobs.token_logprobs(base.expand(3, 400), t)
    r.logprob.sum().backward()
    x = base.detach().expand(3, 400)
    want, size = plain_grad(x, t, torch.ones(3, device=DEV), torch.zeros(3, device=DEV), 1.0)
    close(base.grad, want.sum(0, keepdim=True), 4 * s_eps(400) * size.sum(0, keepdim=True) + 8 * EPS)


def test_second_derivative_is_refused(pkg):
    x, t = rows_of(2, 50, torch.float32, 1)
    x = x.detach().requires_grad_(True)
    d, = torch.autograd.grad(pkg.logprobs.token_logprobs(x, t).logprob.sum(), (x,), create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()


def test_transposed_logits(pkg):
    x, t = rows_of(40, 30, torch.float32, 2)
    y = x.t().contiguous().t()
    check(pkg.logprobs.token_logprobs(y, t, top=4), x, t, 1.0, 4)
    z = x[:1].expand(40, 30)
    check(pkg.logprobs.token_logprobs(z, t, top=4), z, t, 1.0, 4)


def test_streams_and_graph(pkg):
    """Two streams at once, and forward with gradient captured and replayed on new inputs."""
    lp = pkg.logprobs
    xs, ts_ = zip(*(rows_of(33, 20_000, torch.bfloat16, 20 + i) for i in range(2)))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(lp.token_logprobs(xs[i], ts_[i], top=5))
    torch.cuda.synchronize()
    for i in range(2):
        for r in outs[i]:
            check(r, xs[i], ts_[i], 1.0, 5)
    leaf = xs[0].clone().requires_grad_(True)
    tok = ts_[0].clone()
    gl = torch.randn(33, device=DEV)

    def step():
        r = lp.token_logprobs(leaf, tok, top=5)
        return r, torch.autograd.grad((r.logprob, r.entropy), (leaf,), (gl, gl))[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, capture_error_mode="thread_local"):
        r, d = step()
    for i in (1, 0):
        with torch.no_grad():
            leaf.copy_(xs[i])
        tok.copy_(ts_[i])
        g.replay()
        check(lp.TokenLogprobs(*(v.detach() for v in r)), xs[i], ts_[i], 1.0, 5)
        want, size = plain_grad(xs[i], ts_[i], gl, gl, 1.0)
        close(d, want, 2 * (s_eps(20_000) + 120 * EPS) * size + 2.0 ** -8 * want.abs() + 2.0 ** -126)
    del g


def test_agrees_with_the_sampler(pkg):
    """The sampled token is among the alternatives of the processed rows, and its log probability there is what the
    sampler drew it with; the greedy token has rank 0."""
    ts, th, lp = pkg.talker_sampler, pkg.thinker_sampler, pkg.logprobs
    x, _ = rows_of(64, 6562, torch.bfloat16, 9)
    cfg = ts.TalkerSampling(semantics="omni", rng="counter", top_k=20, min_new_tokens=0)
    hist = torch.full((64, 16), -1, dtype=torch.int64, device=DEV)
    steps, seeds = torch.ones(64, dtype=torch.int64, device=DEV), torch.arange(64, device=DEV)
    tok = ts.sample(x, hist, steps, seeds, 6561, cfg)
    proc = ts.processed_logits(x, hist, steps, 6561, cfg)
    r = lp.token_logprobs(proc, tok, top=32)
    check(r, proc, tok, 1.0, 32)
    assert bool((r.rank < 20).all()) and bool(torch.isfinite(r.logprob).all())
    assert torch.equal(r.top_ids.gather(1, r.rank[:, None])[:, 0], tok)
    assert bool((lp.token_logprobs(x, th.argmax(x)).rank == 0).all())


# ---------------------------------------------------------------- from a head

def exact_operands(n, V, H, seed, scale=0.25):
    """Operands whose products and sums are exact in fp32 (small multiples of 1/4, fewer than 2^20 of them), so that
    the kernel's logits are the exact ones whatever the order of its sums, scaled to a spread of a few units."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    h = torch.randint(-4, 5, (n, H), device=DEV, generator=g).to(torch.bfloat16) * scale
    w = torch.randint(-4, 5, (V, H), device=DEV, generator=g).to(torch.bfloat16) * scale
    t = torch.randint(0, V, (n,), device=DEV, generator=g)
    return h, w, t, 0.3 * math.sqrt(H) * scale * scale * 40 / 6


HEAD_SIZES = [(1, 1, 8), (1, 700, 64), (3, 64, 72), (5, 65, 8), (16, 6562, 768), (17, 1000, 1000), (64, 20_001, 256),
              (127, 513, 128), (128, 512, 64), (129, 4096, 192), (300, 6561, 512), (2100, 777, 80), (40, 33_000, 768),
              # whole waves of column tiles and a few over, split along k
              (3, 148 * 256 + 700, 1024), (100, 148 * 256 * 2 + 1, 1104)]


@pytest.mark.parametrize("n,V,H", HEAD_SIZES)
def test_head_forward(pkg, n, V, H):
    h, w, t, T = exact_operands(n, V, H, n + V + H)
    if n > 3:
        t[1] = -1
        t[2] = V
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    r = pkg.logprobs.LMHeadLogprobs(w)(h, t, temperature=T, status=st)
    x = h.double() @ w.double().t()
    lp, ent = plain(x, t, T)[:2]
    close(r.logprob, lp, s_eps(V) + 4 * EPS * lp.abs())
    close(r.entropy, ent, 2 * s_eps(V) * (2 + ent.abs()))
    assert int(st) == (32 if n > 3 else 0)


@pytest.mark.parametrize("n,V,H", HEAD_SIZES)
def test_head_gradient(pkg, n, V, H):
    """dz is rounded once to bf16 (half a step, 2^-8) as the products' operand: the sums are off by at most 2^-8 of
    the sums of magnitudes plus fp32's, then half a step of their own bf16 rounding."""
    h, w, t, T = exact_operands(n, V, H, n + V + H)
    if n > 3:
        t[1] = -1
    g = torch.Generator(device=DEV).manual_seed(4)
    gl, gh = torch.randn(n, device=DEV, generator=g), 0.1 * torch.randn(n, device=DEV, generator=g)
    hl, wl = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    r = pkg.logprobs.LMHeadLogprobs(wl)(hl, t, temperature=T)
    dh, dw = torch.autograd.grad((r.logprob, r.entropy), (hl, wl), (gl, gh))
    x = h.double() @ w.double().t()
    dz, size = plain_grad(x, t, gl, gh, T)
    tol_z = 2.0 ** -8 * dz.abs() + 4 * (s_eps(V) + 64 * EPS) * size
    more = 1 + 2.0 ** -8
    for got, want, tol in ((dh, dz @ w.double(), tol_z @ w.double().abs()),
                           (dw, dz.t() @ h.double(), tol_z.t() @ h.double().abs())):
        close(got, want, more * (tol * (1 + 2.0 ** -10) + 2.0 ** -8 * want.abs()) + 2.0 ** -100)
    # one gradient alone is the same one
    r = pkg.logprobs.LMHeadLogprobs(w)(hl, t, temperature=T)
    assert torch.equal(torch.autograd.grad((r.logprob, r.entropy), (hl,), (gl, gh))[0], dh)
    r = pkg.logprobs.LMHeadLogprobs(wl)(h, t, temperature=T)
    assert torch.equal(torch.autograd.grad((r.logprob, r.entropy), (wl,), (gl, gh))[0], dw)


def test_head_gradient_against_differences(pkg):
    h, w, t, T = exact_operands(6, 300, 64, 1)
    gl, gh = torch.randn(6, device=DEV), torch.randn(6, device=DEV)
    hl, wl = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    r = pkg.logprobs.LMHeadLogprobs(wl)(hl, t, temperature=T)
    ((r.logprob * gl).sum() + (r.entropy * gh).sum()).backward()

    def f(a, b):
        lp, H = plain(a @ b.t(), t, T)[:2]
        return float((lp * gl.double()).sum() + (H * gh.double()).sum())

    for k, leaf in enumerate((hl, wl)):
        d = torch.randn(leaf.shape, device=DEV, dtype=torch.float64)
        a, b = h.double(), w.double()
        s = 1e-5
        up = f(a + s * d, b) if k == 0 else f(a, b + s * d)
        dn = f(a - s * d, b) if k == 0 else f(a, b - s * d)
        got = (leaf.grad.double() * d).sum()
        # two bf16 roundings on the way to each element, at most 2^-7 of the terms' magnitudes; they are few-fold larger
        # than the elements themselves
        assert abs((up - dn) / (2 * s) - float(got)) <= 2.0 ** -7 * float((leaf.grad.double() * d).abs().sum()) * 4


def test_head_strided_operands_and_empty_batch(pkg):
    h, w, t, T = exact_operands(20, 500, 128, 2)
    wide = torch.zeros(20, 200, dtype=torch.bfloat16, device=DEV)
    wide[:, 3:131] = h                                    # rows off 16-byte boundaries: copied within the call
    big = torch.zeros(500, 136, dtype=torch.bfloat16, device=DEV)
    big[:, :128] = w                                      # rows further apart than their length
    want = pkg.logprobs.LMHeadLogprobs(w)(h, t, temperature=T)
    got = pkg.logprobs.LMHeadLogprobs(big[:, :128])(wide[:, 3:131], t, temperature=T)
    assert torch.equal(got.logprob, want.logprob) and torch.equal(got.entropy, want.entropy)
    got = pkg.logprobs.LMHeadLogprobs(w)(h.t().contiguous().t(), t, temperature=T)
    assert torch.equal(got.logprob, want.logprob)
    wl = w.detach().requires_grad_(True)
    r = pkg.logprobs.LMHeadLogprobs(wl)(h[:0], t[:0])
    assert r.logprob.shape == (0,)
    assert not bool(torch.autograd.grad(r.logprob.sum(), (wl,))[0].any())


def test_head_special_rows(pkg):
    """A NaN hidden row makes its own outputs NaN and nobody else's; a -inf logit has probability 0."""
    h, w, t, T = exact_operands(10, 300, 64, 3)
    want = pkg.logprobs.LMHeadLogprobs(w)(h, t, temperature=T)
    h2 = h.clone()
    h2[4, 7] = float("nan")
    got = pkg.logprobs.LMHeadLogprobs(w)(h2, t, temperature=T)
    assert bool(torch.isnan(got.logprob[4])) and bool(torch.isnan(got.entropy[4]))
    keep = torch.arange(10, device=DEV) != 4
    assert torch.equal(got.logprob[keep], want.logprob[keep]) and torch.equal(got.entropy[keep], want.entropy[keep])
    h3, w3 = h.clone(), w.clone()
    h3[:, 0] = 1.0
    w3[5, 0] = float("-inf")
    t3 = torch.full_like(t, 5)
    r = pkg.logprobs.LMHeadLogprobs(w3)(h3, t3, temperature=T)
    ent = plain(h3.double() @ w3.double().t(), t3, T)[1]
    assert bool(torch.isneginf(r.logprob).all())
    close(r.entropy, ent, 2 * s_eps(300) * (2 + ent.abs()))


def test_head_streams_and_graph(pkg):
    lp = pkg.logprobs
    h, w, t, T = exact_operands(200, 9000, 256, 5)
    h2, _, t2, _ = exact_operands(200, 9000, 256, 6)
    op = lp.LMHeadLogprobs(w)
    want, want2 = op(h, t, temperature=T), op(h2, t2, temperature=T)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(op((h, h2)[i], (t, t2)[i], temperature=T))
    torch.cuda.synchronize()
    for i in range(2):
        for r in outs[i]:
            assert torch.equal(r.logprob, (want, want2)[i].logprob)
    hl, wl = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    tok, gl = t.clone(), torch.randn(200, device=DEV)
    opw = lp.LMHeadLogprobs(wl)

    def step():
        r = opw(hl, tok, temperature=T)
        return (r.logprob, *torch.autograd.grad(r.logprob, (hl, wl), gl))

    eager = [v.detach().clone() for v in step()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, capture_error_mode="thread_local"):
        out = step()
    with torch.no_grad():
        hl.copy_(h2)
    tok.copy_(t2)
    g.replay()
    assert torch.equal(out[0], want2.logprob)
    with torch.no_grad():
        hl.copy_(h)
    tok.copy_(t)
    g.replay()
    for a, b in zip(out, eager):
        assert torch.equal(a, b)
    del g


def test_capture_beside_a_live_eager_graph_is_refused(pkg):
    """A leaf whose eager graph is alive: torch's engine would tie the captured backward pass to the eager stream and
    invalidate the capture; the operators say so instead, and work once the eager graph is gone."""
    x, t = rows_of(5, 300, torch.float32, 1)
    h, w, t2, T = exact_operands(5, 300, 64, 1)
    lx, lh, lw = (v.clone().requires_grad_(True) for v in (x, h, w))
    calls = ((lambda: pkg.logprobs.token_logprobs(lx, t).logprob, (lx,)),
             (lambda: pkg.logprobs.LMHeadLogprobs(lw)(lh, t2, temperature=T).logprob, (lh, lw)),
             (lambda: pkg.projection.linear(lh, lw), (lh, lw)))
    for f, leaves in calls:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            y = f()
            want = [v.clone() for v in torch.autograd.grad(y, leaves, torch.ones_like(y))]
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
            got = torch.autograd.grad(y, leaves, one)
        g.replay()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        del g, y


def test_calls_from_a_new_thread(pkg):
    """A thread whose first CUDA work is the call itself (its allocations come from the cache), as autograd's device
    threads are: the products' tensor maps need a current context."""
    import threading

    h, w, t, T = exact_operands(16, 300, 64, 9)
    greedy = pkg.thinker_sampler.LMHeadArgmax(w, 16)
    calls = {"head": lambda: pkg.logprobs.LMHeadLogprobs(w)(h, t, temperature=T).logprob,
             "linear": lambda: pkg.projection.linear(h, w), "greedy": lambda: greedy(h),
             "logits": lambda: pkg.logprobs.token_logprobs((h @ w.t()), t, top=3).logprob}
    want = {k: f().clone() for k, f in calls.items()}
    torch.cuda.synchronize()
    for k, f in calls.items():
        got = []

        def run():
            try:
                got.append(f())
            except Exception as e:  # reported below, in the test's own thread
                got.append(e)

        th = threading.Thread(target=run)
        th.start()
        th.join()
        torch.cuda.synchronize()
        assert isinstance(got[0], torch.Tensor), (k, got[0])
        assert torch.equal(got[0], want[k]), k


def test_head_agrees_with_logits(pkg):
    """The head's form and the logits' form of the same rows, and the greedy step: the argmax has the largest logprob."""
    h, w, _, T = exact_operands(33, 6562, 768, 8)
    logits = h.float() @ w.float().t()
    t = pkg.thinker_sampler.argmax(logits)
    a = pkg.logprobs.LMHeadLogprobs(w)(h, t, temperature=T)
    b = pkg.logprobs.token_logprobs(logits, t, temperature=T)
    close(a.logprob, b.logprob, 2 * (s_eps(6562) + 4 * EPS * b.logprob.abs()))
    close(a.entropy, b.entropy, 4 * s_eps(6562) * (2 + b.entropy))
    assert bool((b.rank == 0).all())
