"""The head's log probabilities at the models' real width and vocabulary, on operands whose sums are not exact in fp32.

Tolerance of the logits.  The tensor cores add 16 products a step to a sum whose fp32 tail they cut off, half an ulp or
2^-24 of the sum on average.  Over the 64 steps of 1024 k the sum of a random walk with standard deviation s after all K
loses 2^-24 sum_i E|s_i| = 2^-24 (0.8 * 64 * 2 / 3) s / sqrt(Q), Q = K / 1024, a quarter more in the mean square; Q such
parts, whose signs are independent, give 2^-24 * 43 s.  (Handed over only at the end it would be 2^-24 * 171 s at K = 4096.)
The log probability has its own arithmetic beside it, 4 roundings of which the mean square counts one each: 2^-24 * 2
|logprob|.  A single row is allowed six times the mean square.
"""

import pytest
import torch

from tests.test_gpu_logprobs import DEV, EPS, close, exact_operands, plain, plain_grad, s_eps

pytestmark = pytest.mark.gpu


def operands(n, V, H, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    h = torch.randn(n, H, device=DEV, generator=g).bfloat16()
    w = torch.empty(V, H, device=DEV, dtype=torch.bfloat16).normal_(0.0, 2.0 / H ** 0.5, generator=g)
    return h, w, torch.randint(0, V, (n,), device=DEV, generator=g)


def logits64(h, w):
    return torch.cat([h.double() @ w[a:a + 20_000].double().t() for a in range(0, w.shape[0], 20_000)], 1)


# one CTA's tiles, a pair's, and a step's with its last column tiles split along k
@pytest.mark.parametrize("n,V,H", [(512, 20_001, 4096), (1000, 6562, 768), (700, 3001, 2056), (64, 151_936, 4096),
                                   (200, 151_936, 4096)])
def test_forward(pkg, n, V, H):
    h, w, t = operands(n, V, H, n)
    for T in (1.0, 0.7):
        r = pkg.logprobs.LMHeadLogprobs(w)(h, t, temperature=T)
        x = logits64(h, w) / T
        lse = torch.logsumexp(x, 1)
        lp = x.gather(1, t[:, None])[:, 0] - lse
        ent = lse - (torch.softmax(x, 1) * x).sum(1)
        s = float(x.std())
        err = EPS * (43 * s + 2 * float(lp.square().mean().sqrt()))
        off = r.logprob.double() - lp
        assert float(off.square().mean().sqrt()) <= err, (float(off.square().mean().sqrt()), err)
        assert float(off.abs().max()) <= 6 * err
        close(r.entropy, ent, 2 * s_eps(V) * (2 + ent.abs()) + 6 * err)


@pytest.mark.parametrize("n,V,H", [(64, 151_936, 4096), (300, 20_001, 4096)])
def test_gradient(pkg, n, V, H):
    """dz is rounded once to bf16 (half a step, 2^-8) as the products' operand, p is off by the logits' error."""
    h, w, t = operands(n, V, H, n)
    g = torch.Generator(device=DEV).manual_seed(2)
    gl, gh = torch.randn(n, device=DEV, generator=g), 0.1 * torch.randn(n, device=DEV, generator=g)
    hl, wl = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    r = pkg.logprobs.LMHeadLogprobs(wl)(hl, t)
    dh, dw = torch.autograd.grad((r.logprob, r.entropy), (hl, wl), (gl, gh))
    x = logits64(h, w)
    err = 6 * EPS * (43 * float(x.std()) + 28)
    dz, size = plain_grad(x, t, gl, gh, 1.0)
    tol = 2.0 ** -8 * dz.abs() + (4 * (s_eps(V) + 64 * EPS) + 2 * err) * size
    del x, size
    more = 1 + 2.0 ** -8

    def product(a, b):  # a [p, V] times b [V, q] by parts of V
        return sum(a[:, v:v + 20_000] @ b[v:v + 20_000].double() for v in range(0, V, 20_000))

    want = product(dz, w)
    close(dh, want, more * (product(tol, w.abs()) * (1 + 2.0 ** -10) + 2.0 ** -8 * want.abs()) + 2.0 ** -100)
    for v in range(0, V, 20_000):
        want = dz[:, v:v + 20_000].t() @ h.double()
        bound = tol[:, v:v + 20_000].t() @ h.double().abs()
        close(dw[v:v + 20_000], want, more * (bound * (1 + 2.0 ** -10) + 2.0 ** -8 * want.abs()) + 2.0 ** -100)


@pytest.mark.parametrize("n,V,H", [(1, 148 * 256 + 300, 2304), (64, 148 * 256 + 1, 2056), (65, 148 * 256 + 5, 2048),
                                   (128, 148 * 512 + 257, 3600), (33, 148 * 256 + 1500, 4096)])
def test_left_over_column_tiles(pkg, n, V, H):
    """Whole waves of column tiles and a few over, split along k: exact sums, tokens in the split tiles and outside."""
    h, w, t, T = exact_operands(n, V, H, n + H)
    t[::2] = V - 1 - torch.arange(t[::2].numel(), device=DEV) % (V - 148 * 256 * (V // (148 * 256)))
    r = pkg.logprobs.LMHeadLogprobs(w)(h, t, temperature=T)
    lp, ent = plain(h.double() @ w.double().t(), t, T)[:2]
    close(r.logprob, lp, s_eps(V) + 4 * EPS * lp.abs())
    close(r.entropy, ent, 2 * s_eps(V) * (2 + ent.abs()))
