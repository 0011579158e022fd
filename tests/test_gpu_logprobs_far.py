"""Log probabilities of rows far from zero: finite masks (-1e9 .. the type's lowest value, alone and beside ordinary
logits), large logits and small temperatures, on every path of the logits kernel, of its gradient and of the head.

Tolerances: as in ``test_gpu_logprobs``, where y = (x - m) c takes one rounding more than fma(x, c, -m c), and the
temperature's own rounding to fp32 is counted: 4 eps |y| in the place of 2, with a p-weighted |y| of at most log2 V, and
8 eps |logprob| in the place of 4.
"""

import pytest
import torch

from tests.test_gpu_logprobs import DEV, EPS, HALF_STEP, close, plain, plain_grad

pytestmark = pytest.mark.gpu
MASKS = (-1e9, -1e10, -1e20, -1e30, None)  # None: the type's lowest value
# a cluster of CTAs per row, one CTA of 512 threads, of 256, of 128, and a warp per row (the last two without alternatives)
SHAPES = [(3, 151_936, 8), (3, 151_936, 0), (5, 6562, 8), (7, 700, 0), (300, 14_001, 5), (300, 40_003, 0), (300, 6000, 3),
          (310, 701, 0), (1800, 6561, 0)]


def s_of(V):
    """The sums' share (see test_gpu_logprobs), of a row per warp: the largest of the paths."""
    return EPS * (V / 64 + 96)


FMAX = torch.finfo(torch.float32).max


def close_fp32(got, want, tol):
    """`close`, where what is beyond fp32 may be infinite (no row here has an infinity of its own)."""
    close(got.double().clamp(-FMAX, FMAX), want.clamp(-FMAX, FMAX), tol.clamp(max=FMAX))


def far_rows(n, V, dtype, T, seed):
    """Rows of every kind in turn, and tokens that are ordinary, masked or at the row's end."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    i = torch.arange(V, device=DEV)
    base = torch.randn(n, V, device=DEV, generator=g) * 2
    edge = 2.0 ** 20 * T / 1.4426950408889634  # logits of about 2^20 in base 2
    rows = []
    for r in range(n):
        value = MASKS[(r // 8) % len(MASKS)]
        value = torch.finfo(dtype).min if value is None else value
        kind = r % 8 if n >= 8 else (r + seed) % 8
        x = base[r]
        if kind == 0:
            x = torch.where(i < V - 3, value, x)                  # masked first, a few left
        elif kind == 1:
            x = torch.full_like(x, value)                         # nothing but the mask
        elif kind == 2:
            x = torch.where(base[(r + 1) % n].abs() < 2.0, value, x)
        elif kind == 3:
            x = -value * (1.0 + 2.0 ** -7 * (i % 5))              # far above zero
            x = torch.where(torch.isfinite(x.to(dtype)), x, -value)
        elif kind == 4:
            x = x * 1500.0
        elif kind == 5:
            x = edge + 4.0 * T * x                                # both sides of the border between the two forms of y
        elif kind == 6:
            x = torch.where(i % 2 == 0, -edge + 4.0 * T * x, value)
        else:
            x = torch.where(i % 777 == 5, -value, value)          # the two ends
        rows.append(x)
    x = torch.stack(rows).to(dtype)
    t = torch.randint(0, V, (n,), device=DEV, generator=g)
    t[1::3] = V - 1
    t[2::3] = x[2::3].float().argmax(1)
    return x, t


@pytest.mark.parametrize("T", [1e-6, 0.1, 0.7, 1.0, 2.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,V,top", SHAPES)
def test_forward(pkg, n, V, top, dtype, T):
    for seed in range(8 if n < 8 else 1):
        x, t = far_rows(n, V, dtype, T, seed)
        r = pkg.logprobs.token_logprobs(x, t, top=top, temperature=T)
        lp, H, rank, ids, vals, _, _ = plain(x, t, T, top)
        close_fp32(r.logprob, lp, s_of(V) + 8 * EPS * lp.abs())
        if top:
            close_fp32(r.top_logprobs, vals, s_of(V) + 8 * EPS * vals.abs())
        close(r.entropy, H, 2 * s_of(V) * (2 + H.abs()))
        assert torch.equal(r.rank, rank)
        if top:
            assert torch.equal(r.top_ids, ids)


@pytest.mark.parametrize("T", [1e-6, 0.1, 1.0, 2.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,V", [(3, 20_001), (310, 701), (1800, 700)])
def test_gradient(pkg, n, V, dtype, T):
    for seed in range(8 if n < 8 else 1):
        x, t = far_rows(n, V, dtype, T, seed)
        g = torch.Generator(device=DEV).manual_seed(seed)
        gl, gh = torch.randn(n, device=DEV, generator=g), torch.randn(n, device=DEV, generator=g)
        leaf = x.detach().requires_grad_(True)
        r = pkg.logprobs.token_logprobs(leaf, t, temperature=T)
        d, = torch.autograd.grad((r.logprob, r.entropy), (leaf,), (gl, gh))
        want, size = plain_grad(x, t, gl, gh, T)
        logp = plain(x, t, T)[6]
        near = torch.where(logp > -200, logp.abs(), 0.0)  # p is 0 in fp32 below that
        rel = s_of(V) + 8 * EPS * near
        close(d, want, 2 * rel * size + HALF_STEP[dtype] * want.abs() + 2.0 ** -110 / T)


@pytest.mark.parametrize("n", [4, 300])
def test_head(pkg, n):
    """Logits of a head that are all but equal and far from zero, masked by a far feature, or large."""
    V, H = 1001, 64
    g = torch.Generator(device=DEV).manual_seed(n)
    for far in (1e5, -1e9, -1e20, 1e20, 1e28):
        for kind in range(3):
            h = torch.zeros(n, H, device=DEV)
            w = torch.zeros(V, H, device=DEV)
            if kind != 1:  # beside far logits the small ones are lost in fp32: only the masked rows have them
                h[:, 1:] = torch.randint(-4, 5, (n, H - 1), device=DEV, generator=g) * 0.25
                w[:, 1:] = torch.randint(-4, 5, (V, H - 1), device=DEV, generator=g) * 0.25
            h[:, 0] = far
            if kind == 0:
                w[:, 0] = torch.where(torch.rand(V, device=DEV, generator=g) < 0.7, -1.0 if far > 0 else 1.0, 0.0)
                w[:, 1:] *= (w[:, :1] == 0)   # a masked logit is the mask alone
            elif kind == 1:
                w[:, 0] = 1.0                 # uniform
            else:
                w[:, 0] = torch.randint(-4, 5, (V,), device=DEV, generator=g) * 0.25
                w[:, 1:] = 0.0
            h, w = h.bfloat16(), w.bfloat16()
            t = torch.randint(0, V, (n,), device=DEV, generator=g)
            gl, gh = torch.randn(n, device=DEV, generator=g), torch.randn(n, device=DEV, generator=g)
            x = h.double() @ w.double().t()
            for T in (0.7, 1.0, 3.0):
                hl, wl = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
                r = pkg.logprobs.LMHeadLogprobs(wl)(hl, t, temperature=T)
                lp, ent = plain(x, t, T)[:2]
                close(r.logprob, lp, s_of(V) + 8 * EPS * lp.abs())
                close(r.entropy, ent, 2 * s_of(V) * (2 + ent.abs()))
                dh, dw = torch.autograd.grad((r.logprob, r.entropy), (hl, wl), (gl, gh))
                d, size = plain_grad(x, t, gl, gh, T)
                # dz is rounded once to bf16 (half a step), the products' sums and their rounding follow
                td = 2.0 ** -8 * d.abs() + 2.0 ** -12 * size + 2.0 ** -120
                for got, want, tol in ((dh, d @ w.double(), td @ w.double().abs()),
                                       (dw, d.t() @ h.double(), td.t() @ h.double().abs())):
                    close(got, want, tol * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs() + 2.0 ** -60)
