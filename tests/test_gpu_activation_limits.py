"""The projections' activations at infinite pre-activations: act(-inf) is the limit, 0, and so is its slope; act(inf) is inf and
NaN stays NaN, whichever way a product is cut (few rows, whole tiles, tiles split along k and joined).

All of it is exact: a column whose bias is infinite has that pre-activation whatever its (finite) sums are.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
INF = float("inf")
SIZES = [(1, 64, 200), (3, 64, 200), (40, 64, 200), (300, 64, 200), (300, 64, 1537), (40, 4096, 200), (16, 16384, 256)]


def problem(pkg, form, n, k, m, activation):
    g = torch.Generator(device=DEV).manual_seed(n + k + m)
    x, w, b, r, dy = ((torch.randn(*s, device=DEV, generator=g) * f).bfloat16()
                      for s, f in (((n, k), 1.0), ((m, k), k ** -0.5), ((m,), 0.5), ((n, m), 1.0), ((n, m), 1.0)))
    if form == "mx":
        q = pkg.mx.quantize(w)
        return lambda x, b, r=None: pkg.mx.linear(x, q, b, activation=activation, residual=r), x, b, r, dy
    kept = "e4m3" if form == "kept" else None
    return (lambda x, b, r=None: pkg.projection.linear(x, w, b, activation=activation, residual=r, checkpoint=kept)), x, b, r, dy


@pytest.mark.parametrize("activation", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("form", ["mx", "plain", "kept"])
@pytest.mark.parametrize("n,k,m", SIZES)
def test_limits(pkg, n, k, m, form, activation):
    call, x, b, r, _ = problem(pkg, form, n, k, m, activation)
    far = b.clone()
    far[0] = far[7] = far[m - 1] = -INF
    far[100], far[101] = INF, float("nan")
    keep = torch.ones(m, dtype=torch.bool, device=DEV)
    keep[[0, 7, 100, 101, m - 1]] = False
    for res in (None, r):
        y, clean = call(x, far, res), call(x, b, res)
        assert torch.equal(y[:, keep], clean[:, keep])
        for c in (0, 7, m - 1):
            assert torch.equal(y[:, c], torch.zeros_like(y[:, c]) if res is None else r[:, c])
        assert bool((y[:, 100] == INF).all()) and bool(torch.isnan(y[:, 101]).all())


@pytest.mark.parametrize("activation", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("form", ["mx", "plain"])
@pytest.mark.parametrize("n,k,m", SIZES)
def test_gradients_there(pkg, n, k, m, form, activation):
    """A column at -inf takes no part in the gradients: they are those of a column whose output has none."""
    call, x, b, _, dy = problem(pkg, form, n, k, m, activation)
    far, without = b.clone(), dy.clone()
    far[7] = -INF
    without[:, 7] = 0
    for bias, g in ((far, dy), (b, without)):
        leaves = [v.detach().requires_grad_(True) for v in (x, bias)]
        got = torch.autograd.grad(call(*leaves), leaves, g)
        assert all(bool(torch.isfinite(v).all()) for v in got)
        if bias is far:
            want = got
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
