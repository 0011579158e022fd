"""Waits that give up (``b2s_wait_limit``): the outputs say so themselves, with a status word or without one.

With a limit of 0 a call starts no copy and no product and gives up before its first wait, so that nothing is in flight
when it returns; the calls are otherwise sound.
"""

import contextlib
import ctypes

import pytest
import torch

DEV = torch.device("cuda:0")


def set_limit(lib, clocks):
    before = ctypes.c_int64()
    assert lib.b2s_wait_limit(clocks, ctypes.byref(before)) == 0
    return before.value


@contextlib.contextmanager
def limit(lib, clocks):
    before = set_limit(lib, clocks)
    try:
        yield before
    finally:
        set_limit(lib, before)


def test_the_limit_itself(pkg):
    lib = pkg._native.capi()
    default = set_limit(lib, -1)
    assert default > 10 ** 8
    with limit(lib, 0) as before:
        assert before == default and set_limit(lib, -1) == 0
        with limit(lib, 1234):
            assert set_limit(lib, -1) == 1234
            assert set_limit(lib, 1 << 60) == 1234 and set_limit(lib, -1) == default  # never beyond the default
        assert set_limit(lib, -1) == 0
    assert lib.b2s_wait_limit(-1, None) == 0 and set_limit(lib, -1) == default


def word():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("top", [0, 7])
@pytest.mark.parametrize("n,V", [(1, 6562), (3, 151_936), (300, 6000), (300, 40_003)])
def test_logits(pkg, n, V, top, dtype):
    """One CTA of 512, a cluster, 128 and 256 threads a row (a warp per row waits for nothing)."""
    lp, lib = pkg.logprobs, pkg._native.capi()
    x, t = torch.randn(n, V, device=DEV).to(dtype), torch.randint(0, V, (n,), device=DEV)
    if n > 1:
        t[1] = -1
    want = lp.token_logprobs(x, t, top=top)
    leaf, st = x.clone().requires_grad_(True), word()
    with limit(lib, 0):
        r = lp.token_logprobs(leaf, t, top=top, status=st)
        s = lp.token_logprobs(x, t, top=top)
    d, = torch.autograd.grad((r.logprob, r.entropy), (leaf,), (torch.ones(n, device=DEV), torch.ones(n, device=DEV)))
    torch.cuda.synchronize()
    assert int(st) == 4
    for got in (r, s):
        assert bool(torch.isnan(got.logprob[t >= 0]).all()) and bool(torch.isnan(got.entropy).all())
        assert bool((got.rank == -1).all())
        if top:
            assert bool((got.top_ids == -1).all()) and bool(torch.isnan(got.top_logprobs).all())
    assert bool(torch.isnan(d).all())
    got = lp.token_logprobs(x, t, top=top, status=st)  # and the next call is sound again
    assert torch.equal(got.logprob, want.logprob) and torch.equal(got.rank, want.rank) and int(st) == 4


@pytest.mark.gpu
@pytest.mark.parametrize("n,V,H", [(1, 700, 64), (16, 6562, 768), (100, 148 * 256 * 2 + 1, 1104), (100, 148 * 256 + 1, 2056), (300, 6561, 2056), (777, 6562, 768)])
def test_head(pkg, n, V, H):
    """Tiles of one CTA and of a pair, column tiles split along k; a given-up forward and a given-up gradient."""
    lp, lib = pkg.logprobs, pkg._native.capi()
    h = torch.randn(n, H, device=DEV).bfloat16().requires_grad_(True)
    w = (torch.randn(V, H, device=DEV) / H ** 0.5).bfloat16().requires_grad_(True)
    t = torch.randint(0, V, (n,), device=DEV)
    op, g = lp.LMHeadLogprobs(w), torch.ones(n, device=DEV)
    want = op(h, t)
    exact = torch.autograd.grad(want.logprob, (h, w), g)
    st, st2 = word(), word()
    with limit(lib, 0):
        r = op(h, t, status=st)
    assert int(st) == 4 and bool(torch.isnan(r.logprob).all()) and bool(torch.isnan(r.entropy).all())
    for d in torch.autograd.grad(r.logprob, (h, w), g):  # of a forward that gave up
        assert bool(torch.isnan(d).all())
    r = op(h, t, status=st2)
    with limit(lib, 0):
        grads = torch.autograd.grad(r.logprob, (h, w), g)
    assert int(st2) == 4 and all(bool(torch.isnan(d).all()) for d in grads)
    r = op(h, t)
    assert torch.equal(r.logprob, want.logprob)
    for a, b in zip(torch.autograd.grad(r.logprob, (h, w), g), exact):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("activation", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("n,k,m", [(17, 640, 333), (64, 4096, 768), (100, 200, 129), (513, 768, 1537), (2050, 80, 64),
                                   (1300, 2048, 4096)])
def test_linear(pkg, n, k, m, activation):
    """Whole and split tiles of one CTA and of a pair, with the join; a given-up forward, and gradients of a sound one."""
    linear, lib = pkg.projection.linear, pkg._native.capi()
    x, w, b, r = (torch.randn(*s, device=DEV).bfloat16().requires_grad_(True) for s in ((n, k), (m, k), (m,), (n, m)))
    dy = torch.randn(n, m, device=DEV).bfloat16()
    want = linear(x, w, b, activation=activation, residual=r)
    exact = torch.autograd.grad(want, (x, w, b), dy)
    st, st2 = word(), word()
    with limit(lib, 0):
        y = linear(x, w, b, activation=activation, residual=r, status=st)
        z = linear(x, w)
    assert int(st) == 4 and bool(torch.isnan(y).all()) and bool(torch.isnan(z).all())
    y = linear(x, w, b, activation=activation, residual=r, status=st2)
    with limit(lib, 0):
        dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert int(st2) == 4 and bool(torch.isnan(dx).all()) and bool(torch.isnan(dw).all())
    y = linear(x, w, b, activation=activation, residual=r)
    assert torch.equal(y, want)
    for a, c in zip(torch.autograd.grad(y, (x, w, b), dy), exact):
        assert torch.equal(a, c)
