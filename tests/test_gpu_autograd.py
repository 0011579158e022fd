"""The differentiable operators inside what a training program puts around them: checkpointing, vmap, a traced graph,
captures, shared status words."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def data(n=6, k=64, V=40):
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(n, k, device=DEV, generator=g).bfloat16()
    w = (torch.randn(k, k, device=DEV, generator=g) / 8).bfloat16()
    head = (torch.randn(V, k, device=DEV, generator=g) / 4).bfloat16()
    return x, w, head, torch.randint(0, V, (n,), device=DEV, generator=g)


def chain(pkg, x, w, head, t):
    """A projection into a head, and the logits form beside it."""
    y = pkg.projection.linear(x, w, activation="silu", residual=x)
    a = pkg.logprobs.LMHeadLogprobs(head)(y, t)
    b = pkg.logprobs.token_logprobs(torch.nn.functional.linear(y, head).float(), t)
    return a.logprob.sum() + 0.1 * a.entropy.sum() + b.logprob.sum()


def leaves(*v):
    return [u.detach().requires_grad_(True) for u in v]


@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpoint(pkg, reentrant):
    x, w, head, t = data()
    a, b = leaves(x, w, head), leaves(x, w, head)
    chain(pkg, *a, t).backward()
    checkpoint(lambda *v: chain(pkg, *v, t), *b, use_reentrant=reentrant).backward()
    for u, v in zip(a, b):
        assert torch.equal(u.grad, v.grad)


def test_vmap(pkg):
    """Slices in turn: the same bits, and gradients through them."""
    x, w, head, t = data(12)
    xs, ts_ = x.view(3, 4, 64), t.view(3, 4)
    lin = lambda v: pkg.projection.linear(v, w, activation="gelu")
    assert torch.equal(torch.func.vmap(lin)(xs), torch.stack([lin(v) for v in xs]))
    logits = torch.randn(3, 4, 50, device=DEV)
    score = lambda v, i: pkg.logprobs.token_logprobs(v, i).logprob
    assert torch.equal(torch.func.vmap(score)(logits, ts_), torch.stack([score(v, i) for v, i in zip(logits, ts_)]))
    a, b = logits.clone().requires_grad_(True), logits.clone().requires_grad_(True)
    torch.func.vmap(score)(a, ts_).sum().backward()
    torch.stack([score(v, i) for v, i in zip(b, ts_)]).sum().backward()
    assert torch.equal(a.grad, b.grad)


def test_traced(pkg):
    """The nodes' backward ops in a traced joint graph (no generated kernels)."""
    x, w, head, t = data()
    a, b = leaves(x, w, head), leaves(x, w, head)
    ops = pkg._native.ops()

    def f(x, w, head, t):
        y, _ = ops.linear(x, w, None, x, 3, False, None)
        lp, ent, _ = ops.lmhead_logprobs(y, head, t, 1.0, False, None)
        return lp.sum() + 0.1 * ent.sum() + ops.token_logprobs(y.float(), t, 1.0, 0, False, None)[0].sum()

    want = f(*a, t)
    want.backward()
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(*b, t)
    got.backward()
    assert torch.equal(got, want)
    for u, v in zip(a, b):
        assert torch.equal(u.grad, v.grad)


def test_capture_of_views_beside_a_live_eager_graph_is_refused(pkg):
    """Leaves reached through a reshape, the operator's own or the caller's: refused with the reason, and captured once
    the eager graph is gone."""
    x, w, head, t = data()
    lx = x.view(2, 3, 64).clone().requires_grad_(True)
    calls = (lambda: pkg.projection.linear(lx, w), lambda: pkg.logprobs.LMHeadLogprobs(head)(lx.reshape(-1, 64), t).logprob,
             lambda: pkg.logprobs.token_logprobs(lx.flatten(0, 1).float(), t).logprob)
    for f in calls:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            y = f()
            want = torch.autograd.grad(y, lx, torch.ones_like(y))[0].clone()
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
            got = torch.autograd.grad(y, lx, one)[0]
        g.replay()
        assert torch.equal(got, want)
        del g, y


def test_status_word_shared_and_cleared(pkg):
    x, w, head, t = data()
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    a, b = leaves(x, w, head), leaves(x, w, head)
    t[0] = head.shape[0]  # no token, and said so
    y = pkg.projection.linear(a[0], a[1], activation="relu", status=st)
    r = pkg.logprobs.LMHeadLogprobs(a[2])(y, t, status=st)
    assert int(st) == 32
    st.zero_()
    r.logprob.sum().backward()
    assert int(st) == 0
    y = pkg.projection.linear(b[0], b[1], activation="relu")
    pkg.logprobs.LMHeadLogprobs(b[2])(y, t).logprob.sum().backward()
    for u, v in zip(a, b):
        assert torch.equal(u.grad, v.grad)
