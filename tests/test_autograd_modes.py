"""The differentiable operators under torch's ways of differentiating other than a plain backward pass, on Meta tensors
(no GPU needed: the graph nodes run, the kernels do not)."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def calls(ops, device="meta"):
    """Each operator as a function of its differentiable inputs, and those inputs."""
    def empty(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device=device)

    t = empty(3, dtype=torch.int64)
    return {
        "token_logprobs": (lambda x: ops.token_logprobs(x, t, 1.0, 0, False, None)[0], [empty(3, 40, dtype=torch.float32)]),
        "lmhead_logprobs": (lambda h, w: ops.lmhead_logprobs(h, w, t, 1.0, False, None)[0], [empty(3, 16), empty(40, 16)]),
        "linear": (lambda x, w, b, r: ops.linear(x, w, b, r, 3, False, None)[0],
                   [empty(3, 16), empty(40, 16), empty(40), empty(3, 40)]),
    }


@pytest.mark.parametrize("name,which", [("token_logprobs", 0), ("lmhead_logprobs", 0), ("lmhead_logprobs", 1),
                                        ("linear", 0), ("linear", 1), ("linear", 2), ("linear", 3)])
def test_tangents_are_refused(pkg, name, which):
    f, inputs = calls(pkg._native.ops())[name]
    with fwAD.dual_level():
        dual = list(inputs)
        dual[which] = fwAD.make_dual(inputs[which], torch.ones_like(inputs[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            f(*dual)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            f(*dual)
        with fwAD._set_fwd_grad_enabled(False):  # tangents are not asked for
            assert f(*dual).shape[0] == 3
        assert f(*inputs).shape[0] == 3
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(f, tuple(inputs), tuple(torch.ones_like(v) for v in inputs))


@pytest.mark.parametrize("name", ["token_logprobs", "lmhead_logprobs", "linear"])
def test_traced_with_gradients(pkg, name):
    """Shapes of outputs and gradients are known without running anything, with no device and no driver either."""
    f, inputs = calls(pkg._native.ops())[name]
    leaves = [v.requires_grad_(True) for v in inputs]
    y = f(*leaves)
    grads = torch.autograd.grad(y, leaves, torch.ones_like(y))
    assert [g.shape for g in grads] == [v.shape for v in leaves] and all(g.is_meta for g in grads)
    got = torch.func.vmap(f, in_dims=(0,) + (None,) * (len(leaves) - 1))(meta(5, *leaves[0].shape, dtype=leaves[0].dtype), *inputs[1:])
    assert got.shape == (5, *y.shape)
    with pytest.raises(RuntimeError):  # the engine's nodes do not run under torch.func's transforms: refused, never dropped
        torch.func.grad(lambda x: f(x, *inputs[1:]).sum())(meta(*leaves[0].shape, dtype=leaves[0].dtype))


@pytest.mark.parametrize("name", ["token_logprobs", "lmhead_logprobs", "linear"])
def test_traced_with_fake_tensors(pkg, name):
    """CUDA tensors that are none, on a machine with or without a driver (the engine's own backward needs one)."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        f, inputs = calls(pkg._native.ops(), "cuda")[name]
        y = f(*[v.requires_grad_(True) for v in inputs])
    assert y.shape[0] == 3 and y.device.type == "cuda" and y.requires_grad


def test_status_word_cleared_between_the_passes(pkg):
    """The word is an output: reading and clearing it after a forward, or sharing it by two, leaves the backward alone."""
    ops = pkg._native.ops()
    st, t = meta(1, dtype=torch.int32), meta(3, dtype=torch.int64)
    x, h, w = (v.requires_grad_(True) for v in (meta(3, 40, dtype=torch.float32), meta(3, 16), meta(40, 16)))
    first = [ops.token_logprobs(x, t, 1.0, 0, False, st)[0], ops.lmhead_logprobs(h, w, t, 1.0, False, st)[0],
             ops.linear(h, w, None, None, 2, False, st)[0]]
    st.zero_()
    second = [ops.lmhead_logprobs(h, w, t, 1.0, False, st)[0], ops.linear(h, w, None, None, 0, False, st)[0]]
    st.zero_()
    for y in first + second:
        y.sum().backward()
    assert h.grad.shape == h.shape and w.grad.shape == w.shape and x.grad.shape == x.shape
