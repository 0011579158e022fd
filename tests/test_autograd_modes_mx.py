"""The embedding, the microscaled product and the projection with kept activations under torch's ways of differentiating other
than a plain backward pass, on Meta tensors (no GPU needed: the graph nodes run, the kernels do not)."""

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
    codes, scales = empty(40, 16, dtype=torch.uint8), empty(1, 1, 1024, dtype=torch.uint8)
    return {
        "embedding": (lambda w: ops.embedding(t, w, 2.0, None), [empty(40, 16)]),
        "mx_linear": (lambda x, b, r: ops.mx_linear(x, None, codes, scales, 16, b, r, 3, False, None)[0],
                      [empty(3, 16), empty(40), empty(3, 40)]),
        "linear_kept": (lambda x, w, b, r: ops.linear_kept(x, w, b, r, 3, False, False, None)[0],
                        [empty(3, 16), empty(40, 16), empty(40), empty(3, 40)]),
    }


NAMES = ["embedding", "mx_linear", "linear_kept"]


@pytest.mark.parametrize("name,which", [("embedding", 0), ("mx_linear", 0), ("mx_linear", 1), ("mx_linear", 2),
                                        ("linear_kept", 0), ("linear_kept", 1), ("linear_kept", 2), ("linear_kept", 3)])
def test_tangents_are_refused(pkg, name, which):
    f, inputs = calls(pkg._native.ops())[name]
    with fwAD.dual_level():
        dual = list(inputs)
        dual[which] = fwAD.make_dual(inputs[which], torch.ones_like(inputs[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            f(*dual)
        with fwAD._set_fwd_grad_enabled(False):  # tangents are not asked for
            assert f(*dual).shape[0] == 3
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(f, tuple(inputs), tuple(torch.ones_like(v) for v in inputs))


@pytest.mark.parametrize("name", NAMES)
def test_traced_with_gradients(pkg, name):
    f, inputs = calls(pkg._native.ops())[name]
    leaves = [v.requires_grad_(True) for v in inputs]
    y = f(*leaves)
    grads = torch.autograd.grad(y, leaves, torch.ones_like(y))
    assert [g.shape for g in grads] == [v.shape for v in leaves] and all(g.is_meta for g in grads)
    got = torch.func.vmap(f, in_dims=(0,) + (None,) * (len(leaves) - 1))(meta(5, *leaves[0].shape, dtype=leaves[0].dtype), *inputs[1:])
    assert got.shape == (5, *y.shape)
    with pytest.raises(RuntimeError):  # the engine's nodes do not run under torch.func's transforms: refused, never dropped
        torch.func.grad(lambda x: f(x, *inputs[1:]).sum())(meta(*leaves[0].shape, dtype=leaves[0].dtype))


@pytest.mark.parametrize("name", NAMES)
def test_second_derivatives_are_refused(pkg, name):
    f, inputs = calls(pkg._native.ops())[name]
    x = inputs[0].requires_grad_(True)
    y = f(x, *inputs[1:])
    g, = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()


@pytest.mark.parametrize("name", NAMES)
def test_traced_with_fake_tensors(pkg, name):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        f, inputs = calls(pkg._native.ops(), "cuda")[name]
        y = f(*[v.requires_grad_(True) for v in inputs])
    assert y.shape[0] == 3 and y.device.type == "cuda" and y.requires_grad


def test_status_word_cleared_between_the_passes(pkg):
    ops = pkg._native.ops()
    st, t = meta(1, dtype=torch.int32), meta(3, dtype=torch.int64)
    codes, scales = meta(40, 16, dtype=torch.uint8), meta(1, 1, 1024, dtype=torch.uint8)
    table, x, w = (v.requires_grad_(True) for v in (meta(40, 16), meta(3, 16), meta(40, 16)))
    outs = [ops.embedding(t, table, 1.0, st), ops.mx_linear(x, None, codes, scales, 16, None, None, 2, False, st)[0],
            ops.linear_kept(x, w, None, None, 1, False, False, st)[0]]
    st.zero_()
    for y in outs:
        y.sum().backward()
    assert table.grad.shape == table.shape and x.grad.shape == x.shape and w.grad.shape == w.shape
