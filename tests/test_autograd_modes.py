"""The differentiable operators under torch's ways of differentiating other than a plain backward pass, on Meta tensors
(no GPU needed: the graph nodes run, the kernels do not)."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def calls(ops):
    """Each operator as a function of its differentiable inputs, and those inputs."""
    t = meta(3, dtype=torch.int64)
    return {
        "token_logprobs": (lambda x: ops.token_logprobs(x, t, 1.0, 0, False, None)[0], [meta(3, 40, dtype=torch.float32)]),
        "lmhead_logprobs": (lambda h, w: ops.lmhead_logprobs(h, w, t, 1.0, False, None)[0], [meta(3, 16), meta(40, 16)]),
        "linear": (lambda x, w, b, r: ops.linear(x, w, b, r, 3, False, None)[0],
                   [meta(3, 16), meta(40, 16), meta(40), meta(3, 40)]),
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
