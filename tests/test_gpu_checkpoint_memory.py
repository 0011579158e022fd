"""The kept projection's backward pass with a frozen weight: no bf16 copy of x, which only the weight's gradient reads."""

import ctypes

import pytest
import torch

DEV = torch.device("cuda:0")


def test_workspace_without_the_weights_gradient(pkg):
    """The C entry takes the plain gradient's workspace then (no GPU needed: refusals come before any launch)."""
    lib, nat = pkg._native.capi(), pkg._native
    plain, kept = ctypes.c_int64(), ctypes.c_int64()
    assert lib.b2s_linear_grad_workspace(64, 128, 96, ctypes.byref(plain)) == 0
    assert lib.b2s_linear_checkpoint_grad_workspace(64, 128, 96, ctypes.byref(kept)) == 0 and kept.value > plain.value
    at = [0x100000 * (i + 1) for i in range(8)]

    def refused(size, **o):
        # without any gradient asked for, a call that passes the checks launches nothing
        a = nat.LinearGradArgs()
        for f, v in dict(grad_out=at[0], grad_out_row_stride=96, weight=at[1], weight_row_stride=128, rows=64, in_features=128,
                         out_features=96, activation=0, workspace=at[2], workspace_bytes=size, **o).items():
            setattr(a, f, v)
        k = nat.LinearKept(at[4], at[5], at[6], at[7])
        return lib.b2s_linear_checkpoint_grad(ctypes.byref(a), ctypes.byref(k), None) == 1

    assert refused(kept.value - 1, grad_weight=at[3]) and refused(plain.value, grad_weight=at[3])
    assert refused(plain.value - 1) and not refused(plain.value)


@pytest.mark.gpu
@pytest.mark.parametrize("activation", [None, "gelu"])
def test_peak_of_a_backward_with_a_frozen_weight(pkg, activation):
    n, k, m = 4096, 2048, 1024
    g = torch.Generator(device=DEV).manual_seed(3)
    x, w, b, dy = ((torch.randn(*s, device=DEV, generator=g) * f).bfloat16()
                   for s, f in (((n, k), 1.0), ((m, k), k ** -0.5), ((m,), 0.5), ((n, m), 1.0)))

    def peak(weight_too, **o):
        leaves = [v.detach().requires_grad_(True) for v in ((x, b, w) if weight_too else (x, b))]
        y = pkg.projection.linear(leaves[0], leaves[2] if weight_too else w, leaves[1], activation=activation, **o)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        got = torch.autograd.grad(y, leaves, dy)
        torch.cuda.synchronize()
        return torch.cuda.max_memory_allocated() - before, got

    bare, _ = peak(False)
    kept, frozen = peak(False, checkpoint="e4m3")
    every, whole = peak(True, checkpoint="e4m3")
    assert kept == bare and every >= kept + 2 * n * k  # x's way back to bf16
    assert torch.equal(frozen[0], whole[0]) and torch.equal(frozen[1], whole[1])
