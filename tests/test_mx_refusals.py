"""What the embedding and the microscaled entry points refuse, before anything is launched (no GPU needed)."""

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

FAKE = [ctypes.c_void_p(0x10000 * (i + 1)) for i in range(12)]
ODD = ctypes.c_void_p(0x10001)
OFF = ctypes.c_void_p(0x10008)


def test_python_entry_points_refuse_cpu_tensors(pkg):
    t, table = torch.zeros(3, dtype=torch.int64), torch.zeros(5, 8)
    with pytest.raises(ValueError):
        pkg.embedding.lookup(t, table)
    with pytest.raises(ValueError):
        pkg.mx.quantize(table)
    with pytest.raises(ValueError):
        pkg.mx.MXTensor(torch.zeros(5, 16, dtype=torch.uint8), torch.zeros(1, 1, 1024, dtype=torch.uint8), (5, 8))
    with pytest.raises(ValueError):
        pkg.mx.linear(table.bfloat16(), table)
    with pytest.raises(ValueError):
        pkg.mx.dequantize(table)
    with pytest.raises(ValueError):
        pkg.projection.linear(table.bfloat16(), table.bfloat16(), checkpoint="e4m3")


def test_embedding_arguments(pkg):
    lib = pkg._native.capi()

    def call(tokens=FAKE[0], n=4, table=FAKE[1], dtype=1, vocab=100, width=64, stride=64, scale=1.0, out=FAKE[2]):
        return lib.b2s_embedding(tokens, n, table, dtype, vocab, width, stride, scale, out, None, None)

    assert call(n=0) == 0
    for bad in (dict(tokens=None), dict(n=-1), dict(table=None), dict(dtype=2), dict(vocab=0), dict(width=0), dict(stride=63),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(out=None), dict(table=ODD), dict(out=ODD),
                dict(dtype=0, table=ctypes.c_void_p(0x10002))):
        assert call(**bad) == 1, bad
    for big in (dict(n=0x7fffffff), dict(vocab=0x7fffffff), dict(width=0x7fffffff, stride=0x7fffffff),
                dict(n=0x7fff0000, width=0x7fff0000, stride=0x7fff0000)):
        assert call(**big) == 2, big

    def mx(tokens=FAKE[0], n=4, codes=FAKE[1], scales=FAKE[2], vocab=100, width=64, scale=1.0, out=FAKE[3]):
        return lib.b2s_embedding_mx(tokens, n, codes, scales, vocab, width, scale, out, None, None)

    assert mx(n=0) == 0 and mx(n=0x7fffffff) == 2
    for bad in (dict(tokens=None), dict(n=-1), dict(codes=None), dict(scales=None), dict(vocab=0), dict(width=0),
                dict(scale=float("nan")), dict(out=None), dict(codes=OFF), dict(scales=OFF), dict(out=ODD)):
        assert mx(**bad) == 1, bad


def test_embedding_gradient_arguments(pkg):
    lib = pkg._native.capi()
    need = ctypes.c_int64()
    assert lib.b2s_embedding_grad_workspace(4, 100, 64, ctypes.byref(need)) == 0 and need.value > 0
    for bad in ((-1, 100, 64), (4, 0, 64), (4, 100, 0)):
        assert lib.b2s_embedding_grad_workspace(*bad, ctypes.byref(need)) == 1
    lib.b2s_embedding_grad_workspace(4, 100, 64, ctypes.byref(need))

    def call(tokens=FAKE[0], n=4, grad=FAKE[1], stride=64, dtype=1, vocab=100, width=64, scale=1.0, out=FAKE[2], ws=FAKE[3],
             size=need.value):
        return lib.b2s_embedding_grad(tokens, n, grad, stride, dtype, vocab, width, scale, out, ws, size, None)

    for bad in (dict(tokens=None), dict(n=-1), dict(grad=None), dict(stride=63), dict(dtype=5), dict(vocab=0), dict(width=0),
                dict(scale=float("inf")), dict(out=None), dict(out=ODD), dict(grad=ODD), dict(ws=None), dict(ws=OFF),
                dict(size=need.value - 1), dict(n=0, out=None)):
        assert call(**bad) == 1, bad
    assert call(n=0x7fffffff) == 2 and call(vocab=0x7fffffff) == 2


def test_quantisation_arguments(pkg):
    lib = pkg._native.capi()
    for fn, order in ((lib.b2s_mx_quantize, lambda x, d, r, k, s, c, t: (x, d, r, k, s, c, t)),
                      (lib.b2s_mx_dequantize, lambda x, d, r, k, s, c, t: (c, t, r, k, d, x, s))):
        def call(x=FAKE[0], dtype=1, rows=4, k=64, stride=64, codes=FAKE[1], scales=FAKE[2]):
            return fn(*order(x, dtype, rows, k, stride, codes, scales), None)

        assert call(rows=0) == 0
        for bad in (dict(x=None), dict(dtype=2), dict(rows=-1), dict(k=0), dict(stride=63), dict(codes=None), dict(scales=None),
                    dict(codes=OFF), dict(scales=OFF), dict(x=ODD), dict(dtype=0, x=ctypes.c_void_p(0x10002))):
            assert call(**bad) == 1, bad
        assert call(rows=0x7fffffff) == 2 and call(k=0x7fffffff, stride=0x7fffffff) == 2


OK = dict(x=FAKE[0].value, x_row_stride=64, x_codes=None, x_scales=None, weight_codes=FAKE[1].value,
          weight_scales=FAKE[2].value, rows=5, in_features=64, out_features=50, activation=0, bias=None, residual=None,
          residual_row_stride=0, out=FAKE[3].value, out_row_stride=50, preact=None, preact_row_stride=0,
          workspace=FAKE[4].value, workspace_bytes=1 << 40, status=None)


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(in_features=0), dict(out_features=0), dict(activation=4), dict(activation=-1),
                                 dict(x=None), dict(x_codes=FAKE[5].value, x_scales=FAKE[6].value),
                                 dict(x=None, x_codes=FAKE[5].value), dict(x=None, x_codes=0x10008, x_scales=FAKE[6].value),
                                 dict(x=None, x_codes=FAKE[5].value, x_scales=0x10008), dict(x_row_stride=63),
                                 dict(weight_codes=None), dict(weight_scales=None), dict(weight_codes=0x10008),
                                 dict(weight_scales=0x10004), dict(out=None), dict(out=0x10001), dict(x=0x10001),
                                 dict(out_row_stride=49), dict(bias=0x10001), dict(residual=FAKE[7].value, residual_row_stride=49),
                                 dict(residual=0x10001, residual_row_stride=50), dict(preact=FAKE[8].value, preact_row_stride=50),
                                 dict(preact=0x10008, preact_row_stride=56)], ids=str)
def test_product_arguments(pkg, bad):
    lib, nat = pkg._native.capi(), pkg._native
    assert lib.b2s_mx_linear(ctypes.byref(nat.MxLinearArgs(**{**OK, **bad})), None) == 1


def test_product_sizes(pkg):
    lib, nat = pkg._native.capi(), pkg._native
    assert lib.b2s_mx_linear(None, None) == 1
    assert lib.b2s_mx_linear(ctypes.byref(nat.MxLinearArgs(**{**OK, "rows": 0})), None) == 0
    assert lib.b2s_mx_linear(ctypes.byref(nat.MxLinearArgs(**{**OK, "rows": 0x7fffffff})), None) == 2
    n = ctypes.c_int64()
    assert lib.b2s_mx_linear_workspace(5, 64, 50, ctypes.byref(n)) == 0 and n.value >= 0
    for bad in ((-1, 64, 50), (5, 0, 50), (5, 64, 0)):
        assert lib.b2s_mx_linear_workspace(*bad, ctypes.byref(n)) == 1


@pytest.mark.parametrize("bad", [dict(x_codes=None), dict(x_scales=None), dict(z_codes=None), dict(z_scales=None),
                                 dict(x_codes=0x10008), dict(z_codes=0x10008)], ids=str)
def test_checkpoint_arguments(pkg, bad):
    lib, nat = pkg._native.capi(), pkg._native
    whole = dict(x_codes=FAKE[0].value, x_scales=FAKE[1].value, z_codes=FAKE[2].value, z_scales=FAKE[3].value)
    fwd = dict(x=FAKE[4].value, x_row_stride=64, weight=FAKE[5].value, weight_row_stride=64, rows=5, in_features=64,
               out_features=50, activation=3, out=FAKE[6].value, out_row_stride=50, workspace=FAKE[7].value, workspace_bytes=1 << 40)
    grad = dict(grad_out=FAKE[4].value, grad_out_row_stride=50, weight=FAKE[5].value, weight_row_stride=64, rows=5,
                in_features=64, out_features=50, activation=3, grad_x=FAKE[6].value, grad_weight=FAKE[8].value,
                workspace=FAKE[7].value, workspace_bytes=1 << 40)
    kept = ctypes.byref(nat.LinearKept(**{**whole, **bad}))
    assert lib.b2s_linear_checkpoint(ctypes.byref(nat.LinearArgs(**fwd)), kept, None) == 1
    assert lib.b2s_linear_checkpoint_grad(ctypes.byref(nat.LinearGradArgs(**grad)), kept, None) == 1
    good = ctypes.byref(nat.LinearKept(**whole))
    for f, g in ((dict(x=None), dict(weight=None)), (dict(rows=-1), dict(rows=-1)), (dict(workspace=None), dict(workspace=None)),
                 (dict(preact=FAKE[9].value, preact_row_stride=56), dict(workspace_bytes=64)),
                 (dict(activation=4), dict(activation=4)), (dict(in_features=60), dict(in_features=60))):
        if "workspace" not in f:
            assert lib.b2s_linear_checkpoint(ctypes.byref(nat.LinearArgs(**{**fwd, **f})), good, None) == 1, f
        assert lib.b2s_linear_checkpoint_grad(ctypes.byref(nat.LinearGradArgs(**{**grad, **g})), good, None) == 1, g
    assert lib.b2s_linear_checkpoint(ctypes.byref(nat.LinearArgs(**fwd)), None, None) == 1
    assert lib.b2s_linear_checkpoint_grad(ctypes.byref(nat.LinearGradArgs(**grad)), None, None) == 1
    assert lib.b2s_linear_checkpoint(ctypes.byref(nat.LinearArgs(**{**fwd, "rows": 0})), good, None) == 0
    n = ctypes.c_int64()
    assert lib.b2s_linear_checkpoint_grad_workspace(5, 64, 50, ctypes.byref(n)) == 0 and n.value >= 5 * 64 * 2
    assert lib.b2s_linear_checkpoint_workspace(-1, 64, 50, ctypes.byref(n)) == 1


@pytest.mark.parametrize("name,mirror", [("b2s_mx_linear_args", "MxLinearArgs"), ("b2s_linear_kept", "LinearKept")])
def test_argument_layout_matches_c(pkg, tmp_path, name, mirror):
    header = Path(__file__).resolve().parents[1] / "include" / "b2s_sampler.h"
    cls = getattr(pkg._native, mirror)
    src = tmp_path / "layout.c"
    src.write_text("\n".join(["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void) {",
                              'printf("%zu\\n", sizeof(' + name + '));',
                              *[f'printf("%zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_], "return 0; }"]))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-x", "c", str(src), "-o", str(exe)], check=True)
    out = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert out == [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]


def test_meta_kernels(pkg):
    """Shapes are known without running anything, with gradients asked for too."""
    ops = pkg._native.ops()
    t, table = torch.empty(7, dtype=torch.int64, device="meta"), torch.empty(100, 33, device="meta", requires_grad=True)
    y = ops.embedding(t, table, 2.0, None)
    d, = torch.autograd.grad(y, table, torch.empty_like(y))
    assert y.shape == (7, 33) and d.shape == (100, 33)
    codes, scales = ops.mx_quantize(torch.empty(300, 300, device="meta"))
    assert codes.shape == (300, 160) and scales.shape == (3, 2, 1024)
    assert ops.mx_dequantize(codes, scales, 300, torch.bfloat16).shape == (300, 300)
    assert ops.embedding_mx(t, codes, scales, 300, 1.0, None).shape == (7, 300)
    x = torch.empty(5, 300, dtype=torch.bfloat16, device="meta", requires_grad=True)
    w = torch.empty(90, 304, dtype=torch.bfloat16, device="meta", requires_grad=True)
    h = torch.empty(5, 304, dtype=torch.bfloat16, device="meta")
    kept = ops.linear_kept(h, w, None, None, 3, False, False, None)
    assert [tuple(v.shape) for v in kept] == [(5, 90), (5, 320), (10, 5), (5, 96), (3, 5)]
    assert torch.autograd.grad(kept[0], w, torch.empty_like(kept[0]))[0].shape == (90, 304)
    y, pre = ops.mx_linear(x, None, codes, scales, 300, None, None, 3, True, None)
    d, = torch.autograd.grad(y, x, torch.empty_like(y))
    assert y.shape == (5, 300) and pre.shape == (5, 304) and d.shape == (5, 300)


def test_tangents_and_second_derivatives_are_refused(pkg):
    import torch.autograd.forward_ad as fw

    ops = pkg._native.ops()
    t, table = torch.empty(7, dtype=torch.int64, device="meta"), torch.empty(100, 32, device="meta", requires_grad=True)
    with fw.dual_level(), pytest.raises(NotImplementedError):
        ops.embedding(t, fw.make_dual(table, torch.empty_like(table)), 1.0, None)
    w = torch.empty(7, 32, device="meta", requires_grad=True)
    d, = torch.autograd.grad(ops.embedding(t, table, 1.0, None), table, w, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        d.sum().backward()
