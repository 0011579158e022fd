"""What the log-probability and projection entry points refuse, before anything is launched (no GPU needed)."""

import ctypes

import pytest
import torch

FAKE = [ctypes.c_void_p(0x10000 * (i + 1)) for i in range(12)]


def test_python_entry_points_refuse_cpu_tensors(pkg):
    x, t = torch.zeros(2, 16), torch.zeros(2, dtype=torch.int64)
    w = torch.zeros(16, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        pkg.logprobs.token_logprobs(x, t)
    with pytest.raises(ValueError):
        pkg.logprobs.LMHeadLogprobs(w)
    with pytest.raises(ValueError):
        pkg.projection.linear(torch.zeros(2, 8, dtype=torch.bfloat16), w)


def test_token_logprobs_arguments(pkg):
    lib = pkg._native.capi()

    def call(dtype=1, rows=4, vocab=100, stride=100, T=1.0, top=0, logits=FAKE[0], ids=FAKE[4], vals=FAKE[5], stats=None):
        return lib.b2s_token_logprobs(logits, dtype, rows, vocab, stride, FAKE[1], T, top, FAKE[2], FAKE[3], FAKE[6], ids,
                                      vals, stats, None, None)

    assert call(rows=0) == 0
    for bad in (dict(dtype=2), dict(rows=-1), dict(vocab=0), dict(stride=99), dict(T=0.0), dict(T=-1.0),
                dict(T=float("nan")), dict(T=float("inf")), dict(top=-1), dict(logits=None), dict(top=3, ids=None),
                dict(top=3, vals=None), dict(stats=ctypes.c_void_p(0x10008)), dict(vocab=5, stride=5, top=6),
                dict(logits=ctypes.c_void_p(0x10001)), dict(dtype=0, logits=ctypes.c_void_p(0x10002))):
        assert call(**bad) == 1, bad
    assert call(top=33) == 2
    assert call(rows=0x7fffffff) == 2 and call(vocab=0x7fffffff, stride=0x7fffffff) == 2  # indices beyond 32 bits

    def grad(dtype=1, rows=4, vocab=100, stride=100, T=1.0, stats=FAKE[2], out=FAKE[3], ostride=100):
        return lib.b2s_token_logprobs_grad(FAKE[0], dtype, rows, vocab, stride, FAKE[1], T, stats, FAKE[4], None, out,
                                           ostride, None)

    assert grad(rows=0) == 0
    for bad in (dict(dtype=3), dict(rows=-2), dict(vocab=0), dict(stride=50), dict(ostride=99), dict(T=0.0),
                dict(stats=None), dict(out=None), dict(stats=ctypes.c_void_p(0x10004)), dict(out=ctypes.c_void_p(0x10001))):
        assert grad(**bad) == 1, bad


def _head(nat, **kw):
    d = dict(hidden=FAKE[0].value, hidden_row_stride=64, head=FAKE[1].value, head_row_stride=64, hidden_dim=64,
             vocab=1000, rows=5, temperature=1.0, tokens=FAKE[2].value, workspace=FAKE[3].value,
             workspace_bytes=1 << 40, status=None)
    d.update(kw)
    return nat.LMHeadArgs(**d)


HEAD_BAD = (dict(rows=-1), dict(vocab=0), dict(hidden_dim=60), dict(hidden_dim=4), dict(hidden_row_stride=56),
            dict(hidden_row_stride=68), dict(head_row_stride=63), dict(head_row_stride=66), dict(temperature=0.0),
            dict(hidden=None), dict(head=None), dict(hidden=0x10008), dict(head=0x10002), dict(tokens=None),
            dict(workspace=None), dict(workspace_bytes=8), dict(workspace=0x10008))


@pytest.mark.parametrize("bad", HEAD_BAD, ids=str)
def test_head_arguments(pkg, bad):
    lib, nat = pkg._native.capi(), pkg._native
    a = _head(nat, **bad)
    assert lib.b2s_lmhead_logprobs(ctypes.byref(a), FAKE[4], FAKE[5], None, None) == 1
    assert lib.b2s_lmhead_logprobs_grad(ctypes.byref(a), FAKE[6], FAKE[4], FAKE[5], FAKE[7], FAKE[8], None) == 1


def test_head_more_arguments(pkg):
    lib, nat = pkg._native.capi(), pkg._native
    a = _head(nat)
    assert lib.b2s_lmhead_logprobs(None, FAKE[4], FAKE[5], None, None) == 1
    for big in (dict(rows=0x7fffffff), dict(vocab=0x7ffffff8)):
        assert lib.b2s_lmhead_logprobs(ctypes.byref(_head(nat, **big)), FAKE[4], FAKE[5], None, None) == 2
    assert lib.b2s_linear(ctypes.byref(nat.LinearArgs(**{**LINEAR_OK, "rows": 0x7fffffff})), None) == 2
    assert lib.b2s_lmhead_logprobs(ctypes.byref(a), FAKE[4], FAKE[5], ctypes.c_void_p(0x10008), None) == 1
    assert lib.b2s_lmhead_logprobs(ctypes.byref(_head(nat, rows=0)), FAKE[4], FAKE[5], None, None) == 0
    assert lib.b2s_lmhead_logprobs_grad(ctypes.byref(a), None, FAKE[4], FAKE[5], FAKE[7], FAKE[8], None) == 1
    assert lib.b2s_lmhead_logprobs_grad(ctypes.byref(a), FAKE[6], FAKE[4], FAKE[5], ctypes.c_void_p(0x10008), None, None) == 1
    assert lib.b2s_lmhead_logprobs_grad(ctypes.byref(a), FAKE[6], FAKE[4], FAKE[5], None, ctypes.c_void_p(0x10008), None) == 1
    n = ctypes.c_int64()
    assert lib.b2s_lmhead_logprobs_workspace(5, 1000, 64, ctypes.byref(n)) == 0 and n.value > 0
    assert lib.b2s_lmhead_logprobs_workspace(-1, 1000, 64, ctypes.byref(n)) == 1
    assert lib.b2s_lmhead_logprobs_grad_workspace(5, 1001, 64, ctypes.byref(n)) == 0 and n.value >= 5 * 1008 * 2


LINEAR_OK = dict(x=FAKE[0].value, x_row_stride=64, weight=FAKE[1].value, weight_row_stride=64, rows=5, in_features=64,
                 out_features=50, activation=0, bias=None, residual=None, residual_row_stride=0, out=FAKE[2].value,
                 out_row_stride=50, preact=None, preact_row_stride=0, workspace=FAKE[3].value, workspace_bytes=1 << 40,
                 status=None)


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(in_features=60), dict(in_features=0), dict(out_features=0),
                                 dict(activation=4), dict(activation=-1), dict(x=None), dict(weight=None), dict(out=None),
                                 dict(x=0x10008), dict(weight=0x10008), dict(out=0x10001), dict(x_row_stride=60),
                                 dict(x_row_stride=68), dict(weight_row_stride=56), dict(out_row_stride=49),
                                 dict(bias=0x10002), dict(residual=FAKE[4].value, residual_row_stride=49),
                                 dict(preact=FAKE[5].value, preact_row_stride=50),
                                 dict(preact=0x10008, preact_row_stride=56)], ids=str)
def test_linear_arguments(pkg, bad):
    lib, nat = pkg._native.capi(), pkg._native
    assert lib.b2s_linear(ctypes.byref(nat.LinearArgs(**{**LINEAR_OK, **bad})), None) == 1


GRAD_OK = dict(grad_out=FAKE[0].value, grad_out_row_stride=50, x=FAKE[1].value, x_row_stride=64, weight=FAKE[2].value,
               weight_row_stride=64, preact=FAKE[3].value, preact_row_stride=56, rows=5, in_features=64, out_features=50,
               activation=3, grad_x=FAKE[4].value, grad_weight=FAKE[5].value, grad_bias=FAKE[6].value,
               workspace=FAKE[7].value, workspace_bytes=1 << 40, status=None)


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(in_features=60), dict(out_features=0), dict(activation=9),
                                 dict(grad_out=None), dict(grad_out_row_stride=49), dict(preact=None),
                                 dict(preact_row_stride=50), dict(x=None), dict(weight=None), dict(x_row_stride=12),
                                 dict(weight_row_stride=65), dict(grad_x=0x10008), dict(grad_weight=0x10008),
                                 dict(workspace=None), dict(workspace_bytes=16)], ids=str)
def test_linear_grad_arguments(pkg, bad):
    lib, nat = pkg._native.capi(), pkg._native
    assert lib.b2s_linear_grad(ctypes.byref(nat.LinearGradArgs(**{**GRAD_OK, **bad})), None) == 1


@pytest.mark.parametrize("name,mirror", [("b2s_lmhead_args", "LMHeadArgs"), ("b2s_linear_args", "LinearArgs"),
                                         ("b2s_linear_grad_args", "LinearGradArgs")])
def test_struct_layout_matches_c(pkg, tmp_path, name, mirror):
    import subprocess
    from pathlib import Path

    header = Path(__file__).resolve().parents[1] / "include" / "b2s_sampler.h"
    cls = getattr(pkg._native, mirror)
    src = tmp_path / "layout.c"
    src.write_text("\n".join(["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void) {",
                              f'printf("%zu\\n", sizeof({name}));',
                              *[f'printf("%zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_], "return 0; }"]))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-x", "c", str(src), "-o", str(exe)], check=True)
    out = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert out == [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]


def test_ops_have_meta_kernels(pkg):
    """Shapes are known without running anything (tracing, fake tensors)."""
    ops = pkg._native.ops()
    x, t = torch.empty(3, 100, device="meta"), torch.empty(3, dtype=torch.int64, device="meta")
    lp, ent, rank, ids, vals, stats = ops.token_logprobs(x, t, 1.0, 5, True, None)
    assert lp.shape == ent.shape == rank.shape == (3,) and ids.shape == vals.shape == (3, 5) and stats.shape == (3, 4)
    assert ops.token_logprobs_grad(x, t, stats, lp, None, 1.0).shape == (3, 100)
    h, w = (torch.empty(s, dtype=torch.bfloat16, device="meta") for s in ((3, 64), (100, 64)))
    assert [tuple(v.shape) for v in ops.lmhead_logprobs(h, w, t, 1.0, False, None)] == [(3,), (3,), (0, 4)]
    assert [tuple(v.shape) for v in ops.lmhead_logprobs_grad(h, w, t, stats, lp, None, 1.0, True, False, None)] == [(3, 64), (0, 64)]
    assert [tuple(v.shape) for v in ops.linear(h, w, None, None, 2, True, None)] == [(3, 100), (3, 104)]
    assert [tuple(v.shape) for v in ops.linear_grad(torch.empty(3, 100, dtype=torch.bfloat16, device="meta"), h, w, None, 0,
                                                    True, True, True, None)] == [(3, 64), (100, 64), (100,)]
