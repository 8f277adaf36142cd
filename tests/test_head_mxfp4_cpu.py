"""Refusals of the head losses and the 4-bit operators, and the descriptor's layout: nothing here runs on a GPU."""
import ctypes as C
import os
import subprocess

import pytest
import torch

import cellseg_amd as ca
from cellseg_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
H, W, T = torch.randn(4, 8), torch.randn(10, 8), torch.zeros(4, dtype=torch.int64)
IDS, LOGITS = torch.zeros(4, 3, dtype=torch.int64), torch.zeros(4, 3)


def test_head_descriptor_layout_matches_the_c_header(tmp_path):
    fields = [f[0] for f in _lib.HeadLoss._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "cellseg_hip.h"\nint main(void) {\n  printf("%zu", sizeof(cs_head_loss));\n'
                   + "".join(f'  printf(" %zu", offsetof(cs_head_loss, {f}));\n' for f in fields) + "  return 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [C.sizeof(_lib.HeadLoss)] + [getattr(_lib.HeadLoss, f).offset for f in fields]


@pytest.mark.parametrize("call,error", [
    (lambda: ca.linear_cross_entropy(H, W, T), ca.CellSegHipError),                                   # CPU tensors: no fallback
    (lambda: ca.linear_cross_entropy(H, W.bfloat16(), T), TypeError),
    (lambda: ca.linear_cross_entropy(H.double(), W.double(), T), TypeError),
    (lambda: ca.linear_cross_entropy(H, W, T.float()), TypeError),
    (lambda: ca.linear_cross_entropy(H, W[:, :7], T), ValueError),
    (lambda: ca.linear_cross_entropy(H, W[:0], T), ValueError),
    (lambda: ca.linear_cross_entropy(H, W[None], T), ValueError),
    (lambda: ca.linear_cross_entropy(H, W, T, reduction="batchmean"), ValueError),
    (lambda: ca.linear_distillation(H, W, IDS, LOGITS), ca.CellSegHipError),
    (lambda: ca.LinearCrossEntropyLoss(reduction="x"), ValueError),
    (lambda: ca.LinearDistillationLoss(temperature=0.0), ValueError),
    (lambda: ca.mxfp4_quantize(H), ca.CellSegHipError),
    (lambda: ca.mxfp4_quantize(H.double()), TypeError),
    (lambda: ca.mxfp4_quantize(H[:, :0]), ValueError),
    (lambda: ca.mxfp4_quantize(H.clone().requires_grad_()), ValueError),
    (lambda: ca.mxfp4_linear(H, W), TypeError),
    (lambda: ca.MXFP4Tensor(torch.zeros(3, 15, dtype=torch.uint8), torch.zeros(3, 1, dtype=torch.uint8), 32), ValueError),
    (lambda: ca.MXFP4Tensor(torch.zeros(3, 16, dtype=torch.uint8), torch.zeros(3, 2, dtype=torch.uint8), 32), ValueError),
    (lambda: ca.MXFP4Tensor(torch.zeros(3, 16), torch.zeros(3, 1, dtype=torch.uint8), 32), ValueError),
    (lambda: ca.MXFP4Tensor(torch.zeros(3, 16, dtype=torch.uint8), torch.zeros(3, 1, dtype=torch.uint8), 32, torch.int8), TypeError),
    (lambda: ca.mxfp4_linear(H[:, :7], ca.MXFP4Tensor(torch.zeros(3, 16, dtype=torch.uint8), torch.zeros(3, 1, dtype=torch.uint8), 8)), ValueError),
    (lambda: ca.mxfp4_linear(H.clone().requires_grad_(), ca.MXFP4Tensor(torch.zeros(3, 16, dtype=torch.uint8), torch.zeros(3, 1, dtype=torch.uint8), 8)), ValueError),
    (lambda: ca.mxfp4_linear(H, ca.MXFP4Tensor(torch.zeros(3, 16, dtype=torch.uint8), torch.zeros(3, 1, dtype=torch.uint8), 8)), ca.CellSegHipError),
])
def test_refusals(call, error):
    with pytest.raises(error):
        call()


def head(**over):
    d = dict(hidden=4096, weight=8192, ids=4096, teacher=None, hidden_pitch=8, weight_pitch=8, ids_pitch=1, teacher_pitch=0, rows=4, vocab=10, width=8, ignore_index=-100,
             temperature=1.0, type=0, kind=0, reduction=1, ids_bits=64, teacher_type=0, top=1)
    d.update(over)
    return _lib.HeadLoss(**d)


@pytest.mark.parametrize("over", [dict(rows=-1), dict(rows=1 << 26), dict(vocab=0), dict(vocab=1 << 30), dict(width=0), dict(width=1 << 21), dict(type=3), dict(kind=2), dict(reduction=3),
                                  dict(ids_bits=16), dict(top=2), dict(temperature=2.0), dict(kind=1, top=0), dict(kind=1, top=1025), dict(kind=1, temperature=0.0),
                                  dict(kind=1, temperature=float("nan")), dict(kind=1, teacher_type=4), dict(hidden_pitch=7), dict(weight_pitch=7)])
def test_the_c_entry_refuses(over):
    """Bad descriptors and NULL pointers are refused before anything is launched (no GPU is needed to see that)."""
    h = head(**over)
    assert _lib.lib.cs_head_loss_saved_bytes(C.byref(h)) == 0 and _lib.lib.cs_head_loss_workspace_bytes(C.byref(h), 3) == 0
    assert _lib.lib.cs_head_loss_forward(C.byref(h), None, 4096, 4096, 1 << 40, 4096, 1 << 40, None) == -1
    assert _lib.lib.cs_head_loss_backward(C.byref(h), 4096, 1 << 40, 4096, 0, 4096, 4096, 4096, 1 << 40, None) == -1


def test_the_c_entry_refuses_small_workspaces_and_null():
    h = head()
    saved, ws = _lib.lib.cs_head_loss_saved_bytes(C.byref(h)), _lib.lib.cs_head_loss_workspace_bytes(C.byref(h), 0)
    assert saved > 0 and ws > 0
    assert _lib.lib.cs_head_loss_forward(C.byref(h), None, 4096, 4096, saved - 1, 4096, ws, None) == -3
    assert _lib.lib.cs_head_loss_forward(C.byref(h), None, 4096, 4096, saved, 4096, ws - 1, None) == -3
    assert _lib.lib.cs_head_loss_forward(C.byref(h), None, 4096, None, saved, 4096, ws, None) == -1
    back = _lib.lib.cs_head_loss_workspace_bytes(C.byref(h), 3)
    assert _lib.lib.cs_head_loss_backward(C.byref(h), 4096, saved, 4096, 0, 4096, 4096, 4096, back - 1, None) == -3
    assert _lib.lib.cs_head_loss_backward(C.byref(h), 4096, saved, None, 0, 4096, 4096, 4096, back, None) == -1
    assert _lib.lib.cs_head_loss_backward(C.byref(h), 4096, saved, 4096, 0, 4100, 4096, 4096, back, None) == -1
    assert _lib.lib.cs_mxfp4_quantize(4096, 8, 4, 0, 0, 4096, 4096, None) == -1
    assert _lib.lib.cs_mxfp4_quantize(4096, 8, 4, 8, 5, 4096, 4096, None) == -1
    assert _lib.lib.cs_mxfp4_quantize(None, 8, 4, 8, 0, 4096, 4096, None) == -1
    assert _lib.lib.cs_mxfp4_dequantize(4098, 4096, 4, 8, 0, 4096, None) == -1
    size = _lib.lib.cs_mxfp4_linear_workspace_bytes(40, 8, 6)
    assert size > 0 and _lib.lib.cs_mxfp4_linear(4096, 8, 40, 8, 0, 4096, 4096, 6, 4096, 4096, size - 1, None) == -3
    assert _lib.lib.cs_mxfp4_linear(4096, 8, 40, 8, 0, 4096, 4096, 6, 4096, None, size, None) == -1
    assert _lib.lib.cs_mxfp4_linear(4096, 8, 40, 8, 0, 4100, 4096, 6, 4096, 4096, size, None) == -1


def test_workspaces_of_no_rows():
    h = head(rows=0, hidden=None)
    assert _lib.lib.cs_head_loss_saved_bytes(C.byref(h)) > 0
    for backward in range(4):
        assert _lib.lib.cs_head_loss_workspace_bytes(C.byref(h), backward) == 0


def test_kept_scores_are_counted_and_bounded_by_the_weight():
    """keep_scores: 64 rows at most, whole 16 rows of 128 words in fp32, and no more than the weight's own row."""
    size = lambda **over: _lib.lib.cs_head_loss_saved_bytes(C.byref(head(hidden_pitch=512, weight_pitch=512, width=512, vocab=1000, **over)))
    assert size(keep_scores=1) - size(keep_scores=0) == 1024 * 16 * 4
    assert size(rows=64, keep_scores=1) - size(rows=64) == 1024 * 64 * 4
    assert size(rows=65, keep_scores=1) == size(rows=65)
    for rows, width, kind, kept in ((64, 128, 0, True), (64, 127, 0, False), (64, 64, 2, True), (64, 63, 2, False), (1, 32, 1, True), (1, 31, 1, False), (0, 64, 0, False)):
        d = dict(rows=rows, width=width, type=kind, hidden_pitch=width, weight_pitch=width)
        with_scores, without = (_lib.lib.cs_head_loss_saved_bytes(C.byref(head(keep_scores=k, **d))) for k in (1, 0))
        assert (with_scores > without) == kept, (rows, width, kind)


def test_kept_float32_scores_are_bounded():
    size = lambda **over: _lib.lib.cs_head_loss_saved_bytes(C.byref(head(hidden_pitch=64, weight_pitch=64, width=64, **over)))
    assert size(rows=100, vocab=1000, type=2, keep_scores=1) - size(rows=100, vocab=1000, type=2) == -(-100 * (1024 + 32) * 4 // 256) * 256
    assert size(rows=100, vocab=1000, type=0, keep_scores=1) == size(rows=100, vocab=1000, type=0)
    assert size(rows=1024, vocab=131072, type=2, keep_scores=1) > size(rows=1024, vocab=131072, type=2)
    assert size(rows=1025, vocab=131072, type=2, keep_scores=1) == size(rows=1025, vocab=131072, type=2)


def test_sizes_beyond_a_launch_are_refused():
    h = head(rows=1 << 24)
    assert _lib.lib.cs_head_loss_saved_bytes(C.byref(h)) == 0
    assert _lib.lib.cs_mxfp4_linear(4096, 8, 1, 8, 0, 4096, 4096, 1 << 28, 4096, 4096, 1 << 60, None) == -1
    assert _lib.lib.cs_mxfp4_linear(4096, 8, 1 << 29, 8, 0, 4096, 4096, 1 << 29, 4096, 4096, 1 << 60, None) == -1


def test_a_forward_mode_tangent_is_refused():
    """A dual tensor has requires_grad False; its result would come back without a tangent."""
    weight = ca.MXFP4Tensor(torch.zeros(3, 16, dtype=torch.uint8), torch.zeros(3, 1, dtype=torch.uint8), 8)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(H, torch.ones_like(H))
        for call in (lambda: ca.mxfp4_quantize(dual), lambda: ca.mxfp4_linear(dual, weight), lambda: ca.mxfp4_linear(dual[0], weight)):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="forward-mode"):
                    call()
        with pytest.raises(ca.CellSegHipError):                          # without its tangent it is taken, and refused for being on the CPU
            ca.mxfp4_quantize(dual.detach())


@pytest.mark.parametrize("temperature", [1e-45, 4e-39, 1e-8, 9.9e-6, float("inf")])
def test_temperatures_that_leave_the_range_of_the_exponents_are_refused(temperature):
    """Below 1e-8 logits of an ordinary size would come back as NaN."""
    with pytest.raises(ValueError, match="temperature"):
        ca.LinearDistillationLoss(temperature=temperature)
    h = head(kind=1, teacher=4096, temperature=temperature)
    assert _lib.lib.cs_head_loss_saved_bytes(C.byref(h)) == 0 and _lib.lib.cs_head_loss_workspace_bytes(C.byref(h), 3) == 0


def test_the_lowest_temperature_is_taken():
    assert ca.LinearDistillationLoss(temperature=1e-5).temperature == 1e-5
    assert _lib.lib.cs_head_loss_saved_bytes(C.byref(head(kind=1, teacher=4096, temperature=1e-5))) > 0
