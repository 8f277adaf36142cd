"""``linear_cross_entropy`` / ``linear_distillation`` - the losses of a linear head over a large vocabulary, next to ``DiceCELoss``.

The logits ``hidden @ weight.T`` of a large call are never held whole: the forward pass keeps the maximum and the sum of exponentials of every row, the backward
pass rebuilds the logits in pieces of the vocabulary (``cs_head_loss_forward`` / ``cs_head_loss_backward``, csrc/kernels_head.hip).  That bounds the memory of
a step, but does not make it small: a backward pass has a workspace for the logits' gradient of a piece, up to 512 MiB in the inputs' type, once as it is and
once transposed, for that piece of the weight transposed, and for sums of the gradient of hidden.  8192 rows of 4096 over 131072 words, bf16: 1.5 GB, where
the logits in float32 take 4.3; but 4096 x 2048 over 50000 words: 1.1 against 0.8 GB, and 100 x 2048 over 65536: 370 against 26 MB.
With rows i, vocabulary j, ``z = hidden weight^T``, ``p_i = softmax(z_i / T)``:

    cross entropy   loss_i = -log p_i[target_i]                                       T = 1
    distillation    loss_i = T^2 sum_k q_ik (log q_ik - log p_i[teacher_ids_ik])      q_i = softmax(teacher_logits_i / T)

``hidden`` ``[..., D]`` and ``weight`` ``[V, D]`` share one type (bfloat16, float16 or float32) and get gradients of that type; products are
summed, and losses returned, in float32.  16-bit gradients of the logits are rounded once to the type of the inputs before they are
multiplied, an error of the size of the gradients' own last rounding (up to 64 rows they are kept as the sum of two 16-bit values).  For gradients of up to
64 rows the logits are kept where they take no more memory than the weight, and in float32, where to build them again takes longest, up to 512 MiB of
them.  A float16 net wants the usual loss scale: a mean over many rows makes gradients smaller than float16 holds.

Both directions can be captured into a graph; capture ``torch.autograd.grad``, as ``.backward()`` in a capture joins the stream on which an
earlier, still living graph of the same leaves was built, which torch does not survive.
"""
from __future__ import annotations

import ctypes as C

import torch
import torch.nn as nn

from . import _lib
from ._lib import check, lib

TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}          # CS_TYPE_*
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}                            # CS_REDUCE_*
_CROSS_ENTROPY, _DISTILLATION = 0, 1
MAX_TOP = 1024
MIN_TEMPERATURE = 1e-5


def _pitch(t: torch.Tensor) -> int:
    """Elements between the rows of a 2-d tensor with unit inner stride (of one row: its length)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def rows_of(t: torch.Tensor) -> torch.Tensor:
    """[..., D] -> [rows, D] with unit inner stride and rows that do not overlap; a copy only where the strides do not allow a view."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t


def _checked(hidden: torch.Tensor, weight: torch.Tensor, reduction: str, ids: torch.Tensor, name: str):
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction is one of {', '.join(_REDUCTIONS)}, got {reduction!r}")
    if hidden.dtype not in TYPES or weight.dtype != hidden.dtype:
        raise TypeError(f"hidden and weight share one of bfloat16, float16 and float32, got {hidden.dtype} and {weight.dtype}")
    if hidden.dim() < 1 or weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"expected hidden [..., D] and weight [V, D], got {tuple(hidden.shape)} and {tuple(weight.shape)}")
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{name} holds int64 or int32, got {ids.dtype}")
    for t in (hidden, weight, ids):
        if not t.is_cuda:
            _lib.require_gpu(t)
    if weight.device != hidden.device or ids.device != hidden.device:
        raise ValueError(f"hidden, weight and {name} are on one device, got {hidden.device}, {weight.device} and {ids.device}")


def _has_backward(hidden: torch.Tensor, weight: torch.Tensor) -> bool:
    """Whether a backward pass can follow (``ctx.needs_input_grad`` does not know of ``torch.no_grad()``)."""
    return torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad)


def _check_temperature(temperature: float) -> None:
    if not MIN_TEMPERATURE <= float(temperature) < 1e30:
        raise ValueError(f"temperature is at least {MIN_TEMPERATURE:g} and finite, got {temperature}")


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, *, ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """Softmax cross entropy of the logits ``hidden @ weight.T`` against ``target`` (``hidden.shape[:-1]``, int64 or int32) -> float32.

    Rows whose target is ``ignore_index`` have loss 0, no gradient, and are not counted; a mean over no row is 0.  Any other target
    outside ``[0, V)`` makes the loss and the gradients NaN (it is seen on the device only)."""
    _checked(hidden, weight, reduction, target, "target")
    if target.shape != hidden.shape[:-1]:
        raise ValueError(f"expected target {tuple(hidden.shape[:-1])}, got {tuple(target.shape)}")
    losses = _HeadLoss.apply(rows_of(hidden), rows_of(weight), target if target.dim() == 1 else target.reshape(-1), None, _CROSS_ENTROPY, _REDUCTIONS[reduction], int(ignore_index), 1.0,
                             _has_backward(hidden, weight))
    return losses.reshape(target.shape) if reduction == "none" else losses


def linear_distillation(hidden: torch.Tensor, weight: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor, *, temperature: float = 1.0,
                        reduction: str = "mean") -> torch.Tensor:
    """T^2 KL(teacher || student) of the student logits ``hidden @ weight.T`` against a teacher's top logits -> float32.

    ``teacher_ids`` (int64 or int32) and ``teacher_logits`` (bfloat16, float16 or float32) are ``[..., K]``, K up to 1024, in any order; the
    teacher's mass is spread over them alone, the student's over the whole vocabulary.  An entry with a negative id or a logit of -inf
    carries no mass; rows without mass have loss 0, no gradient, and are not counted; an id may come twice.  An id >= V makes the loss
    and the gradients NaN.  The teacher gets no gradient.

    ``temperature`` is 1e-5 or more: student logits beyond about 1e9 times the temperature make the loss infinite or NaN."""
    _checked(hidden, weight, reduction, teacher_ids, "teacher_ids")
    if teacher_ids.dim() != hidden.dim() or teacher_ids.shape[:-1] != hidden.shape[:-1] or teacher_logits.shape != teacher_ids.shape:
        raise ValueError(f"expected teacher_ids and teacher_logits {tuple(hidden.shape[:-1])} + (K,), got {tuple(teacher_ids.shape)} and {tuple(teacher_logits.shape)}")
    if not 1 <= teacher_ids.shape[-1] <= MAX_TOP:
        raise ValueError(f"a teacher gives 1 to {MAX_TOP} logits per row, got {teacher_ids.shape[-1]}")
    if teacher_logits.dtype not in TYPES:
        raise TypeError(f"teacher_logits holds bfloat16, float16 or float32, got {teacher_logits.dtype}")
    if teacher_logits.device != hidden.device:
        raise ValueError(f"teacher_logits is on {teacher_logits.device}, hidden on {hidden.device}")
    if teacher_logits.requires_grad and torch.is_grad_enabled():
        raise ValueError("the teacher gets no gradient: pass teacher_logits.detach()")
    _check_temperature(temperature)
    losses = _HeadLoss.apply(rows_of(hidden), rows_of(weight), rows_of(teacher_ids), rows_of(teacher_logits), _DISTILLATION, _REDUCTIONS[reduction], 0, float(temperature),
                             _has_backward(hidden, weight))
    return losses.reshape(hidden.shape[:-1]) if reduction == "none" else losses


class LinearCrossEntropyLoss(nn.Module):
    """``linear_cross_entropy`` as a module: ``loss(hidden, weight, target)``."""

    def __init__(self, ignore_index: int = -100, reduction: str = "mean"):
        super().__init__()
        if reduction not in _REDUCTIONS:
            raise ValueError(f"reduction is one of {', '.join(_REDUCTIONS)}, got {reduction!r}")
        self.ignore_index, self.reduction = ignore_index, reduction

    def forward(self, hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor) -> torch.Tensor:
        return linear_cross_entropy(hidden, weight, target, ignore_index=self.ignore_index, reduction=self.reduction)


class LinearDistillationLoss(nn.Module):
    """``linear_distillation`` as a module: ``loss(hidden, weight, teacher_ids, teacher_logits)``."""

    def __init__(self, temperature: float = 1.0, reduction: str = "mean"):
        super().__init__()
        if reduction not in _REDUCTIONS:
            raise ValueError(f"reduction is one of {', '.join(_REDUCTIONS)}, got {reduction!r}")
        _check_temperature(temperature)
        self.temperature, self.reduction = temperature, reduction

    def forward(self, hidden: torch.Tensor, weight: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor) -> torch.Tensor:
        return linear_distillation(hidden, weight, teacher_ids, teacher_logits, temperature=self.temperature, reduction=self.reduction)


def _descriptor(hidden, weight, kind, reduction, ignore_index, temperature, top, ids=None, teacher=None) -> _lib.HeadLoss:
    return _lib.HeadLoss(hidden=hidden.data_ptr(), weight=weight.data_ptr(), ids=ids.data_ptr() if ids is not None else None,
                         teacher=teacher.data_ptr() if teacher is not None else None, hidden_pitch=_pitch(hidden), weight_pitch=_pitch(weight),
                         ids_pitch=(ids.stride(0) if ids.shape[0] > 1 else top) if ids is not None else 0, teacher_pitch=_pitch(teacher) if teacher is not None else 0,
                         rows=hidden.shape[0], vocab=weight.shape[0], width=weight.shape[1], ignore_index=ignore_index, temperature=temperature,
                         type=TYPES[hidden.dtype], kind=kind, reduction=reduction, ids_bits=32 if ids is not None and ids.dtype == torch.int32 else 64,
                         teacher_type=TYPES[teacher.dtype] if teacher is not None else 0, top=top)


class _HeadLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, ids, teacher, kind, reduction, ignore_index, temperature, keep):
        top = 1 if teacher is None else ids.shape[1]
        head = _descriptor(hidden, weight, kind, reduction, ignore_index, temperature, top, ids, teacher)
        head.keep_scores = int(keep)
        with _lib.on_device(hidden.device):
            size = lib.cs_head_loss_saved_bytes(head)
            if not size:
                check(-1, "cs_head_loss_saved_bytes")
            saved = torch.empty(size, dtype=torch.uint8, device=hidden.device)
            ws = torch.empty(lib.cs_head_loss_workspace_bytes(head, 0) or 1, dtype=torch.uint8, device=hidden.device)
            loss = torch.empty((hidden.shape[0],) if reduction == 0 else (), dtype=torch.float32, device=hidden.device)
            to = loss.data_ptr()
            check(lib.cs_head_loss_forward(head, to if reduction == 0 else None, None if reduction == 0 else to, saved.data_ptr(), saved.numel(), ws.data_ptr(), ws.numel(),
                                           _lib.raw_stream(hidden.device)), "cs_head_loss_forward")
        ctx.save_for_backward(hidden, weight, saved)
        ctx.head = head
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        hidden, weight, saved = ctx.saved_tensors
        head = ctx.head
        head.hidden, head.weight = hidden.data_ptr(), weight.data_ptr()      # a saved-tensor hook may have moved them, with new strides
        head.hidden_pitch, head.weight_pitch = _pitch(hidden), _pitch(weight)
        need = ctx.needs_input_grad
        if grad.dtype != torch.float32:
            grad = grad.float()
        with _lib.on_device(hidden.device):
            gh = torch.empty_like(hidden, memory_format=torch.contiguous_format) if need[0] else None
            gw = torch.empty_like(weight, memory_format=torch.contiguous_format) if need[1] else None
            ws = torch.empty(lib.cs_head_loss_workspace_bytes(head, need[0] + 2 * need[1]) or 1, dtype=torch.uint8, device=hidden.device)
            check(lib.cs_head_loss_backward(head, saved.data_ptr(), saved.numel(), grad.data_ptr(), grad.stride(0) if grad.dim() else 0, gh.data_ptr() if need[0] else None,
                                            gw.data_ptr() if need[1] else None, ws.data_ptr(), ws.numel(), _lib.raw_stream(hidden.device)), "cs_head_loss_backward")
        return gh, gw, None, None, None, None, None, None, None
