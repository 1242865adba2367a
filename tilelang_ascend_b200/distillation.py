"""Distillation of logits from a teacher's top entries, and through it the training of the lightning indexer (no reference
counterpart: its indexer examples are forward only).

* ``topk_distillation``  rows of logits against the teacher's top K entries of each row, differentiable in the logits
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .adapter import current_stream, ptr

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_TEACHERS = {"weights": 0, "logits": 1}
_OVER = {"list": 0, "row": 1}


class _Rows:
    """Checked arguments of a distillation: [..., V] student rows, [..., K] teacher entries."""

    def __init__(self, student, teacher, indices, teacher_kind, over, temperature):
        if teacher_kind not in _TEACHERS:
            raise ValueError(f"teacher_kind must be 'weights' or 'logits', got {teacher_kind!r}")
        if over not in _OVER:
            raise ValueError(f"over must be 'list' or 'row', got {over!r}")
        self.temperature = float(temperature)
        if not 0.0 < self.temperature < float("inf"):
            raise ValueError(f"temperature must be positive and finite, got {temperature}")
        for t, name in ((student, "student"), (teacher, "teacher")):
            if not isinstance(t, torch.Tensor) or t.dim() < 1:
                raise ValueError(f"{name} must be a tensor of rows")
            if t.dtype not in _TYPES:
                raise ValueError(f"Input tensor {name} has dtype {t.dtype}, expected bfloat16, float16 or float32")
        self.lead, self.V, self.K = student.shape[:-1], student.shape[-1], teacher.shape[-1]
        if teacher.shape[:-1] != self.lead:
            raise ValueError(f"student {tuple(student.shape)} and teacher {tuple(teacher.shape)} must have the same rows")
        if self.V < 1 or self.K < 1:
            raise ValueError("rows need at least one column and one entry")
        if not teacher.is_contiguous():
            raise ValueError("Input tensor teacher must be contiguous")
        if indices is None:
            if self.K != self.V:
                raise ValueError(f"without indices the teacher has one entry per column (got {self.K} for {self.V})")
        else:
            if indices.dtype != torch.int32:
                raise ValueError(f"Input tensor indices has dtype {indices.dtype}, expected torch.int32")
            if indices.shape != teacher.shape or not indices.is_contiguous():
                raise ValueError(f"indices must be contiguous {tuple(teacher.shape)}, got {tuple(indices.shape)}")
        try:
            rows = student.view(-1, self.V) if student.numel() else student
        except RuntimeError:
            rows = None
        if rows is None or (student.numel() and self.V > 1 and rows.stride(1) != 1):
            raise ValueError("student must have unit inner stride and evenly spaced rows")
        self.rows = student.numel() // self.V
        self.row_stride = rows.stride(0) if student.numel() else self.V
        self.dev = student.device
        for t, name in ((teacher, "teacher"), (indices, "indices")):
            if t is not None and t.device != self.dev:
                raise ValueError(f"Input tensor {name} is on {t.device}, expected {self.dev}")
        self.head = (ptr(student), _TYPES[student.dtype], self.row_stride, ptr(teacher), _TYPES[teacher.dtype], ptr(indices))
        self.tail = (self.rows, self.V, self.K, _OVER[over], _TEACHERS[teacher_kind], self.temperature)

    def require_cuda(self) -> None:
        if self.dev.type != "cuda":
            raise ValueError(f"kernels run on CUDA tensors only (got device {self.dev}); there is no CPU path")


def topk_distillation_raw(student, teacher, indices=None, *, teacher_kind: str = "weights", over: str = "list",
                          temperature: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss [...], stats [rows, 4]) of :func:`topk_distillation`; the backward takes the stats."""
    r = _Rows(student, teacher, indices, teacher_kind, over, temperature)
    r.require_cuda()
    loss = torch.empty(r.lead, dtype=torch.float32, device=r.dev)
    stats = torch.empty((r.rows, 4), dtype=torch.float32, device=r.dev)
    if r.rows:
        with torch.cuda.device(r.dev):
            _lib.check(_lib.load().dsa_topk_distillation(*r.head, ptr(loss), ptr(stats), *r.tail, current_stream(r.dev)))
    return loss, stats


def topk_distillation_bwd_raw(student, teacher, indices, stats, grad, *, teacher_kind: str = "weights", over: str = "list", temperature: float = 1.0):
    """Gradient of the student's rows (contiguous, the student's dtype) for ``grad`` [...] of the losses."""
    r = _Rows(student, teacher, indices, teacher_kind, over, temperature)
    for t, name, shape in ((stats, "stats", (r.rows, 4)), (grad, "grad", tuple(r.lead))):
        if t.dtype != torch.float32 or tuple(t.shape) != shape or not t.is_contiguous() or t.device != r.dev:
            raise ValueError(f"{name} must be contiguous float32 {shape} on {r.dev}")
    r.require_cuda()
    d_student = torch.empty(student.shape, dtype=student.dtype, device=r.dev)
    if r.rows:
        with torch.cuda.device(r.dev):
            _lib.check(_lib.load().dsa_topk_distillation_bwd(*r.head, ptr(stats), ptr(grad), ptr(d_student), *r.tail, current_stream(r.dev)))
    return d_student


class TopkDistillationFunction(torch.autograd.Function):
    """Autograd node over the forward / backward kernels."""

    @staticmethod
    def forward(ctx, student, teacher, indices, teacher_kind, over, temperature):
        ctx.how = dict(teacher_kind=teacher_kind, over=over, temperature=temperature)
        loss, stats = topk_distillation_raw(student, teacher, indices, **ctx.how)
        ctx.save_for_backward(student, teacher, indices, stats)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        student, teacher, indices, stats = ctx.saved_tensors
        if not ctx.needs_input_grad[0]:
            return (None,) * 6
        return (topk_distillation_bwd_raw(student, teacher, indices, stats, grad.contiguous(), **ctx.how),) + (None,) * 5


def topk_distillation(student, teacher, indices: Optional[torch.Tensor] = None, *, teacher_kind: str = "weights", over: str = "list",
                      temperature: float = 1.0):
    """KL divergence, row by row, of a student's logits from a teacher's top entries: ``loss = sum_j p_j (log p_j - log s_j)``.

    student [..., V] fp32 / bf16 / fp16 logits (unit inner stride, evenly spaced rows); teacher [..., K] the entries' ``"weights"``
    (not below 0, any sum) or ``"logits"``; indices [..., K] int32 their columns, or None when every column has its entry (K = V).
    An entry takes part when its column lies in [0, V) and the student's logit there is not -inf; -1 pads a list, and what the
    teacher holds at entries that take no part is not looked at.  p are the participating entries normalised (logits: softmax of
    logit / temperature), s the softmax of student / temperature ``over`` the participating entries (``"list"``) or over the whole row
    (``"row"``).  A row whose teacher holds nothing has loss 0 and gradient 0.  Returns fp32 losses [...]; the gradient reaches the
    student only.  A column that a row lists twice counts twice in p (and in a list's s)."""
    return TopkDistillationFunction.apply(student, teacher, indices, teacher_kind, over, temperature)
