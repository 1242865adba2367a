"""Distillation of logits from a teacher's top entries, and through it the training of the lightning indexer (no reference
counterpart: its indexer examples are forward only).

* ``topk_distillation``               rows of logits against the teacher's top K entries of each row, differentiable in the logits
* ``lightning_indexer_distillation``  the same with the indexer's scores of a query's listed keys as its logits, differentiable in the
                                      indexer's queries, keys and head weights
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .adapter import check_inputs, current_stream, dtype_code, ptr

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


def _check_indexer(query, key, weights, indices, lists) -> torch.device:
    """Shapes and types of the indexer's inputs, its lists and the fp32 tensors [B,S1,1,K] that go with them."""
    if query.dim() != 4 or key.dim() != 4 or indices.dim() != 4:
        raise ValueError("query, key and indices must be 4-dimensional ([B,S1,N1,128], [B,S2,1,128], [B,S1,1,K])")
    B, S1, N1, D = query.shape
    if D != 128 or not 1 <= N1 <= 64:
        raise ValueError(f"the indexer's gradient needs head dim 128 and at most 64 heads, got {N1} heads of {D}")
    if key.shape != (B, key.shape[1], 1, D) or weights.shape != (B, S1, N1) or indices.shape[:3] != (B, S1, 1):
        raise ValueError(f"shape mismatch: query {tuple(query.shape)}, key {tuple(key.shape)}, weights {tuple(weights.shape)}, indices {tuple(indices.shape)}")
    if key.shape[1] < 1 or not 1 <= indices.shape[3] <= 8192:
        raise ValueError(f"at least one key and lists of 1 to 8192 entries are needed, got {key.shape[1]} and {indices.shape[3]}")
    dtype_code(query.dtype)
    for t, name in lists:
        if t.shape != indices.shape:
            raise ValueError(f"{name} must be {tuple(indices.shape)}, got {tuple(t.shape)}")
    return check_inputs([query, key, weights, indices] + [t for t, _ in lists],
                        [None, query.dtype, torch.float32, torch.int32] + [torch.float32] * len(lists),
                        ["query", "key", "weights", "indices"] + [name for _, name in lists])


def lightning_indexer_bwd_raw(query, key, weights, indices, d_values):
    """Gradients of the indexer's scores at listed keys: (d_query in the query's dtype, d_key fp32, d_weights fp32) for ``d_values``
    [B,S1,1,K] fp32.  Entries of ``indices`` outside [0, S2) take no part, whatever d_values holds there.  relu'(0) = 0.  The key
    gradient is summed with fp32 atomics: its last bits depend on their order."""
    dev = _check_indexer(query, key, weights, indices, [(d_values, "d_values")])
    B, S1, N1, D = query.shape
    d_query, d_weights = torch.empty_like(query), torch.empty_like(weights)
    d_key = torch.zeros(key.shape, dtype=torch.float32, device=dev)
    if B * S1:
        with torch.cuda.device(dev):
            _lib.check(_lib.load().dsa_lightning_indexer_bwd(
                ptr(query), ptr(key), ptr(weights), ptr(indices), ptr(d_values), ptr(d_query), ptr(d_key), ptr(d_weights), B, S1, key.shape[1], N1, D,
                indices.shape[3], dtype_code(query.dtype), current_stream(dev)))
    return d_query, d_key, d_weights


class LightningIndexerDistillationFunction(torch.autograd.Function):
    """Autograd node: distillation of the listed scores, and their gradient through the indexer."""

    @staticmethod
    def forward(ctx, query, key, weights, indices, values, teacher, teacher_kind, temperature):
        _check_indexer(query, key, weights, indices, [(values, "values"), (teacher, "teacher")])
        ctx.how = dict(teacher_kind=teacher_kind, temperature=temperature)
        loss, stats = topk_distillation_raw(values, teacher, None, **ctx.how)
        ctx.save_for_backward(query, key, weights, indices, values, teacher, stats)
        return loss.squeeze(2)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        query, key, weights, indices, values, teacher, stats = ctx.saved_tensors
        d_values = topk_distillation_bwd_raw(values, teacher, None, stats, grad.contiguous().unsqueeze(2), **ctx.how)
        d_query, d_key, d_weights = lightning_indexer_bwd_raw(query, key, weights, indices, d_values)
        return d_query, d_key.to(key.dtype), d_weights, None, None, None, None, None


def lightning_indexer_distillation(query, key, weights, indices, values, teacher, *, teacher_kind: str = "weights", temperature: float = 1.0):
    """Loss [B,S1] that trains the lightning indexer: KL divergence of its softmax over a query's listed keys from the teacher's
    (:func:`topk_distillation` over the list).  Gradients reach ``query``, ``key`` and ``weights``.

    query [B,S1,N1,128], key [B,S2,1,128] bf16 / fp16, weights [B,S1,N1] fp32 (at most 64 heads); ``indices`` and ``values``
    [B,S1,1,K] are what :func:`lightning_indexer_raw` returned for them (int32, -1 pads; fp32 scores, -inf there); ``teacher``
    [B,S1,1,K] fp32 its entries, e.g. from :func:`sparse_mla_key_weights`.  ``values`` are taken as the scores of these inputs: no
    gradient flows through them or through the teacher.  An entry takes part when its value is not -inf and its index lies in
    [0, S2)."""
    return LightningIndexerDistillationFunction.apply(query, key, weights, indices, values, teacher, teacher_kind, float(temperature))
