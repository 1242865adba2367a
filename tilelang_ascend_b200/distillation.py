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
from .adapter import check_inputs, dtype_code, on_device, ptr, raw_stream

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_TEACHERS = {"weights": 0, "logits": 1}
_OVER = {"list": 0, "row": 1}


def _check_rows(student, teacher, indices, teacher_kind, over, temperature) -> torch.device:
    """Arguments of a distillation: [..., V] student rows, [..., K] teacher entries."""
    if teacher_kind not in _TEACHERS:
        raise ValueError(f"teacher_kind must be 'weights' or 'logits', got {teacher_kind!r}")
    if over not in _OVER:
        raise ValueError(f"over must be 'list' or 'row', got {over!r}")
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"temperature must be in [1e-30, 1e30], got {temperature}")
    for t, name in ((student, "student"), (teacher, "teacher")):
        if not isinstance(t, torch.Tensor) or t.dim() < 1:
            raise ValueError(f"{name} must be a tensor of rows")
        if t.dtype not in _TYPES:
            raise ValueError(f"Input tensor {name} has dtype {t.dtype}, expected bfloat16, float16 or float32")
    V, K, dev = student.shape[-1], teacher.shape[-1], student.device
    if teacher.shape[:-1] != student.shape[:-1]:
        raise ValueError(f"student {tuple(student.shape)} and teacher {tuple(teacher.shape)} must have the same rows")
    if V < 1 or K < 1:
        raise ValueError("rows need at least one column and one entry")
    if not teacher.is_contiguous():
        raise ValueError("Input tensor teacher must be contiguous")
    if indices is None:
        if K != V:
            raise ValueError(f"without indices the teacher has one entry per column (got {K} for {V})")
    else:
        if indices.dtype != torch.int32:
            raise ValueError(f"Input tensor indices has dtype {indices.dtype}, expected torch.int32")
        if indices.shape != teacher.shape or not indices.is_contiguous():
            raise ValueError(f"indices must be contiguous {tuple(teacher.shape)}, got {tuple(indices.shape)}")
    _row_stride(student)
    for t, name in ((teacher, "teacher"), (indices, "indices")):
        if t is not None and t.device != dev:
            raise ValueError(f"Input tensor {name} is on {t.device}, expected {dev}")
    return dev


def _row_stride(student) -> int:
    """Elements between a student's rows."""
    if student.is_contiguous():
        return student.shape[-1]
    try:
        rows = student.view(-1, student.shape[-1])
    except RuntimeError:
        rows = None
    if rows is None or (rows.stride(1) != 1 and rows.shape[1] > 1):
        raise ValueError("student must have unit inner stride and evenly spaced rows")
    return rows.stride(0)


def _head(student, teacher, indices):
    return student.data_ptr(), _TYPES[student.dtype], _row_stride(student), teacher.data_ptr(), _TYPES[teacher.dtype], ptr(indices)


def _tail(student, teacher, teacher_kind, over, temperature):
    V = student.shape[-1]
    return student.numel() // V, V, teacher.shape[-1], _OVER[over], _TEACHERS[teacher_kind], temperature


def _require_cuda(dev) -> None:
    if dev.type != "cuda":
        raise ValueError(f"kernels run on CUDA tensors only (got device {dev}); there is no CPU path")


def topk_distillation_raw(student, teacher, indices=None, *, teacher_kind: str = "weights", over: str = "list",
                          temperature: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss [...], stats [rows, 4]) of :func:`topk_distillation`; the backward takes the stats."""
    temperature = float(temperature)
    dev = _check_rows(student, teacher, indices, teacher_kind, over, temperature)
    _require_cuda(dev)
    tail = _tail(student, teacher, teacher_kind, over, temperature)
    loss = torch.empty(student.shape[:-1], dtype=torch.float32, device=dev)
    stats = torch.empty((tail[0], 4), dtype=torch.float32, device=dev)
    if tail[0]:
        lib = _lib.load()
        nbytes = lib.dsa_topk_distillation_workspace_bytes(tail[0], tail[1], tail[3], 1) if indices is not None else 0
        workspace = torch.empty((nbytes,), dtype=torch.uint8, device=dev) if nbytes else None
        with on_device(dev):
            _lib.check(lib.dsa_topk_distillation(*_head(student, teacher, indices), loss.data_ptr(), stats.data_ptr(), *tail, ptr(workspace), nbytes,
                                                 raw_stream(dev)))
    return loss, stats


def _gradient(student, teacher, indices, stats, grad, teacher_kind, over, temperature):
    """Gradient of checked rows."""
    dev, tail = student.device, _tail(student, teacher, teacher_kind, over, temperature)
    d_student = torch.empty(student.shape, dtype=student.dtype, device=dev)
    if tail[0]:
        with on_device(dev):
            _lib.check(_lib.load().dsa_topk_distillation_bwd(*_head(student, teacher, indices), stats.data_ptr(), grad.data_ptr(), d_student.data_ptr(), *tail,
                                                             raw_stream(dev)))
    return d_student


def topk_distillation_bwd_raw(student, teacher, indices, stats, grad, *, teacher_kind: str = "weights", over: str = "list", temperature: float = 1.0):
    """Gradient of the student's rows (contiguous, the student's dtype) for ``grad`` [...] of the losses."""
    temperature = float(temperature)
    dev = _check_rows(student, teacher, indices, teacher_kind, over, temperature)
    for t, name, shape in ((stats, "stats", (student.numel() // student.shape[-1], 4)), (grad, "grad", student.shape[:-1])):
        if t.dtype != torch.float32 or t.shape != shape or not t.is_contiguous() or t.device != dev:
            raise ValueError(f"{name} must be contiguous float32 {tuple(shape)} on {dev}")
    _require_cuda(dev)
    return _gradient(student, teacher, indices, stats, grad, teacher_kind, over, temperature)


class TopkDistillationFunction(torch.autograd.Function):
    """Autograd node over the forward / backward kernels."""

    @staticmethod
    def forward(ctx, student, teacher, indices, teacher_kind, over, temperature):
        loss, stats = topk_distillation_raw(student, teacher, indices, teacher_kind=teacher_kind, over=over, temperature=temperature)
        ctx.how = teacher_kind, over, float(temperature)
        ctx.save_for_backward(student, teacher, indices, stats)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return _gradient(*ctx.saved_tensors, grad.contiguous(), *ctx.how), None, None, None, None, None


def topk_distillation(student, teacher, indices: Optional[torch.Tensor] = None, *, teacher_kind: str = "weights", over: str = "list",
                      temperature: float = 1.0):
    """KL divergence, row by row, of a student's logits from a teacher's top entries: ``loss = sum_j p_j (log p_j - log s_j)``.

    student [..., V] fp32 / bf16 / fp16 logits (unit inner stride, evenly spaced rows); teacher [..., K] the entries' ``"weights"``
    (not below 0, any sum from 1e-30 to 3e38; what fp32 cannot add up gives NaN) or ``"logits"``; indices [..., K] int32 their columns,
    or None when every column has its entry (K = V).
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
    [B,S1,1,K] fp32.  Entries of ``indices`` outside [0, S2) take no part, whatever d_values holds there.  relu'(0) = 0, and a score
    that is NaN is passed on, as autograd's relu does.  The key gradient is summed with fp32 atomics: its last bits depend on their
    order (the others' only where a list names a key three times or more)."""
    _check_indexer(query, key, weights, indices, [(d_values, "d_values")])
    return _indexer_gradients(query, key, weights, indices, d_values)


def _indexer_gradients(query, key, weights, indices, d_values):
    """The same for checked tensors."""
    B, S1, N1, D = query.shape
    dev = query.device
    d_query, d_weights = torch.empty_like(query), torch.empty_like(weights)
    d_key = torch.zeros(key.shape, dtype=torch.float32, device=dev)
    if B * S1:
        lib = _lib.load()
        sizes = B, S1, key.shape[1], N1, D, indices.shape[3], dtype_code(query.dtype)
        nbytes = lib.dsa_lightning_indexer_bwd_workspace_bytes(*sizes)
        workspace = torch.empty((nbytes,), dtype=torch.uint8, device=dev) if nbytes else None
        with on_device(dev):
            _lib.check(lib.dsa_lightning_indexer_bwd(
                query.data_ptr(), key.data_ptr(), weights.data_ptr(), indices.data_ptr(), d_values.data_ptr(), d_query.data_ptr(), d_key.data_ptr(),
                d_weights.data_ptr(), *sizes, ptr(workspace), nbytes, raw_stream(dev)))
    return d_query, d_key, d_weights


class LightningIndexerDistillationFunction(torch.autograd.Function):
    """Autograd node: distillation of the listed scores, and their gradient through the indexer."""

    @staticmethod
    def forward(ctx, query, key, weights, indices, values, teacher, teacher_kind, temperature):
        _check_indexer(query, key, weights, indices, [(values, "values"), (teacher, "teacher")])
        loss, stats = topk_distillation_raw(values, teacher, None, teacher_kind=teacher_kind, temperature=temperature)
        ctx.how = teacher_kind, "list", float(temperature)
        ctx.save_for_backward(query, key, weights, indices, values, teacher, stats)
        return loss.squeeze(2)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        query, key, weights, indices, values, teacher, stats = ctx.saved_tensors
        d_values = _gradient(values, teacher, None, stats, grad.contiguous(), *ctx.how)
        d_query, d_key, d_weights = _indexer_gradients(query, key, weights, indices, d_values)
        return d_query, d_key.to(key.dtype), d_weights, None, None, None, None, None


def lightning_indexer_distillation(query, key, weights, indices, values, teacher, *, teacher_kind: str = "weights", temperature: float = 1.0):
    """Loss [B,S1] that trains the lightning indexer: KL divergence of its softmax over a query's listed keys from the teacher's
    (:func:`topk_distillation` over the list).  Gradients reach ``query``, ``key`` and ``weights``.

    query [B,S1,N1,128], key [B,S2,1,128] bf16 / fp16, weights [B,S1,N1] fp32 (at most 64 heads); ``indices`` and ``values``
    [B,S1,1,K] are what :func:`lightning_indexer_raw` returned for them (int32, -1 pads; fp32 scores, -inf there); ``teacher``
    [B,S1,1,K] fp32 its entries, e.g. from :func:`sparse_mla_key_weights`.  ``values`` are taken as the scores of these inputs: no
    gradient flows through them or through the teacher.  An entry takes part when its value is not -inf; one whose index lies
    outside [0, S2) must have the value -inf, as it has there."""
    return LightningIndexerDistillationFunction.apply(query, key, weights, indices, values, teacher, teacher_kind, float(temperature))
