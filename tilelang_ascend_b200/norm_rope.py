"""Norm of every head's query and key rows and rotation by their tokens' positions, in one pass.

The attention and indexer entry points of this package take rotated queries and keys, and their decode forms read them from
paged caches; these calls make both (no reference counterpart: its examples start from rotated tensors):

* ``qk_norm_rope``         differentiable, returns the rows as new tensors (prefill, training)
* ``qk_norm_rope_cached``  writes the key rows straight into a paged cache, kept in one part ([num_blocks, block_size, heads, D]) or
                           in two (``key_cache_rope``: the rotated tail apart, as the MLA decode entry points read it)
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .adapter import current_stream, dtype_code, ptr

NORMS = {None: 0, "rms": 1, "layer": 2}


def _check_rows(x, name: str, like=None) -> None:
    if not isinstance(x, torch.Tensor):
        raise ValueError(f"{name}: expected a torch.Tensor, got {type(x).__name__}")
    if x.dim() != 4:
        raise ValueError(f"{name} must be [B, S, heads, D], got {tuple(x.shape)}")
    if x.shape[3] > 1 and x.stride(3) != 1 and x.numel():
        raise ValueError(f"Input tensor {name} must have unit inner stride")
    dtype_code(x.dtype)
    if like is not None and (x.shape[:2] != like.shape[:2] or x.shape[3] != like.shape[3] or x.dtype != like.dtype):
        raise ValueError(f"q and k must agree in B, S, D and dtype (got {tuple(like.shape)} {like.dtype}, {tuple(x.shape)} {x.dtype})")


def _check_vector(t, name: str, n: int, dtypes) -> None:
    if t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector of {n} values, got {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"Input tensor {name} has dtype {t.dtype}, expected one of {', '.join(str(d) for d in dtypes)}")


def _token_numbers(t, name: str, B: int, S: int) -> int:
    """1 for int64, 0 for int32."""
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be an int32 or int64 tensor")
    if tuple(t.shape) != (B, S) or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous [{B}, {S}], got {tuple(t.shape)}")
    return int(t.dtype == torch.int64)


class _Call:
    """Checked arguments of a call, without its outputs."""

    def __init__(self, q, k, positions, inv_freq, rope_start, interleaved, rope_scale, q_norm, k_norm, q_weight, q_bias, k_weight, k_bias,
                 norm_dim, eps, others=()):
        first = q if q is not None else k
        if first is None:
            raise ValueError("queries or keys must be given")
        if q is not None:
            _check_rows(q, "q")
        if k is not None:
            _check_rows(k, "k", q)
        self.B, self.S, _, self.D = first.shape
        self.dtype, self.code, self.dev = first.dtype, dtype_code(first.dtype), first.device
        self.positions, self.inv_freq = positions, inv_freq
        self.positions64 = _token_numbers(positions, "positions", self.B, self.S)
        if not isinstance(inv_freq, torch.Tensor) or inv_freq.dim() != 1:
            raise ValueError("inv_freq must be a vector with one frequency per rotated pair")
        _check_vector(inv_freq, "inv_freq", inv_freq.shape[0], (torch.float32,))
        self.R, self.rope_start = 2 * inv_freq.shape[0], int(rope_start)
        if self.R < 2 or self.rope_start < 0 or self.rope_start + self.R > self.D:
            raise ValueError(f"the rotated dims [{self.rope_start}, {self.rope_start + self.R}) must lie inside rows of {self.D}")
        self.norm_dim = self.D if norm_dim is None else int(norm_dim)
        if not 1 <= self.norm_dim <= self.D:
            raise ValueError(f"norm_dim must be in [1, {self.D}], got {norm_dim}")
        self.interleaved, self.rope_scale, self.eps = bool(interleaved), float(rope_scale), float(eps)
        self.norms, self.params, self.rows = (q_norm, k_norm), ((q_weight, q_bias), (k_weight, k_bias)), (q, k)
        tensors = [(positions, "positions"), (inv_freq, "inv_freq"), *others]
        for side, x, norm, (weight, bias) in (("q", q, q_norm, self.params[0]), ("k", k, k_norm, self.params[1])):
            if norm not in NORMS:
                raise ValueError(f"{side}_norm must be None, 'rms' or 'layer', got {norm!r}")
            given = [(t, f"{side}_{what}") for t, what in ((weight, "weight"), (bias, "bias")) if t is not None]
            if given and (norm is None or x is None):
                raise ValueError(f"{given[0][1]} needs {side} and its norm")
            for t, name in given:
                _check_vector(t, name, self.norm_dim, (torch.float32, self.dtype))
            if len(given) == 2 and weight.dtype != bias.dtype:
                raise ValueError(f"{side}_weight and {side}_bias must have one dtype")
            tensors += given + ([(x, side)] if x is not None else [])
        for t, name in tensors:
            if t.device != self.dev:
                raise ValueError(f"Input tensor {name} is on {t.device}, expected {self.dev}")

    def require_cuda(self) -> None:
        if self.dev.type != "cuda":
            raise ValueError(f"kernels run on CUDA tensors only (got device {self.dev}); there is no CPU path")

    def side(self, i: int, out, tail=None, split: Optional[int] = None, slots=None, y_slots: int = 0):
        """The C struct of queries (0) or keys (1) written to ``out``; None when they are not there."""
        x = self.rows[i]
        if x is None:
            return None
        weight, bias = self.params[i]
        param = weight if weight is not None else bias
        st = x.stride()
        return _lib.RopeRows(x=ptr(x), stride_b=st[0], stride_s=st[1], stride_h=st[2], heads=x.shape[2], norm=NORMS[self.norms[i]],
                             weight=ptr(weight), bias=ptr(bias), params_fp32=int(param is not None and param.dtype == torch.float32),
                             split=self.D if split is None else split, y=ptr(out), y_tail=ptr(tail), slots=ptr(slots), y_slots=y_slots,
                             slots_int64=int(slots is not None and slots.dtype == torch.int64))

    def scalars(self):
        return (ptr(self.positions), self.positions64, ptr(self.inv_freq), self.B, self.S, self.D, self.R, self.rope_start, self.norm_dim,
                1 if self.interleaved else 0, self.rope_scale, self.eps)

    def run(self, q_side, k_side) -> None:
        with torch.cuda.device(self.dev):
            ref = [None if s is None else ctypes.byref(s) for s in (q_side, k_side)]
            _lib.check(_lib.load().dsa_norm_rope(*ref, *self.scalars(), self.code, current_stream(self.dev)))


def _new_rows(x):
    return None if x is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)


class QkNormRopeFunction(torch.autograd.Function):
    """Autograd node over the forward / backward kernels."""

    @staticmethod
    def forward(ctx, q, k, q_weight, q_bias, k_weight, k_bias, positions, inv_freq, rope_start, interleaved, rope_scale, q_norm, k_norm, norm_dim, eps):
        call = _Call(q, k, positions, inv_freq, rope_start, interleaved, rope_scale, q_norm, k_norm, q_weight, q_bias, k_weight, k_bias, norm_dim, eps)
        call.require_cuda()
        outs = [_new_rows(q), _new_rows(k)]
        if call.B * call.S and any(o is not None and o.numel() for o in outs):
            sides = [None if o is None or not o.numel() else call.side(i, o) for i, o in enumerate(outs)]
            call.run(*sides)
        # (rows without a norm are not needed again: their gradient is the rotation of the outputs')
        keep = [x if norm is not None else None for x, norm in zip((q, k), call.norms)]
        ctx.save_for_backward(*keep, q_weight, q_bias, k_weight, k_bias, positions, inv_freq)
        ctx.shapes = [None if x is None else (x.shape, x.dtype) for x in (q, k)]
        ctx.rest = (rope_start, interleaved, rope_scale, q_norm, k_norm, norm_dim, eps)
        return tuple(outs)

    @staticmethod
    @once_differentiable
    def backward(ctx, *d_outs):
        q, k, q_weight, q_bias, k_weight, k_bias, positions, inv_freq = ctx.saved_tensors
        rope_start, interleaved, rope_scale, q_norm, k_norm, norm_dim, eps = ctx.rest
        grads = [None] * 15
        for i, (d_y, x, norm, weight, bias) in enumerate(zip(d_outs, (q, k), (q_norm, k_norm), (q_weight, k_weight), (q_bias, k_bias))):
            need_x, need_w, need_b = ctx.needs_input_grad[i], ctx.needs_input_grad[2 + 2 * i], ctx.needs_input_grad[3 + 2 * i]
            if d_y is None or ctx.shapes[i] is None or not (need_x or need_w or need_b):
                continue
            grads[i], grads[2 + 2 * i], grads[3 + 2 * i] = qk_norm_rope_bwd_raw(
                d_y, x, positions, inv_freq, rope_start=rope_start, interleaved=interleaved, rope_scale=rope_scale, norm=norm, weight=weight,
                bias=bias, norm_dim=norm_dim, eps=eps, need_params=(need_w, need_b))
        return tuple(grads)


def qk_norm_rope_bwd_raw(d_y, x, positions, inv_freq, *, rope_start: int = 0, interleaved: bool = True, rope_scale: float = 1.0, norm=None, weight=None,
                         bias=None, norm_dim: Optional[int] = None, eps: float = 1e-6, need_params: Tuple[bool, bool] = (True, True)):
    """(dx, dweight or None, dbias or None) of one side: ``d_y`` [B,S,heads,D], ``x`` the forward's input (None without a norm).
    The parameters' sums are taken in fp32 and in a fixed order."""
    if d_y.stride(-1) != 1:
        d_y = d_y.contiguous()
    rows = d_y if norm is None else x
    call = _Call(rows, None, positions, inv_freq, rope_start, interleaved, rope_scale, norm, None, weight if norm is not None else None,
                 bias if norm is not None else None, None, None, norm_dim, eps, others=((d_y, "d_y"),))
    _check_rows(d_y, "d_y")
    if d_y.shape != rows.shape or d_y.dtype != rows.dtype:
        raise ValueError(f"d_y {tuple(d_y.shape)} {d_y.dtype} does not fit x {tuple(rows.shape)} {rows.dtype}")
    call.require_cuda()
    dx = torch.empty(d_y.shape, dtype=d_y.dtype, device=d_y.device)
    d_weight = torch.empty_like(weight) if norm is not None and weight is not None and need_params[0] else None
    d_bias = torch.empty_like(bias) if norm is not None and bias is not None and need_params[1] else None
    if not dx.numel():
        for t in (d_weight, d_bias):
            if t is not None:
                t.zero_()
        return dx, d_weight, d_bias
    lib = _lib.load()
    with torch.cuda.device(call.dev):
        workspace, nbytes = None, 0
        if d_weight is not None or d_bias is not None:
            nbytes = int(lib.dsa_norm_rope_bwd_workspace_bytes(call.norm_dim))
            workspace = torch.empty((nbytes,), dtype=torch.uint8, device=call.dev)
        side = call.side(0, dx)
        _lib.check(lib.dsa_norm_rope_bwd(ctypes.byref(side), ptr(d_y), d_y.stride(0), d_y.stride(1), d_y.stride(2), *call.scalars(), ptr(d_weight),
                                         ptr(d_bias), ptr(workspace), nbytes, call.code, current_stream(call.dev)))
    return dx, d_weight, d_bias


def qk_norm_rope(q, k, positions, inv_freq, *, rope_start: int = 0, interleaved: bool = True, rope_scale: float = 1.0, q_norm=None, k_norm=None,
                 q_weight=None, q_bias=None, k_weight=None, k_bias=None, norm_dim: Optional[int] = None, eps: float = 1e-6):
    """Differentiable ``(q', k')``: every head's row normed over its leading ``norm_dim`` dims (default: all), then its dims
    ``[rope_start, rope_start + 2 * len(inv_freq))`` rotated by ``positions * inv_freq``.

    q [B,S,H,D] and k [B,S,Hk,D] bf16 / fp16 with unit inner stride (slices of a projection are read in place; either may be None);
    positions [B,S] int32 / int64, any value; inv_freq fp32, one frequency per rotated pair; pairs are (2i, 2i+1) when
    ``interleaved``, else (i, i + half).  ``q_norm`` / ``k_norm``: None, "rms" (x / sqrt(mean x^2 + eps)) or "layer"; weights and
    biases [norm_dim] (fp32 or the rows' type) are shared by the heads.  ``rope_scale`` multiplies cosines and sines.
    Everything is computed in fp32 (the angles in 64 bits) and rounded once.  Outputs are contiguous; gradients reach q, k,
    weights and biases."""
    return QkNormRopeFunction.apply(q, k, q_weight, q_bias, k_weight, k_bias, positions, inv_freq, int(rope_start), bool(interleaved), float(rope_scale),
                                    q_norm, k_norm, norm_dim, float(eps))


def qk_norm_rope_cached(q, k, positions, inv_freq, key_cache, slots, *, key_cache_rope=None, rope_start: int = 0, interleaved: bool = True,
                        rope_scale: float = 1.0, q_norm=None, k_norm=None, q_weight=None, q_bias=None, k_weight=None, k_bias=None,
                        norm_dim: Optional[int] = None, eps: float = 1e-6):
    """``qk_norm_rope`` of a serving step: the key rows go to rows ``slots`` of a paged cache; returns q' (None without q).

    key_cache [num_blocks, block_size, Hk, D], or with ``key_cache_rope`` [num_blocks, block_size, Hk, R] the dims before the
    rotated ones, [num_blocks, block_size, Hk, D - R] (then the rotated dims are the last R).  slots [B,S] int32 / int64: block *
    block_size + offset; a token whose slot lies outside the cache (-1: padding) writes nothing.  Two tokens of a call never
    share a slot.  One launch; no gradients (an input that asks for one is refused)."""
    inputs = [t for t in (q, k, q_weight, q_bias, k_weight, k_bias) if t is not None]
    if k is None:
        raise ValueError("k must be given")
    if torch.is_grad_enabled() and any(t.requires_grad for t in inputs):
        raise ValueError("qk_norm_rope_cached has no gradient; use qk_norm_rope, or call it under torch.no_grad()")
    caches = [(key_cache, "key_cache")] + ([] if key_cache_rope is None else [(key_cache_rope, "key_cache_rope")])
    for t, name in caches:
        if not isinstance(t, torch.Tensor) or t.dim() != 4 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous [num_blocks, block_size, heads, dims] tensor")
    call = _Call(q, k, positions, inv_freq, rope_start, interleaved, rope_scale, q_norm, k_norm, q_weight, q_bias, k_weight, k_bias, norm_dim, eps,
                 others=(*caches, (slots, "slots")))
    _token_numbers(slots, "slots", call.B, call.S)
    split = call.D if key_cache_rope is None else call.D - call.R
    if key_cache_rope is not None and (call.rope_start != split or split == 0):
        raise ValueError("a cache in two parts needs the rotated dims at the end of the row")
    for (t, name), dims in zip(caches, (split, call.R)):
        if t.dtype != k.dtype or t.shape[2] != k.shape[2] or t.shape[3] != dims or t.shape[:2] != key_cache.shape[:2]:
            raise ValueError(f"{name} {tuple(t.shape)} {t.dtype} does not fit keys {tuple(k.shape)} {k.dtype} of {dims} dims")
    call.require_cuda()
    out = _new_rows(q)
    if call.B * call.S and (k.shape[2] or (q is not None and q.shape[2])):
        q_side = None if q is None or not out.numel() else call.side(0, out)
        k_side = call.side(1, key_cache, key_cache_rope, split, slots, key_cache.shape[0] * key_cache.shape[1]) if key_cache.numel() else None
        if q_side is not None or k_side is not None:
            call.run(q_side, k_side)
    return out
