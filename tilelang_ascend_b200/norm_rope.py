"""Norm of every head's query and key rows and rotation by their tokens' positions, in one pass.

The attention and indexer entry points of this package take rotated queries and keys, and their decode forms read them from
paged caches; these calls make both (no reference counterpart: its examples start from rotated tensors):

* ``qk_norm_rope``         differentiable, returns the rows as new tensors (prefill, training)
* ``qk_norm_rope_cached``  writes the key rows straight into a paged cache, kept in one part ([num_blocks, block_size, heads, D]) or
                           in two (``key_cache_rope``: the rotated tail apart, as the MLA decode entry points read it)
"""
from __future__ import annotations

from ctypes import byref
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .adapter import dtype_code, on_device, ptr, raw_stream

NORMS = {None: 0, "rms": 1, "layer": 2}


def _check_rows(x, name: str) -> None:
    if not isinstance(x, torch.Tensor):
        raise ValueError(f"{name}: expected a torch.Tensor, got {type(x).__name__}")
    if x.dim() != 4:
        raise ValueError(f"{name} must be [B, S, heads, D], got {tuple(x.shape)}")
    if x.stride(3) != 1 and x.shape[3] > 1 and x.numel():
        raise ValueError(f"Input tensor {name} must have unit inner stride")


def _check_vector(t, name: str, n: int, dtypes) -> None:
    if t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector of {n} values, got {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"Input tensor {name} has dtype {t.dtype}, expected one of {', '.join(str(d) for d in dtypes)}")


def _token_numbers(t, name: str, B: int, S: int) -> int:
    """1 for int64, 0 for int32."""
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be an int32 or int64 tensor")
    if t.shape != (B, S) or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous [{B}, {S}], got {tuple(t.shape)}")
    return int(t.dtype == torch.int64)


class _Call:
    """Checked arguments of a call, without its outputs."""

    def __init__(self, rows, positions, inv_freq, rope_start, interleaved, rope_scale, norms, params, norm_dim, eps, others=()):
        first = rows[0] if rows[0] is not None else rows[1]
        if first is None:
            raise ValueError("queries or keys must be given")
        for x, name in zip(rows, ("q", "k")):
            if x is not None:
                _check_rows(x, name)
        q, k = rows
        if q is not None and k is not None and (q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3] or q.dtype != k.dtype):
            raise ValueError(f"q and k must agree in B, S, D and dtype (got {tuple(q.shape)} {q.dtype}, {tuple(k.shape)} {k.dtype})")
        B, S, _, D = first.shape
        code, dev = dtype_code(first.dtype), first.device
        positions64 = _token_numbers(positions, "positions", B, S)
        if not isinstance(inv_freq, torch.Tensor) or inv_freq.dim() != 1:
            raise ValueError("inv_freq must be a vector with one frequency per rotated pair")
        _check_vector(inv_freq, "inv_freq", inv_freq.shape[0], (torch.float32,))
        R, rope_start = 2 * inv_freq.shape[0], int(rope_start)
        if R < 2 or rope_start < 0 or rope_start + R > D:
            raise ValueError(f"the rotated dims [{rope_start}, {rope_start + R}) must lie inside rows of {D}")
        norm_dim = D if norm_dim is None else int(norm_dim)
        if not 1 <= norm_dim <= D:
            raise ValueError(f"norm_dim must be in [1, {D}], got {norm_dim}")
        for side, x, norm, (weight, bias) in zip(("q", "k"), rows, norms, params):
            if norm not in NORMS:
                raise ValueError(f"{side}_norm must be None, 'rms' or 'layer', got {norm!r}")
            for t, what in ((weight, "weight"), (bias, "bias")):
                if t is not None:
                    if norm is None or x is None:
                        raise ValueError(f"{side}_{what} needs {side} and its norm")
                    _check_vector(t, f"{side}_{what}", norm_dim, (torch.float32, first.dtype))
                    if t.device != dev:
                        raise ValueError(f"Input tensor {side}_{what} is on {t.device}, expected {dev}")
            if weight is not None and bias is not None and weight.dtype != bias.dtype:
                raise ValueError(f"{side}_weight and {side}_bias must have one dtype")
        for t, name in ((q, "q"), (k, "k"), (positions, "positions"), (inv_freq, "inv_freq"), *others):
            if t is not None and t.device != dev:
                raise ValueError(f"Input tensor {name} is on {t.device}, expected {dev}")
        self.B, self.S, self.D, self.R, self.rope_start, self.norm_dim = B, S, D, R, rope_start, norm_dim
        self.code, self.dev, self.positions64 = code, dev, positions64
        self.norms = norms
        self.rest = (B, S, D, R, rope_start, norm_dim, 1 if interleaved else 0, float(rope_scale), float(eps))

    def require_cuda(self) -> None:
        if self.dev.type != "cuda":
            raise ValueError(f"kernels run on CUDA tensors only (got device {self.dev}); there is no CPU path")

    def scalars(self, positions, inv_freq):
        return (positions.data_ptr(), self.positions64, inv_freq.data_ptr(), *self.rest)

    def side(self, i: int, x, heads: int, params, out, tail=None, split: Optional[int] = None, slots=None, y_slots: int = 0):
        """The C struct of queries (0) or keys (1): rows x (None: not read) to ``out``."""
        weight, bias = params
        param = weight if weight is not None else bias
        sb, ss, sh = (0, 0, 0) if x is None else x.stride()[:3]
        return _lib.RopeRows(ptr(x), sb, ss, sh, heads, NORMS[self.norms[i]], ptr(weight), ptr(bias),
                             0 if param is None else int(param.dtype == torch.float32), self.D if split is None else split, out.data_ptr(), ptr(tail),
                             ptr(slots), y_slots, 0 if slots is None else int(slots.dtype == torch.int64), 0)

    def run(self, q_side, k_side, positions, inv_freq) -> None:
        with on_device(self.dev):
            _lib.check(_lib.load().dsa_norm_rope(None if q_side is None else byref(q_side), None if k_side is None else byref(k_side),
                                                 *self.scalars(positions, inv_freq), self.code, raw_stream(self.dev)))


def _new_rows(x):
    return None if x is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _backward(call: _Call, d_outs, rows, params, positions, inv_freq, need_rows, need_params):
    """([dq, dk], [(dweight, dbias) of q, of k]) of a checked call; None where nothing is asked for."""
    d_rows, d_params, sides = [None, None], [[None, None], [None, None]], [None, None]
    lines, empty = 0, call.B * call.S == 0
    for i in range(2):
        d_y, norm = d_outs[i], call.norms[i]
        wanted = [t is not None and need for t, need in zip(params[i], need_params[i])]
        if d_y is None or not (need_rows[i] or wanted[0] or wanted[1]):
            continue
        d_rows[i] = torch.empty(d_y.shape, dtype=d_y.dtype, device=call.dev)
        d_params[i] = [torch.empty_like(t) if w else None for t, w in zip(params[i], wanted)]
        if empty or not d_y.numel():
            for t in d_params[i]:
                if t is not None:
                    t.zero_()
            continue
        if d_y.stride(3) != 1 and call.D > 1:
            d_y = d_y.contiguous()
        x = None if norm is None else rows[i]
        sb, ss, sh, _ = d_y.stride()
        sides[i] = (_lib.RopeGrads(call.side(i, x, d_y.shape[2], params[i], d_rows[i]), d_y.data_ptr(), sb, ss, sh, ptr(d_params[i][0]), ptr(d_params[i][1])), d_y)
        lines += wanted[0] or wanted[1]
    if sides[0] is not None or sides[1] is not None:
        lib = _lib.load()
        with on_device(call.dev):
            workspace, nbytes = None, 0
            if lines:
                nbytes = lines * int(lib.dsa_norm_rope_bwd_workspace_bytes(call.norm_dim))
                workspace = torch.empty((nbytes,), dtype=torch.uint8, device=call.dev)
            _lib.check(lib.dsa_norm_rope_bwd(None if sides[0] is None else byref(sides[0][0]), None if sides[1] is None else byref(sides[1][0]),
                                             *call.scalars(positions, inv_freq), ptr(workspace), nbytes, call.code, raw_stream(call.dev)))
    return d_rows, d_params


class QkNormRopeFunction(torch.autograd.Function):
    """Autograd node over the forward / backward kernels."""

    @staticmethod
    def forward(ctx, q, k, q_weight, q_bias, k_weight, k_bias, positions, inv_freq, rope_start, interleaved, rope_scale, q_norm, k_norm, norm_dim, eps):
        params = ((q_weight, q_bias), (k_weight, k_bias))
        call = _Call((q, k), positions, inv_freq, rope_start, interleaved, rope_scale, (q_norm, k_norm), params, norm_dim, eps)
        call.require_cuda()
        outs = _new_rows(q), _new_rows(k)
        sides = [None if o is None or not o.numel() else call.side(i, x, x.shape[2], params[i], o) for i, (x, o) in enumerate(zip((q, k), outs))]
        if sides[0] is not None or sides[1] is not None:
            call.run(*sides, positions, inv_freq)
        # (rows without a norm are not needed again: their gradient is the rotation of the outputs')
        ctx.save_for_backward(None if q_norm is None else q, None if k_norm is None else k, q_weight, q_bias, k_weight, k_bias, positions, inv_freq)
        ctx.call = call
        ctx.set_materialize_grads(False)
        return outs

    @staticmethod
    @once_differentiable
    def backward(ctx, d_q, d_k):
        q, k, q_weight, q_bias, k_weight, k_bias, positions, inv_freq = ctx.saved_tensors
        need = ctx.needs_input_grad
        (dq, dk), ((dqw, dqb), (dkw, dkb)) = _backward(ctx.call, (d_q, d_k), (q, k), ((q_weight, q_bias), (k_weight, k_bias)), positions, inv_freq, need[:2],
                                                       (need[2:4], need[4:6]))
        return dq, dk, dqw, dqb, dkw, dkb, None, None, None, None, None, None, None, None, None


def qk_norm_rope_bwd_raw(d_q, d_k, q, k, positions, inv_freq, *, rope_start: int = 0, interleaved: bool = True, rope_scale: float = 1.0, q_norm=None,
                         k_norm=None, q_weight=None, q_bias=None, k_weight=None, k_bias=None, norm_dim: Optional[int] = None, eps: float = 1e-6):
    """(dq, dk, dq_weight, dq_bias, dk_weight, dk_bias) of :func:`qk_norm_rope` for the gradients ``d_q`` / ``d_k`` of its outputs (either may be
    None); ``q`` / ``k`` are the forward's inputs, looked at on sides with a norm only.  None where there is nothing to derive.  The
    parameters' sums are taken in fp32 and in a fixed order."""
    for d_y, x, norm, name in ((d_q, q, q_norm, "d_q"), (d_k, k, k_norm, "d_k")):
        if d_y is not None:
            _check_rows(d_y, name)
            if norm is not None and (x is None or d_y.shape != x.shape or d_y.dtype != x.dtype):
                raise ValueError(f"{name} {tuple(d_y.shape)} {d_y.dtype} does not fit the forward's input")
    rows = tuple(None if d_y is None else (d_y if norm is None else x) for d_y, x, norm in ((d_q, q, q_norm), (d_k, k, k_norm)))
    params = tuple((None, None) if d_y is None else pair for d_y, pair in ((d_q, (q_weight, q_bias)), (d_k, (k_weight, k_bias))))
    call = _Call(rows, positions, inv_freq, rope_start, interleaved, rope_scale, (q_norm, k_norm), params, norm_dim, eps, others=((d_q, "d_q"), (d_k, "d_k")))
    call.require_cuda()
    (dq, dk), (dqp, dkp) = _backward(call, (d_q, d_k), rows, params, positions, inv_freq, (True, True), ((True, True), (True, True)))
    return dq, dk, dqp[0], dqp[1], dkp[0], dkp[1]


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
    return QkNormRopeFunction.apply(q, k, q_weight, q_bias, k_weight, k_bias, positions, inv_freq, rope_start, interleaved, rope_scale, q_norm, k_norm,
                                    norm_dim, eps)


def qk_norm_rope_cached(q, k, positions, inv_freq, key_cache, slots, *, key_cache_rope=None, rope_start: int = 0, interleaved: bool = True,
                        rope_scale: float = 1.0, q_norm=None, k_norm=None, q_weight=None, q_bias=None, k_weight=None, k_bias=None,
                        norm_dim: Optional[int] = None, eps: float = 1e-6):
    """``qk_norm_rope`` of a serving step: the key rows go to rows ``slots`` of a paged cache; returns q' (None without q).

    key_cache [num_blocks, block_size, Hk, D], or with ``key_cache_rope`` [num_blocks, block_size, Hk, R] the dims before the
    rotated ones, [num_blocks, block_size, Hk, D - R] (then the rotated dims are the last R).  slots [B,S] int32 / int64: block *
    block_size + offset; a token whose slot lies outside the cache (-1: padding) writes nothing.  Two tokens of a call never
    share a slot, and q and k are no part of the cache.  One launch; no gradients (an input that asks for one is refused)."""
    if k is None:
        raise ValueError("k must be given")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, q_bias, k_weight, k_bias)):
        raise ValueError("qk_norm_rope_cached has no gradient; use qk_norm_rope, or call it under torch.no_grad()")
    if not isinstance(slots, torch.Tensor):
        raise ValueError("slots must be an int32 or int64 tensor")
    caches = ((key_cache, "key_cache"),) if key_cache_rope is None else ((key_cache, "key_cache"), (key_cache_rope, "key_cache_rope"))
    for t, name in caches:
        if not isinstance(t, torch.Tensor) or t.dim() != 4 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous [num_blocks, block_size, heads, dims] tensor")
    params = ((q_weight, q_bias), (k_weight, k_bias))
    call = _Call((q, k), positions, inv_freq, rope_start, interleaved, rope_scale, (q_norm, k_norm), params, norm_dim, eps, others=(*caches, (slots, "slots")))
    _token_numbers(slots, "slots", call.B, call.S)
    split = call.D if key_cache_rope is None else call.D - call.R
    if key_cache_rope is not None and (call.rope_start != split or split == 0):
        raise ValueError("a cache in two parts needs the rotated dims at the end of the row")
    num_blocks, block_size = key_cache.shape[:2]
    for (t, name), dims in zip(caches, (split, call.R)):
        if t.dtype != k.dtype or t.shape != (num_blocks, block_size, k.shape[2], dims):
            raise ValueError(f"{name} {tuple(t.shape)} {t.dtype} does not fit keys {tuple(k.shape)} {k.dtype} of {dims} dims")
    call.require_cuda()
    out = _new_rows(q)
    q_side = None if out is None or not out.numel() else call.side(0, q, q.shape[2], params[0], out)
    k_side = call.side(1, k, k.shape[2], params[1], key_cache, key_cache_rope, split, slots, num_blocks * block_size) if k.numel() and key_cache.numel() else None
    if q_side is not None or k_side is not None:
        call.run(q_side, k_side, positions, inv_freq)
    return out
