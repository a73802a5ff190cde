"""Attention over the atoms of a batch: the operators of an attention block as HIP kernels.

=========================  ========================================================
:func:`embedding`          rows of a table by index with a scale; the table's gradient
                           by sorted indices
:func:`head_norm_rotate`   norms of queries and keys for each head and their rotation
                           in the same pass
:func:`structure_attention`  softmax attention of every atom to the atoms of its
                           structure; the backward pass forms the probabilities again
:func:`dropout_add`        dropout from a counter-based generator, with a residual; the
                           mask is never stored
=========================  ========================================================

They take GPU tensors of float32, bfloat16 or float16 (arithmetic and sums in float32, every
output rounded once) and raise on any other; there is no fallback. They run on the
current stream without host reads (:func:`attention_plan` makes one), every sum has a fixed
order, and the kernels may be captured in a HIP graph. :func:`embedding` and :func:`dropout_add`
are differentiable to any order, the other two once. The per-edge reference path has no
counterpart.
"""
from __future__ import annotations

import ctypes
import functools
import math
from dataclasses import dataclass
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _lib

MAX_HEAD_DIM = 128


def _on_gpu(**tensors: Optional[Tensor]) -> torch.device:
    device = None
    for name, t in tensors.items():
        if t is None:
            continue
        if t.device.type != "cuda":
            raise RuntimeError("xnn_amd ops run on the GPU only (got a tensor on "
                               f"{t.device}); there is no CPU fallback")
        if device is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, not on {device}")
        device = t.device
    return device


_FUNCTIONS: dict = {}


def _call(name: str, *args) -> None:
    """:func:`xnn_amd._lib.call` without its lookups: at these operators' smallest sizes the host's
    microseconds are the time of a call."""
    if _lib.timed:
        return _lib.call(name, *args)
    fn = _FUNCTIONS.get(name)
    if fn is None:
        fn = _FUNCTIONS[name] = getattr(_lib.load(), name)
    _lib.calls[name] = _lib.calls.get(name, 0) + 1
    code = fn(*args)
    if code:
        _lib.check(name, code)


def _once_differentiable() -> None:
    if torch.is_grad_enabled():
        raise RuntimeError("the xnn_amd backward is differentiable once; double backward "
                           "(create_graph=True) needs the PyTorch form (use_fast=False)")


def _stream(t: Tensor) -> int:
    """The current stream of the tensor's device: the handle alone, without the object around it
    (2 us less a call)."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _wanted(*tensors: Optional[Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


@functools.lru_cache(maxsize=256)
def _work_bytes(name: str, *sizes: int) -> int:
    need = ctypes.c_size_t()
    _lib.check(name, getattr(_lib.load(), name)(*sizes, ctypes.byref(need)))
    return need.value


def _workspace(name: str, device: torch.device, *sizes: int) -> Tuple[Tensor, int]:
    need = _work_bytes(name, *sizes)
    return torch.empty(max(need, 1), dtype=torch.uint8, device=device), need


# --------------------------------------------------------------------------- embedding
def _embedding(ids: Tensor, table: Tensor, scale: float) -> Tensor:
    out = table.new_empty((*ids.shape, table.shape[1]))
    _call("xnn_embedding", _lib.storage_code(table.dtype), ids.data_ptr(), ids.numel(),
              table.data_ptr(), table.shape[0], table.shape[1], scale, out.data_ptr(),
              _stream(table))
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale):
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale = table.shape[0], scale
        return _embedding(ids, table, scale)

    @staticmethod
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        apply = _EmbeddingGrad.apply if torch.is_grad_enabled() else _embedding_grad
        return None, apply(ids, grad, ctx.rows, ctx.scale), None


def _embedding_grad(ids: Tensor, grad: Tensor, rows: int, scale: float) -> Tensor:
    grad = grad.contiguous()
    channels = grad.shape[-1]
    out = grad.new_empty((rows, channels))
    work, size = _workspace("xnn_embedding_grad_work_size", grad.device, ids.numel(), rows, channels)
    _call("xnn_embedding_grad", _lib.storage_code(grad.dtype), ids.data_ptr(), ids.numel(),
              grad.data_ptr(), rows, channels, scale, out.data_ptr(), work.data_ptr(), size,
              _stream(grad))
    return out


class _EmbeddingGrad(torch.autograd.Function):
    """The adjoint of :class:`_Embedding`, and the other way round."""

    @staticmethod
    def forward(ctx, ids, grad, rows, scale):
        ctx.save_for_backward(ids)
        ctx.scale = scale
        return _embedding_grad(ids, grad, rows, scale)

    @staticmethod
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        return None, _Embedding.apply(ids, grad.contiguous(), ctx.scale), None, None


def embedding(ids: Tensor, table: Tensor, scale: float = 1.0) -> Tensor:
    """``scale * table[ids]``, of shape ``ids.shape + (C,)``, for ``table`` (V, C).

    ``ids`` of any integer type; one outside the table gives a row of NaN and counts in no
    gradient. The gradient of the table sorts the ids and sums each row's tokens in their order
    (float32, rounded once), the same bits at every call."""
    device = table.get_device()
    if device < 0 or ids.get_device() != device:
        _on_gpu(table=table, ids=ids)
    if table.dim() != 2:
        raise ValueError(f"table must be (rows, channels), got {tuple(table.shape)}")
    if ids.dtype.is_floating_point or ids.dtype == torch.bool or ids.dtype.is_complex:
        raise TypeError(f"ids must be integers, got {ids.dtype}")
    _lib.storage_code(table.dtype)
    ids = ids.to(torch.int64).contiguous()
    table = table.contiguous()
    if _wanted(table):
        return _Embedding.apply(ids, table, float(scale))
    return _embedding(ids, table, float(scale))


# --------------------------------------------------------------------------- dropout
def _dropout(x, residual, drop, seed, offset, counter):
    out = torch.empty_like(x)
    _call("xnn_dropout_add", _lib.storage_code(x.dtype), x.data_ptr(),
              None if residual is None else residual.data_ptr(), x.numel(), drop, seed, offset,
              None if counter is None else counter.data_ptr(), out.data_ptr(),
              _stream(x))
    return out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, drop, seed, offset, counter):
        ctx.args = (drop, seed, offset)
        ctx.save_for_backward(counter)
        return _dropout(x, residual, drop, seed, offset, counter)

    @staticmethod
    def backward(ctx, grad):
        (counter,) = ctx.saved_tensors
        need = ctx.needs_input_grad
        apply = _Dropout.apply if torch.is_grad_enabled() else _dropout
        dx = apply(grad.contiguous(), None, *ctx.args, counter) if need[0] else None
        return dx, grad if need[1] else None, None, None, None, None


def dropout_add(x: Tensor, residual: Optional[Tensor], p: float, seed: int,
                offset=0) -> Tensor:
    """``residual + keep * x / (1 - p)`` in ``x``'s dtype (``residual`` None: without it).

    Element ``e`` of ``x`` (in index order) is kept when its 16-bit draw is at least
    ``round(65536 p)``: half word ``e % 8`` of the Philox4x32-10 block with counter ``(e // 8,
    offset)`` and key ``seed``. The factor is that of the rounded probability, so the mean is
    kept exactly. The same ``(seed, offset)`` gives the same mask; the backward pass draws it
    again. ``seed`` is an integer, ``offset`` an integer or, for a captured graph that advances
    it between replays, an int64 tensor of one element on the device (the backward pass reads it
    again: change it after that)."""
    device = x.get_device()
    if device < 0 or (residual is not None and residual.get_device() != device):
        _on_gpu(x=x, residual=residual)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be in [0, 1], got {p}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual {tuple(residual.shape)} {residual.dtype} does not match x "
                         f"{tuple(x.shape)} {x.dtype}")
    counter = None
    if isinstance(offset, Tensor):
        if offset.dtype != torch.int64 or offset.numel() != 1:
            raise ValueError("an offset tensor holds one int64")
        _on_gpu(x=x, offset=offset)
        counter, offset = offset, 0
    mask64 = (1 << 64) - 1
    drop, seed, offset = int(round(p * 65536)), int(seed) & mask64, int(offset) & mask64
    _lib.storage_code(x.dtype)
    x = x.contiguous()
    residual = None if residual is None else residual.contiguous()
    if _wanted(x, residual):
        return _Dropout.apply(x, residual, drop, seed, offset, counter)
    return _dropout(x, residual, drop, seed, offset, counter)


# --------------------------------------------------------------------------- norm and rotation
def _heads_of(t: Tensor) -> "_lib.Heads":
    return _lib.Heads(t.data_ptr(), t.stride(0), t.stride(1), t.shape[1])


def _unit_stride(t: Tensor) -> Tensor:
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _norm_args(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
    return (_lib.storage_code(q.dtype), ctypes.byref(_heads_of(q)), ctypes.byref(_heads_of(k)),
            q.shape[0], q.shape[2], 2 * cos.shape[1], q_weight.data_ptr(), k_weight.data_ptr(),
            cos.data_ptr(), sin.data_ptr(), cos.shape[0],
            None if positions is None else positions.data_ptr(), eps, int(interleaved))


def _norm_rotate(q, k, args):
    q_out, k_out = q.new_empty(q.shape), k.new_empty(k.shape)
    _call("xnn_head_norm_rotate", *args, q_out.data_ptr(), k_out.data_ptr(), _stream(q))
    return q_out, k_out


class _NormRotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.args = (eps, interleaved)
        return _norm_rotate(q, k, _norm_args(q, k, q_weight, k_weight, cos, sin, positions, eps,
                                             interleaved))

    @staticmethod
    def backward(ctx, grad_q, grad_k):
        _once_differentiable()
        saved = ctx.saved_tensors
        q, k, q_weight, k_weight, cos, sin, _ = saved
        need = ctx.needs_input_grad
        weights, tables = need[2] or need[3], need[4] or need[5]
        d_q, d_k = q.new_empty(q.shape), k.new_empty(k.shape)
        d_qw = d_kw = d_cos = d_sin = work = None
        size = 0
        if weights:
            d_qw, d_kw = torch.empty_like(q_weight), torch.empty_like(k_weight)
            work, size = _workspace("xnn_head_norm_rotate_backward_work_size", q.device, q.shape[2])
        if tables:
            d_cos, d_sin = torch.empty_like(cos), torch.empty_like(sin)
        grad_q, grad_k = grad_q.contiguous(), grad_k.contiguous()
        _call("xnn_head_norm_rotate_backward", *_norm_args(*saved, *ctx.args),
                  grad_q.data_ptr(), grad_k.data_ptr(), d_q.data_ptr(), d_k.data_ptr(),
                  *(_lib.ptr(t) for t in (d_qw, d_kw, d_cos, d_sin, work)), size,
                  _stream(q))
        grads = (d_q, d_k, d_qw, d_kw, d_cos, d_sin)
        return (*(g if n else None for g, n in zip(grads, need)), None, None, None)


def head_norm_rotate(q: Tensor, k: Tensor, q_weight: Tensor, k_weight: Tensor, cos: Tensor,
                     sin: Tensor, positions: Optional[Tensor] = None, eps: float = 1e-6,
                     interleaved: bool = False) -> Tuple[Tensor, Tensor]:
    """Queries ``q`` (T, H, D) and keys ``k`` (T, K, D), each head divided by its root mean square
    (``sqrt(mean x^2 + eps)``), times ``q_weight`` / ``k_weight`` (D,), its first ``R`` elements
    rotated: pairs ``(i, i + R/2)``, or ``(2 i, 2 i + 1)`` when ``interleaved``, by the angle with
    cosine ``cos`` and sine ``sin`` (rows, R/2; float32).

    Token ``t`` takes row ``positions[t]`` of the tables (one outside gives NaN), or row ``t`` when
    ``positions`` is None; only then do the tables have gradients (phases that depend on the
    geometry lead to forces). Tokens and heads may be strided (views of one projection's output)."""
    device = q.get_device()
    if device < 0 or not (device == k.get_device() == q_weight.get_device() == k_weight.get_device()
                          == cos.get_device() == sin.get_device()) \
            or (positions is not None and positions.get_device() != device):
        _on_gpu(q=q, k=k, q_weight=q_weight, k_weight=k_weight, cos=cos, sin=sin, positions=positions)
    if q.dim() != 3 or k.dim() != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError("q and k must be (tokens, heads, head_dim) of the same tokens and head_dim, "
                         f"got {tuple(q.shape)} and {tuple(k.shape)}")
    T, D = q.shape[0], q.shape[2]
    if not 1 <= D <= MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be in [1, {MAX_HEAD_DIM}], got {D}")
    if q.shape[1] < 1 or k.shape[1] < 1:
        raise ValueError("no heads")
    if not q.dtype == k.dtype == q_weight.dtype == k_weight.dtype:
        raise TypeError(f"q, k and their weights must have one dtype, got {q.dtype}, {k.dtype}, "
                        f"{q_weight.dtype} and {k_weight.dtype}")
    if q_weight.shape != (D,) or k_weight.shape != (D,):
        raise ValueError(f"the weights must be ({D},)")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise TypeError("cos and sin must be float32")
    if cos.dim() != 2 or cos.shape != sin.shape or 2 * cos.shape[1] > D:
        raise ValueError(f"cos and sin must be (rows, R / 2) with R <= {D}, got {tuple(cos.shape)} "
                         f"and {tuple(sin.shape)}")
    if positions is None:
        if cos.shape[0] != T:
            raise ValueError(f"without positions the tables have a row a token: {cos.shape[0]} "
                             f"rows, {T} tokens")
    else:
        if positions.shape != (T,) or positions.dtype.is_floating_point \
                or positions.dtype == torch.bool:
            raise ValueError(f"positions must be ({T},) integers")
        if _wanted(cos, sin):
            raise ValueError("tables read by position have no gradient here (gather their rows "
                             "and leave positions out)")
        positions = positions.to(torch.int64).contiguous()
    args = (_unit_stride(q), _unit_stride(k), q_weight.contiguous(), k_weight.contiguous(),
            cos.contiguous(), sin.contiguous(), positions, float(eps), bool(interleaved))
    if _wanted(*args[:6]):
        return _NormRotate.apply(*args)
    return _norm_rotate(args[0], args[1], _norm_args(*args))


# --------------------------------------------------------------------------- attention
@dataclass
class AttentionPlan:
    """The row tiles of a batch of structures (:func:`attention_plan`)."""
    n_tokens: int
    n_structures: int
    max_atoms: int
    tiles32: Tensor                  # (tiles, 3) int32: first row, end and begin of its structure
    tiles128: Tensor
    ptr: Tensor                      # (B + 1,) int64

    def __post_init__(self):
        self.c = _lib.AttentionTiles(self.n_tokens, self.max_atoms, self.tiles32.shape[0],
                                     self.tiles128.shape[0], self.tiles32.data_ptr(),
                                     self.tiles128.data_ptr())
        self._bytes = {}

    def work_bytes(self, name: str, *sizes: int) -> int:
        """Bytes of a workspace for this plan: a function of the sizes alone."""
        need = self._bytes.get((name, sizes))
        if need is None:
            c = ctypes.c_size_t()
            _lib.check(name, getattr(_lib.load(), name)(self.n_tokens, *sizes, ctypes.byref(self.c),
                                                        ctypes.byref(c)))
            need = self._bytes[name, sizes] = c.value
        return need


def attention_plan(n_atoms: Tensor, n_tokens: Optional[int] = None) -> AttentionPlan:
    """The plan of structures with ``n_atoms`` (B,) consecutive atoms each (a graph's
    ``n_atoms``), kept as long as the batch: two launches and one host read (of the checks and
    sizes). ``n_tokens``: the atoms of the batch, read from the sum where it is not given.

    Raises ``ValueError`` for negative counts or counts that do not sum to ``n_tokens``."""
    device = _on_gpu(n_atoms=n_atoms)
    if n_atoms.dim() != 1 or n_atoms.dtype.is_floating_point or n_atoms.dtype == torch.bool:
        raise ValueError(f"n_atoms must be (B,) integers, got {tuple(n_atoms.shape)} {n_atoms.dtype}")
    n_atoms = n_atoms.to(torch.int64).contiguous()
    n_tokens = int(n_atoms.sum()) if n_tokens is None else int(n_tokens)
    if n_tokens < 0:
        raise ValueError(f"negative number of atoms ({n_tokens})")
    B = n_atoms.shape[0]
    caps = [n_tokens // 32 + B, n_tokens // 128 + B]
    ints = torch.empty(3 * sum(caps), dtype=torch.int32, device=device)
    longs = torch.empty(4 * B + 8, dtype=torch.int64, device=device)
    ptr, tile_ptr, order, info = longs.split([B + 1, 2 * (B + 1), B, 5])
    lists = ints.split([3 * c for c in caps])
    _call("xnn_attention_plan", n_atoms.data_ptr(), B, n_tokens, ptr.data_ptr(),
              tile_ptr.data_ptr(), order.data_ptr(), lists[0].data_ptr(), caps[0], lists[1].data_ptr(), caps[1],
              info.data_ptr(), _stream(n_atoms))
    n32, n128, longest, status, total = info.tolist()
    if status == 1:
        raise ValueError(f"n_atoms holds a count outside [0, {n_tokens}]")
    if status == 2:
        raise ValueError(f"n_atoms sums to {total}, the batch has {n_tokens} atoms")
    return AttentionPlan(n_tokens, B, longest, lists[0][:3 * n32].view(-1, 3),
                         lists[1][:3 * n128].view(-1, 3), ptr)


def _attention_args(q, k, v, plan, mask, scale):
    return (_lib.storage_code(q.dtype), ctypes.byref(_heads_of(q)), ctypes.byref(_heads_of(k)),
            ctypes.byref(_heads_of(v)), q.shape[0], q.shape[2], ctypes.byref(plan.c),
            None if mask is None else mask.data_ptr(), scale)


def _attention(q, plan, args, want_lse):
    out = q.new_empty(q.shape)
    size = plan.work_bytes("xnn_attention_work_size", q.shape[1], q.shape[2])
    work = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
    lse = torch.empty(q.shape[1], q.shape[0], dtype=torch.float32, device=q.device) if want_lse else None
    _call("xnn_attention", *args, out.data_ptr(), _lib.ptr(lse),
              _lib.ptr(work), size, _stream(q))
    return out, lse


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, plan, mask, scale):
        ctx.plan, ctx.scale = plan, scale
        out, lse = _attention(q, plan, _attention_args(q, k, v, plan, mask, scale), True)
        ctx.save_for_backward(q, k, v, mask, out, lse)
        return out

    @staticmethod
    def backward(ctx, grad):
        _once_differentiable()
        q, k, v, mask, out, lse = ctx.saved_tensors
        grad = grad.contiguous()
        dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
        size = ctx.plan.work_bytes("xnn_attention_backward_work_size", q.shape[1], k.shape[1], q.shape[2])
        work = torch.empty(size, dtype=torch.uint8, device=q.device)
        _call("xnn_attention_backward", *_attention_args(q, k, v, ctx.plan, mask, ctx.scale),
                  out.data_ptr(), lse.data_ptr(), grad.data_ptr(), dq.data_ptr(), dk.data_ptr(),
                  dv.data_ptr(), work.data_ptr(), size, _stream(q))
        need = ctx.needs_input_grad
        return (*(g if n else None for g, n in zip((dq, dk, dv), need)), None, None, None)


def structure_attention(q: Tensor, k: Tensor, v: Tensor, plan: AttentionPlan,
                        mask: Optional[Tensor] = None, scale: Optional[float] = None) -> Tensor:
    """``softmax(scale q k^T) v`` of every atom over the atoms of its structure.

    ``q`` (T, H, D); ``k`` and ``v`` (T, K, D) with ``H`` a multiple of ``K`` (query heads ``h`` read
    head ``h // (H / K)``); ``D <= 128``; tokens and heads may be strided (views of one projection's
    output). ``plan`` from :func:`attention_plan`. ``mask`` (T,), bool: atoms that may be attended
    to (None: all); an atom that is masked out reaches no other, whatever its values, and gets zero
    key and value gradients; atoms with nothing to attend to get zeros. ``scale``: ``D ** -0.5``
    by default, positive. Returns (T, H, D). Neither scores nor probabilities are stored; the backward
    pass forms them again from the rows' log-sums."""
    device = q.get_device()
    if device < 0 or not device == k.get_device() == v.get_device() == plan.ptr.get_device() \
            or (mask is not None and mask.get_device() != device):
        _on_gpu(q=q, k=k, v=v, mask=mask, plan=plan.ptr)
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or q.shape[0] != k.shape[0] \
            or q.shape[2] != k.shape[2]:
        raise ValueError("q must be (tokens, heads, head_dim), k and v (tokens, kv_heads, head_dim), "
                         f"got {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    T, H, D = q.shape
    if not 1 <= D <= MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be in [1, {MAX_HEAD_DIM}], got {D}")
    if k.shape[1] < 1 or H < 1 or H % k.shape[1] != 0:
        raise ValueError(f"{H} heads cannot share {k.shape[1]} heads of keys and values")
    if not q.dtype == k.dtype == v.dtype:
        raise TypeError(f"q, k and v must have one dtype, got {q.dtype}, {k.dtype} and {v.dtype}")
    if plan.n_tokens != T:
        raise ValueError(f"the plan is of {plan.n_tokens} tokens, q holds {T}")
    if mask is not None:
        if mask.shape != (T,) or mask.dtype != torch.bool:
            raise ValueError(f"mask must be ({T},) bool, got {tuple(mask.shape)} {mask.dtype}")
        mask = mask.contiguous()
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    _lib.storage_code(q.dtype)
    q, k, v = _unit_stride(q), _unit_stride(k), _unit_stride(v)
    if _wanted(q, k, v):
        return _Attention.apply(q, k, v, plan, mask, scale)
    return _attention(q, plan, _attention_args(q, k, v, plan, mask, scale), False)[0]
