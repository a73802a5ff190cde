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
order, and the kernels may be captured in a HIP graph. Checks, autograd and launches are native code
(``csrc/attention_ops.cpp``), registered as operators (``torch.ops.xnn_amd``) with a form for shapes
alone, so that tracers, fake tensors and compilers record them. They have no forward-mode derivative and
no batching rule (``vmap``), and raise there. :func:`embedding` and :func:`dropout_add`
are differentiable to any order, the other two once. The per-edge reference path has no
counterpart.
"""
from __future__ import annotations

import os
from dataclasses import dataclass
from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.compiler import is_compiling

from . import _lib
from .plan import capturing, hold_captured

_native, _failure = None, None
try:
    # registers the operators (torch.ops.xnn_amd) with their shapes and derivatives
    from . import _attention_ops as _built
    _built.set_library(os.path.abspath(_lib.LIBRARY))
    _lib.calls.join(_built.entries(), _built.calls)
except (ImportError, AttributeError) as err:     # not built, or from other sources: the first call says so
    _built, _failure = None, err


def _ops():
    """The native operators, checked on first use (raises when they are not built)."""
    global _native
    if _native is None:
        _lib.load()
        if _built is None:
            raise RuntimeError("xnn_amd/_attention_ops.so is missing, old or does not load: build it with "
                               "`python -m xnn_amd.build` (the kernels have no fallback)") from _failure
        _native = _built
    return _native


_U64 = (1 << 64) - 1


def _signed(x: int) -> int:
    """The low 64 bits of ``x`` as a signed integer."""
    x = int(x) & _U64
    return x - (1 << 64) if x >> 63 else x


def embedding(ids: Tensor, table: Tensor, scale: float = 1.0) -> Tensor:
    """``scale * table[ids]``, of shape ``ids.shape + (C,)``, for ``table`` (V, C).

    ``ids`` of any integer type; one outside the table gives a row of NaN and counts in no
    gradient. The gradient of the table sorts the ids and sums each row's tokens in their order
    (float32, rounded once), the same bits at every call."""
    if is_compiling():               # a compiler cannot look into the native entry: the same operator by name
        return torch.ops.xnn_amd.embedding_rows(ids, table, scale)
    return (_native or _ops()).embedding(ids, table, scale)


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
    counter = None
    if isinstance(offset, Tensor):
        counter, offset = offset, 0
    if is_compiling():
        return torch.ops.xnn_amd.dropout_add(x, residual, p, _signed(seed), _signed(offset), counter)
    return (_native or _ops()).dropout_add(x, residual, p, int(seed) & _U64, int(offset) & _U64, counter)


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
    if is_compiling():
        return torch.ops.xnn_amd.head_norm_rotate(q, k, q_weight, k_weight, cos, sin, positions, eps,
                                                  interleaved)
    return (_native or _ops()).head_norm_rotate(q, k, q_weight, k_weight, cos, sin, positions, eps,
                                                interleaved)


@dataclass
class AttentionPlan:
    """The row tiles of a batch of structures (:func:`attention_plan`)."""
    n_tokens: int
    n_structures: int
    max_atoms: int
    tiles32: Tensor                  # (tiles, 3) int32: first row, end and begin of its structure
    tiles128: Tensor
    ptr: Tensor                      # (B + 1,) int64: where each structure's atoms begin

    def __post_init__(self):
        self.native = _ops().Plan(self.n_tokens, self.max_atoms, self.tiles32, self.tiles128)

    # a graph that keeps its plan is copied and pickled with it
    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k != "native"}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self.__post_init__()


def attention_plan(n_atoms: Tensor, n_tokens: Optional[int] = None) -> AttentionPlan:
    """The plan of structures with ``n_atoms`` (B,) consecutive atoms each, kept as long as the
    batch (:meth:`~xnn_amd.data.AtomicGraph.attention_plan` keeps it with the graph): two launches and
    one host read, of the checks and sizes. ``n_tokens``: the atoms of the batch; where it is not
    given their sum is read as well.

    Raises ``ValueError`` for negative counts or counts that do not sum to ``n_tokens``."""
    device = n_atoms.device
    if device.type != "cuda":
        raise RuntimeError(f"xnn_amd ops run on the GPU only (got a tensor on {device}); there is no "
                           "CPU fallback")
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
    with torch.cuda.device(device):
        _lib.call("xnn_attention_plan", n_atoms.data_ptr(), B, n_tokens, ptr.data_ptr(),
                  tile_ptr.data_ptr(), order.data_ptr(), lists[0].data_ptr(), caps[0],
                  lists[1].data_ptr(), caps[1], info.data_ptr(), _lib.stream(device))
    n32, n128, longest, status, total = info.tolist()
    if status == 1:
        raise ValueError(f"n_atoms holds a count outside [0, {n_tokens}]")
    if status == 2:
        raise ValueError(f"n_atoms sums to {total}, the batch has {n_tokens} atoms")
    return AttentionPlan(n_tokens, B, longest, lists[0][:3 * n32].view(-1, 3),
                         lists[1][:3 * n128].view(-1, 3), ptr)


def plan_for(graph) -> AttentionPlan:
    """The cached plan of an :class:`~xnn_amd.data.AtomicGraph` (made again when ``n_atoms`` is another tensor
    or was written to, or the number of atoms changes). One that a capture takes stays as long as ``n_atoms``."""
    n_atoms = graph.n_atoms
    version = None if n_atoms.is_inference() else n_atoms._version
    key = (version, graph.num_nodes)
    cached = getattr(graph, "_xnn_attention_plan", None)
    if cached is not None and cached[0] is n_atoms and cached[1] == key:
        if capturing(n_atoms.device):
            hold_captured(n_atoms, cached[2])
        return cached[2]
    with torch.inference_mode(False):                      # it serves a training step, too
        plan = attention_plan(n_atoms, graph.num_nodes)
    object.__setattr__(graph, "_xnn_attention_plan", (n_atoms, key, plan))
    return plan


def structure_attention(q: Tensor, k: Tensor, v: Tensor, plan: AttentionPlan,
                        mask: Optional[Tensor] = None, scale: Optional[float] = None) -> Tensor:
    """``softmax(scale q k^T) v`` of every atom over the atoms of its structure.

    ``q`` (T, H, D); ``k`` and ``v`` (T, K, D) with ``H`` a multiple of ``K`` (query heads ``h`` read
    head ``h // (H / K)``); ``D <= 128``; tokens and heads may be strided (views of one projection's
    output). ``plan`` from :func:`attention_plan`. ``mask`` (T,), bool: atoms that may be attended
    to (None: all); an atom that is masked out reaches no other through its key and value, whatever they
    hold, and gets zero gradients of them; atoms with nothing to attend to get zeros. ``scale``: ``D ** -0.5``
    by default, positive. A masked atom's own row is computed as any other: where its query is not
    finite, neither are its output and, through its row's gradient, those of its structure's keys.
    Returns (T, H, D). Neither scores nor probabilities are stored; the backward
    pass forms them again from the rows' log-sums.

    Scores, softmax statistics and all sums are float32. float32 operands enter the products as three
    planes of 8 bits: a key or value that is not finite and not masked makes its structure's rows NaN,
    also where its weight would be zero. In 16 bits probabilities and score gradients are rounded to the
    type between the two products, with their rounding errors as a second term where the batch has few
    scores (``T * H * max_atoms`` up to 2^23), and the backward pass takes the rows' ``g . out``
    from the stored output in structures of more than 32 atoms."""
    if is_compiling():
        return torch.ops.xnn_amd.structure_attention(q, k, v, plan.tiles32, plan.tiles128, mask,
                                                     plan.n_tokens, plan.max_atoms, scale)
    return (_native or _ops()).structure_attention(q, k, v, plan.native, mask, scale)
