"""The feed-forward half of an attention block over atoms, its operators as HIP kernels.

=======================  ============================================================
:func:`layer_norm`       norm of rows; the backward pass sums the weight's and the bias's
                         gradients over the rows
:func:`linear`           product with a weight; bias, activation and residual in its
                         epilogue
:func:`grouped_linear`   the same with the weight of each row's group (the species of an
                         atom, the expert that it is routed to)
:func:`group_plan`       the rows of each group, for :func:`grouped_linear`
=======================  ============================================================

As the operators of :mod:`xnn_amd.attention` (whose manner they share: types, streams, errors,
registration with the dispatcher) they take GPU tensors of float32, bfloat16 or float16, do
arithmetic and sums in float32 and round every output once, raise on any other tensor, run on
the current stream without host reads, sum in a fixed order and may be captured in a HIP graph.
They are differentiable once. The per-edge reference path has no counterpart.
"""
from __future__ import annotations

import ctypes
import os
from dataclasses import dataclass
from typing import Optional

import torch
from torch import Tensor
from torch.compiler import is_compiling

from . import _lib
from .plan import captured_plans, capturing, hold_captured

_native, _failure = None, None
try:
    # registers the operators (torch.ops.xnn_amd) with their shapes and derivatives
    from . import _feed_forward_ops as _built
    _built.set_library(os.path.abspath(_lib.LIBRARY))
    _lib.calls.join(_built.entries(), _built.calls)
except (ImportError, AttributeError) as err:     # not built, or from other sources: the first call says so
    _built, _failure = None, err

#: activations by name, with their codes in the C ABI
ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2, "tanh": 3}


def _ops():
    """The native operators, checked on first use (raises when they are not built)."""
    global _native
    if _native is None:
        _lib.load()
        if _built is None:
            raise RuntimeError("xnn_amd/_feed_forward_ops.so is missing, old or does not load: build it with "
                               "`python -m xnn_amd.build` (the kernels have no fallback)") from _failure
        _native = _built
    return _native


def _activation(name: Optional[str]) -> int:
    try:
        return ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError(f"unknown activation {name!r} (None, 'silu', 'gelu' or 'tanh')") from None


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None,
               eps: float = 1e-5) -> Tensor:
    """``(x - mean) / sqrt(mean (x - mean)^2 + eps) * weight + bias`` over the last dimension of ``x``
    (..., C), ``C <= 16384``; ``weight`` and ``bias`` (C,), each of which may be left out. Rows may
    be strided (a part of wider ones).

    The squares are those of the centered values. Each gradient is summed over the rows in a fixed
    order, float32 within a block of rows and float64 over the blocks."""
    if is_compiling():               # a compiler cannot look into the native entry: the same operator by name
        return torch.ops.xnn_amd.layer_norm(x, weight, bias, eps)
    return (_native or _ops()).layer_norm(x, weight, bias, eps)


def linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, activation: Optional[str] = None,
           residual: Optional[Tensor] = None) -> Tensor:
    """``residual + f(x @ weight + bias)`` for ``x`` (..., K), ``weight`` (K, N), ``bias`` (N,) and
    ``residual`` (..., N), the last two where they are given; ``activation`` ``f``: None, ``"silu"``,
    ``"gelu"`` (``z Phi(z)``, by the error function) or ``"tanh"``. Rows of ``x`` may be strided.

    Where a gradient is wanted the forward pass keeps ``f'(z)`` (beside the 16-bit types in 16 bits of a form of its
    own: off by 2^-11 of it at most down to 2^-29 in bfloat16; in float16 by 2^-14.8 of it near 1 and 2^-11 down to
    2^-19), and the backward pass rounds ``d = grad f'(z)`` to ``x``'s type once, between ``f'`` and the two products. float32 operands enter the products as three
    planes of 8 bits: one that is not finite makes the outputs it reaches NaN (the forward pass of one or two rows of
    up to 1,500 inputs multiplies in float32, and gives infinities where that does)."""
    code = _activation(activation)
    if is_compiling():
        return torch.ops.xnn_amd.dense(x, weight, bias, code, residual, None)
    return (_native or _ops()).dense(x, weight, bias, code, residual, None)


@dataclass
class GroupPlan:
    """The rows of each group (:func:`group_plan`)."""
    n_rows: int
    n_groups: int
    rows: Tensor                     # int32: the sorted rows, where the groups begin, their tiles


def group_plan(ids: Tensor, n_groups: int) -> GroupPlan:
    """The plan of rows whose groups are ``ids`` (T,), integers; kept as long as they are
    (:meth:`~xnn_amd.data.AtomicGraph.species_plan` keeps that of the species with the graph). A row with
    an id outside ``[0, n_groups)`` is of no group. At most 4,096 groups. Three launches and no host
    read: a plan of ids that are made on the device may be captured with what uses it."""
    if is_compiling():
        rows = torch.ops.xnn_amd.group_plan(ids, n_groups)
    else:
        rows = (_native or _ops()).group_plan(ids, n_groups)
    return GroupPlan(ids.shape[0], int(n_groups), rows)


class _KeptPlans:
    """A graph's plans by stream and number of groups, of one tensor of species at one version. Copied or pickled it is
    empty: versions start again there."""

    def __init__(self, ids=None, version=None):
        self.ids, self.version, self.plans = ids, version, {}

    def __reduce__(self):
        return _KeptPlans, ()


def _form_again(plan: GroupPlan, ids: Tensor) -> None:
    """``plan`` formed in its own memory once more (from other ids, of another content). A backward pass of before that
    has kept it is told, and raises."""
    torch.autograd.graph.increment_version(plan.rows)
    ids = ids.to(torch.int64).contiguous()
    sizes = [ctypes.c_size_t(), ctypes.c_size_t()]
    _lib.call("xnn_group_plan_size", plan.n_rows, plan.n_groups, *map(ctypes.byref, sizes))
    work = torch.empty(sizes[1].value, dtype=torch.uint8, device=ids.device)
    with torch.cuda.device(ids.device):
        _lib.call("xnn_group_plan", ids.data_ptr(), plan.n_rows, plan.n_groups, plan.rows.data_ptr(),
                  work.data_ptr(), work.numel(), _lib.stream(ids.device))


def species_plan_for(graph, n_groups: int) -> GroupPlan:
    """The plan of an :class:`~xnn_amd.data.AtomicGraph`'s species, kept for each stream and number of groups, and
    made again when its ``atomic_numbers`` are another tensor or were written to (of an inference tensor, which
    does not tell, at every call).

    What a capture uses is formed in it, so that each replay follows the atomic numbers as they are then: a new plan
    in the captured graph's memory, or, the first time, a kept one in its own, which serves no later call and stays as
    long as the species that the captured kernels read."""
    ids = graph.atomic_numbers
    if not ids.is_cuda or ids.is_inference():
        return group_plan(ids, n_groups)                   # (refused on a CPU)
    captured = capturing(ids.device)
    kept = getattr(graph, "_xnn_species_plan", None)
    if kept is None or kept.ids is not ids or kept.version != ids._version:
        kept = _KeptPlans(ids, ids._version)
        if not captured:
            object.__setattr__(graph, "_xnn_species_plan", kept)
    if captured:
        key = next((k for k in kept.plans if k[1] == n_groups), None)
        if key is None or any(p.n_groups == n_groups for p in captured_plans(ids)):
            return group_plan(ids, n_groups)
        plan = kept.plans.pop(key)
        hold_captured(ids, plan)
        _form_again(plan, ids)
        return plan
    key = (torch.cuda.current_stream(ids.device).cuda_stream, int(n_groups))
    plan = kept.plans.get(key)
    if plan is None:
        with torch.inference_mode(False):                  # it serves a training step, too
            plan = kept.plans[key] = group_plan(ids, n_groups)
    return plan


def grouped_linear(x: Tensor, weight: Tensor, plan: GroupPlan, bias: Optional[Tensor] = None,
                   activation: Optional[str] = None, residual: Optional[Tensor] = None) -> Tensor:
    """:func:`linear` with the weight of each row's group: row ``t`` of ``x`` (T, K) is multiplied by
    ``weight[ids[t]]``, with ``weight`` (G, K, N), ``bias`` (G, N) and ``plan`` =
    :func:`group_plan` ``(ids, G)``. Rows are read and written where they stand, in any order of groups.

    A row of no group gives a row of NaN, counts in no weight's gradient and gets zero gradients of
    its own; the weights of a group without rows get zero gradients."""
    code = _activation(activation)
    if not isinstance(plan, GroupPlan):
        raise TypeError(f"plan must be a GroupPlan (group_plan), got {type(plan).__name__}")
    if weight.dim() == 3 and weight.shape[0] != plan.n_groups:
        raise ValueError(f"the plan is of {plan.n_groups} groups, weight {tuple(weight.shape)} has "
                         f"{weight.shape[0]}")
    if is_compiling():
        return torch.ops.xnn_amd.dense(x, weight, bias, code, residual, plan.rows)
    return (_native or _ops()).dense(x, weight, bias, code, residual, plan.rows)
