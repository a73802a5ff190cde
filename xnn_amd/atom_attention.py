"""Attention and feed-forward blocks over atoms and :class:`AtomAttentionPotential`, the model that runs
the operators of :mod:`xnn_amd.attention` and :mod:`xnn_amd.feed_forward` together.

Every module has two evaluations of the same function, as the other fast-path modules
(common/models/fast.py:73-91): the HIP kernels, and a PyTorch formulation that is differentiable
to any order (``use_fast=False``, a CPU, float64, or a training step on forces).
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Union

import torch
from torch import Tensor, nn

from .attention import (AttentionPlan, attention_plan, dropout_add, embedding, head_norm_rotate,
                        structure_attention)
from .feed_forward import GroupPlan, group_plan, grouped_linear, layer_norm, linear
from .fast import MI355X_POLICY, FastPathModule, fast_modules, select
from .models import ShEdgePotential, register_model


def _takes(device: torch.device, dtype: torch.dtype) -> bool:
    return device.type == "cuda" and dtype in (torch.float32, torch.bfloat16, torch.float16)


# --------------------------------------------------------------------------- PyTorch forms
def dropout_keep(shape, p: float, seed: int, offset: Union[int, Tensor], device) -> Tensor:
    """The mask of :func:`~xnn_amd.attention.dropout_add`, bool of ``shape``."""
    m, n = 0xFFFFFFFF, math.prod(shape)
    i = torch.arange((n + 7) // 8, device=device)

    def words(x):
        return x.to(device).reshape(1).expand_as(i) if isinstance(x, Tensor) else torch.full_like(i, x)
    c = [i & m, i >> 32, words(offset & m), words((offset >> 32) & m)]
    k = [seed & m, (seed >> 32) & m]
    for _ in range(10):
        # 64-bit products in int64: the shifts' sign bits are masked away
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & m) ^ c[1] ^ k[0], b & m, ((a >> 32) & m) ^ c[3] ^ k[1], a & m]
        k = [(k[0] + 0x9E3779B9) & m, (k[1] + 0xBB67AE85) & m]
    w = torch.stack(c, 1)
    draws = torch.stack((w & 0xFFFF, w >> 16), 2).flatten()[:n]
    return (draws >= int(round(65536 * p))).view(shape)


def dropout_add_torch(x: Tensor, residual: Tensor, p: float, seed: int,
                      offset: Union[int, Tensor]) -> Tensor:
    drop = int(round(65536 * p))
    keep = dropout_keep(x.shape, p, seed, offset, x.device)
    factor = 65536.0 / (65536 - drop) if drop < 65536 else 0.0
    return residual + torch.where(keep, x * factor, 0.0)


def head_norm_rotate_torch(x: Tensor, weight: Tensor, cos: Tensor, sin: Tensor,
                           eps: float) -> Tensor:
    """One of queries and keys, pairs ``(i, i + R/2)``, a row of the tables a token."""
    h = cos.shape[1]
    u = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight
    a, b, c, s = u[..., :h], u[..., h:2 * h], cos[:, None], sin[:, None]
    return torch.cat((a * c - b * s, a * s + b * c, u[..., 2 * h:]), -1)


def structure_attention_torch(q: Tensor, k: Tensor, v: Tensor, n_atoms: Tensor) -> Tensor:
    """Attention within structures, padded to the longest one."""
    n = n_atoms.to(device=q.device, dtype=torch.int64)
    B, L, T = n.shape[0], int(n.max()) if n.numel() else 0, q.shape[0]
    if T == 0:
        return q.new_zeros(q.shape)
    start = torch.cumsum(n, 0) - n
    where = torch.repeat_interleave(torch.arange(B, device=q.device), n)
    rows = where * L + torch.arange(T, device=q.device) - start[where]

    def padded(x):
        x = x.repeat_interleave(q.shape[1] // x.shape[1], 1)
        full = x.new_zeros((B * L,) + x.shape[1:]).index_copy(0, rows, x)
        return full.view(B, L, *x.shape[1:]).transpose(1, 2)
    s = (padded(q) * q.shape[2] ** -0.5) @ padded(k).transpose(2, 3)
    beyond = torch.arange(L, device=q.device) >= n[:, None]
    p = torch.softmax(s.masked_fill(beyond[:, None, None, :], -math.inf), -1)
    # structures without atoms have rows of nothing, which no atom reads
    out = (p @ padded(v)).transpose(1, 2).reshape(B * L, *q.shape[1:])
    return out.index_select(0, rows)


def layer_norm_torch(x: Tensor, weight: Tensor, bias: Tensor, eps: float) -> Tensor:
    centered = x - x.mean(-1, keepdim=True)
    return centered * torch.rsqrt(centered.square().mean(-1, keepdim=True) + eps) * weight + bias


_ACTIVATIONS = {None: lambda z: z, "silu": nn.functional.silu, "gelu": nn.functional.gelu, "tanh": torch.tanh}


def linear_torch(x: Tensor, weight: Tensor, bias: Tensor, activation: Optional[str],
                 residual: Optional[Tensor] = None) -> Tensor:
    y = _ACTIVATIONS[activation](x @ weight + bias)
    return y if residual is None else residual + y


def grouped_linear_torch(x: Tensor, weight: Tensor, ids: Tensor, bias: Tensor, activation: Optional[str],
                         residual: Optional[Tensor] = None) -> Tensor:
    """The rows of each group that has some with its weight; NaN for those of no group."""
    order = torch.argsort(ids, stable=True)
    groups, counts = torch.unique(ids, return_counts=True)
    parts = [_ACTIVATIONS[activation](x[rows] @ weight[g] + bias[g]) if 0 <= g < weight.shape[0]
             else x.new_full((len(rows), weight.shape[2]), float("nan"), dtype=(x[:0] @ weight[0]).dtype)
             for g, rows in zip(groups.tolist(), order.split(counts.tolist()))]
    y = torch.cat(parts)[torch.argsort(order)] if parts else x @ weight[0]
    return y if residual is None else residual + y


# --------------------------------------------------------------------------- modules
class SpeciesEmbedding(nn.Module, FastPathModule):
    """A row of ``channels`` features a species, times ``scale``."""

    def __init__(self, n_species: int, channels: int, scale: float = 1.0,
                 generator: Optional[torch.Generator] = None):
        super().__init__()
        self.scale = float(scale)
        self.weight = nn.Parameter(torch.randn(n_species, channels, generator=generator))
        self.fast_active = False

    def fast_supported(self, device: torch.device, dtype: torch.dtype) -> bool:
        return _takes(device, dtype)

    def forward(self, z: Tensor, weight: Optional[Tensor] = None) -> Tensor:
        weight = self.weight if weight is None else weight
        if self.fast_active:
            return embedding(z, weight, self.scale)
        return self.scale * weight[z]


class AtomAttention(nn.Module, FastPathModule):
    """``x + dropout(W_o attention(rotate(norm(q)), rotate(norm(k)), v))`` with ``q, k, v = W x``.

    The heads of queries and keys are normalized and rotated by each atom's phases; an atom attends to
    the atoms of its structure. In training mode the dropout of call ``n`` draws with counter ``n``
    (:attr:`calls`, kept in the state dict: a resumed run goes on with the next one) and the module's
    ``seed``. A call that is given its ``offset`` draws with that one and leaves the counter alone:
    what is computed again in the backward pass (``torch.utils.checkpoint``) needs it, since the
    counter is by then another call's, and raises without."""

    def __init__(self, channels: int, heads: int, kv_heads: Optional[int] = None,
                 dropout: float = 0.0, seed: int = 0, eps: float = 1e-6,
                 generator: Optional[torch.Generator] = None):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if channels % heads != 0 or heads % kv_heads != 0:
            raise ValueError(f"{channels} channels, {heads} heads and {kv_heads} key and value "
                             "heads: each must divide the one before")
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, channels // heads
        self.dropout, self.seed, self.eps, self.calls = float(dropout), int(seed), float(eps), 0
        self.fast_active = False

        def weight(n_in, n_out):
            return nn.Parameter(torch.randn(n_in, n_out, generator=generator) / n_in ** 0.5)
        self.qkv = weight(channels, (heads + 2 * kv_heads) * self.head_dim)
        self.out = weight(channels, channels)
        self.q_weight = nn.Parameter(torch.ones(self.head_dim))
        self.k_weight = nn.Parameter(torch.ones(self.head_dim))

    def fast_supported(self, device: torch.device, dtype: torch.dtype) -> bool:
        return _takes(device, dtype) and self.head_dim <= 128

    def get_extra_state(self) -> Tensor:
        return torch.tensor(self.calls)

    def set_extra_state(self, state: Tensor) -> None:
        self.calls = int(state)

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys,
                              unexpected_keys, error_msgs):
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys,
                                      unexpected_keys, error_msgs)
        # a state that was saved without the counter leaves it as it is
        key = prefix + "_extra_state"
        if key in missing_keys:
            missing_keys.remove(key)

    def _next_offset(self) -> int:
        if torch._C._current_graph_task_id() != -1:
            raise RuntimeError("the dropout of a block that is computed again in a backward pass (activation "
                               "checkpointing) would draw another mask: call it with its offset")
        self.calls += 1
        return self.calls

    def forward(self, x: Tensor, cos: Tensor, sin: Tensor, n_atoms: Tensor,
                plan: Optional[AttentionPlan] = None, param_grads: bool = True,
                offset: Union[None, int, Tensor] = None) -> Tensor:
        """``x`` (N, channels), the phases' cosines and sines (N, R/2), ``n_atoms`` (B,); ``plan``
        of ``n_atoms`` for the kernels (made here when None); ``offset`` of the dropout's draws, an
        integer or an int64 tensor of one element (None: the next of :attr:`calls`)."""
        n, H, K, D = x.shape[0], self.heads, self.kv_heads, self.head_dim
        # under autocast the projections are of its type, in which the heads go on; x keeps its own
        q, k, v = (x @ self.qkv.to(x.dtype)).view(n, H + 2 * K, D).split([H, K, K], 1)
        q_weight, k_weight = self.q_weight.to(q.dtype), self.k_weight.to(q.dtype)
        if not param_grads:
            q_weight, k_weight = q_weight.detach(), k_weight.detach()
        if self.fast_active:
            q, k = head_norm_rotate(q, k, q_weight, k_weight, cos.float(), sin.float(),
                                    eps=self.eps)
            plan = attention_plan(n_atoms, n) if plan is None else plan
            y = structure_attention(q, k, v, plan)
        else:
            q, k = (head_norm_rotate_torch(t, w, cos.to(t.dtype), sin.to(t.dtype), self.eps)
                    for t, w in ((q, q_weight), (k, k_weight)))
            y = structure_attention_torch(q, k, v, n_atoms)
        y = (y.reshape(n, H * D) @ self.out.to(y.dtype)).to(x.dtype)
        if not self.training or self.dropout == 0.0:
            return x + y
        offset = self._next_offset() if offset is None else offset
        add = dropout_add if self.fast_active else dropout_add_torch
        return add(y, x, self.dropout, self.seed, offset)


class AtomFeedForward(nn.Module, FastPathModule):
    """``x + W_2 f(W_1 layer_norm(x) + b_1) + b_2``, the weights shared by all atoms or, with ``n_species``,
    those of each atom's atomic number (below ``n_species``)."""

    def __init__(self, channels: int, hidden: int, activation: Optional[str] = "silu",
                 n_species: Optional[int] = None, eps: float = 1e-5,
                 generator: Optional[torch.Generator] = None):
        super().__init__()
        if channels < 1 or hidden < 1 or (n_species is not None and n_species < 1):
            raise ValueError(f"{channels} channels, {hidden} hidden ones and {n_species} species: each must be positive")
        if activation not in _ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r} (None, 'silu', 'gelu' or 'tanh')")
        self.activation, self.n_species, self.eps = activation, n_species, float(eps)
        self.fast_active = False
        lead = () if n_species is None else (n_species,)

        def weight(n_in, n_out):
            return nn.Parameter(torch.randn(*lead, n_in, n_out, generator=generator) / n_in ** 0.5)
        self.norm_weight = nn.Parameter(torch.ones(channels))
        self.norm_bias = nn.Parameter(torch.zeros(channels))
        self.up, self.up_bias = weight(channels, hidden), nn.Parameter(torch.zeros(*lead, hidden))
        self.down, self.down_bias = weight(hidden, channels), nn.Parameter(torch.zeros(*lead, channels))

    def fast_supported(self, device: torch.device, dtype: torch.dtype) -> bool:
        return (_takes(device, dtype) and self.norm_weight.shape[0] <= 16384 and self.up.shape[-1] < 1 << 20
                and (self.n_species is None or self.n_species <= 4096))

    def forward(self, x: Tensor, z: Optional[Tensor] = None, plan: Optional[GroupPlan] = None,
                param_grads: bool = True) -> Tensor:
        """``x`` (N, channels); with species ``z`` (N,), the atomic numbers, and ``plan`` of them for the
        kernels (made here when None)."""
        params = (self.norm_weight, self.norm_bias, self.up, self.up_bias, self.down, self.down_bias)
        nw, nb, up, ub, down, db = (p.to(x.dtype) if param_grads else p.detach().to(x.dtype) for p in params)
        if self.n_species is not None and z is None:
            raise ValueError("weights of species need the atomic numbers")
        if not self.fast_active:
            n = layer_norm_torch(x, nw, nb, self.eps)
            if self.n_species is None:
                return linear_torch(linear_torch(n, up, ub, self.activation), down, db, None, x)
            return grouped_linear_torch(grouped_linear_torch(n, up, z, ub, self.activation), down, z, db, None, x)
        n, residual = layer_norm(x, nw, nb, self.eps), x
        if torch.is_autocast_enabled("cuda") and x.dtype == torch.float32:
            # under autocast the products are of its type; x keeps its own
            low = torch.get_autocast_dtype("cuda")
            n, up, ub, down, db = (t.to(low) for t in (n, up, ub, down, db))
            residual = None
        if self.n_species is None:
            y = linear(linear(n, up, ub, self.activation), down, db, None, residual)
        else:
            plan = group_plan(z, self.n_species) if plan is None else plan
            y = grouped_linear(grouped_linear(n, up, plan, ub, self.activation), down, plan, db, None, residual)
        return y if residual is not None else x + y.to(x.dtype)


@register_model("atom_attention")
class AtomAttentionPotential(ShEdgePotential):
    """Edge messages, then attention among the atoms of a structure.

    The message sums ``A_i`` of :class:`~xnn_amd.models.ShEdgePotential` give each atom the invariants
    ``s_i = log(1 + sum_m A_i[c, l, m]^2)``; features ``x_i = s_i W + embedding(Z_i)`` pass through
    ``layers`` blocks of :class:`AtomAttention`, whose phases are linear in ``s_i`` (so the energy
    does not change when the structure is turned, moved or its atoms reordered), each followed by an
    :class:`AtomFeedForward` of ``feed_forward`` hidden channels where that is not zero (with the weights of
    each atom's species where ``species_weights``), and are read out as
    ``E_i = <U, x_i> + atom_ref[Z_i]``. All geometry enters through the edge vectors: forces and
    stress come from the edge backward. ``use_fast=False``, a CPU or a training step on forces
    (``create_graph=True``) takes the PyTorch formulation.

    Block ``i`` draws its dropout with key ``(i, dropout_seed)``; ``dropout_seed`` is ``seed`` by default
    (of no ``seed``, that of torch's generator). Data-parallel ranks that are to draw different
    masks from the same weights take different ones.
    """

    def __init__(self, species: Sequence[int] = (1, 6, 7, 8), n_rbf: int = 8, l_max: int = 3,
                 channels: int = 128, cutoff: float = 5.0, heads: int = 4,
                 kv_heads: Optional[int] = None, layers: int = 2, dropout: float = 0.0,
                 embedding_scale: float = 1.0, seed: Optional[int] = 0,
                 dropout_seed: Optional[int] = None, feed_forward: int = 0, species_weights: bool = False,
                 activation: Optional[str] = "silu", **kwargs):
        super().__init__(species=species, n_rbf=n_rbf, l_max=l_max, channels=channels,
                         cutoff=cutoff, seed=seed, **kwargs)
        gen = torch.Generator().manual_seed(seed + 1) if seed is not None else None
        n_inv = channels * (l_max + 1)
        self.embed = SpeciesEmbedding(max(species) + 1, channels, embedding_scale, gen)
        if dropout_seed is None:
            dropout_seed = torch.initial_seed() if seed is None else seed
        self.blocks = nn.ModuleList(
            AtomAttention(channels, heads, kv_heads, dropout, seed=(int(dropout_seed) & 0xFFFFFFFF) << 32 | i,
                          generator=gen)
            for i in range(layers))
        self.mix = nn.Parameter(torch.randn(n_inv, channels, generator=gen) / n_inv ** 0.5)
        half = self.blocks[0].head_dim // 2 if layers else 0
        self.phase = nn.Parameter(torch.randn(n_inv, half, generator=gen) / n_inv ** 0.5)
        self.U = nn.Parameter(torch.randn(channels, generator=gen) / channels ** 0.5)
        # after the weights that a model without them has: those draw the same numbers
        self.feed_forward = nn.ModuleList(
            AtomFeedForward(channels, feed_forward, activation, max(species) + 1 if species_weights else None,
                            generator=gen)
            for _ in range(layers if feed_forward else 0))
        orders = torch.cat([torch.full((2 * l + 1,), l) for l in range(l_max + 1)])
        self.register_buffer("per_order", torch.nn.functional.one_hot(orders).float())

    def forward(self, data, offset: Union[None, int, Tensor] = None) -> dict:
        """``offset``: of the blocks' dropout (:class:`AtomAttention`)."""
        dtype = data.model_dtype
        select(fast_modules(self), self.use_fast, MI355X_POLICY, data.pos.device, dtype,
               data.num_edges, double_backward=self.double_backward)
        A = self.messages(data, data.edge_vectors())
        s = torch.log1p(A.square() @ self.per_order.to(A.dtype)).flatten(1)
        weight = self.embed.weight.to(s.dtype)
        x = s @ self.mix.to(s.dtype) + self.embed(
            data.atomic_numbers, weight if self.param_grads else weight.detach())
        angle = s @ self.phase.to(s.dtype)
        cos, sin = torch.cos(angle), torch.sin(angle)
        plan = None
        if self.blocks and self.blocks[0].fast_active:
            plan = data.attention_plan()                   # one host read a graph, not a step
        species = None
        if self.feed_forward and self.feed_forward[0].fast_active and self.feed_forward[0].n_species is not None:
            species = data.species_plan(self.feed_forward[0].n_species)
        for i, block in enumerate(self.blocks):
            x = block(x, cos, sin, data.n_atoms, plan, self.param_grads, offset)
            if self.feed_forward:
                x = self.feed_forward[i](x, data.atomic_numbers, species, self.param_grads)
        ref = self.atom_ref.to(x.dtype)
        if x.is_cuda and self.embed.fast_active:
            from .ops import node_readout_op
            U = self.U
            if not self.param_grads:
                U, ref = U.detach(), ref.detach()
            node_energy = node_readout_op(x, U, data.atomic_numbers, ref)
        else:
            node_energy = torch.addmv(ref[data.atomic_numbers], x, self.U.to(x.dtype))
        return {"node_energy": node_energy, "energy": self.aggregate_energy(node_energy, data)}
