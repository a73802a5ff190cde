"""The operators over atoms inside a checkpoint, which computes the forward pass again while the backward pass asks for what it
kept: the gradients are the same bits."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

import xnn_amd as xa

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _normal(*shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(sum(shape))).to(DEV)


def _feed_forward(name):
    plan = xa.group_plan(torch.arange(40, device=DEV) % 3, 3)
    return {"layer_norm": (xa.layer_norm, (_normal(40, 12), _normal(12), _normal(1, 12)[0])),
            "linear": (lambda x, w, b: xa.linear(x, w, b, "silu"), (_normal(40, 12), _normal(12, 20), _normal(20))),
            "linear of a constant weight": (lambda x: xa.linear(x, _normal(12, 20)), (_normal(40, 12),)),
            "grouped_linear": (lambda x, w, b: xa.grouped_linear(x, w, plan, b, "gelu"),
                               (_normal(40, 12), _normal(3, 12, 20), _normal(3, 20)))}[name]


def _same(f, args, use_reentrant, stop=True):
    grads = []
    for again in (True, False):
        leaves = [a.clone().requires_grad_(True) for a in args]
        with torch.utils.checkpoint.set_checkpoint_early_stop(stop):
            out = checkpoint(f, *leaves, use_reentrant=use_reentrant) if again else f(*leaves)
            grads.append(torch.autograd.grad(out, leaves, torch.cos(out).detach()) if not use_reentrant else None)
            if use_reentrant:
                out.backward(torch.cos(out).detach())
                grads[-1] = [t.grad for t in leaves]
    for a, b in zip(*grads):
        assert torch.equal(a, b)


@pytest.mark.parametrize("name", ["layer_norm", "linear", "linear of a constant weight", "grouped_linear"])
@pytest.mark.parametrize("use_reentrant", [False, True])
def test_feed_forward(name, use_reentrant):
    for stop in (True, False):
        _same(*_feed_forward(name), use_reentrant, stop)


@pytest.mark.parametrize("species", [None, 9])
def test_a_feed_forward_block(species):
    block = xa.AtomFeedForward(12, 20, "gelu", species).to(DEV)
    block.fast_active = True
    z = torch.tensor([1, 6, 7, 8], device=DEV)[torch.arange(40, device=DEV) % 4]
    _same(lambda x: block(x, z), (_normal(40, 12),), False)


def _attention(name):
    plan = xa.attention_plan(torch.tensor([17, 3, 20], device=DEV)) if name == "structure_attention" else None
    ids = torch.arange(40, device=DEV) % 5
    phase = torch.linspace(0, 3, 160, device=DEV).view(40, 4)
    return {"structure_attention": (lambda q, k, v: xa.structure_attention(q, k, v, plan),
                                    (_normal(40, 4, 8), _normal(40, 2, 8), _normal(2, 40, 8).transpose(0, 1))),
            "head_norm_rotate": (lambda q, k, a, b: torch.cat(xa.head_norm_rotate(q, k, a, b, phase.cos(), phase.sin()), 1),
                                 (_normal(40, 4, 8), _normal(40, 2, 8), _normal(8), _normal(1, 8)[0])),
            "embedding": (lambda w: xa.embedding(ids, w), (_normal(5, 12),)),
            "dropout_add": (lambda x, r: xa.dropout_add(x, r, 0.3, 7, 11), (_normal(40, 12), _normal(1, 40, 12)[0]))}[name]


@pytest.mark.parametrize("name", ["structure_attention", "head_norm_rotate", "embedding", "dropout_add"])
@pytest.mark.parametrize("use_reentrant", [False, True])
def test_attention(name, use_reentrant):
    _same(*_attention(name), use_reentrant)
