"""The attention blocks' dropout masks under activation checkpointing, in a resumed run and between
models: which offset and key each call draws with."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

import xnn_amd as xa
from xnn_amd import synthetic


def _block(device="cpu", dtype=torch.float64):
    gen = torch.Generator().manual_seed(0)
    block = xa.AtomAttention(32, 4, 2, dropout=0.4, seed=7, generator=gen).to(device, dtype).train()
    block.fast_active = device != "cpu"
    x = torch.randn(30, 32, generator=gen).to(device, dtype)
    angle = torch.randn(30, 4, generator=gen).to(device, dtype)
    n_atoms = torch.tensor([21, 9], device=device)
    return block, (x, angle.cos(), angle.sin(), n_atoms)


def _gradients(block, args, offset, how):
    """The block's output and gradients; ``how``: not checkpointed (None), or which checkpoint."""
    x = args[0].clone().requires_grad_(True)
    call = (x, *args[1:], None, True, offset)
    y = block(*call) if how is None else checkpoint(block, *call, use_reentrant=how == "reentrant")
    block.zero_grad()
    y.square().sum().backward()
    return (y.detach(), x.grad, *(p.grad for p in block.parameters()))


DEVICES = [("cpu", torch.float64), pytest.param("cuda", torch.float32, marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device,dtype", DEVICES)
@pytest.mark.parametrize("how", ["kept", "reentrant"])
@pytest.mark.parametrize("as_tensor", [False, True])
def test_a_checkpointed_block_draws_its_mask_again(device, dtype, how, as_tensor):
    block, args = _block(device, dtype)
    offset = torch.tensor([5], device=device) if as_tensor else 5
    want = _gradients(block, args, offset, None)
    got = _gradients(block, args, offset, how)
    assert block.calls == 0
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert not torch.equal(_gradients(block, args, 6, None)[0], want[0])


@pytest.mark.parametrize("device,dtype", DEVICES)
@pytest.mark.parametrize("how", ["kept", "reentrant"])
def test_a_checkpointed_block_without_its_offset_is_refused(device, dtype, how):
    block, args = _block(device, dtype)
    if device == "cuda" and how == "kept":
        # the kernels' node holds the draw itself, and nothing that is needed again comes after it
        for a, b in zip(_gradients(block, args, None, how), _gradients(block, args, 1, None)):
            assert torch.equal(a, b)
    else:
        with pytest.raises(RuntimeError, match="offset"):
            _gradients(block, args, None, how)
    assert block.calls == 1                                         # the forward pass's own
    block.eval()
    for a, b in zip(_gradients(block, args, None, how), _gradients(block, args, None, None)):
        assert torch.equal(a, b)


def test_the_counter_is_the_default_offset():
    block, args = _block()
    for n in (1, 2):
        assert torch.equal(block(*args), block(*args, offset=n))
        assert block.calls == n


def test_a_resumed_run_draws_the_next_masks(tmp_path):
    block, args = _block()
    for _ in range(3):
        block(*args)
    torch.save(block.state_dict(), tmp_path / "state.pt")
    want = block(*args)
    other, _ = _block()
    other.load_state_dict(torch.load(tmp_path / "state.pt", weights_only=True))
    assert other.calls == 3 and torch.equal(other(*args), want)
    # a state without the counter is loaded, and nothing else may be missing
    state = {k: v for k, v in block.state_dict().items() if not k.endswith("_extra_state")}
    other.load_state_dict(state)
    assert other.calls == 4
    state.popitem()
    with pytest.raises(RuntimeError, match="Missing"):
        other.load_state_dict(state)


def _graph(device="cpu"):
    graphs = [xa.structure_to_graph(s.as_dict(), 4.0) for s in synthetic.random_molecules(2, seed=2)]
    return xa.collate(graphs).to(device)


def test_models_draw_with_their_seeds():
    def energies(**kw):
        torch.manual_seed(1)
        model = xa.AtomAttentionPotential(channels=16, heads=2, cutoff=4.0, dropout=0.5, **kw).train()
        weights = xa.AtomAttentionPotential(channels=16, heads=2, cutoff=4.0).state_dict()
        model.load_state_dict({k: v for k, v in weights.items() if "_extra_state" not in k})
        g = _graph()
        g.pos = g.pos.float()
        first = model(g)["energy"]
        assert torch.equal(model(g, offset=1)["energy"], first)
        return first
    base = energies(seed=0)
    assert torch.equal(base, energies(seed=3, dropout_seed=0))
    assert torch.equal(energies(seed=3), energies(seed=3))
    others = [energies(seed=3), energies(seed=0, dropout_seed=1), energies(seed=None)]
    assert not any(torch.equal(base, e) for e in others)
    assert not torch.equal(others[0], others[1])


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_a_checkpointed_model(device):
    model = xa.AtomAttentionPotential(channels=16, heads=2, cutoff=4.0, dropout=0.5).to(device).train()
    g = _graph(device)
    g.pos = g.pos.float()
    grads = []
    for f in (lambda: model(g, 9)["energy"],
              lambda: checkpoint(lambda d: model(d, 9)["energy"], g, use_reentrant=False)):
        loss = f().square().sum()
        grads.append(torch.autograd.grad(loss, list(model.parameters()), allow_unused=True))
    for a, b in zip(*grads):
        assert (a is None and b is None) or torch.equal(a, b)
    y = checkpoint(lambda d: model(d)["energy"], g, use_reentrant=False)
    with pytest.raises(RuntimeError, match="offset"):
        y.square().sum().backward()
