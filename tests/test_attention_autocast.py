"""The attention block and model under torch.autocast."""
import pytest
import torch

import xnn_amd as xa
from xnn_amd import synthetic

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dropout", [0.0, 0.3])
def test_a_block_under_autocast(device, dtype, dropout):
    """Norm of the error against float64: the output has nine roundings to 16 bits behind it (two operands and
    the result of each projection, norm, probabilities and attention), the gradients those of both
    passes; each is of half a unit at most."""
    if device == "cpu" and dtype == torch.float16:
        pytest.skip("float16 products on a CPU")
    gen = torch.Generator().manual_seed(0)
    block = xa.AtomAttention(64, 4, 2, dropout=dropout, generator=gen).double().train()
    x = torch.randn(90, 64, generator=gen, dtype=torch.float64)
    angle = torch.randn(90, 8, generator=gen, dtype=torch.float64)
    g = torch.randn(90, 64, generator=gen, dtype=torch.float64)
    n_atoms = torch.tensor([64, 26])

    def run(block, x, angle, g, n_atoms):
        leaf = x.clone().requires_grad_(True)
        y = block(leaf, angle.cos(), angle.sin(), n_atoms, offset=1)
        assert y.dtype == x.dtype
        return (y.detach(), *torch.autograd.grad(y, (leaf, *block.parameters()), g))
    want = run(block, x, angle, g, n_atoms)
    block = block.float().to(device)
    block.fast_active = device != "cpu"
    with torch.autocast(device, dtype):
        got = run(block, *(t.float().to(device) for t in (x, angle, g)), n_atoms.to(device))
    unit = torch.finfo(dtype).eps
    for i, (a, b) in enumerate(zip(got, want)):
        assert a.dtype == torch.float32
        off = float((a.cpu().double() - b).norm() / b.norm())
        assert off <= (9 if i == 0 else 18) * unit / 2, (i, off)


@pytest.mark.gpu
def test_a_fitting_step_under_autocast():
    from xnn_amd import _lib
    graphs = [xa.structure_to_graph(s.as_dict(), 4.0) for s in synthetic.random_molecules(5, seed=2)]
    grads = []
    for cast in (False, True):
        model = xa.AtomAttentionPotential(channels=32, heads=4, cutoff=4.0, dropout=0.25).to("cuda").train()
        g = xa.collate(graphs).to("cuda")
        before = _lib.calls.get("xnn_attention_backward", 0)
        with torch.autocast("cuda", torch.bfloat16, enabled=cast):
            loss = model(g)["energy"].square().mean()
        loss.backward()
        assert _lib.calls.get("xnn_attention_backward", 0) == before + len(model.blocks)
        grads.append(torch.cat([p.grad.double().flatten() for p in model.parameters()]))
    assert grads[1].isfinite().all()
    # the direction of the float32 step, up to the roundings of two blocks and the readout
    cosine = float(grads[0] @ grads[1] / (grads[0].norm() * grads[1].norm()))
    assert cosine > 1 - (2 * 18 * 2.0 ** -9) ** 2 - 1e-3, cosine
