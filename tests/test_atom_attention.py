"""The attention potential's PyTorch formulation against the operators' definitions, its symmetries,
its forces against differences, and (on a GPU) the HIP evaluation against it."""
import pytest
import torch

import oracle.attention as R
import xnn_amd as xa
from xnn_amd import atom_attention as AA
from xnn_amd import synthetic


@pytest.fixture
def float64():
    old = torch.get_default_dtype()
    torch.set_default_dtype(torch.float64)
    yield
    torch.set_default_dtype(old)


def _graph(device="cpu", n=3, cutoff=4.0):
    graphs = [xa.structure_to_graph(s.as_dict(), cutoff) for s in synthetic.random_molecules(n, seed=2)]
    return xa.collate(graphs).to(device)


def test_pytorch_forms_equal_the_definitions():
    gen = torch.Generator().manual_seed(0)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, dtype=torch.float64)
    counts = [3, 0, 11, 1]
    q, k, v = normal(15, 4, 6), normal(15, 2, 6), normal(15, 2, 6)
    got = AA.structure_attention_torch(q, k, v, torch.tensor(counts))
    torch.testing.assert_close(got, R.attention(q, k, v, counts)[0], rtol=1e-12, atol=1e-12)
    angle, w = normal(15, 2), normal(6)
    got = AA.head_norm_rotate_torch(q, w, angle.cos(), angle.sin(), 1e-6)
    torch.testing.assert_close(got, R.norm_rotate(q, w, angle.cos(), angle.sin(), 1e-6, False),
                               rtol=1e-12, atol=1e-12)
    keep = AA.dropout_keep((7, 9), 0.3, 1 << 63 | 5, (1 << 33) + 1, "cpu")
    assert torch.equal(keep.flatten(), R.keep_mask(0, 63, round(65536 * 0.3), 1 << 63 | 5, (1 << 33) + 1))


def test_philox_known_answers():
    """The test vectors published with Philox4x32-10 (Salmon, Moraes, Dror and Shaw, SC 2011)."""
    m = 0xFFFFFFFF
    assert R.philox((0,) * 4, (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert R.philox((m,) * 4, (m, m)) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_definition_gradients_are_those_of_autograd():
    """The formulas of the float64 definition against automatic differentiation."""
    gen = torch.Generator().manual_seed(1)
    counts, mask = [5, 9, 2], torch.rand(16, generator=gen) > 0.3
    mask[14:] = False
    q, k, v = (torch.randn(16, h, 4, generator=gen, dtype=torch.float64) for h in (4, 2, 2))
    g = torch.randn(16, 4, 4, generator=gen, dtype=torch.float64)
    out, *grads, _ = R.attention(q, k, v, counts, mask, 0.7, g)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    total, start = 0.0, 0
    for n in counts:
        rows = torch.arange(start, start + n)
        start += n
        keys = rows[mask[rows]]
        if len(keys) == 0:
            assert (out[rows] == 0).all()
            continue
        a = leaves[0][rows].transpose(0, 1)
        b, c = (t[keys].repeat_interleave(2, 1).transpose(0, 1) for t in leaves[1:])
        o = torch.softmax(0.7 * a @ b.transpose(1, 2), -1) @ c
        torch.testing.assert_close(o.detach().transpose(0, 1), out[rows], rtol=1e-12, atol=1e-12)
        total = total + (o.transpose(0, 1) * g[rows]).sum()
    for a, b in zip(torch.autograd.grad(total, leaves), grads):
        torch.testing.assert_close(a, b, rtol=1e-11, atol=1e-12)


def test_the_model_is_registered_and_invariant(float64):
    model = xa.build_model(xa.ModelConfig("atom_attention", dict(channels=16, heads=2, kv_heads=1,
                                                                 cutoff=4.0, layers=2))).eval()
    assert isinstance(model, xa.AtomAttentionPotential)
    g = _graph()
    want = model(g)["energy"]
    turn = torch.linalg.qr(torch.randn(3, 3, generator=torch.Generator().manual_seed(3)))[0]
    moved = _graph()
    moved.pos = moved.pos @ turn.T + 1.5
    torch.testing.assert_close(model(moved)["energy"], want, rtol=1e-10, atol=1e-10)
    # a molecule's energy does not depend on what else is in the batch
    alone = xa.structure_to_graph(synthetic.random_molecules(3, seed=2)[1].as_dict(), 4.0)
    alone = xa.collate([alone])
    torch.testing.assert_close(model(alone)["energy"][0], want[1], rtol=1e-10, atol=1e-10)


def test_forces_against_differences(float64):
    model = xa.AtomAttentionPotential(channels=16, heads=2, cutoff=4.0, layers=1).eval()
    g = _graph(n=1)
    forces = xa.ForceStressOutput(model, compute_stress=False).eval()(g)["forces"].detach()
    step = torch.randn(g.pos.shape, generator=torch.Generator().manual_seed(4))
    h = 1e-5

    def energy(sign):
        moved = _graph(n=1)
        moved.pos = moved.pos + sign * h * step
        return float(model(moved)["energy"].detach().sum())
    slope = (energy(1) - energy(-1)) / (2 * h)
    assert abs(-float((forces * step).sum()) - slope) < 1e-6 * max(1.0, float(forces.norm()))


def test_training_on_forces_takes_the_pytorch_form(float64):
    model = xa.AtomAttentionPotential(channels=16, heads=2, cutoff=4.0, dropout=0.2).train()
    out = xa.ForceStressOutput(model, compute_stress=False).train()(_graph())
    loss = out["energy"].square().sum() + out["forces"].square().sum()
    loss.backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in model.parameters())
    assert [b.calls for b in model.blocks] == [1, 1]


def test_refused_shapes():
    with pytest.raises(ValueError, match="divide"):
        xa.AtomAttention(32, 3)
    with pytest.raises(ValueError, match="divide"):
        xa.AtomAttention(32, 4, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("periodic", [False, True])
def test_hip_evaluation_equals_the_pytorch_form(periodic):
    from xnn_amd import _lib
    model = xa.AtomAttentionPotential(channels=32, heads=4, kv_heads=2, cutoff=4.0, layers=2)
    model = model.to("cuda").eval()

    def graph():
        if not periodic:
            return _graph("cuda", 5)
        s = synthetic.water_box(n_molecules=64, box=12.4, grid=4, seed=3)
        return xa.structure_to_graph(s.as_dict(), 4.0, device="cuda")
    before = {n: _lib.calls.get(n, 0) for n in ("xnn_attention", "xnn_attention_backward",
                                                "xnn_head_norm_rotate_backward", "xnn_embedding")}
    got = xa.ForceStressOutput(model, compute_stress=periodic).eval()(graph())
    assert all(_lib.calls.get(n, 0) > c for n, c in before.items())
    model.use_fast = False
    want = xa.ForceStressOutput(model, compute_stress=periodic).eval()(graph())
    # float32 on both sides: energies of a few hundred terms, forces their derivatives
    torch.testing.assert_close(got["energy"], want["energy"], rtol=2e-5, atol=2e-4)
    scale = float(want["forces"].abs().max())
    assert float((got["forces"] - want["forces"]).abs().max()) <= 2e-4 * scale
    if periodic:
        scale = float(want["stress"].abs().max())
        assert float((got["stress"] - want["stress"]).abs().max()) <= 2e-4 * scale


@pytest.mark.gpu
def test_a_fitting_step_uses_every_kernel():
    """Energies of a batch in training mode: the same loss and gradients as the PyTorch form (the
    same dropout masks), every operator's backward on its kernel."""
    from xnn_amd import _lib
    grads = []
    for fast in (True, False):
        model = xa.AtomAttentionPotential(channels=32, heads=4, cutoff=4.0, dropout=0.25,
                                          use_fast=fast).to("cuda").train()
        names = ("xnn_embedding_grad", "xnn_dropout_add", "xnn_attention_backward",
                 "xnn_head_norm_rotate_backward")
        before = {n: _lib.calls.get(n, 0) for n in names}
        loss = model(_graph("cuda", 5))["energy"].square().sum()
        loss.backward()
        if fast:
            assert all(_lib.calls.get(n, 0) > c for n, c in before.items())
        grads.append({n: p.grad.double() for n, p in model.named_parameters()})
    for n, a in grads[0].items():
        b = grads[1][n]
        assert float((a - b).norm()) <= 2e-4 * float(b.norm()) + 1e-6, n
