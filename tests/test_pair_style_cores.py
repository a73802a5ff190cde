"""Which models the pair-style wrapper evaluates by the fused edge-potential call, and the attention
potential behind it."""
import pytest
import torch

import xnn_amd as xa
from xnn_amd import synthetic
from xnn_amd.deploy import LAMMPSWrapper


class OtherEnergy(xa.ShEdgePotential):
    def forward(self, data):
        out = super().forward(data)
        return {k: 2 * v for k, v in out.items()}


class OtherMessages(xa.ShEdgePotential):
    def messages(self, data, vec):
        return super().messages(data, vec).tanh()


class OtherName(xa.ShEdgePotential):
    """The same function under another name."""


class OtherReadout(xa.ShEdgePotential):
    def __init__(self):
        super().__init__()
        self.U = torch.nn.Parameter(self.U.detach()[:, 0].clone())


def test_only_the_edge_potential_itself_takes_the_fused_call():
    assert LAMMPSWrapper(xa.ShEdgePotential()).fused_core
    assert LAMMPSWrapper(OtherName()).fused_core
    for model in (xa.AtomAttentionPotential(channels=128, heads=4), OtherEnergy(), OtherMessages(),
                  OtherReadout()):
        assert not LAMMPSWrapper(model).fused_core, type(model).__name__


@pytest.mark.gpu
@pytest.mark.parametrize("periodic", [False, True])
def test_attention_potential_behind_the_pair_style_wrapper(periodic):
    from xnn_amd import _lib
    model = xa.AtomAttentionPotential(channels=64, heads=4, kv_heads=2, cutoff=4.0).to("cuda").eval()
    if periodic:
        s = synthetic.water_box(n_molecules=64, box=12.4, grid=4, seed=3)
    else:
        s = synthetic.random_molecules(1, seed=9)[0]
    g = xa.structure_to_graph(s.as_dict(), 4.0, device="cuda")
    g.pos = g.pos.float()
    cell = torch.zeros(3, 3, device="cuda")
    if periodic:
        g.cell = g.cell.float()
        cell = g.cell[0]
    before = {n: _lib.calls.get(n, 0) for n in ("xnn_sh_pair_energy_forces", "xnn_attention")}
    pair = LAMMPSWrapper(model)(g.pos, g.edge_index, g.cell_shifts, g.atomic_numbers, cell)
    assert _lib.calls.get("xnn_sh_pair_energy_forces", 0) == before["xnn_sh_pair_energy_forces"]
    assert _lib.calls.get("xnn_attention", 0) > before["xnn_attention"]
    out = xa.ForceStressOutput(model, compute_stress=periodic).eval()(g)
    # one evaluation on the same tensors, its sums in a fixed order
    assert torch.equal(pair["node_energy"], out["node_energy"].detach().double())
    assert torch.equal(pair["forces"], out["forces"].detach())
    if periodic:
        want = -torch.det(cell.double()) * out["stress"].detach()[0].double()
    else:
        m = g.pos.detach().double().T @ out["forces"].detach().double()
        want = 0.5 * (m + m.T)
    torch.testing.assert_close(pair["virial"], want, rtol=1e-6, atol=1e-6 * float(want.abs().max()))
