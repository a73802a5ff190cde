"""The attention plan of a graph: made once, made again when the structures change, and a model's whole
step captured as a HIP graph."""
import copy

import pytest
import torch

import xnn_amd as xa
from xnn_amd import _lib, synthetic

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _graph(n=4):
    graphs = [xa.structure_to_graph(s.as_dict(), 4.0) for s in synthetic.random_molecules(n, seed=2)]
    return xa.collate(graphs).to(DEV)


def _plans():
    return _lib.calls.get("xnn_attention_plan", 0)


def test_a_graph_has_one_plan_until_its_structures_change():
    g = _graph()
    before = _plans()
    plan = g.attention_plan()
    assert g.attention_plan() is plan and copy.copy(g).attention_plan() is plan
    assert _plans() == before + 1
    counts = g.n_atoms.tolist()
    g.n_atoms[0] += counts[1]                                       # written to: the first two structures are one
    g.n_atoms[1] = 0
    joined = g.attention_plan()
    assert joined is not plan and joined.max_atoms == counts[0] + counts[1]
    g.n_atoms = torch.tensor(counts, device=DEV)
    assert g.attention_plan().max_atoms == plan.max_atoms
    assert _plans() == before + 3
    g.n_atoms = torch.tensor(counts[:-1], device=DEV)
    with pytest.raises(ValueError, match="sums to"):
        g.attention_plan()


def test_a_graph_is_copied_and_pickled_with_its_plan():
    import pickle
    g = _graph()
    plan = g.attention_plan()
    q = torch.randn(g.num_nodes, 2, 16, device=DEV)
    want = xa.structure_attention(q, q, q, plan)
    for other in (copy.deepcopy(g), pickle.loads(pickle.dumps(g))):
        again = other.attention_plan()
        assert again is not plan and torch.equal(again.tiles32, plan.tiles32)
        assert torch.equal(xa.structure_attention(q, q, q, again), want)


def test_a_step_of_the_model_reads_nothing_on_the_host():
    g = _graph()
    wrapped = xa.ForceStressOutput(xa.AtomAttentionPotential(channels=32, heads=4, cutoff=4.0).to(DEV)).eval()
    g.plan()
    g.attention_plan()
    want = wrapped(copy.copy(g))
    before = _plans()
    torch.cuda.set_sync_debug_mode("error")
    try:
        got = wrapped(copy.copy(g))
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert _plans() == before
    assert torch.equal(got["forces"], want["forces"])


@pytest.mark.parametrize("periodic", [False, True])
def test_graph_replays_match_the_eager_step(periodic):
    if periodic:
        s = synthetic.water_box(n_molecules=64, box=12.4, grid=4, seed=3)
        g = xa.structure_to_graph(s.as_dict(), 4.0, device=DEV)
    else:
        g = _graph()
    model = xa.AtomAttentionPotential(channels=32, heads=4, kv_heads=2, cutoff=4.0).to(DEV)
    wrapped = xa.ForceStressOutput(model, compute_stress=periodic).eval()
    keys = ("energy", "forces", "stress") if periodic else ("energy", "forces")
    g.plan()

    def step():
        return wrapped(copy.copy(g))
    side = torch.cuda.Stream()
    g.attention_plan()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    start = g.pos.clone()
    for k in range(4):
        g.pos.copy_(start + 0.01 * k * torch.sin(start))
        graph.replay()
        torch.cuda.synchronize()
        got = {key: static[key].clone() for key in keys}
        eager = step()
        torch.cuda.synchronize()
        for key in keys:
            assert torch.equal(got[key], eager[key]), (k, key)
