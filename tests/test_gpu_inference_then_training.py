"""The plans that a graph keeps, made by an evaluation in inference mode, serve a training step afterwards."""
import pytest
import torch

import xnn_amd as xa
from xnn_amd import synthetic

pytestmark = pytest.mark.gpu
MODELS = {"edges": lambda: xa.ShEdgePotential(n_rbf=8, l_max=2, channels=32, cutoff=4.0, seed=0),
          "attention": lambda: xa.AtomAttentionPotential(channels=32, heads=4, cutoff=4.0),
          "species": lambda: xa.AtomAttentionPotential(channels=32, heads=4, cutoff=4.0, feed_forward=48,
                                                       species_weights=True)}


def _graph():
    graphs = [xa.structure_to_graph(s.as_dict(), 4.0) for s in synthetic.random_molecules(3, seed=2)]
    return xa.collate(graphs).to("cuda")


@pytest.mark.parametrize("name", MODELS)
def test_a_graph_is_evaluated_in_inference_mode_and_trained_on(name):
    grads = []
    for first in (True, False):
        model, g = MODELS[name]().to("cuda"), _graph()
        if first:
            with torch.inference_mode():
                model(g)
        out = model(g)["energy"]
        out.square().sum().backward()
        grads.append([out.detach()] + [p.grad for p in model.parameters() if p.grad is not None])
    assert len(grads[0]) > 2
    for a, b in zip(*grads):
        assert torch.equal(a, b)


def test_a_graph_that_inference_mode_made():
    """Its tensors are inference tensors, and so it serves evaluations alone."""
    model = MODELS["species"]().to("cuda")
    want = model(_graph())["energy"].detach()
    with torch.inference_mode():
        g = _graph()
        for _ in range(2):
            assert torch.equal(model(g)["energy"], want)
