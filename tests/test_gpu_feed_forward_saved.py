"""What the backward passes of the feed-forward operators keep: x for the gradients of weight and bias alone, the weight
for that of x alone. The rest may go, or be written to, before the backward pass."""
import pytest
import torch

import xnn_amd as xa

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_layer_norm_keeps_its_weight_for_x_alone():
    gen = torch.Generator().manual_seed(2)
    x, w, g = (torch.randn(*s, generator=gen).to(DEV) for s in ((30, 24), (24,), (30, 24)))
    leaf = w.clone().requires_grad_(True)
    out = xa.layer_norm(x, leaf)
    want, = torch.autograd.grad(out, leaf, g, retain_graph=True)
    with torch.no_grad():
        leaf.mul_(3.0)
    got, = torch.autograd.grad(out, leaf, g)
    assert torch.equal(got, want)
