"""Sizes and species at the limits of the feed-forward block over atoms."""
import pytest
import torch

import xnn_amd as xa


@pytest.mark.parametrize("channels,hidden,species,fits", [
    (4, 8, None, True), (1, (1 << 20) - 1, None, True), (1, 1 << 20, None, False), (16385, 1, None, False),
    (4, 8, 4096, True), (4, 8, 4097, False)])
def test_sizes_that_the_kernels_refuse_take_the_pytorch_form(channels, hidden, species, fits):
    block = xa.AtomFeedForward(channels, hidden, n_species=species)
    assert block.fast_supported(torch.device("cuda"), torch.float32) is fits


def test_a_species_without_weights_gives_nan_in_the_pytorch_form_too():
    """As the kernels' rows of no group: no other species' weights (those of -1 were the last one's), no gradient."""
    block = xa.AtomFeedForward(4, 8, n_species=3).double()
    x = torch.randn(6, 4, dtype=torch.float64, generator=torch.Generator().manual_seed(1), requires_grad=True)
    z = torch.tensor([0, -1, 2, 3, 1, 2])
    out = block(x, z)
    known = torch.tensor([True, False, True, False, True, True])
    assert out[~known].isnan().all() and torch.equal(out[known], block(x[known], z[known]))
    got = torch.autograd.grad(out, list(block.parameters()), torch.ones_like(out))
    want = torch.autograd.grad(block(x[known], z[known]).sum(), list(block.parameters()))
    for (name, _), a, b in zip(block.named_parameters(), got, want):
        if name.startswith(("up", "down")):
            torch.testing.assert_close(a, b)
    assert block(x[:0], z[:0]).shape == (0, 4)
