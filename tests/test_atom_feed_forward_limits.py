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
