"""Tiles that are not of the tokens they are given with: the kernels stay within the tokens."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [16, 33, 128])
@pytest.mark.parametrize("tile", [(0, 400, 0), (96, 1 << 30, -64), (-32, 100, -5), (300, 500, 290), (50, 40, 45)])
def test_a_tile_beyond_the_tokens(dtype, D, tile):
    """100 tokens in the middle of larger tensors: what surrounds them is neither read (NaN) nor written."""
    import xnn_amd as xa
    ops = torch.ops.xnn_amd
    xa.attention_plan(torch.tensor([1], device=DEV))                # opens the library
    gen = torch.Generator().manual_seed(D)

    def surrounded(*shape):
        wide = torch.full((300, *shape[1:]), float("nan"), dtype=dtype, device=DEV)
        wide[100:200] = torch.randn(shape, generator=gen).to(dtype)
        return wide[100:200]
    q, k, v, g = (surrounded(100, 2, D) for _ in range(4))
    tiles = torch.tensor([tile], dtype=torch.int32, device=DEV)
    args = (q, k, v, tiles, tiles, None, 100, 100, None)
    out, lse = ops.structure_attention_lse(*args)
    ops.structure_attention_backward(g.contiguous(), torch.zeros_like(q), torch.zeros_like(lse), *args)
    first, end, begin = max(tile[0], 0), min(tile[1], 100), max(tile[2], 0)
    rows = slice(first, end)
    if first < end:
        a, b, c = (t.double().transpose(0, 1) for t in (q[rows], k[begin:end], v[begin:end]))
        want = (torch.softmax(a @ b.transpose(1, 2).contiguous() * D ** -0.5, -1) @ c).transpose(0, 1)
        torch.testing.assert_close(out[rows].double(), want, rtol=0.02, atol=0.02)
