"""The accuracy of float32 attention, head size by head size: the norm of the error is that of float32
arithmetic. The kernels form float32 products from three planes of 8 bits; the loss of one, 2^-16 of every
operand, is thirty times what these bounds allow."""
import pytest
import torch

import oracle.attention as R

DEV = "cuda:0"
# Unit roundoffs of float32, 2^-24, in the norm: a sum's dropped products and roundings (independent signs, which
# grow with the root of their number) stay below eight. Behind the output are two sums and the exponential of one,
# which a score of up to 2^2 makes four times as large; behind a gradient the same twice.
OUT, GRADIENT = 32 * 2.0 ** -24, 64 * 2.0 ** -24


def _inputs(counts, H, K, D):
    gen = torch.Generator().manual_seed(sum(counts) + D)
    T = sum(counts)
    q, k, v, g = (torch.randn(T, h, D, generator=gen) for h in (H, K, K, H))
    return q, k, v, g


def _errors(got, want):
    return [float((a.detach().cpu().double() - b).norm() / b.norm()) for a, b in zip(got, want)]


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [[30] * 12, [100] * 12, [1100]], ids=["short", "whole", "parts"])
@pytest.mark.parametrize("D", [13, 16, 27, 32, 50, 64, 81, 96, 111, 128])
@pytest.mark.parametrize("shift", [0, 1], ids=["aligned", "shifted"])
def test_float32_attention_errs_as_float32(counts, D, shift):
    import xnn_amd as xa
    H, K = 2, 1
    q, k, v, g = _inputs(counts, H, K, D)
    *want, _ = R.attention(*(t.double() for t in (q, k, v)), counts, None, None, g.double())
    leaves = []
    for t in (q, k, v):
        d = torch.empty(t.numel() + shift, device=DEV)[shift:].view(t.shape)
        leaves.append(d.copy_(t).requires_grad_(True))
    out = xa.structure_attention(*leaves, xa.attention_plan(torch.tensor(counts, device=DEV)))
    got = (out, *torch.autograd.grad(out, leaves, g.to(DEV)))
    for name, e, bound in zip(("out", "dq", "dk", "dv"), _errors(got, want), (OUT, *(GRADIENT,) * 3)):
        assert e <= bound, (name, e)


@pytest.mark.parametrize("D", [16, 32, 64, 128])
def test_the_bounds_notice_a_lost_plane(D):
    """The definition with every operand of a product cut to two planes of 8 bits: no output passes."""
    counts = [200]
    q, k, v, g = _inputs(counts, 2, 1, D)
    *want, _ = R.attention(*(t.double() for t in (q, k, v)), counts, None, None, g.double())

    def cut(x):
        # 24 significant bits, the last eight of them zero
        x = x.float()
        return (x.view(torch.int32) & ~0xFF).view(torch.float32).double()
    scale = D ** -0.5
    k, v = (cut(t).repeat_interleave(2, 1).transpose(0, 1) for t in (k, v))
    q, g = cut(q * scale).transpose(0, 1), cut(g).transpose(0, 1)
    p = torch.softmax(q @ k.transpose(1, 2), -1)
    out = cut(p) @ v
    dp = g @ v.transpose(1, 2)
    ds = cut(p * (dp - (g * out).sum(-1, keepdim=True)))
    got = [out, scale * ds @ k, (ds.transpose(1, 2) @ q).sum(0, keepdim=True),
           (cut(p).transpose(1, 2) @ g).sum(0, keepdim=True)]
    for e, bound in zip(_errors([t.transpose(0, 1) for t in got], want), (OUT, *(GRADIENT,) * 3)):
        assert e > 2 * bound, e
