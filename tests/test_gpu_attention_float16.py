"""float16 gradients of attention whose score gradients pass the type's largest number while the
gradients themselves do not, against the definition in float64."""
import pytest
import torch

import oracle.attention as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = torch.finfo(torch.float32).eps
UNIT = 2.0 ** -11


def _compare(q, k, v, grad, counts, mask):
    import xnn_amd as xa
    *want, bounds = R.attention(*(t.double() for t in (q, k, v)), counts, mask, None, grad.double())
    assert all(float(t.abs().max()) < 65504 for t in want)          # what float16 can hold
    plan = xa.attention_plan(torch.tensor(counts, device=DEV))
    leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    out = xa.structure_attention(*leaves, plan, mask=None if mask is None else mask.to(DEV))
    got = (out, *torch.autograd.grad(out, leaves, grad.to(DEV)))
    for name, a, b, e in zip(("out", "dq", "dk", "dv"), got, want, bounds(EPS, UNIT, UNIT)):
        a = a.detach().cpu().double()
        assert torch.isfinite(a).all(), name
        worst = float(((a - b).abs() - e - 2.0 ** -25).max())
        assert worst <= 0, (name, worst, float(b.abs().max()))


def _largest_score_gradient(q, k, v, grad, mask, head=0):
    """Of one structure and one head, without its mask's keys."""
    a, b, c, g = (t[:, head].double() for t in (q, k, v, grad))
    b, c = (b, c) if mask is None else (b[mask], c[mask])
    p = torch.softmax(a @ b.T * a.shape[1] ** -0.5, 1)
    dp = g @ c.T
    return float((p * (dp - (p * dp).sum(1, keepdim=True))).abs().max())


@pytest.mark.parametrize("D", [16, 33, 64, 128])
@pytest.mark.parametrize("left", [2, 3])
def test_few_keys_of_a_long_structure_and_large_cotangents(D, left):
    """16,500 atoms of which the mask leaves two or three, cotangents of some hundreds: the probabilities are
    large although the structure is long."""
    n = 16500
    gen = torch.Generator().manual_seed(D + left)
    q, k, v, g = (torch.randn(n, 1, D, generator=gen) for _ in range(4))
    g[::40] *= 800
    mask = torch.zeros(n, dtype=torch.bool)
    mask[torch.randperm(n, generator=gen)[:left]] = True
    q, k, v, g = (t.half() for t in (q, k, v, g))
    assert _largest_score_gradient(q, k, v, g, mask) > 65504 / 32
    _compare(q, k, v, g, [n], mask)


@pytest.mark.parametrize("counts", [[20], [64, 40], [150], [1100, 70]])
@pytest.mark.parametrize("D", [16, 32, 64, 96, 128])
def test_score_gradients_beyond_the_largest_number(counts, D):
    """Cotangents of some thousands in a few rows, three keys a structure, two heads that share them; queries
    and keys are small, and so are their gradients."""
    gen = torch.Generator().manual_seed(sum(counts) + D)
    T, first = sum(counts), counts[0]
    q, k, v, g = (torch.randn(T, h, D, generator=gen) for h in (2, 1, 1, 2))
    g *= 0.01
    g[::150] = g[::150].sign() * 2.5e5 / D
    v[0], v[1] = g[0, 1].sign(), -g[0, 1].sign()
    q, k, v, g = (t.half() for t in (0.01 * q, 0.01 * k, 4 * v, g))
    mask = torch.zeros(T, dtype=torch.bool)
    mask[:3] = mask[T - 3:] = True
    assert _largest_score_gradient(q[:first], *(t[:first].repeat_interleave(2, 1) for t in (k, v)), g[:first],
                                   mask[:first], 1) > 65504
    _compare(q, k, v, g, counts, mask)
