"""The attention operators over atoms against float64 evaluations of their definitions: odd sizes,
strides, masks that leave nothing, values that are not finite, shared heads, other streams."""
import math

import pytest
import torch

import oracle.attention as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = torch.finfo(torch.float32).eps
# unit roundoff of the stored values (float32: two, a factor and a sum may each round); below
# 2^-14 a float16 is rounded to a multiple of 2^-24, whatever its size
UNIT = {torch.float32: EPS, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = list(UNIT)


def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen).to(dtype)


def _close(got, want, bound):
    stored, got = got.dtype, got.detach().cpu().double()
    assert got.shape == want.shape
    assert torch.isfinite(got).all()
    if stored == torch.float16:
        bound = bound + 2.0 ** -25
    worst = ((got - want).abs() - bound).max() if got.numel() else torch.tensor(-1.0)
    assert worst <= 0, f"beyond the bound by {float(worst):.3e} of {float(want.abs().max()):.3e}"


# --------------------------------------------------------------------------- embedding
@pytest.mark.parametrize("n,V,C", [(1, 1, 1), (0, 5, 16), (21, 119, 128), (33, 3, 65), (4097, 2, 64),
                                   (700, 70000, 24), (5000, 300, 250), (2500, 1000, 1024),
                                   (16384, 256, 8), (20000, 1000, 8), (70000, 300, 4), (40000, 70000, 3),
                                   (3000, 255, 40), (1100000, 4, 4)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_embedding_and_its_gradient(n, V, C, dtype):
    import xnn_amd as xa
    gen = torch.Generator().manual_seed(n + V)
    table, grad = _normal(gen, V, C, dtype=dtype), _normal(gen, n, C, dtype=dtype)
    ids = (torch.rand(n, generator=gen) ** 3 * V).long()
    t = table.to(DEV).requires_grad_(True)
    out = xa.embedding(ids.to(DEV), t, 1.7)
    want = R.embedding(ids, table.double(), 1.7)
    _close(out, want, (UNIT[dtype] + EPS) * want.abs())
    (got,) = torch.autograd.grad(out, t, grad.to(DEV))
    want = R.embedding_grad(ids, grad.double(), V, 1.7)
    size = R.embedding_grad(ids, grad.double().abs(), V, 1.7)
    # a row's terms added one after the other at the worst
    _close(got, want, UNIT[dtype] * want.abs() + (n + 2) * EPS * size)


def test_embedding_of_ids_outside_the_table():
    import xnn_amd as xa
    table = torch.ones(4, 8, device=DEV, requires_grad=True)
    ids = torch.tensor([[0, -1, 3], [4, 1 << 40, -(1 << 62)]], device=DEV)
    out = xa.embedding(ids, table, 2.0)
    good = torch.tensor([[True, False, True], [False] * 3], device=DEV)
    assert (out[good] == 2).all() and out[~good].isnan().all()
    (g,) = torch.autograd.grad(out, table, torch.ones_like(out))
    assert g[:, 0].tolist() == [2, 0, 0, 2]


def test_embedding_is_differentiable_twice():
    import xnn_amd as xa
    gen = torch.Generator().manual_seed(0)
    ids = torch.randint(0, 5, (40,), generator=gen).to(DEV)
    table = _normal(gen, 5, 12).to(DEV).requires_grad_(True)
    out = xa.embedding(ids, table, 0.5)
    (g,) = torch.autograd.grad((out ** 2).sum(), table, create_graph=True)
    (h,) = torch.autograd.grad(g.sum(), table)
    count = torch.bincount(ids, minlength=5)[:, None].float()
    torch.testing.assert_close(h, 0.5 * count.expand_as(h), rtol=1e-5, atol=1e-6)


# --------------------------------------------------------------------------- dropout
@pytest.mark.parametrize("shape", [(1,), (0, 3), (7, 33), (129, 64), (5, 3, 17)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("p,residual", [(0.0, True), (0.1, True), (0.5, False), (1.0, True)])
def test_dropout(shape, dtype, p, residual):
    import xnn_amd as xa
    gen = torch.Generator().manual_seed(len(shape))
    x, r, g = (_normal(gen, *shape, dtype=dtype) for _ in range(3))
    seed, offset = 0x9123456789ABCDEF, (1 << 40) + 7
    xd, rd = x.to(DEV).requires_grad_(True), r.to(DEV).requires_grad_(True) if residual else None
    out = xa.dropout_add(xd, rd, p, seed, offset)
    drop = round(65536 * p)
    keep = R.keep_mask(0, x.numel(), drop, seed, offset).view(shape)
    factor = keep.double() * (65536 / max(65536 - drop, 1))
    want = x.double() * factor + (r.double() if residual else 0.0)
    size = (x.double() * factor).abs() + (r.double().abs() if residual else 0.0)
    _close(out, want, UNIT[dtype] * want.abs() + 2 * EPS * size)
    got = torch.autograd.grad(out, [xd] + ([rd] if residual else []), g.to(DEV))
    want = g.double() * factor
    _close(got[0], want, (UNIT[dtype] + EPS) * want.abs())
    if residual:
        assert torch.equal(got[1].cpu(), g)


def test_dropout_draws_by_index_seed_and_offset():
    import xnn_amd as xa
    x = torch.ones(1000, 33, device=DEV)
    a = xa.dropout_add(x, None, 0.25, 5, 9)
    view = torch.ones(1000, 66, device=DEV)[:, ::2]
    assert torch.equal(a, xa.dropout_add(view, None, 0.25, 5, 9))
    shifted = torch.ones(33001, device=DEV)[1:].view(1000, 33)      # an address of its own alignment
    assert torch.equal(a, xa.dropout_add(shifted, None, 0.25, 5, 9))
    assert torch.equal(a, xa.dropout_add(x, None, 0.25, 5, torch.tensor([9], device=DEV)))
    assert not torch.equal(a, xa.dropout_add(x, None, 0.25, 6, 9))
    assert not torch.equal(a, xa.dropout_add(x, None, 0.25, 5, 10))
    # 33,000 draws: five standard deviations
    kept = (a != 0).float().mean().item()
    assert abs(kept - 0.75) < 5 * math.sqrt(0.75 * 0.25 / 33000)
    x[0] = float("nan")
    out = xa.dropout_add(x, torch.zeros_like(x), 0.25, 5, 9)
    assert (out[0][a[0] == 0] == 0).all()                           # a dropped value is not read


def test_dropout_beyond_32_bits_of_elements():
    import xnn_amd as xa
    n = (1 << 31) + 1000
    x = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    out = xa.dropout_add(x, None, 0.5, 3, 4)
    first = n - 777
    keep = R.keep_mask(first, 777, 32768, 3, 4)
    assert torch.equal(out[first:].cpu() != 0, keep)


# --------------------------------------------------------------------------- norm and rotation
@pytest.mark.parametrize("T,H,K,D,rot", [(1, 1, 1, 2, 2), (3, 4, 4, 32, 32), (65, 8, 2, 128, 128),
                                         (130, 3, 1, 48, 24), (17, 2, 1, 33, 20), (40, 40, 8, 64, 64),
                                         (9, 1, 1, 1, 0), (2100, 4, 2, 16, 8), (0, 2, 2, 16, 16)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mode", ["rows", "positions", "interleaved"])
def test_head_norm_rotate(T, H, K, D, rot, dtype, mode):
    import xnn_amd as xa
    gen = torch.Generator().manual_seed(T + D)
    qk = _normal(gen, T, H + K, D, dtype=dtype)
    wq, wk = (1 + 0.1 * _normal(gen, D)).to(dtype), (1 + 0.1 * _normal(gen, D)).to(dtype)
    rows = 50 if mode == "positions" else T
    angle = 6.3 * torch.rand(rows, rot // 2, generator=gen)
    cos, sin = torch.cos(angle), torch.sin(angle)
    pos = torch.randint(0, 50, (T,), generator=gen) if mode == "positions" else None
    g = _normal(gen, T, H, D, dtype=dtype), _normal(gen, T, K, D, dtype=dtype)
    inter = mode == "interleaved"

    leaves = [t.double().requires_grad_(True) for t in (qk[:, :H], qk[:, H:], wq, wk, cos, sin)]
    c, s = (t if pos is None else t[pos] for t in leaves[4:])
    want = [R.norm_rotate(x, w, c, s, 1e-5, inter) for x, w in zip(leaves[:2], leaves[2:4])]
    n_grads = 4 if pos is not None else 6
    want_g = torch.autograd.grad(want, leaves[:n_grads], [t.double() for t in g], allow_unused=True)

    d = qk.to(DEV)
    dev = [d[:, :H], d[:, H:], wq.to(DEV), wk.to(DEV), cos.to(DEV), sin.to(DEV)]
    dev = [t.detach().requires_grad_(i < n_grads) for i, t in enumerate(dev)]
    got = xa.head_norm_rotate(*dev, positions=None if pos is None else pos.to(DEV), eps=1e-5,
                              interleaved=inter)
    got_g = torch.autograd.grad(got, dev[:n_grads], [t.to(DEV) for t in g])
    u = UNIT[dtype]
    for a, b, w in zip(got, want, (wq, wk)):
        # the norm is a sum of D squares; a pair's two products, each at most the head's largest
        size = b.detach().abs() + (b.detach().abs().amax(-1, keepdim=True) if rot else 0.0)
        _close(a, b.detach(), u * b.detach().abs() + (D + 12) * EPS * size)
    if T == 0:
        assert all((x == 0).all() for x in got_g)
        return
    for i, (a, b) in enumerate(zip(got_g, want_g)):
        if b is None:
            b = torch.zeros_like(leaves[i])
        x = leaves[i % 2].detach() if i < 4 else None
        if i < 2:
            gi, w = g[i].double(), (wq, wk)[i].double()
            r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5)
            # dx = r (w g - n mean(w g n)): D-term sums of at most |w| |g| and |n|, 2 products a turn
            n = (x * r).abs()
            top = 2 * w.abs().max() * gi.abs().amax(-1, keepdim=True)
            _close(a, b, u * b.abs() + (D + 16) * EPS * r * top * (1 + n * n.mean(-1, keepdim=True)))
        elif i < 4:
            gi = g[i - 2].double()
            x = leaves[i - 2].detach()
            n = (x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5)).abs()
            heads = gi.shape[1]
            size = (2 * gi.abs().amax(-1, keepdim=True) * n).sum((0, 1))
            # T heads terms a column in runs, at worst one after the other
            _close(a, b, u * b.abs() + (T * heads + D + 16) * EPS * size)
        else:
            size = sum((2 * gi.double().abs().amax(-1) * y.detach().abs().amax(-1) * 2).sum(1)
                       for gi, y in zip(g, want))[:, None]
            _close(a, b, (D + H + K + 20) * EPS * size.expand_as(b))


def test_head_norm_rotate_positions_outside_the_tables():
    import xnn_amd as xa
    q = torch.ones(3, 2, 8, device=DEV)
    w = torch.ones(8, device=DEV)
    cos, sin = torch.ones(4, 2, device=DEV), torch.zeros(4, 2, device=DEV)
    a, b = xa.head_norm_rotate(q, q, w, w, cos, sin, positions=torch.tensor([0, 4, -1], device=DEV))
    assert a[0].isfinite().all() and a[1:, :, :4].isnan().all() and b[1:, :, :4].isnan().all()
    assert a[:, :, 4:].isfinite().all()                             # elements that are not turned


# --------------------------------------------------------------------------- attention
def _attention_inputs(counts, H, K, D, dtype, masked, packed, seed=0):
    gen = torch.Generator().manual_seed(seed + sum(counts) + D)
    T = sum(counts)
    qkv = _normal(gen, T, H + 2 * K, D, dtype=dtype)
    grad = _normal(gen, T, H, D, dtype=dtype)
    mask = None
    if masked:
        mask = torch.rand(T, generator=gen) >= 0.3
        if len(counts) > 1:                                         # the first structure has none left
            mask[:counts[0]] = False
    parts = qkv.split([H, K, K], 1)
    d = qkv.to(DEV)
    dev = d.split([H, K, K], 1) if packed else [p.contiguous().to(DEV) for p in parts]
    return parts, [t.detach().requires_grad_(True) for t in dev], grad, mask


@pytest.mark.parametrize("counts,H,K,D", [
    ([1], 1, 1, 1), ([21], 4, 4, 32), ([63, 0, 64, 65, 1], 2, 1, 16), ([129, 3], 4, 2, 33),
    ([300], 2, 2, 64), ([40, 17, 128], 8, 2, 128), ([200, 31], 1, 1, 96), ([70] * 9, 2, 2, 20),
    ([1100], 1, 1, 8), ([500, 600, 257], 4, 4, 48)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("masked,packed", [(False, True), (True, False)])
def test_structure_attention(counts, H, K, D, dtype, masked, packed):
    import xnn_amd as xa
    parts, dev, grad, mask = _attention_inputs(counts, H, K, D, dtype, masked, packed)
    *want, bounds = R.attention(*(t.double() for t in parts), counts, mask, None, grad.double())
    plan = xa.attention_plan(torch.tensor(counts, device=DEV), sum(counts))
    m = None if mask is None else mask.to(DEV)
    out = xa.structure_attention(*dev, plan, mask=m)
    got = (out, *torch.autograd.grad(out, dev, grad.to(DEV)))
    u = UNIT[dtype]
    for name, a, b, e in zip(("out", "dq", "dk", "dv"), got, want,
                             bounds(EPS, u, 0.0 if dtype == torch.float32 else u)):
        try:
            _close(a, b, e + 1e-30)
        except AssertionError as err:
            raise AssertionError(f"{name}: {err}") from None
    with torch.no_grad():
        assert torch.equal(xa.structure_attention(*dev, plan, mask=m), out)


@pytest.mark.parametrize("counts,H,K,D", [
    ([65], 2, 2, 65), ([33, 129], 2, 1, 72), ([64, 1, 200], 4, 4, 80), ([700], 4, 1, 95),
    ([31, 60], 1, 1, 96), ([1500, 3], 2, 2, 96), ([129, 300], 2, 2, 97)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("masked,packed", [(False, True), (True, True), (True, False)])
def test_structure_attention_around_heads_of_96(counts, H, K, D, dtype, masked, packed):
    test_structure_attention(counts, H, K, D, dtype, masked, packed)


@pytest.mark.parametrize("runs", [[(0, 64)], [(64, 128), (192, 448)], [(10, 447)], [(0, 447)]])
@pytest.mark.parametrize("D", [16, 32])
@pytest.mark.parametrize("dtype", DTYPES)
def test_whole_tiles_that_the_mask_leaves_out(runs, D, dtype):
    import xnn_amd as xa
    counts, H, K = [448, 20], 2, 1
    parts, dev, grad, _ = _attention_inputs(counts, H, K, D, dtype, False, True)
    mask = torch.ones(sum(counts), dtype=torch.bool)
    for a, b in runs:
        mask[a:b] = False
    *want, bounds = R.attention(*(t.double() for t in parts), counts, mask, None, grad.double())
    plan = xa.attention_plan(torch.tensor(counts, device=DEV), sum(counts))
    with torch.no_grad():
        for t in dev[1:]:                                           # what they hold reaches nothing
            t[~mask.to(DEV)] = float("nan")
    out = xa.structure_attention(*dev, plan, mask=mask.to(DEV))
    got = (out, *torch.autograd.grad(out, dev, grad.to(DEV)))
    u = UNIT[dtype]
    for a, b, e in zip(got, want, bounds(EPS, u, 0.0 if dtype == torch.float32 else u)):
        _close(a, b, e + 1e-30)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [16, 64])
def test_a_long_structure_loses_no_more_than_short_ones(dtype, D):
    """20,000 atoms: the average probability is below float16's least normal number. The norm of the
    errors is at most that of two roundings, of the output and of the weights, each of half a unit at
    most."""
    import xnn_amd as xa
    n = 20000
    gen = torch.Generator(device=DEV).manual_seed(D)
    q, k, v, g = (torch.randn(n, 1, D, generator=gen, device=DEV).to(dtype) for _ in range(4))
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = xa.structure_attention(*leaves, xa.attention_plan(torch.tensor([n], device=DEV)))
    got = (out, *torch.autograd.grad(out, leaves, g))
    a, b, c, e = (t[:, 0].double() for t in (q, k, v, g))
    want = [torch.zeros_like(a) for _ in range(4)]
    for i in range(0, n, 2500):
        r = slice(i, i + 2500)
        p = torch.softmax(a[r] @ b.T * D ** -0.5, 1)
        o, dp = p @ c, e[r] @ c.T
        ds = p * (dp - (e[r] * o).sum(1, keepdim=True)) * D ** -0.5
        want[0][r], want[1][r] = o, ds @ b
        want[2] += ds.T @ a[r]
        want[3] += p.T @ e[r]
    for name, x, y in zip(("out", "dq", "dk", "dv"), got, want):
        off = float((x[:, 0].double() - y).norm() / y.norm())
        assert off <= 2 * UNIT[dtype] / 2, (name, off)


def test_attention_gradients_against_differences():
    """Central differences of the float64 definition along a direction and the kernels' gradients."""
    import xnn_amd as xa
    counts = [37, 90]
    parts, dev, grad, mask = _attention_inputs(counts, 4, 2, 24, torch.float32, True, True)
    plan = xa.attention_plan(torch.tensor(counts, device=DEV))
    out = xa.structure_attention(*dev, plan, mask=mask.to(DEV), scale=0.3)
    got = torch.autograd.grad(out, dev, grad.to(DEV))
    gen = torch.Generator().manual_seed(9)
    h = 1e-5
    for i in range(3):
        step = torch.randn(parts[i].shape, generator=gen, dtype=torch.float64)

        def value(sign):
            moved = [t.double() + (sign * h * step if j == i else 0) for j, t in enumerate(parts)]
            return float((R.attention(*moved, counts, mask, 0.3)[0] * grad.double()).sum())
        slope = (value(1) - value(-1)) / (2 * h)
        mine = float((got[i].cpu().double() * step).sum())
        size = float((got[i].cpu().double() * step).norm())
        # float32 gradients (a few hundred roundings a term) and the differences' own h^2
        assert abs(mine - slope) <= 1e-4 * size, (i, mine, slope)


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_masked_atoms_and_other_structures_hold_reaches_nothing(dtype):
    import xnn_amd as xa
    counts = [50, 70, 20]
    parts, _, grad, _ = _attention_inputs(counts, 2, 2, 32, dtype, False, False)
    mask = torch.ones(140, dtype=torch.bool)
    mask[55:60] = False                                             # of the second structure
    mask[120:] = False                                              # all of the third
    plan = xa.attention_plan(torch.tensor(counts, device=DEV))

    def run(bad):
        q, k, v = (t.clone() for t in parts)
        g = grad.clone()
        if bad is not None:
            k[55:60], v[55:60], k[120:], v[120:] = bad, bad, bad, bad
            q[:50], k[:50], v[:50] = bad, bad, bad                  # the first structure entirely
        dev = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
        out = xa.structure_attention(*dev, plan, mask=mask.to(DEV))
        return (out, *torch.autograd.grad(out, dev, g.to(DEV)))
    clean = run(None)
    for bad in (float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min):
        for a, b in zip(clean, run(bad)):
            assert torch.equal(a[50:], b[50:])
    for a in clean[2:]:
        assert (a[55:60] == 0).all()
    for a in clean:
        assert (a[120:] == 0).all()


def test_rows_without_keys_pass_no_cotangent_on():
    import xnn_amd as xa
    q, k, v = (torch.randn(30, 2, 16, device=DEV, requires_grad=True) for _ in range(3))
    plan = xa.attention_plan(torch.tensor([10, 20], device=DEV))
    mask = torch.ones(30, dtype=torch.bool, device=DEV)
    mask[:10] = False
    out = xa.structure_attention(q, k, v, plan, mask=mask)
    g = torch.randn_like(out)
    g[:10] = float("nan")
    for a in torch.autograd.grad(out, (q, k, v), g):
        assert (a[:10] == 0).all() and a[10:].isfinite().all()


def test_attention_of_far_apart_scores():
    """Scores of tens of thousands apart: the largest takes all, nothing overflows."""
    import xnn_amd as xa
    n, D = 200, 32
    q = torch.zeros(n, 1, D, device=DEV)
    q[:, 0, 0] = 1000.0
    k = torch.zeros(n, 1, D, device=DEV)
    k[:, 0, 0] = torch.arange(n, device=DEV).float() * 10 - 1000
    v = torch.randn(n, 1, D, device=DEV)
    plan = xa.attention_plan(torch.tensor([n], device=DEV))
    q.requires_grad_(True)
    out = xa.structure_attention(q, k, v, plan)
    assert torch.equal(out.detach(), v[-1:].expand_as(v))
    assert (torch.autograd.grad(out.sum(), q)[0] == 0).all()


@pytest.mark.parametrize("counts", [[], [0, 0]])
def test_batches_without_atoms(counts):
    import xnn_amd as xa
    plan = xa.attention_plan(torch.tensor(counts, dtype=torch.int64, device=DEV))
    assert (plan.n_tokens, plan.max_atoms) == (0, 0)
    q = torch.randn(0, 2, 8, device=DEV, requires_grad=True)
    out = xa.structure_attention(q, q, q, plan, mask=torch.ones(0, dtype=torch.bool, device=DEV))
    assert out.shape == (0, 2, 8) and torch.autograd.grad(out.sum(), q)[0].shape == q.shape


def test_only_wanted_gradients_are_formed():
    """Gradients asked for one at a time are those asked for together; an output without a cotangent
    counts as zeros."""
    import xnn_amd as xa
    gen = torch.Generator().manual_seed(8)
    leaves = [_normal(gen, *s).to(DEV).requires_grad_(True)
              for s in ((40, 2, 16), (40, 1, 16), (16,), (16,), (40, 8), (40, 8))]
    grads = [_normal(gen, 40, h, 16).to(DEV) for h in (2, 1)]
    outs = xa.head_norm_rotate(*leaves)
    together = torch.autograd.grad(outs, leaves, grads, retain_graph=True)
    for x, g in zip(leaves, together):
        assert torch.equal(torch.autograd.grad(outs, x, grads, retain_graph=True)[0], g)
    alone = torch.autograd.grad(outs[0], leaves[:2], grads[0], retain_graph=True)
    assert torch.equal(alone[0], together[0]) and (alone[1] == 0).all()
    v = _normal(gen, 40, 1, 16).to(DEV).requires_grad_(True)
    out = xa.structure_attention(leaves[0], leaves[1], v, xa.attention_plan(torch.tensor([40], device=DEV)))
    g = torch.randn_like(out)
    together = torch.autograd.grad(out, (leaves[0], leaves[1], v), g, retain_graph=True)
    for x, a in zip((leaves[0], leaves[1], v), together):
        assert torch.equal(torch.autograd.grad(out, x, g, retain_graph=True)[0], a)


def test_dropout_is_differentiable_twice():
    import xnn_amd as xa
    x = torch.randn(50, 9, device=DEV, requires_grad=True)
    y = xa.dropout_add(x, None, 0.4, 11, 3)
    (g,) = torch.autograd.grad((y ** 2).sum(), x, create_graph=True)
    (h,) = torch.autograd.grad(g.sum(), x)
    factor = torch.where(y.detach() != 0, 65536 / (65536 - round(0.4 * 65536)), 0.0)
    torch.testing.assert_close(h, 2 * factor ** 2, rtol=1e-5, atol=1e-6)


def test_forward_mode_and_batched_transforms_are_refused():
    import torch.autograd.forward_ad as fa
    import xnn_amd as xa
    x = torch.randn(4, 8, device=DEV)
    with fa.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            xa.dropout_add(fa.make_dual(x, torch.ones_like(x)), None, 0.5, 1)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: xa.dropout_add(t, None, 0.5, 1))(x)


def test_attention_with_strides_beyond_32_bits():
    import xnn_amd as xa
    T, D, stride = 66, 16, 1 << 26                                  # 66 x 2^26 elements: 8.9 GB
    store = torch.empty(T * stride, dtype=torch.bfloat16, device=DEV)
    gen = torch.Generator().manual_seed(4)
    small = [_normal(gen, T, 1, D, dtype=torch.bfloat16).to(DEV) for _ in range(3)]
    views = []
    for i, t in enumerate(small):
        w = store.as_strided((T, 1, D), (stride, D, 1), 1024 * i)
        w.copy_(t)
        views.append(w)
    plan = xa.attention_plan(torch.tensor([T], device=DEV))
    want, got = ([t.detach().requires_grad_(True) for t in s] for s in (small, views))
    outs = [xa.structure_attention(*s, plan) for s in (want, got)]
    assert torch.equal(*outs)
    g = torch.randn_like(outs[0])
    for a, b in zip(*(torch.autograd.grad(o, s, g) for o, s in zip(outs, (want, got)))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("shift", [1, 2, 4])
def test_results_do_not_depend_on_the_alignment(shift):
    import xnn_amd as xa
    gen = torch.Generator().manual_seed(5)
    plan = xa.attention_plan(torch.tensor([100, 33], device=DEV))
    w = torch.ones(32, device=DEV)
    angle = torch.rand(133, 16, generator=gen).to(DEV)

    def block(ts, grad):
        q, k, v = (t.requires_grad_(True) for t in ts)
        a, b = xa.head_norm_rotate(q, k, w, w, angle.cos(), angle.sin())
        out = xa.structure_attention(a, b, v, plan)
        return (out, *torch.autograd.grad(out, (q, k, v), grad))
    parts = [_normal(gen, 133, 2, 32).to(DEV) for _ in range(4)]
    shifted = [torch.empty(t.numel() + shift, device=DEV)[shift:].view(t.shape).copy_(t) for t in parts]
    want = block([t.clone() for t in parts[:3]], parts[3])
    got = block(shifted[:3], shifted[3])
    for a, b in zip(want, got):
        torch.testing.assert_close(a, b, rtol=2e-5, atol=2e-5)


@pytest.mark.parametrize("D", [1, 5, 17, 33, 50, 66, 97, 127])
@pytest.mark.parametrize("dtype", DTYPES)
def test_what_lies_between_the_heads_reaches_nothing(D, dtype):
    """Heads of odd sizes and strides with NaN after each: the same bits as without gaps."""
    import xnn_amd as xa
    counts = [130, 1, 64, 65]
    parts, dev, grad, _ = _attention_inputs(counts, 2, 1, D, dtype, False, False)
    plan = xa.attention_plan(torch.tensor(counts, device=DEV))
    gaps = []
    for x in parts:
        wide = torch.full((*x.shape[:2], D + 9), float("nan"), dtype=dtype, device=DEV)
        wide[..., :D] = x.to(DEV)
        gaps.append(wide[..., :D].detach().requires_grad_(True))
    for mask in (None, torch.arange(sum(counts), device=DEV) % 3 != 0):
        got = []
        for qkv in (dev, gaps):
            out = xa.structure_attention(*qkv, plan, mask=mask)
            got.append((out, *torch.autograd.grad(out, qkv, grad.to(DEV))))
        for a, b in zip(*got):
            assert a.isfinite().all() and torch.equal(a, b)


def test_the_operators_repeat_bit_for_bit_on_any_stream():
    import xnn_amd as xa
    gen = torch.Generator().manual_seed(6)
    counts = torch.tensor([700, 300, 21], device=DEV)
    T, H, D = 1021, 4, 32
    ids = torch.randint(0, 9, (T,), generator=gen).to(DEV)
    table = _normal(gen, 9, H * D).to(DEV).requires_grad_(True)
    angle = torch.rand(T, D // 2, generator=gen).to(DEV).requires_grad_(True)
    w = torch.ones(D, device=DEV, requires_grad=True)

    def block():
        plan = xa.attention_plan(counts)
        x = xa.embedding(ids, table, 0.7)
        h = x.view(T, H, D)
        q, k = xa.head_norm_rotate(h, h, w, w, angle.cos(), angle.sin())
        y = xa.dropout_add(xa.structure_attention(q, k, h, plan).reshape(T, -1), x, 0.1, 1, 2)
        return (y.detach(), *torch.autograd.grad(y.square().sum(), (table, angle, w)))
    first = block()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = block()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_the_operators_replay_from_a_graph():
    """Captured once, replayed with new inputs between eager work; the dropout counter advances
    between the replays."""
    import xnn_amd as xa
    T, H, D = 130, 2, 16
    plan = xa.attention_plan(torch.tensor([100, 30], device=DEV))
    ids = torch.zeros(T, dtype=torch.int64, device=DEV)
    table = torch.randn(9, H * D, device=DEV, requires_grad=True)
    w = torch.ones(D, device=DEV, requires_grad=True)
    angle = torch.rand(T, D // 2, device=DEV)
    cos, sin = angle.cos(), angle.sin()
    counter = torch.zeros(1, dtype=torch.int64, device=DEV)

    def step():
        x = xa.embedding(ids, table, 0.7)
        h = x.view(T, H, D)
        q, k = xa.head_norm_rotate(h, h, w, w, cos, sin)
        y = xa.dropout_add(xa.structure_attention(q, k, h, plan).reshape(T, -1), x, 0.3, 1, counter)
        return (y, *torch.autograd.grad(y, (table, w), x.detach()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for r in range(4):
        ids.copy_(torch.randint(0, 9, (T,), device=DEV))
        counter.fill_(100 + r)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_gradients_with_saved_tensors_kept_elsewhere():
    """Saved tensors packed to the host and brought back to other memory (offloading hooks)."""
    import xnn_amd as xa
    plan = xa.attention_plan(torch.tensor([30, 34], device=DEV))
    w = torch.ones(16, device=DEV, requires_grad=True)
    ids = torch.arange(64, device=DEV) % 5
    table = torch.randn(5, 96, device=DEV, requires_grad=True)
    angle = torch.rand(64, 8, device=DEV)

    def step():
        x = xa.embedding(ids, table, 1.0).view(64, 6, 16)
        q, k = xa.head_norm_rotate(x[:, :2], x[:, 2:4], w, w, angle.cos(), angle.sin())
        y = xa.dropout_add(xa.structure_attention(q, k, x[:, 4:], plan), q, 0.2, 1, 2)
        return y
    y = step()
    want = torch.autograd.grad(y, (table, w), torch.ones_like(y))
    with torch.autograd.graph.save_on_cpu():
        y = step()
    junk = [torch.full((64, 96), float("nan"), device=DEV) for _ in range(64)]
    got = torch.autograd.grad(y, (table, w), torch.ones_like(y))
    del junk
    for a, b in zip(want, got):
        assert torch.equal(a, b)


# --------------------------------------------------------------------------- refusals
def test_refusals():
    import xnn_amd as xa
    q = torch.randn(10, 4, 16, device=DEV)
    k = torch.randn(10, 2, 16, device=DEV)
    plan = xa.attention_plan(torch.tensor([4, 6], device=DEV))
    mask = torch.ones(10, dtype=torch.bool, device=DEV)
    bad = [
        (ValueError, lambda: xa.attention_plan(torch.tensor([4, -1], device=DEV), 3)),
        (ValueError, lambda: xa.attention_plan(torch.tensor([4, 5], device=DEV), 10)),
        (ValueError, lambda: xa.attention_plan(torch.tensor([4.0], device=DEV))),
        (RuntimeError, lambda: xa.attention_plan(torch.tensor([4]))),
        (ValueError, lambda: xa.structure_attention(q[:9], k[:9], k[:9], plan)),
        (ValueError, lambda: xa.structure_attention(q[:, :3], k, k, plan)),
        (ValueError, lambda: xa.structure_attention(q, k, k[:, :1], plan)),
        (ValueError, lambda: xa.structure_attention(q, k, k, plan, mask=mask[:9])),
        (ValueError, lambda: xa.structure_attention(q, k, k, plan, mask=mask.float())),
        (ValueError, lambda: xa.structure_attention(q, k, k, plan, scale=0.0)),
        (ValueError, lambda: xa.structure_attention(q, k, k, plan, scale=float("nan"))),
        (TypeError, lambda: xa.structure_attention(q, k.half(), k.half(), plan)),
        (TypeError, lambda: xa.structure_attention(q.double(), k.double(), k.double(), plan)),
        (RuntimeError, lambda: xa.structure_attention(q.cpu(), k, k, plan)),
        (ValueError, lambda: xa.structure_attention(*(torch.randn(10, 1, 129, device=DEV),) * 3, plan)),
        (TypeError, lambda: xa.embedding(torch.zeros(3, device=DEV), q[0])),
        (ValueError, lambda: xa.embedding(torch.zeros(3, dtype=torch.int64, device=DEV), q)),
        (TypeError, lambda: xa.embedding(torch.zeros(3, dtype=torch.int64, device=DEV), q[0].double())),
        (ValueError, lambda: xa.dropout_add(q, None, 1.5, 0)),
        (ValueError, lambda: xa.dropout_add(q, k, 0.5, 0)),
        (ValueError, lambda: xa.dropout_add(q, None, 0.5, 0, torch.zeros(2, dtype=torch.int64, device=DEV))),
    ]
    w, t = torch.ones(16, device=DEV), torch.ones(10, 8, device=DEV)
    pos = torch.zeros(10, dtype=torch.int64, device=DEV)
    bad += [
        (ValueError, lambda: xa.head_norm_rotate(q, k, w, w, t[:9], t[:9])),
        (ValueError, lambda: xa.head_norm_rotate(q, k, w, w, torch.ones(10, 9, device=DEV), torch.ones(10, 9, device=DEV))),
        (TypeError, lambda: xa.head_norm_rotate(q, k, w, w, t.half(), t.half())),
        (TypeError, lambda: xa.head_norm_rotate(q, k, w.half(), w, t, t)),
        (ValueError, lambda: xa.head_norm_rotate(q, k, w[:8], w, t, t)),
        (ValueError, lambda: xa.head_norm_rotate(q, k, w, w, t, t, positions=pos[:3])),
        (ValueError, lambda: xa.head_norm_rotate(q, k, w, w, t.clone().requires_grad_(True), t, positions=pos)),
    ]
    for error, call in bad:
        with pytest.raises(error):
            call()
    out = xa.structure_attention(q.requires_grad_(True), k, k, plan)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(out.sum(), q, create_graph=True)
