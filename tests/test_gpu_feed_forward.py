"""The feed-forward operators over atoms on the GPU against the same operations in float64.

A result is off by its own rounding (half a step of the type, u) and by what the operator documents: float32
sums, the products of float32 operands left out of the planes (2^-23 of each product) and, in 16 bits, the
form in which f'(z) is kept and the rounding of d = grad f'(z). The bounds below add these up over each output's own terms."""
import math

import numpy as np
import pytest
import torch

import xnn_amd as xa

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
FUNCTIONS = {None: lambda z: z, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
             "tanh": torch.tanh}
TINY = {"f32": 2.0 ** -126, "bf16": 2.0 ** -126, "f16": 2.0 ** -24}


def _u(dtype):
    """Half a step of the type, relative."""
    return torch.finfo(TYPES[dtype]).eps / 2


def _term(dtype, n):
    """Error of a sum of ``n`` products, of the sum of their sizes: float32 partial sums in any order, and in
    float32 the planes' products that are left out."""
    return (n + 8) * 2.0 ** -24 + (2.0 ** -22 if dtype == "f32" else 0.0)


def _random(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen) * scale).to(TYPES[dtype]).to(DEV)


def _close(got, want, bound, what):
    got, err = got.double(), (got.double() - want).abs()
    assert got.isfinite().all(), what
    worst = float((err / bound.clamp_min(1e-300)).max()) if err.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} of the bound"


# --------------------------------------------------------------------------- layer norm
def _norm_case(dtype, rows, width, affine=True, strided=False, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = _random(gen, (rows, width + (5 if strided else 0)), dtype) * 2 + 1
    x = x[:, 3:3 + width] if strided else x
    w, b = (1 + 0.2 * _random(gen, (width,), dtype), _random(gen, (width,), dtype)) if affine else (None, None)
    return x, w, b, _random(gen, (rows, width), dtype)


def _check_norm(dtype, x, w, b, g, eps=1e-5):
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, w, b)]
    out = xa.layer_norm(*leaves, eps=eps)
    grads = torch.autograd.grad(out, [t for t in leaves if t is not None], g)
    dbl = [None if t is None else t.detach().double().requires_grad_(True) for t in (x, w, b)]
    y, wd, bd = dbl
    mean = y.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((y - mean).square().mean(-1, keepdim=True) + eps)
    n = (y - mean) * r
    ref = n if wd is None else n * wd + bd
    want = torch.autograd.grad(ref, [t for t in dbl if t is not None], g.double())
    C, T, u, s = x.shape[-1], x.numel() // x.shape[-1], _u(dtype), 2.0 ** -24
    with torch.no_grad():
        # The mean of C values is off by (C + 2) s of the mean of their sizes (a thread's sums are far shorter than
        # C), and r by (C + 8) s and the mean's share of it; n carries both
        k = (min(C, 64) + 16) * s
        size = (y.abs().mean(-1, keepdim=True) + y.abs()) * r
        dn = k * (size + n.abs() * (1 + size))
        one = torch.ones_like(n) if wd is None else wd.abs()
        bound = u * ref.abs() + 4 * s * ((n * one).abs() + (0 if bd is None else bd.abs())) + dn * one + TINY[dtype]
        _close(out, ref, bound, "output")
        gw = g.double() * (1 if wd is None else wd)
        m1, m2 = gw.abs().mean(-1, keepdim=True), (gw * n).abs().mean(-1, keepdim=True)
        e2 = (gw.abs() * dn).mean(-1, keepdim=True) + k * m2
        d = r * (k * (gw.abs() + m1) + n.abs() * e2 + dn * m2 + 8 * s * (gw.abs() + m1 + n.abs() * m2))
        d = d + want[0].abs() * (u + k * (1 + size)) + TINY[dtype]
        _close(grads[0], want[0], d, "dx")
        if w is None:
            return
        gn = (g.double() * n).abs().reshape(T, C).sum(0)
        gdn = (g.double().abs() * dn).reshape(T, C).sum(0)
        rows = (min(T, 2048) + 16) * s
        _close(grads[1], want[1], u * want[1].abs() + rows * gn + gdn + TINY[dtype], "dw")
        _close(grads[2], want[2], u * want[2].abs() + rows * g.double().abs().reshape(T, C).sum(0) + TINY[dtype], "db")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 2), (3, 7), (21, 128), (64, 64), (130, 65), (7, 511), (33, 1000),
                                        (300, 256), (5, 4097), (3, 8192), (2, 9001), (2, 16384), (5000, 33)])
def test_layer_norm(dtype, rows, width):
    _check_norm(dtype, *_norm_case(dtype, rows, width))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", [(1, 5), (40, 64), (9, 513), (2000, 130)])
def test_layer_norm_of_a_part_of_wider_rows_and_without_weights(dtype, rows, width):
    _check_norm(dtype, *_norm_case(dtype, rows, width, strided=True))
    _check_norm(dtype, *_norm_case(dtype, rows, width, affine=False, strided=True))


def test_layer_norm_of_more_dimensions():
    x, w, b, g = _norm_case("f32", 24, 16)
    out = xa.layer_norm(x.view(2, 3, 4, 16), w, b)
    assert out.shape == (2, 3, 4, 16) and torch.equal(out.view(24, 16), xa.layer_norm(x, w, b))
    assert torch.equal(xa.layer_norm(x[0], w, b), xa.layer_norm(x, w, b)[0])
    moved = x.t().contiguous().t()
    assert torch.equal(xa.layer_norm(moved, w, b), xa.layer_norm(x, w, b))
    assert torch.equal(xa.layer_norm(x[:1].expand(24, 16), w, b), xa.layer_norm(x[:1], w, b).expand(24, 16))


def test_layer_norm_of_no_rows_and_single_gradients():
    x, w, b, g = _norm_case("f32", 40, 24)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    full = torch.autograd.grad(xa.layer_norm(*leaves), leaves, g)
    for i, leaf in enumerate(leaves):
        args = [t.detach() for t in (x, w, b)]
        args[i] = leaf
        alone, = torch.autograd.grad(xa.layer_norm(*args), leaf, g)
        assert torch.equal(alone, full[i])
    empty = x[:0].detach().requires_grad_(True)
    out = xa.layer_norm(empty, *leaves[1:])
    grads = torch.autograd.grad(out, (empty, *leaves[1:]), g[:0])
    assert out.shape == (0, 24) and grads[0].shape == (0, 24)
    assert all(not t.any() for t in grads[1:])


def test_layer_norm_of_a_constant_row_and_of_large_offsets():
    """The squares are of the centered values: an offset far above the spread costs what its own rounding costs."""
    x = torch.full((3, 512), 7.25, device=DEV)
    assert not xa.layer_norm(x).any()
    x = torch.randn(64, 512, generator=torch.Generator().manual_seed(1)).to(DEV) + 1000.0
    y = x.double()
    want = (y - y.mean(1, keepdim=True)) / torch.sqrt(y.var(1, unbiased=False, keepdim=True) + 1e-5)
    assert float((xa.layer_norm(x).double() - want).abs().max()) < 1000 * 16 * 2.0 ** -24
    x[5, 17] = float("nan")
    bad = xa.layer_norm(x).isnan().any(1)
    assert bad[5] and int(bad.sum()) == 1


# --------------------------------------------------------------------------- dense layers
def _dense_case(dtype, rows, n_in, n_out, groups=None, bias=True, residual=False, strided=False, seed=0, some=None):
    gen = torch.Generator().manual_seed(seed)
    x = _random(gen, (rows, n_in + (3 if strided else 0)), dtype)
    x = x[:, 1:1 + n_in] if strided else x
    lead = () if groups is None else (groups,)
    w = _random(gen, lead + (n_in, n_out), dtype, n_in ** -0.5)
    b = _random(gen, lead + (n_out,), dtype) if bias else None
    r = _random(gen, (rows, n_out), dtype) if residual else None
    g = _random(gen, (rows, n_out), dtype)
    ids = None
    if groups is not None:
        ids = torch.randint(0, groups, (rows,), generator=gen)
        if some is not None:                                # the groups that have rows; -1: none
            ids = torch.tensor(some)[torch.randint(0, len(some), (rows,), generator=gen)]
        ids = ids.to(DEV)
    return x, w, b, r, g, ids


def _check_dense(dtype, case, activation):
    x, w, b, r, g, ids = case
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, w, b, r)]
    if ids is None:
        out = xa.linear(*leaves[:3], activation, leaves[3])
    else:
        plan = xa.group_plan(ids, w.shape[0])
        out = xa.grouped_linear(leaves[0], leaves[1], plan, leaves[2], activation, leaves[3])
    grads = list(torch.autograd.grad(out, [t for t in leaves if t is not None], g))
    out = out.detach()
    K, N, u = x.shape[1], w.shape[-1], _u(dtype)
    tiny = TINY[dtype]
    seen = torch.zeros(len(x), dtype=torch.bool, device=DEV)
    for group in range(1 if ids is None else w.shape[0]):
        rows = torch.arange(len(x), device=DEV) if ids is None else (ids == group).nonzero()[:, 0]
        seen[rows] = True
        xd, wd = x[rows].double(), (w if ids is None else w[group]).double()
        bd = None if b is None else (b if ids is None else b[group]).double()
        z = (xd @ wd + (0 if bd is None else bd)).requires_grad_(True)
        y = FUNCTIONS[activation](z)
        slope, = torch.autograd.grad(y.sum(), z)
        y, z = y.detach(), z.detach()
        want = y if r is None else y + r[rows].double()
        # z, then f (Lipschitz to 1.13, evaluated to a few float32 steps of its size), the residual and the rounding
        dz = _term(dtype, K) * (xd.abs() @ wd.abs() + (0 if bd is None else bd.abs()))
        f32 = 0.0 if activation is None else 2.0 ** -21
        bound = 1.2 * dz + f32 * (1 + z.abs()) + (u + 2.0 ** -23) * want.abs() + 2.0 ** -23 * y.abs() + tiny
        _close(out[rows], want, bound, f"output of {group}")
        gd = g[rows].double()
        d = gd * slope
        # f' changes by at most |f''| <= 1. It is kept in float16 beside bfloat16; beside float16 its root is, in units
        # of 1 / 30,000, so it is off by 2 root(f') e + e^2 with e half a unit. d is rounded to the type
        e = 0.0 if activation is None or dtype != "f16" else 1.01 / 60000
        kept = 2 * e * slope.abs().sqrt() + e * e
        if dtype == "bf16" and activation is not None:
            kept = 2.0 ** -11 * slope.abs() + 2.0 ** -24
        dd = gd.abs() * (dz + f32 * (1 + z.abs()) + kept)
        dd = dd + (0 if activation is None else u * d.abs() + tiny)
        dx = d @ wd.t()
        _close(grads[0][rows], dx, _term(dtype, N) * (d.abs() @ wd.abs().t()) + dd @ wd.abs().t() + u * dx.abs() + tiny,
               f"dx of {group}")
        dw = xd.t() @ d
        n = min(len(rows), 4096) + 64
        got = grads[1] if ids is None else grads[1][group]
        _close(got, dw, _term(dtype, n) * (xd.abs().t() @ d.abs()) + xd.abs().t() @ dd + u * dw.abs() + tiny,
               f"dw of {group}")
        if b is not None:
            got = grads[2] if ids is None else grads[2][group]
            db = d.sum(0)
            _close(got, db, n * 2.0 ** -24 * d.abs().sum(0) + dd.sum(0) + u * db.abs() + tiny, f"db of {group}")
    if r is not None:
        assert torch.equal(grads[-1], g)
    assert out[~seen].isnan().all() and not grads[0][~seen].any()


@pytest.mark.parametrize("n_in", [40, 300])
def test_slopes_far_from_one_keep_their_digits_in_bfloat16(n_in):
    """silu at z = -10 -+ 2: f' of 1e-3 to 1e-5, its error half a float16 step of it (2^-11) and, of the exponential,
    |z| 2^-23 and two roundings of z itself; d and dx are rounded to the type."""
    gen = torch.Generator().manual_seed(n_in)
    x, g = _random(gen, (200, n_in), "bf16"), _random(gen, (200, 96), "bf16")
    w = _random(gen, (n_in, 96), "bf16", 0.5 * n_in ** -0.5)
    b = torch.full((96,), -10.0, device=DEV, dtype=torch.bfloat16)
    leaf = x.detach().requires_grad_(True)
    got, = torch.autograd.grad(xa.linear(leaf, w, b, "silu"), leaf, g)
    z = (x.double() @ w.double() - 10).requires_grad_(True)
    slope, = torch.autograd.grad(torch.nn.functional.silu(z).sum(), z)
    z = z.detach()
    d = g.double() * slope
    dz = _term("bf16", n_in) * (x.double().abs() @ w.double().abs() + 10)
    dd = d.abs() * (2.0 ** -11 + 2.0 ** -8 + z.abs() * 2.0 ** -22 + 4 * 2.0 ** -24 + 2 * dz) * 1.01
    dx = d @ w.double().t()
    bound = dd @ w.double().abs().t() + _term("bf16", 96) * (d.abs() @ w.double().abs().t()) + 2.0 ** -8 * dx.abs()
    _close(got, dx, bound, "dx")


SHAPES = [(1, 1, 1), (1, 8, 8), (1, 1024, 4096), (5, 3, 7), (2, 64, 1), (21, 128, 512), (64, 64, 64), (65, 129, 33),
          (300, 250, 511), (257, 40, 300), (31, 512, 17), (1000, 17, 129)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n_in,n_out", SHAPES)
def test_linear(dtype, rows, n_in, n_out):
    activation = [None, "silu", "gelu", "tanh"][(rows + n_in) % 4]
    _check_dense(dtype, _dense_case(dtype, rows, n_in, n_out, residual=rows % 2 == 1), activation)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", FUNCTIONS)
@pytest.mark.parametrize("bias", [True, False])
def test_linear_activations(dtype, activation, bias):
    _check_dense(dtype, _dense_case(dtype, 100, 48, 72, bias=bias, residual=bias), activation)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n_in,n_out", [(4300, 72, 1000), (4300, 1000, 72), (16700, 40, 1030), (16700, 1030, 40),
                                             (33000, 65, 300), (6000, 512, 128), (70001, 24, 20)])
def test_linear_of_many_tiles(dtype, rows, n_in, n_out):
    _check_dense(dtype, _dense_case(dtype, rows, n_in, n_out, residual=n_in == 72), "silu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 9])
@pytest.mark.parametrize("n_in,n_out", [(1, 3), (33, 1000), (1500, 65), (5000, 40), (64, 2100)])
def test_linear_of_few_rows(dtype, rows, n_in, n_out):
    _check_dense(dtype, _dense_case(dtype, rows, n_in, n_out, residual=rows % 2 == 0, strided=rows == 5), "silu")
    _check_dense(dtype, _dense_case(dtype, rows, n_in, n_out, 3, some=[-1, 0, 2], bias=rows != 4), None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n_in,n_out", [(1, 4096, 70), (3, 70, 4097), (100, 3001, 130), (130, 200, 2900),
                                             (64, 1030, 1030)])
def test_linear_of_long_sums_for_few_outputs(dtype, rows, n_in, n_out):
    _check_dense(dtype, _dense_case(dtype, rows, n_in, n_out, residual=True), "tanh")
    _check_dense(dtype, _dense_case(dtype, rows, n_in, n_out, 5, some=[-1, 1, 1, 4]), "gelu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n_in,n_out", [(1, 5, 3), (70, 64, 64), (129, 33, 65)])
def test_linear_of_a_part_of_wider_rows(dtype, rows, n_in, n_out):
    _check_dense(dtype, _dense_case(dtype, rows, n_in, n_out, strided=True), "gelu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n_in,n_out,groups,some", [
    (1, 8, 8, 1, None), (1, 7, 5, 3, [1]), (21, 128, 512, 9, [1, 6, 7, 8]), (100, 16, 24, 5, [4]), (300, 33, 65, 40, None),
    (1000, 65, 130, 3, [2, 0]), (64, 8, 8, 4096, None), (50, 12, 20, 4, [-1, 4, 9000000000, 2]), (30, 8, 8, 2, [-1]),
    (9000, 128, 512, 9, [1, 8]), (5000, 250, 511, 119, [1, 6, 7, 8, 16, 17])])
def test_grouped_linear(dtype, rows, n_in, n_out, groups, some):
    activation = ["silu", None][rows % 2]
    _check_dense(dtype, _dense_case(dtype, rows, n_in, n_out, groups, residual=groups % 2 == 0, some=some), activation)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n_in,n_out", [(33000, 72, 300), (70000, 24, 130), (9000, 1030, 1000)])
def test_grouped_linear_of_many_tiles(dtype, rows, n_in, n_out):
    _check_dense(dtype, _dense_case(dtype, rows, n_in, n_out, 7, some=[0, 0, 0, 1, 1, 3, 6], strided=True), "silu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("groups", [62, 63, 64, 65, 254, 255, 256, 257, 300])
def test_grouped_linear_of_as_many_groups_as_lanes(dtype, groups):
    """Tiles are found in lists of up to a wave's lanes, up to four of them, and longer ones."""
    some = [0, 1, groups - 1, groups - 1, groups - 1, groups // 2, -1, groups]
    _check_dense(dtype, _dense_case(dtype, 700, 40, 72, groups, residual=True, some=some), "gelu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_in,n_out", [(256, 1024), (130, 900), (100, 520)])
def test_grouped_linear_of_uneven_groups_with_many_parts(dtype, n_in, n_out):
    """The weight's gradient in parts of different lengths, a weight's tiles a multiple of the dies and not."""
    some = [3] * 30 + [20] * 18 + list(range(4, 20)) + [-1]
    _check_dense(dtype, _dense_case(dtype, 12000, n_in, n_out, 24, some=some), "silu")


def test_a_row_that_is_not_finite_reaches_no_other():
    for dtype in TYPES:
        x, w, b, r, g, ids = _dense_case(dtype, 200, 70, 90, 4)
        plan = xa.group_plan(ids, 4)
        want = xa.grouped_linear(x, w, plan, b)
        x[7] = float("nan")
        x[8, 69] = float("inf")
        got = xa.grouped_linear(x, w, plan, b)
        keep = torch.ones(200, dtype=torch.bool, device=DEV)
        keep[7:9] = False
        assert torch.equal(got[keep], want[keep]) and not got[~keep].isfinite().any()
        # a weight that is not finite stays with its group
        w[2] = float("nan")
        got = xa.grouped_linear(x, w, plan, b)
        keep &= ids != 2
        assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 2, 3, 70])
@pytest.mark.parametrize("n_in", [1, 2, 10, 33, 1000, 4097])
def test_an_infinite_input_gives_infinities_of_its_weights_signs(dtype, rows, n_in):
    """In 16 bits products are the type's own: an infinity in the last place of the sum meets no zero."""
    x, w, _, _, _, _ = _dense_case(dtype, rows, n_in, 40, bias=False)
    w = torch.where(w == 0, torch.ones_like(w), w)
    x[:, -1] = math.inf
    assert torch.equal(xa.linear(x, w), (w[-1].sign() * math.inf).expand(rows, 40))


def test_what_lies_around_the_operands_is_not_read_into_sums():
    """Rows of a tensor that ends where they end, amid NaN: odd widths, whose 16-byte pieces reach beyond a row."""
    for dtype in TYPES:
        for rows, n_in, n_out in [(3, 5, 7), (67, 33, 65), (130, 129, 127)]:
            x, w, b, r, g, _ = _dense_case(dtype, rows, n_in, n_out, residual=True)

            def amid(t):
                wide = torch.full((t.numel() + 64,), float("nan"), dtype=t.dtype, device=DEV)
                wide[31:31 + t.numel()] = t.flatten()
                return wide[31:31 + t.numel()].view(t.shape)
            args = [amid(t) for t in (x, w, b, r)]
            leaves = [t.detach().requires_grad_(True) for t in (x, w, b, r)]
            others = [t.detach().requires_grad_(True) for t in args]
            out, got = (xa.linear(*a[:3], "silu", a[3]) for a in (leaves, others))
            assert torch.equal(out, got)
            for a, c in zip(torch.autograd.grad(out, leaves, g), torch.autograd.grad(got, others, amid(g))):
                assert torch.equal(a, c)


def test_linear_of_no_rows_and_single_gradients():
    x, w, b, r, g, _ = _dense_case("f32", 90, 24, 40, residual=True)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b, r)]
    full = torch.autograd.grad(xa.linear(*leaves[:3], "silu", leaves[3]), leaves, g)
    for i, leaf in enumerate(leaves):
        args = [t.detach() for t in (x, w, b, r)]
        args[i] = leaf
        alone, = torch.autograd.grad(xa.linear(*args[:3], "silu", args[3]), leaf, g)
        assert torch.equal(alone, full[i])
    empty = x[:0].detach().requires_grad_(True)
    grads = torch.autograd.grad(xa.linear(empty, *leaves[1:3]), (empty, *leaves[1:3]), g[:0])
    assert grads[0].shape == (0, 24) and not grads[1].any() and not grads[2].any()
    ids = torch.zeros(0, dtype=torch.int64, device=DEV)
    w3, b3 = (t.detach()[None].expand(3, *t.shape).contiguous().requires_grad_(True) for t in (w, b))
    grads = torch.autograd.grad(xa.grouped_linear(empty, w3, xa.group_plan(ids, 3), b3), (empty, w3, b3), g[:0])
    assert grads[0].shape == (0, 24) and not grads[1].any() and not grads[2].any()


def test_linear_of_more_dimensions_and_transposed_weights():
    x, w, b, r, g, _ = _dense_case("bf16", 24, 16, 32, residual=True)
    want = xa.linear(x, w, b, "gelu", r)
    got = xa.linear(x.view(2, 3, 4, 16), w, b, "gelu", r.view(2, 3, 4, 32))
    assert got.shape == (2, 3, 4, 32) and torch.equal(got.view(24, 32), want)
    assert torch.equal(xa.linear(x, w.t().contiguous().t(), b, "gelu", r), want)
    assert torch.equal(xa.linear(x.t().contiguous().t(), w, b, "gelu", r), want)


def test_gradients_against_differences():
    """Along a direction, in float32: the slope of sum(cos(out)) by central differences of the float64 formula."""
    x, w, b, r, g, ids = _dense_case("f32", 30, 12, 20, 3, residual=True)
    plan = xa.group_plan(ids, 3)
    nw, nb = 1 + 0.1 * torch.randn(12, device=DEV), 0.1 * torch.randn(12, device=DEV)
    leaves = [t.detach().requires_grad_(True) for t in (x, nw, nb, w, b, r)]

    def energy(x, nw, nb, w, b, r):
        n = (x - x.mean(-1, keepdim=True)) / torch.sqrt(x.var(-1, unbiased=False, keepdim=True) + 1e-5)
        z = torch.einsum("tk,tkn->tn", n * nw + nb, w[ids]) + b[ids]
        return torch.cos(torch.nn.functional.silu(z) + r).sum()
    out = xa.grouped_linear(xa.layer_norm(*leaves[:3]), leaves[3], plan, leaves[4], "silu", leaves[5])
    grads = torch.autograd.grad(out, leaves, -torch.sin(out).detach())
    gen = torch.Generator().manual_seed(9)
    for i, leaf in enumerate(leaves):
        step = torch.randn(leaf.shape, generator=gen, dtype=torch.float64).to(DEV)
        at = [[t.detach().double() for t in leaves] for _ in range(2)]
        at[0][i] = at[0][i] + 1e-5 * step
        at[1][i] = at[1][i] - 1e-5 * step
        slope = float((energy(*at[0]) - energy(*at[1])) / 2e-5)
        got = float((grads[i].double() * step).sum())
        assert abs(got - slope) <= 1e-4 * float((grads[i].double() * step).abs().sum()), i


# --------------------------------------------------------------------------- plans
@pytest.mark.parametrize("rows,groups", [(0, 3), (1, 1), (63, 2), (1000, 9), (5000, 119), (20000, 4096), (70001, 300)])
def test_group_plan(rows, groups):
    rng = np.random.default_rng(rows)
    ids = rng.integers(-1, groups + 1, size=rows)
    for dtype in (torch.int64, torch.int32):
        plan = xa.group_plan(torch.from_numpy(ids).to(DEV).to(dtype), groups)
        got = plan.rows.cpu().numpy()
        bucket = np.where((ids < 0) | (ids >= groups), groups, ids)
        assert (plan.n_rows, plan.n_groups) == (rows, groups)
        assert np.array_equal(got[:rows], np.argsort(bucket, kind="stable"))
        counts = np.bincount(bucket, minlength=groups + 1)
        lists = got[rows:].reshape(53, groups + 2)
        assert np.array_equal(lists[0], np.concatenate([[0], np.cumsum(counts)]))
        sizes = [32, 64, 128, 256] + [(256 << o) // 4 * q for o in range(12) for q in (5, 6, 7, 8)]
        for level, size in enumerate(sizes):
            tiles = -(-counts // size)
            assert np.array_equal(lists[1 + level], np.concatenate([[0], np.cumsum(tiles)])), level


@pytest.mark.parametrize("rows,groups", [(2, 3), (2, 200), (300, 3), (300, 200), (5000, 70)])
def test_a_plan_of_other_numbers_reaches_nothing_outside(rows, groups):
    """The registered operators take a plan as it is given: every index of it is held to the rows and groups."""
    gen = torch.Generator().manual_seed(rows)
    for dtype in ("f32", "bf16"):
        x, w, b, r, g, ids = _dense_case(dtype, rows, 72, 130, groups, residual=True)
        plan = xa.group_plan(ids, groups)
        want = xa.grouped_linear(x, w, plan, b, "silu", r)
        around = [torch.full((1 << 16,), 5.0, device=DEV) for _ in range(8)]
        n = plan.rows.numel()
        for bad in (torch.full((n,), -1), torch.full((n,), 2 ** 31 - 1), torch.full((n,), -2 ** 31),
                    torch.arange(n, 0, -1), torch.randint(-2 ** 31, 2 ** 31 - 1, (n,), generator=gen),
                    torch.randint(-3, 2 * rows, (n,), generator=gen)):
            bad = bad.to(torch.int32).to(DEV)
            out, slope = torch.ops.xnn_amd.dense_slope(x, w, b, 1, r, bad)
            dx, dw, db = torch.ops.xnn_amd.dense_backward(g, slope, x, w, bad, True, True, True)
            torch.cuda.synchronize()
            assert out.shape == want.shape and dx.shape == x.shape and dw.shape == w.shape and db.shape == b.shape
        assert all((t == 5.0).all() for t in around)
        assert torch.equal(xa.grouped_linear(x, w, plan, b, "silu", r), want)


def test_the_species_plan_is_kept_with_the_graph():
    from xnn_amd import synthetic
    g = xa.structure_to_graph(synthetic.random_molecules(1, seed=2)[0].as_dict(), 4.0).to(DEV)
    plan = g.species_plan(9)
    assert g.species_plan(9) is plan and g.species_plan(10) is not plan
    plan = g.species_plan(9)
    g.atomic_numbers[0] = 1
    assert g.species_plan(9) is not plan


def test_a_species_plan_that_a_capture_makes_is_not_kept():
    """Its rows are there once the graph is replayed, and in the graph's memory; one that is kept serves a capture, and
    another stream makes its own."""
    from xnn_amd import synthetic
    g = xa.structure_to_graph(synthetic.random_molecules(1, seed=2)[0].as_dict(), 4.0).to(DEV)
    want = xa.group_plan(g.atomic_numbers, 9).rows
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = g.species_plan(9)
    plan = g.species_plan(9)
    assert plan is not inside and torch.equal(plan.rows, want)
    for _ in range(3):
        inside.rows.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(inside.rows, want) and g.species_plan(9) is plan
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert g.species_plan(9) is plan
        rows = plan.rows + 1
    graph.replay()
    assert torch.equal(rows, want + 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = g.species_plan(9)
        assert other is not plan and g.species_plan(9) is other
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other.rows, want)


# --------------------------------------------------------------------------- streams, graphs, refusals
def test_the_same_bits_at_every_call_and_on_another_stream():
    x, w, b, r, g, ids = _dense_case("bf16", 5000, 128, 256, 5, residual=True)
    plan = xa.group_plan(ids, 5)

    def once():
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b, r)]
        out = xa.grouped_linear(leaves[0], leaves[1], plan, leaves[2], "gelu", leaves[3])
        y = xa.layer_norm(out)
        return [out.detach(), y.detach(), *torch.autograd.grad(y, leaves, g)]
    want = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = once()
    torch.cuda.current_stream().wait_stream(side)
    for a, c, d in zip(want, got, once()):
        assert torch.equal(a, c) and torch.equal(a, d)


def test_two_streams_at_once():
    """Calls in flight on two streams, forward and backward, share no workspace and no state."""
    cases = [_dense_case("f32", 3000, 256, 96, 6, residual=True, seed=1), _dense_case("bf16", 40, 4096, 64, 3, seed=2)]

    def once(case):
        x, w, b, r, g, ids = case
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        out = xa.grouped_linear(leaves[0], leaves[1], xa.group_plan(ids, w.shape[0]), leaves[2], "silu", r)
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]
    want = [once(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(6):
        for case, stream, ref in zip(cases, streams, want):
            with torch.cuda.stream(stream):
                got.append((once(case), ref))
    torch.cuda.synchronize()
    for a, ref in got:
        for t, u in zip(a, ref):
            assert torch.equal(t, u)


def test_a_captured_step_replays_the_plan_the_layers_and_their_gradients():
    """Ids, inputs and cotangents change between the replays; every replay equals the eager result."""
    x, w, b, r, g, ids = _dense_case("f32", 700, 64, 96, 5, residual=True)
    nw = torch.ones(64, device=DEV)

    def step(x, ids, g, leaves):
        plan = xa.group_plan(ids, 5)
        out = xa.grouped_linear(xa.layer_norm(x, leaves[0]), leaves[1], plan, leaves[2], "silu", r)
        out = xa.linear(out, leaves[3], None, "tanh")
        return [out.detach(), *torch.autograd.grad(out, (x, *leaves), g)]
    w2 = _random(torch.Generator().manual_seed(3), (96, 64), "f32", 0.1)
    static = [x.clone().requires_grad_(True), ids.clone(), _random(torch.Generator().manual_seed(4), (700, 64), "f32")]
    leaves = [t.detach().requires_grad_(True) for t in (nw, w, b, w2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static, leaves)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static, leaves)
    for seed in range(4):
        gen = torch.Generator().manual_seed(20 + seed)
        with torch.no_grad():
            static[0].copy_(_random(gen, (700, 64), "f32"))
            static[1].copy_(torch.randint(-1, 5, (700,), generator=gen))
            static[2].copy_(_random(gen, (700, 64), "f32"))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        eager = [t.detach().requires_grad_(True) for t in leaves]
        want = step(static[0].detach().requires_grad_(True), static[1], static[2], eager)
        for a, c in zip(got, want):
            assert torch.equal(a.nan_to_num(7.0), c.nan_to_num(7.0))


def test_operands_of_more_than_4_GB():
    """Offsets beyond 32 bits: in rows of x and of the output, and in the weights of the last group."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    gen = torch.Generator(device=DEV).manual_seed(5)

    def rand(*shape):
        return torch.randn(shape, generator=gen, device=DEV, dtype=torch.bfloat16)
    pick = [0, 1, 65_535, 65_536, 130_999, 131_071, 139_998, 139_999]
    x = rand(140_000, 16_384)                               # 4.6 GB, 2.3e9 elements
    nw, nb = rand(16_384), rand(16_384)
    leaf = x.requires_grad_(True)
    out = xa.layer_norm(leaf, nw, nb)
    dx, = torch.autograd.grad(out, leaf, out.detach())
    part = x.detach()[pick].requires_grad_(True)
    alone = xa.layer_norm(part, nw, nb)
    assert torch.equal(out[pick], alone)
    assert torch.equal(dx[pick], torch.autograd.grad(alone, part, alone.detach())[0])
    del out, dx, alone, part
    w = rand(16_384, 40) / 128
    leaf = x.detach().requires_grad_(True)
    wl = w.detach().requires_grad_(True)
    out = xa.linear(leaf, wl, None, "silu")
    g = rand(140_000, 40)
    dx, dw = torch.autograd.grad(out, (leaf, wl), g)
    z = x.detach()[pick].double() @ w.double()
    u = 2.0 ** -8
    size = x.detach()[pick].double().abs() @ w.double().abs()
    dz = _term("bf16", 16_384) * size
    y = torch.nn.functional.silu(z)
    _close(out.detach()[pick], y, 1.2 * dz + 2.0 ** -21 * (1 + z.abs()) + (u + 2.0 ** -23) * y.abs(), "out")
    s = torch.sigmoid(z)
    d = g[pick].double() * s * (1 + z * (1 - s))
    dd = g[pick].double().abs() * (dz + 2.0 ** -21 * (1 + z.abs()) + 1.13 * 2.0 ** -11) + u * d.abs()
    ref = d @ w.double().t()
    _close(dx[pick], ref, dd @ w.double().abs().t() + _term("bf16", 40) * (d.abs() @ w.double().abs().t())
           + u * ref.abs(), "dx")
    # the weight's gradient: the rows behind the 32-bit offset alone, the others' cotangents zero
    g[:132_000] = 0
    dw, = torch.autograd.grad(xa.linear(leaf, wl), wl, g)
    tail, gt = x.detach()[132_000:].double(), g[132_000:].double()
    ref = tail.t() @ gt
    _close(dw, ref, _term("bf16", 8_000) * (tail.abs().t() @ gt.abs()) + u * ref.abs(), "dw")
    del x, leaf, out, dx, dw, tail, size
    w = rand(4096, 1024, 600)                               # 5 GB of weights
    ids = torch.tensor([4095, 0, 4095, 3500, 3600, 7], device=DEV)
    x, g, plan = rand(6, 1024), rand(6, 600), xa.group_plan(ids, 4096)
    wl, leaf = w.requires_grad_(True), x.requires_grad_(True)
    out = xa.grouped_linear(leaf, wl, plan)
    dx, dw = torch.autograd.grad(out, (leaf, wl), g)
    for i, group in enumerate(ids.tolist()):
        wd, xd, gd = w.detach()[group].double(), x.detach()[i].double(), g[i].double()
        ref = xd @ wd
        _close(out.detach()[i], ref, _term("bf16", 1024) * (xd.abs() @ wd.abs()) + u * ref.abs(), "grouped out")
        ref = gd @ wd.t()
        _close(dx[i], ref, _term("bf16", 600) * (gd.abs() @ wd.t().abs()) + u * ref.abs(), "grouped dx")
        rows = (ids == group).nonzero()[:, 0]
        ref = x.detach()[rows].double().t() @ g[rows].double()
        _close(dw[group], ref, 2.0 ** -20 * ref.abs() + u * ref.abs() + 2.0 ** -20, "grouped dw")
    assert not dw[1:7].any() and not dw[3601:4095].any()


def test_rows_behind_the_output_are_left():
    """Outputs are written row by row: what follows the last row in memory stays."""
    from xnn_amd import _lib
    for rows, n_out in [(1, 1), (65, 33), (130, 100)]:
        x, w, _, _, _, _ = _dense_case("f32", rows, 24, n_out)
        out = torch.full((rows * n_out + 256,), -7.0, device=DEV)
        _lib.call("xnn_linear", 0, x.data_ptr(), 24, rows, 24, n_out, w.data_ptr(), None, 0, None, None, 1,
                  out.data_ptr(), None, None, 0, _lib.stream(torch.device(DEV)))
        assert torch.equal(out[:rows * n_out].view(rows, n_out), xa.linear(x, w))
        assert (out[rows * n_out:] == -7.0).all()


def test_refusals():
    x, w, b, r, g, ids = _dense_case("f32", 12, 8, 16, 3)
    plan, w1 = xa.group_plan(ids, 3), w[0]
    for call, err, text in [
            (lambda: xa.linear(x, w1[:7]), ValueError, "weight must be"),
            (lambda: xa.linear(x, w), ValueError, "weight must be"),
            (lambda: xa.linear(x, w1.bfloat16()), TypeError, "weight is"),
            (lambda: xa.linear(x.double(), w1.double()), TypeError, "unsupported dtype"),
            (lambda: xa.linear(x, w1, b[0, :3]), ValueError, "bias must be"),
            (lambda: xa.linear(x, w1, b[0].half()), TypeError, "bias is"),
            (lambda: xa.linear(x, w1, None, None, r if r is not None else x), ValueError, "residual must be"),
            (lambda: xa.linear(x, w1.cpu()), RuntimeError, "GPU only"),
            (lambda: xa.linear(x[:, :0], w1[:0]), ValueError, "width at least 1"),
            (lambda: xa.linear(x, w1[:, :0]), ValueError, "weight must be"),
            (lambda: xa.grouped_linear(x, w1, plan), ValueError, "weight must be"),
            (lambda: xa.grouped_linear(x[:11], w, plan), ValueError, "the plan is not of 11 rows"),
            (lambda: xa.grouped_linear(x, w, plan, b[:2]), ValueError, "bias must be"),
            (lambda: torch.ops.xnn_amd.dense(x, w[:2], None, 0, None, plan.rows), ValueError, "not of 12 rows"),
            (lambda: torch.ops.xnn_amd.dense(x, w1, None, 9, None, None), ValueError, "unknown activation"),
            (lambda: xa.group_plan(ids.float(), 3), TypeError, "integers"),
            (lambda: xa.group_plan(ids[None], 3), ValueError, "ids must be"),
            (lambda: xa.group_plan(ids, 0), ValueError, "n_groups"),
            (lambda: xa.group_plan(ids, 5000), ValueError, "n_groups"),
            (lambda: xa.layer_norm(x, b[0]), ValueError, "weight must be"),
            (lambda: xa.layer_norm(x, None, x[0].half()), TypeError, "bias is"),
            (lambda: xa.layer_norm(x, eps=-1.0), ValueError, "eps"),
            (lambda: xa.layer_norm(x, eps=math.nan), ValueError, "eps"),
            (lambda: xa.layer_norm(x.long()), TypeError, "unsupported dtype"),
            (lambda: xa.layer_norm(torch.zeros(2, 16385, device=DEV)), ValueError, "width")]:
        with pytest.raises(err, match=text):
            call()
    with pytest.raises(NotImplementedError, match="forward-mode"):
        import torch.autograd.forward_ad as fwd
        with fwd.dual_level():
            xa.linear(fwd.make_dual(x, x), w1)
    leaf = x.detach().requires_grad_(True)
    for f in (lambda: xa.linear(leaf, w1, None, "silu"), lambda: xa.layer_norm(leaf)):
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(f().square().sum(), leaf, create_graph=True)
