"""Which variant of the dense layers' kernels a call of given sizes takes: the rules, on the host (no GPU needed), and on
the GPU the results of each of them against float64."""
import ctypes

import pytest

CODES = {"f32": 0, "bf16": 2, "f16": 3}
FIELDS = ("forward", "forward_parts", "input", "input_parts", "weight", "weight_parts", "weight_rows", "pass")


@pytest.fixture(scope="module")
def lib():
    from xnn_amd import _lib
    return _lib.load()


@pytest.mark.parametrize("dtype", [0, 2, 3])
@pytest.mark.parametrize("grouped", [0, 1])
def test_long_reductions_of_one_or_two_rows_are_cut_into_parts(lib, dtype, grouped):
    """A stream of the weight, which needs no workspace, up to 1,500 inputs; then tiles, whose parts have sums there."""
    size = ctypes.c_size_t()
    for rows in (1, 2):
        for n_in, parts in ((64, False), (1500, False), (4096, True), (8192, True)):
            assert lib.xnn_linear_work_size(dtype, rows, n_in, 1024, 1 + 2 * grouped, grouped, ctypes.byref(size)) == 0
            assert (size.value > 0) is parts, (rows, n_in)


def _variant(lib, dtype, rows, n_in, n_out, groups, slope):
    out = (ctypes.c_int32 * 8)()
    assert lib.xnn_linear_variants(CODES[dtype], rows, n_in, n_out, groups or 1, int(groups is not None), int(slope),
                                   out) == 0
    return dict(zip(FIELDS, out))


WATER, FEW, UNEVEN = [1, 1, 8], [-1, 3, 3, 3, 5], [0] * 20 + [1] * 9 + list(range(2, 30)) + [-1]
# type, rows, inputs, outputs, groups and those that have rows, activation, bias; rows of the tiles of the forward pass, of
# x's gradient and the weight's, whether the latter is in parts, whether a pass forms d
CASES = [
    ("f32", 40000, 128, 512, 9, WATER, "silu", True, 128, 128, 128, True, False),
    ("f32", 40000, 128, 512, None, None, "silu", True, 128, 128, 128, True, False),
    ("bf16", 40000, 128, 512, 9, WATER, "silu", True, 128, 128, 128, True, False),
    ("bf16", 72000, 128, 512, None, None, "silu", True, 128, 128, 128, True, False),
    ("f16", 40000, 127, 511, 9, WATER, "tanh", True, 128, 128, 128, True, False),
    ("f16", 72000, 127, 511, None, None, "tanh", False, 128, 128, 128, True, False),
    ("bf16", 40000, 100, 1000, None, None, "silu", True, 256, 128, 128, True, False),
    ("f16", 60000, 100, 1000, 9, WATER, "gelu", True, 256, 128, 128, True, False),
    ("bf16", 9000, 512, 2048, None, None, "gelu", True, 128, 128, 128, True, True),
    ("bf16", 30000, 1024, 1024, 9, WATER, "gelu", True, 256, 256, 128, True, True),
    ("bf16", 24000, 1024, 4096, None, None, "gelu", True, 256, 256, 256, True, True),
    ("bf16", 24000, 1024, 4096, None, None, None, True, 256, 256, 256, True, False),
    ("f16", 6000, 2090, 2101, None, None, None, True, 256, 256, 256, True, False),
    ("bf16", 6000, 2090, 2101, None, None, None, False, 256, 256, 256, True, False),
    ("f16", 1500, 2090, 2101, None, None, "silu", True, 64, 64, 128, False, True),
    ("bf16", 16384, 1024, 1024, 64, UNEVEN, None, True, 128, 128, 128, True, False),
    ("f16", 16384, 1024, 1024, 64, UNEVEN, "silu", True, 128, 128, 128, True, True),
    ("f32", 6000, 1100, 2100, None, None, "silu", True, 128, 128, 128, True, True),
    ("f32", 6000, 1100, 2100, 9, FEW, None, True, 128, 128, 128, True, False),
    ("f32", 6000, 1100, 2100, None, None, None, True, 128, 128, 128, True, False),
    ("f32", 21, 1024, 4096, None, None, None, True, 64, 64, 128, False, False),
    ("bf16", 21, 1024, 4096, None, None, "silu", True, 64, 64, 128, False, True),
    ("f32", 5000, 70, 130, 9, FEW, "silu", True, 64, 64, 64, True, False),
    ("f16", 5000, 70, 130, 9, FEW, "silu", True, 64, 64, 64, True, False),
    ("bf16", 5000, 70, 130, None, None, "silu", True, 64, 64, 64, True, False),
    ("f32", 5000, 70, 130, None, None, "silu", True, 64, 64, 64, True, False),
    ("bf16", 5000, 70, 130, 9, FEW, None, True, 64, 64, 64, True, False),
    ("f16", 5000, 70, 130, None, None, None, True, 64, 64, 64, True, False),
    ("f32", 5000, 70, 130, 9, FEW, None, True, 64, 64, 64, True, False),
    ("f32", 5000, 70, 130, None, None, None, True, 64, 64, 64, True, False),
    ("f32", 1, 1024, 512, None, None, "silu", True, 0, 64, 64, False, True),
]


def _name(case):
    dtype, rows, n_in, n_out, groups, _, activation, bias = case[:8]
    return f"{dtype}-{rows}x{n_in}-{n_out}-{groups}-{activation}{'-bias' if bias else ''}"


@pytest.mark.parametrize("case", CASES, ids=_name)
def test_the_variant_that_a_call_takes(lib, case):
    dtype, rows, n_in, n_out, groups, _, activation, _, forward, inputs, weight, parts, formed = case
    v = _variant(lib, dtype, rows, n_in, n_out, groups, activation is not None)
    assert (v["forward"], v["input"], v["weight"], bool(v["pass"])) == (forward, inputs, weight, formed), v
    assert (rows > v["weight_rows"]) is parts, v


def test_the_cases_take_every_variant():
    """Of products: 64 and 128 of all types and 256 of the 16-bit ones, of one weight and of groups; x's and the weight's
    gradients with d formed as it is staged (up to 128 tiles); the weight's of one weight alone in 256."""
    def kinds(size, column, slope=None):
        return {(c[column], c[4] is not None) for c in CASES if (c[0] == "f32") == (size == 4)
                and (slope is None or (c[6] is not None and not c[12]) is slope)}
    both = {(t, g) for t in (64, 128) for g in (False, True)}
    for size in (2, 4):
        wide = {(256, False), (256, True)} if size == 2 else set()
        assert kinds(size, 8) - {(0, False)} == both | wide
        assert kinds(size, 9, True) == both and kinds(size, 10, True) == both
        assert kinds(size, 9, False) >= both and kinds(size, 10, False) >= both
    assert {(256, False), (256, True)} <= kinds(2, 9, False) and (256, False) in kinds(2, 10, False)
    assert {c[7] for c in CASES if c[10] == 256} == {True, False}


def test_variants_arguments(lib):
    from xnn_amd import _lib
    out = (ctypes.c_int32 * 8)()
    for args, text in (((1, 5, 8, 8, 1, 0, 0, out), b"dtype"), ((0, 0, 8, 8, 1, 0, 0, out), b"no rows"),
                       ((0, 5, 0, 8, 1, 0, 0, out), b"widths"), ((0, 5, 8, 8, 5000, 1, 0, out), b"n_groups"),
                       ((0, 5, 8, 8, 1, 0, 0, None), b"NULL")):
        assert lib.xnn_linear_variants(*args) == _lib.XNN_EINVAL and text in lib.xnn_last_error()


# --------------------------------------------------------------------------- on the GPU
@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=_name)
def test_each_variant_against_float64(case):
    from test_gpu_feed_forward import _check_dense, _dense_case
    dtype, rows, n_in, n_out, groups, some, activation, bias = case[:8]
    _check_dense(dtype, _dense_case(dtype, rows, n_in, n_out, groups, bias=bias, some=some, seed=rows + n_in), activation)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 3, 70])
@pytest.mark.parametrize("n_in", [10, 1500, 1501])
def test_an_infinite_float32_input(rows, n_in):
    """NaN, for infinity has no planes; in one or two rows of up to 1,500 inputs the product's own infinity."""
    import torch
    import xnn_amd as xa
    x = torch.ones(rows, n_in, device="cuda")
    x[:, n_in // 2] = float("inf")
    w = torch.randn(n_in, 40, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    w = torch.where(w == 0, torch.ones_like(w), w)
    got = xa.linear(x, w)
    if rows <= 2 and n_in <= 1500:
        assert torch.equal(got, (w[n_in // 2].sign() * float("inf")).expand(rows, 40))
    else:
        assert got.isnan().all()
