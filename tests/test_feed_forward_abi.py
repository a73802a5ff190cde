"""Argument checks of the feed-forward operators' C entry points: refused on the host before any launch
(no GPU needed), and CPU tensors refused by the functions."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from xnn_amd import _lib
    return _lib.load()


def _refused(lib, code, text):
    from xnn_amd import _lib
    assert code == _lib.XNN_EINVAL
    assert text in lib.xnn_last_error(), lib.xnn_last_error()


BUF = (ctypes.c_double * 64)()
SIZE, MORE = ctypes.c_size_t(), ctypes.c_size_t()


def test_layer_norm_arguments(lib):
    f = lib.xnn_layer_norm

    def call(dtype=0, x=BUF, stride=8, rows=4, width=8, out=BUF):
        return f(dtype, x, stride, rows, width, None, None, 1e-5, out, None, None)
    _refused(lib, call(dtype=1), b"dtype")
    _refused(lib, call(rows=-1), b"n_rows")
    _refused(lib, call(rows=1 << 31), b"n_rows")
    _refused(lib, call(width=0), b"width")
    _refused(lib, call(width=16385), b"width")
    _refused(lib, call(stride=7), b"overlap")
    _refused(lib, call(x=None), b"NULL")
    _refused(lib, call(out=None), b"NULL")
    assert call(rows=0, x=None, out=None) == 0
    assert lib.xnn_layer_norm_backward_work_size(8, ctypes.byref(SIZE)) == 0 and SIZE.value > 0
    _refused(lib, lib.xnn_layer_norm_backward_work_size(0, ctypes.byref(SIZE)), b"width")
    _refused(lib, lib.xnn_layer_norm_backward_work_size(8, None), b"NULL size")
    g = lib.xnn_layer_norm_backward

    def back(grad=BUF, stats=BUF, dw=BUF, work=BUF, size=None, rows=4, stride=8):
        return g(0, grad, BUF, stride, rows, 8, None, stats, BUF, dw, None, work,
                 SIZE.value if size is None else size, None)
    _refused(lib, back(grad=None), b"NULL")
    _refused(lib, back(stats=None), b"NULL")
    _refused(lib, back(stride=4), b"overlap")
    _refused(lib, back(size=SIZE.value - 1), b"work too small")
    _refused(lib, back(work=None), b"work too small")
    assert g(0, None, None, 0, 0, 8, None, None, None, None, None, None, 0, None) == 0


def test_group_plan_arguments(lib):
    size, f = lib.xnn_group_plan_size, lib.xnn_group_plan
    two = (ctypes.byref(SIZE), ctypes.byref(MORE))
    assert size(1000, 9, *two) == 0
    assert SIZE.value == 4 * (1000 + 53 * 11) and MORE.value > 0
    _refused(lib, size(-1, 9, *two), b"n must")
    _refused(lib, size(1 << 30, 9, *two), b"n must")
    _refused(lib, size(10, 0, *two), b"n_groups")
    _refused(lib, size(10, 4097, *two), b"n_groups")
    _refused(lib, size(10, 9, None, None), b"NULL size")
    _refused(lib, f(BUF, 1000, 9, None, BUF, MORE.value, None), b"NULL plan")
    _refused(lib, f(None, 1000, 9, BUF, BUF, MORE.value, None), b"NULL ids")
    _refused(lib, f(BUF, 1000, 9, BUF, BUF, MORE.value - 1, None), b"work too small")
    _refused(lib, f(BUF, 1000, 5000, BUF, BUF, 1 << 30, None), b"n_groups")


def test_linear_arguments(lib):
    f, size = lib.xnn_linear, lib.xnn_linear_work_size
    assert size(0, 100000, 64, 64, 1, 0, ctypes.byref(SIZE)) == 0 and SIZE.value == 0
    assert size(0, 20, 4096, 64, 1, 0, ctypes.byref(SIZE)) == 0 and SIZE.value > 0     # a long sum for few outputs
    need = SIZE.value
    _refused(lib, size(0, 20, 4096, 64, 1, 0, None), b"NULL size")
    _refused(lib, size(1, 20, 4096, 64, 1, 0, ctypes.byref(SIZE)), b"dtype")

    def call(dtype=0, x=BUF, stride=None, rows=4, n_in=8, n_out=4, w=BUF, act=0, plan=None, groups=1, out=BUF,
             slope=None, work=BUF, room=0):
        return f(dtype, x, n_in if stride is None else stride, rows, n_in, n_out, w, None, act, None, plan, groups,
                 out, slope, work, room, None)
    _refused(lib, call(rows=20, n_in=4096, n_out=64, room=need - 1), b"work too small")
    _refused(lib, call(rows=20, n_in=4096, n_out=64, room=need, work=None), b"work too small")
    _refused(lib, call(rows=20, n_in=4096, n_out=64, room=need, work=ctypes.addressof(BUF) + 4), b"aligned")
    _refused(lib, call(dtype=1), b"dtype")
    _refused(lib, call(rows=-1), b"n_rows")
    _refused(lib, call(rows=1 << 30), b"n_rows")
    _refused(lib, call(n_in=0), b"widths")
    _refused(lib, call(n_out=1 << 20), b"widths")
    _refused(lib, call(rows=(1 << 30) - 1, n_out=(1 << 20) - 1), b"too many tiles")
    _refused(lib, call(act=4), b"activation")
    _refused(lib, call(act=-1), b"activation")
    _refused(lib, call(slope=BUF), b"no slope")
    _refused(lib, call(groups=2), b"plan")
    _refused(lib, call(groups=0, plan=BUF), b"n_groups")
    _refused(lib, call(groups=4097, plan=BUF), b"n_groups")
    _refused(lib, call(stride=7), b"overlap")
    _refused(lib, call(x=None), b"NULL")
    _refused(lib, call(w=None), b"NULL")
    _refused(lib, call(out=None), b"NULL")
    assert call(rows=0, x=None, out=None, w=None) == 0


def test_linear_backward_arguments(lib):
    def size(dtype, rows, groups, grouped=0, slope=0, weight=1, bias=0, out=None):
        return lib.xnn_linear_backward_work_size(dtype, rows, 64, 64, groups, grouped, slope, 0, weight, bias,
                                                 ctypes.byref(SIZE) if out is None else out)
    assert size(0, 20, 1) == 0 and SIZE.value == 0
    assert size(2, 1000, 1, slope=1, weight=0) == 0 and SIZE.value == 0
    assert lib.xnn_linear_backward_work_size(2, 1000, 200, 64, 1, 0, 1, 0, 0, 0, ctypes.byref(SIZE)) == 0
    assert SIZE.value == 1000 * 64 * 2                      # d
    assert size(0, 100000, 1) == 0
    need = SIZE.value
    assert need > 0
    _refused(lib, size(0, 20, 5000, 1), b"n_groups")
    _refused(lib, size(1, 20, 1), b"dtype")
    _refused(lib, lib.xnn_linear_backward_work_size(0, 20, 64, 64, 1, 0, 0, 0, 1, 0, None), b"NULL size")
    f = lib.xnn_linear_backward

    def call(grad=BUF, slope=None, x=BUF, stride=64, rows=100000, w=BUF, dx=None, dw=BUF, db=None, work=BUF,
             size=need):
        return f(0, grad, slope, x, stride, rows, 64, 64, w, None, 1, dx, dw, db, work, size, None)
    _refused(lib, call(grad=None), b"NULL cotangent")
    _refused(lib, call(w=None, dx=BUF), b"NULL weight")
    _refused(lib, call(x=None), b"NULL input")
    _refused(lib, call(stride=63), b"overlap")
    _refused(lib, call(size=need - 1), b"work too small")
    _refused(lib, call(db=BUF), b"work too small")
    _refused(lib, call(dw=None, db=BUF), b"goes with")
    _refused(lib, call(work=None), b"work too small")
    _refused(lib, call(work=ctypes.addressof(BUF) + 4), b"aligned")
    assert call(dw=None) == 0
    assert f(0, None, None, None, 0, 0, 64, 64, None, None, 1, BUF, None, None, None, 0, None) == 0


def test_sizes_whose_launches_pass_32_bits_of_threads(lib):
    def forward(rows, n_in, n_out, groups):
        return lib.xnn_linear_work_size(2, rows, n_in, n_out, groups, int(groups > 1), ctypes.byref(SIZE))

    def backward(rows, n_in, n_out, groups, slope=0, weight=1, bias=1):
        return lib.xnn_linear_backward_work_size(2, rows, n_in, n_out, groups, int(groups > 1), slope, 1, weight, bias,
                                                 ctypes.byref(SIZE))
    wide = (1 << 20) - 1
    _refused(lib, forward((1 << 30) - 1, 1, 1, 1), b"too many tiles")
    _refused(lib, forward(1, 1, wide, 4096), b"too many tiles")
    _refused(lib, backward((1 << 30) - 1, 1, 1, 1), b"too many tiles")
    assert forward(1 << 29, 1, 1, 1) == 0 and backward(1 << 29, 1, 1, 1) == 0
    assert forward(5000, 1, wide, 200) == 0
    # a weight of 2^37 elements; groups' biases take no blocks of their own
    _refused(lib, backward(100, 1 << 19, 1 << 18, 1), b"too many tiles")
    assert backward(100, 1 << 18, 1 << 17, 1) == 0
    assert backward(100, 1, 1 << 17, 4000) == 0
    assert backward(100, 1, 1 << 17, 4000, weight=0, bias=0) == 0


def test_functions_refuse_cpu_tensors():
    import xnn_amd as xa
    x, w = torch.zeros(4, 8), torch.zeros(8, 8)
    for call in (lambda: xa.layer_norm(x), lambda: xa.linear(x, w),
                 lambda: xa.group_plan(torch.zeros(4, dtype=torch.int64), 3),
                 lambda: xa.grouped_linear(x, w[None], xa.GroupPlan(4, 1, torch.zeros(163, dtype=torch.int32)))):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_refused_names_and_plans():
    import xnn_amd as xa
    x, w = torch.zeros(4, 8), torch.zeros(8, 8)
    with pytest.raises(ValueError, match="unknown activation"):
        xa.linear(x, w, activation="swish")
    with pytest.raises(ValueError, match="unknown activation"):
        xa.linear(x, w, activation=["silu"])
    with pytest.raises(TypeError, match="GroupPlan"):
        xa.grouped_linear(x, w[None], torch.zeros(4))
    with pytest.raises(ValueError, match="groups"):
        xa.grouped_linear(x, torch.zeros(3, 8, 8), xa.GroupPlan(4, 2, torch.zeros(216, dtype=torch.int32)))
