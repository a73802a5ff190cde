"""Argument checks of the attention operators' C entry points: refused on the host before any launch
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
SIZE, SPLIT = ctypes.c_size_t(), ctypes.c_size_t()


def test_embedding_arguments(lib):
    f = lib.xnn_embedding
    _refused(lib, f(1, BUF, 4, BUF, 4, 4, 1.0, BUF, None), b"dtype")
    _refused(lib, f(0, BUF, -1, BUF, 4, 4, 1.0, BUF, None), b"negative")
    _refused(lib, f(0, None, 4, BUF, 4, 4, 1.0, BUF, None), b"NULL")
    assert f(0, None, 0, None, 0, 4, 1.0, None, None) == 0
    assert lib.xnn_embedding_grad_work_size(1000, 119, 128, ctypes.byref(SIZE)) == 0
    need = SIZE.value
    _refused(lib, lib.xnn_embedding_grad_work_size(1 << 31, 119, 128, ctypes.byref(SIZE)), b"too many")
    g = lib.xnn_embedding_grad
    _refused(lib, g(0, BUF, 1000, BUF, 119, 128, 1.0, BUF, BUF, need - 1, None), b"too small")
    _refused(lib, g(0, BUF, 1000, BUF, 119, 128, 1.0, BUF, ctypes.addressof(BUF) + 4, need, None), b"aligned")
    _refused(lib, g(7, BUF, 1000, BUF, 119, 128, 1.0, BUF, BUF, need, None), b"dtype")
    assert g(0, None, 0, None, 0, 128, 1.0, None, None, 0, None) == 0


def test_dropout_arguments(lib):
    f = lib.xnn_dropout_add
    _refused(lib, f(1, BUF, None, 4, 0, 0, 0, None, BUF, None), b"dtype")
    _refused(lib, f(0, BUF, None, 4, 65537, 0, 0, None, BUF, None), b"drop")
    _refused(lib, f(0, None, None, 4, 0, 0, 0, None, BUF, None), b"NULL")
    assert f(0, None, None, 0, 0, 0, 0, None, None, None) == 0


def _heads(n, data=None):
    from xnn_amd import _lib
    return ctypes.byref(_lib.Heads(ctypes.addressof(BUF) if data is None else data, n * 16, 16, n))


def test_head_norm_arguments(lib):
    f = lib.xnn_head_norm_rotate

    def call(q=4, k=2, T=3, D=16, R=16, rows=3, pos=None, out=BUF):
        return f(0, _heads(q), _heads(k), T, D, R, BUF, BUF, BUF, BUF, rows, pos, 1e-6, 0, out, BUF, None)
    _refused(lib, call(D=129), b"head_dim")
    _refused(lib, call(R=15), b"rotated")
    _refused(lib, call(R=18), b"rotated")
    _refused(lib, call(q=0), b"no heads")
    _refused(lib, call(rows=4), b"row a token")
    _refused(lib, call(out=None), b"NULL output")
    assert call(T=0, out=None) == 0
    g = lib.xnn_head_norm_rotate_backward

    def back(pos=None, dqw=BUF, dkw=BUF, dc=BUF, ds=BUF, size=1 << 30):
        return g(0, _heads(4), _heads(2), 3, 16, 16, BUF, BUF, BUF, BUF, 3, pos, 1e-6, 0, BUF, BUF,
                 BUF, BUF, dqw, dkw, dc, ds, BUF, size, None)
    _refused(lib, back(dkw=None), b"weights' gradients")
    _refused(lib, back(dc=None), b"tables' gradients")
    _refused(lib, back(pos=BUF), b"by position")
    _refused(lib, back(size=16), b"work too small")


def test_attention_arguments(lib):
    from xnn_amd import _lib

    def plan(tokens=10, n32=1, n128=1, tiles=True):
        at = ctypes.addressof(BUF) if tiles else None
        return ctypes.byref(_lib.AttentionTiles(tokens, 10, n32, n128, at, at))

    def call(dtype=0, H=4, K=2, KV=2, T=10, D=16, p=None, scale=0.25, out=BUF, q=None):
        return lib.xnn_attention(dtype, _heads(H, q), _heads(K), _heads(KV), T, D, p or plan(), None,
                                 scale, out, None, None, 0, None)
    _refused(lib, call(dtype=1), b"dtype")
    _refused(lib, call(D=0), b"head_dim")
    _refused(lib, call(D=129), b"head_dim")
    _refused(lib, call(H=3), b"multiple")
    _refused(lib, call(KV=1), b"multiple")
    _refused(lib, call(T=9), b"another number")
    _refused(lib, call(p=plan(n32=0)), b"empty plan")
    _refused(lib, call(p=plan(tiles=False)), b"empty plan")
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        _refused(lib, call(scale=scale), b"scale")
    _refused(lib, call(out=None), b"NULL output")
    _refused(lib, call(q=0), b"NULL input")
    assert call(T=0, p=plan(tokens=0, tiles=False), out=None) == 0
    _refused(lib, lib.xnn_attention_plan(BUF, 2, 100, BUF, BUF, BUF, BUF, 2, BUF, 2, BUF, None), b"too small")
    _refused(lib, lib.xnn_attention_plan(BUF, 2, 1 << 31, BUF, BUF, BUF, BUF, 2, BUF, 2, BUF, None), b"too many")
    assert lib.xnn_attention_backward_work_size(0, 10, 4, 2, 16, plan(), ctypes.byref(SIZE)) == 0
    long = ctypes.byref(_lib.AttentionTiles(9000, 9000, 141, 71, None, None))
    assert lib.xnn_attention_work_size(0, 9000, 4, 32, long, ctypes.byref(SPLIT)) == 0 and SPLIT.value > 0
    assert lib.xnn_attention_work_size(0, 10, 4, 16, plan(), ctypes.byref(SPLIT)) == 0 and SPLIT.value == 0
    _refused(lib, lib.xnn_attention_backward(0, _heads(4), _heads(2), _heads(2), 10, 16, plan(), None,
                                             0.25, BUF, BUF, BUF, BUF, BUF, BUF, BUF, SIZE.value - 1,
                                             None), b"too small")


def test_functions_refuse_cpu_tensors():
    import xnn_amd as xa
    x = torch.zeros(4, 2, 8)
    for call in (lambda: xa.attention_plan(torch.tensor([4])),
                 lambda: xa.embedding(torch.zeros(3, dtype=torch.int64), x[0]),
                 lambda: xa.dropout_add(x, None, 0.5, 0),
                 lambda: xa.head_norm_rotate(x, x, x[0, 0], x[0, 0], x[:, 0, :4], x[:, 0, :4])):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
