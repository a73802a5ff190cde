"""The counts of the entry points' calls: Python's and native code's as one mapping."""
import pytest

from xnn_amd import _lib


def test_python_and_native_calls_count_together():
    native = {"a": 2, "b": 0}
    calls = _lib.CallCounts()
    calls["p"] = 3
    calls.join(native, lambda name: native.get(name, 0))
    assert dict(calls) == {"p": 3, "a": 2}
    assert "a" in calls and "b" not in calls and "q" not in calls
    assert calls["a"] == calls.get("a") == 2 and calls.get("b", 7) == 7
    with pytest.raises(KeyError):
        calls["b"]
    calls["a"] = calls["a"] + 1
    native["a"] += 4
    assert calls["a"] == 7 and len(calls) == 2 and sorted(calls) == ["a", "p"]
    before = dict(calls)
    calls.clear()
    assert dict(calls) == {} and before == {"p": 3, "a": 7}
    native["b"] += 1
    assert dict(calls) == {"b": 1}
    del calls["b"]
    assert "b" not in calls


def test_counting_a_call(monkeypatch):
    calls = _lib.CallCounts()
    monkeypatch.setattr(_lib, "calls", calls)
    calls.join(["x"], lambda name: 5 if name == "x" else 0)
    for _ in range(2):
        _lib.count_call("x")
    assert calls["x"] == 7


def test_the_attention_operators_are_counted():
    import xnn_amd.attention as A
    names = A._ops().entries()
    assert "xnn_attention" in names and "xnn_embedding_grad" in names
    assert all(isinstance(_lib.calls.get(n, 0), int) for n in names)
