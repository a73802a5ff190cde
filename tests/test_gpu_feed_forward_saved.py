"""What the backward passes of the feed-forward operators keep: x for the gradients of weight and bias alone, the weight
for that of x alone. The rest may go, or be written to, before the backward pass."""
import pytest
import torch

import xnn_amd as xa

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _case(groups):
    gen = torch.Generator().manual_seed(1)

    def normal(*shape):
        return torch.randn(*shape, generator=gen).to(DEV)
    lead = () if groups is None else (groups,)
    plan = None if groups is None else xa.group_plan(torch.arange(70, device=DEV) * 7 % (groups + 1), groups)
    return dict(x=normal(70, 24), w=normal(*lead, 24, 40), b=normal(*lead, 40), r=normal(70, 40), g=normal(70, 40)), plan


def _run(x, w, b, r, plan, activation):
    if plan is None:
        return xa.linear(x, w, b, activation, r)
    return xa.grouped_linear(x, w, plan, b, activation, r)


NEEDS = {"x": "w", "w": "x", "b": "x", "r": ""}


@pytest.mark.parametrize("activation", [None, "silu"])
@pytest.mark.parametrize("groups", [None, 4])
@pytest.mark.parametrize("leaf", NEEDS)
def test_a_gradient_needs_no_other_operand(leaf, groups, activation):
    t, plan = _case(groups)
    g = t.pop("g")
    leaves = {k: v.clone().requires_grad_(True) for k, v in t.items()}
    want, = torch.autograd.grad(_run(**leaves, plan=plan, activation=activation), leaves[leaf], g)
    for other in t:
        if other == leaf or other in NEEDS[leaf]:
            continue
        args = {k: v.clone() for k, v in t.items()}
        args[leaf].requires_grad_(True)
        out = _run(**args, plan=plan, activation=activation)
        args[other].add_(1.0)
        got, = torch.autograd.grad(out, args[leaf], g)
        assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0)), other
    for other in NEEDS[leaf]:
        args = {k: v.clone() for k, v in t.items()}
        args[leaf].requires_grad_(True)
        out = _run(**args, plan=plan, activation=activation)
        args[other].add_(1.0)
        with pytest.raises(RuntimeError, match="inplace operation"):
            torch.autograd.grad(out, args[leaf], g)


def test_its_own_operand_may_be_written_to():
    t, _ = _case(None)
    for leaf in ("x", "w", "b", "r"):
        args = {k: t[k].clone() for k in ("x", "w", "b", "r")}
        args[leaf].requires_grad_(True)
        out = _run(**args, plan=None, activation="gelu")
        want, = torch.autograd.grad(out, args[leaf], t["g"], retain_graph=True)
        with torch.no_grad():
            args[leaf].mul_(3.0)
        got, = torch.autograd.grad(out, args[leaf], t["g"])
        assert torch.equal(got, want)


def test_memory_of_an_input_that_is_not_needed():
    """x of 64 MB, of which the gradient of x itself needs nothing."""
    x = torch.randn(1 << 14, 1024, device=DEV, requires_grad=True)
    w = torch.randn(1024, 8, device=DEV)
    start = torch.cuda.memory_allocated()
    out = xa.linear(x * 2.0, w)
    assert torch.cuda.memory_allocated() - start < 8 << 20
    torch.autograd.grad(out.sum(), x)


def test_layer_norm_keeps_its_weight_for_x_alone():
    gen = torch.Generator().manual_seed(2)
    x, w, g = (torch.randn(*s, generator=gen).to(DEV) for s in ((30, 24), (24,), (30, 24)))
    leaf = w.clone().requires_grad_(True)
    out = xa.layer_norm(x, leaf)
    want, = torch.autograd.grad(out, leaf, g, retain_graph=True)
    with torch.no_grad():
        leaf.mul_(3.0)
    got, = torch.autograd.grad(out, leaf, g)
    assert torch.equal(got, want)


def test_the_backward_operator_with_what_each_gradient_needs():
    ops = torch.ops.xnn_amd
    for groups in (None, 4):
        t, plan = _case(groups)
        rows = None if plan is None else plan.rows
        slope = ops.dense_slope(t["x"], t["w"], t["b"], 1, None, rows)[1]
        full = ops.dense_backward(t["g"], slope, t["x"], t["w"], rows, True, True, True)
        dx = ops.dense_backward(t["g"], slope, None, t["w"], rows, True, False, False)
        dw = ops.dense_backward(t["g"], slope, t["x"], None, rows, False, True, True)
        for a, b in ((dx[0], full[0]), (dw[1], full[1]), (dw[2], full[2])):
            assert torch.equal(a, b)
        for args in ((t["g"], slope, None, t["w"], rows, True, False, False),
                     (t["g"], slope, t["x"], None, rows, False, True, True)):
            torch.library.opcheck(ops.dense_backward.default, args,
                                  test_utils=("test_schema", "test_faketensor", "test_aot_dispatch_dynamic"))
        for args, text in (((t["g"], slope, None, t["w"], rows, True, True, False), "need x"),
                           ((t["g"], slope, t["x"], None, rows, True, True, False), "needs the weight"),
                           ((t["g"][:5], slope, None, t["w"], rows, True, False, False),
                            "slope is not" if groups is None else "the plan is not of 5 rows"),
                           ((t["g"], slope, t["x"][:5], None, rows, False, True, False), "x must be"),
                           ((t["g"][:, :3], None, None, t["w"], rows, True, False, False), "weight must be")):
            with pytest.raises(ValueError, match=text):
                ops.dense_backward(*args)
