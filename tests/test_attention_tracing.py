"""The attention operators under tracers, fake tensors and compilers: they are recorded as operators
(never as memory that nothing fills) and give the same results from there."""
import pytest
import torch

import xnn_amd as xa

DEV = "cuda:0"


def _cases(device, T=40, H=4, K=2, D=16):
    """name -> (function, inputs), the plan apart."""
    gen = torch.Generator().manual_seed(3)

    def normal(*shape):
        return torch.randn(*shape, generator=gen).to(device)
    angle = normal(T, D // 2)
    heads = (normal(T, H, D), normal(T, K, D), normal(D), normal(D), angle.cos(), angle.sin())
    return {
        "xnn_amd.embedding_rows": (lambda i, t: xa.embedding(i, t, 0.5),
                                   (torch.arange(T, device=device) % 7, normal(7, 12))),
        "xnn_amd.dropout_add": (lambda x, r: xa.dropout_add(x, r, 0.3, 1 << 63 | 9, 4),
                                (normal(T, 9), normal(T, 9))),
        "xnn_amd.head_norm_rotate": (lambda *a: torch.cat(xa.head_norm_rotate(*a), 1), heads),
    }


@pytest.mark.parametrize("name", ["xnn_amd.embedding_rows", "xnn_amd.dropout_add", "xnn_amd.head_norm_rotate"])
def test_shapes_alone_are_enough_to_record_an_operator(name):
    """No memory and no GPU: the operator is in the graph, its output has the shape and type."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    f, args = _cases("cpu")[name]
    with FakeTensorMode() as mode:
        fake = [torch.empty(a.shape, dtype=a.dtype, device="cuda") for a in args]
        graph = make_fx(f)(*fake)
        out = f(*fake)
    assert any(name in str(n.target) for n in graph.graph.nodes if n.op == "call_function"), graph.code
    assert out.dtype == torch.float32 and out.device.type == "cuda"
    want = {"xnn_amd.embedding_rows": (40, 12), "xnn_amd.dropout_add": (40, 9),
            "xnn_amd.head_norm_rotate": (40, 6, 16)}[name]
    assert tuple(out.shape) == want


def test_attention_of_shapes_alone():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        q, k = (torch.empty(40, h, 16, dtype=torch.bfloat16, device="cuda") for h in (4, 2))
        tiles = torch.empty(2, 3, dtype=torch.int32, device="cuda")
        ops = torch.ops.xnn_amd
        out = ops.structure_attention(q, k, k, tiles, tiles, None, 40, 40, None)
        also, lse = ops.structure_attention_lse(q, k, k, tiles, tiles, None, 40, 40, None)
        grads = ops.structure_attention_backward(out, also, lse, q, k, k, tiles, tiles, None, 40, 40, 0.5)
        assert [tuple(t.shape) for t in (out, also, lse, *grads)] == [
            (40, 4, 16), (40, 4, 16), (4, 40), (40, 4, 16), (40, 2, 16), (40, 2, 16)]
        assert lse.dtype == torch.float32 and all(t.dtype == torch.bfloat16 for t in (out, *grads))


# --------------------------------------------------------------------------- on the GPU
def _gpu_cases():
    plan = xa.attention_plan(torch.tensor([25, 15], device=DEV))
    mask = torch.arange(40, device=DEV) % 5 != 0
    gen = torch.Generator().manual_seed(4)
    qkv = [torch.randn(40, h, 16, generator=gen).to(DEV) for h in (4, 2, 2)]
    return {**_cases(DEV),
            "xnn_amd.structure_attention": (lambda q, k, v: xa.structure_attention(q, k, v, plan, mask=mask), qkv)}


def _others(args):
    """Other inputs of the same kind."""
    return [a * 0.5 + 0.25 if a.is_floating_point() else a.flip(0) for a in args]


NAMES = ["xnn_amd.embedding_rows", "xnn_amd.dropout_add", "xnn_amd.head_norm_rotate",
         "xnn_amd.structure_attention"]


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("tracer", ["jit", "make_fx", "compile"])
def test_a_recorded_function_gives_what_the_function_gives(name, tracer):
    f, args = _gpu_cases()[name]
    if tracer == "jit":
        recorded = torch.jit.trace(f, tuple(args), check_trace=False)
    elif tracer == "make_fx":
        from torch.fx.experimental.proxy_tensor import make_fx
        recorded = make_fx(f)(*args)
    else:
        recorded = torch.compile(f, backend="aot_eager", fullgraph=True)
    for inputs in (args, _others(args)):
        assert torch.equal(recorded(*inputs), f(*inputs))
    if tracer == "make_fx":
        return                                                      # records the forward pass alone
    leaves = [[a.clone().requires_grad_(True) if a.is_floating_point() else a for a in _others(args)]
              for _ in range(2)]
    grads = []
    for g, inputs in zip((recorded, f), leaves):
        out = g(*inputs)
        grads.append(torch.autograd.grad(out, [a for a in inputs if a.requires_grad], torch.cos(out).detach()))
    for a, b in zip(*grads):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_the_operators_registration():
    """Schema, shapes and recording of the operators and of those that their backward passes call."""
    plan = xa.attention_plan(torch.tensor([25, 15], device=DEV))
    cases = _gpu_cases()
    ops = torch.ops.xnn_amd
    ids, table = cases["xnn_amd.embedding_rows"][1]
    x, r = cases["xnn_amd.dropout_add"][1]
    heads = cases["xnn_amd.head_norm_rotate"][1]
    q, k, v = cases["xnn_amd.structure_attention"][1]
    tiles = (plan.tiles32, plan.tiles128, None, 40, plan.max_atoms, None)
    out, lse = ops.structure_attention_lse(q, k, v, *tiles)
    checks = ("test_schema", "test_faketensor", "test_aot_dispatch_dynamic")
    for op, args in ((ops.embedding_rows, (ids, table, 0.5)), (ops.embedding_rows_grad, (ids, table[ids], 7, 0.5)),
                     (ops.dropout_add, (x, r, 0.25, 3, 4, None)),
                     (ops.head_norm_rotate, (*heads, None, 1e-6, False)),
                     (ops.head_norm_rotate_backward, (heads[0], heads[1], *heads, None, 1e-6, True, True, True)),
                     (ops.structure_attention, (q, k, v, *tiles)),
                     (ops.structure_attention_lse, (q, k, v, *tiles)),
                     (ops.structure_attention_backward, (q, out, lse, q, k, v, *tiles))):
        torch.library.opcheck(op.default, args, test_utils=checks)


@pytest.mark.gpu
def test_functional_gradients():
    """torch.func.grad records the backward pass too: the operators that are differentiable once refuse."""
    for name, (f, args) in _gpu_cases().items():
        at = [i for i, a in enumerate(args) if a.is_floating_point()]
        gradient = torch.func.grad(lambda *a: f(*a).square().sum(), argnums=tuple(at))
        if name in ("xnn_amd.head_norm_rotate", "xnn_amd.structure_attention"):
            with pytest.raises(RuntimeError, match="once"):
                gradient(*args)
            continue
        leaves = [a.clone().requires_grad_(True) if a.is_floating_point() else a for a in args]
        want = torch.autograd.grad(f(*leaves).square().sum(), [leaves[i] for i in at])
        for a, b in zip(gradient(*args), want):
            assert torch.equal(a, b), name


@pytest.mark.gpu
def test_a_batch_of_cotangents_is_a_loop_over_them():
    for name, (f, args) in _gpu_cases().items():
        leaves = [a.clone().requires_grad_(True) if a.is_floating_point() else a for a in args]
        wanted = [a for a in leaves if a.requires_grad]
        out = f(*leaves)
        batch = torch.stack([torch.cos(out), torch.sin(out)]).detach()
        got = torch.autograd.grad(out, wanted, batch, is_grads_batched=True, retain_graph=True)
        each = [torch.autograd.grad(out, wanted, g, retain_graph=True) for g in batch]
        for a, *b in zip(got, *each):
            assert torch.equal(a, torch.stack(b)), name


@pytest.mark.gpu
def test_batches_of_calls_are_refused():
    for name, (f, args) in _gpu_cases().items():
        with pytest.raises(RuntimeError, match="batching rule"):
            torch.func.vmap(f, randomness="different")(*(a[None] for a in args))
