"""The feed-forward block over atoms and the attention potential with it: the PyTorch formulation against the
definition, symmetries and forces, and (on a GPU) the HIP evaluation against it."""
import pytest
import torch

import xnn_amd as xa
from xnn_amd import atom_attention as AA
from xnn_amd import synthetic


@pytest.fixture
def float64():
    old = torch.get_default_dtype()
    torch.set_default_dtype(torch.float64)
    yield
    torch.set_default_dtype(old)


def _graph(device="cpu", n=3, cutoff=4.0):
    graphs = [xa.structure_to_graph(s.as_dict(), cutoff) for s in synthetic.random_molecules(n, seed=2)]
    return xa.collate(graphs).to(device)


def _block(n_species, dtype=torch.float64, activation="gelu"):
    gen = torch.Generator().manual_seed(5)
    block = xa.AtomFeedForward(12, 20, activation, n_species, generator=gen).to(dtype)
    with torch.no_grad():
        for p in block.parameters():
            p += 0.1 * torch.randn(p.shape, generator=gen).to(dtype)
    return block


@pytest.mark.parametrize("n_species", [None, 9])
@pytest.mark.parametrize("activation", [None, "silu", "gelu", "tanh"])
def test_pytorch_form_equals_the_definition(n_species, activation):
    """Atom by atom."""
    block = _block(n_species, activation=activation)
    gen = torch.Generator().manual_seed(6)
    x = torch.randn(17, 12, generator=gen, dtype=torch.float64)
    z = torch.tensor([1, 6, 7, 8])[torch.randint(0, 4, (17,), generator=gen)]
    f = {None: lambda t: t, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
         "tanh": torch.tanh}[activation]
    want = []
    for row, species in zip(x, z.tolist()):
        def of(p):
            return p if n_species is None else p[species]
        n = (row - row.mean()) / torch.sqrt(row.var(unbiased=False) + 1e-5) * block.norm_weight + block.norm_bias
        hidden = f(of(block.up).T @ n + of(block.up_bias))
        want.append(row + of(block.down).T @ hidden + of(block.down_bias))
    torch.testing.assert_close(block(x, z), torch.stack(want), rtol=1e-12, atol=1e-12)
    empty = block(x[:0], z[:0])
    assert empty.shape == (0, 12)


def test_a_model_without_it_is_what_it_was(float64):
    """The weights before the feed-forward blocks draw the same numbers, with and without them."""
    old = xa.AtomAttentionPotential(channels=16, heads=2, cutoff=4.0)
    new = xa.AtomAttentionPotential(channels=16, heads=2, cutoff=4.0, feed_forward=24, species_weights=True)
    assert not old.feed_forward and len(new.feed_forward) == 2
    state = new.state_dict()
    for name, p in old.state_dict().items():
        assert torch.equal(p, state[name]), name
    assert new.feed_forward[0].up.shape == (9, 16, 24)


@pytest.mark.parametrize("species_weights", [False, True])
def test_the_model_is_invariant_and_its_forces_are_slopes(float64, species_weights):
    model = xa.build_model(xa.ModelConfig("atom_attention", dict(
        channels=16, heads=2, cutoff=4.0, layers=1, feed_forward=24, species_weights=species_weights))).eval()
    g = _graph()
    want = model(g)["energy"]
    turn = torch.linalg.qr(torch.randn(3, 3, generator=torch.Generator().manual_seed(3)))[0]
    moved = _graph()
    moved.pos = moved.pos @ turn.T + 1.5
    torch.testing.assert_close(model(moved)["energy"], want, rtol=1e-10, atol=1e-10)
    forces = xa.ForceStressOutput(model, compute_stress=False).eval()(_graph(n=1))["forces"].detach()
    step = torch.randn(forces.shape, generator=torch.Generator().manual_seed(4))

    def energy(sign):
        at = _graph(n=1)
        at.pos = at.pos + sign * 1e-5 * step
        return float(model(at)["energy"].detach().sum())
    slope = (energy(1) - energy(-1)) / 2e-5
    assert abs(-float((forces * step).sum()) - slope) < 1e-6 * max(1.0, float(forces.norm()))


def test_training_on_forces_takes_the_pytorch_form(float64):
    model = xa.AtomAttentionPotential(channels=16, heads=2, cutoff=4.0, layers=1, feed_forward=8,
                                      species_weights=True).train()
    out = xa.ForceStressOutput(model, compute_stress=False).train()(_graph())
    (out["energy"].square().sum() + out["forces"].square().sum()).backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in model.parameters())


def test_refused():
    with pytest.raises(ValueError, match="positive"):
        xa.AtomFeedForward(8, 0)
    with pytest.raises(ValueError, match="positive"):
        xa.AtomFeedForward(8, 8, n_species=0)
    with pytest.raises(ValueError, match="activation"):
        xa.AtomFeedForward(8, 8, "relu")
    with pytest.raises(ValueError, match="atomic numbers"):
        xa.AtomFeedForward(8, 8, n_species=3)(torch.zeros(2, 8))


# --------------------------------------------------------------------------- on the GPU
@pytest.mark.gpu
@pytest.mark.parametrize("species_weights", [False, True])
@pytest.mark.parametrize("periodic", [False, True])
def test_hip_evaluation_equals_the_pytorch_form(periodic, species_weights):
    from xnn_amd import _lib
    model = xa.AtomAttentionPotential(channels=32, heads=4, cutoff=4.0, layers=2, feed_forward=96,
                                      species_weights=species_weights).to("cuda").eval()

    def graph():
        if not periodic:
            return _graph("cuda", 5)
        s = synthetic.water_box(n_molecules=64, box=12.4, grid=4, seed=3)
        return xa.structure_to_graph(s.as_dict(), 4.0, device="cuda")
    names = ["xnn_layer_norm", "xnn_layer_norm_backward", "xnn_linear", "xnn_linear_backward"]
    names += ["xnn_group_plan"] if species_weights else []
    before = {n: _lib.calls.get(n, 0) for n in names}
    got = xa.ForceStressOutput(model, compute_stress=periodic).eval()(graph())
    assert all(_lib.calls.get(n, 0) > c for n, c in before.items())
    model.use_fast = False
    want = xa.ForceStressOutput(model, compute_stress=periodic).eval()(graph())
    # float32 on both sides: energies of a few hundred terms, forces their derivatives
    torch.testing.assert_close(got["energy"], want["energy"], rtol=2e-5, atol=2e-4)
    scale = float(want["forces"].abs().max())
    assert float((got["forces"] - want["forces"]).abs().max()) <= 2e-4 * scale


@pytest.mark.gpu
@pytest.mark.parametrize("species_weights", [False, True])
def test_a_fitting_step_has_the_gradients_of_the_pytorch_form(species_weights):
    grads = []
    for fast in (True, False):
        model = xa.AtomAttentionPotential(channels=32, heads=4, cutoff=4.0, feed_forward=64, activation="gelu",
                                          species_weights=species_weights, use_fast=fast).to("cuda").train()
        model(_graph("cuda", 5))["energy"].square().sum().backward()
        grads.append({n: p.grad.double() for n, p in model.named_parameters()})
    for n, a in grads[0].items():
        b = grads[1][n]
        assert float((a - b).norm()) <= 2e-4 * float(b.norm()) + 1e-6, n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n_species", [None, 9])
def test_a_block_under_autocast(dtype, n_species):
    """Norms of the errors against float64: the sum that is added to x has six roundings to 16 bits behind it (the
    operands and results of two products), the gradients those of both passes, each of half a unit at most."""
    block = _block(n_species)
    gen = torch.Generator().manual_seed(6)
    x, g = (torch.randn(90, 12, generator=gen, dtype=torch.float64) for _ in range(2))
    z = torch.tensor([1, 6, 7, 8])[torch.randint(0, 4, (90,), generator=gen)]

    def run(block, x, g, z):
        leaf = x.clone().requires_grad_(True)
        y = block(leaf, z)
        assert y.dtype == x.dtype
        return (y.detach(), *torch.autograd.grad(y, (leaf, *block.parameters()), g))
    want = run(block, x, g, z)
    block = block.float().to("cuda")
    block.fast_active = True
    with torch.autocast("cuda", dtype):
        got = run(block, *(t.to("cuda") for t in (x.float(), g.float(), z)))
    unit = torch.finfo(dtype).eps
    for i, (a, b) in enumerate(zip(got, want)):
        assert a.dtype == torch.float32
        off = float((a.cpu().double() - b).norm() / b.norm())
        assert off <= (3 if i == 0 else 6) * unit, (i, off / unit)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["layer_norm", "linear", "grouped_linear"])
@pytest.mark.parametrize("tracer", ["jit", "make_fx", "compile"])
def test_a_recorded_function_gives_what_the_function_gives(name, tracer):
    gen = torch.Generator().manual_seed(7)

    def normal(*shape):
        return torch.randn(*shape, generator=gen).to("cuda")
    plan = xa.group_plan(torch.arange(40, device="cuda") % 3, 3)
    f, args = {"layer_norm": (lambda x, w, b: xa.layer_norm(x, w, b), (normal(40, 12), normal(12), normal(12))),
               "linear": (lambda x, w, b, r: xa.linear(x, w, b, "gelu", r),
                          (normal(40, 12), normal(12, 20), normal(20), normal(40, 20))),
               "grouped_linear": (lambda x, w, b: xa.grouped_linear(x, w, plan, b, "silu"),
                                  (normal(40, 12), normal(3, 12, 20), normal(3, 20)))}[name]
    if tracer == "jit":
        recorded = torch.jit.trace(f, args, check_trace=False)
    elif tracer == "make_fx":
        from torch.fx.experimental.proxy_tensor import make_fx
        recorded = make_fx(f)(*args)
    else:
        recorded = torch.compile(f, backend="aot_eager", fullgraph=True)
    others = [a * 0.5 + 0.25 for a in args]
    for inputs in (args, others):
        assert torch.equal(recorded(*inputs), f(*inputs))
    if tracer == "make_fx":
        return                                                      # records the forward pass alone
    grads = []
    for h in (recorded, f):
        leaves = [a.clone().requires_grad_(True) for a in others]
        out = h(*leaves)
        grads.append(torch.autograd.grad(out, leaves, torch.cos(out).detach()))
    for a, b in zip(*grads):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_the_operators_registration():
    """Schema, shapes and recording of the operators and of those that their backward passes call."""
    gen = torch.Generator().manual_seed(8)

    def normal(*shape):
        return torch.randn(*shape, generator=gen).to("cuda")
    ops = torch.ops.xnn_amd
    ids = torch.arange(40, device="cuda") % 3
    plan = ops.group_plan(ids, 3)
    x, w, b, w3, b3, r, n, g = (normal(40, 12), normal(12, 20), normal(20), normal(3, 12, 20), normal(3, 20),
                                normal(40, 20), normal(12), normal(40, 20))
    stats = ops.layer_norm_stats(x, n, n, 1e-5)[1]
    slope = ops.dense_slope(x, w, b, 2, r, None)[1]
    checks = ("test_schema", "test_faketensor", "test_aot_dispatch_dynamic")
    for op, args in ((ops.layer_norm, (x, n, n, 1e-5)), (ops.layer_norm_stats, (x, None, n, 1e-5)),
                     (ops.layer_norm_backward, (x, x, n, stats, True, True, False)), (ops.group_plan, (ids, 3)),
                     (ops.dense, (x, w, b, 2, r, None)), (ops.dense, (x, w3, b3, 1, None, plan)),
                     (ops.dense_slope, (x, w, None, 2, r, None)), (ops.dense_slope, (x, w3, b3, 0, None, plan)),
                     (ops.dense_backward, (g, slope, x, w, None, True, True, True)),
                     (ops.dense_backward, (g, None, x, w3, plan, False, True, False))):
        torch.library.opcheck(op.default, args, test_utils=checks)


@pytest.mark.gpu
def test_batches_of_calls_are_refused_and_batches_of_cotangents_are_loops():
    x, w = torch.randn(5, 6, device="cuda"), torch.randn(6, 4, device="cuda")
    for f in (lambda a: xa.linear(a, w), xa.layer_norm):
        with pytest.raises(RuntimeError, match="batching rule"):
            torch.func.vmap(f)(x[None])
        leaf = x.clone().requires_grad_(True)
        out = f(leaf)
        batch = torch.stack([torch.cos(out), torch.sin(out)]).detach()
        got, = torch.autograd.grad(out, leaf, batch, is_grads_batched=True, retain_graph=True)
        for a, b in zip(got, batch):
            assert torch.equal(a, torch.autograd.grad(out, leaf, b, retain_graph=True)[0])
