"""Which species plan a graph gives, and who holds it: on the host, with stand-ins for streams, captures and the
plan's kernels; on the GPU the replays of captured steps."""
import copy
import gc
import pickle
import types
import weakref

import pytest
import torch

import xnn_amd as xa
from xnn_amd import feed_forward as FF


class Ids:
    """A species tensor on the device, as far as the cache looks at it."""
    device, is_cuda = "device", True

    def __init__(self, inference=False):
        self._version, self.inference = 0, inference

    def is_inference(self):
        return self.inference


class Graph:
    def __init__(self, inference=False):
        self.atomic_numbers = Ids(inference)


class Rows:
    pass


@pytest.fixture
def card(monkeypatch):
    """The stream that is current, whether it captures, and the plans that were formed again."""
    state = types.SimpleNamespace(stream=0, capturing=False, made=0, again=[])

    def make(ids, n_groups):
        state.made += 1
        return xa.GroupPlan(4, n_groups, Rows())
    monkeypatch.setattr(FF, "group_plan", make)
    monkeypatch.setattr(FF, "_form_again", lambda plan, ids: state.again.append(plan), raising=False)
    monkeypatch.setattr(torch.cuda, "device", lambda device: torch.no_grad())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state.capturing)
    monkeypatch.setattr(torch.cuda, "current_stream",
                        lambda device=None: types.SimpleNamespace(cuda_stream=state.stream))
    return state


def _captured(graph, card, n_groups=9):
    card.capturing = True
    plan = FF.species_plan_for(graph, n_groups)
    card.capturing = False
    return weakref.ref(plan.rows)


@pytest.mark.parametrize("act", ["stream", "groups", "write", "other ids", "copy"])
def test_a_plan_that_a_capture_takes_lives_on(card, act):
    """The captured kernels have its address: no later call may give it back to the allocator."""
    graph = Graph()
    ids = graph.atomic_numbers                              # which the captured kernels read, too
    FF.species_plan_for(graph, 9)
    if act == "copy":                                        # a model's step on a copy of the graph, which then goes
        rows = _captured(copy.copy(graph), card)
        ids._version += 1
    else:
        rows = _captured(graph, card)
        if act == "stream":
            card.stream = 7
        elif act == "write":
            ids._version += 1
        elif act == "other ids":
            graph.atomic_numbers = Ids()
    FF.species_plan_for(graph, 10 if act == "groups" else 9)
    gc.collect()
    assert rows() is not None


def test_a_replay_follows_the_atomic_numbers_whether_a_plan_was_kept_or_not(card):
    """What a capture uses is formed in it: at every replay, from the numbers as they are then."""
    graph = Graph()
    made = card.made
    _captured(graph, card)
    assert card.made == made + 1 and not card.again          # no plan was there: made in the capture
    kept = FF.species_plan_for(graph, 9)
    assert FF.species_plan_for(graph, 9) is kept and not card.again
    _captured(graph, card)
    assert len(card.again) == 1 and card.again[0] is kept
    # the replays write to that one: calls outside them have another, and so has a second capture, of its own
    other = FF.species_plan_for(graph, 9)
    assert other is not kept
    made = card.made
    for _ in range(3):
        assert _captured(graph, card)() is not other.rows
    assert card.made == made + 3 and len(card.again) == 1 and FF.species_plan_for(graph, 9) is other


def test_a_plan_of_numbers_that_were_written_to_is_not_taken_by_a_capture(card):
    graph = Graph()
    FF.species_plan_for(graph, 9)
    graph.atomic_numbers._version += 1
    made = card.made
    _captured(graph, card)
    assert card.made == made + 1 and not card.again


def test_streams_and_numbers_of_groups_keep_a_plan_each(card):
    graph = Graph()
    plans = {}
    for _ in range(2):
        for stream in (0, 7):
            for groups in (9, 10):
                card.stream = stream
                plan = FF.species_plan_for(graph, groups)
                assert plans.setdefault((stream, groups), plan) is plan and plan.n_groups == groups
    assert card.made == 4


def test_numbers_without_a_version_have_a_new_plan_each_time(card):
    """A write to an inference tensor can't be noticed."""
    graph = Graph(inference=True)
    assert FF.species_plan_for(graph, 9) is not FF.species_plan_for(graph, 9)


@pytest.mark.parametrize("other", [copy.deepcopy, lambda graph: pickle.loads(pickle.dumps(graph))])
def test_a_copied_graph_makes_its_own(card, other):
    """The version of copied numbers starts again, and may come to that of the numbers which the plan is of."""
    graph = Graph()
    graph.atomic_numbers._version = 2
    FF.species_plan_for(graph, 9)
    _captured(graph, card)
    FF.species_plan_for(graph, 9)
    made, another = card.made, other(graph)
    another.atomic_numbers._version = 2                     # 1 after the copy, and one write
    FF.species_plan_for(another, 9)
    assert card.made == made + 1


# --------------------------------------------------------------------------- on the GPU
def _graph(n=4):
    from xnn_amd import synthetic
    graphs = [xa.structure_to_graph(s.as_dict(), 4.0) for s in synthetic.random_molecules(n, seed=2)]
    return xa.collate(graphs).to("cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("kept", [True, False])
def test_replays_after_the_kept_plan_is_gone_and_the_numbers_changed(kept):
    g = _graph()
    if kept:
        g.species_plan(9)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows = g.species_plan(9).rows + 0
    others = [torch.tensor([1, 6, 7, 8], device="cuda")[(torch.arange(g.num_nodes, device="cuda") * k) % 4]
              for k in range(4)]
    side = torch.cuda.Stream()
    for ids in others:
        g.atomic_numbers.copy_(ids)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            g.species_plan(9)
        g.species_plan(10)
        junk = [torch.full((g.num_nodes + 53 * 11,), -1, dtype=torch.int32, device="cuda") for _ in range(16)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(rows, xa.group_plan(ids, 9).rows)
        assert torch.equal(rows, g.species_plan(9).rows)
        assert all((t == -1).all() for t in junk)


@pytest.mark.gpu
@pytest.mark.parametrize("kept", [True, False])
def test_a_captured_model_with_weights_of_species_follows_them(kept):
    g = _graph()
    model = xa.AtomAttentionPotential(channels=32, heads=4, cutoff=4.0, feed_forward=48,
                                      species_weights=True).to("cuda")
    wrapped = xa.ForceStressOutput(model, compute_stress=False).eval()
    g.plan()
    g.attention_plan()
    if kept:
        g.species_plan(9)

    def step():
        return wrapped(copy.copy(g))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    start = g.atomic_numbers.clone()
    for k in range(4):
        g.atomic_numbers.copy_(start.roll(k))
        graph.replay()
        torch.cuda.synchronize()
        got = {key: static[key].clone() for key in ("energy", "forces")}
        eager = step()
        torch.cuda.synchronize()
        for key, value in got.items():
            assert torch.equal(value, eager[key]), (k, key)


@pytest.mark.gpu
def test_a_backward_pass_whose_plan_a_capture_took_raises():
    """Replays after a write to the numbers would give it others' weights."""
    g = _graph()
    x = torch.randn(g.num_nodes, 8, device="cuda", requires_grad=True)
    w = torch.randn(9, 8, 8, device="cuda")
    out = xa.grouped_linear(x, w, g.species_plan(9))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g.species_plan(9)
    with pytest.raises(RuntimeError, match="inplace operation"):
        out.sum().backward()
    xa.grouped_linear(x, w, g.species_plan(9)).sum().backward()
    assert x.grad.isfinite().all()


@pytest.mark.gpu
def test_inference_numbers_that_were_written_to():
    with torch.inference_mode():
        ids = torch.tensor([1, 6, 8, 1], device="cuda")
        g = Graph()
        g.atomic_numbers = ids
        FF.species_plan_for(g, 9)
        ids[0] = 8
        assert torch.equal(FF.species_plan_for(g, 9).rows, xa.group_plan(ids, 9).rows)
