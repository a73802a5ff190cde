"""An attention plan that a capture takes lives on, whatever becomes of the graph's cache (stand-ins for the plan's kernels
and for the capture: no GPU needed)."""
import copy
import gc
import types
import weakref

import pytest
import torch

from xnn_amd import attention
from xnn_amd.plan import captured_plans, hold_captured


class Thing:
    pass


class Counts(Thing):
    device, _version = "device", 0

    def is_inference(self):
        return False


@pytest.mark.parametrize("act", ["write", "atoms", "copy"])
def test_a_plan_that_a_capture_takes_lives_on(monkeypatch, act):
    state = types.SimpleNamespace(capturing=False)
    monkeypatch.setattr(attention, "attention_plan", lambda n_atoms, n: Thing())
    monkeypatch.setattr(torch.cuda, "device", lambda device: torch.no_grad())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state.capturing)
    graph = Thing()
    graph.n_atoms, graph.num_nodes = Counts(), 12
    attention.plan_for(graph)
    state.capturing = True
    plan = weakref.ref(attention.plan_for(copy.copy(graph) if act == "copy" else graph))
    assert plan() is attention.plan_for(graph)
    state.capturing = False
    if act == "atoms":
        graph.num_nodes = 13
    else:
        graph.n_atoms._version += 1
    attention.plan_for(graph)
    gc.collect()
    assert plan() is not None and len(captured_plans(graph.n_atoms)) == 1
    assert not captured_plans(copy.deepcopy(graph).n_atoms)
    del graph
    gc.collect()
    assert plan() is None


def test_a_tensor_that_plans_are_held_for_is_saved_as_any_other():
    import io
    counts = torch.tensor([3, 4])
    hold_captured(counts, Thing())
    file = io.BytesIO()
    torch.save(counts, file)
    file.seek(0)
    assert torch.equal(torch.load(file, weights_only=True), counts) and not captured_plans(torch.tensor([3, 4]))
    # an object of Python that went and came back, the tensor having stayed
    plan = weakref.ref(captured_plans(counts)[0])
    holder = torch.nn.Module()
    holder.register_buffer("counts", counts)
    del counts
    gc.collect()
    assert captured_plans(holder.counts)[0] is plan()
    del holder
    gc.collect()
    assert plan() is None
