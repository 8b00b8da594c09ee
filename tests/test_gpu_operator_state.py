"""Memory of a scheduled model with attention and layer norm against what its plan counts."""
import pytest
import torch

from monet_amd.graph import Graph
from monet_amd.schedule import Schedule
from monet_amd.solver import Model
from monet_amd.solver_info import SolverInfo
from test_operator_state import LAYERS, T, WIDTH, Stack

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode, frac", [("normal", 1.5), ("normal", 0.7), ("multiway_newnode", 0.6)])
def test_a_step_stays_within_its_budget(cuda, mode, frac):
    """Measured costs and a budget below what the model takes; heads of two elements, where attention's
    fp32 logarithms are half of its output.  The allocator rounds each tensor up to 512 bytes: at most
    20 per graph node (an operator's arguments, outputs and gradients)."""
    torch.manual_seed(0)
    bs = 2048
    model = Stack().to(cuda)
    graph = Graph.create(Stack(), (T, WIDTH))
    si = SolverInfo(bs, "stack", mode)
    x = torch.randn(bs, T, WIDTH, device=cuda)
    state = list(model.state_dict(keep_vars=True).values())
    si.extract(graph, x, *state)
    total = sum(n.mem for i, n in si.nodes.items() if i < si.loss) + si.nodes[si.loss].fixed_mem
    budget = frac * total / 2 ** 30
    sched = Schedule(graph, si)
    sched.init_schedule(Model(si, budget, time_limit=60, mip_rel_gap=0.1).solve(), si.mode)
    gout = torch.randn(bs, T, 3, device=cuda)

    def step():
        for p in model.parameters():
            p.grad = None
        sched.backward(sched.forward(x, *state).mul(0).add(gout))

    step()
    rounding = 512 * 20 * len(graph.nodes)
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    outside = held - sum(t.numel() * t.element_size() for t in [x] + state) - gout.numel() * 4
    torch.cuda.reset_peak_memory_stats()
    step()
    torch.cuda.synchronize()
    # (two products of the model's output are this test's own)
    peak = torch.cuda.max_memory_allocated() - outside - 3 * gout.numel() * 4
    assert peak <= budget * 2 ** 30 + rounding, (peak, budget * 2 ** 30)
    # nothing but the gradients stays behind a step
    assert torch.cuda.memory_allocated() <= held + rounding
    for p in model.parameters():
        p.grad = None
    assert torch.cuda.memory_allocated() <= outside + sum(
        t.numel() * t.element_size() for t in [x, gout] + state) + rounding
