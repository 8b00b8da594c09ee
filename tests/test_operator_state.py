"""What an operator keeps in `params` for its backward and grows with the batch - the logarithm of the
sums of attention's rows, the statistics of layer norm - is part of the memory the solver plans with,
and the executor lets go of it when the operator's backward has run.  No GPU."""
import weakref

import pytest
import torch
import torch.nn as nn

import monet_amd.lm_ops as lm_ops
from monet_amd import functional as MF
from monet_amd.graph import Graph
from monet_amd.schedule import _BWD, _FWD, Schedule
from monet_amd.solver import Model
from monet_amd.solver_info import SolverInfo
from test_solver import synthetic_cost

T, HEADS, SIZE, LAYERS = 40, 6, 2, 4
WIDTH = HEADS * SIZE


class Stack(nn.Module):
    """Layer norm over the last or the last two dimensions, then attention."""

    def __init__(self):
        super().__init__()
        self.norms = nn.ModuleList(nn.LayerNorm(WIDTH) if k % 2 else nn.LayerNorm((T, WIDTH)) for k in range(LAYERS))
        self.head = nn.Linear(WIDTH, 3)

    def forward(self, x):
        for norm in self.norms:
            h = norm(x).view(-1, T, HEADS, SIZE)
            x = x + torch.flatten(MF.window_attention(h, h, h, left=5), 2)
        return self.head(x)


def counted_cost(si):
    base = synthetic_cost(si)
    return lambda n, op, bwd_op: (*base(n, op, bwd_op), si.state_bytes(op, n))


def plan(mode, bs, frac):
    torch.manual_seed(0)
    graph = Graph.create(Stack(), (T, WIDTH))
    si = SolverInfo(bs, "stack", mode)
    si.extract(graph, cost_fn=counted_cost(si))
    total = sum(n.mem for i, n in si.nodes.items() if i < si.loss) + si.nodes[si.loss].fixed_mem
    sol = Model(si, frac * total / 2 ** 30, time_limit=60, mip_rel_gap=0.1).solve()
    sched = Schedule(graph, si)
    sched.init_schedule(sol, si.mode)
    return graph, si, sched


@pytest.mark.parametrize("elem", [torch.float32, torch.bfloat16])
def test_the_solver_counts_it(elem):
    bs = 5
    graph = Graph.create(Stack(), (T, WIDTH))
    si = SolverInfo(bs, "stack", "normal")
    si.extract(graph, torch.empty(bs, T, WIDTH, dtype=elem), cost_fn=counted_cost(si))
    eb = si.elem_bytes
    params = 2 * (LAYERS // 2) * (WIDTH + T * WIDTH) + WIDTH * 3 + 3
    leaves = eb * (params + bs * T * WIDTH * 2)      # x is read by the norm and the add
    rows = (LAYERS // 2) * bs * T + (LAYERS // 2) * bs                 # over the last dimension, over both
    states = 4 * LAYERS * bs * HEADS * T + 8 * rows
    assert si.nodes[si.loss].fixed_mem == leaves + states
    # backward: parameter gradients come, states go after their operator's step
    grads, gone = 0, 0
    for i in range(si.loss + 1, len(si.nodes)):
        b = si.nodes[i]
        grads += sum(eb * int(torch.Size(p.shape).numel()) for p in b.stored)
        assert b.fixed_mem == leaves + states + grads - gone, (i, b)
        if b.fwd_node.op == "monet::window_attention":
            gone += 4 * bs * HEADS * T
        elif b.fwd_node.op == "aten::layer_norm":
            gone += 8 * bs * (T if b.fwd_node.args[1].value == [WIDTH] else 1)
    assert gone == states


@pytest.mark.parametrize("mode, frac", [("normal", 2.0), ("normal", 0.6), ("multiway_newnode", 0.6)])
def test_the_executor_holds_no_more(mode, frac, monkeypatch):
    """Two steps with stand-ins for the kernels: what is alive of the states never exceeds what the
    plan counts at that point, and nothing stays behind a step."""
    bs, alive = 3, {}

    def track(t):
        alive[id(t)] = t.numel() * 4
        weakref.finalize(t, alive.pop, id(t))
        return t

    def attention(q, k, v, **how):
        return q * 1.0, track(torch.zeros(q.shape[0], q.shape[2], q.shape[1]))

    def norm(x, shape, w, b, eps):
        lead = x.shape[:x.dim() - len(shape)]
        return x * 1.0, track(torch.zeros(lead)), track(torch.zeros(lead))

    monkeypatch.setattr(lm_ops.attention, "window_attention_forward", attention)
    monkeypatch.setattr(lm_ops.attention, "window_attention_backward",
                        lambda g, q, k, v, out, lse, **how: (g * 1.0, g * 1.0, g * 1.0))
    monkeypatch.setattr(lm_ops.layernorm, "layer_norm_forward", norm)
    monkeypatch.setattr(lm_ops.layernorm, "layer_norm_backward",
                        lambda g, x, m, r, w, b, need: (g * 1.0, w * 0.0, b * 0.0))
    graph, si, sched = plan(mode, bs, frac)
    states = {k: c.state_bytes(n) for k, n in enumerate(graph.nodes) if hasattr(n, "op")
              for c in lm_ops.list_ops("normal", n.op)[:1]}
    counted = sum(-b * bs for b in states.values() if b < 0)
    again = sum(ins[0] == _FWD and states[ins[2]] != 0 for p in sched._plan[1:] for ins in p)
    assert again > 0 or frac > 1
    model = Stack()
    run, left = sched._run, []

    def one_by_one(instructions):
        nonlocal counted
        for ins in instructions:
            run([ins])
            assert sum(alive.values()) <= counted, ins
            if ins[0] == _BWD and ins[5]:
                counted += states[ins[2]] * bs       # (negative: per sample)
                assert sum(alive.values()) <= counted, ins
    monkeypatch.setattr(sched, "_run", one_by_one)
    whole = counted
    for _ in range(2):
        counted = whole
        y = sched.forward(torch.randn(bs, T, WIDTH), *model.state_dict(keep_vars=True).values())
        assert sum(alive.values()) == whole
        sched.backward(torch.ones_like(y))
        assert not alive and counted == 0


def test_profiles_read_from_a_file_count_it(tmp_path):
    """Costs that were written before (a file holds run times and workspaces) give the same plan."""
    graph = Graph.create(Stack(), (T, WIDTH))
    fixed = []
    for _ in range(2):
        si = SolverInfo(4, "stack", "normal", data_dir=tmp_path)
        si.extract(graph, cost_fn=counted_cost(si))
        fixed.append([n.fixed_mem for n in si.nodes.values()])
    assert fixed[0] == fixed[1] and max(n.state_mem for n in si.nodes.values()) == 4 * 4 * HEADS * T
