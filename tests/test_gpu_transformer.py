"""The transformer-block operators together: a model trained through stock autograd with the
differentiable calls, the same model through solved schedules, against 64 bits."""
import copy
import math

import pytest
import torch
import torch.nn as nn

import monet_amd.lm_ops as lm_ops
from monet_amd import functional as MF
from transformer_net import PATCH, TOKENS, PatchNet, cheap_dropout_cost

pytestmark = pytest.mark.gpu


def _rel(a, b, floor):
    return float((a - b).detach().abs().max() / b.detach().abs().max().clamp_min(floor))


def _plain(model, x):
    """PatchNet without dropout in elementary operations, in the tensors' own type."""
    x = model.embed(x)
    T = x.shape[1]
    i, j = torch.arange(T, device=x.device)[:, None], torch.arange(T, device=x.device)[None]
    see = (j <= i + 2) & ((j >= i - 13) | (j < 1))

    def norm(m, t):
        t = (t - t.mean(-1, keepdim=True)) / torch.sqrt(t.var(-1, correction=0, keepdim=True) + m.eps)
        return t if m.weight is None else t * m.weight + m.bias

    def turn(t, pos):
        out = [t[..., k] for k in range(t.shape[-1])]
        pairs, k = 5, 0
        for a, s in enumerate((2, 2, 1)):
            for f in range(s):
                ang = pos[a].to(t.dtype)[None, :, None] * 10000.0 ** (-f / s)
                p, q = t[..., k], t[..., k + pairs]
                out[k], out[k + pairs] = p * ang.cos() - q * ang.sin(), p * ang.sin() + q * ang.cos()
                k += 1
        return torch.stack(out, -1)

    for blk in model.blocks:
        n = norm(blk.norm1, x)
        q, k, v = (m(n).view(x.shape[0], T, -1, blk.size) for m in (blk.q, blk.k, blk.v))
        q, k = turn(q, blk.positions), turn(k, blk.positions)
        k, v = (t.repeat_interleave(blk.heads // blk.shared, 2) for t in (k, v))
        s = torch.matmul(q.transpose(1, 2), k.permute(0, 2, 3, 1).contiguous()) / math.sqrt(blk.size)
        P = torch.softmax(s.masked_fill(~see, -math.inf), -1)
        y = torch.matmul(P, v.transpose(1, 2).contiguous()).transpose(1, 2)
        x = x + blk.out(torch.flatten(y, 2))
        x = x + blk.down(torch.relu(blk.up(norm(blk.norm2, x))))
    return model.head(torch.flatten(norm(model.norm, x), 1))


def _grads(model, y, gout):
    model.zero_grad()
    y.backward(gout)
    return {n: p.grad.clone() for n, p in model.named_parameters()}


def test_autograd_against_64_bits(cuda):
    """fp32 through the differentiable calls against the same model in fp64: relative to a gradient's
    largest entry the two differ by a few hundred roundings (layers of at most 2880 terms)."""
    torch.manual_seed(0)
    model = PatchNet(p=0.0).to(cuda)
    x, gout = torch.randn(6, TOKENS, PATCH, device=cuda), torch.randn(6, 7, device=cuda)
    wide = copy.deepcopy(model).double()
    y, y64 = model(x), _plain(wide, x.double())
    assert _rel(y.double(), y64, 1e-30) < 1e-5
    got, want = _grads(model, y, gout), _grads(wide, y64, gout.double())
    floor = 1e-3 * max(float(g.abs().max()) for g in want.values())
    for n in want:
        assert _rel(got[n].double(), want[n], floor) < 2e-5, n


def _solve(model, mode, bs, cuda, cost=None):
    from monet_amd.graph import Graph, fusion_level
    from monet_amd.solver_info import SolverInfo
    graph = Graph.create(copy.deepcopy(model).cpu(), (TOKENS, PATCH), fuse_bn_relu=fusion_level(mode))
    si = SolverInfo(bs, "patch", mode)
    if cost is None:     # measured on the GPU
        si.extract(graph, torch.randn(bs, TOKENS, PATCH, device=cuda),
                   *list(model.state_dict(keep_vars=True).values()))
    else:
        si.extract(graph, cost_fn=cost(si))
    return graph, si


@pytest.mark.parametrize("mode", ["normal", "inplace_conv_multiway_newnode", "fused_inplace_conv_multiway_newnode"])
def test_schedules_match_autograd_with_dropout(cuda, mode):
    """One seed, one mask: the schedule's output and gradients are autograd's although tight budgets
    run dropouts again, and every step draws new masks."""
    from monet_amd.schedule import _FWD, Schedule
    from monet_amd.solver import Model
    torch.manual_seed(1)
    bs = 64
    model = PatchNet(p=0.3).to(cuda).train()
    x, gout = torch.randn(bs, TOKENS, PATCH, device=cuda), torch.randn(bs, 7, device=cuda)
    want = {}
    for seed in (5, 6):
        torch.manual_seed(seed)
        y = model(x)
        want[seed] = y.detach(), _grads(model, y, gout)
    assert not torch.allclose(want[5][0], want[6][0])
    graph, si = _solve(model, mode, bs, cuda, cheap_dropout_cost)
    total = sum(n.mem for i, n in si.nodes.items() if i < si.loss) + si.nodes[si.loss].fixed_mem
    again = 0
    for frac in (2.0, 0.6, 0.45):
        sol = Model(si, frac * total / 2 ** 30, time_limit=60, mip_rel_gap=0.1).solve()
        m = copy.deepcopy(model)
        m.zero_grad()
        sched = Schedule(graph, si)
        sched.init_schedule(sol, si.mode)
        again += sum(ins[0] == _FWD and type(ins[1]).__name__ == "CounterDropout"
                     for plan in sched._plan[1:] for ins in plan)
        for seed in (5, 6, 5):
            y0, g0 = want[seed]
            floor = 1e-3 * max(float(g.abs().max()) for g in g0.values())
            torch.manual_seed(seed)
            for p in m.parameters():
                p.grad = None
            y = sched.forward(x, *list(m.state_dict(keep_vars=True).values()))
            assert _rel(y, y0, 1e-30) < 1e-5
            sched.backward(gout)
            for n, p in m.named_parameters():
                assert _rel(p.grad, g0[n], floor) < 2e-5, (frac, seed, n)
    # (with in-place ReLUs the solver gets by without)
    assert again > 0 or mode != "normal"


def test_wrapper_and_evaluation(cuda, tmp_path):
    import pickle
    from monet_amd.monet_wrapper import MONeTWrapper
    from monet_amd.solver import Model
    torch.manual_seed(2)
    model = PatchNet(p=0.25).to(cuda).train()
    graph, si = _solve(model, "multiway_newnode", 8, cuda)
    sol = Model(si, 1.0, time_limit=60, mip_rel_gap=0.05).solve()
    with open(tmp_path / "s.pkl", "wb") as f:
        pickle.dump([si, sol], f)
    net = MONeTWrapper(copy.deepcopy(model), str(tmp_path / "s.pkl"), (TOKENS, PATCH)).cuda()
    x, gout = torch.randn(8, TOKENS, PATCH, device=cuda), torch.randn(8, 7, device=cuda)
    torch.manual_seed(9)
    want = model(x)
    grads = _grads(model, want, gout)
    torch.manual_seed(9)
    got = net(x.clone())
    got.backward(gout)
    assert _rel(got.detach(), want.detach(), 1e-30) < 1e-5
    for n, p in net.model.named_parameters():
        assert _rel(p.grad, grads[n], 1e-3 * max(float(g.abs().max()) for g in grads.values())) < 2e-5, n
    # a model in evaluation mode drops nothing
    model.eval()
    quiet = copy.deepcopy(model)
    for b in quiet.blocks:
        b.p = 0.0
    assert torch.equal(model(x), quiet(x))


def test_low_precision_block_steps(cuda):
    """A bf16 block through the differentiable calls: gradients arrive in the parameters' type and
    follow the fp32 ones to a bf16 network's accuracy (a dozen roundings of 2^-8 along the path,
    each gradient an average over thousands of terms)."""
    torch.manual_seed(3)
    model = PatchNet(p=0.0).to(cuda)
    x, gout = torch.randn(4, TOKENS, PATCH, device=cuda), torch.randn(4, 7, device=cuda)
    want = _grads(model, model(x), gout)
    low = copy.deepcopy(model).bfloat16()
    got = _grads(low, low(x.bfloat16()), gout.bfloat16())
    for n, g in want.items():
        assert got[n].dtype == torch.bfloat16
        num = float((got[n].float() - g).norm() / g.norm().clamp_min(1e-2))
        assert num < 16 * 2.0 ** -8, (n, num)


def test_gradients_only_where_wanted(cuda):
    q, k, v = (torch.randn(1, 20, 2, 16, device=cuda, requires_grad=r) for r in (False, True, False))
    MF.window_attention(q, k, v, left=3).sum().backward()
    assert q.grad is None and v.grad is None and k.grad.shape == k.shape
    x = torch.randn(1, 20, 2, 16, device=cuda, requires_grad=True)
    y = MF.rotary(MF.dropout(x, 0.4), torch.arange(20, device=cuda)[None], (8,))
    y.sum().backward()
    assert x.grad is not None and not bool(torch.isnan(x.grad).any())
    with pytest.raises(RuntimeError, match="once_differentiable|twice"):
        (g,) = torch.autograd.grad(MF.rotary(x, torch.arange(20, device=cuda)[None], (8,)).pow(2).sum(), x,
                                   create_graph=True)
        g.sum().backward()


def test_captured_training_step(cuda):
    """Forward and backward of the operators under one graph, replayed with new inputs: each replay
    equals the eager step with the masks it drew."""
    B, T, H, D = 2, 300, 2, 32
    x, w, b, g = (torch.randn(s, device=cuda) for s in ((B, T, H * D), (H * D,), (H * D,), (B, T, H * D)))
    pos = torch.arange(T, device=cuda)[None]
    L = lm_ops

    def step(state):
        y, mean, rstd = L.layernorm.layer_norm_forward(x, H * D, w, b)
        q = L.rotary.rotary_forward(y.view(B, T, H, D), pos, (16,))
        o, lse = L.attention.window_attention_forward(q, q, q, left=50, sinks=2)
        z = L.dropout.dropout_forward(o.view(B, T, H * D), 0.3, state)
        dz = L.dropout.dropout_backward(g, 0.3, state).view(B, T, H, D)
        dq, dk, dv = L.attention.window_attention_backward(dz, q, q, q, o, lse, left=50, sinks=2)
        dy = L.rotary.rotary_backward(dq + dk + dv, pos, (16,)).view(B, T, H * D)
        return (z,) + L.layernorm.layer_norm_backward(dy, x, mean, rstd, w, b)

    step(L.dropout.dropout_state(cuda))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        state = L.dropout.dropout_state(cuda)
        out = step(state)
    for k in range(4):
        x.copy_(torch.randn_like(x))
        g.copy_(torch.randn_like(g))
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, step(state)):
            assert torch.equal(p, q), k
