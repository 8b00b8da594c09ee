"""The transformer-block operators at large sizes and through a schedule, against 64 bits."""
import copy

import pytest
import torch
import torch.nn as nn

import monet_amd.lm_ops as lm_ops
from monet_amd import functional as MF
from test_gpu_attention import check, make, run

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def test_layer_norm_parameter_gradients_of_many_rows(cuda):
    """2^21 + 3 rows of 1032 in bf16: 1024 workgroups of one row at a time, so a sum is a chain of 2049
    additions, joined by 1024 / 32 + 5 more, then rounded; dw's terms are four roundings each (x - mean,
    times rstd, times grad; mean and rstd are the kernel's own)."""
    D, rows = 1032, (1 << 21) + 3
    x = torch.empty(rows, D, device=cuda, dtype=torch.bfloat16)
    g = torch.empty_like(x)
    for t in (x, g):
        t.view(-1)[: 1 << 30].normal_()
        t.view(-1)[1 << 30:].normal_()
    x[:, 5] += 3
    g += 0.25
    w = torch.ones(D, device=cuda)
    _, mean, rstd = lm_ops.layernorm.layer_norm_forward(x, D, w, w)
    _, dw, db = lm_ops.layernorm.layer_norm_backward(g, x, mean, rstd, w, w, need_input=False)
    want, size = torch.zeros(2, 2, D, device=cuda, dtype=torch.float64)
    for r in range(0, rows, 1 << 18):
        part = slice(r, r + (1 << 18))
        gp = g[part].double()
        xh = (x[part].double() - mean[part].double()[:, None]) * rstd[part].double()[:, None]
        for k, terms in enumerate((gp * xh, gp)):
            want[k] += terms.sum(0)
            size[k] += terms.abs().sum(0)
    for k, got in enumerate((dw, db)):
        assert bool(((got.double() - want[k]).abs() <= (2049 + 37 + 5) * U * size[k]).all()), k


@pytest.mark.parametrize("mean", [0.0, 1.0])
def test_sinks_of_a_million_tokens(cuda, mean):
    """2^31 elements: the gradients of the sinks, which every query sees, are sums over workgroups all
    along the sequence.  Against 64 bits from the kernel's own lse and output.  Per term (8 heads x 2^20
    queries): P within 2 (D + 8) u E + 4 u |lse|, rounded to bf16 (2^-8) as is dS; dP within D u of its
    sum of magnitudes; a workgroup adds at most 2^17 terms in a chain, and 129 parts are joined.  (With
    queries and gradients of mean one the terms do not cancel, and the bound is a small part of the sum.)"""
    T, H, K, D, sinks = (1 << 20) + 77, 16, 2, 128, 3
    q, g = (torch.empty(1, T, H, D, device=cuda, dtype=torch.bfloat16) for _ in range(2))
    for t in (q, g):
        t.view(-1)[: 1 << 30].normal_(mean)
        t.view(-1)[1 << 30:].normal_(mean)
    k, v = (torch.randn(1, T, K, D, device=cuda).bfloat16() for _ in range(2))
    k[:, :sinks] *= 3                                     # they get a share of every row's weight
    how = dict(left=64, right=0, sinks=sinks)
    out, lse = lm_ops.attention.window_attention_forward(q, k, v, **how)
    _, dk, dv = lm_ops.attention.window_attention_backward(g, q, k, v, out, lse, **how)
    scale, h = D ** -0.5, 2.0 ** -8
    sums = torch.zeros(2, 2, K, sinks, D, device=cuda, dtype=torch.float64)      # dk / dv; value, bound
    share, chain = 0.0, (2 ** 17 + 200) * U
    for r in range(0, T, 1 << 15):
        part = slice(r, min(r + (1 << 15), T))
        i = torch.arange(part.start, part.stop, device=cuda)
        see = i[:, None] >= torch.arange(sinks, device=cuda)
        for hh in range(H):
            c = hh // (H // K)
            kd, vd = k[0, :sinks, c].double(), v[0, :sinks, c].double()
            qd, gd, od = q[0, part, hh].double(), g[0, part, hh].double(), out[0, part, hh].double()
            z = lse[0, hh, part].double()[:, None]
            s = scale * (qd @ kd.t().contiguous())
            P = torch.where(see, torch.exp(s - z), 0.0)
            eP = U * (2 * (D + 8) * scale * (qd.abs() @ kd.abs().t().contiguous()) + 4 * z.abs() + 8)
            dP, delta = gd @ vd.t().contiguous(), (gd * od).sum(1, keepdim=True)
            e_dP = 2 * D * U * (gd.abs() @ vd.abs().t().contiguous() + (gd * od).abs().sum(1, keepdim=True))
            dS = P * (dP - delta)
            e_dS = P * ((dP - delta).abs() * eP + e_dP) + (h + chain) * dS.abs()
            sums[0, 0, c] += scale * (dS.t().contiguous() @ qd)
            sums[0, 1, c] += scale * (e_dS.t().contiguous() @ qd.abs())
            sums[1, 0, c] += P.t().contiguous() @ gd
            sums[1, 1, c] += (P * (eP + h + chain)).t().contiguous() @ gd.abs()
            share = max(share, float(P.sum(1).min()) if r else 0.0)
    assert share > 0
    for got, (want, bound) in zip((dk, dv), sums):
        err = (got[0, :sinks].double() - want.transpose(0, 1)).abs()
        assert bool((err <= 1.1 * bound.transpose(0, 1) + h * want.transpose(0, 1).abs()).all())
        if mean:
            assert bool((bound < 0.25 * want.abs().amax(-1, keepdim=True)).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values_of_one_over_a_long_sequence(cuda, dtype):
    """16000 tokens with v = 1, where every row of probabilities sums to one and dS vanishes: all
    results against 64 bits, dq and dk among them."""
    q, k, v, g = make(cuda, 1, 16000, 2, 1, 128, dtype)
    ones = torch.ones_like(v)
    got = run(q, k, ones, g, 512, 0, 4)
    check(q, k, ones, g, 512, 0, 4, None, None, got)
    # rounding level: |dP - delta| is that of the output, about one step of it
    step = {torch.bfloat16: 2.0 ** -8, torch.float32: 200 * U}[dtype]
    e = (g.double().abs() * ((got[0].double() - 1).abs() + 260 * U)).sum(-1).max()
    lim = float(e) * 128 ** -0.5 * 1.01 + 1e-30
    assert float(got[2].abs().max()) <= lim * float(k.abs().max()) * (1 + step)


class Padded(nn.Module):
    """Attention over sequences of given lengths, a buffer of the model, three times."""

    def __init__(self, batch, tokens, width, heads):
        super().__init__()
        self.tokens, self.heads, self.size = tokens, heads, width // heads
        self.norms = nn.ModuleList(nn.LayerNorm(width) for _ in range(3))
        self.qkv = nn.ModuleList(nn.Linear(width, width) for _ in range(9))
        self.head = nn.Linear(width, 5)
        self.register_buffer("lengths", torch.arange(batch, dtype=torch.int32) * tokens // (batch - 1))

    def forward(self, x):
        for b in range(3):
            n = self.norms[b](x)
            q, k, v = (m(n).view(-1, self.tokens, self.heads, self.size) for m in self.qkv[3 * b:3 * b + 3])
            y = MF.window_attention(q, k, v, left=9, right=3, sinks=2, lengths=self.lengths)
            x = x + torch.flatten(y, 2)
        return self.head(x)


@pytest.mark.parametrize("mode, frac", [("normal", 2.0), ("normal", 0.6), ("multiway_newnode", 0.6)])
def test_lengths_through_a_schedule(cuda, mode, frac):
    """A padded batch, from an empty sequence to a full one: a schedule's results are autograd's."""
    from monet_amd.graph import Graph
    from monet_amd.schedule import _FWD, Schedule
    from monet_amd.solver import Model
    from monet_amd.solver_info import SolverInfo
    from test_solver import synthetic_cost
    torch.manual_seed(4)
    bs, tokens, width = 9, 70, 32
    model = Padded(bs, tokens, width, 4)
    graph = Graph.create(model, (tokens, width))
    model = model.to(cuda)
    x, gout = torch.randn(bs, tokens, width, device=cuda), torch.randn(bs, tokens, 5, device=cuda)
    y0 = model(x)
    y0.backward(gout)
    want = {n: p.grad.clone() for n, p in model.named_parameters()}
    si = SolverInfo(bs, "padded", mode)
    si.extract(graph, cost_fn=synthetic_cost(si))
    total = sum(n.mem for i, n in si.nodes.items() if i < si.loss) + si.nodes[si.loss].fixed_mem
    sched = Schedule(graph, si)
    sched.init_schedule(Model(si, frac * total / 2 ** 30, time_limit=60, mip_rel_gap=0.1).solve(), si.mode)
    again = sum(ins[0] == _FWD and type(ins[1]).__name__ == "WindowAttention" for p in sched._plan[1:] for ins in p)
    assert again > 0 or frac > 1
    m = copy.deepcopy(model)
    for lengths in (m.lengths.clone(), m.lengths.flip(0)):       # the buffer is read anew every step
        m.lengths.copy_(lengths)
        for p in m.parameters():
            p.grad = None
        y = sched.forward(x, *m.state_dict(keep_vars=True).values())
        sched.backward(gout)
        if torch.equal(lengths, model.lengths):
            # the same operators in the same order on the same operands, but for sums of gradients
            assert float((y - y0).detach().abs().max()) <= 1e-5 * float(y0.detach().abs().max())
            floor = 1e-3 * max(float(g.abs().max()) for g in want.values())
            for n, p in m.named_parameters():
                off = float((p.grad - want[n]).abs().max() / want[n].abs().max().clamp_min(floor))
                assert off < 2e-5, (n, off)
        else:
            assert not torch.allclose(y, y0)


def test_windows_of_any_number(cuda):
    """Python's numbers do not end at 64 bits: a window beyond the sequence is no limit."""
    q, k, v, g = make(cuda, 1, 150, 2, 1, 16, torch.float32)
    want = run(q, k, v, g, -1, -1, 0)
    for huge in (150, 2 ** 62, 2 ** 63, 2 ** 64 + 3):
        for how in ((huge, huge, 0), (3, huge, huge), (huge, -1, huge)):
            for a, b in zip(run(q, k, v, g, *how), want):
                assert torch.equal(a, b), how
