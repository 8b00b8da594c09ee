"""Attention with a sliding window and sinks against the formula in 64 bits: sizes on both sides of
the tiles, every window, shared heads, padded batches, strides, special values, gradients."""
import math

import pytest
import torch

import monet_amd.lm_ops as lm_ops
from monet_amd import _lib

pytestmark = pytest.mark.gpu
at = lm_ops.attention
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
OPERAND = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DENORMAL = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def make(cuda, B, T, H, K, D, dtype, seed=0, scale=1.0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    r = lambda h: (torch.randn(B, T, h, D, device=cuda, generator=g) * scale).to(dtype)
    return r(H), r(K), r(K), r(H)


def visible(T, n, left, right, sinks, dev):
    i, j = torch.arange(T, device=dev)[:, None], torch.arange(T, device=dev)[None]
    see = (i < n) & (j < n)
    if right >= 0:
        see &= j <= i + right
    if left >= 0:
        see &= (j >= i - left) | (j < sinks)
    return see


def check(q, k, v, g, left, right, sinks, lengths, scale, got):
    """Compares with the formula, head by head.  Bounds (u = 2^-24, h = the half step to which P and
    dS are rounded as operands of 16-bit products, 0 for fp32; n = terms of a sum):
      scores     |s - s'| <= (D + 8) u E, E = max_j scale sum_d |q k|
      P          relative: twice that, n + 40 roundings of the sum and the quotient, 3 u |lse|: eP
      out        sum_j P |v| (eP + h + n u)
      delta      sum_d |do| |o| (half step of o + D u)
      dP         D u sum_d |do| |v|
      dS         P (|dP - delta| (eP + 3 u) + both errors), then h |dS|
      dq, dk, dv sums of those with |k|, |q|, |do|, n u of the terms more
    A 16-bit result is rounded once more, and fp16 operands below 2^-14 keep 2^-25 absolutely."""
    out, lse, dq, dk, dv = got
    B, T, H, D = q.shape
    K = k.shape[2]
    dt = q.dtype
    hf, h, tiny = HALF[dt], OPERAND[dt], DENORMAL[dt]
    scale = 1 / math.sqrt(D) if scale is None else scale
    worst = {}

    def near(name, a, b, bound):
        a = a.double()
        lim = bound * 1.01 + b.abs() * hf + (DENORMAL[dt] if name != "lse" else 0.0)
        err = (a - b).abs()
        ok = (err <= lim) | (a == b)
        assert bool(ok.all()), (name, float((err / lim)[~ok].max()))
        if (lim > 0).any():
            worst[name] = max(worst.get(name, 0.0), float((err / lim.clamp_min(1e-300))[a != b].max())
                              if bool((a != b).any()) else 0.0)

    for b in range(B):
        n = T if lengths is None else int(lengths[b])
        see = visible(T, n, left, right, sinks, q.device)
        rows = torch.arange(T, device=q.device) < n
        dk_sum = torch.zeros(2, T, K, D, device=q.device, dtype=torch.float64)
        dv_sum = torch.zeros_like(dk_sum)
        for hh in range(H):
            c = hh * K // H
            clean = lambda t: torch.where(rows[:, None], t.double(), 0.0)
            qd, kd, vd, gd = clean(q[b, :, hh]), clean(k[b, :, c]), clean(v[b, :, c]), clean(g[b, :, hh])
            s = (qd @ kd.t().contiguous()) * scale
            s = s.masked_fill(~see, -math.inf)
            z = torch.logsumexp(s, 1)
            P = torch.where(see, torch.exp(s - torch.where(rows, z, 0.0)[:, None]), 0.0)
            E = (scale * (qd.abs() @ kd.abs().t().contiguous())).masked_fill(~see, 0.0).amax(1)
            cnt = see.sum(1).double()
            zz = torch.where(rows, z, 0.0).abs()
            eP = U * (2 * (D + 8) * E + cnt + 40 + 3 * zz)
            o = P @ vd
            Pv = P @ vd.abs()
            eo = Pv * (eP + h + cnt * U)[:, None] + tiny * (see.double() @ vd.abs())
            near("out", out[b, :, hh], o, eo)
            fin = lse[b, hh][rows].double()
            near("lse", fin, z[rows], (eP + 4 * U * (1 + zz))[rows])
            assert bool((lse[b, hh][~rows] == -math.inf).all())
            if dq is None:
                continue
            dP = gd @ vd.t().contiguous()
            delta = (gd * o).sum(1, keepdim=True)
            e_delta = (gd.abs() * (o.abs() * (hf + D * U) + eo)).sum(1, keepdim=True)
            e_dP = D * U * (gd.abs() @ vd.abs().t().contiguous())
            dS = P * (dP - delta)
            e_dS = P * ((dP - delta).abs() * (eP + 3 * U)[:, None] + e_dP + e_delta)
            e_dS = e_dS + h * (dS.abs() + e_dS) + torch.where(see, tiny, 0.0)
            near("dq", dq[b, :, hh], scale * (dS @ kd),
                 scale * ((e_dS + (cnt * U)[:, None] * dS.abs()) @ kd.abs()))
            terms = (see.sum(0).double() * H / K + 40) * U
            dk_sum[0, :, c] += scale * (dS.t().contiguous() @ qd)
            dk_sum[1, :, c] += scale * ((e_dS + terms[None] * dS.abs()).t().contiguous() @ qd.abs())
            dv_sum[0, :, c] += P.t().contiguous() @ gd
            dv_sum[1, :, c] += (P * (eP[:, None] + h + terms[None]) + torch.where(see, tiny, 0.0)
                                ).t().contiguous() @ gd.abs()
        if dq is not None:
            near("dk", dk[b], *dk_sum)
            near("dv", dv[b], *dv_sum)
    return worst


def run(q, k, v, g, left=-1, right=0, sinks=0, lengths=None, scale=None, backward=True):
    how = dict(left=left, right=right, sinks=sinks, lengths=lengths, scale=scale)
    out, lse = at.window_attention_forward(q, k, v, **how)
    assert out.dtype == q.dtype and out.is_contiguous() and lse.dtype == torch.float32
    grads = at.window_attention_backward(g, q, k, v, out, lse, **how) if backward else (None,) * 3
    return (out, lse) + tuple(grads)


TYPES = [torch.float32, torch.bfloat16, torch.float16]
WINDOWS = [(-1, 0, 0), (-1, -1, 0), (7, 0, 2), (0, 0, 0), (0, 0, 1), (40, 40, 1), (5, 90, 70), (100, 3, 0),
           (-1, 5, 3), (64, 0, 1000)]


@pytest.mark.parametrize("T", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 257, 385])
@pytest.mark.parametrize("dtype", TYPES)
def test_lengths_and_windows(cuda, T, dtype):
    for w, (left, right, sinks) in enumerate(WINDOWS):
        q, k, v, g = make(cuda, 2, T, 2, 1, 64, dtype, seed=T + w)
        lengths = torch.tensor([T, T // 2], device=cuda, dtype=torch.int32) if w % 2 else None
        got = run(q, k, v, g, left, right, sinks, lengths)
        check(q, k, v, g, left, right, sinks, lengths, None, got)


@pytest.mark.parametrize("D", [1, 2, 7, 8, 16, 31, 32, 33, 40, 64, 72, 80, 96, 97, 100, 120, 127, 128])
@pytest.mark.parametrize("dtype", TYPES)
def test_head_sizes(cuda, D, dtype):
    for T, H, K in ((70, 3, 3), (141, 4, 2)):
        q, k, v, g = make(cuda, 1, T, H, K, D, dtype, seed=D)
        check(q, k, v, g, 50, 0, 3, None, None, run(q, k, v, g, 50, 0, 3))


@pytest.mark.parametrize("H,K", [(1, 1), (6, 6), (8, 2), (5, 1), (12, 4)])
@pytest.mark.parametrize("dtype", TYPES)
def test_shared_heads(cuda, H, K, dtype):
    q, k, v, g = make(cuda, 2, 150, H, K, 48, dtype, seed=H)
    check(q, k, v, g, -1, 0, 0, None, 0.3, run(q, k, v, g, -1, 0, 0, scale=0.3))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,left,right,sinks", [(1100, 60, 0, 1), (1500, 100, 0, 3), (2600, 64, 10, 200),
                                                (3000, 1, 0, 128), (2049, 0, 0, 129), (1300, 500, 0, 4),
                                                (8300, 0, 0, 1000)])
def test_sinks_split_over_their_queries(cuda, T, left, right, sinks, dtype):
    """Sequences long enough that the sinks' gradients are partial sums of several workgroups."""
    q, k, v, g = make(cuda, 2, T, 2, 1, 64, dtype, seed=T)
    lengths = torch.tensor([T, T - 700], device=cuda, dtype=torch.int32)
    got = run(q, k, v, g, left, right, sinks, lengths)
    check(q, k, v, g, left, right, sinks, lengths, None, got)
    for p, s in zip(got, run(q, k, v, g, left, right, sinks, lengths)):
        assert torch.equal(p, s)    # sums in a fixed order


@pytest.mark.parametrize("dtype", TYPES)
def test_padded_batches(cuda, dtype):
    """Lengths of zero, one, the whole; behind them NaN, which is neither read nor passed on."""
    T = 140
    lens = [0, 1, 2, 64, 65, 128, 139, 140]
    q, k, v, g = make(cuda, len(lens), T, 4, 2, 40, dtype)
    lengths = torch.tensor(lens, device=cuda, dtype=torch.int32)
    for b, n in enumerate(lens):
        for t in (q, k, v, g):
            t[b, n:] = float("nan")
    for left, right, sinks in ((-1, -1, 0), (30, 0, 2), (3, 3, 0)):
        got = run(q, k, v, g, left, right, sinks, lengths)
        check(q, k, v, g, left, right, sinks, lengths, None, got)
        for t in (got[0],) + got[2:]:
            for b, n in enumerate(lens):
                assert bool((t[b, n:] == 0).all())
    # lengths beyond the tensor mean all of it, negative ones nothing
    wild = torch.tensor([-5, 1000] + lens[2:], device=cuda, dtype=torch.int32)
    q, k, v, g = make(cuda, len(lens), T, 4, 2, 40, dtype)
    tame = wild.clamp(0, T)
    for p, s in zip(run(q, k, v, g, 30, 0, 2, wild), run(q, k, v, g, 30, 0, 2, tame)):
        assert torch.equal(p, s)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(cuda, dtype):
    """Views of one projection, heads before tokens, odd starts, a broadcast key head."""
    B, T, H, K, D = 2, 90, 4, 2, 24
    g = make(cuda, B, T, H, K, D, dtype)[3]
    packed = torch.randn(B, T, H + 2 * K, D + 1, device=cuda).to(dtype)
    heads_first = torch.randn(3, B, H, T, D, device=cuda).to(dtype)
    odd = torch.randn(1 + 3 * B * T * H * D, device=cuda).to(dtype)[1:].view(3, B, T, H, D)
    every_other = torch.randn(3, B, T, H, 2 * D, device=cuda).to(dtype)[..., ::2]
    sets = [(packed[:, :, :H, 1:], packed[:, :, H:H + K, 1:], packed[:, :, H + K:, :D]),
            tuple(t.transpose(1, 2) for t in heads_first), tuple(odd), tuple(every_other),
            (odd[0], odd[1][:, :, :1].expand(-1, -1, H, -1), odd[2][:, :, :1].expand(-1, -1, H, -1)),
            (odd[0].flip(1).contiguous().flip(1), odd[1], odd[1])]
    for q, k, v in sets:
        want = run(q.contiguous(), k.contiguous(), v.contiguous(), g, 20, 0, 1)
        got = run(q, k, v, g.transpose(1, 2).contiguous().transpose(1, 2), 20, 0, 1)
        for p, s in zip(got, want):
            assert torch.equal(p, s)


def test_large_scores_and_infinities(cuda):
    for dtype in TYPES:
        # scores of +-1000: one key takes it all, nothing overflows
        q, k, v, g = make(cuda, 1, 130, 1, 1, 64, dtype, scale=8.0)
        got = run(q, k, v, g, 40, 0, 1, scale=2.0)
        assert all(bool(torch.isfinite(t).all()) for t in got)
        check(q, k, v, g, 40, 0, 1, None, 2.0, (got[0], got[1], None, None, None))
        # a NaN key poisons the queries that see it, the others stay what they were
        q, k, v, g = make(cuda, 1, 300, 1, 1, 64, dtype)
        clean = run(q, k, v, g, 10, 0, 0, backward=False)[0]
        k2 = k.clone()
        k2[0, 200] = float("nan")
        out = run(q, k2, v, g, 10, 0, 0, backward=False)[0]
        assert bool(torch.isnan(out[0, 200:211]).all())
        assert torch.equal(out[0, :200], clean[0, :200]) and torch.equal(out[0, 211:], clean[0, 211:])


def test_against_differences(cuda):
    """fp32 gradients against central differences of the operator's own forward: step 2^-6,
    truncation below 2^-12 of the third derivative, rounding 2^-24 * 64 of the loss's scale."""
    q, k, v, g = make(cuda, 1, 37, 2, 1, 16, torch.float32)
    lengths = torch.tensor([33], device=cuda, dtype=torch.int32)
    how = dict(left=9, right=2, sinks=2, lengths=lengths)
    _, _, dq, dk, dv = run(q, k, v, g, **how)

    def loss(*qkv):
        return float((at.window_attention_forward(*qkv, **how)[0].double() * g.double()).sum())

    h = 2.0 ** -6
    for which, grad in enumerate((dq, dk, dv)):
        for e in range(0, grad.numel(), 53):
            step = torch.zeros_like(grad)
            step.view(-1)[e] = h
            lo, hi = [q, k, v], [q, k, v]
            lo[which], hi[which] = lo[which] - step, hi[which] + step
            num = (loss(*hi) - loss(*lo)) / (2 * h)
            assert abs(num - float(grad.reshape(-1)[e])) < 2e-3 * (1 + abs(num)), (which, e)


def test_long_sequence_properties(cuda):
    """16000 tokens: rows of probabilities sum to one (v = 1), a window's result is that of the
    window cut out, and sum_i dv = sum_i do where every row sums to one."""
    T = 16000
    for dtype in (torch.bfloat16, torch.float32):
        q, k, v, g = make(cuda, 1, T, 2, 1, 128, dtype)
        ones = torch.ones_like(v)
        out, lse, dq, dk, dv = run(q, k, ones, g, 512, 0, 4)
        assert float((out.double() - 1).abs().max()) <= HALF[dtype] + 700 * (OPERAND[dtype] / 16 + U)
        # do v^T is the same for every key: dS is 0 but for roundings of dP and delta
        full = run(q, k, v, g, 100, 0, 0)
        at_end = slice(T - 200, T)
        part = run(*(t[:, T - 400:] for t in (q, k, v, g)), 100, 0, 0)
        # (tiles start elsewhere: the order of the sums differs)
        assert float((full[0][:, at_end] - part[0][:, 200:]).abs().max()) < 8 * max(HALF[dtype], 64 * U)
        s = full[4].double().sum((0, 1, 2)) - g.double().sum((0, 1, 2))
        # 3.2e4 roundings of do-sized terms, independent: six times their root
        assert float(s.abs().max()) < 6 * (2 * T) ** 0.5 * 2 * max(HALF[dtype], 64 * U) * 3


@pytest.mark.parametrize("D", [64, 128])
def test_graph_capture_and_streams(cuda, D):
    q, k, v, g = make(cuda, 2, 1400, 4, 2, D, torch.bfloat16)
    lengths = torch.tensor([1400, 900], device=cuda, dtype=torch.int32)
    how = dict(left=100, right=0, sinks=4, lengths=lengths)
    want = run(q, k, v, g, **how)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run(q, k, v, g, **how)
    torch.cuda.current_stream().wait_stream(s)
    for p, r in zip(want, got):
        assert torch.equal(p, r)
    graphs = []
    for _ in range(2):          # two graphs, each with a workspace of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, run(q, k, v, g, **how)))
        graphs[-1] = (graph, graphs[-1][1])
    for seed in (1, 2, 3):
        for t, new in zip((q, k, v, g), make(cuda, 2, 1400, 4, 2, D, torch.bfloat16, seed)):
            t.copy_(new)
        lengths.copy_(torch.tensor([1400 - 300 * seed, 900 + seed], dtype=torch.int32))
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = run(q, k, v, g, **how)
        for _, got in graphs:
            for p, r in zip(want, got):
                assert torch.equal(p, r)


def test_empty(cuda):
    for B, T in ((0, 5), (3, 0)):
        q, k, v, g = make(cuda, B, T, 4, 2, 16, torch.float32)
        out, lse, dq, dk, dv = run(q, k, v, g, 3, 0, 1)
        assert out.shape == dq.shape == (B, T, 4, 16) and dk.shape == dv.shape == (B, T, 2, 16)
        assert lse.shape == (B, 4, T)


def test_refusals(cuda):
    q, k, v, g = make(cuda, 2, 10, 4, 2, 16, torch.float32)
    fwd, bwd = at.window_attention_forward, at.window_attention_backward
    out, lse = fwd(q, k, v)
    n = torch.tensor([10, 5], device=cuda, dtype=torch.int32)
    for call, text in [
            (lambda: fwd(q[0], k, v), "must be"),
            (lambda: fwd(q, k, v[:, :, :1]), "must be"),
            (lambda: fwd(q, k[:, :9], v[:, :9]), "differ in batch"),
            (lambda: fwd(q, k[..., :8], v[..., :8]), "differ in batch"),
            (lambda: fwd(q[:, :, :3], k, v), "evenly"),
            (lambda: fwd(q, k.half(), v), "dtype"),
            (lambda: fwd(q.double(), k.double(), v.double()), "dtype"),
            (lambda: fwd(q, k, v, left=-2), "left and right"),
            (lambda: fwd(q, k, v, right=-3), "left and right"),
            (lambda: fwd(q, k, v, sinks=-1), "sinks"),
            (lambda: fwd(q, k, v, scale=0.0), "scale"),
            (lambda: fwd(q, k, v, scale=-1.0), "scale"),
            (lambda: fwd(q, k, v, scale=float("nan")), "scale"),
            (lambda: fwd(q, k, v, lengths=n.long()), "dtype"),
            (lambda: fwd(q, k, v, lengths=n[:1]), "one number per sequence"),
            (lambda: fwd(q, k, v, lengths=n.cpu()), "GPU tensor"),
            (lambda: fwd(*make(cuda, 1, 3, 1, 1, 129, torch.float32)[:3]), "unsupported"),
            (lambda: bwd(g[:, :5], q, k, v, out, lse), "grad_output"),
            (lambda: bwd(g.half(), q, k, v, out, lse), "dtype"),
            (lambda: bwd(g, q, k, v, out, lse.transpose(1, 2)), "lse")]:
        with pytest.raises(RuntimeError, match=text):
            call()
