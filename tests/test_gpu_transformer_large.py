"""Tensors of more than 2^31 elements and batches of more workgroups than a launch takes: the last
rows, tokens, elements and sequences are where they belong."""
import pytest
import torch

import monet_amd.lm_ops as lm_ops

pytestmark = pytest.mark.gpu


def test_layer_norm(cuda):
    D, rows = 1032, (1 << 21) + 3          # 2.2e9 elements
    x = torch.empty(rows, D, device=cuda, dtype=torch.bfloat16)
    x.view(-1)[: 1 << 30].normal_()
    x.view(-1)[1 << 30:].normal_()
    w, b = torch.rand(D, device=cuda) + 0.5, torch.randn(D, device=cuda)
    y, mean, rstd = lm_ops.layernorm.layer_norm_forward(x, D, w, b)
    dx, dw, db = lm_ops.layernorm.layer_norm_backward(y, x, mean, rstd, w, b)
    tail = x[-40:].clone()
    ty, tm, tr = lm_ops.layernorm.layer_norm_forward(tail, D, w, b)
    assert torch.equal(y[-40:], ty) and torch.equal(mean[-40:], tm) and torch.equal(rstd[-40:], tr)
    tdx = lm_ops.layernorm.layer_norm_backward(ty, tail, tm, tr, w, b)[0]
    assert torch.equal(dx[-40:], tdx)
    del dx
    # db = sum of y over 2.1e6 rows: chains of 2^21 / 4096 additions and a few dozen more
    step, want, size = 1 << 18, torch.zeros(D, device=cuda, dtype=torch.float64), torch.zeros(D, device=cuda)
    size = size.double()
    for r in range(0, rows, step):
        part = y[r:r + step].double()
        want += part.sum(0)
        size += part.abs().sum(0)
    assert bool(((db.double() - want).abs() <= 600 * 2.0 ** -24 * size).all())


def test_rotary(cuda):
    T, H, D = (1 << 20) + 5, 16, 130       # 2.2e9 elements
    x = torch.empty(1, T, H, D, device=cuda, dtype=torch.bfloat16)
    x.view(-1)[: 1 << 30].normal_()
    x.view(-1)[1 << 30:].normal_()
    pos = torch.arange(T, device=cuda)[None]
    for interleaved in (False, True):
        y = lm_ops.rotary.rotary_forward(x, pos, (64,), interleaved=interleaved)
        tail = lm_ops.rotary.rotary_forward(x[:, -70:].clone(), pos[:, -70:], (64,), interleaved=interleaved)
        assert torch.equal(y[:, -70:], tail)
        del y


def test_attention(cuda):
    """A window of 64 over a million tokens: the end equals that of the last thousand alone, up to
    the order of sums (two roundings of bf16 at most between them), and the sink's share of every
    row's weight adds up."""
    T, H, D = (1 << 20) + 77, 16, 128      # 2.1e9 elements
    q = torch.empty(1, T, H, D, device=cuda, dtype=torch.bfloat16)
    q.view(-1)[: 1 << 30].normal_()
    q.view(-1)[1 << 30:].normal_()
    k = torch.randn(1, T, 2, D, device=cuda).bfloat16()
    v = torch.randn(1, T, 2, D, device=cuda).bfloat16()
    how = dict(left=64, right=0, sinks=0)
    out, lse = lm_ops.attention.window_attention_forward(q, k, v, **how)
    cut = [t[:, -1024:].clone() for t in (q, k, v)]
    o, l = lm_ops.attention.window_attention_forward(*cut, **how)
    assert float((out[:, -900:].float() - o[:, -900:].float()).abs().max()) < 2 * 2.0 ** -8 * 8
    assert float((lse[:, :, -900:] - l[:, :, -900:]).abs().max()) < 1e-4
    dq, dk, dv = lm_ops.attention.window_attention_backward(out, q, k, v, out, lse, **how)
    cq, ck, cv = lm_ops.attention.window_attention_backward(o, *cut, o, l, **how)
    for a, b in ((dq, cq), (dk, ck), (dv, cv)):
        scale = float(b.float().abs().max())
        assert float((a[:, -800:].float() - b[:, -800:].float()).abs().max()) < 8 * 2.0 ** -8 * scale


def test_attention_of_more_workgroups_than_a_launch_takes(cuda):
    """Many short sequences: a batch that is run in parts.  A sequence's result does not depend on
    the batch around it, so small batches taken out of it give the same bits."""
    B, T, H, K, D = 720_000, 3, 8, 4, 8     # a part is at most 2^32 / 256 / 6 / 8 = 349 525 entries
    q = torch.randn(B, T, H, D, device=cuda, dtype=torch.float16)
    k, v = (torch.randn(B, T, K, D, device=cuda, dtype=torch.float16) for _ in range(2))
    lengths = torch.randint(0, T + 1, (B,), device=cuda, dtype=torch.int32)
    how = dict(left=1, right=0, sinks=1)
    fwd, bwd = lm_ops.attention.window_attention_forward, lm_ops.attention.window_attention_backward
    out, lse = fwd(q, k, v, lengths=lengths, **how)
    grads = bwd(q, q, k, v, out, lse, lengths=lengths, **how)
    for b in (0, 349_500, 699_000, B - 100):
        cut = lambda t: t[b:b + 100]
        o, l = fwd(cut(q), cut(k), cut(v), lengths=cut(lengths), **how)
        assert torch.equal(cut(out), o) and torch.equal(cut(lse), l), b
        for name, a, c in zip("qkv", grads, bwd(cut(q), cut(q), cut(k), cut(v), o, l, lengths=cut(lengths), **how)):
            assert torch.equal(cut(a), c), (b, name)
