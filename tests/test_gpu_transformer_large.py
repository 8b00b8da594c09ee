"""Tensors of more than 2^31 elements: the last rows, tokens and elements are where they belong."""
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
