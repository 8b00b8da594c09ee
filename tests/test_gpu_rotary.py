"""Rotary positions against rotations in 64 bits: one to three axes, both layouts of the pairs,
both runs of frequencies, far, negative and fractional positions, strides, the inverse."""
import math

import pytest
import torch

import monet_amd.lm_ops as lm_ops

pytestmark = pytest.mark.gpu
ro = lm_ops.rotary
STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def exact(x, positions, sections, base, joint, interleaved, sign=1.0):
    x, n = x.double().cpu(), sum(sections)
    B, T = x.shape[:2]
    pos = positions.double().cpu()
    if pos.dim() == 2:
        pos = pos[:, None].expand(-1, B, -1)
    y = x.clone()
    k = 0
    for a, s in enumerate(sections):
        for i in range(s):
            f = base ** (-k / n if joint else -i / s)
            c, sn = torch.cos(pos[a] * f)[..., None], sign * torch.sin(pos[a] * f)[..., None]
            p, q = (2 * k, 2 * k + 1) if interleaved else (k, k + n)
            y[..., p] = x[..., p] * c - x[..., q] * sn
            y[..., q] = x[..., p] * sn + x[..., q] * c
            k += 1
    return y


def check(got, want, x, far=0.0):
    """An angle is off by 2^-28 turns (1.5 * 2^-25.3 radians) after its reduction and by 2^-52 of
    itself before; sine and cosine round by 2 u more, two products and their sum by 3 u, of a pair
    whose length is at most sqrt(2) max|x|: 8 u of that length in all, then the result's rounding."""
    length = 2 ** 0.5 * x.double().abs().amax(-1, keepdim=True).cpu()
    lim = (8 * 2.0 ** -24 + far * 2.0 ** -52) * length * 1.01 + want.abs() * STEP[got.dtype] + \
        (2.0 ** -25 if got.dtype == torch.float16 else 0)
    err = (got.double().cpu() - want).abs()
    assert bool((err <= lim).all()), float((err / lim).max())


CASES = [  # B, T, H, D, sections
    (1, 1, 1, 2, (1,)),
    (2, 5, 3, 7, (3,)),
    (1, 33, 2, 64, (32,)),
    (3, 12, 4, 64, (16, 16)),
    (2, 50, 1, 80, (10, 11, 12)),
    (1, 17, 5, 96, (0, 20, 20)),
    (70, 3, 2, 33, (5, 7)),
    (2, 130, 12, 256, (64, 64)),
    (5, 9, 3, 24, (0,)),
]


@pytest.mark.parametrize("B,T,H,D,sections", CASES)
@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("interleaved", [False, True])
def test_against_rotations(cuda, B, T, H, D, sections, dtype, interleaved):
    torch.manual_seed(B * T + D)
    x = torch.randn(B, T, H, D, device=cuda).to(dtype)
    for joint in (False, True):
        for pos in (torch.randint(-50, 50, (len(sections), T), device=cuda),
                    torch.randint(0, 900, (len(sections), B, T), device=cuda, dtype=torch.int32),
                    torch.rand(len(sections), T, device=cuda) * 30):
            how = (pos, sections, 1000.0, joint, interleaved)
            y = ro.rotary_forward(x, *how)
            assert y.is_contiguous() and y.dtype == dtype
            check(y, exact(x, *how), x, far=900)
            check(ro.rotary_backward(x, *how), exact(x, *how, sign=-1.0), x, far=900)


def test_far_positions(cuda):
    """A position of 2^40: the angle keeps 2^40 * 2^-52 radians and the result follows."""
    x = torch.randn(1, 64, 2, 32, device=cuda)
    pos = (torch.arange(64, device=cuda) + (1 << 40))[None]
    check(ro.rotary_forward(x, pos, (16,)), exact(x, pos, (16,), 10000.0, False, False), x, far=2.0 ** 42)
    pos = torch.tensor([[10 ** 6, -10 ** 6, 123457]], device=cuda)
    x = x[:, :3]
    check(ro.rotary_forward(x, pos, (16,)), exact(x, pos, (16,), 10000.0, False, False), x, far=2.0 ** 22)


def test_backward_is_the_transpose(cuda):
    """<turn(x), g> = <x, turn_back(g)>, and turning back a turned tensor gives it again."""
    x, g = torch.randn(2, 3, 40, 4, 48, device=cuda).unbind(0)
    pos = torch.arange(40, device=cuda)[None] * 3
    a = float((ro.rotary_forward(x, pos, (20,)).double() * g.double()).sum())
    b = float((x.double() * ro.rotary_backward(g, pos, (20,)).double()).sum())
    n = x.numel()
    # each product carries 16 u of |x| |g| ~ 1, as good as independent: ten times the root of n
    assert abs(a - b) < 10 * 16 * 2.0 ** -24 * n ** 0.5
    back = ro.rotary_backward(ro.rotary_forward(x, pos, (20,)), pos, (20,))
    assert float((back - x).abs().max()) <= 20 * 2.0 ** -24 * 2 ** 0.5 * float(x.abs().max())


def test_strides_and_empty(cuda):
    qkv = torch.randn(3, 11, 9, 24, device=cuda)
    pos = torch.arange(44, device=cuda).view(2, 22)[:, ::2]          # strided positions
    how = (pos, (4, 6))
    for x in (qkv[:, :, 3:6], qkv.transpose(1, 2)[:, :, :4], qkv[..., 1:23], qkv[..., ::2]):
        p = pos if x.shape[1] == 11 else pos[:, :9]
        want = ro.rotary_forward(x.contiguous(), p, how[1]) if x.shape[3] >= 20 else None
        if want is None:
            with pytest.raises(RuntimeError, match="sections"):
                ro.rotary_forward(x, p, how[1])
            want = ro.rotary_forward(x.contiguous(), p, (2, 4))
            assert torch.equal(ro.rotary_forward(x, p, (2, 4)), want)
        else:
            assert torch.equal(ro.rotary_forward(x, p, how[1]), want)
    assert ro.rotary_forward(qkv[:0], pos, (4, 6)).shape == (0, 11, 9, 24)
    assert ro.rotary_forward(qkv[:, :0], pos[:, :0], (4, 6)).shape == (3, 0, 9, 24)
    one = qkv[:1].expand(5, -1, -1, -1)                              # a broadcast batch
    assert torch.equal(ro.rotary_forward(one, pos, (4, 6))[4], ro.rotary_forward(qkv, pos, (4, 6))[0])


def test_refusals(cuda):
    x = torch.randn(1, 4, 2, 8, device=cuda)
    p = torch.zeros(1, 4, device=cuda, dtype=torch.int64)
    for call, text in [
            (lambda: ro.rotary_forward(x[0], p, (2,)), "must be"),
            (lambda: ro.rotary_forward(x, p, (5,)), "sections"),
            (lambda: ro.rotary_forward(x, p, (-1,)), "sections"),
            (lambda: ro.rotary_forward(x, p, ()), "sections"),
            (lambda: ro.rotary_forward(x, p, (1, 1, 1, 1)), "sections"),
            (lambda: ro.rotary_forward(x, p, (1, 1)), "positions"),
            (lambda: ro.rotary_forward(x, p[:, :3], (1,)), "positions"),
            (lambda: ro.rotary_forward(x, p.double(), (1,)), "int64, int32"),
            (lambda: ro.rotary_forward(x, p.cpu(), (1,)), "GPU tensor"),
            (lambda: ro.rotary_forward(x, p, (1,), 0.0), "base"),
            (lambda: ro.rotary_forward(x.double(), p, (1,)), "dtype"),
            (lambda: ro.rotary_forward(torch.zeros(1, 4, 1, 300, device=cuda), p, (129,)), "unsupported")]:
        with pytest.raises(RuntimeError, match=text):
            call()


def test_graph_replays(cuda):
    x = torch.randn(2, 30, 4, 32, device=cuda)
    pos = torch.arange(30, device=cuda)[None].clone()
    ro.rotary_forward(x, pos, (16,))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ro.rotary_forward(x, pos, (16,))
    for k in range(3):
        pos.add_(7)
        x.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ro.rotary_forward(x, pos, (16,)))
