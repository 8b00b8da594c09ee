"""Dropout from a counter-based generator: published test vectors of the generator, the mask
against a computation in Python integers, forward and backward, every type and alignment."""
import pytest
import torch

import monet_amd.lm_ops as lm_ops

pytestmark = pytest.mark.gpu
dr = lm_ops.dropout
TYPES = [torch.float32, torch.bfloat16, torch.float16]
M = 0xFFFFFFFF


def philox(c, k):
    """Philox4x32-10 on Python integers."""
    c, k = list(c), list(k)
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & M, (p0 >> 32) ^ c[3] ^ k[1], p0 & M]
        k = [(k[0] + 0x9E3779B9) & M, (k[1] + 0xBB67AE85) & M]
    return c


def test_published_vectors():
    # the known answers that the authors publish with Random123 for ten rounds
    assert philox((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert philox((M, M, M, M), (M, M)) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert philox((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0)) == \
        [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def numbers(n, state):
    seed, off = [v & (2 ** 64 - 1) for v in state]
    out = []
    for g in range((n + 7) // 8):
        hi, lo = (philox((g & M, (g >> 32) | b, off & M, off >> 32), (seed & M, seed >> 32))
                  for b in (0, 1 << 31))
        for e in range(8):
            s = 16 * (e & 1)
            out.append(((hi[e // 2] >> s & 0xFFFF) << 16) | (lo[e // 2] >> s & 0xFFFF))
    return out[:n]


def state(cuda, *v):
    return torch.tensor(v, dtype=torch.int64, device=cuda)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 3, 7, 8, 9, 64, 1001, 4096])
def test_mask_and_values(cuda, dtype, n):
    for p, st in ((0.0, (1, 2)), (0.1, (5, 0)), (0.5, (-7, 1 << 40)), (0.9371, (1 << 62, -3)), (1.0, (3, 4))):
        x = torch.randn(n, device=cuda).to(dtype)
        u = torch.tensor(numbers(n, st), dtype=torch.int64)
        keep = (u >= round(p * 2 ** 32)) & (p < 1)
        want = torch.where(keep, x.cpu().double() / max(1 - p, 1e-300), 0.0)
        for y in (dr.dropout_forward(x, p, state(cuda, *st)), dr.dropout_backward(x, p, state(cuda, *st))):
            y = y.cpu()
            assert y.dtype == dtype and torch.equal(y != 0, keep & (x.cpu() != 0))
            # the factor is rounded to fp32, the product to fp32 and to the result's type
            step = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
            lim = want.abs() * (step + 2.01 * 2.0 ** -24) + (2.0 ** -25 if dtype == torch.float16 else 0)
            assert bool(((y.double() - want).abs() <= lim).all())


def test_ties_of_the_high_half(cuda):
    """The low half decides where the high one equals the threshold's: thresholds put on, below and
    above the numbers of single elements."""
    n, st = 512, (11, 13)
    x = torch.ones(n, device=cuda)
    u = torch.tensor(numbers(n, st), dtype=torch.int64)
    for e in range(0, n, 41):
        for d in (-1, 0, 1):
            t = int(u[e]) + d
            y = dr.dropout_forward(x, t / 2 ** 32, state(cuda, *st)).cpu()
            assert torch.equal(y != 0, u >= t), (e, d)


def test_rate_and_independence(cuda):
    n, p = 1 << 22, 0.3
    x = torch.ones(n, device=cuda)
    a = dr.dropout_forward(x, p, state(cuda, 1, 0)) != 0
    b = dr.dropout_forward(x, p, state(cuda, 1, 1)) != 0
    c = dr.dropout_forward(x, p, state(cuda, 2, 0)) != 0
    # six standard deviations of a mean of n yes / no answers
    six = 6 * (p * (1 - p) / n) ** 0.5
    for m in (a, b, c):
        assert abs(float(m.double().mean()) - (1 - p)) < six
    for m, o in ((a, b), (a, c), (a[1:], a[:-1]), (a[8:], a[:-8])):
        assert abs(float((m & o).double().mean()) - (1 - p) ** 2) < 6 * 0.5 / n ** 0.5
    assert torch.equal(a, dr.dropout_forward(x, p, state(cuda, 1, 0)) != 0)


@pytest.mark.parametrize("dtype", TYPES)
def test_views_and_special_values(cuda, dtype):
    st = state(cuda, 21, 5)
    base = torch.randn(1 + 37 * 19, device=cuda).to(dtype)
    odd = base[1:].view(37, 19)                      # starts at an odd element
    want = dr.dropout_forward(odd.clone(), 0.4, st)
    assert torch.equal(dr.dropout_forward(odd, 0.4, st), want)
    t = odd.t().contiguous().t()                     # other strides, the same elements
    assert torch.equal(dr.dropout_forward(t, 0.4, st), want)
    bad = odd.clone()
    bad[want == 0] = float("inf")
    bad[0] = torch.where(want[0] == 0, float("nan"), odd[0])
    assert torch.equal(dr.dropout_forward(bad, 0.4, st), want)   # what is dropped is zero, whatever it was
    assert dr.dropout_forward(odd[:0], 0.4, st).shape == (0, 19)
    assert dr.dropout_forward(odd[0, 0], 0.0, st).shape == ()


def test_refusals(cuda):
    x, st = torch.ones(8, device=cuda), state(cuda, 1, 2)
    for call, text in [
            (lambda: dr.dropout_forward(x, -0.1, st), "between 0 and 1"),
            (lambda: dr.dropout_forward(x, float("nan"), st), "between 0 and 1"),
            (lambda: dr.dropout_forward(x.double(), 0.1, st), "dtype"),
            (lambda: dr.dropout_forward(x, 0.1, st.int()), "dtype"),
            (lambda: dr.dropout_forward(x, 0.1, st[:1]), "seed, offset"),
            (lambda: dr.dropout_forward(x, 0.1, st.cpu()), "GPU tensor")]:
        with pytest.raises(RuntimeError, match=text):
            call()


def test_state_follows_torchs_generator_and_graphs(cuda):
    torch.manual_seed(5)
    a, b = dr.dropout_state(cuda), dr.dropout_state(cuda)
    torch.manual_seed(5)
    assert torch.equal(a, dr.dropout_state(cuda)) and not torch.equal(a, b)
    x = torch.ones(5000, device=cuda)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st = dr.dropout_state(cuda)
        y = dr.dropout_forward(x, 0.5, st)
        dx = dr.dropout_backward(x, 0.5, st)
    seen = []
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, dx) and torch.equal(y, dr.dropout_forward(x, 0.5, st))
        seen.append(y.clone())
    for k in range(3):
        assert not torch.equal(seen[k], seen[k + 1])   # every replay draws another state


def test_large_tensor_on_another_stream(cuda):
    """More elements than 2^31 bytes; the last ones against the numbers of their own groups."""
    n = (1 << 31) + 24
    x = torch.ones(n, device=cuda, dtype=torch.bfloat16)
    st = (3, 9)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = dr.dropout_forward(x, 0.5, state(cuda, *st))
    s.synchronize()
    tail = y[-24:].cpu() != 0
    for g in range(3):
        gg = (n - 24) // 8 + g
        hi = philox((gg & M, gg >> 32, st[1], 0), (st[0], 0))
        for e in range(8):
            h = hi[e // 2] >> 16 * (e & 1) & 0xFFFF
            if h != 0x8000:
                assert bool(tail[8 * g + e]) == (h > 0x8000)
