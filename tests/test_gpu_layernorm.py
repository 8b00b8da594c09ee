"""Layer normalisation against the formula in 64 bits: row lengths on both sides of every kernel's
limits, the element and weight types, rows that start at odd addresses, gradients."""
import pytest
import torch

import monet_amd.lm_ops as lm_ops
from monet_amd import _lib

pytestmark = pytest.mark.gpu
ln = lm_ops.layernorm
U = 2.0 ** -24
STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}   # half a denormal step


def _data(cuda, rows, D, dtype, wtype, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    x = (torch.randn(rows, D, device=cuda, generator=g) *
         (0.3 + torch.rand(rows, 1, device=cuda, generator=g)) +
         2.0 * torch.randn(rows, 1, device=cuda, generator=g)).to(dtype)
    w = (1 + 0.3 * torch.randn(D, device=cuda, generator=g)).to(wtype)
    b = (0.2 * torch.randn(D, device=cuda, generator=g)).to(wtype)
    gr = torch.randn(rows, D, device=cuda, generator=g).to(dtype)
    return x, w, b, gr


def _exact(x, w, b, gr, eps):
    x, gr = x.double(), gr.double()
    D = x.shape[-1]
    w = torch.ones(D, device=x.device, dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(D, device=x.device, dtype=torch.float64) if b is None else b.double()
    mu = x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - mu) * r
    gw = gr * w
    dx = r * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
    return dict(y=xh * w + b, mean=mu[:, 0], rstd=r[:, 0], dx=dx, dw=(gr * xh).sum(0), db=gr.sum(0), xh=xh,
                w=w, b=b, gw=gw)


def _check(got, want, bound, dtype, what):
    """|got - want| <= half a step of the result's type, and `bound` for the fp32 arithmetic."""
    err = (got.double() - want).abs()
    lim = want.abs() * STEP[dtype] + bound * (1 + STEP[dtype]) + TINY[dtype]
    assert bool((err <= lim).all()), (what, float((err / lim).max()))


def _check_all(x, w, b, gr, eps, out, grads):
    """Bounds on the fp32 arithmetic.  A sum of D values is made of chains of at most 32 additions
    in a lane, 6 across a wave and 16 across waves (54, with the product and the factor 1/D 56
    roundings), so it is off by 56 u times the sum of magnitudes.  With M = max|x| of a row,
    A = M r, N = max|xh|:  mean: 56 u M;  xh = (x - mu) r: 56 u A from the mean, 56/2 + 60 A u... of
    itself from the variance (whose own error is 56 u, and twice the mean's relative to the
    deviation, second order), 3 u for its own roundings: together at most u (60 A + 34 N) =: e.
    dx = r (gw - s1 - xh s2) with G = max|gw|: s1 off by 58 u G, s2 by 58 u G N + G e, xh by e
    (|s2| <= G N), r by 34 u, four roundings of values up to G (2 + N^2):
    r G (58 u + 58 u N^2 + 2 N e + 38 u (2 + N^2)).  dw, db: `rows` more additions at most."""
    y, mean, rstd = out
    dx, dw, db = grads
    rows, D = x.shape
    e = _exact(x, w, b, gr, eps)
    M = x.double().abs().amax(1, keepdim=True)
    r = e["rstd"][:, None]
    N = e["xh"].abs().amax(1, keepdim=True)
    exh = U * (60 * M * r + 34 * N)
    _check(mean, e["mean"], 56 * U * M[:, 0], torch.float32, "mean")
    _check(rstd, e["rstd"], (U * 34 + 56 * 56 * U * U * (M * r)[:, 0] ** 2) * e["rstd"], torch.float32, "rstd")
    _check(y, e["y"], exh * e["w"].abs() + 3 * U * (e["b"].abs() + (e["xh"] * e["w"]).abs()), x.dtype, "y")
    G = e["gw"].abs().amax(1, keepdim=True)
    bdx = r * G * (58 * U + 58 * U * N ** 2 + 2 * N * exh + 38 * U * (2 + N ** 2))
    if dx is not None:
        _check(dx, e["dx"], bdx, x.dtype, "dx")
    depth = rows + 40
    ga = gr.double().abs()
    if dw is not None:
        _check(dw, e["dw"], (depth * U * (ga * e["xh"].abs()) + ga * exh).sum(0), w.dtype, "dw")
    if db is not None:
        _check(db, e["db"], (depth * U * ga).sum(0), (w if w is not None else x).dtype, "db")


# below, at and above what a group of 8, 16, 32, 64 lanes, a wave's registers and a workgroup hold
DIMS = [1, 2, 7, 31, 32, 33, 64, 65, 127, 129, 256, 257, 384, 512, 513, 1023, 1024, 1025, 2047, 2048, 2049,
        4096, 4097, 8191, 8193, 16384, 16385, 20001]


@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("dtype,wtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                         (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                         (torch.float16, torch.float32)])
def test_against_the_formula(cuda, D, dtype, wtype):
    for rows in (1, 5, 67):
        x, w, b, gr = _data(cuda, rows, D, dtype, wtype, seed=D + rows)
        out = ln.layer_norm_forward(x, (D,), w, b, 1e-5)
        assert out[0].dtype == dtype and out[1].dtype == out[2].dtype == torch.float32
        grads = ln.layer_norm_backward(gr, x, out[1], out[2], w, b)
        assert grads[0].dtype == dtype and grads[1].dtype == grads[2].dtype == wtype
        _check_all(x, w, b, gr, 1e-5, out, grads)


@pytest.mark.parametrize("rows,D", [(5000, 96), (2300, 700), (20000, 24), (1500, 3000)])
def test_many_rows(cuda, rows, D):
    """More rows than workgroups: partial sums of the parameters' gradients are joined."""
    for dtype, wtype in ((torch.float32, torch.float32), (torch.bfloat16, torch.float32)):
        x, w, b, gr = _data(cuda, rows, D, dtype, wtype)
        out = ln.layer_norm_forward(x, D, w, b)
        grads = ln.layer_norm_backward(gr, x, out[1], out[2], w, b)
        _check_all(x, w, b, gr, 1e-5, out, grads)
        again = ln.layer_norm_backward(gr, x, out[1], out[2], w, b)
        for p, q in zip(grads, again):
            assert torch.equal(p, q)     # fixed order of the sums


def test_against_differences(cuda):
    """The gradient against central differences of the operator's own forward, in fp32: step h,
    truncation h^2 f''' / 6 and rounding 2^-23 |f| / h, both below 1e-3 of the loss's scale here."""
    x, w, b, gr = _data(cuda, 6, 20, torch.float32, torch.float32)
    _, mean, rstd = ln.layer_norm_forward(x, 20, w, b)
    dx, dw, db = ln.layer_norm_backward(gr, x, mean, rstd, w, b)
    h = 2.0 ** -7

    def loss(x, w, b):
        return float((ln.layer_norm_forward(x, 20, w, b)[0].double() * gr.double()).sum())

    scale = float(gr.double().abs().sum())
    for t, d, args in ((x, dx, 0), (w, dw, 1), (b, db, 2)):
        for i in range(0, t.numel(), 7):
            step = torch.zeros_like(t)
            step.view(-1)[i] = h
            lo, hi = [x, w, b], [x, w, b]
            lo[args], hi[args] = t - step, t + step
            num = (loss(*hi) - loss(*lo)) / (2 * h)
            assert abs(num - float(d.reshape(-1)[i])) < 1e-3 * scale, (args, i)


def test_without_parameters_and_more_dimensions(cuda):
    x = torch.randn(3, 4, 5, 6, device=cuda)
    gr = torch.randn_like(x)
    w = torch.randn(5, 6, device=cuda)
    flat = lambda t: t.reshape(12, 30)
    for ww, bb in ((None, None), (w, None), (None, w)):
        y, mean, rstd = ln.layer_norm_forward(x, (5, 6), ww, bb)
        assert y.shape == x.shape and mean.shape == rstd.shape == (3, 4)
        dx, dw, db = ln.layer_norm_backward(gr, x, mean, rstd, ww, bb)
        assert (dw is None) == (ww is None) and (db is None) == (bb is None)
        fw = None if ww is None else ww.reshape(-1)
        fb = None if bb is None else bb.reshape(-1)
        _check_all(flat(x), fw, fb, flat(gr), 1e-5, (flat(y), mean.reshape(-1), rstd.reshape(-1)),
                   (flat(dx), None if dw is None else dw.reshape(-1), None if db is None else db.reshape(-1)))
    assert ln.layer_norm_backward(gr, x, mean, rstd, w, None, need_input=False)[0] is None


def test_empty_and_odd_views(cuda):
    w = torch.ones(8, device=cuda)
    y, mean, rstd = ln.layer_norm_forward(torch.empty(0, 8, device=cuda), 8, w, w)
    assert y.shape == (0, 8) and mean.shape == (0,)
    dx, dw, db = ln.layer_norm_backward(y, y, mean, rstd, w, w)
    assert dx.shape == (0, 8) and not bool(dw.any()) and not bool(db.any())
    for dtype in (torch.float32, torch.bfloat16):
        base = torch.randn(1 + 9 * 33, device=cuda).to(dtype)
        x = base[1:].view(9, 33)                      # rows of odd length from an odd element on
        gr = torch.randn(33, 9, device=cuda).to(dtype).t()   # a transposed gradient
        wt = torch.randn(66, device=cuda)[::2]
        out = ln.layer_norm_forward(x, 33, wt, wt)
        _check_all(x, wt, wt, gr, 1e-5, out, ln.layer_norm_backward(gr, x, out[1], out[2], wt, wt))


def test_special_values(cuda):
    x, w, b, gr = _data(cuda, 6, 40, torch.float32, torch.float32)
    clean = ln.layer_norm_forward(x, 40, w, b)[0]
    x2 = x.clone()
    x2[1, 3], x2[4, 0] = float("nan"), float("inf")
    y = ln.layer_norm_forward(x2, 40, w, b)[0]
    for row in (0, 2, 3, 5):
        assert torch.equal(y[row], clean[row])        # a row's NaN stays in its row
    assert bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[4]).any())
    same = torch.full((3, 40), 7.25, device=cuda)     # no deviation at all: xh = 0
    y, mean, rstd = ln.layer_norm_forward(same, 40, w, b)
    assert torch.equal(y, b.expand(3, 40)) and torch.equal(mean, same[:, 0])
    far = torch.full((1, 512), 1e4, device=cuda)      # far off zero: the variance is taken around the mean
    far[0, ::2] += 1.0
    mean, rstd = ln.layer_norm_forward(far, 512)[1:]
    assert abs(float(rstd) - 1 / (0.25 + 1e-5) ** 0.5) < 1e-3


def test_refusals(cuda):
    x = torch.randn(4, 8, device=cuda)
    w = torch.ones(8, device=cuda)
    cases = [
        (lambda: ln.layer_norm_forward(x, (4,)), "normalized shape"),
        (lambda: ln.layer_norm_forward(x, ()), "normalized shape"),
        (lambda: ln.layer_norm_forward(x, (2, 4, 8)), "normalized shape"),
        (lambda: ln.layer_norm_forward(x, 8, torch.ones(7, device=cuda)), "weight"),
        (lambda: ln.layer_norm_forward(x, 8, w.half()), "dtype"),
        (lambda: ln.layer_norm_forward(x.half(), 8, w, w.half()), "differ in dtype"),
        (lambda: ln.layer_norm_forward(x.double(), 8), "dtype"),
        (lambda: ln.layer_norm_forward(x, 8, w.cpu()), "GPU tensor"),
        (lambda: ln.layer_norm_backward(x[:2], x, x[:, 0], x[:, 0]), "shape"),
        (lambda: ln.layer_norm_backward(x.half(), x, x[:, 0], x[:, 0]), "dtype"),
        (lambda: ln.layer_norm_backward(x, x, x[:3, 0], x[:, 0]), "does not belong"),
        (lambda: ln.layer_norm_backward(x, x, x, x), "does not belong"),
    ]
    for call, text in cases:
        with pytest.raises(RuntimeError, match=text):
            call()


def test_streams_and_graphs(cuda):
    x, w, b, gr = _data(cuda, 300, 200, torch.bfloat16, torch.float32)
    want = ln.layer_norm_forward(x, 200, w, b)
    gwant = ln.layer_norm_backward(gr, x, want[1], want[2], w, b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ln.layer_norm_forward(x, 200, w, b)
        ggot = ln.layer_norm_backward(gr, x, got[1], got[2], w, b)
    torch.cuda.current_stream().wait_stream(s)
    for p, q in zip(want + gwant, got + ggot):
        assert torch.equal(p, q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ln.layer_norm_forward(x, 200, w, b)
        grads = ln.layer_norm_backward(gr, x, out[1], out[2], w, b)
    for seed in (1, 2, 3):
        x2, _, _, g2 = _data(cuda, 300, 200, torch.bfloat16, torch.float32, seed)
        x.copy_(x2)
        gr.copy_(g2)
        graph.replay()
        torch.cuda.synchronize()
        e = ln.layer_norm_forward(x, 200, w, b)
        for p, q in zip(out + grads, e + ln.layer_norm_backward(gr, x, e[1], e[2], w, b)):
            assert torch.equal(p, q)


@pytest.mark.parametrize("D", [24, 700, 3000, 20001])
def test_in_place_through_the_c_entry(cuda, D):
    """y may take x's place, dx the gradient's."""
    x, w, b, gr = _data(cuda, 70, D, torch.bfloat16, torch.float32)
    y, mean, rstd = ln.layer_norm_forward(x, D, w, b)
    want = ln.layer_norm_backward(gr, x, mean, rstd, w, b)
    xi, gi = x.clone(), gr.clone()
    dw, db = torch.empty_like(w), torch.empty_like(b)
    nbytes = _lib.load().mn_layer_norm_ws_bytes(70, D)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=cuda)
    s = _lib.stream_ptr(cuda)
    _lib.call("mn_layer_norm_bwd", gi.data_ptr(), x.data_ptr(), mean.data_ptr(), rstd.data_ptr(), w.data_ptr(),
              gi.data_ptr(), dw.data_ptr(), db.data_ptr(), 70, D, _lib.BF16, _lib.F32, ws.data_ptr(), nbytes, s)
    for p, q in zip(want, (gi, dw, db)):
        assert torch.equal(p, q)
    _lib.call("mn_layer_norm_fwd", xi.data_ptr(), w.data_ptr(), b.data_ptr(), xi.data_ptr(), None, None, 70, D,
              1e-5, _lib.BF16, _lib.F32, s)
    assert torch.equal(xi, y)
