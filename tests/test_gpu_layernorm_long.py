"""Layer norm of very long rows: the limits of a launch, and sums of many terms."""
import pytest
import torch

import monet_amd.lm_ops as lm_ops

pytestmark = pytest.mark.gpu
ln = lm_ops.layernorm


def test_parameter_gradients_of_rows_beyond_a_launch(cuda):
    """2^27 + 33 columns: more than 2^32 threads where a workgroup of 1024 takes 32 of them.  Two rows:
    dw = sum g xh and db = sum g are one rounded addition of two products, each within three roundings
    (x - mean, times rstd, times g), and the result's own: 4u of the sum of magnitudes."""
    D, rows = 2 ** 27 + 33, 2
    g = torch.randn(rows, D, device=cuda, dtype=torch.float16)
    x = torch.randn(rows, D, device=cuda, dtype=torch.float16)
    w = torch.ones(D, device=cuda, dtype=torch.float32)
    mean, rstd = torch.tensor([0.25, -0.5], device=cuda), torch.tensor([1.5, 0.75], device=cuda)
    _, dw, db = ln.layer_norm_backward(g, x, mean, rstd, w, w, need_input=False)
    u = 2.0 ** -24
    for lo in range(0, D, 2 ** 25):
        part = slice(lo, min(lo + 2 ** 25, D))
        gp = g[:, part].double()
        xh = (x[:, part].double() - mean.double()[:, None]) * rstd.double()[:, None]
        for got, terms in ((dw, gp * xh), (db, gp)):
            bound = 4 * u * terms.abs().sum(0) + 1e-30
            assert bool(((got[part].double() - terms.sum(0)).abs() <= bound).all()), lo


U = 2.0 ** -24
CHAIN = 2 ** 22      # 4096 terms a thread


def _far(cuda, D):
    """A row far from zero: 1000.1 and 0.05 to either side."""
    x = torch.full((1, D), 1000.1, device=cuda)
    x[:, ::2] += 0.05
    x[:, 1::2] -= 0.05
    return x


def test_mean_of_a_long_row_far_from_zero(cuda):
    """The mean is the exact sum's (64-bit partial sums: 2^-53 a term) rounded once, u |mean|; x - mean
    is exact (both lie in one binade, and multiples of its step), so y is off by that error times rstd,
    by rstd's (division, root, sum with eps, its own rounding, and the squared error of the mean, which
    is 2^-20 of the variance here: 4u + 2^-20) and two roundings more.  (A chain of 4096 fp32 additions of
    1000.1 drifts by up to 2^-25 a term: 0.06, more than the deviation.)"""
    x = _far(cuda, CHAIN)
    y, mean, rstd = ln.layer_norm_forward(x, CHAIN, eps=1e-5)
    wide = x.double()
    mu = wide.mean()
    want_r = 1 / (wide.var(correction=0) + 1e-5).sqrt()
    assert abs(float(mean[0]) - float(mu)) <= 1.01 * U * 1000.1
    var_off = (U * 1000.1) ** 2 * 1.1 / float(wide.var(correction=0))
    assert abs(float(rstd[0]) / float(want_r) - 1) <= 5 * U + var_off
    want = (wide - mu) * want_r
    bound = 1.01 * U * 1000.1 * float(want_r) + (8 * U + var_off) * want.abs()
    assert bool(((y.double() - want).abs() <= bound).all())


def test_sums_of_the_gradient_of_a_long_row(cuda):
    """dx = r (g - s1 - xh s2) from the same mean and rstd.  xh carries 2u; s1 u of itself; s2 3u of the
    mean of |g xh| and u of itself; the three operations 3u of their operands, the factor r u."""
    x = _far(cuda, CHAIN)
    g = torch.full((1, CHAIN), 0.1, device=cuda)
    g[:, ::3] += 0.013
    _, mean, rstd = ln.layer_norm_forward(x, CHAIN, eps=1e-5)
    dx, _, _ = ln.layer_norm_backward(g, x, mean, rstd)
    r, gw = float(rstd[0]), g.double()
    xh = (x.double() - mean.double()) * r
    s1, s2 = float(gw.mean()), float((gw * xh).mean())
    want = r * (gw - s1 - xh * s2)
    s2_off = 4 * U * float((gw * xh).abs().mean()) + U * abs(s2)
    bound = r * (U * abs(s1) + xh.abs() * s2_off + 3 * U * ((gw - s1).abs() + (2 * xh * s2).abs())) \
        + 2 * U * want.abs() + 1e-30
    assert bool(((dx.double() - want).abs() <= 1.01 * bound).all())


def test_parameter_gradients_of_many_long_rows(cuda):
    """65536 rows in 64 slices of 1024: 64-bit sums rounded once, joined by 7 fp32 additions (two slices
    to a thread of 32, five levels), rounded: 8u of the sum of magnitudes, and 2u of xh for dw."""
    rows, D = 1 << 16, 16400
    g = torch.full((rows, D), 0.1, device=cuda)
    x = torch.full((rows, D), 0.7, device=cuda)
    mean, rstd = torch.zeros(rows, device=cuda), torch.ones(rows, device=cuda)
    w = torch.ones(D, device=cuda)
    _, dw, db = ln.layer_norm_backward(g, x, mean, rstd, w, w, need_input=False)
    c, d = float(g[0, 0]), float(x[0, 0])
    assert float((db.double() / (rows * c) - 1).abs().max()) <= 8 * U
    assert float((dw.double() / (rows * c * d) - 1).abs().max()) <= 10 * U
