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
