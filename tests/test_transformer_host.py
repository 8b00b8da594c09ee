"""Host side of the transformer-block operators that needs no GPU: refusals of the C entry points
(decided before anything is launched), of the operators, sizes of workspaces, the registry."""
import ctypes

import pytest
import torch

import monet_amd.lm_ops as lm_ops
from monet_amd import _lib

F32, BF16, F16 = _lib.F32, _lib.BF16, _lib.F16
P = 64   # stands for a device pointer: these calls are refused, or have nothing to do


def lib():
    return _lib.load()


def test_layer_norm_refusals():
    f = lib().mn_layer_norm_fwd

    def fwd(x=P, y=P, rows=4, D=8, dtype=F32, wdtype=F32):
        return f(x, P, P, y, P, P, rows, D, 1e-5, dtype, wdtype, None)

    assert fwd(rows=-1) == _lib.MN_EINVAL
    assert fwd(D=0) == _lib.MN_EINVAL and fwd(D=-3) == _lib.MN_EINVAL
    assert fwd(x=None) == _lib.MN_EINVAL and fwd(y=None) == _lib.MN_EINVAL
    assert fwd(dtype=3) == _lib.MN_EUNSUPPORTED and fwd(dtype=-1) == _lib.MN_EUNSUPPORTED
    assert fwd(dtype=F32, wdtype=BF16) == _lib.MN_EUNSUPPORTED
    assert fwd(dtype=F16, wdtype=BF16) == _lib.MN_EUNSUPPORTED
    assert fwd(D=1 << 40) == _lib.MN_EUNSUPPORTED and fwd(rows=1 << 41) == _lib.MN_EUNSUPPORTED
    assert fwd(rows=0) == _lib.MN_OK                    # nothing to do
    b = lib().mn_layer_norm_bwd

    def bwd(g=P, x=P, mean=P, rstd=P, dw=P, rows=4, D=8, ws=P, nbytes=None):
        nbytes = lib().mn_layer_norm_ws_bytes(rows, D) if nbytes is None else nbytes
        return b(g, x, mean, rstd, P, P, dw, None, rows, D, F32, F32, ws, nbytes, None)

    for missing in ("g", "x", "mean", "rstd", "ws"):
        assert bwd(**{missing: None}) == _lib.MN_EINVAL, missing
    assert bwd(nbytes=4) == _lib.MN_EINVAL and bwd(ws=P + 2) == _lib.MN_EINVAL
    assert bwd(rows=-1) == _lib.MN_EINVAL and bwd(D=0) == _lib.MN_EINVAL


def test_layer_norm_workspace():
    size = lib().mn_layer_norm_ws_bytes
    assert size(0, 8) == 0 and size(-1, 8) == 0 and size(4, 0) == 0
    for rows in (1, 7, 36064, 1 << 20):
        for D in (1, 31, 512, 2048, 2049, 16385):
            n = size(rows, D)
            assert n % (8 * D) == 0 and 1 <= n // (8 * D) <= 1024, (rows, D)


def test_dropout_refusals():
    f = lib().mn_dropout
    assert f(P, P, -1, 0.5, P, F32, None) == _lib.MN_EINVAL
    for p in (-0.1, 1.1, float("nan"), float("inf")):
        assert f(P, P, 8, p, P, F32, None) == _lib.MN_EINVAL, p
    for hole in range(3):
        a = [P, P, P]
        a[hole] = None
        assert f(a[0], a[1], 8, 0.5, a[2], F32, None) == _lib.MN_EINVAL
    assert f(P, P, 8, 0.5, P, 7, None) == _lib.MN_EUNSUPPORTED
    assert f(None, None, 0, 0.5, None, F32, None) == _lib.MN_OK


def _rotary(**kw):
    d = _lib.RotaryDesc(B=1, T=4, H=2, D=16, axes=2, base=10000.0)
    d.sections[:] = (4, 4, 0)
    d.x_stride[:] = (128, 32, 16)
    d.pos_stride[:] = (4, 0, 1)
    for k, v in kw.items():
        if k == "sections":
            d.sections[:] = v
        else:
            setattr(d, k, v)
    return d


def test_rotary_refusals():
    f = lib().mn_rotary

    def call(x=P, pos=P, y=P, dtype=F32, **kw):
        return f(ctypes.byref(_rotary(**kw)), x, pos, y, 0, dtype, None)

    assert f(None, P, P, P, 0, F32, None) == _lib.MN_EINVAL
    for bad in (dict(B=-1), dict(T=-1), dict(H=-1), dict(D=0), dict(axes=0), dict(axes=4), dict(base=0.0),
                dict(base=float("nan")), dict(sections=(-1, 4, 0)), dict(sections=(5, 4, 0)),
                dict(x=None), dict(pos=None), dict(y=None)):
        assert call(**bad) == _lib.MN_EINVAL, bad
    for bad in (dict(D=400, sections=(100, 100, 0)), dict(H=1 << 20), dict(B=1 << 31), dict(pos_type=3),
                dict(dtype=9)):
        assert call(**bad) == _lib.MN_EUNSUPPORTED, bad
    for empty in (dict(B=0), dict(T=0), dict(H=0)):
        assert call(**empty) == _lib.MN_OK, empty


def test_operators_refuse_cpu_tensors():
    x = torch.zeros(2, 4)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        lm_ops.layernorm.layer_norm_forward(x, (4,))
    with pytest.raises(RuntimeError, match="GPU tensor"):
        lm_ops.layernorm.layer_norm_backward(x, x, x[:, 0], x[:, 0])
    with pytest.raises(RuntimeError, match="GPU tensor"):
        lm_ops.dropout.dropout_forward(x, 0.5, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="lives on the GPU"):
        lm_ops.dropout.dropout_state("cpu")
    with pytest.raises(RuntimeError, match="GPU tensor"):
        lm_ops.rotary.rotary_forward(x[None, None], torch.zeros(1, 2), (2,))


def test_registered_in_every_solver_mode():
    for mode in ("normal", "multiway", "newnode", "multiway_newnode", "conv_multiway_newnode",
                 "conv_normal"):
        for name, cls in (("aten::layer_norm", lm_ops.layernorm.InputActLayerNorm),
                          ("monet::dropout", lm_ops.dropout.CounterDropout),
                          ("monet::rotary", lm_ops.rotary.Rotary)):
            assert lm_ops.list_ops(mode, name) == [cls]
        # the operator that replays torch's own dropout stays what it was
        assert lm_ops.list_ops(mode, "aten::dropout") == [lm_ops.elementary.Dropout]
