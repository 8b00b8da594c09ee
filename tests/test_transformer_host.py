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


def _attention(**kw):
    d = _lib.AttentionDesc(B=2, T=300, Hq=4, Hkv=2, D=64, left=10, right=0, sinks=1, scale=0.125)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_attention_refusals():
    f, b, size = lib().mn_attention_fwd, lib().mn_attention_bwd, lib().mn_attention_bwd_ws_bytes

    def fwd(q=P, k=P, v=P, out=P, lse=P, dtype=F32, **kw):
        return f(ctypes.byref(_attention(**kw)), q, k, v, None, out, lse, dtype, None)

    assert f(None, P, P, P, None, P, P, F32, None) == _lib.MN_EINVAL and size(None) == 0
    for bad in (dict(B=-1), dict(T=-1), dict(Hq=0), dict(Hkv=0), dict(D=0), dict(Hq=5), dict(left=-2),
                dict(right=-2), dict(sinks=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                dict(scale=float("inf")), dict(q=None), dict(k=None), dict(v=None), dict(out=None),
                dict(lse=None)):
        assert fwd(**bad) == _lib.MN_EINVAL, bad
    for bad in (dict(D=129), dict(T=1 << 28), dict(B=1 << 28), dict(Hq=1 << 20, Hkv=1 << 20),
                dict(B=1 << 20, T=1 << 20), dict(dtype=5)):
        assert fwd(**bad) == _lib.MN_EUNSUPPORTED, bad
    for empty in (dict(B=0), dict(T=0)):
        assert fwd(**empty) == _lib.MN_OK, empty

    def bwd(hole=None, ws=P, nbytes=None, **kw):
        d = _attention(**kw)
        ptrs = [None if k == hole else P for k in range(10)]
        return b(ctypes.byref(d), *ptrs, F32, ws, size(ctypes.byref(d)) if nbytes is None else nbytes, None)

    for hole in (0, 1, 2, 3, 4, 5, 7, 8, 9):       # 6 is `lengths`, which may be missing
        assert bwd(hole) == _lib.MN_EINVAL, hole
    assert bwd(ws=None) == _lib.MN_EINVAL and bwd(ws=P + 2) == _lib.MN_EINVAL and bwd(nbytes=8) == _lib.MN_EINVAL
    assert bwd(D=129, nbytes=1 << 40) == _lib.MN_EUNSUPPORTED


def test_attention_workspace():
    size = lambda **kw: lib().mn_attention_bwd_ws_bytes(ctypes.byref(_attention(**kw)))
    rows = 4 * 2 * 4          # fp32 per token: batch 2, 4 heads
    assert size() == rows * 300 and size(sinks=0) == rows * 300 and size(left=-1, T=5000) == rows * 5000
    assert size(T=0) == 0 and size(D=129) == 0
    # sinks behind a window: partial results of at most 129 workgroups per sink
    for T, left, sinks in ((1100, 60, 1), (15808, 1024, 4), (1 << 20, 0, 200), (40000, 128, 4000)):
        parts = size(T=T, left=left, sinks=sinks) - rows * T
        key = 2 * 2 * 2 * 64 * 4          # batch, key heads, dk and dv
        kept = sinks if sinks < 128 else (sinks + 127) // 128 * 128
        assert parts % (key * kept) == 0 and 2 <= parts // (key * kept) <= 129, (T, left, sinks)
    assert size(T=2000, left=10, sinks=300) == rows * 2000   # more than an eighth of the keys
    # a batch beyond a launch (2^32 threads, six workgroups to a tile and head) shares one part's
    part = ((1 << 32) - 1) // 256 // 6 // (4 * 3)
    assert size(B=part, sinks=0) == size(B=part + 1, sinks=0) == part * 4 * 300 * 4


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
    with pytest.raises(RuntimeError, match="GPU tensor"):
        lm_ops.attention.window_attention_forward(x[None, None], x[None, None], x[None, None])


def test_registered_in_every_solver_mode():
    for mode in ("normal", "multiway", "newnode", "multiway_newnode", "conv_multiway_newnode",
                 "conv_normal"):
        for name, cls in (("aten::layer_norm", lm_ops.layernorm.InputActLayerNorm),
                          ("monet::dropout", lm_ops.dropout.CounterDropout),
                          ("monet::rotary", lm_ops.rotary.Rotary),
                          ("monet::window_attention", lm_ops.attention.WindowAttention)):
            assert lm_ops.list_ops(mode, name) == [cls]
        # the operator that replays torch's own dropout stays what it was
        assert lm_ops.list_ops(mode, "aten::dropout") == [lm_ops.elementary.Dropout]


# ------------------------------------------------------------------ traced, solved, compiled
def _traced():
    from transformer_net import PATCH, TOKENS, PatchNet
    from monet_amd.graph import Graph
    torch.manual_seed(0)
    return Graph.create(PatchNet(), (TOKENS, PATCH))


def test_a_traced_model_names_the_operators():
    g = _traced()
    ops = [n.op for n in g.nodes if hasattr(n, "op")]
    assert ops.count("monet::rotary") == 4 and ops.count("monet::window_attention") == 2
    assert ops.count("monet::dropout") == 4 and ops.count("aten::layer_norm") == 5
    from transformer_net import TOKENS
    for n in g.nodes:
        if getattr(n, "op", "") == "monet::window_attention":
            assert n.shape == [-1, TOKENS, 4, 12] and n.has_backward
            assert [a.value for a in n.args[3:]] == [None, 13, 2, 1, None]


def test_outside_a_trace_cpu_tensors_are_refused():
    from monet_amd import functional as MF
    x = torch.zeros(1, 2, 2, 8)
    for call in (lambda: MF.dropout(x, 0.5), lambda: MF.window_attention(x, x, x),
                 lambda: MF.rotary(x, torch.zeros(1, 2), (2,))):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    assert MF.dropout(x, 0.5, training=False) is x and MF.dropout(x, 0.0) is x
    with pytest.raises(RuntimeError, match="between 0 and 1"):
        MF.dropout(x, 1.5)


@pytest.mark.parametrize("mode", ["normal", "multiway_newnode", "inplace_conv_multiway_newnode"])
def test_schedules_of_a_traced_model_compile(mode):
    """The solver's plan, generous and tight, compiles; dropouts that run again in the backward are
    marked to find the state of their first run."""
    from monet_amd.schedule import Schedule, _FWD
    from monet_amd.solver import Model
    from monet_amd.solver_info import SolverInfo
    from transformer_net import cheap_dropout_cost
    g = _traced()
    si = SolverInfo(16, "patch", mode)
    si.extract(g, cost_fn=cheap_dropout_cost(si))
    total = sum(n.mem for i, n in si.nodes.items() if i < si.loss) + si.nodes[si.loss].fixed_mem
    again = 0
    for frac in (1.5, 0.55, 0.45):
        sol = Model(si, frac * total / 2 ** 30, time_limit=60, mip_rel_gap=0.1).solve()
        sched = Schedule(g, si)
        sched.init_schedule(sol, si.mode)
        for t, plan in enumerate(sched._plan):
            for ins in plan:
                if ins[0] == _FWD and type(ins[1]).__name__ == "CounterDropout":
                    assert ins[5] == (t > 0)
                    again += t > 0
    assert again > 0
