"""Attention over a sliding window and a few first tokens that stay visible
(`monet::window_attention`, traced from `monet_amd.functional.window_attention`).

Scores are never stored: the forward keeps the logarithm of every row's sum, four bytes a row and
head, next to BatchNorm's statistics in `params`, and the backward computes the probabilities
again from q, k, v, the output and that.  The reference has no counterpart.

Query i of a sequence sees key j if j <= i + right and (j >= i - left or j < sinks), both inside
the sequence's length; -1 means no limit.  right=0 is causal; left=right=w is a band.
"""
import math

import torch

from .. import _lib
from .base import OP, InputStorage, OutputStorage, implements


def _rows(t):
    """`t` with a head's elements next to each other."""
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def _describe(q, k, v, left, right, sinks, scale, lengths):
    """(dtype code, q, k, v, lengths, struct mn_attention)."""
    code = _lib.dtype_code(q, "q")
    for t, name in ((k, "k"), (v, "v")):
        _lib.require_gpu_tensor(t, name, q.dtype)
        _lib.require_same_device(q, t, name)
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise RuntimeError("q must be [batch, tokens, heads, head size], k and v alike [batch, tokens, "
                           f"key heads, head size]; got {list(q.shape)}, {list(k.shape)}, {list(v.shape)}")
    B, T, Hq, D = q.shape
    Hkv = k.shape[2]
    if k.shape[0] != B or k.shape[1] != T or k.shape[3] != D:
        raise RuntimeError(f"q of shape {list(q.shape)} and k of shape {list(k.shape)} differ in batch, tokens "
                           "or head size")
    if Hq == 0 or Hkv == 0 or D == 0 or Hq % Hkv:
        raise RuntimeError(f"{Hq} query heads cannot share {Hkv} key heads of {D} elements evenly")
    left, right, sinks = int(left), int(right), int(sinks)
    if left < -1 or right < -1 or sinks < 0:
        raise RuntimeError("left and right must be -1 (no limit) or a number of tokens, sinks a number of "
                           f"tokens; got {left}, {right}, {sinks}")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 < scale <= 1e30:
        raise RuntimeError(f"the scale must be positive, got {scale}")
    if lengths is not None:
        _lib.require_gpu_tensor(lengths, "lengths", torch.int32)
        _lib.require_same_device(q, lengths, "lengths")
        if lengths.shape != (B,):
            raise RuntimeError(f"lengths must hold one number per sequence, {B}, got {list(lengths.shape)}")
        lengths = lengths.contiguous()
    q, k, v = _rows(q), _rows(k), _rows(v)
    # (numbers beyond the sequence are all the same, and ctypes would keep the low 64 bits of any)
    d = _lib.AttentionDesc(B=B, T=T, Hq=Hq, Hkv=Hkv, D=D, left=min(left, T), right=min(right, T),
                           sinks=min(sinks, T), scale=scale)
    d.q_stride[:] = q.stride()[:3]
    d.k_stride[:] = k.stride()[:3]
    d.v_stride[:] = v.stride()[:3]
    return code, q, k, v, lengths, d


def window_attention_forward(q, k, v, left=-1, right=0, sinks=0, scale=None, lengths=None):
    """(out, lse) for q [batch, tokens, heads, head size], k and v [batch, tokens, key heads, head
    size] (any strides; heads a multiple of key heads; head size up to 128).

    scale    of the scores, 1 / sqrt(head size) unless given
    lengths  int32 [batch] on the GPU: tokens of each padded sequence.  What lies behind them is
             not read, and comes out as zeros (lse -inf).  (A NaN inside a sequence may reach
             every query of it, as in a product of a masked softmax with v.)
    out [batch, tokens, heads, head size] has q's type; lse [batch, heads, tokens] is fp32.
    """
    code, q, k, v, lengths, d = _describe(q, k, v, left, right, sinks, scale, lengths)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(d.B, d.Hq, d.T, dtype=torch.float32, device=q.device)
    _lib.call_on(q.device, "mn_attention_fwd", _lib.byref(d), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                 _lib.ptr(lengths), out.data_ptr(), lse.data_ptr(), code)
    return out, lse


def window_attention_backward(grad, q, k, v, out, lse, left=-1, right=0, sinks=0, scale=None, lengths=None):
    """(dq, dk, dv) from the forward's inputs and results."""
    code, q, k, v, lengths, d = _describe(q, k, v, left, right, sinks, scale, lengths)
    for t, name, shape, dtype in ((grad, "grad_output", q.shape, q.dtype), (out, "out", q.shape, q.dtype),
                                  (lse, "lse", (d.B, d.Hq, d.T), torch.float32)):
        _lib.require_gpu_tensor(t, name, dtype)
        _lib.require_same_device(q, t, name)
        if tuple(t.shape) != tuple(shape):
            raise RuntimeError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    grad, out, lse = grad.contiguous(), out.contiguous(), lse.contiguous()
    dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dk = torch.empty(k.shape, dtype=q.dtype, device=q.device)
    dv = torch.empty(v.shape, dtype=q.dtype, device=q.device)
    nbytes = _lib.load().mn_attention_bwd_ws_bytes(_lib.byref(d))
    ws = torch.empty(max(nbytes, 4), dtype=torch.uint8, device=q.device)
    _lib.call_on(q.device, "mn_attention_bwd", _lib.byref(d), grad.data_ptr(), q.data_ptr(), k.data_ptr(),
                 v.data_ptr(), out.data_ptr(), lse.data_ptr(), _lib.ptr(lengths), dq.data_ptr(), dk.data_ptr(),
                 dv.data_ptr(), code, ws.data_ptr(), nbytes)
    return dq, dk, dv


@implements(['monet::window_attention'],
            ['normal', 'multiway', 'newnode', 'multiway_newnode', 'conv_multiway_newnode',
             'conv_normal'])
class WindowAttention(OP):
    """Backward from the stored q, k, v and output."""
    backward_storage = [InputStorage(0, 1, 2), OutputStorage()]
    params = None   # (lse, lengths, window)

    @staticmethod
    def state_bytes(node):
        B, T, H, _ = node.shape
        return 4 * B * T * H

    def forward(self, q, k, v, lengths, left, right, sinks, scale):
        with torch.no_grad():
            how = dict(left=left, right=right, sinks=sinks, scale=scale)
            out, lse = window_attention_forward(q, k, v, lengths=lengths, **how)
            self.params = lse, lengths, how
            return out

    def backward(self, grad_output, stored, nodel=False):
        with torch.no_grad():
            q, k, v, out = stored
            if not nodel:
                del stored[:]
            lse, lengths, how = self.params
            grads = window_attention_backward(grad_output, q, k, v, out, lse, lengths=lengths, **how)
            # one gradient per tensor argument of the forward
            return grads if lengths is None else grads + (None,)
