"""Layer normalisation over the last dimensions (`aten::layer_norm`).

The reference has no such operator; it follows the contract of its operator classes
(monet/lm_ops/base.py:2-53).  The forward records mean and reciprocal standard deviation, eight
bytes a row, next to BatchNorm's statistics in `params`; the backward needs the stored input.
fp32, bf16 or fp16; weight and bias have the input's type or fp32.
"""
import math

import torch

from .. import _lib
from .base import OP, InputStorage, implements


def _parameter(t, name, shape, x):
    if t is None:
        return None
    if t.device != x.device:
        _lib.require_gpu_tensor(t, name)
        _lib.require_same_device(x, t, name)
    if t.shape != shape:
        raise RuntimeError(f"{name} must have the normalized shape {list(shape)}, got {list(t.shape)}")
    if t.dtype != x.dtype and t.dtype != torch.float32:
        raise RuntimeError(f"{name} must have dtype {x.dtype} or torch.float32, got {t.dtype}")
    return t if t.is_contiguous() else t.contiguous()


def _weight_type(weight, bias, x):
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError(f"weight and bias differ in dtype: {weight.dtype} and {bias.dtype}")
    t = weight if weight is not None else bias
    return x.dtype if t is None else t.dtype


def layer_norm_forward(x, normalized_shape, weight=None, bias=None, eps=1e-5):
    """(y, mean, rstd): `x` normalised over its last len(normalized_shape) dimensions; the fp32
    statistics have the shape of the dimensions before them."""
    code = _lib.dtype_code(x, "input")
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    k = len(shape)
    if k == 0 or x.dim() < k or x.shape[x.dim() - k:] != shape:
        raise RuntimeError(f"an input of shape {list(x.shape)} does not end in the normalized shape "
                           f"{list(shape)}")
    w, b = _parameter(weight, "weight", shape, x), _parameter(bias, "bias", shape, x)
    wcode = _lib.DTYPE_CODES[_weight_type(w, b, x)]
    xc = x if x.is_contiguous() else x.contiguous()
    D = math.prod(shape)
    lead = x.shape[:x.dim() - k]
    rows = math.prod(lead)
    y = torch.empty_like(xc)
    mean = x.new_empty(lead, dtype=torch.float32)
    rstd = x.new_empty(lead, dtype=torch.float32)
    _lib.call_on(x.device, "mn_layer_norm_fwd", xc.data_ptr(), _lib.ptr(w), _lib.ptr(b), y.data_ptr(),
                 mean.data_ptr(), rstd.data_ptr(), rows, D, float(eps), code, wcode)
    return y, mean, rstd


def layer_norm_backward(grad, x, mean, rstd, weight=None, bias=None, need_input=True):
    """(dx, dw, db) from the forward's input and statistics; dw / db are None without a weight /
    bias, dx without `need_input`.  `bias` only says whether its gradient is wanted, and in which
    type."""
    code = _lib.dtype_code(x, "stored input")
    _lib.require_gpu_tensor(grad, "grad_output", x.dtype)
    if grad.shape != x.shape:
        raise RuntimeError("grad_output and the stored input differ in shape")
    lead = x.shape[:mean.dim()]
    shape = tuple(x.shape[mean.dim():])
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        _lib.require_gpu_tensor(t, name, torch.float32)
        _lib.require_same_device(x, t, name)
        if t.shape != lead or not shape:
            raise RuntimeError(f"{name} of shape {list(t.shape)} does not belong to an input of shape "
                               f"{list(x.shape)}")
    _lib.require_same_device(x, grad, "grad_output")
    w, b = _parameter(weight, "weight", shape, x), _parameter(bias, "bias", shape, x)
    wtype = _weight_type(w, b, x)
    xc = x if x.is_contiguous() else x.contiguous()
    g = grad if grad.is_contiguous() else grad.contiguous()
    mean = mean if mean.is_contiguous() else mean.contiguous()
    rstd = rstd if rstd.is_contiguous() else rstd.contiguous()
    D = math.prod(shape)
    rows = mean.numel()
    dx = torch.empty_like(xc) if need_input else None
    dw = None if w is None else torch.empty(shape, dtype=wtype, device=x.device)
    db = None if b is None else torch.empty(shape, dtype=wtype, device=x.device)
    ws, nbytes = None, 0
    if dw is not None or db is not None:
        nbytes = _lib.load().mn_layer_norm_ws_bytes(rows, D)
        ws = torch.empty(max(nbytes, 4), dtype=torch.uint8, device=x.device)
    _lib.call_on(x.device, "mn_layer_norm_bwd", g.data_ptr(), xc.data_ptr(), mean.data_ptr(),
                 rstd.data_ptr(), _lib.ptr(w), _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db), rows, D, code,
                 _lib.DTYPE_CODES[wtype], _lib.ptr(ws), nbytes)
    return dx, dw, db


@implements(['aten::layer_norm'],
            ['normal', 'multiway', 'newnode', 'multiway_newnode', 'conv_multiway_newnode',
             'conv_normal'])
class InputActLayerNorm(OP):
    """Backward from the stored input; weight and bias are parameters, alive all the time."""
    backward_storage = InputStorage(0)
    params = None   # (mean, rstd, weight, bias, does the input need a gradient)

    @staticmethod
    def state_bytes(node):
        normalized_shape = node.args[1].value
        return 8 * math.prod(node.shape[:len(node.shape) - len(normalized_shape)])

    def forward(self, input_, normalized_shape, weight=None, bias=None, eps=1e-5, *rest):
        with torch.no_grad():
            y, mean, rstd = layer_norm_forward(input_, normalized_shape, weight, bias, eps)
            self.params = mean, rstd, weight, bias, input_.requires_grad
            return y

    def backward(self, grad_output, stored, nodel=False):
        with torch.no_grad():
            input_ = stored[0]
            if not nodel:
                del stored[0]
            mean, rstd, weight, bias, need_input = self.params
            dx, dw, db = layer_norm_backward(grad_output, input_, mean, rstd, weight, bias, need_input)
            # one gradient per tensor argument of the forward
            return (dx,) + ((dw,) if weight is not None else ()) + ((db,) if bias is not None else ())
