"""Dropout whose mask is a function of (seed, offset, element number) and is never stored
(`monet::dropout`, traced from `monet_amd.functional.dropout`).

The replayed `aten::dropout` (monet/lm_ops/elementary.py:83-94) keeps a byte per element inside an
autograd node, where the solver does not see it, and drops OTHER elements when a schedule runs it
again.  This operator keeps 16 bytes, {seed, offset} in device memory: the backward and every
recomputation of a step ask the generator again and get the same elements.
"""
import torch

from .. import _lib
from .base import OP, implements


def dropout_state(device=None):
    """int64 [2] on the GPU: {seed, offset} drawn from torch's generator of that device (so
    torch.manual_seed decides it, and every replay of a captured graph draws another)."""
    device = torch.device("cuda") if device is None else torch.device(device)
    if device.type != "cuda":
        raise RuntimeError("the state of a dropout lives on the GPU")
    return torch.randint(-2 ** 63, 2 ** 63 - 1, (2,), dtype=torch.int64, device=device)


def _dropout(x, p, state, name):
    code = _lib.dtype_code(x, name)
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise RuntimeError(f"the probability must lie between 0 and 1, got {p}")
    _lib.require_gpu_tensor(state, "state", torch.int64)
    if state.shape != (2,) or not state.is_contiguous():
        raise RuntimeError("state must be two contiguous int64 numbers, {seed, offset}")
    _lib.require_same_device(x, state, "state")
    xc = x if x.is_contiguous() else x.contiguous()
    y = torch.empty_like(xc)
    _lib.call_on(x.device, "mn_dropout", xc.data_ptr(), y.data_ptr(), xc.numel(), p, state.data_ptr(),
                 code)
    return y


def dropout_forward(x, p, state):
    """x / (1 - p) where an element stays, 0 where it is dropped (probability p, in steps of
    2^-32), in a dense tensor of x's shape.  Elements are numbered row by row, whatever x's
    strides are."""
    return _dropout(x, p, state, "input")


def dropout_backward(grad, p, state):
    """The gradient of dropout_forward with the same p and state."""
    return _dropout(grad, p, state, "grad_output")


@implements(['monet::dropout'],
            ['normal', 'multiway', 'newnode', 'multiway_newnode', 'conv_multiway_newnode',
             'conv_normal'])
class CounterDropout(OP):
    backward_storage = None
    params = None   # (p, state); state None: nothing is dropped
    # a forward that finds `params` repeats the step's first forward
    recompute_needs_params = True

    def forward(self, x, p, training=True):
        with torch.no_grad():
            if self.params is None:
                drops = bool(training) and p > 0
                self.params = p, dropout_state(x.device) if drops else None
            p, state = self.params
            return x.clone() if state is None else dropout_forward(x, p, state)

    def backward(self, grad_output, stored, nodel=False):
        assert len(stored) == 0
        with torch.no_grad():
            p, state = self.params
            return grad_output if state is None else dropout_backward(grad_output, p, state)
