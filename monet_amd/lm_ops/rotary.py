"""Rotary positions over one to three axes - row and column of an image's patches, frame of a
video (`monet::rotary`, traced from `monet_amd.functional.rotary`).

Turning is linear in x and keeps its length, so the backward stores nothing of x: it turns the
gradient back.  The reference has no counterpart.
"""
import torch

from .. import _lib
from .base import OP, implements

_POS_TYPES = {torch.int64: 0, torch.int32: 1, torch.float32: 2}


def _rotary(x, positions, sections, base, joint, interleaved, inverse, name):
    code = _lib.dtype_code(x, name)
    if x.dim() != 4:
        raise RuntimeError(f"{name} must be [batch, tokens, heads, head size], got {list(x.shape)}")
    B, T, H, D = x.shape
    sections = [int(s) for s in sections]
    axes = len(sections)
    if not 1 <= axes <= 3 or min(sections) < 0 or 2 * sum(sections) > D or D == 0:
        raise RuntimeError(f"one to three sections that turn at most the head's {D} elements in pairs "
                           f"are needed, got {sections}")
    if not base > 0:
        raise RuntimeError(f"base must be positive, got {base}")
    _lib.require_gpu_tensor(positions, "positions")
    if positions.dtype not in _POS_TYPES:
        raise RuntimeError(f"positions must be int64, int32 or float32, got {positions.dtype}")
    if tuple(positions.shape) not in ((axes, T), (axes, B, T)):
        raise RuntimeError(f"positions must be [{axes}, {T}] or [{axes}, {B}, {T}], got "
                           f"{list(positions.shape)}")
    _lib.require_same_device(x, positions, "positions")
    if x.stride(3) != 1 and D > 1:
        x = x.contiguous()
    ps = positions.stride()
    d = _lib.RotaryDesc(B=B, T=T, H=H, D=D, axes=axes, joint=bool(joint), interleaved=bool(interleaved),
                        pos_type=_POS_TYPES[positions.dtype], base=float(base))
    d.sections[:axes] = sections
    d.x_stride[:] = x.stride()[:3]
    d.pos_stride[:] = (ps[0], 0, ps[1]) if len(ps) == 2 else ps
    y = torch.empty(B, T, H, D, dtype=x.dtype, device=x.device)
    _lib.call_on(x.device, "mn_rotary", _lib.byref(d), x.data_ptr(), positions.data_ptr(), y.data_ptr(),
                 int(inverse), code)
    return y


def rotary_forward(x, positions, sections, base=10000.0, joint=False, interleaved=False):
    """`x` [batch, tokens, heads, head size] with its pairs turned, in a dense tensor.

    positions  [axes, tokens] or [axes, batch, tokens], whole or fp32 numbers
    sections   pairs turned by each axis, 2 * sum(sections) <= head size; the rest is copied
    joint      False: the frequencies of every axis run from 1 down to 1 / base;
               True: one run over all pairs, axis after axis
    interleaved  pairs are neighbours (2k, 2k + 1) instead of (k, k + sum(sections))
    """
    return _rotary(x, positions, sections, base, joint, interleaved, False, "input")


def rotary_backward(grad, positions, sections, base=10000.0, joint=False, interleaved=False):
    """The gradient of rotary_forward: `grad` turned back."""
    return _rotary(grad, positions, sections, base, joint, interleaved, True, "grad_output")


@implements(['monet::rotary'],
            ['normal', 'multiway', 'newnode', 'multiway_newnode', 'conv_multiway_newnode',
             'conv_normal'])
class Rotary(OP):
    backward_storage = None
    params = None   # (positions, sections, base, joint, interleaved); positions never get a gradient

    def forward(self, x, positions, sections, base, joint, interleaved):
        with torch.no_grad():
            self.params = positions, sections, base, joint, interleaved
            return rotary_forward(x, *self.params)

    def backward(self, grad_output, stored, nodel=False):
        assert len(stored) == 0
        with torch.no_grad():
            return rotary_backward(grad_output, *self.params), None
