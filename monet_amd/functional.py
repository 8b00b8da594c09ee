"""Operators a transformer block calls between its linear layers and that torch has no counterpart
of: dropout whose mask is never stored, rotary positions over several axes, attention with a
sliding window and sinks.  (Layer normalisation is torch's own call, `nn.LayerNorm`; under a
schedule it runs this framework's kernel.)

Called on GPU tensors they run the kernels of `monet_amd.lm_ops` and are differentiable.  While
`Graph.create` traces a model on the CPU they only record a `monet::` node of the right shape,
which a schedule then runs through the operator classes; outside a trace CPU tensors are refused,
as everywhere in this package.
"""
import torch
from torch.autograd.function import once_differentiable

from .lm_ops import attention as _attention
from .lm_ops import dropout as _dropout
from .lm_ops import rotary as _rotary

_library = torch.library.Library("monet", "DEF")
_library.define("dropout(Tensor x, float p, bool training) -> Tensor")
_library.define("rotary(Tensor x, Tensor positions, int[] sections, float base, bool joint, "
                "bool interleaved) -> Tensor")
_library.define("window_attention(Tensor q, Tensor k, Tensor v, Tensor? lengths, int left, int right, "
                "int sinks, float? scale) -> Tensor")
# what a trace needs: the shape, dense as the operators' results are (a copy, since an operator may
# not return its argument)
for _name in ("dropout", "rotary", "window_attention"):
    _library.impl(_name, lambda x, *rest: x.detach().clone(memory_format=torch.contiguous_format),
                  "CompositeExplicitAutograd")


def _recorded(x):
    return torch.jit.is_tracing() and not x.is_cuda


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p):
        ctx.p, ctx.state = p, _dropout.dropout_state(x.device)
        return _dropout.dropout_forward(x, p, ctx.state)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return _dropout.dropout_backward(grad, ctx.p, ctx.state), None


def dropout(x, p=0.5, training=True):
    """As `torch.nn.functional.dropout`, with 16 bytes kept for the backward pass instead of a mask.
    The elements that are dropped follow from torch's generator of x's device."""
    if not 0.0 <= p <= 1.0:
        raise RuntimeError(f"the probability must lie between 0 and 1, got {p}")
    if _recorded(x):
        return torch.ops.monet.dropout(x, float(p), bool(training))
    if not training or p == 0:
        return x
    if not x.is_cuda:
        _dropout.dropout_forward(x, p, None)   # refuses
    return _Dropout.apply(x, float(p))


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, *how):
        ctx.how = how
        ctx.save_for_backward(positions)
        return _rotary.rotary_forward(x, positions, *how)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return (_rotary.rotary_backward(grad, ctx.saved_tensors[0], *ctx.how),) + (None,) * 5


def rotary(x, positions, sections, base=10000.0, joint=False, interleaved=False):
    """`lm_ops.rotary.rotary_forward`, differentiable in x (not in the positions)."""
    sections = [int(s) for s in sections]
    if _recorded(x):
        return torch.ops.monet.rotary(x, positions, sections, float(base), bool(joint), bool(interleaved))
    return _Rotary.apply(x, positions, sections, base, joint, interleaved)


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, *how):
        ctx.how = dict(zip(("left", "right", "sinks", "scale"), how))
        out, lse = _attention.window_attention_forward(q, k, v, lengths=lengths, **ctx.how)
        ctx.save_for_backward(q, k, v, out, lse, lengths)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, v, out, lse, lengths = ctx.saved_tensors
        grads = _attention.window_attention_backward(grad, q, k, v, out, lse, lengths=lengths, **ctx.how)
        return grads + (None,) * 5


def window_attention(q, k, v, left=-1, right=0, sinks=0, scale=None, lengths=None):
    """The output of `lm_ops.attention.window_attention_forward`, differentiable in q, k and v."""
    left, right, sinks = int(left), int(right), int(sinks)
    scale = None if scale is None else float(scale)
    if _recorded(q):
        return torch.ops.monet.window_attention(q, k, v, lengths, left, right, sinks, scale)
    return _WindowAttention.apply(q, k, v, lengths, left, right, sinks, scale)
