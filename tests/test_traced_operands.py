"""What an operator of a traced model may read besides activations: parameters and buffers as they
are.  Values computed from them inside forward() are refused when the model is traced; a schedule
would otherwise hand the operator the parameter in their place.  No GPU."""
import pytest
import torch
import torch.nn as nn

from monet_amd import functional as MF
from monet_amd.graph import Graph

T, D = 8, 8


class Net(nn.Module):
    def __init__(self, f):
        super().__init__()
        self.f = f
        self.register_buffer("positions", torch.stack([torch.arange(T), torch.arange(T)]))
        self.register_buffer("scale", torch.tensor(3.0))
        self.lin = nn.Linear(D, D)
        self.square = nn.Parameter(torch.randn(D, D))
        self.register_buffer("passing", torch.arange(T)[None], persistent=False)
        self.attribute = torch.arange(T)[None]

    def forward(self, x):
        return self.f(self, x)

    def heads(self, x):
        return self.lin(x).view(-1, T, 1, D)


def trace(f, shape=(T, D)):
    return Graph.create(Net(f), shape)


def graph_ops(g):
    return [n.op for n in g.nodes if hasattr(n, "op")]


@pytest.mark.parametrize("name, f", [
    ("neg", lambda s, x: MF.rotary(s.heads(x), -s.positions, (2, 2))),
    ("slice", lambda s, x: MF.rotary(s.heads(x), s.positions[:, :T], (2, 2))),
    ("float", lambda s, x: MF.rotary(s.heads(x), s.positions.float(), (2, 2))),
    ("stack", lambda s, x: MF.rotary(s.heads(x), torch.stack([s.positions[0], s.positions[1]]), (2, 2))),
    ("scale", lambda s, x: s.lin(x) * (-s.scale)),
    ("linear of a transposed weight", lambda s, x: nn.functional.linear(x, s.square.t(), s.lin.bias)),
    ("linear of exp", lambda s, x: nn.functional.linear(x, s.square.exp(), s.lin.bias)),
    ("product with a transposed weight", lambda s, x: s.lin(x) * s.square.t()),
    ("cat", lambda s, x: torch.cat([s.lin(x), s.lin(x) + (-s.scale)], 1)),
])
def test_functions_of_parameters_are_refused(name, f):
    with pytest.raises(ValueError, match="parameters and buffers"):
        trace(f)


def test_parameters_as_they_are():
    """What stays: parameters and buffers themselves, numbers, and the transposed weight of addmm."""
    g = trace(lambda s, x: MF.rotary(s.heads(x), s.positions, (2, 2)))
    assert graph_ops(g)[-1] == "monet::rotary"
    assert graph_ops(trace(lambda s, x: s.lin(x) * s.scale)) == ["aten::linear", "aten::mul"]
    assert graph_ops(trace(lambda s, x: s.lin(x) * 2)) == ["aten::linear", "aten::mul"]
    g = trace(lambda s, x: torch.addmm(s.lin.bias, x, s.square.t()), (D,))
    add = g.nodes[-1]
    assert add.op == "aten::addmm" and list(g.nodes[add.args[2].index].shape) == [D, D]
    assert not hasattr(g.nodes[add.args[2].index], "op") and add.args[2].requires_grad


@pytest.mark.parametrize("name, f", [
    ("parameter", lambda s, x: torch.addmm(s.lin.bias, x, s.square)),
    ("activation", lambda s, x: torch.addmm(s.scale, x, s.lin(x).t())),
])
def test_addmm_of_another_operand_is_refused(name, f):
    """Its operator multiplies with the transposed of the parameter it is given."""
    with pytest.raises(ValueError, match="transposed"):
        trace(f, (D,))


@pytest.mark.parametrize("name, f", [
    ("arange", lambda s, x: MF.rotary(s.heads(x), torch.arange(T)[None], (4,))),
    ("lengths", lambda s, x: MF.window_attention(s.heads(x), s.heads(x), s.heads(x),
                                                 lengths=torch.full((23,), T, dtype=torch.int32))),
    ("factors", lambda s, x: s.lin(x) * torch.arange(float(D))),
    ("buffer that is not persistent", lambda s, x: MF.rotary(s.heads(x), s.passing, (4,))),
    ("attribute", lambda s, x: MF.rotary(s.heads(x), s.attribute, (4,))),
])
def test_tensors_outside_the_state_dict_are_refused(name, f):
    """The trace runs on the CPU: they would be constants there."""
    with pytest.raises(ValueError, match="persistent"):
        trace(f)


@pytest.mark.parametrize("name, f", [
    ("positions", lambda s, x: MF.rotary(s.heads(x), x.permute(2, 0, 1), (1,) * 3)),
    ("lengths", lambda s, x: MF.window_attention(s.heads(x), s.heads(x), s.heads(x), lengths=s.lin(x))),
])
def test_computed_positions_and_lengths_are_refused(name, f):
    """Neither has a gradient to pass on, which the backward of what computed it would wait for."""
    with pytest.raises(ValueError, match="no gradient"):
        trace(f)


def test_traced_outputs_are_dense():
    """As those of the operators: a view of one is traced where it would run."""
    def turned(s, x):
        y = s.lin(x).view(-1, 2, T, D // 2).transpose(1, 2)        # [batch, tokens, heads, head size]
        return y

    for f in (lambda s, x: MF.window_attention(turned(s, x), turned(s, x), turned(s, x)),
              lambda s, x: MF.rotary(turned(s, x), s.positions, (1, 1)),
              lambda s, x: MF.dropout(turned(s, x), 0.5, True)):
        g = trace(lambda s, x: f(s, x).view(-1, T, D))
        assert graph_ops(g)[-1] == "aten::view" and g.nodes[-1].shape == [-1, T, D]


@pytest.mark.parametrize("p", [-0.5, 1.5, float("nan")])
def test_traced_dropout_refuses_what_an_eager_one_refuses(p):
    with pytest.raises(RuntimeError, match="between 0 and 1"):
        trace(lambda s, x: MF.dropout(s.lin(x), p, True))
