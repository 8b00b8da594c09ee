"""Dropout at probabilities next to one."""
import pytest
import torch

import monet_amd.lm_ops as lm_ops
from test_gpu_dropout import M, numbers, state

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed, element", [(2677174, 1007), (3076271, 407)])
def test_probabilities_that_round_to_one(cuda, seed, element):
    """round(p 2^32) = 2^32 is above every number: not even the largest, 2^32 - 1, stays.  One step
    below it stays, times 2^32."""
    n = 1024
    u = numbers(n, (seed, 0))
    assert u[element] == M and u.count(M) == 1
    x = torch.ones(n, device=cuda)
    st = state(cuda, seed, 0)
    for p in (1 - 2.0 ** -34, 1 - 2.0 ** -53, 1.0):
        assert not bool(lm_ops.dropout.dropout_forward(x, p, st).any())
    y = lm_ops.dropout.dropout_forward(x, 1 - 2.0 ** -32, st)
    assert float(y[element]) == 2.0 ** 32 and int((y != 0).sum()) == 1
