"""linear_cross_entropy where something stands that has no part in the result: the columns of a tile behind the last
row, rows that are not scored, masked tokens."""

import math

import pytest
import torch

import prlstm_amd
import test_gpu_cross_entropy as xent
from test_gpu_cross_entropy import TYPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [5, 40, 130, 300, 515])
@pytest.mark.parametrize("forced", [89.0, 100.0, 3000.0])
def test_a_token_that_the_bias_forces(dev, dtype, n, forced):
    """A bias whose exponential is infinite: the rows' largest logit takes it back, and a tile's columns behind the last
    row, whose logits it is alone, add nothing."""
    x, w, t, b, dloss = xent.inputs(dev, dtype, n, 700, 40, bias=True, pad=True)
    b[77] = forced
    b[300] = -math.inf
    t[t == 300] = 77
    xent.check(x, w, t, b, dloss)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [5, 300])
def test_an_infinite_bias_where_nothing_is_scored(dev, dtype, n):
    x, w, t, b, dloss = xent.inputs(dev, dtype, n, 700, 40, bias=True)
    b[77] = math.inf
    t[:] = -1
    leaves = [s.detach().requires_grad_(True) for s in (x, w, b)]
    loss = prlstm_amd.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
    assert not bool(loss.any())
    for g in torch.autograd.grad(loss, leaves, dloss):
        assert not bool(g.any())
