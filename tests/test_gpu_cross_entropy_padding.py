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


def _grads(x, w, t, b, dloss):
    leaves = [s.detach().requires_grad_(True) for s in (x, w, b)]
    loss = prlstm_amd.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
    return loss.detach(), torch.autograd.grad(loss, leaves, dloss)


def _within(got, x, w, t, b, dloss):
    """The gradients, against the 64-bit ones of operands whose other rows are ordinary."""
    _, dl, parts, size = xent.reference(x, w, t, b, dloss)
    shift = (x.shape[1] + 4) * xent.U * size
    slack, bound_x, bound_w = xent.bounds(x, w, t, dl, parts, shift, dloss)
    xent.within("dx", got[0], dl @ w.double().cpu(), bound_x)
    xent.within("dw", got[1], dl.t() @ x.double().cpu(), bound_w)
    xent.within("dbias", got[2], dl.sum(0), slack.sum(0) + 40 * xent.U * parts.sum(0) + len(x) * 2.0 ** -126)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [5, 40, 150, 300, 600])
@pytest.mark.parametrize("held", ["largest", "inf", "nan"])
@pytest.mark.parametrize("d", [40, 17])
def test_what_rows_that_are_not_scored_hold(dev, dtype, n, held, d):
    """Padding that nothing has written: the other rows' results are those beside ordinary padding, as precise, and its
    own gradient is 0; rows whose loss has a gradient of 0 likewise."""
    x, w, t, b, dloss = xent.inputs(dev, dtype, n, 700, d, bias=True)
    out = torch.arange(n, device=dev) % 3 == 1
    t[out] = -1
    out[-1], dloss[-1] = True, 0.0
    bad = x.clone()
    bad[out] = {"largest": torch.finfo(dtype).max, "inf": math.inf, "nan": math.nan}[held]
    bad[out, ::2] *= -1
    x[out] = 0.0  # the size of what is scored alone
    loss, want = _grads(x, w, t, b, dloss)
    loss2, got = _grads(bad, w, t, b, dloss)
    assert not bool(loss2[t < 0].any()) and not bool(got[0][out].any())
    scored = ~out
    assert torch.allclose(loss2[scored], loss[scored], rtol=1e-5, atol=1e-5)
    _within(got, x, w, t, b, dloss)
    if dtype is not torch.float32:
        for g, k in zip(got, want):
            assert torch.equal(g, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [5, 40, 150, 300, 600])
def test_what_masked_tokens_weigh(dev, dtype, n):
    """Large weights of tokens that a bias of -inf masks: nothing of the other results is less precise."""
    x, w, t, b, dloss = xent.inputs(dev, dtype, n, 700, 40, bias=True, pad=True)
    b[3::7] = -math.inf
    t = torch.where(t % 7 == 3, t - 1, t)
    bad = w.clone()
    bad[3::7] = 6e4 if dtype is torch.float16 else 1e30
    w[3::7] = 0.0  # the size of what is not masked alone
    loss, want = _grads(x, w, t, b, dloss)
    loss2, got = _grads(x, bad, t, b, dloss)
    assert torch.equal(loss, loss2) and not bool(got[1][3::7].any()) and not bool(got[2][3::7].any())
    _within(got, x, w, t, b, dloss)
    for g, k in zip(got, want):
        assert torch.equal(g, k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [5, 300])
def test_an_infinite_weight_that_rules_a_token_out(dev, dtype, n):
    """Logits of -inf from the product: no gradient of that token's bias, whatever 0 times the weight is behind the last
    row."""
    x, w, t, b, dloss = xent.inputs(dev, dtype, n, 700, 40, bias=True)
    x, t = x.abs() + 0.1, t.clamp_min(1)
    w[0] = -math.inf
    loss, (_, dw, db) = _grads(x, w, t, b, dloss)
    assert bool(torch.isfinite(loss).all()) and bool(torch.isfinite(db).all()) and bool(torch.isfinite(dw).all())
    assert not bool(dw[0].any()) and db[0].item() == 0 and bool(db.any())
