"""linear_cross_entropy's backward where a workgroup takes many tiles of a short product, whatever is asked for."""

import pytest
import torch

import prlstm_amd
import test_gpu_cross_entropy as xent

pytestmark = pytest.mark.gpu


def _gradients(x, w, t, b, dloss, bias_too):
    leaves = [s.detach().requires_grad_(True) for s in ((x, w, b) if bias_too else (x, w))]
    loss = prlstm_amd.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2] if bias_too else b)
    return torch.autograd.grad(loss, leaves, dloss)[:2]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,v", [(1100, 20500), (1100, 40000), (500, 40000)])
@pytest.mark.parametrize("d", [24, 32, 64, 128, 136])
def test_without_a_gradient_of_the_bias(dev, dtype, n, v, d):
    """Up to a width of 128 a tile's product has no more slices than are in LDS.  405 tiles of 256 x 256 and 1570 and
    628 of 128 x 256 on 256 CUs: dx and dw are the same bits without a bias, with one of zeros that needs no gradient
    and with one that needs its own, whose sums meet behind a barrier of their own; and every time."""
    x, w, t, _, dloss = xent.inputs(dev, dtype, n, v, d, pad=True)
    zeros = torch.zeros(v, device=dev)
    want = _gradients(x, w, t, zeros, dloss, True)
    for bias in (None, zeros, None):
        for g, k in zip(_gradients(x, w, t, bias, dloss, False), want):
            assert torch.equal(g, k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_short_tiles_against_64_bits(dev, dtype):
    xent.check(*xent.inputs(dev, dtype, 1100, 20500, 72, pad=True))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [8, 9, 16, 17])
@pytest.mark.parametrize("v,d", [(32768, 264), (32768, 256), (26300, 264), (26100, 264)])
def test_few_rows_of_tiles_that_fill_the_chip(dev, dtype, n, v, d):
    """From 9 to 16 rows the vocabulary and the width decide whether the scoring runs on tiles (256, 206 or 204 of
    128 tokens on 256 CUs)."""
    xent.check(*xent.inputs(dev, dtype, n, v, d, bias=True, pad=True))
