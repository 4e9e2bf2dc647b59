"""linear_cross_entropy's backward of 16-bit operands in scaled fp16 (more than 128 bf16 rows; fp16 ones in two numbers
up to 512 rows): gradients and operands of sizes far apart.  Tolerances as in test_gpu_cross_entropy."""

import pytest
import torch

import prlstm_amd
import test_gpu_cross_entropy as xent

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("n", [129, 150, 600])
def test_gradients_of_unlike_rows(dev, n):
    """Rows' gradients over 30 decades, each as precise as alone; whatever comes with a row that is not scored."""
    x, w, t, b, dloss = xent.inputs(dev, BF16, n, 400, 24, bias=True)
    dloss = dloss * 10.0 ** torch.linspace(-15, 15, n, device=dev)
    xent.check(x, w, t, b, dloss)
    t[7], t[40], t[41] = -1, -1, -5
    want = xent.check(x, w, t, b, dloss)[1]
    for other in (1e30, float("inf"), float("nan"), 0.0):
        dloss[[7, 40, 41]] = other
        leaves = [s.detach().requires_grad_(True) for s in (x, w, b)]
        loss = prlstm_amd.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
        for g, k in zip(torch.autograd.grad(loss, leaves, dloss), want):
            assert torch.equal(g, k)


@pytest.mark.parametrize("n", [150, 600])
def test_gradients_of_unlike_rows_in_fp16(dev, n):
    """Over six decades, which leave the results within fp16's range."""
    x, w, t, b, dloss = xent.inputs(dev, F16, n, 400, 24, bias=True, pad=True)
    xent.check(x, w, t, b, dloss * 10.0 ** torch.linspace(-3, 3, n, device=dev))


@pytest.mark.parametrize("n", [129, 150, 600])
@pytest.mark.parametrize("up", [2.0 ** 60, 2.0 ** -60, 0.0])
def test_sizes_of_the_operands(dev, n, up):
    """Operands near the ends of bf16's range, whose products fp16 could not hold."""
    x, w, t, b, dloss = xent.inputs(dev, BF16, n, 300, 24)
    if up:
        xent.check(x * up, w / up, t, b, dloss)
    else:
        xent.check(x * 0, w, t, b, dloss)
        xent.check(x, w * 0, t, b, dloss)


@pytest.mark.parametrize("dtype,n", [(BF16, 150), (BF16, 600), (F16, 150), (F16, 600)])
def test_elements_of_unlike_sizes(dev, dtype, n):
    """Columns of x over eight decades (fp16: six), the weight's the other way."""
    x, w, t, b, dloss = xent.inputs(dev, dtype, n, 300, 24)
    far = 4 if dtype is BF16 else 3
    by = 2.0 ** torch.linspace(-far * 3.3, far * 3.3, 24, device=dev).round()
    xent.check((x.float() * by).to(dtype), (w.float() / by).to(dtype), t, b, dloss)
