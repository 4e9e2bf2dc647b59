"""linear_cross_entropy against its formulas in 64 bits.

Tolerances.  A logit is a sum of D exact products (16-bit operands) or of D products, in fp32: off by at most
(D + 4) 2^-24 of the sum of the products' sizes; `shift` is the largest of these of a row.  The loss is off
by twice that and a few roundings of its parts.  A probability is off by the factor exp(2 shift + 2^-18), the
last for exp's and the sum's own roundings.  16-bit operands: dl is rounded to fp16 (2^-11 of itself), then a
product's sum of n terms is off by (n + 8) 2^-24 of their sizes, and the result is rounded once.  fp16's last
place is 2^-24, so that what is rounded there is off by 2^-25; the scales put 2^14 or more at each row's g, at
the largest element of x times the largest g (an element of a row whose g is smaller has as much less), and at
that of a bf16 w: 2^-39 of g for dl, 2^-39 max|x| max|g| / |g| for x, 2^-39 max|w| for w.  What is below the
smallest normal number, 2^-126, may be 0: a probability, a gradient dl, or either of the later two of the three
pieces that an fp32 product's operand is split into: 4 2^-126 of each dl.
"""

import math

import pytest
import torch

import prlstm_amd

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def reference(x, w, targets, bias, dloss):
    """loss, dl, and the sizes that the tolerances are measured against, in 64 bits on the CPU."""
    x, w, dloss = (t.detach().double().cpu() for t in (x, w, dloss))
    t = targets.cpu().long()
    b = torch.zeros(w.shape[0], dtype=torch.float64) if bias is None else bias.detach().double().cpu()
    l = x @ w.t() + b
    size = x.abs() @ w.abs().t() + torch.where(torch.isinf(b), torch.zeros_like(b), b.abs())
    there = (t >= 0) & (t < w.shape[0])
    empty = (l == -math.inf).all(1)
    lse = torch.logsumexp(l, 1)
    loss = torch.where(there, lse - l.gather(1, t.clamp(0, w.shape[0] - 1)[:, None])[:, 0], torch.zeros_like(lse))
    loss[there & empty] = math.inf
    loss[t >= w.shape[0]] = math.nan
    g = torch.where(there & ~empty, dloss, torch.zeros_like(dloss))
    p = torch.exp(l - torch.where(empty, torch.zeros_like(lse), lse)[:, None])
    hot = torch.zeros_like(p)
    hot[there, t[there]] = 1.0
    masked = l == -math.inf
    dl = torch.where(masked, torch.zeros_like(p), g[:, None] * (p - hot))
    parts = torch.where(masked, torch.zeros_like(p), g.abs()[:, None] * (p + hot))  # of dl
    return loss, dl, parts, size.amax(1) if size.numel() else lse * 0


def within(name, got, want, bound):
    half = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype is torch.float16 else 0.0
    g = got.detach().double().cpu()
    assert g.shape == want.shape, (name, g.shape, want.shape)
    same = (g == want) | (torch.isnan(g) & torch.isnan(want))
    off = (g - want).abs() - (half * want.abs() + bound + tiny)
    bad = ~same & ~(off <= 0)
    assert not bool(bad.any()), (name, int(bad.sum()), off[bad].max().item())


def bounds(x, w, targets, dl, parts, shift, dloss):
    """The error of dl in fp32, and those of dx and dw before they are rounded."""
    (n, v), d = dl.shape, x.shape[1]
    slack = (torch.expm1(2 * shift)[:, None] + 2 ** -18) * parts
    x64, w64, g = x.detach().double().cpu().abs(), w.detach().double().cpu().abs(), dloss.detach().double().cpu().abs()
    err, off_x, off_w = slack + 4 * 2.0 ** -126, torch.zeros(n, 1), 0.0
    if x.dtype is not torch.float32 and n:
        g = torch.where((targets.cpu() >= 0) & (targets.cpu() < v), g, torch.zeros_like(g))
        err = err + 2.0 ** -11 * dl.abs() + 2.0 ** -39 * g[:, None]
        off_x = 2.0 ** -39 * x64.max() * (g.max() / torch.where(g > 0, g, g.max().clamp_min(1e-300)))[:, None]
        if x.dtype is torch.bfloat16:
            off_w = 2.0 ** -39 * w64.max()
    reach = parts + err  # what dl is at most
    bound_x = err @ w64 + (reach * off_w).sum(1, keepdim=True) + (v + 8) * U * (reach @ w64)
    bound_w = err.t() @ x64 + (reach * off_x).sum(0)[:, None] + (n + 8) * U * (reach.t() @ x64)
    return slack, bound_x, bound_w


def check(x, w, targets, bias, dloss):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, bias) if t is not None]
    loss = prlstm_amd.linear_cross_entropy(leaves[0], leaves[1], targets, bias=leaves[2] if bias is not None else None)
    grads = torch.autograd.grad(loss, leaves, dloss)
    with torch.no_grad():
        alone = prlstm_amd.linear_cross_entropy(x, w, targets, bias=bias)
    want, dl, parts, size = reference(x, w, targets, bias, dloss)
    n, d = x.shape
    v = w.shape[0]
    shift = (d + 4) * U * size
    finite = torch.where(torch.isfinite(want), want.abs(), torch.zeros_like(want))
    if n > (64 if x.dtype is torch.float32 else 16):  # fewer rows alone are summed in another order
        assert torch.equal(torch.nan_to_num(alone, -1.0), torch.nan_to_num(loss, -1.0))
    within("loss alone", alone, want, 2 * shift + 16 * U * (finite + size + math.log(v + 1)) + 2 ** -20)
    within("loss", loss, want, 2 * shift + 16 * U * (finite + size + math.log(v + 1)) + 2 ** -20)
    slack, bound_x, bound_w = bounds(x, w, targets, dl, parts, shift, dloss)
    x64, w64 = x.detach().double().cpu(), w.detach().double().cpu()
    assert grads[0].dtype is x.dtype and grads[1].dtype is w.dtype
    within("dx", grads[0], dl @ w64, bound_x)
    within("dw", grads[1], dl.t() @ x64, bound_w)
    if bias is not None:
        # each of the n terms may be 0 where it is below 2^-126
        within("dbias", grads[2], dl.sum(0), slack.sum(0) + 40 * U * parts.sum(0) + n * 2.0 ** -126)
    return loss, grads


def inputs(dev, dtype, n, v, d, bias=False, pad=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    x, w = torch.randn(n, d, generator=g), 1.5 * d ** -0.5 * torch.randn(v, d, generator=g)
    t = torch.randint(0, v, (n,), generator=g)
    if n:
        x = x + 3 * torch.rand(n, 1, generator=g) * w[t]
    b = torch.randn(v, generator=g).to(dev) if bias else None
    if pad and n:
        t[torch.rand(n, generator=g) < 0.3] = -1
    dloss = torch.randn(n, generator=g) / max(1, n)
    return x.to(dtype).to(dev), w.to(dtype).to(dev), t.to(dev), b, dloss.to(dev)


SIZES = [(1, 1, 1), (9, 40, 3), (40, 100, 2), (20, 77, 6), (64, 90, 1100), (1, 300, 8), (2, 2, 5), (3, 257, 64), (5, 1000, 72), (70, 513, 130), (256, 256, 64),
         (300, 700, 264), (257, 255, 17), (33, 5000, 40), (600, 90, 500), (1, 20000, 128)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,d", SIZES)
@pytest.mark.parametrize("extra", [False, True])
def test_against_64_bits(dev, dtype, n, v, d, extra):
    check(*inputs(dev, dtype, n, v, d, bias=extra, pad=extra))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,v,d", [(64, 70000, 32), (20000, 500, 24)])
def test_sums_split_between_workgroups(dev, dtype, n, v, d):
    """Long sums of few results."""
    check(*inputs(dev, dtype, n, v, d, bias=True))


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_tokens(dev, dtype):
    """-inf in the bias: no probability and no gradient; a masked target has loss inf."""
    x, w, t, b, dloss = inputs(dev, dtype, 40, 600, 48, bias=True)
    b[::3] = -math.inf
    b[300:560] = -math.inf  # a whole tile's worth
    t = t // 3 * 3 + 1
    t[t >= 300] = 1
    t[7] = 3
    t[9] = -5
    loss, grads = check(x, w, t, b, dloss)
    assert loss[7].item() == math.inf and loss[9].item() == 0
    assert not bool(grads[1][::3].any()) and not bool(grads[2][::3].any()) and not bool(grads[0][9].any())


@pytest.mark.parametrize("dtype", TYPES)
def test_nothing_but_masks(dev, dtype):
    x, w, t, b, dloss = inputs(dev, dtype, 5, 300, 16, bias=True)
    b[:] = -math.inf
    t[1] = -1
    leaves = [s.detach().requires_grad_(True) for s in (x, w, b)]
    loss = prlstm_amd.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
    assert loss.tolist() == [math.inf, 0.0] + [math.inf] * 3
    for g in torch.autograd.grad(loss, leaves, dloss):
        assert not bool(g.any())


@pytest.mark.parametrize("dtype", TYPES)
def test_non_finite_rows_stay_apart(dev, dtype):
    """A row of x with NaN or infinities makes its own loss and gradient NaN and no other row's; where its
    target is negative it makes nothing but its loss of 0."""
    x, w, t, b, dloss = inputs(dev, dtype, 300, 700, 40)
    loss, _ = check(x, w, t, b, dloss)
    bad = x.clone()
    bad[5], bad[290, 3] = math.nan, math.inf
    xs = bad.requires_grad_(True)
    l2 = prlstm_amd.linear_cross_entropy(xs, w, t)
    dx, = torch.autograd.grad(l2, xs, dloss)
    rest = torch.ones(300, dtype=torch.bool, device=dev)
    rest[[5, 290]] = False
    assert torch.isnan(l2[~rest]).all() and torch.equal(l2[rest], loss[rest])
    assert bool(torch.isnan(dx[~rest]).any(1).all()) and bool(torch.isfinite(dx[rest]).all())


def test_large_logits(dev):
    """Logits far beyond exp's range, of both signs."""
    x, w, t, b, dloss = inputs(dev, torch.float32, 50, 400, 24)
    check(x * 100, w, t, b, dloss)
    x, w, t, b, dloss = inputs(dev, torch.bfloat16, 50, 400, 24)
    check(x * 64, w, t, b, dloss)


@pytest.mark.parametrize("scale", [0.0, 1e-30, 1e30])
def test_sizes_of_the_gradient(dev, scale):
    """fp16's products run on scaled gradients."""
    x, w, t, b, dloss = inputs(dev, torch.float16, 30, 400, 24, bias=True)
    leaves = [s.detach().requires_grad_(True) for s in (x, w, b)]
    loss = prlstm_amd.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
    got = torch.autograd.grad(loss, leaves, dloss * scale)
    assert all(bool(torch.isfinite(g).all()) for g in (got if scale < 1 else got[2:]))
    _, dl, parts, size = reference(x, w, t, b, dloss * scale)  # a gradient may cancel, its parts do not
    slack = (torch.expm1(2 * (24 + 4) * U * size)[:, None] + 2 ** -18) * parts + 4 * 2.0 ** -126
    within("dbias", got[2], dl.sum(0), slack.sum(0) + 40 * U * parts.sum(0))
    if scale == 1e30:
        assert not bool(torch.isnan(got[0]).any())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 7, 16, 17, 33, 64, 65, 128, 129])
def test_few_rows(dev, dtype, n):
    """Around the sizes where another kernel takes over: whole runs of tokens masked, among them targets, rows not
    scored, logits far below zero, a row of NaN."""
    x, w, t, b, dloss = inputs(dev, dtype, n, 1100, 72, bias=True, pad=n > 7)
    b[100:700] = -math.inf
    check(x, w, t, b, dloss)
    check(x * 16, w, t, b - 300, dloss)
    loss = prlstm_amd.linear_cross_entropy(x, w, t, bias=b)
    size = reference(x, w, t, b, dloss)[3].max().item()
    x[n // 2] = math.nan
    again = prlstm_amd.linear_cross_entropy(x, w, t, bias=b)
    rest = torch.arange(n, device=dev) != n // 2
    if dtype is torch.float32:
        # tiles of an fp32 product that hold a NaN are computed by other instructions: both results are within
        # the loss's bound, (2 (72 + 4) + 3 * 16) 2^-24 of size + log v and 2^-20 at most where it is finite
        far = 2 * ((2 * 76 + 48) * U * (size + 8) + 2 ** -20)
        assert bool(((again - loss)[rest].nan_to_num(0.0).abs() <= far).all()) and not bool(again[rest].isnan().any())
    else:
        assert torch.equal(again[rest], loss[rest])
    assert t[n // 2] < 0 or bool(torch.isnan(again[n // 2]))
    b[:] = -math.inf
    again = prlstm_amd.linear_cross_entropy(x, w, t, bias=b)
    assert bool(torch.isinf(again[rest & (t >= 0)]).all())


def test_gradients_of_unlike_rows(dev):
    """Rows' gradients over 30 decades, each as precise as alone; whatever comes with a row that is not scored."""
    x, w, t, b, dloss = inputs(dev, torch.bfloat16, 61, 400, 24, bias=True)
    check(x, w, t, b, dloss * 10.0 ** torch.linspace(-15, 15, 61, device=dev))
    t[7], t[40], t[41] = -1, -1, -5
    want = check(x, w, t, b, dloss)[1]
    for other in (1e30, float("inf"), float("nan"), 0.0):
        dloss[[7, 40, 41]] = other
        for g, k in zip(check(x, w, t, b, torch.where(t < 0, torch.zeros_like(dloss), dloss))[1], want):
            assert torch.equal(g, k)
        leaves = [s.detach().requires_grad_(True) for s in (x, w, b)]
        loss = prlstm_amd.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
        for g, k in zip(torch.autograd.grad(loss, leaves, dloss), want):
            assert torch.equal(g, k)


def test_sizes_of_the_operands(dev):
    """Operands near the ends of bf16's range, whose products fp16 could not hold."""
    x, w, t, b, dloss = inputs(dev, torch.bfloat16, 40, 300, 24)
    for up in (2.0 ** 60, 2.0 ** -60):
        check(x * up, w / up, t, b, dloss)
    check(x * 0, w, t, b, dloss)
    check(x, w * 0, t, b, dloss)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,d", [(300, 17000, 40), (300, 40000, 24), (1100, 20500, 24)])
def test_many_tiles(dev, dtype, n, v, d):
    """Tiles of 256 tokens (134, 405 of them) and of 128 (628), one and several for a workgroup."""
    check(*inputs(dev, dtype, n, v, d, bias=True, pad=True))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 2, 200])
def test_gradients_are_rounded_once(dev, dtype, n):
    """As far from the exact ones as their rounding, not as two of them: the products' own error is at most
    2^-11 of their terms' sizes, an eighth of bf16's half step."""
    x, w, t, b, dloss = inputs(dev, dtype, n, 500, 32)
    grads = check(x, w, t, b, dloss)[1]
    _, dl, _, _ = reference(x, w, t, b, dloss)
    for g, k in zip(grads, (dl @ w.double().cpu(), dl.t() @ x.double().cpu())):
        once = (k.to(dtype).double() - k).norm()
        own = 2.0 ** -11 * k.norm() * 2  # sums of terms of random signs are as large as their errors
        assert (g.double().cpu() - k).norm() <= once + own


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_shapes(dev, dtype):
    """Rows cut from wider tensors, at odd offsets, transposed, repeated; leading dimensions; int32."""
    x, w, t, b, dloss = inputs(dev, dtype, 60, 300, 40, bias=True)
    want, grads = check(x, w, t, b, dloss)
    wide_x, wide_w = torch.zeros(60, 101, device=dev, dtype=dtype), torch.zeros(300, 64, device=dev, dtype=dtype)
    wide_x[:, 3:43], wide_w[:, 8:48] = x, w
    for xs, ws in ((wide_x[:, 3:43], wide_w[:, 8:48]), (x.t().contiguous().t(), w.t().contiguous().t())):
        leaves = [s.detach().requires_grad_(True) for s in (xs, ws, b)]
        loss = prlstm_amd.linear_cross_entropy(leaves[0], leaves[1], t.int(), bias=leaves[2])
        assert torch.equal(loss, want)
        for g, k in zip(torch.autograd.grad(loss, leaves, dloss), grads):
            assert torch.equal(g, k)
    lead = prlstm_amd.linear_cross_entropy(x.reshape(3, 4, 5, 40), w, t.reshape(3, 4, 5), bias=b)
    assert lead.shape == (3, 4, 5)
    assert torch.equal(lead.reshape(-1), prlstm_amd.linear_cross_entropy(x, w, t, bias=b))
    check(x[:1].expand(60, 40), w, t, b, dloss)
    assert prlstm_amd.linear_cross_entropy(x[0], w, t[0], bias=b).shape == ()


@pytest.mark.parametrize("dtype", TYPES)
def test_of_nothing(dev, dtype):
    x, w, t, b, dloss = inputs(dev, dtype, 0, 30, 8, bias=True)
    leaves = [s.detach().requires_grad_(True) for s in (x, w, b)]
    loss = prlstm_amd.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
    assert loss.shape == (0,)
    for g in torch.autograd.grad(loss, leaves, dloss):
        assert not bool(g.any())


def test_some_gradients(dev):
    """Only what is asked for, whatever the rest is."""
    x, w, t, b, dloss = inputs(dev, torch.bfloat16, 60, 300, 40, bias=True)
    leaves = [s.detach().requires_grad_(True) for s in (x, w, b)]
    loss = prlstm_amd.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
    all_of = torch.autograd.grad(loss, leaves, dloss)
    for k in range(3):
        args = [x, w, b]
        args[k] = leaves[k]
        g, = torch.autograd.grad(prlstm_amd.linear_cross_entropy(args[0], args[1], t, bias=args[2]), leaves[k], dloss)
        assert torch.equal(g, all_of[k])


def test_targets_beyond_the_vocabulary(dev):
    prlstm_amd.check_errors()
    x, w, t, b, dloss = inputs(dev, torch.bfloat16, 60, 300, 40)
    t[3], t[5] = 300, 1 << 40
    leaves = [s.detach().requires_grad_(True) for s in (x, w)]
    loss = prlstm_amd.linear_cross_entropy(leaves[0], leaves[1], t)
    assert torch.isnan(loss).nonzero()[:, 0].tolist() == [3, 5]
    dx, dw = torch.autograd.grad(loss, leaves, dloss)
    assert not bool(dx[[3, 5]].any()) and bool(torch.isfinite(dw).all())
    with pytest.raises(RuntimeError, match="vocabulary"):
        prlstm_amd.check_errors()


def test_refusals(dev):
    z = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device=dev)  # noqa: E731
    t = torch.zeros(3, dtype=torch.int64, device=dev)
    f = prlstm_amd.linear_cross_entropy
    for call, text in ((lambda: f(z(3, 4), z(5, 6), t), "weight"), (lambda: f(z(3, 4), z(5, 4), t[:2]), "targets must"),
                       (lambda: f(z(3, 4), z(5, 4, dt=torch.bfloat16), t), "weight must be"),
                       (lambda: f(z(3, 4, dt=torch.float64), z(5, 4, dt=torch.float64), t), "x must be"),
                       (lambda: f(z(3, 4), z(5, 4), t.float()), "int64 or int32"),
                       (lambda: f(z(3, 4), z(5, 4), t, bias=z(4)), "bias must"),
                       (lambda: f(z(3, 4), z(0, 4), t), "must not be empty"),
                       (lambda: f(z(3, 0), z(5, 0), t), "must not be empty"),
                       (lambda: f(z(3, 4), z(5, 4), t.cpu()), "targets is on"),
                       (lambda: f(z(3, 4), z(5, 4).cpu(), t), "weight must be")):
        with pytest.raises(RuntimeError, match=text):
            call()


@pytest.mark.parametrize("dtype", TYPES)
def test_captured_training_step(dev, dtype):
    x, w, t, b, dloss = inputs(dev, dtype, 300, 700, 40, bias=True)

    def step():
        leaves = [s.detach().requires_grad_(True) for s in (x, w, b)]
        loss = prlstm_amd.linear_cross_entropy(leaves[0], leaves[1], t, bias=leaves[2])
        return loss.detach(), *torch.autograd.grad(loss, leaves, dloss)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        for old, new in zip((x, w, t, b, dloss), inputs(dev, dtype, 300, 700, 40, bias=True, seed=seed + 3)):
            old.copy_(new)
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        for got, k in zip(captured, want):
            assert torch.equal(got, k)
