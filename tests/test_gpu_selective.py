"""The selective layers (prlstm_amd.selective) against their formulas in 64 bits.

Tolerances: a result is rounded once to its type (half a step, eps / 2 of its value), and what it
sums is off by at most ``k`` roundings of 2^-24 of each term, where k counts the operations that a term
passes: per step of the recurrence the exponent's product, v_exp_f32, softplus and the two
products and sums (8 in all), so 8 T + 40 with the sums over states, channels and waves; for the
weights' sums the fp32 part of at most 256 steps and 8 waves.
"""

import pytest
import torch

import prlstm_amd
import selective_reference as ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def check(name, got, want, size, k):
    half = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype is torch.float16 else 0.0  # half of the smallest subnormal
    g = got.detach().double().cpu()
    assert g.shape == want.shape, (name, g.shape, want.shape)
    off = (g - want).abs() - (half * want.abs() + k * U * size + tiny)
    assert not bool(torch.isnan(off).any()), name
    assert off.numel() == 0 or off.max().item() <= 0, (name, off.max().item(), (g - want).abs().max().item())


def ordered(g, shape, dtype, order, dev):
    """Random [T, B, n] whose outer dimension in memory is time's, or the batch's."""
    t, b, n = shape
    if order == "time":
        return torch.randn(t, b, n, generator=g).to(dtype).to(dev)
    return torch.randn(b, t, n, generator=g).to(dtype).to(dev).transpose(0, 1)


def scan_inputs(dev, dtype, T, B, D, N, order="time", reset=0.0, state=True, gate=True, bias=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    # b and c are columns of one projection
    proj = ordered(g, (T, B, 2 * N + 3), dtype, order, dev)
    s = {"x": ordered(g, (T, B, D), dtype, order, dev), "delta": ordered(g, (T, B, D), dtype, order, dev),
         "a": (-torch.rand(D, N, generator=g) * 8 - 0.01).to(dev), "b": proj[..., 1:1 + N], "c": proj[..., 3 + N:]}
    s["d"] = torch.randn(D, generator=g).to(dev) if bias else None
    s["z"] = ordered(g, (T, B, D), dtype, order, dev) if gate else None
    s["delta_bias"] = (torch.randn(D, generator=g) - 2).to(dev) if bias else None
    s["h0"] = torch.randn(B, D, N, generator=g).to(dev) if state else None
    s["reset"] = (torch.rand(T, B, generator=g) < reset).to(dev) if reset else None
    return s, ordered(g, (T, B, D), dtype, order, dev), torch.randn(B, D, N, generator=g).to(dev)


def check_scan(s, dout, dh_n, **kw):
    leaves = {k: v.detach().requires_grad_(True) for k, v in s.items() if v is not None and k != "reset"}
    y, h = prlstm_amd.selective_scan(**{**s, **leaves}, **kw)
    T, k = y.shape[0], 8 * y.shape[0] + 40
    pairs = [(o, d) for o, d in ((y, dout), (h, dh_n)) if d is not None]
    grads = dict(zip(leaves, torch.autograd.grad([o for o, _ in pairs], list(leaves.values()),
                                                 [d for _, d in pairs])))
    want, size = (ref.scan(**s, **kw, dout=dout, dh_n=dh_n, magnitude=m) for m in (False, True))
    check("y", y, want["y"], size["y"], k)
    check("h", h, want["h"], size["h"], k)
    for name, grad in grads.items():
        assert grad.shape == leaves[name].shape and grad.dtype == leaves[name].dtype
        check(name, grad, want[name], size[name], 2 * k + 8)
    with torch.no_grad():
        y2, h2 = prlstm_amd.selective_scan(**s, **kw)
    if T == 1:  # the step's kernel, which sums in another order
        check("y", y2, want["y"], size["y"], k)
        check("h", h2, want["h"], size["h"], k)
    else:
        assert torch.equal(y2, y) and torch.equal(h2, h)
    return grads


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,B,D,N,order,reset,state,gate,bias", [
    (1, 1, 1, 1, "time", 0, False, False, False),
    (1, 2, 65, 16, "time", 0, True, True, True),
    (2, 3, 5, 3, "batch", 0.5, True, True, False),
    (16, 2, 64, 4, "time", 0, True, False, True),
    (17, 1, 130, 5, "batch", 0.2, False, True, True),
    (33, 2, 70, 16, "time", 0.1, True, True, True),
    (40, 3, 64, 17, "batch", 0, True, True, True),
    (31, 1, 66, 32, "time", 0.1, True, False, True),
    (25, 2, 65, 33, "batch", 0.1, True, True, True),
    (9, 1, 64, 64, "time", 0, False, True, False),
    (8, 2, 3, 2, "batch", 1.0, True, True, True),
])
def test_scan(dev, dtype, T, B, D, N, order, reset, state, gate, bias):
    check_scan(*scan_inputs(dev, dtype, T, B, D, N, order, reset, state, gate, bias))


@pytest.mark.parametrize("T,B,D,N,reset", [(130, 1, 70, 16, 0), (300, 2, 5, 3, 0.02), (257, 1, 64, 40, 0.01),
                                           (129, 1, 3, 8, 0), (400, 1, 65, 20, 0.3)])
def test_scan_in_segments(dev, T, B, D, N, reset):
    """Few channels: the time is cut into segments that run side by side."""
    check_scan(*scan_inputs(dev, torch.float32, T, B, D, N, "time", reset))


def test_scan_gradient_of_one_output(dev):
    s, dout, dh_n = scan_inputs(dev, torch.float32, 20, 2, 10, 6, reset=0.1)
    check_scan(s, dout, None)
    check_scan(s, None, dh_n)


def test_scan_without_softplus(dev):
    s, dout, dh_n = scan_inputs(dev, torch.float32, 40, 2, 20, 6, bias=False)
    s["delta"] = s["delta"].abs()
    check_scan(s, dout, dh_n, softplus=False)


def test_scan_of_extreme_steps(dev):
    """delta from far below, where softplus is exp, to far above, where it is delta itself."""
    s, dout, dh_n = scan_inputs(dev, torch.float32, 30, 1, 40, 4, bias=False)
    s["delta"] = torch.linspace(-40, 60, 1200, device=dev).reshape(30, 1, 40)
    check_scan(s, dout, dh_n)


@pytest.mark.parametrize("T,B,D,N", [(0, 2, 5, 4), (5, 0, 5, 4), (5, 2, 0, 4), (0, 0, 0, 1)])
def test_scan_of_nothing(dev, T, B, D, N):
    s, dout, dh_n = scan_inputs(dev, torch.bfloat16, T, B, D, N)
    leaves = {k: v.detach().requires_grad_(True) for k, v in s.items() if v is not None}
    y, h = prlstm_amd.selective_scan(**{**s, **leaves})
    assert y.shape == (T, B, D)
    grads = dict(zip(leaves, torch.autograd.grad((y, h), list(leaves.values()), (dout, dh_n))))
    if T == 0:
        assert torch.equal(h, s["h0"]) and torch.equal(grads["h0"], dh_n)
    for k, g in grads.items():
        assert g.shape == leaves[k].shape and (k == "h0" or not bool(g.any()))


@pytest.mark.parametrize("T", [20, 300])
def test_scan_keeps_sequences_apart(dev, T):
    """NaN and infinities of one sequence, of its state and of its gradients reach no other."""
    s, dout, dh_n = scan_inputs(dev, torch.float32, T, 2, 10, 6, state=True)
    cut = T // 2 + 1
    s["reset"] = torch.zeros(T, 2, dtype=torch.bool, device=dev)
    s["reset"][cut] = True

    def results(s, dout):
        leaves = {k: v.detach().requires_grad_(True) for k, v in s.items() if v is not None and k != "reset"}
        y, h = prlstm_amd.selective_scan(**{**s, **leaves})
        return y, h, dict(zip(leaves, torch.autograd.grad((y, h), list(leaves.values()), (dout, dh_n))))

    y, h, g = results(s, dout)
    bad = {k: v if v is None else v.clone() for k, v in s.items()}
    bad["x"][cut - 2], bad["h0"][0], bad["h0"][1] = float("inf"), float("nan"), float("inf")
    bad["b"][0] = float("nan")
    y2, h2, g2 = results(bad, dout)
    assert torch.equal(y2[cut:], y[cut:]) and torch.equal(h2, h)
    for k in ("x", "delta", "b", "c", "z"):
        assert torch.equal(g2[k][cut:], g[k][cut:]), k
    d2 = dout.clone()
    d2[cut + 1] = float("nan")
    _, _, g2 = results(s, d2)
    for k in ("x", "delta", "b", "c", "z"):
        assert torch.equal(g2[k][:cut], g[k][:cut]), k
    assert torch.equal(g2["h0"], g["h0"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,D,N", [(1, 1, 1), (3, 65, 16), (2, 10, 64), (5, 7, 5), (2, 33, 24)])
def test_scan_steps(dev, dtype, B, D, N):
    """Token by token, the state in place, against the whole sequence's formulas."""
    T = 6
    s, _, _ = scan_inputs(dev, dtype, T, B, D, N, reset=0.3)
    want, size = (ref.scan(**s, magnitude=m) for m in (False, True))
    h, pick = s["h0"].clone(), lambda k, t: None if s[k] is None else s[k][t]  # noqa: E731
    for t in range(T):
        args = {k: pick(k, t) for k in ("x", "delta", "b", "c", "z", "reset")}
        y, h2 = prlstm_amd.selective_scan_step(**args, a=s["a"], d=s["d"], delta_bias=s["delta_bias"], h=h)
        y3, h3 = prlstm_amd.selective_scan_step(**args, a=s["a"], d=s["d"], delta_bias=s["delta_bias"], h=h, h_out=h)
        assert h3 is h and torch.equal(h, h2) and torch.equal(y, y3)
        check("y", y, want["y"][t], size["y"][t], 8 * t + 48)
    check("h", h, want["h"], size["h"], 8 * T + 40)
    none, _ = prlstm_amd.selective_scan_step(**{k: pick(k, 0) for k in ("x", "delta", "b", "c")}, a=s["a"], h=None)
    alone = {k: s[k][:1] for k in ("x", "delta", "b", "c")}
    check("y", none, ref.scan(**alone, a=s["a"])["y"][0], ref.scan(**alone, a=s["a"], magnitude=True)["y"][0], 48)


def conv_inputs(dev, dtype, T, B, D, K, order="time", reset=0.0, state=True, bias=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    s = {"x": ordered(g, (T, B, D), dtype, order, dev), "weight": torch.randn(D, K, generator=g).to(dev),
         "bias": torch.randn(D, generator=g).to(dev) if bias else None,
         "state": torch.randn(B, K - 1, D, generator=g).to(dtype).to(dev) if state else None,
         "reset": (torch.rand(T, B, generator=g) < reset).to(dev) if reset else None}
    return s, ordered(g, (T, B, D), dtype, order, dev), torch.randn(B, K - 1, D, generator=g).to(dtype).to(dev)


def check_conv(s, dout, dstate_n, act=True):
    leaves = {k: v.detach().requires_grad_(True) for k, v in s.items() if v is not None and k != "reset"}
    y, n = prlstm_amd.causal_conv(**{**s, **leaves}, activation="silu" if act else None)
    pairs = [(o, d) for o, d in ((y, dout), (n, dstate_n)) if d is not None]
    grads = dict(zip(leaves, torch.autograd.grad([o for o, _ in pairs], list(leaves.values()),
                                                 [d for _, d in pairs], allow_unused=True)))
    want, size = (ref.conv(**s, act=act, dout=dout, dstate_n=dstate_n, magnitude=m) for m in (False, True))
    # a term passes K + 1 sums and, in silu or its slope, about 8 roundings and |u| <= size of exp's argument
    reach = size["y"].max().item() if size["y"].numel() else 0.0
    k = 20 + 4 * reach
    check("y", y, want["y"], size["y"], k)
    assert torch.equal(n.double().cpu(), want["state_n"])
    for name, grad in grads.items():
        if grad is None:
            assert want[name].numel() == 0
            continue
        # slope's error is absolute: it is a sum of s and u s (1 - s), each below 1.2
        grew = ref.conv(**s, act=False, dout=dout, dstate_n=dstate_n, magnitude=True)[name]
        check(name, grad, want[name], 2 * grew + size[name], k + (280 if name in ("weight", "bias") else 0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,B,D,K,order,reset,state,bias,act", [
    (1, 1, 1, 1, "time", 0, False, False, True),
    (1, 2, 9, 4, "time", 0.5, True, True, True),
    (2, 3, 5, 4, "batch", 0.3, True, True, True),
    (3, 1, 7, 4, "time", 0, True, False, False),
    (8, 2, 64, 3, "time", 0, False, True, True),
    (17, 3, 130, 2, "batch", 0.2, True, True, True),
    (33, 2, 65, 4, "time", 0.2, True, True, True),
    (40, 1, 515, 3, "batch", 0.1, True, True, False),
    (66, 2, 8, 4, "time", 1.0, True, True, True),
    (20, 5, 3, 1, "time", 0.2, False, True, True),
    (300, 3, 12, 4, "batch", 0.05, True, True, True),
])
def test_conv(dev, dtype, T, B, D, K, order, reset, state, bias, act):
    check_conv(*conv_inputs(dev, dtype, T, B, D, K, order, reset, state, bias), act)


def test_conv_gradient_of_one_output(dev):
    s, dout, dn = conv_inputs(dev, torch.float32, 20, 2, 10, 4, reset=0.1)
    check_conv(s, dout, None)
    check_conv(s, None, dn)
    s, dout, dn = conv_inputs(dev, torch.float32, 2, 2, 10, 4)
    check_conv(s, None, dn)


@pytest.mark.parametrize("T,B,D", [(0, 2, 5), (5, 0, 5), (5, 2, 0)])
def test_conv_of_nothing(dev, T, B, D):
    s, dout, dn = conv_inputs(dev, torch.bfloat16, T, B, D, 4)
    leaves = {k: v.detach().requires_grad_(True) for k, v in s.items() if v is not None}
    y, n = prlstm_amd.causal_conv(**leaves)
    assert y.shape == (T, B, D)
    grads = dict(zip(leaves, torch.autograd.grad((y, n), list(leaves.values()), (dout, dn))))
    if T == 0:
        assert torch.equal(n, s["state"]) and torch.equal(grads["state"], dn)
    assert not bool(grads["weight"].any()) and not bool(grads["bias"].any())


def test_conv_keeps_sequences_apart(dev):
    T, cut = 40, 21
    s, dout, dn = conv_inputs(dev, torch.float32, T, 2, 10, 4)
    s["reset"] = torch.zeros(T, 2, dtype=torch.bool, device=dev)
    s["reset"][cut] = True

    def results(s, dout):
        leaves = {k: v.detach().requires_grad_(True) for k, v in s.items() if v is not None and k != "reset"}
        y, n = prlstm_amd.causal_conv(**{**s, **leaves})
        return y, n, dict(zip(leaves, torch.autograd.grad((y, n), list(leaves.values()), (dout, dn))))

    y, n, g = results(s, dout)
    bad = {k: v.clone() for k, v in s.items()}
    bad["x"][cut - 1], bad["x"][cut - 3], bad["state"][0] = float("nan"), float("inf"), float("nan")
    y2, n2, g2 = results(bad, dout)
    assert torch.equal(y2[cut:], y[cut:]) and torch.equal(n2, n) and torch.equal(g2["x"][cut:], g["x"][cut:])
    d2 = dout.clone()
    d2[cut] = float("nan")
    _, _, g2 = results(s, d2)
    assert torch.equal(g2["x"][:cut], g["x"][:cut]) and torch.equal(g2["state"], g["state"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,D,K", [(1, 1, 1), (3, 65, 4), (2, 10, 3), (5, 7, 2)])
def test_conv_steps(dev, dtype, B, D, K):
    T = 7
    s, _, _ = conv_inputs(dev, dtype, T, B, D, K, reset=0.3)
    want, size = (ref.conv(**s, magnitude=m) for m in (False, True))
    state, k = s["state"].clone(), 20 + 4 * size["y"].max().item()
    for t in range(T):
        args = dict(x=s["x"][t], weight=s["weight"], bias=s["bias"], reset=s["reset"][t])
        y, n = prlstm_amd.causal_conv_step(state=state, **args)
        y2, n2 = prlstm_amd.causal_conv_step(state=state, state_out=state, **args)
        assert n2 is state and torch.equal(n, state) and torch.equal(y, y2)
        check("y", y, want["y"][t], size["y"][t], k)
    assert torch.equal(state.double().cpu(), want["state_n"])


def test_strides(dev):
    """Inputs that are columns of wider tensors, or not dense at all, or repeated over the batch."""
    s, dout, dh_n = scan_inputs(dev, torch.bfloat16, 20, 3, 20, 6)
    wide = torch.randn(20, 3, 70, device=dev).bfloat16()
    s.update(x=wide[..., 3:23], delta=wide[..., 25:45], z=wide[..., 50:70].flip(-1))
    s["b"] = wide[:, :1, :6].expand(20, 3, 6)
    s["c"] = wide[..., :12:2]
    check_scan(s, dout[:, :1].expand_as(dout), dh_n.transpose(0, 1).contiguous().transpose(0, 1))
    c, dout, dn = conv_inputs(dev, torch.bfloat16, 20, 3, 20, 4)
    c["x"], c["weight"] = wide[..., 5:25], torch.randn(4, 20, device=dev).t()
    check_conv(c, dout[:, :1].expand_as(dout), dn)


def test_weights_of_another_type(dev):
    """16-bit weights count as their values, and their gradients are rounded to their type."""
    s, dout, dh_n = scan_inputs(dev, torch.bfloat16, 12, 2, 10, 4)
    for k in ("a", "d", "delta_bias", "h0"):
        s[k] = s[k].bfloat16()
    check_scan(s, dout, dh_n)


def test_captured_training_step(dev):
    """Forward and backward of both in a graph that is replayed on new inputs, between eager calls."""
    c, _, _ = conv_inputs(dev, torch.bfloat16, 200, 2, 72, 4, reset=0.02)
    s, dout, dh_n = scan_inputs(dev, torch.bfloat16, 200, 2, 72, 16, reset=0.02)

    def step(c, s, dout):
        conv = {k: v.detach().requires_grad_(True) for k, v in c.items() if v is not None and k != "reset"}
        leaves = {k: v.detach().requires_grad_(True) for k, v in s.items() if v is not None and k not in ("x", "reset")}
        x, _ = prlstm_amd.causal_conv(**{**c, **conv})
        y, h = prlstm_amd.selective_scan(**{**s, **leaves, "x": x})
        every = {**{"conv_" + k: v for k, v in conv.items()}, **leaves}
        return y.detach(), h.detach(), *torch.autograd.grad((y, h), list(every.values()), (dout, dh_n))

    step(c, s, dout)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(c, s, dout)
    for seed in range(3):
        c2, _, _ = conv_inputs(dev, torch.bfloat16, 200, 2, 72, 4, reset=0.02, seed=seed + 5)
        s2, d2, _ = scan_inputs(dev, torch.bfloat16, 200, 2, 72, 16, reset=0.02, seed=seed + 5)
        for old, new in ((c, c2), (s, s2)):
            for k, v in new.items():
                if v is not None:
                    old[k].copy_(v)
        dout.copy_(d2)
        graph.replay()
        want = step(c, s, dout)
        torch.cuda.synchronize()
        for got, w in zip(captured, want):
            assert torch.equal(got, w)


def test_on_another_stream(dev):
    s, dout, dh_n = scan_inputs(dev, torch.bfloat16, 200, 2, 72, 16)
    c, _, _ = conv_inputs(dev, torch.bfloat16, 200, 2, 72, 4)
    want = prlstm_amd.selective_scan(**s), prlstm_amd.causal_conv(**c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = prlstm_amd.selective_scan(**s), prlstm_amd.causal_conv(**c)
    torch.cuda.current_stream().wait_stream(side)
    for g, w in zip(got, want):
        assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])


def test_state_changed_in_place_is_known(dev):
    """A backward that has saved a state which a step then overwrites is refused, as torch's own are."""
    state = torch.zeros(2, 3, 8, device=dev)
    w = torch.ones(8, 4, device=dev, requires_grad=True)
    y, _ = prlstm_amd.causal_conv(torch.ones(5, 2, 8, device=dev), w, state=state)
    prlstm_amd.causal_conv_step(torch.ones(2, 8, device=dev), state, w, state_out=state)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


def test_results_repeat(dev):
    s, dout, dh_n = scan_inputs(dev, torch.bfloat16, 100, 4, 200, 16)
    first = check_scan(s, dout, dh_n)
    for _ in range(3):
        again = check_scan(s, dout, dh_n)
        assert all(torch.equal(first[k], again[k]) for k in first)
