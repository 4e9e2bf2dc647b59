"""The selective layers and the loss without logits at their limits: offsets beyond 2^31 elements, refused calls,
gradients of other layouts, operands that overlap, graphs beside each other."""

import math

import pytest
import torch
import torch.autograd.forward_ad as fwad

import prlstm_amd
import selective_reference as ref
import test_gpu_cross_entropy as xent
import test_gpu_selective as sel

pytestmark = pytest.mark.gpu
TAIL = 40  # steps or rows at the end that are compared
BF16 = torch.bfloat16


def _long(dev, t, tail):
    """[t, *tail.shape[1:]] of sevens that ends with tail."""
    x = torch.full((t, *tail.shape[1:]), 7.0, dtype=tail.dtype, device=dev)
    x[t - len(tail):] = tail
    return x


def test_conv_beyond_32_bits(dev):
    """More than 2^31 elements, the last document of which is compared with what it is alone."""
    T, B, D = (1 << 18) + TAIL, 2, 4100
    s, dout, dn = sel.conv_inputs(dev, BF16, TAIL, B, D, 4, state=False)
    x = _long(dev, T, s["x"]).requires_grad_(True)
    w, b = s["weight"].requires_grad_(True), s["bias"].requires_grad_(True)
    s["reset"] = torch.zeros(TAIL, B, dtype=torch.bool, device=dev)
    s["reset"][0] = True
    reset = torch.zeros(T, B, dtype=torch.bool, device=dev)
    reset[T - TAIL] = True
    y, n = prlstm_amd.causal_conv(x, w, b, reset=reset)
    dy = torch.zeros_like(y)
    dy[T - TAIL:] = dout
    dx, dw, db = torch.autograd.grad((y, n), (x, w, b), (dy, dn))
    want, size = (ref.conv(**s, dout=dout, dstate_n=dn, magnitude=m) for m in (False, True))
    grew = ref.conv(**s, act=False, dout=dout, dstate_n=dn, magnitude=True)
    k = 20 + 4 * size["y"].max().item()
    sel.check("y", y[T - TAIL:], want["y"], size["y"], k)
    assert torch.equal(n.double().cpu(), want["state_n"])
    sel.check("dx", dx[T - TAIL:], want["x"], 2 * grew["x"] + size["x"], k)
    for name, grad in (("weight", dw), ("bias", db)):
        sel.check(name, grad, want[name], 2 * grew[name] + size[name], k + 280)
    assert not bool(dx[:T - TAIL].any())


def test_scan_beyond_32_bits(dev):
    T, B, D, N = (1 << 18) + TAIL, 2, 4100, 2
    s, dout, dh_n = sel.scan_inputs(dev, BF16, TAIL, B, D, N, state=False)
    s["b"], s["c"] = s["b"].contiguous(), s["c"].contiguous()
    s["reset"] = torch.zeros(TAIL, B, dtype=torch.bool, device=dev)
    s["reset"][0] = True
    streams = ("x", "delta", "b", "c", "z")
    leaves = {k: (_long(dev, T, v) if k in streams else v).requires_grad_(True) for k, v in s.items()
              if v is not None and k != "reset"}
    reset = torch.zeros(T, B, dtype=torch.bool, device=dev)
    reset[T - TAIL] = True
    y, h = prlstm_amd.selective_scan(**leaves, reset=reset)
    dy = torch.zeros_like(y)
    dy[T - TAIL:] = dout
    grads = dict(zip(leaves, torch.autograd.grad((y, h), list(leaves.values()), (dy, dh_n))))
    for k in streams:
        assert not bool(grads[k][:T - TAIL].any()), k
        grads[k] = grads[k][T - TAIL:]
    want, size = (ref.scan(**s, dout=dout, dh_n=dh_n, magnitude=m) for m in (False, True))
    k = 8 * TAIL + 40
    sel.check("y", y[T - TAIL:], want["y"], size["y"], k)
    sel.check("h_n", h, want["h"], size["h"], k)
    for name, grad in grads.items():
        sel.check(name, grad, want[name], size[name], 2 * k + 8)


@pytest.mark.parametrize("n,v,d,dtype", [((1 << 21) + 70, 64, 1024, BF16), (70, (1 << 21) + 1000, 1024, BF16),
                                          (3, 9000011, 16, BF16), ((1 << 21) + 70, 5, 1030, torch.float32),
                                          (30, 4500011, 500, torch.float32),
                                          (30, 2200011, 257, torch.float32)])
def test_loss_beyond_32_bits(dev, n, v, d, dtype):
    """Only the last rows have a gradient, and all tokens but the first and last 500 are masked."""
    rows, kept = min(n, 70), torch.arange(v)
    if v > 1000:
        kept = torch.cat((kept[:500], kept[-500:]))
    x, w, t, _, dloss = xent.inputs(dev, dtype, rows, len(kept), d)
    big_x = _long(dev, n, x).requires_grad_(True)
    bias = torch.full((v,), -math.inf, device=dev)
    bias[kept.to(dev)] = 0.0
    big_w = torch.full((v, d), 7.0, dtype=dtype, device=dev)
    big_w[kept.to(dev)] = w
    big_w.requires_grad_(True)
    big_t = torch.zeros(n, dtype=torch.int64, device=dev)
    big_t[n - rows:] = kept.to(dev)[t]
    loss = prlstm_amd.linear_cross_entropy(big_x, big_w, big_t, bias=bias)
    dl = torch.zeros(n, device=dev)
    dl[n - rows:] = dloss
    dx, dw = torch.autograd.grad(loss, (big_x, big_w), dl)
    want, ref_dl, parts, size = xent.reference(x, w, t, None, dloss)
    shift = (d + 4) * xent.U * size
    xent.within("loss", loss[n - rows:], want,
                2 * shift + 16 * xent.U * (want.abs() + size + math.log(v + 1)) + 2 ** -20)
    _, bound_x, bound_w = xent.bounds(x, w, t, ref_dl, parts, shift, dloss)
    xent.within("dx", dx[n - rows:], ref_dl @ w.double().cpu(), bound_x)
    xent.within("dw", dw[kept.to(dev)], ref_dl.t() @ x.double().cpu(), bound_w)
    assert not bool(dx[:n - rows].any())
    assert v <= 1000 or not bool(dw[500:v - 500].any())


def _calls(dev):
    """(name, the call on a dict of operands, the operands)."""
    r = lambda *s: torch.randn(*s, device=dev)  # noqa: E731
    t = torch.zeros(6, 2, dtype=torch.int64, device=dev)
    return [
        ("conv", lambda o: prlstm_amd.causal_conv(**o)[0],
         dict(x=r(6, 2, 5), weight=r(5, 4), bias=r(5), state=r(2, 3, 5))),
        ("conv_step", lambda o: prlstm_amd.causal_conv_step(**o)[0],
         dict(x=r(2, 5), state=r(2, 3, 5), weight=r(5, 4), bias=r(5))),
        ("scan", lambda o: prlstm_amd.selective_scan(**o)[0],
         dict(x=r(6, 2, 5), delta=r(6, 2, 5), a=-r(5, 3).abs(), b=r(6, 2, 3), c=r(6, 2, 3), d=r(5), z=r(6, 2, 5),
              delta_bias=r(5), h0=r(2, 5, 3))),
        ("scan_step", lambda o: prlstm_amd.selective_scan_step(**o)[0],
         dict(x=r(2, 5), delta=r(2, 5), a=-r(5, 3).abs(), b=r(2, 3), c=r(2, 3), h=r(2, 5, 3), d=r(5), z=r(2, 5),
              delta_bias=r(5))),
        ("loss", lambda o: prlstm_amd.linear_cross_entropy(targets=t, **o),
         dict(x=r(6, 2, 5), weight=r(7, 5), bias=r(7))),
    ]


def test_operands_that_do_not_fit(dev):
    """Every operand of every call: too few dimensions, another size, another device; streams also another type."""
    for name, call, operands in _calls(dev):
        call(operands)
        for k, v in operands.items():
            others = [v[0], torch.cat((v, v), -1), torch.cat((v, v)), v.cpu(), v.double() if k == "x" else v.int()]
            if k in ("delta", "b", "c", "z") or (name, k) in (("conv", "state"), ("conv_step", "state"),
                                                              ("loss", "weight")):
                others.append(v.bfloat16())
            for i, other in enumerate(others):
                if (name, k, i) == ("conv", "x", 2):
                    continue  # more steps
                with pytest.raises(RuntimeError):
                    call({**operands, k: other})
                    pytest.fail(f"{name}: {k} {tuple(other.shape)} {other.dtype} was taken")


def test_forward_mode_is_refused(dev):
    for name, call, operands in _calls(dev):
        for k, v in operands.items():
            with fwad.dual_level(), pytest.raises(NotImplementedError):
                call({**operands, k: fwad.make_dual(v, torch.ones_like(v))})
                pytest.fail(f"{name}: {k}")


def test_derivatives_once(dev):
    for name, call, operands in _calls(dev):
        if name.endswith("step"):
            continue
        x = operands["x"].requires_grad_(True)
        dx, = torch.autograd.grad(call(operands).square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            dx.sum().backward()


def test_gradients_of_any_layout(dev):
    """Expanded and transposed gradients, and outputs that are changed in place before the backward."""
    for name, call, operands in _calls(dev):
        if name.endswith("step"):
            continue
        leaves = {k: v.requires_grad_(True) for k, v in operands.items()}
        y = call(leaves)
        dense = torch.randn_like(y)
        lists = []
        for dy in (torch.ones_like(y), torch.ones((), device=dev).expand_as(y), dense,
                   dense.transpose(0, 1).contiguous().transpose(0, 1)):
            lists.append(torch.autograd.grad(y, list(leaves.values()), dy, retain_graph=True))
        y.mul_(2.0)
        lists.append(torch.autograd.grad(y, list(leaves.values()), dense / 2))  # of y before: dense
        for a, b in ((0, 1), (2, 3), (2, 4)):
            for k, g, w in zip(leaves, lists[a], lists[b]):
                assert torch.equal(g, w), (name, k, a, b)


def test_states_that_overlap(dev):
    """The new state may take the old one's place; a part of it is refused."""
    buf = torch.zeros(4, 3, 8, device=dev)
    x, w = torch.ones(2, 8, device=dev), torch.ones(8, 4, device=dev)
    with pytest.raises(RuntimeError, match="state_out overlaps"):
        prlstm_amd.causal_conv_step(x, buf[:2], w, state_out=buf[1:3])
    _, n = prlstm_amd.causal_conv_step(x, buf[:2], w, state_out=buf[2:])
    assert bool(n[:, 2].eq(1).all()) and not bool(buf[:2].any())
    h = torch.zeros(3, 8, 4, device=dev)
    bc, a = torch.ones(2, 4, device=dev), -torch.ones(8, 4, device=dev)
    with pytest.raises(RuntimeError, match="h_out overlaps"):
        prlstm_amd.selective_scan_step(x, x, a, bc, bc, h[:2], h_out=h[1:])
    _, n = prlstm_amd.selective_scan_step(x, x, a, bc, bc, h[:2], h_out=h[:2])
    assert n.data_ptr() == h.data_ptr() and bool(h[:2].all()) and not bool(h[2].any())


def test_two_graphs(dev):
    """Two graphs of the whole chain, replayed in turn and one behind the other: neither sees the other's
    workspaces."""
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).to(dev)  # noqa: E731
    sizes = ((300, 2, 40, 16, 500), (4200, 1, 72, 10, 300))  # the second scan in segments
    made = []
    for T, B, D, N, V in sizes:
        o = dict(u=r(T, B, D), taps=r(D, 4), delta=r(T, B, D), a=-r(D, N).abs() - 0.1, b=r(T, B, N), c=r(T, B, N),
                 w=r(V, D) * D ** -0.5)
        t = torch.randint(0, V, (T, B), generator=g).to(dev)

        dl = r(T, B)

        def step(o=o, t=t, dl=dl):
            leaves = {k: v.detach().requires_grad_(True) for k, v in o.items()}
            x, _ = prlstm_amd.causal_conv(leaves["u"], leaves["taps"])
            y, _ = prlstm_amd.selective_scan(x, *(leaves[k] for k in ("delta", "a", "b", "c")))
            loss = prlstm_amd.linear_cross_entropy(y.bfloat16(), leaves["w"].bfloat16(), t)
            return loss.detach(), *torch.autograd.grad(loss, list(leaves.values()), dl)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        made.append((graph, out, step))
    for order in ((0, 1), (1, 0), (0, 0, 1)):
        for i in order:
            made[i][0].replay()
        want = [m[2]() for m in made]
        torch.cuda.synchronize()
        for (_, out, _), w in zip(made, want):
            assert all(torch.equal(a, b) for a, b in zip(out, w)), order


def test_two_streams(dev):
    """The whole chain on two streams at a time: neither call sees the other's workspaces."""
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).to(dev)  # noqa: E731
    chains = []
    for T, B, D, N, V, dtype in ((2000, 1, 128, 16, 3000, BF16), (600, 3, 72, 7, 700, torch.float32)):
        o = dict(u=r(T, B, D).to(dtype), taps=r(D, 4), delta=r(T, B, D).to(dtype), a=-r(D, N).abs() - 0.1,
                 b=r(T, B, N).to(dtype), c=r(T, B, N).to(dtype), w=(r(V, D) * D ** -0.5).to(dtype))
        t, dl = torch.randint(0, V, (T, B), generator=g).to(dev), r(T, B)

        def chain(o=o, t=t, dl=dl):
            leaves = {k: v.detach().requires_grad_(True) for k, v in o.items()}
            x, _ = prlstm_amd.causal_conv(leaves["u"], leaves["taps"])
            y, _ = prlstm_amd.selective_scan(x, *(leaves[k] for k in ("delta", "a", "b", "c")))
            loss = prlstm_amd.linear_cross_entropy(y, leaves["w"], t)
            return loss.detach(), *torch.autograd.grad(loss, list(leaves.values()), dl)

        chains.append(chain)
    want = [chain() for chain in chains]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in chains]
    for _ in range(4):
        got = []
        for s, chain in zip(streams, chains):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(chain())
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
