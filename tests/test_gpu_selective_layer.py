"""The selective operators and the loss without logits together, as the example language model uses them."""

import pytest
import torch

from prlstm_amd import language_model
from prlstm_amd.lm import token_logprobs

pytestmark = pytest.mark.gpu

# A gradient passes four products of at most 80 terms, a convolution and a scan of 37 steps (at most 8 * 37 + 40
# roundings), twice: below 1100 roundings of 2^-24, of terms whose sizes are at most 10 times those of their sums.
CLOSE = 11000 * 2.0 ** -24


def plain_layer(p, x, reset):
    """SelectiveLayer over x [T, B, width] with parameters p, step by step."""
    states, taps = p["log_a"].shape[1], p["taps"].shape[1]
    rank = p["choose.weight"].shape[0] - 2 * states
    u, z = (torch.nn.functional.layer_norm(x, x.shape[-1:], p["norm.weight"], p["norm.bias"])
            @ p["enter.weight"].T).chunk(2, -1)
    window = [torch.zeros_like(u[0])] * taps
    h = x.new_zeros(*u.shape[1:], states)
    a, out = -torch.exp(p["log_a"]), []
    for t in range(len(x)):
        keep = ~reset[t][:, None]
        window = [torch.where(keep, w, torch.zeros_like(w)) for w in window[1:]] + [u[t]]
        v = torch.nn.functional.silu(p["taps_bias"] + sum(p["taps"][:, k] * window[k] for k in range(taps)))
        delta, b, c = (v @ p["choose.weight"].T).split((rank, states, states), -1)
        dt = torch.nn.functional.softplus(delta @ p["widen.weight"].T + p["delta_bias"])[..., None]
        h = torch.where(keep[..., None], h, torch.zeros_like(h))
        h = torch.exp(dt * a) * h + dt * v[..., None] * b[:, None]
        y = (h * c[:, None]).sum(-1) + p["skip"] * v
        out.append(x[t] + (y * torch.nn.functional.silu(z[t])) @ p["leave.weight"].T)
    return torch.stack(out)


def test_layer_against_64_bits(dev):
    """The output, every parameter's gradient and the input's, and their sum along a random direction
    against a difference."""
    torch.manual_seed(0)
    layer = language_model.SelectiveLayer(20, 5)
    x, dy = torch.randn(37, 3, 20), torch.randn(37, 3, 20).double()
    reset = torch.rand(37, 3) < 0.1
    p = {k: v.detach().double().requires_grad_(True) for k, v in layer.named_parameters()}
    x64 = x.double().requires_grad_(True)
    y64 = plain_layer(p, x64, reset)
    want = torch.autograd.grad(y64, [*p.values(), x64], dy)
    layer.to(dev)
    xd = x.to(dev).requires_grad_(True)
    y, _ = layer(xd, None, reset.to(dev))
    got = torch.autograd.grad(y, [*layer.parameters(), xd], dy.float().to(dev))
    names = ["y", *p, "x"]
    got = [g.detach().double().cpu() for g in (y, *got)]
    for name, g, w in zip(names, got, (y64, *want)):
        assert (g - w).norm() <= CLOSE * w.norm(), (name, float((g - w).norm() / w.norm()))
    way = [torch.randn_like(v) for v in (*p.values(), x64)]
    with torch.no_grad():
        ends = []
        for h in (1e-6, -1e-6):
            moved = [v + h * d for v, d in zip((*p.values(), x64), way)]
            ends.append((plain_layer(dict(zip(p, moved)), moved[-1], reset) * dy).sum())
    slope = (ends[0] - ends[1]) / 2e-6
    along = sum((g * d).sum() for g, d in zip(got[1:], way))
    size = sum(g.norm() * d.norm() for g, d in zip(got[1:], way))
    # the difference itself: a third derivative times 1e-12, and 2^-52 of sums of 2220 terms over 1e-6
    assert abs(along - slope) <= (CLOSE + 1e-6) * size


def test_steps_follow_the_sequence(dev):
    """As the sequence form, one token at a time and in two halves; the same sums in fp32 in other orders:
    1e-4 of activations of order 10 over 20 steps."""
    torch.manual_seed(0)
    m = language_model.LanguageModel(50, 32, layers=1, selective=2, states=6).to(dev)
    ids = torch.randint(0, 50, (20, 3), device=dev)
    ids[5, 1] = -1
    with torch.no_grad():
        logits, (_, last) = m(ids)
        a, state = m(ids[:7])
        b, _ = m(ids[7:], state)
    assert torch.allclose(torch.cat((a, b)), logits, rtol=1e-4, atol=1e-4)
    state = m.state(3)
    whole = token_logprobs(logits, top=5)
    for t in range(20):
        r = m.step(ids[t], state, top=5)
        assert torch.allclose(r.entropy, whole.entropy[t], rtol=1e-3, atol=1e-3), t
        assert torch.allclose(r.top_logp, whole.top_logp[t], rtol=1e-3, atol=1e-3), t
    for got, want in zip(state[1][1:], last[1:]):
        for x, y in zip(got, want):
            assert torch.allclose(x, y, rtol=1e-3, atol=1e-3)


def test_reset_cuts_the_selective_layers(dev):
    torch.manual_seed(0)
    m = language_model.LanguageModel(50, 32, layers=0, selective=2).to(dev)
    ids = torch.randint(0, 50, (24, 2), device=dev)
    reset = torch.zeros(24, 2, dtype=torch.bool, device=dev)
    reset[10, 0] = True
    logits, _ = m(ids, reset=reset)
    alone, _ = m(ids[10:, :1])
    assert torch.allclose(logits[10:, 0], alone[:, 0], rtol=1e-4, atol=1e-4)
    logits[10:, 0].square().sum().backward()
    unseen = torch.ones(50, dtype=torch.bool, device=dev)
    unseen[ids[10:, 0]] = False
    assert float(m.weight.grad[unseen].abs().max()) == 0.0


@pytest.mark.parametrize("selective", [0, 1])
def test_loss_without_logits(dev, selective):
    """The loss and its gradients are those of the loss with logits, of the same sums in other orders."""
    torch.manual_seed(0)
    m = language_model.LanguageModel(300, 48, selective=selective).to(dev)
    ids = torch.randint(0, 300, (37, 3), device=dev)
    targets = torch.roll(ids, -1, 0)
    targets[-1] = -1
    both = []
    for keep in (True, False):
        loss = m.loss(ids, targets, keep_logits=keep)
        grads = torch.autograd.grad(loss, list(m.parameters()), allow_unused=True)
        both.append((loss, grads))
    (a, ga), (b, gb) = both
    assert abs(a.item() - b.item()) <= CLOSE * a.item()
    for (name, _), x, y in zip(m.named_parameters(), ga, gb):
        assert (x is None) == (y is None), name
        if x is not None:
            assert (x - y).norm() <= CLOSE * x.norm(), name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_training_step_in_16_bits(dev, dtype):
    torch.manual_seed(0)
    m = language_model.LanguageModel(300, 64, selective=1).to(dev, dtype)
    ids = torch.randint(0, 300, (40, 4), device=dev)
    targets = torch.roll(ids, -1, 0)
    targets[-1] = -1
    loss = m.loss(ids, targets, keep_logits=False)
    loss.backward()
    assert loss.dtype is torch.float32
    for name, p in m.named_parameters():
        assert p.grad is None or (p.grad.dtype is dtype and bool(torch.isfinite(p.grad).all())), name
    state = m.state(4)
    assert bool(torch.isfinite(m.step(ids[0], state).entropy).all())
