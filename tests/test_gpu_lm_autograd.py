"""What the language-model operators (prlstm_amd.lm) refuse or notice as torch's own operations do."""

import pytest
import torch
from torch.autograd import forward_ad

import prlstm_amd

pytestmark = pytest.mark.gpu


def test_forward_mode_derivatives_are_refused(dev):
    """The operators have no forward-mode derivative: a tangent is an error, not a derivative of zero."""
    ids = torch.zeros(3, dtype=torch.int64, device=dev)
    zeros = lambda *s: torch.zeros(*s, device=dev)  # noqa: E731
    with forward_ad.dual_level():
        dual = lambda *s: forward_ad.make_dual(zeros(*s), torch.ones(*s, device=dev))  # noqa: E731
        for call in (lambda: prlstm_amd.embedding(ids, dual(4, 6)),
                     lambda: prlstm_amd.gated_recurrence(dual(5, 2, 8)),
                     lambda: prlstm_amd.gated_recurrence(zeros(5, 2, 8), dual(2, 4)),
                     lambda: prlstm_amd.gated_recurrence_step(dual(2, 8), zeros(2, 4)),
                     lambda: prlstm_amd.gated_recurrence_step(zeros(2, 8), dual(2, 4)),
                     lambda: prlstm_amd.token_logprobs(dual(3, 5), ids)):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
                    call()
        # without a tangent the calls are as ever
        assert prlstm_amd.embedding(ids, zeros(4, 6)).shape == (3, 6)
        assert prlstm_amd.gated_recurrence(zeros(5, 2, 8))[0].shape == (5, 2, 4)
        assert prlstm_amd.gated_recurrence_step(zeros(2, 8), zeros(2, 4))[0].shape == (2, 4)
        assert prlstm_amd.token_logprobs(zeros(3, 5), ids).logp.shape == (3,)


def test_tangents_of_incoming_gradients_are_refused(dev):
    ids = torch.zeros(3, dtype=torch.int64, device=dev)
    w = torch.zeros(4, 6, device=dev, requires_grad=True)
    zv = torch.zeros(5, 2, 8, device=dev, requires_grad=True)
    x = torch.zeros(3, 5, device=dev, requires_grad=True)
    for out, arg in ((prlstm_amd.embedding(ids, w), w), (prlstm_amd.gated_recurrence(zv)[0], zv),
                     (prlstm_amd.gated_recurrence(zv)[1], zv), (prlstm_amd.token_logprobs(x, ids).logp, x),
                     (prlstm_amd.token_logprobs(x).entropy, x)):
        with forward_ad.dual_level():
            g = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(NotImplementedError):
                torch.autograd.grad(out, arg, g)


def test_scale_that_is_a_tensor(dev):
    """The scale has no gradient and is not fetched from the device: a tensor that asks for either
    is refused; a number of another kind is one."""
    ids, w = torch.zeros(3, dtype=torch.int64, device=dev), torch.ones(4, 6, device=dev)
    for scale in (torch.tensor(2.0, requires_grad=True), torch.tensor(2.0, device=dev, requires_grad=True),
                  torch.tensor(2.0, device=dev)):
        with pytest.raises(RuntimeError, match="scale must be a number"):
            prlstm_amd.embedding(ids, w, scale)
    for scale in (2, 2.0, torch.tensor(2.0), torch.tensor(2)):
        assert torch.equal(prlstm_amd.embedding(ids, w, scale), torch.full((3, 6), 2.0, device=dev))
    with torch.no_grad():
        out = prlstm_amd.embedding(ids, w, torch.nn.Parameter(torch.tensor(2.0)))
        assert torch.equal(out, torch.full((3, 6), 2.0, device=dev))
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        prlstm_amd.embedding(ids, w, forward_ad.make_dual(torch.tensor(2.0), torch.tensor(1.0)))


@pytest.mark.parametrize("order", ["time", "batch"])
def test_output_changed_in_place(dev, order):
    """A residual added to the output in place, in either order of time and batch."""
    g = torch.Generator().manual_seed(0)
    zv = torch.randn(6, 3, 10, generator=g).to(dev)
    if order == "batch":
        zv = zv.transpose(0, 1).contiguous().transpose(0, 1)
    dout = torch.randn(6, 3, 5, generator=g).to(dev)
    a, b = (zv.clone(memory_format=torch.preserve_format).requires_grad_(True) for _ in range(2))
    out, _ = prlstm_amd.gated_recurrence(a)
    assert (out.stride(0) > out.stride(1)) == (order == "time")
    out += a[..., 5:]
    want = prlstm_amd.gated_recurrence(b)[0] + b[..., 5:]
    assert torch.equal(out, want)
    assert torch.equal(*(torch.autograd.grad(o, x, dout)[0] for o, x in ((out, a), (want, b))))


def test_state_updated_in_place_is_noticed(dev):
    """A state that a backward pass needs and a step has overwritten is an error there."""
    w = torch.ones(2, 4, device=dev, requires_grad=True)
    h = torch.ones(2, 4, device=dev)
    y = (w * h).sum()
    version = h._version
    prlstm_amd.gated_recurrence_step(torch.zeros(2, 8, device=dev), h, h_out=h)
    assert h._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():  # whose tensors have no version
        h = torch.zeros(2, 4, device=dev)
        _, h2 = prlstm_amd.gated_recurrence_step(torch.zeros(2, 8, device=dev), h, h_out=h)
        assert h2 is h
