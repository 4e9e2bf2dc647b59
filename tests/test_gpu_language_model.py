"""The example language model: its sequence form, its step form and its training agree."""

import pytest
import torch

from prlstm_amd import language_model
from prlstm_amd.lm import token_logprobs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("parallel", [True, False])
def test_steps_follow_the_sequence(dev, parallel):
    """Log probabilities one token at a time equal those of the whole sequence, and of its halves
    with the state carried over.  Both compute the same sums in fp32 in other orders: 1e-4 of
    activations of order 10 over 20 steps."""
    torch.manual_seed(0)
    m = language_model.LanguageModel(50, 32, parallel=parallel).to(dev)
    ids = torch.randint(0, 50, (20, 3), device=dev)
    ids[5, 1] = -1  # a padded position
    with torch.no_grad():
        logits, (lstm, gated) = m(ids)
        a, state = m(ids[:7])
        b, _ = m(ids[7:], state)
    assert torch.allclose(torch.cat((a, b)), logits, rtol=1e-4, atol=1e-4)
    state = m.state(3)
    whole = token_logprobs(logits, top=5)
    for t in range(20):
        r = m.step(ids[t], state, top=5)
        assert torch.allclose(r.entropy, whole.entropy[t], rtol=1e-3, atol=1e-3), t
        assert torch.allclose(r.top_logp, whole.top_logp[t], rtol=1e-3, atol=1e-3), t
    for x, y in zip((*state[0], *state[1]), (*lstm, *gated)):
        assert torch.allclose(x, y, rtol=1e-3, atol=1e-3)


def test_documents_in_one_sequence(dev):
    """With a reset between two documents the gated layers see the second one alone (the loss of a
    model without its LSTM's state is the same as of the documents apart)."""
    torch.manual_seed(0)
    m = language_model.LanguageModel(50, 32).to(dev)
    with torch.no_grad():  # the LSTM forgets everything: its forget gate shut, the scan's floor 1e-6
        m.lstm.bias_ih_l0[32:64] = -200.0
    ids = torch.randint(0, 50, (24, 2), device=dev)
    reset = torch.zeros(24, 2, dtype=torch.bool, device=dev)
    reset[10] = True
    with torch.no_grad():
        both, _ = m(ids, reset=reset)
        second, _ = m(ids[10:])
    assert torch.allclose(both[10:], second, rtol=1e-3, atol=1e-3)


def test_it_learns(dev):
    first, last, share = language_model.main()
    assert last < 0.5 * first and share > 0.8, (first, last, share)


def test_bf16_training_step(dev):
    torch.manual_seed(0)
    m = language_model.LanguageModel(300, 64).to(dev, torch.bfloat16)
    ids = torch.randint(0, 300, (40, 4), device=dev)
    targets = torch.roll(ids, -1, 0)
    targets[-1] = -1
    loss = m.loss(ids, targets)
    loss.backward()
    assert all(p.grad is None or bool(torch.isfinite(p.grad).all()) for p in m.parameters())
    assert m.weight.grad.dtype == torch.bfloat16 and abs(loss.item() - torch.log(torch.tensor(300.0)).item()) < 2.0
