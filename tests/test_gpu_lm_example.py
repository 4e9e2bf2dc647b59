"""Documents packed into one sequence of the example language model."""

import pytest
import torch

from prlstm_amd import language_model

pytestmark = pytest.mark.gpu


def test_reset_cuts_every_layers_state(dev):
    """The second of two documents in one sequence is what it is alone, rows cut at different steps,
    and its loss has no gradient in the first."""
    torch.manual_seed(0)
    for parallel in (True, False):
        m = language_model.LanguageModel(50, 32, parallel=parallel).to(dev)
        ids = torch.randint(0, 50, (24, 3), device=dev)
        reset = torch.zeros(24, 3, dtype=torch.bool, device=dev)
        reset[10, 0] = reset[17, 1] = reset[0, 2] = True
        logits, state = m(ids, reset=reset)
        for row, cut in ((0, 10), (1, 17), (2, 0)):
            alone, (lstm, gated) = m(ids[cut:, row:row + 1])
            # the same sums in fp32 in other orders over 24 steps
            assert torch.allclose(logits[cut:, row], alone[:, 0], rtol=1e-4, atol=1e-4), (parallel, row)
            for a, b in zip((*state[0], *state[1]), (*lstm, *gated)):
                assert torch.allclose(a[row], b[0], rtol=1e-4, atol=1e-4)
        m.weight.grad = None
        logits[10:, 0].square().sum().backward()
        unseen = torch.ones(50, dtype=torch.bool, device=dev)
        unseen[ids[10:, 0]] = False
        assert float(m.weight.grad[unseen].abs().max()) == 0.0


def test_reset_of_nothing_changes_nothing(dev):
    torch.manual_seed(0)
    m = language_model.LanguageModel(50, 32).to(dev)
    ids = torch.randint(0, 50, (12, 3), device=dev)
    with torch.no_grad():
        assert torch.equal(m(ids)[0], m(ids, reset=torch.zeros(12, 3, dtype=torch.bool, device=dev))[0])
