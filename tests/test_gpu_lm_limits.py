"""The language-model operators (prlstm_amd.lm) at the ends of the sizes that they take."""

import pytest
import torch

import prlstm_amd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,V", [((1 << 26) + 300, 2), ((1 << 24) + 300, 2100)])
def test_logprobs_of_more_rows_than_a_launch_has(dev, N, V):
    """Rows of one wave and of a workgroup; each is one of few, so the results are too."""
    two = torch.zeros(2, V, dtype=torch.bfloat16, device=dev)
    two[0, 0], two[1, 1] = 1.0, 3.0
    x = two.repeat((N + 1) // 2, 1)[:N] if V == 2 else two[:1].expand(N, V)
    tokens = torch.zeros(N, dtype=torch.int32, device=dev)
    tokens[-1] = 1
    r = prlstm_amd.token_logprobs(x, tokens, top=1)
    few = prlstm_amd.token_logprobs(two, torch.zeros(2, dtype=torch.int32, device=dev), top=1)
    last = prlstm_amd.token_logprobs(x[-1:], torch.ones(1, dtype=torch.int32, device=dev))
    k = len(two) if V == 2 else 1
    at = torch.arange(N - 1, device=dev) % k
    assert torch.equal(r.logp[:-1], few.logp[at]) and torch.equal(r.logp[-1:], last.logp)
    del at
    at = torch.arange(N, device=dev) % k
    assert torch.equal(r.entropy, few.entropy[at])
    assert torch.equal(r.top_ids[:, 0], few.top_ids[at, 0]) and torch.equal(r.top_logp[:, 0], few.top_logp[at, 0])
