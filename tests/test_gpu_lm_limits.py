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


def test_embedding_gradient_of_more_rows_than_a_grid_has_in_y(dev):
    """33.6 million tokens: 131072 classes."""
    V, D = (1 << 25) + 40000, 1
    ids = torch.tensor([0, V - 1, 1 << 25, 5, V - 1, 65536 * 511, -1], device=dev)
    # one token of more than a chunk of positions, in a class above 65535
    ids = torch.cat((ids, torch.full((40,), 100000, device=dev)))
    w = torch.zeros(V, D, dtype=torch.bfloat16, device=dev, requires_grad=True)
    dout = torch.arange(1, len(ids) + 1, device=dev, dtype=torch.bfloat16)[:, None]
    dw, = torch.autograd.grad(prlstm_amd.embedding(ids, w), w, dout)
    want = torch.zeros(V, device=dev).index_add_(0, ids.clamp_min(0), dout[:, 0].float() * (ids >= 0))
    assert torch.equal(dw[:, 0].float(), want.bfloat16().float())


def test_embedding_of_more_rows_than_a_launch_has(dev):
    """257 columns are 33 vectors, so a workgroup of 256 threads has 16 rows, and 2^28 rows are two
    launches."""
    N, D = (1 << 28) + 100, 257
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 170e9:
        pytest.skip("needs 138 GB")
    ids = torch.zeros(N, dtype=torch.int32, device=dev)
    ids[-1], ids[-50], ids[5] = 2, -1, 1
    w = torch.arange(3 * D, device=dev).reshape(3, D).remainder(256).bfloat16()
    out = prlstm_amd.embedding(ids, w)
    assert torch.equal(out[-1], w[2]) and torch.equal(out[5], w[1]) and not bool(out[-50].any())
    out[-1] = out[5] = out[-50] = w[0]
    for rows in out.split(1 << 24):
        assert bool((rows == w[0]).all())
    del out, rows
    torch.cuda.empty_cache()


@pytest.mark.parametrize("T", [1, 3])
def test_gated_recurrence_of_many_channels(dev, T):
    """More channels than a square weight of 2^31 elements would have."""
    B, H = 2, 40001
    g = torch.Generator().manual_seed(T)
    zv = torch.randn(T, B, 2 * H, generator=g).to(dev).requires_grad_(True)
    out, h_n = prlstm_amd.gated_recurrence(zv)
    dz, = torch.autograd.grad(h_n.sum(), zv)
    for lo in (0, H // 2, H - 7):
        part = torch.cat((zv.detach()[..., lo:lo + 7], zv.detach()[..., H + lo:H + lo + 7]), -1).requires_grad_(True)
        o, h = prlstm_amd.gated_recurrence(part)
        d, = torch.autograd.grad(h.sum(), part)
        assert torch.equal(out[..., lo:lo + 7], o) and torch.equal(h_n[:, lo:lo + 7], h)
        assert torch.equal(torch.cat((dz[..., lo:lo + 7], dz[..., H + lo:H + lo + 7]), -1), d)


def test_sizes_beyond_32_bits_are_refused(dev):
    """Sizes that a 32-bit argument would take for others: 2^32 + 5 is not 5."""
    n = (1 << 32) + 5
    one = torch.zeros(1, 1, device=dev)
    ids = torch.tensor([7], device=dev)
    for call in (lambda: prlstm_amd.embedding(ids, one.expand(n, 1)),
                 lambda: prlstm_amd.embedding(ids[:0], one.expand(3, n)),
                 lambda: prlstm_amd.gated_recurrence(one[None].expand(n, 0, 2)),
                 lambda: prlstm_amd.gated_recurrence(one[None].expand(0, n, 2)),
                 lambda: prlstm_amd.gated_recurrence_step(one.expand(0, 2 * n), None),
                 lambda: prlstm_amd.token_logprobs(one.expand(0, n))):
        with pytest.raises(RuntimeError, match="2\\^31"):
            call()
    prlstm_amd.check_errors(dev)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_tokens_of_a_large_entropy_gradient(dev, dtype):
    """A masked token has no gradient, whatever the entropy's is; the others' are finite."""
    x = torch.tensor([[0.0, -float("inf"), 1.0, -500.0, 2.0]]).to(dtype)
    want = torch.zeros(1, 5, dtype=torch.float64)
    y = x.double()[:, [0, 2, 4]].requires_grad_(True)
    p = torch.softmax(y, 1)
    want[:, [0, 2, 4]] = torch.autograd.grad(-(p * torch.log(p)).sum(), y)[0]
    for dent in (1.0, 1e9, 1e30):
        xd = x.to(dev).requires_grad_(True)
        dx, = torch.autograd.grad(prlstm_amd.token_logprobs(xd).entropy, xd, torch.tensor([dent], device=dev))
        got = dx.double().cpu() / dent
        # fp32 statistics of order 1 and one rounding to the type
        u = 2.0 ** -8 if dtype is torch.bfloat16 else 2.0 ** -24
        assert bool(((got - want).abs() <= 1.01 * u * want.abs() + 64 * 2.0 ** -24).all()), (dent, got, want)
        assert float(got[0, 1]) == 0.0


def test_masked_tokens_of_an_infinite_gradient(dev):
    inf = float("inf")
    x = torch.tensor([[0.0, -inf, 1.0, -inf, 2.0]], device=dev, requires_grad=True)
    r = prlstm_amd.token_logprobs(x, torch.tensor([2], device=dev), top=1)
    for out in (r.logp, r.entropy, r.top_logp):
        for g in (inf, float("nan")):
            dx, = torch.autograd.grad(out, x, torch.full_like(out, g), retain_graph=True)
            assert dx[0, 1] == 0.0 and dx[0, 3] == 0.0 and not bool(torch.isfinite(dx[0, 4]))
