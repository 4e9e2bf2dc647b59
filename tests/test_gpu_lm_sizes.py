"""Sizes of the language-model operators (prlstm_amd.lm) that take other launches or branches than
small calls: large vocabularies and batches of the embedding's gradient, many rows and int32 tokens of
the log probabilities, and long recurrences of many channels.  Bounds as in test_gpu_lm."""

import pytest
import torch

import prlstm_amd
from test_gpu_lm import HALF, _check_gated, _gated_plain, _logprob_plain, _order, _within, u

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,V,D", [(5000, 200003, 40), (270001, 200003, 9), (140000, 300, 16), (9000, 600011, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_embedding_gradient_of_large_vocabularies_and_batches(dev, N, V, D, dtype):
    """More than 256 classes (V above 131072), chunks of 64 positions and more (N above 131072), with
    frequent tokens in classes on both sides of 256."""
    print(f"embedding {N} {V} {D} {dtype}", flush=True)
    g = torch.Generator().manual_seed(N + V)
    ids = (torch.rand(N, generator=g) ** 3 * V).long().clamp_max(V - 1)
    often = torch.rand(N, generator=g)
    ids[often < 0.3] = min(V - 1, 512 * 7 + 300)
    ids[often > 0.9] = 5
    ids[torch.rand(N, generator=g) < 0.05] = -1
    dout = torch.randn(N, D, generator=g).to(dtype)
    there = ids >= 0
    at, d2 = ids[there], dout[there].double()
    want = torch.zeros(V, D, dtype=torch.float64).index_add_(0, at, d2)
    mag = torch.zeros(V, D, dtype=torch.float64).index_add_(0, at, d2.abs())
    bound = (torch.bincount(at, minlength=V)[:, None].double() + 2) * u * mag + HALF[dtype] * 1.01 * want.abs() + 1e-38
    w = torch.randn(V, D, generator=g).to(dtype)
    first = None
    for ids_dtype in (torch.int64, torch.int32):
        wd = w.to(dev).requires_grad_(True)
        out = prlstm_amd.embedding(ids.to(dev, ids_dtype), wd)
        assert torch.equal(out.detach().cpu(), torch.where(there[:, None], w[ids.clamp_min(0)], torch.zeros(()).to(dtype)))
        dw, = torch.autograd.grad(out, wd, dout.to(dev))
        _within("dweight", dw, want, bound)
        first = dw if first is None else first
        assert torch.equal(dw, first)


@pytest.mark.parametrize("N,V,top", [(7, 4099, 3), (65600, 40, 2), (131500, 17, 0), (3, 60000, 8)])
def test_logprobs_of_int32_tokens_and_many_rows(dev, N, V, top):
    """int32 tokens give what int64 ones do, in value and gradient; more than 65535 rows are several
    launches of the backward, checked on both sides of each cut."""
    print(f"logprobs {N} {V} {top}", flush=True)
    g = torch.Generator().manual_seed(N + V)
    x = torch.randn(N, V, generator=g) * 3
    tokens = torch.randint(0, V, (N,), generator=g)
    tokens[torch.rand(N, generator=g) < 0.1] = -1
    dlogp, dent, dtop = torch.randn(N, generator=g), torch.randn(N, generator=g), torch.randn(N, top, generator=g)
    rows = torch.tensor(sorted({r for c in (0, 65535, 131070, N) for r in range(c - 3, c + 4) if 0 <= r < N}))
    want = _logprob_plain(x[rows], tokens[rows], top, dlogp[rows], dent[rows], dtop[rows])
    whole = torch.log_softmax(x.double(), 1)
    got = []
    for dtype in (torch.int64, torch.int32):
        xd = x.to(dev).requires_grad_(True)
        r = prlstm_amd.token_logprobs(xd, tokens.to(dev, dtype), top=top)
        outs, gs = [r.logp, r.entropy], [dlogp.to(dev), dent.to(dev)]
        if top:
            outs, gs = outs + [r.top_logp], gs + [dtop.to(dev)]
            assert torch.equal(r.top_ids.cpu(), _order(x)[:, :top])
            _within("top_logp", r.top_logp[rows], *want["top_logp"])
        dx, = torch.autograd.grad(outs, xd, gs)
        _within("logp", r.logp[rows], *want["logp"])
        _within("entropy", r.entropy[rows], *want["entropy"])
        _within("dlogits", dx[rows], want["dlogits"][0], want["dlogits"][1] + 1.01 * u * want["dlogits"][0].abs() + 1e-38)
        # every row: the value, and a gradient that sums to nothing (p sums to 1; the entropy's to 0)
        every = torch.where(tokens >= 0, whole.gather(1, tokens.clamp_min(0)[:, None])[:, 0], 0.0)
        assert float((r.logp.detach().cpu() - every).abs().max()) < 1e-4
        assert float(dx.double().sum(1).abs().max()) < 1e-4
        got.append((r.logp.detach(), r.entropy.detach(), dx))
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("T,B,H,dtype", [(150, 35, 1000, torch.bfloat16), (300, 33, 513, torch.float32),
                                         (129, 20, 1024, torch.float16)])
def test_gated_recurrence_of_many_workgroups(dev, T, B, H, dtype):
    """512 workgroups over the channels and more take four waves of several chunks, 257 to 511 eight."""
    print(f"gated {T} {B} {H} {dtype}", flush=True)
    g = torch.Generator().manual_seed(T)
    zv = torch.randn(T, B, 2 * H, generator=g)
    zv[..., :H] += 2.0
    zv = zv.to(dtype)
    h0, dout, dh_n = torch.randn(B, H, generator=g), torch.randn(T, B, H, generator=g).to(dtype), torch.randn(B, H, generator=g)
    reset = torch.rand(T, B, generator=g) < 0.02
    for r in (None, reset):
        want = _gated_plain(zv, h0, r, dout, dh_n)
        zd, hd = zv.to(dev).requires_grad_(True), h0.to(dev).requires_grad_(True)
        out, h_n = prlstm_amd.gated_recurrence(zd, hd, None if r is None else r.to(dev))
        dz, dh = torch.autograd.grad((out, h_n), (zd, hd), (dout.to(dev), dh_n.to(dev)))
        for k, v in (("out", out), ("h_n", h_n), ("dzv", dz), ("dh0", dh)):
            _check_gated(k, v, want[k], dtype)
