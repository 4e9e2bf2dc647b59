"""The language-model operators (prlstm_amd.lm) against plain 64-bit evaluations on the CPU.

Tolerances are bounds, worked out from the operations: u = 2^-24 is half a unit in the last place of
fp32 (every sum, state and statistic is fp32), U that of the tensors' type (each output is rounded to
it once).  A sum of n terms in any order is within n u of the sum of the magnitudes; the gates, their
exponentials and reciprocals are within 8 u of their values.
"""

import math
import zlib

import pytest
import torch

import prlstm_amd
from prlstm_amd import _lib
from prlstm_amd import lm

pytestmark = pytest.mark.gpu

u = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: u}
TINY = {torch.bfloat16: 1e-38, torch.float16: 2.0 ** -25, torch.float32: 1e-38}  # of the smallest numbers
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _gen(*key):
    return torch.Generator().manual_seed(zlib.crc32(repr(key).encode()))


def _within(name, got, want, bound):
    """Every element within its bound; infinities and NaN in the same places."""
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    fine = torch.isfinite(want)
    same = torch.where(torch.isnan(want), torch.isnan(got), got == want)
    assert bool(same[~fine].all()), f"{name}: infinities or NaN differ"
    err = (got - want).abs()[fine]
    bound = (torch.as_tensor(bound, dtype=torch.float64).expand_as(want))[fine]
    assert bool(torch.isfinite(got[fine]).all()), f"{name}: not finite"
    bad = err > bound
    assert not bool(bad.any()), f"{name}: {int(bad.sum())} of {bad.numel()} outside, worst {(err / bound).max():.3g}x"


# ---- embedding -----------------------------------------------------------------------------

EMBED = [  # ids' shape, V, D
    ((1,), 1, 1), ((0,), 5, 4), ((3, 0), 5, 4), ((8,), 64, 512), ((5, 7), 10, 33), ((700,), 1003, 65), ((1,), 70001, 8),
    ((2049,), 3, 128), ((300,), 40000, 6), ((4, 250), 129, 650), ((3000,), 2, 257), ((70,), 50, 2050),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,V,D", EMBED)
def test_embedding(dev, shape, V, D, dtype):
    print(f"embedding {shape} {V} {D} {dtype}", flush=True)
    g = _gen("embed", shape, V, D)
    ids = (torch.rand(shape, generator=g) ** 3 * V).long().clamp_max(V - 1)  # a few tokens are frequent
    ids[torch.rand(shape, generator=g) < 0.1] = -1
    w = torch.randn(V, D, generator=g).to(dtype)
    dout = torch.randn(*shape, D, generator=g).to(dtype)
    scale, padding = 1.7, (V // 2 if V > 2 else None)
    there = (ids >= 0)[..., None]
    rows = w[ids.clamp_min(0)].float() * torch.tensor(scale)
    want = torch.where(there, rows, torch.zeros(())).to(dtype)
    keep = (ids >= 0).reshape(-1) & (ids.reshape(-1) != (-1 if padding is None else padding))
    at, d2 = ids.reshape(-1)[keep], dout.reshape(-1, D)[keep].double()
    s32 = float(torch.tensor(scale))
    dw = torch.zeros(V, D, dtype=torch.float64).index_add_(0, at, d2) * s32
    mag = torch.zeros(V, D, dtype=torch.float64).index_add_(0, at, d2.abs()) * s32
    count = torch.bincount(at, minlength=V)[:, None].double()
    first = None
    for ids_dtype in (torch.int64, torch.int32):
        i = ids.to(dev, ids_dtype)
        wd = w.to(dev).requires_grad_(True)
        out = prlstm_amd.embedding(i, wd, scale, padding_idx=padding)
        assert out.dtype == dtype and torch.equal(out.detach().cpu(), want)
        got, = torch.autograd.grad(out, wd, dout.to(dev))
        assert got.dtype == dtype
        _within("dweight", got, dw, (count + 2) * u * mag + HALF[dtype] * dw.abs() * 1.01 + TINY[dtype])
        first = got if first is None else first
        assert torch.equal(got, first)  # the sums' order is fixed
        with torch.no_grad():
            assert torch.equal(prlstm_amd.embedding(i, wd, scale), out)


def test_embedding_frequent_token(dev):
    """One token in nearly every position: a long row is summed in parts."""
    g = _gen("frequent")
    N, V, D = 20011, 50, 70
    ids = torch.where(torch.rand(N, generator=g) < 0.9, torch.full((N,), 17), torch.randint(0, V, (N,), generator=g))
    dout = torch.randn(N, D, generator=g)
    w = torch.zeros(V, D, device=dev, requires_grad=True)
    dw, = torch.autograd.grad(prlstm_amd.embedding(ids.to(dev), w), w, dout.to(dev))
    want = torch.zeros(V, D, dtype=torch.float64).index_add_(0, ids, dout.double())
    mag = torch.zeros(V, D, dtype=torch.float64).index_add_(0, ids, dout.double().abs())
    _within("dweight", dw, want, torch.bincount(ids, minlength=V)[:, None].double() * u * mag + u)


@pytest.mark.parametrize("kind", ["one", "few", "half"])
def test_embedding_many_positions_of_few_tokens(dev, kind):
    """More positions of a class than a workgroup lists: one token, a few, and half of them one."""
    g = _gen("many", kind)
    N, V, D = 40003, 600, 24
    ids = torch.randint(0, V, (N,), generator=g)
    if kind == "one":
        ids[:] = 256
    elif kind == "few":
        ids = ids % 2 * 256 + 5
    else:
        ids[torch.rand(N, generator=g) < 0.5] = 599
    dout = torch.randn(N, D, generator=g)
    want = torch.zeros(V, D, dtype=torch.float64).index_add_(0, ids, dout.double())
    mag = torch.zeros(V, D, dtype=torch.float64).index_add_(0, ids, dout.double().abs())
    bound = (torch.bincount(ids, minlength=V)[:, None].double() + 2) * u * mag + 1e-36
    for ids_dtype in (torch.int64, torch.int32):
        w = torch.zeros(V, D, device=dev, requires_grad=True)
        out = prlstm_amd.embedding(ids.to(dev, ids_dtype), w)
        dw, = torch.autograd.grad(out, w, dout.to(dev))
        _within("dweight", dw, want, bound)


def test_embedding_strides_and_broadcast_gradient(dev):
    g = _gen("strides")
    ids = torch.randint(0, 40, (6, 9), generator=g)
    base = torch.randn(40, 50, generator=g)
    w = base.to(dev)[:, 3:36].requires_grad_(True)  # rows of a wider table, not 16-byte aligned
    out = prlstm_amd.embedding(ids.to(dev).t(), w)  # ids in another order
    assert torch.equal(out.detach().cpu(), base[:, 3:36][ids.t()])
    gw, = torch.autograd.grad(out.sum(), w)  # an expanded gradient
    count = torch.bincount(ids.reshape(-1), minlength=40)[:, None].float()
    assert torch.equal(gw.cpu(), count.expand(40, 33))
    wt = base.t().contiguous().to(dev).t().requires_grad_(True)  # columns first in memory
    assert torch.equal(prlstm_amd.embedding(ids.to(dev), wt).detach().cpu(), base[ids])


def test_ids_beyond_the_vocabulary_are_loud(dev):
    prlstm_amd.check_errors(dev)
    w = torch.ones(5, 3, device=dev, requires_grad=True)
    out = prlstm_amd.embedding(torch.tensor([1, 5, -2, 1 << 40], device=dev), w)
    gw, = torch.autograd.grad(out, w, torch.ones(4, 3, device=dev))
    with pytest.raises(RuntimeError, match="beyond the vocabulary"):
        prlstm_amd.check_errors(dev)
    prlstm_amd.check_errors(dev)  # cleared
    assert torch.isnan(out[1]).all() and torch.isnan(out[3]).all()
    assert torch.equal(out[2].cpu(), torch.zeros(3)) and torch.equal(gw.cpu().sum(1), torch.tensor([0., 3, 0, 0, 0]))
    r = prlstm_amd.token_logprobs(torch.zeros(3, 5, device=dev), torch.tensor([4, 5, -1], device=dev))
    with pytest.raises(RuntimeError, match="beyond the vocabulary"):
        prlstm_amd.check_errors(dev)
    assert torch.isnan(r.logp[1]) and float(r.logp[2]) == 0.0 and bool(torch.isfinite(r.entropy).all())


# ---- gated recurrence ----------------------------------------------------------------------


def _gated_plain(zv, h0, reset, dout, dh_n):
    """Values and gradients in 64 bits, and the bounds of their fp32 errors.

    M_t (the state's terms in magnitude) is carried by the same recurrence; each term passes one
    product and one sum a step, each factor within 8 u: E_t = f E_{t-1} + 16 u M_t in any
    association.  The gradient mirrors it."""
    zv, dout, dh_n = zv.double(), dout.double(), dh_n.double()
    T, B, n = zv.shape
    H = n // 2
    z, v = zv[..., :H], zv[..., H:]
    f, w = 1 / (1 + torch.exp(-z)), 1 / (1 + torch.exp(z))
    cut = torch.zeros(T, B, 1, dtype=torch.bool) if reset is None else reset[..., None].bool()
    zero = torch.zeros(B, H, dtype=torch.float64)
    h = zero if h0 is None else h0.double()
    M, E, hs, prev, prevE = h.abs(), zero, [], [], []
    Es = []
    for t in range(T):
        p, pM, pE = (torch.where(cut[t], zero, x) for x in (h, M, E))
        prev.append(p)
        prevE.append(pE)
        h = torch.where(cut[t], w[t] * v[t], f[t] * p + w[t] * v[t])
        M = f[t] * pM + w[t] * v[t].abs()
        E = f[t] * pE + 16 * u * M
        hs.append(h)
        Es.append(E)
    res = {"h_n": (h, E + 1e-36)}
    out = torch.stack(hs) if T else torch.zeros(0, B, H, dtype=torch.float64)
    res["out"] = (out, torch.stack(Es) + 1e-36 if T else torch.zeros(0, B, H, dtype=torch.float64))
    U, MU, EU = dh_n, dh_n.abs(), zero
    dzv, ez = torch.zeros_like(zv), torch.zeros_like(zv)
    for t in range(T - 1, -1, -1):
        G, MG = dout[t] + U, dout[t].abs() + MU
        EG = EU + 4 * u * MG
        diff = prev[t] - v[t]
        ediff = prevE[t] + u * (prev[t].abs() + v[t].abs())
        fw = f[t] * w[t]
        dzv[t, :, :H] = G * diff * fw
        dzv[t, :, H:] = w[t] * G
        ez[t, :, :H] = fw * (EG * (diff.abs() + ediff) + G.abs() * ediff + 20 * u * MG * diff.abs())
        ez[t, :, H:] = w[t] * (EG + 10 * u * MG)
        U = torch.where(cut[t], zero, f[t] * G)
        MU = torch.where(cut[t], zero, f[t] * MG)
        EU = torch.where(cut[t], zero, f[t] * EG + 16 * u * MU)
    res["dzv"] = (dzv, ez + 1e-36)
    res["dh0"] = (U, EU + 1e-36)
    return res


def _check_gated(name, got, want, dtype):
    exact, bound = want
    if name in ("out", "dzv"):
        bound = bound + HALF[dtype] * exact.abs().nan_to_num(0, 0, 0) * 1.01 + TINY[dtype]
    _within(name, got, exact, bound)


GATED = [  # T, B, H
    (0, 2, 5), (1, 1, 1), (1, 3, 70), (2, 5, 33), (7, 2, 64), (8, 1, 129), (9, 3, 100), (17, 2, 2), (31, 1, 256),
    (64, 4, 66), (129, 3, 130), (257, 2, 40), (300, 1, 1), (520, 2, 31), (1025, 1, 72), (2050, 3, 20), (40, 70, 9),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,B,H", GATED)
def test_gated_recurrence(dev, T, B, H, dtype):
    print(f"gated {T} {B} {H} {dtype}", flush=True)
    for order, with_reset, with_h0 in (("time", False, True), ("batch", True, True), ("time", True, False),
                                       ("batch", False, False)):
        g = _gen("gated", T, B, H, order)
        zv = torch.randn(T, B, 2 * H, generator=g)
        zv[..., :H] = zv[..., :H] * 2 + 2  # mostly long memories
        zv = zv.to(dtype)
        dout = torch.randn(T, B, H, generator=g).to(dtype)
        dh_n = torch.randn(B, H, generator=g)
        h0 = torch.randn(B, H, generator=g) if with_h0 else None
        reset = torch.rand(T, B, generator=g) < 0.1 if with_reset else None
        want = _gated_plain(zv, h0, reset, dout, dh_n)
        put = (lambda x: x.to(dev)) if order == "time" else (
            lambda x: x.transpose(0, 1).contiguous().to(dev).transpose(0, 1))
        zd = put(zv).requires_grad_(True)
        hd = None if h0 is None else h0.to(dev).requires_grad_(True)
        rd = None if reset is None else put(reset)
        out, h_n = prlstm_amd.gated_recurrence(zd, hd, rd)
        assert out.dtype == dtype and h_n.dtype == torch.float32
        grads = torch.autograd.grad((out, h_n), [x for x in (zd, hd) if x is not None], (put(dout), dh_n.to(dev)))
        got = {"out": out, "h_n": h_n, "dzv": grads[0]}
        if h0 is not None:
            got["dh0"] = grads[1]
        for k, x in got.items():
            _check_gated(k, x, want[k], dtype)
        with torch.no_grad():
            o2, h2 = prlstm_amd.gated_recurrence(zd, hd, rd)
        assert torch.equal(o2, out) and torch.equal(h2, h_n)
        if T == 1 and order == "time":
            o3, h3 = prlstm_amd.gated_recurrence_step(zd[0].detach(), None if hd is None else hd.detach(),
                                                      None if rd is None else rd[0])
            assert torch.equal(o3, out[0]) and torch.equal(h3, h_n)


def test_gated_gradients_of_parts(dev):
    """Only some outputs in the loss, an expanded gradient, and an unused state."""
    g = _gen("parts")
    T, B, H = 50, 2, 24
    zv, h0 = torch.randn(T, B, 2 * H, generator=g), torch.randn(B, H, generator=g)
    zero = torch.zeros(B, H)
    for use_out, use_h in ((True, False), (False, True)):
        zd, hd = zv.to(dev).requires_grad_(True), h0.to(dev).requires_grad_(True)
        out, h_n = prlstm_amd.gated_recurrence(zd, hd)
        loss = (out.sum() if use_out else 0) + (h_n.sum() if use_h else 0)
        grads = torch.autograd.grad(loss, (zd, hd))
        want = _gated_plain(zv, h0, None, torch.ones(T, B, H) * use_out, zero + float(use_h))
        _check_gated("dzv", grads[0], want["dzv"], torch.float32)
        _check_gated("dh0", grads[1], want["dh0"], torch.float32)


def test_gated_parts_of_a_wider_tensor(dev):
    """zv as a part of a wider projection, unaligned, and a dense copy: the same values."""
    g = _gen("wider")
    wide = torch.randn(70, 3, 150, generator=g).to(dev)
    part = wide[:, :, 5:135]
    a, ha = prlstm_amd.gated_recurrence(part)
    b, hb = prlstm_amd.gated_recurrence(part.contiguous())
    want = _gated_plain(part.cpu(), None, None, torch.zeros(70, 3, 65), torch.zeros(3, 65))
    for o, h in ((a, ha), (b, hb)):
        _check_gated("out", o, want["out"], torch.float32)
        _check_gated("h_n", h, want["h_n"], torch.float32)
    steps = wide[:, :1].expand(70, 4, 150)[:, :, :60]  # one sequence for every batch row
    o, _ = prlstm_amd.gated_recurrence(steps)
    assert torch.equal(o[:, 0], o[:, 3])


@pytest.mark.parametrize("T", [40, 700])
def test_gated_reset_stops_nan_and_infinity(dev, T):
    """What is not finite in one sequence reaches no other one, forward or backward."""
    g = _gen("nan", T)
    B, H = 2, 48
    zv = torch.randn(T, B, 2 * H, generator=g)
    reset = torch.zeros(T, B, dtype=torch.bool)
    reset[T // 4], reset[T // 2 + 1] = True, True
    clean = zv.clone()
    bad = range(T // 4, T // 2 + 1)
    zv[T // 4 + 2, 0, H:] = float("inf")
    zv[T // 4 + 3, 1, :] = float("nan")
    zv[T // 4 + 1, 1, H + 3] = -float("inf")
    dout = torch.randn(T, B, H, generator=g)
    bad_dout = dout.clone()
    bad_dout[T // 4 + 4] = float("nan")
    good = [t for t in range(T) if t not in bad]
    want = _gated_plain(clean, None, reset, dout, torch.zeros(B, H))
    zd = zv.to(dev).requires_grad_(True)
    out, h_n = prlstm_amd.gated_recurrence(zd, None, reset.to(dev))
    dz, = torch.autograd.grad((out, h_n), zd, (bad_dout.to(dev), torch.zeros(B, H, device=dev)))
    _check_gated("out", out[good], tuple(x[good] for x in want["out"]), torch.float32)
    _check_gated("h_n", h_n, want["h_n"], torch.float32)
    _check_gated("dzv", dz[good], tuple(x[good] for x in want["dzv"]), torch.float32)
    assert bool(torch.isinf(out[T // 4 + 2, 0]).all()) and bool(torch.isnan(out[T // 4 + 3, 1]).all())


@pytest.mark.parametrize("T", [20, 900])
def test_gated_infinite_state_stays(dev, T):
    """An infinite state stays infinite (no 0 * inf where a product of gates underflows)."""
    zv = torch.zeros(T, 1, 6)
    zv[..., :3] = -9.0  # gates of 1e-4: their product underflows within a dozen steps
    h0 = torch.tensor([[float("inf"), -float("inf"), 1.0]])
    out, h_n = prlstm_amd.gated_recurrence(zv.to(dev), h0.to(dev))
    assert bool((out[:, 0, 0] == float("inf")).all()) and bool((out[:, 0, 1] == -float("inf")).all())
    assert bool(torch.isfinite(out[:, 0, 2]).all()) and float(h_n[0, 0]) == float("inf")


def test_gated_extreme_gates(dev):
    """Gates that are wholly open or shut, and gates of +-inf."""
    z = torch.tensor([-float("inf"), -200.0, -90.0, 0.0, 30.0, 200.0, float("inf")])
    zv = torch.cat((z, torch.full((7,), 3.0))).expand(5, 2, 14).contiguous()
    h0 = torch.full((2, 7), -2.0)
    out, h_n = prlstm_amd.gated_recurrence(zv.to(dev), h0.to(dev))
    want = _gated_plain(zv, h0, None, torch.zeros(5, 2, 7), torch.zeros(2, 7))
    _check_gated("out", out, want["out"], torch.float32)


def test_gated_state_in_place_and_chained_steps(dev):
    """Single steps that update their state in place give the sequence's values."""
    g = _gen("steps")
    T, B, H = 21, 3, 50
    zv = torch.randn(T, B, 2 * H, generator=g).to(dev, torch.bfloat16)
    h = torch.randn(B, H, generator=g).to(dev)
    reset = (torch.rand(T, B, generator=g) < 0.2).to(dev)
    want = _gated_plain(zv.cpu(), h.cpu(), reset.cpu(), torch.zeros(T, B, H), torch.zeros(B, H))
    for t in range(T):
        out, h2 = prlstm_amd.gated_recurrence_step(zv[t], h, reset[t], h_out=h)
        assert h2 is h
        _check_gated("out", out, tuple(x[t] for x in want["out"]), torch.bfloat16)
    _check_gated("h_n", h, want["h_n"], torch.float32)


# ---- log probabilities ---------------------------------------------------------------------


def _order(x):
    """Ids of each row by value, NaN first, the lowest id first among equals."""
    key = torch.where(torch.isnan(x), torch.full_like(x, float("inf")), x)
    nan_last = (~torch.isnan(x)).to(torch.int8)
    idx = torch.sort(key, dim=1, descending=True, stable=True).indices
    again = torch.sort(nan_last.gather(1, idx), dim=1, stable=True).indices
    return idx.gather(1, again)


def _logprob_plain(x, tokens, top, dlogp, dent, dtop):
    """Values, gradient and bounds.  L u bounds a row's sums (no partial sum is longer than L
    terms: a lane's share and the joins)."""
    x = x.double()
    N, V = x.shape
    L = math.ceil(V / 64) + 96
    m = x.amax(1, keepdim=True) if V else torch.zeros(N, 1)
    none = torch.isneginf(x).all(1)
    m0 = torch.where(torch.isneginf(m), torch.zeros(()).double(), m)
    ls = torch.log(torch.exp(x - m0).sum(1, keepdim=True))
    lp = x - m0 - ls
    lp = torch.where(lp < -3.4028236e38, -float("inf"), lp)  # beyond fp32
    p = torch.exp(lp)
    plp = torch.where(p == 0, torch.zeros(()).double(), p * lp)
    ent = -plp.sum(1)
    d = torch.where(p == 0, torch.zeros(()).double(), (x - m).abs())
    spread = (p * d).sum(1)  # mean distance from the largest
    e_lse = u * (L + 8 + 4 * spread + 2 * ls[:, 0].abs())  # of log sum exp(x - m)
    e_lse = torch.where(none, torch.zeros(()).double(), e_lse)
    e_ent = 2 * u * (L + 16) * (1 + spread) + 8 * u * (p * d * d).sum(1)
    ent, e_ent = torch.where(none, 0.0, ent), torch.where(none, 0.0, e_ent)
    lp = torch.where(none[:, None], -float("inf"), lp)
    rows, there = torch.arange(N), tokens >= 0
    at = tokens.clamp(0, V - 1)
    logp = torch.where(there, lp[rows, at], 0.0)
    size = lambda v: v.abs().nan_to_num(0, 0, 0)  # noqa: E731
    res = {"logp": (logp, size(e_lse) + 2 * u * (size(logp) + size(ls[:, 0]))), "entropy": (ent, size(e_ent))}
    idx = _order(x)[:, :top]
    tl = lp.gather(1, idx)
    res["top_ids"] = idx
    res["top_logp"] = (tl, size(e_lse)[:, None] + 2 * u * (size(tl) + size(ls)))
    one = torch.zeros_like(x)
    one[rows[there], at[there]] = dlogp.double()[there]
    one.scatter_add_(1, idx, dtop.double())
    S = one.sum(1, keepdim=True)
    mag = (dlogp.abs() * there).double()[:, None] + dtop.abs().double().sum(1, keepdim=True)
    dh = dent.double()[:, None]
    inner = S + dh * torch.where(p == 0, 0.0, lp + ent[:, None])
    g = one - torch.where(p == 0, 0.0, p * inner)
    g = torch.where(none[:, None], 0.0, g)
    e_lp = size(e_lse)[:, None] + 2 * u * (size(lp) + size(ls))
    e_in = (top + 4) * u * mag + dh.abs() * (e_lp + size(e_ent)[:, None] + 4 * u * (size(lp) + ent[:, None]))
    e_g = size(p) * ((8 * u + e_lp) * (mag + dh.abs() * (size(lp) + size(ent)[:, None])) + e_in) + (top + 4) * u * (
        one.abs() + size(p) * size(inner))
    # a probability below the normal numbers may be 0
    res["dlogits"] = (g, e_g + 1e-36 * (1 + mag + dh.abs() * 1000))
    return res


def _check_logprob(dev, logits, tokens, top, g, dtype, ent=True):
    N, V = logits.shape
    dlogp, dent = torch.randn(N, generator=g), torch.randn(N, generator=g) * float(ent)
    dtop = torch.randn(N, top, generator=g)
    want = _logprob_plain(logits, tokens, top, dlogp, dent, dtop)
    xd = logits.to(dev) if logits.is_contiguous() else torch.empty_strided(
        logits.shape, logits.stride(), dtype=dtype, device=dev).copy_(logits)
    xd.requires_grad_(True)
    r = prlstm_amd.token_logprobs(xd, tokens.to(dev), top=top)
    for k in ("logp", "entropy") + (("top_logp",) if top else ()):
        got = getattr(r, k)
        assert got.dtype == torch.float32
        _within(k, got, *want[k])
    outs, gs = [r.logp], [dlogp.to(dev)]
    if ent:
        outs, gs = outs + [r.entropy], gs + [dent.to(dev)]
    if top:
        assert torch.equal(r.top_ids.cpu(), want["top_ids"])
        outs, gs = outs + [r.top_logp], gs + [dtop.to(dev)]
    dx, = torch.autograd.grad(outs, xd, gs)
    assert dx.dtype == dtype
    exact, bound = want["dlogits"]
    _within("dlogits", dx, exact, bound + HALF[dtype] * exact.abs().nan_to_num(0, 0, 0) * 1.01 + TINY[dtype])
    with torch.no_grad():
        q = prlstm_amd.token_logprobs(xd, tokens.to(dev), top=top)
    for a, b in zip(q, r):
        assert a is None and b is None or torch.equal(a.nan_to_num(7.0), b.detach().nan_to_num(7.0))


LOGPROB = [  # N, V, top
    (0, 7, 2), (1, 1, 1), (3, 2, 0), (5, 31, 31), (2, 64, 32), (7, 65, 5), (4, 255, 3), (3, 257, 1), (2, 1000, 20),
    (1, 2049, 32), (6, 4099, 7), (2, 10007, 5), (1, 70001, 20), (300, 100, 4), (2, 33333, 0), (1, 262144, 32), (40, 20001, 32), (3, 16383, 32), (520, 2049, 32),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V,top", LOGPROB)
def test_logprobs(dev, N, V, top, dtype):
    print(f"logprobs {N} {V} {top} {dtype}", flush=True)
    g = _gen("logprob", N, V, top)
    x = (torch.randn(N, V, generator=g) * 3).to(dtype)
    tokens = torch.randint(0, V, (N,), generator=g)
    tokens[torch.rand(N, generator=g) < 0.2] = -1
    _check_logprob(dev, x, tokens, top, g, dtype)
    _check_logprob(dev, x, tokens.to(torch.int32).long(), 0, g, dtype, ent=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [50, 1500, 9001])
def test_logprobs_masks(dev, V, dtype):
    """Masked tokens, a row with one token left, rows with none, masks of the type's lowest value."""
    g = _gen("mask", V)
    x = (torch.randn(12, V, generator=g) * 2).to(dtype)
    x[torch.rand(12, V, generator=g) < 0.5] = -float("inf")
    low = torch.finfo(dtype).min
    x[1] = -float("inf")
    x[2] = -float("inf")
    x[2, V // 2] = 1.5
    x[3] = low
    x[4, : V // 2] = low
    x[5] = -float("inf")
    x[5, -1] = low
    x[6] = low
    x[6, 3] = -low  # the largest: the others are infinitely far below
    x[7] = 0.25
    x[8, ::3] = -float("inf")
    tokens = torch.randint(0, V, (12,), generator=g)
    tokens[6] = 3
    tokens[11] = -1
    _check_logprob(dev, x, tokens, min(32, V), g, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [70, 5003])
def test_logprobs_of_rows_that_are_not_finite(dev, V, dtype):
    """NaN or +inf in a row makes its results NaN, and the alternatives are still in order."""
    g = _gen("notfinite", V)
    x = torch.randn(6, V, generator=g).to(dtype)
    x[0, V - 1] = float("nan")
    x[1, 5] = float("inf")
    x[2, 9], x[2, 3], x[2, 20] = float("nan"), float("inf"), -float("nan")
    x[3] = float("nan")
    x[4] = -float("inf")
    x[4, 7] = float("nan")
    top = 9
    xd = x.to(dev).requires_grad_(True)
    tokens = torch.arange(6) + 3
    r = prlstm_amd.token_logprobs(xd, tokens.to(dev), top=top)
    dx, = torch.autograd.grad(r.logp.sum(), xd)
    assert torch.equal(r.top_ids.cpu(), _order(x.float())[:, :top])
    for t in (r.logp, r.entropy, r.top_logp):
        assert bool(torch.isnan(t[:5]).all()) and bool(torch.isfinite(t[5]).all())
    assert bool(torch.isnan(dx[:4]).all()) and bool(torch.isfinite(dx[5]).all())


@pytest.mark.parametrize("V", [300, 20000, 100001])
def test_logprobs_alternatives_in_hard_orders(dev, V):
    """Equal logits, zeros of both signs, rising, falling and blockwise rows."""
    g = _gen("hard", V)
    ramp = torch.arange(V, dtype=torch.float32) / V
    rows = [torch.zeros(V), torch.zeros(V).index_fill_(0, torch.arange(0, V, 2), -0.0), ramp, -ramp,
            torch.randint(0, 3, (V,), generator=g).float(), (torch.arange(V) // 40).float() * 1e-3,
            -(torch.arange(V) // 9000).float(), torch.where(torch.arange(V) % 256 == 7, ramp + 5, ramp),
            torch.where(torch.arange(V) < 4000, ramp + 5, ramp), torch.full((V,), -float("inf")),
            torch.full((V,), -3e38), torch.where(torch.arange(V) % 3000 == 5, ramp, torch.full((V,), -float("inf"))),
            torch.where(torch.arange(V) > V - 25, ramp + 1, torch.zeros(V))]
    x = torch.stack(rows)
    for dtype in DTYPES:
        xt = x.clamp_min(torch.finfo(dtype).min).where(x != -float("inf"), x).to(dtype)
        for top in (1, 32):
            r = prlstm_amd.token_logprobs(xt.to(dev), top=top)
            assert r.logp is None
            assert torch.equal(r.top_ids.cpu(), _order(xt.float())[:, :top]), (dtype, top)


def test_logprobs_strides_and_shapes(dev):
    g = _gen("lpstrides")
    for dtype in DTYPES:
        wide = torch.randn(9, 1201, generator=g).to(dtype)
        for part in (wide[:, :1000], wide[:, 1:1000], wide[2:, 3:4], wide[::2, 7:]):
            tokens = torch.randint(0, part.shape[1], (part.shape[0],), generator=g)
            _check_logprob(dev, part, tokens, min(3, part.shape[1]), g, dtype)
    x = torch.randn(3, 4, 77, generator=g).to(dev)
    tokens = torch.randint(0, 77, (3, 4), generator=g).to(dev)
    r = prlstm_amd.token_logprobs(x, tokens, top=2)
    flat = prlstm_amd.token_logprobs(x.reshape(12, 77), tokens.reshape(12), top=2)
    for a, b, tail in zip(r, flat, ((), (), (2,), (2,))):
        assert a.shape == (3, 4, *tail) and torch.equal(a.reshape(b.shape), b)
    cols = x.permute(2, 0, 1).contiguous().permute(1, 2, 0)  # the vocabulary first in memory
    assert torch.equal(prlstm_amd.token_logprobs(cols, tokens).logp, r.logp)
    one = prlstm_amd.token_logprobs(x[0, 0], tokens[0, 0])
    assert one.logp.shape == () and torch.equal(one.logp, r.logp[0, 0])
    row = x[:1, 0].expand(5, 77)  # one row for five tokens
    many = prlstm_amd.token_logprobs(row, tokens[0, 0].expand(5))
    assert torch.equal(many.logp, r.logp[0, 0].expand(5))


# ---- sizes beyond the caches, offsets beyond 32 bits ----------------------------------------


def test_embedding_beyond_the_caches(dev):
    g = torch.Generator(device=dev).manual_seed(1)
    N, V, D = 66000, 70001, 1024
    ids = (torch.rand(N, device=dev, generator=g) ** 3 * V).int().clamp_max(V - 1)
    w = torch.randn(V, D, device=dev, generator=g).bfloat16().requires_grad_(True)
    dout = torch.randn(N, D, device=dev, generator=g).bfloat16()
    out = prlstm_amd.embedding(ids, w, 3.0)
    assert torch.equal(out.detach(), (w.detach()[ids].float() * 3.0).bfloat16())
    dw, = torch.autograd.grad(out, w, dout)
    at = ids.long()
    want = torch.zeros(V, D, dtype=torch.float64, device=dev).index_add_(0, at, dout.double()) * 3.0
    mag = torch.zeros(V, D, dtype=torch.float64, device=dev).index_add_(0, at, dout.double().abs()) * 3.0
    count = torch.bincount(at, minlength=V)[:, None].double()
    bound = (count + 2) * u * mag + HALF[torch.bfloat16] * 1.01 * want.abs() + 1e-38
    assert bool(((dw.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype,T", [(torch.bfloat16, 2900), (torch.float32, 1500)])
def test_gated_beyond_the_caches(dev, dtype, T):
    g = torch.Generator(device=dev).manual_seed(2)
    B, H = 16, 1024
    zv = torch.randn(T, B, 2 * H, device=dev, generator=g)
    zv[..., :H] += 2.0
    zv = zv.to(dtype).requires_grad_(True)
    dout = torch.randn(T, B, H, device=dev, generator=g).to(dtype)
    reset = torch.rand(T, B, device=dev, generator=g) < 0.01
    for r in (None, reset):
        out, h_n = prlstm_amd.gated_recurrence(zv, None, r)
        dzv, = torch.autograd.grad(out, zv, dout)
        pick = torch.randint(0, H, (40,), device=dev, generator=g)  # some channels, in 64 bits
        part = torch.cat((zv.detach()[..., pick], zv.detach()[..., H + pick]), -1)
        want = _gated_plain(part.cpu(), None, None if r is None else r.cpu(), dout[..., pick].cpu(), torch.zeros(B, 40))
        _check_gated("out", out[..., pick], want["out"], dtype)
        _check_gated("h_n", h_n[..., pick], want["h_n"], dtype)
        _check_gated("dzv", torch.cat((dzv[..., pick], dzv[..., H + pick]), -1), want["dzv"], dtype)


def test_logprobs_beyond_the_caches(dev):
    """Sampled rows against 64 bits; every row's gradient sums to its own part."""
    g = torch.Generator().manual_seed(3)
    N, V = 4100, 17001
    gd = torch.Generator(device=dev).manual_seed(3)
    x = (3 * torch.randn(N, V, device=dev, generator=gd)).bfloat16().requires_grad_(True)
    tokens = torch.randint(0, V, (N,), generator=g)
    dlogp, dent = torch.randn(N, generator=g), torch.randn(N, generator=g)
    dtop = torch.randn(N, 3, generator=g)
    r = prlstm_amd.token_logprobs(x, tokens.to(dev), top=3)
    for ent in (False, True):
        outs = [r.logp, r.top_logp] + ([r.entropy] if ent else [])
        gs = [dlogp.to(dev), dtop.to(dev)] + ([dent.to(dev)] if ent else [])
        dx, = torch.autograd.grad(outs, x, gs, retain_graph=True)
        rows = torch.cat((torch.arange(3), torch.randint(0, N, (20,), generator=g), torch.tensor([N - 1])))
        want = _logprob_plain(x.detach()[rows].cpu(), tokens[rows], 3, dlogp[rows], dent[rows] * ent, dtop[rows])
        for k in ("logp", "entropy", "top_logp"):
            _within(k, getattr(r, k)[rows], *want[k])
        assert torch.equal(r.top_ids[rows].cpu(), want["top_ids"])
        exact, bound = want["dlogits"]
        _within("dlogits", dx[rows], exact, bound + HALF[torch.bfloat16] * 1.01 * exact.abs() + 1e-38)


def test_offsets_beyond_32_bits(dev):
    """Rows, steps and batch rows that lie more than 2^32 bytes apart."""
    g = _gen("far")
    far = (1 << 31) + 6  # elements
    buf = torch.empty(2 * far + 4096, dtype=torch.bfloat16, device=dev)

    def place(t):  # [3, n] at rows `far` apart
        v = buf.as_strided((3, t.shape[1]), (far, 1))
        v.copy_(t)
        return v

    x = torch.randn(3, 2001, generator=g).bfloat16()
    tokens = torch.tensor([5, 2000, 17])
    v = place(x)
    near = prlstm_amd.token_logprobs(x.to(dev), tokens.to(dev), top=4)
    for a, b in zip(prlstm_amd.token_logprobs(v, tokens.to(dev), top=4), near):
        assert torch.equal(a, b)
    ids = torch.tensor([2, 0, 1, 2], device=dev)
    assert torch.equal(prlstm_amd.embedding(ids, v, 2.0), prlstm_amd.embedding(ids, x.to(dev), 2.0))
    zv = torch.randn(3, 200, generator=g).bfloat16()
    v = place(zv)
    dense = zv.to(dev)
    for a, b in ((v[:, None], dense[:, None]), (v[None], dense[None])):  # far steps, far batch rows
        a, b = a.detach().requires_grad_(True), b.detach().requires_grad_(True)
        oa, ha = prlstm_amd.gated_recurrence(a)
        ob, hb = prlstm_amd.gated_recurrence(b)
        assert torch.equal(oa, ob) and torch.equal(ha, hb)
        ga, = torch.autograd.grad(oa, a, torch.ones_like(oa))
        gb, = torch.autograd.grad(ob, b, torch.ones_like(ob))
        assert torch.equal(ga, gb)


# ---- gradients against differences ---------------------------------------------------------


def _differences(fn, x, eps=1e-5):
    """Central differences of the scalar fn in 64 bits, for every element of x."""
    x = x.double()
    g = torch.zeros(x.numel(), dtype=torch.float64)
    for i in range(x.numel()):
        step = torch.zeros(x.numel(), dtype=torch.float64)
        step[i] = eps
        step = step.reshape(x.shape)
        g[i] = (fn(x + step) - fn(x - step)) / (2 * eps)
    return g.reshape(x.shape)


# the differences' own error: eps^2 / 6 of a third derivative of order 10 (1.7e-10), and 1e-15 / eps
# of losses of order 100 (1e-8); fp32 gradients of order 10 add 1e-6 and sums of some tens of terms
DIFF = 2e-5


def test_embedding_gradient_against_differences(dev):
    g = _gen("d1")
    ids, w, c = torch.tensor([2, 0, 2, -1, 3, 2]), torch.randn(5, 3, generator=g), torch.randn(6, 3, generator=g)

    def loss(x):
        return (torch.where((ids >= 0)[:, None], 0.7 * x[ids.clamp_min(0)], 0.0) * c.double()).sum()

    wd = w.to(dev).requires_grad_(True)
    (prlstm_amd.embedding(ids.to(dev), wd, 0.7) * c.to(dev)).sum().backward()
    _within("dweight", wd.grad, _differences(loss, w), DIFF)


def test_gated_gradient_against_differences(dev):
    g = _gen("d2")
    T, B, H = 11, 2, 3
    zv, h0 = torch.randn(T, B, 2 * H, generator=g), torch.randn(B, H, generator=g)
    c, ch = torch.randn(T, B, H, generator=g), torch.randn(B, H, generator=g)
    reset = torch.zeros(T, B, dtype=torch.bool)
    reset[4, 0], reset[8, 1] = True, True

    def loss(z, h):
        r = _gated_plain(z, h, reset, torch.zeros(T, B, H), torch.zeros(B, H))
        return (r["out"][0] * c.double()).sum() + (r["h_n"][0] * ch.double()).sum()

    zd, hd = zv.to(dev).requires_grad_(True), h0.to(dev).requires_grad_(True)
    out, h_n = prlstm_amd.gated_recurrence(zd, hd, reset.to(dev))
    ((out * c.to(dev)).sum() + (h_n * ch.to(dev)).sum()).backward()
    _within("dzv", zd.grad, _differences(lambda z: loss(z, h0.double()), zv), DIFF)
    _within("dh0", hd.grad, _differences(lambda h: loss(zv, h), h0), DIFF)


def test_logprob_gradient_against_differences(dev):
    g = _gen("d3")
    x, tokens = torch.randn(3, 11, generator=g), torch.tensor([4, -1, 0])
    x[2, 5] = -float("inf")
    a, b, t = torch.randn(3, generator=g), torch.randn(3, generator=g), torch.randn(3, 2, generator=g)
    zero = torch.zeros(3)

    def loss(y):
        y = torch.where(torch.isneginf(x), -float("inf"), y)
        r = _logprob_plain(y, tokens, 2, zero, zero, torch.zeros(3, 2))
        return (r["logp"][0] * a).sum() + (r["entropy"][0] * b).sum() + (r["top_logp"][0] * t).sum()

    xd = x.to(dev).requires_grad_(True)
    r = prlstm_amd.token_logprobs(xd, tokens.to(dev), top=2)
    ((r.logp * a.to(dev)).sum() + (r.entropy * b.to(dev)).sum() + (r.top_logp * t.to(dev)).sum()).backward()
    _within("dlogits", xd.grad, _differences(loss, x.nan_to_num(neginf=0.0)), DIFF)


# ---- streams, graphs, refusals --------------------------------------------------------------


def _pass(ids, w, zw, tokens, dev):
    x = prlstm_amd.embedding(ids, w, scale=2.0)
    out, h = prlstm_amd.gated_recurrence(x @ zw)
    r = prlstm_amd.token_logprobs(out @ w.t(), tokens, top=3)
    grads = torch.autograd.grad((r.logp.sum() + 0.1 * r.entropy.sum(), h.sum()), (w, zw), (torch.ones_like(r.logp.sum()),) * 2)
    return (out.detach(), h.detach(), r.logp.detach(), r.entropy.detach(), r.top_ids, *grads)


def _pass_inputs(dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    T, B, V, D = 60, 3, 500, 32
    ids = torch.randint(0, V, (T, B), generator=g).to(dev)
    w = (0.3 * torch.randn(V, D, generator=g)).to(dev).requires_grad_(True)
    zw = (0.3 * torch.randn(D, 2 * D, generator=g)).to(dev).requires_grad_(True)
    return ids, w, zw, torch.randint(0, V, (T, B), generator=g).to(dev)


def test_another_stream(dev):
    args = _pass_inputs(dev)
    want = _pass(*args, dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _pass(*args, dev)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_graph_replays(dev):
    """A captured serving pass, replayed with new inputs between eager calls."""
    g = _gen("graph")
    V, B, H, S = 4001, 4, 96, 60000
    w = torch.randn(V, 2 * H, generator=g).to(dev, torch.bfloat16)
    ids = torch.zeros(B, dtype=torch.int64, device=dev)
    seq_ids = torch.zeros(300, B, dtype=torch.int64, device=dev)
    h = torch.zeros(B, H, device=dev)
    logits = torch.zeros(B, S, device=dev)
    dout = torch.ones(300, B, 2 * H, device=dev, dtype=torch.bfloat16)

    def calls():
        out, h2 = prlstm_amd.gated_recurrence_step(prlstm_amd.embedding(ids, w), h)
        seq, _ = prlstm_amd.gated_recurrence(prlstm_amd.embedding(seq_ids, w))
        r = prlstm_amd.token_logprobs(logits, ids, top=8)
        wg = w.detach().requires_grad_(True)
        dw, = torch.autograd.grad(prlstm_amd.embedding(seq_ids, wg), wg, dout)
        return out, h2, seq, r.logp, r.entropy, r.top_logp, r.top_ids, dw

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = calls()
    for k in range(4):
        ids.copy_(torch.randint(0, V, (B,), generator=g))
        seq_ids.copy_((torch.rand(300, B, generator=g) ** 4 * V).long())
        h.copy_(torch.randn(B, H, generator=g))
        logits.copy_(torch.randn(B, S, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(static, calls()):
            assert torch.equal(a, b), k


def test_refusals(dev):
    ids = torch.zeros(3, dtype=torch.int64, device=dev)
    w = torch.zeros(4, 6, device=dev)
    zv = torch.zeros(5, 2, 8, device=dev)
    for match, call in (
            ("must be \\[V, D\\]", lambda: prlstm_amd.embedding(ids, w[0])),
            ("int64 or int32", lambda: prlstm_amd.embedding(ids.float(), w)),
            ("bfloat16, float16 or float32", lambda: prlstm_amd.embedding(ids, w.double())),
            ("ids is on cpu", lambda: prlstm_amd.embedding(ids.cpu(), w)),
            ("padding_idx", lambda: prlstm_amd.embedding(ids, w, padding_idx=4)),
            ("zv must be", lambda: prlstm_amd.gated_recurrence(zv[..., :7])),
            ("zv must be", lambda: prlstm_amd.gated_recurrence(zv[0])),
            ("h0 must have shape", lambda: prlstm_amd.gated_recurrence(zv, torch.zeros(2, 5, device=dev))),
            ("h0 must be a floating", lambda: prlstm_amd.gated_recurrence(zv, torch.zeros(2, 4))),
            ("reset must have shape", lambda: prlstm_amd.gated_recurrence(zv, reset=torch.zeros(2, 5, device=dev).bool())),
            ("reset must be a bool", lambda: prlstm_amd.gated_recurrence(zv, reset=torch.zeros(5, 2, device=dev))),
            ("contiguous float32", lambda: prlstm_amd.gated_recurrence_step(zv[0], torch.zeros(2, 4, device=dev).half())),
            ("contiguous float32", lambda: prlstm_amd.gated_recurrence_step(zv[0], torch.zeros(4, 2, device=dev).t())),
            ("zv must be", lambda: prlstm_amd.gated_recurrence_step(zv, None)),
            ("top must be in 0..6", lambda: prlstm_amd.token_logprobs(w, top=7)),
            ("top must be in 0..32", lambda: prlstm_amd.token_logprobs(torch.zeros(2, 50, device=dev), top=33)),
            ("tokens must have shape", lambda: prlstm_amd.token_logprobs(w, ids)),
            ("int64 or int32", lambda: prlstm_amd.token_logprobs(w, w[:, 0])),
            ("bfloat16, float16 or float32", lambda: prlstm_amd.token_logprobs(w.double()))):
        with pytest.raises(RuntimeError, match=match):
            call()
    x = torch.zeros(2, 5, device=dev, requires_grad=True)
    r = prlstm_amd.token_logprobs(x, ids[:2])
    gx, = torch.autograd.grad(r.logp.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        gx.sum().backward()


def test_an_input_changed_before_the_backward_is_noticed(dev):
    x = torch.zeros(2, 5, device=dev, requires_grad=True)
    y = x * 1.0
    r = prlstm_amd.token_logprobs(y, torch.zeros(2, dtype=torch.int64, device=dev))
    y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.logp.sum().backward()
