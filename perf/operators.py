"""Operators of a language model around the recurrent layer, for timing and for comparing outputs:
the embedding of token ids (with its gradient), the gated linear recurrence (training, and one token
at a time) and the log probabilities of tokens under given logits (with entropy, the best
alternatives and the gradient).

Each case is one pass as a program makes it: a serving call without gradients, or a training step's
forward and backward.  With ``own`` false the pass is computed in elementary torch operations in 32
bits, rounded once at the end; with ``own`` true by the package's operators.
"""

import math

import torch

own = False

DEV = torch.device("cuda", 0)
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
PAD = -1  # id of a position without a token


def _embed(name, call, n, v, d, dtype, ids="int64", pad=False):
    """n ids into a [v, d] table.  pad: a share of the positions hold no token."""
    return {"name": name, "op": "embed", "call": call, "N": n, "V": v, "D": d, "dtype": dtype, "ids": ids, "pad": pad}


def _gated(name, call, t, b, h, dtype, order="time", reset=False, h0=False):
    """order: which of time and batch comes first in memory.  reset: sequences of several
    documents, the state cut between them.  h0: a state from the call before."""
    return {"name": name, "op": "gated", "call": call, "T": t, "B": b, "H": h, "dtype": dtype, "order": order,
            "reset": reset, "h0": h0}


def _score(name, call, n, v, dtype, top=0, pitch=0, masked=False, entropy=False, pad=False):
    """n rows of v logits.  pitch: columns that the projection has beyond the vocabulary; masked:
    tokens that may not follow have -inf, in some rows all have; entropy: the loss has it too."""
    return {"name": name, "op": "score", "call": call, "N": n, "V": v, "dtype": dtype, "top": top, "pitch": pitch,
            "masked": masked, "entropy": entropy, "pad": pad}


def listed():
    return [
        # the next token of eight streams that are being served
        _embed("embed_serve", "infer", 8, 32768, 512, "bf16"),
        # a ragged batch of short sequences, padded, with an odd width and vocabulary
        _embed("embed_train_ragged", "train", 700, 10007, 650, "fp32", pad=True),
        # the headline layer's batch (256 steps of 32 sequences) into its input width
        _embed("embed_train", "train", 8192, 32768, 256, "fp32"),
        # the long-sequence batch (4096 steps of 16) with a large vocabulary
        _embed("embed_train_large", "train", 65536, 131072, 1024, "bf16", ids="int32"),
        # one token of 32 served streams, each with its state
        _gated("gated_serve", "step", 1, 32, 1024, "bf16", h0=True),
        # the headline batch
        _gated("gated_train", "train", 256, 32, 512, "bf16"),
        # few channels and a very long sequence of packed documents, after a window before it
        _gated("gated_train_narrow", "train", 16383, 2, 256, "fp32", order="batch", reset=True, h0=True),
        # the long-sequence batch
        _gated("gated_train_long", "train", 4096, 16, 1024, "bf16"),
        # the best alternatives of a few served streams, from a large vocabulary
        _score("score_serve", "infer", 4, 131072, "bf16", top=20),
        # a batch of prompts scored with a vocabulary that is narrower than its projection
        _score("score_prompts", "infer", 1000, 50021, "fp16", top=5, pitch=155, masked=True),
        # a ragged padded batch, with a bonus on the entropy, in full precision
        _score("score_train_ragged", "train", 700, 10007, "fp32", masked=True, entropy=True, pad=True),
        # the headline batch's loss: the largest pass
        _score("score_train", "train", 8192, 32768, "bf16"),
    ]


def _log_int(rng, lo, hi, odd):
    """An integer spread evenly over the logarithm of [lo, hi]; unless `odd`, of few set bits."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if not odd:
        q = 64 if v >= 256 else 16 if v >= 48 else 4 if v >= 8 else 1
        v = max(q, v // q * q)
    return max(lo, min(hi, v))


def draw(rng):
    odd = rng.random() < 0.5
    op = rng.choice(["embed", "gated", "score"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    flag = lambda p: rng.random() < p  # noqa: E731
    if op == "embed":
        c = _embed(None, rng.choice(["infer", "train", "train"]), _log_int(rng, 1, 65536, True),
                   _log_int(rng, 64, 131072, odd), _log_int(rng, 16, 2048, odd), dtype, rng.choice(["int64", "int32"]),
                   flag(0.3))
        top, shrink = work(listed()[3]), ("N", "V")
    elif op == "gated":
        call = rng.choice(["step", "infer", "train", "train"])
        t = 1 if call == "step" else _log_int(rng, 1, 16384, True)
        c = _gated(None, call, t, _log_int(rng, 1, 64, odd), _log_int(rng, 16, 2048, odd), dtype,
                   rng.choice(["time", "batch"]), flag(0.4), call == "step" or flag(0.4))
        top, shrink = work(listed()[7]), ("T", "B")
    else:
        call = rng.choice(["infer", "infer", "train"])
        c = _score(None, call, _log_int(rng, 1, 8192, True), _log_int(rng, 64, 262144, odd), dtype,
                   rng.choice([0, 1, 5, 20, 32]) if call == "infer" else rng.choice([0, 0, 4]),
                   rng.choice([0, 0, 1, 64, 155]), flag(0.4), call == "train" and flag(0.4), flag(0.3))
        top, shrink = work(listed()[11]), ("N", "V")
    del c["name"]
    while work(c)["bytes"] > 0.9 * top["bytes"] or work(c)["flops"] > 0.9 * top["flops"]:
        k = max(shrink, key=lambda s: c[s])
        c[k] = max(1, c[k] * 3 // 4)
    return c


def _tokens(g, n, v, pad):
    """Ids as text has them: the k-th most frequent token with a share of about 1/k."""
    u = torch.rand(n, device=DEV, generator=g, dtype=torch.float64)
    ids = (torch.exp(u * math.log(v + 1.0)) - 1).long().clamp_(0, v - 1)
    if pad:
        ids[torch.rand(n, device=DEV, generator=g) < 0.2] = PAD
    return ids


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    dt, train = DTYPES[case["dtype"]], case["call"] == "train"
    s = {"op": case["op"], "call": case["call"]}
    if case["op"] == "embed":
        n, v, d = case["N"], case["V"], case["D"]
        s["ids"] = _tokens(g, n, v, case["pad"]).to(torch.int32 if case["ids"] == "int32" else torch.int64)
        s["weight"] = (d ** -0.5 * rand(v, d)).to(dt).requires_grad_(train)
        s["scale"] = d ** 0.5
        if train:
            s["dout"] = rand(n, d).to(dt)
    elif case["op"] == "gated":
        t, b, h = case["T"], case["B"], case["H"]
        shape = (t, b) if case["order"] == "time" else (b, t)
        swap = (lambda x: x) if case["order"] == "time" else (lambda x: x.transpose(0, 1))
        zv = rand(*shape, 2 * h)
        zv[..., :h].mul_(1.5).add_(2.0)  # gates that keep their state for tens of steps
        zv = swap(zv.to(dt))
        s["zv"] = zv[0] if case["call"] == "step" else zv.requires_grad_(train)
        s["reset"] = swap(torch.rand(*shape, device=DEV, generator=g) < 1 / 300) if case["reset"] else None
        if s["reset"] is not None and case["call"] == "step":
            s["reset"] = s["reset"][0]
        s["h0"] = rand(b, h).requires_grad_(train) if case["h0"] else None
        if train:
            s["dout"], s["dh_n"] = swap(rand(*shape, h).to(dt)), 0.5 * rand(b, h)
    else:
        n, v = case["N"], case["V"]
        full = rand(n, v + case["pitch"]).mul_(2.0)
        s["tokens"] = _tokens(g, n, v, case["pad"])
        at = torch.randint(0, v, (n,), device=DEV, generator=g)
        full.scatter_add_(1, at[:, None], 12 * torch.rand(n, 1, device=DEV, generator=g))  # rows of any confidence
        if case["masked"]:
            full.masked_fill_(torch.rand(n, v + case["pitch"], device=DEV, generator=g) < 0.25, -math.inf)
            full[torch.rand(n, device=DEV, generator=g) < 0.02] = -math.inf
        s["logits"] = full.to(dt)[:, :v]
        if train:
            s["logits"].requires_grad_(True)
            s["dlogp"] = -torch.rand(n, device=DEV, generator=g) / n
            s["dent"] = -0.01 * torch.rand(n, device=DEV, generator=g) / n if case["entropy"] else None
            s["dtop"] = -torch.rand(n, case["top"], device=DEV, generator=g) / n if case["top"] else None
        s["top"] = case["top"]
    return s


def run(state):
    return {"embed": _run_embed, "gated": _run_gated, "score": _run_score}[state["op"]](state)


def _run_embed(s):
    ids, weight = s["ids"], s["weight"]
    if own:
        import prlstm_amd
        out = prlstm_amd.embedding(ids, weight, scale=s["scale"])
        if s["call"] == "infer":
            return {"out": out}
        dw, = torch.autograd.grad(out, weight, s["dout"])
        return {"out": out.detach(), "dweight": dw}
    with torch.no_grad():
        dt = weight.dtype
        there = ids >= 0
        at = ids.clamp_min(0).long()
        rows = weight[at].float() * s["scale"]
        out = torch.where(there[:, None], rows, torch.zeros((), device=DEV)).to(dt)
        if s["call"] == "infer":
            return {"out": out}
        d = torch.where(there[:, None], s["dout"].float() * s["scale"], torch.zeros((), device=DEV))
        dw = torch.zeros(weight.shape, device=DEV).index_add_(0, at, d)
        return {"out": out, "dweight": dw.to(dt)}


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t for every t, h_{-1} = 0, in log2(T) passes: after the pass of distance
    k, (a_t, b_t) is the map of the steps t-2k+1 .. t.  Overwrites a and b."""
    k, t = 1, a.shape[0]
    while k < t:
        b[k:] += a[k:] * b[:-k]
        a[k:] = a[k:] * a[:-k]
        k *= 2
    return b


def _run_gated(s):
    zv, reset, h0 = s["zv"], s["reset"], s["h0"]
    if own:
        import prlstm_amd
        if s["call"] == "step":
            out, h = prlstm_amd.gated_recurrence_step(zv, h0, reset=reset)
            return {"out": out, "h_n": h}
        out, h = prlstm_amd.gated_recurrence(zv, h0, reset=reset)
        if s["call"] == "infer":
            return {"out": out, "h_n": h}
        grads = torch.autograd.grad((out, h), [x for x in (zv, h0) if x is not None], (s["dout"], s["dh_n"]))
        return {"out": out.detach(), "h_n": h.detach(), **dict(zip(("dzv", "dh0"), grads))}
    with torch.no_grad():
        dt, n = zv.dtype, zv.shape[-1] // 2
        if s["call"] == "step":
            zv = zv[None]
            reset = None if reset is None else reset[None]
        z, v = zv[..., :n].float(), zv[..., n:].float()
        f, w = torch.sigmoid(z), torch.sigmoid(-z)  # w = 1 - f
        a = f if reset is None else torch.where(reset[..., None], torch.zeros((), device=DEV), f)
        b = w * v
        if h0 is not None:
            b[0] += a[0] * h0
        h = _scan(a.clone(), b)
        out, h_n = h.to(dt), h[-1].clone()
        if s["call"] == "step":
            return {"out": out[0], "h_n": h_n}
        if s["call"] == "infer":
            return {"out": out, "h_n": h_n}
        # G_t = dout_t + a_{t+1} G_{t+1}, the same recurrence from the last step to the first
        e = s["dout"].to(torch.float32, copy=True)
        e[-1] += s["dh_n"]
        nxt = torch.zeros_like(a)
        nxt[:-1] = a[1:]
        grad = _scan(nxt.flip(0), e.flip(0)).flip(0)
        prev = torch.zeros_like(h)
        prev[1:] = h[:-1]
        if h0 is not None:
            prev[0] = h0
        if reset is not None:
            prev = torch.where(reset[..., None], torch.zeros((), device=DEV), prev)
        dzv = torch.cat((grad * (prev - v) * f * w, grad * w), -1).to(dt)
        res = {"out": out, "h_n": h_n, "dzv": dzv}
        if h0 is not None:
            res["dh0"] = a[0] * grad[0]
        return res


def _top(x, k):
    """Ids of the k largest of each row, the lowest id first among equals: one selection over whole
    numbers that hold the value's order above and the id below."""
    bits = (x + 0.0).view(torch.int32)
    order = bits ^ ((bits >> 31) & 0x7FFFFFFF)
    v = x.shape[1]
    key = (order.long() << 32) | torch.arange(v - 1, -1, -1, device=DEV)
    return v - 1 - (torch.topk(key, k, dim=1).values & 0xFFFFFFFF)


def _run_score(s):
    logits, tokens, top = s["logits"], s["tokens"], s["top"]
    train = s["call"] == "train"
    if own:
        import prlstm_amd
        r = prlstm_amd.token_logprobs(logits, tokens, top=top)
        res = {"logp": r.logp.detach(), "entropy": r.entropy.detach()}
        if top:
            res.update(top_logp=r.top_logp.detach(), top_ids=r.top_ids)
        if train:
            pairs = [(o, d) for o, d in ((r.logp, s["dlogp"]), (r.entropy, s["dent"]), (r.top_logp, s["dtop"]))
                     if d is not None]
            res["dlogits"], = torch.autograd.grad([o for o, _ in pairs], logits, [d for _, d in pairs])
        return res
    with torch.no_grad():
        zero = torch.zeros((), device=DEV)
        x = logits.float()
        m = x.amax(1, keepdim=True)
        empty = m == -math.inf  # every token is masked: probability 0 for each
        d = x - torch.where(empty, zero, m)
        e = torch.exp(d)
        total = e.sum(1, keepdim=True)
        lse = (m + torch.log(total))
        ent = torch.log(total) - torch.where(e == 0, zero, e * d).sum(1, keepdim=True) / total
        ent = torch.where(empty, zero, ent)
        there = (tokens >= 0)[:, None]
        at = tokens.clamp_min(0)[:, None]
        gain = lambda ids: torch.where(empty, torch.full_like(zero, -math.inf), x.gather(1, ids) - lse)  # noqa: E731
        res = {"logp": torch.where(there, gain(at), zero)[:, 0], "entropy": ent[:, 0]}
        if top:
            res["top_ids"] = _top(x, top)
            res["top_logp"] = gain(res["top_ids"])
        if not train:
            return res
        dlogp = torch.where(there, s["dlogp"][:, None], zero)
        pull = dlogp if s["dtop"] is None else dlogp + s["dtop"].sum(1, keepdim=True)
        logp = x - lse
        p = torch.exp(logp)
        if s["dent"] is not None:
            pull = pull + s["dent"][:, None] * (logp + ent)
        grad = torch.where(p == 0, zero, -p * pull)
        grad.scatter_add_(1, at, dlogp)
        if s["dtop"] is not None:
            grad.scatter_add_(1, res["top_ids"], s["dtop"])
        res["dlogits"] = torch.where(empty, zero, grad).to(logits.dtype)
        return res


def work(case):
    e, train = BYTES[case["dtype"]], case["call"] == "train"
    if case["op"] == "embed":
        n, v, d = case["N"], case["V"], case["D"]
        size = n * (4 if case["ids"] == "int32" else 8) + (min(n, v) + n) * d * e
        if train:
            size += (n + v) * d * e
        return {"bytes": size, "flops": n * d * (3 if train else 1)}
    if case["op"] == "gated":
        n, states = case["T"] * case["B"] * case["H"], case["B"] * case["H"] * 4
        size = 3 * n * e + states * (2 if case["h0"] else 1) + (case["T"] * case["B"] if case["reset"] else 0)
        if train:
            size += 3 * n * e + states * (2 if case["h0"] else 1)
        return {"bytes": size, "flops": n * (24 if train else 9)}
    n, v = case["N"], case["V"]
    size = n * v * e + n * (16 + 12 * case["top"])
    if train:
        size += n * v * e + n * (8 if case["entropy"] else 4)
    return {"bytes": size, "flops": n * v * (10 if train else 5)}


def exact(case, seed):
    """What run() returns, in 64 bits, step by step from the definitions."""
    s = prepare(case, seed)
    with torch.no_grad():
        return {"embed": _exact_embed, "gated": _exact_gated, "score": _exact_score}[case["op"]](s)


def _exact_embed(s):
    ids, w = s["ids"].long(), s["weight"].double()
    out = torch.zeros(ids.shape[0], w.shape[1], dtype=torch.float64, device=DEV)
    at = (ids >= 0).nonzero()[:, 0]
    out[at] = s["scale"] * w[ids[at]]
    if s["call"] == "infer":
        return {"out": out}
    dw = torch.zeros_like(w)
    dw.index_add_(0, ids[at], s["dout"][at].double())
    return {"out": out, "dweight": dw * s["scale"]}


def _exact_gated(s):
    step = s["call"] == "step"
    zv = s["zv"].detach().double()
    zv = zv[None] if step else zv
    t, b, n = zv.shape[0], zv.shape[1], zv.shape[2] // 2
    keep = torch.ones(t, b, 1, dtype=torch.float64, device=DEV)
    if s["reset"] is not None:
        keep -= s["reset"].reshape(t, b, 1).double()
    f = 1 / (1 + torch.exp(-zv[..., :n]))
    w = 1 / (1 + torch.exp(zv[..., :n]))
    v = zv[..., n:]
    hs = torch.zeros(t + 1, b, n, dtype=torch.float64, device=DEV)
    if s["h0"] is not None:
        hs[0] = s["h0"].double()
    for k in range(t):
        hs[k + 1] = f[k] * keep[k] * hs[k] + w[k] * v[k]
    if step:
        return {"out": hs[1], "h_n": hs[1]}
    res = {"out": hs[1:], "h_n": hs[-1]}
    if s["call"] == "infer":
        return res
    dzv, grad = torch.empty_like(zv), s["dh_n"].double()
    for k in range(t - 1, -1, -1):
        grad = grad + s["dout"][k].double()
        dzv[k, :, :n] = grad * (hs[k] * keep[k] - v[k]) * f[k] * w[k]
        dzv[k, :, n:] = grad * w[k]
        grad = grad * f[k] * keep[k]
    res["dzv"] = dzv
    if s["h0"] is not None:
        res["dh0"] = grad
    return res


def _exact_score(s):
    x, tokens, top = s["logits"].detach().double(), s["tokens"], s["top"]
    empty = torch.isinf(x).all(1)
    lse = torch.logsumexp(x, 1)
    logp = x - lse[:, None]
    logp[empty] = -math.inf
    p = torch.exp(logp)
    ent = -torch.nan_to_num(p * logp, nan=0.0).sum(1)
    rows, there = torch.arange(len(tokens), device=DEV), tokens >= 0
    mine = torch.zeros(len(tokens), dtype=torch.float64, device=DEV)
    mine[there] = logp[rows[there], tokens[there]]
    res = {"logp": mine, "entropy": ent}
    if top:
        best = torch.topk(logp, top, dim=1)
        res["top_logp"], res["top_ids"] = best.values, None
    if s["call"] != "train":
        return res
    g = torch.zeros_like(x)  # of log p, then of the logits
    g[rows[there], tokens[there]] = s["dlogp"].double()[there]
    if top:
        # between equal logits the choice of the lowest id decides where a gradient goes
        order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
        g.scatter_add_(1, order, s["dtop"].double())
    pull = g.sum(1, keepdim=True)
    g -= p * pull
    if s["dent"] is not None:
        g -= s["dent"].double()[:, None] * torch.nan_to_num(p * (logp + ent[:, None]), nan=0.0)
    g[empty] = 0
    res["dlogits"] = g
    return res
