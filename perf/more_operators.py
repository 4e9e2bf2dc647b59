"""Operators of a language model's selective layers and of its loss, for timing and for comparing
outputs: the short causal convolution and the selective scan (training, prompts, and one token at a
time), and the cross entropy of a projection on the vocabulary (scoring, and with its gradients).

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
PAD = -1  # target of a position that is not scored


def _conv(name, call, t, b, d, k, dtype, order="time", reset=False, state=False):
    """A convolution of k taps.  order: which of time and batch comes first in memory.  reset:
    sequences of several documents.  state: inputs of the call before."""
    return {"name": name, "op": "conv", "call": call, "T": t, "B": b, "D": d, "K": k, "dtype": dtype, "order": order,
            "reset": reset, "state": state}


def _scan(name, call, t, b, d, n, dtype, order="time", reset=False, state=False, gate=True):
    """A scan of n states per channel; order, reset and state as above.  gate: the output is gated."""
    return {"name": name, "op": "scan", "call": call, "T": t, "B": b, "D": d, "N": n, "dtype": dtype, "order": order,
            "reset": reset, "state": state, "gate": gate}


def _loss(name, call, n, v, d, dtype, bias=False, pad=False):
    """n rows of width d against v tokens.  bias: of the tokens, the last ones ruled out by -inf.
    pad: a share of the rows is not scored."""
    return {"name": name, "op": "loss", "call": call, "N": n, "V": v, "D": d, "dtype": dtype, "bias": bias, "pad": pad}


def listed():
    return [
        # one token of 32 served streams, each with its last inputs
        _conv("conv_serve", "step", 1, 32, 1024, 4, "bf16", state=True),
        # a ragged batch of packed documents with an odd width, after a window before it
        _conv("conv_train_ragged", "train", 1501, 3, 650, 3, "fp32", order="batch", reset=True, state=True),
        # the long-sequence batch (4096 steps of 16)
        _conv("conv_train_long", "train", 4096, 16, 1024, 4, "bf16"),
        # one token of 32 served streams, each with its states
        _scan("scan_serve", "step", 1, 32, 1024, 16, "bf16", state=True),
        # one long prompt that continues another
        _scan("scan_prompt", "infer", 16383, 1, 1024, 16, "fp16", state=True),
        # the ragged batch of packed documents, without a gate
        _scan("scan_train_ragged", "train", 1501, 3, 650, 10, "fp32", order="batch", reset=True, state=True,
              gate=False),
        # the headline batch (256 steps of 32 sequences)
        _scan("scan_train", "train", 256, 32, 512, 16, "bf16"),
        # the long-sequence batch
        _scan("scan_train_long", "train", 4096, 16, 1024, 16, "bf16"),
        # the last tokens of eight served streams, scored
        _loss("loss_score", "infer", 8, 32768, 512, "bf16"),
        # a ragged padded batch in full precision, with a bias
        _loss("loss_train_ragged", "train", 700, 10007, 650, "fp32", bias=True, pad=True),
        # the headline batch
        _loss("loss_train", "train", 8192, 32768, 512, "bf16", bias=True),
        # as many rows with a large vocabulary and a wide layer: the largest pass
        _loss("loss_train_large", "train", 8192, 131072, 1024, "bf16"),
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
    op = rng.choice(["conv", "scan", "loss"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    flag = lambda p: rng.random() < p  # noqa: E731
    if op == "loss":
        c = _loss(None, rng.choice(["infer", "train", "train"]), _log_int(rng, 1, 8192, True),
                  _log_int(rng, 64, 131072, odd), _log_int(rng, 16, 2048, odd), dtype, flag(0.4), flag(0.3))
        top, shrink = work(listed()[11]), ("N", "V")
    else:
        call = rng.choice(["step", "infer", "train", "train"])
        sizes = (1 if call == "step" else _log_int(rng, 1, 16384, True), _log_int(rng, 1, 64, odd),
                 _log_int(rng, 16, 2048, odd))
        rest = (dtype, rng.choice(["time", "batch"]), flag(0.4), call == "step" or flag(0.4))
        if op == "conv":
            c = _conv(None, call, *sizes, rng.choice([2, 3, 4, 4]), *rest)
            top = work(listed()[2])
        else:
            c = _scan(None, call, *sizes, rng.choice([8, 16, 16, 32, rng.randint(1, 64)]), *rest, flag(0.6))
            top = work(listed()[7])
        shrink = ("T", "B")
    del c["name"]
    while work(c)["bytes"] > 0.9 * top["bytes"] or work(c)["flops"] > 0.9 * top["flops"]:
        k = max(shrink, key=lambda s: c[s])
        c[k] = max(1, c[k] * 3 // 4)
    return c


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    uniform = lambda *s: torch.rand(*s, device=DEV, generator=g)  # noqa: E731
    dt, train = DTYPES[case["dtype"]], case["call"] == "train"
    s = {"op": case["op"], "call": case["call"]}
    leaf = lambda x: x.requires_grad_(train)  # noqa: E731
    if case["op"] == "loss":
        n, v, d = case["N"], case["V"], case["D"]
        # ids as text has them: the k-th most frequent token with a share of about 1/k
        ids = (torch.exp(uniform(n).double() * math.log(v + 1.0)) - 1).long()
        barred = v // 100 if case["bias"] else 0  # of a vocabulary that is filled up to a round size
        ids.clamp_(0, v - 1 - barred)
        w = 1.5 * d ** -0.5 * rand(v, d)
        x = rand(n, d) + 4 * uniform(n, 1) * w[ids]  # rows of any confidence in their token
        if case["pad"]:
            ids[uniform(n) < 0.2] = PAD
        s["targets"] = ids
        s["x"], s["weight"] = leaf(x.to(dt)), leaf(w.to(dt))
        s["bias"] = None
        if case["bias"]:
            s["bias"] = 0.5 * rand(v)
            s["bias"][v - barred:] = -math.inf
            leaf(s["bias"])
        if train:
            s["dloss"] = uniform(n) / n
        return s
    t, b, d = case["T"], case["B"], case["D"]
    step = case["call"] == "step"
    shape = (t, b) if case["order"] == "time" else (b, t)

    def stream(x):
        """As [T, B, ...] (one step: [B, ...])."""
        x = x if case["order"] == "time" else x.transpose(0, 1)
        return x[0] if step else x

    s["x"] = leaf(stream(rand(*shape, d).to(dt)))
    s["reset"] = stream(uniform(*shape) < 1 / 300) if case["reset"] else None
    if train:
        s["dout"] = stream(rand(*shape, d).to(dt))
    if case["op"] == "conv":
        k = case["K"]
        s["weight"] = leaf((2 * uniform(d, k) - 1) * k ** -0.5)
        s["bias"] = leaf(0.2 * rand(d))
        s["state"] = leaf(rand(b, k - 1, d).to(dt)) if case["state"] else None
        return s
    n = case["N"]
    s["delta"] = leaf(stream((0.5 * rand(*shape, d)).to(dt)))
    # b and c are columns of one projection, behind those that delta is made of
    rank = max(1, d // 16)
    proj = stream(rand(*shape, rank + 2 * n).to(dt))
    s["b"], s["c"] = leaf(proj[..., rank:rank + n]), leaf(proj[..., rank + n:])
    s["a"] = leaf(-torch.arange(1, n + 1, device=DEV).float() * torch.exp(0.1 * rand(d, n)))
    first = torch.exp(math.log(0.001) + uniform(d) * math.log(100.0))  # steps of 0.001 to 0.1
    s["delta_bias"] = leaf(first + torch.log(-torch.expm1(-first)))
    s["d"] = leaf(1 + 0.1 * rand(d))
    s["z"] = leaf(stream(rand(*shape, d).to(dt))) if case["gate"] else None
    s["h0"] = leaf(0.3 * rand(b, d, n)) if case["state"] else None
    if train:
        s["dh_n"] = 0.3 * rand(b, d, n)
    return s


def run(state):
    return {"conv": _run_conv, "scan": _run_scan, "loss": _run_loss}[state["op"]](state)


def _silu_slope(u):
    """The derivative of u sigmoid(u)."""
    s = torch.sigmoid(u)
    return s + u * s * (1 - s)


def _run_conv(s):
    x, weight, bias, state, reset = (s[k] for k in ("x", "weight", "bias", "state", "reset"))
    if own:
        import prlstm_amd
        if s["call"] == "step":
            y, after = prlstm_amd.causal_conv_step(x, state, weight, bias, reset=reset)
            return {"y": y, "state": after}
        y, after = prlstm_amd.causal_conv(x, weight, bias, state=state, reset=reset)
        if s["call"] == "infer":
            return {"y": y, "state": after}
        names = [k for k in ("x", "weight", "bias", "state") if s[k] is not None]
        grads = torch.autograd.grad(y, [s[k] for k in names], s["dout"])
        return {"y": y.detach(), "state_n": after.detach(), **{"d" + k: g for k, g in zip(names, grads)}}
    with torch.no_grad():
        dt, k = x.dtype, weight.shape[1]
        if s["call"] == "step":
            x, reset = x[None], None if reset is None else reset[None]
        t, b, d = x.shape
        old = torch.zeros(b, k - 1, d, dtype=dt, device=DEV) if state is None else state
        full = torch.cat((old.transpose(0, 1), x)).float()  # step i of x is row i + k - 1
        there = _same_sequence(t, b, k, reset)
        u = bias.expand(t, b, d).float()
        for j in range(k):
            u = u + weight[:, j] * (full[j:j + t] * there[j])
        y = (u * torch.sigmoid(u)).to(dt)
        after = (full[t:] * _last_sequence(t, b, k, reset)).to(dt).transpose(0, 1)
        if s["call"] == "step":
            return {"y": y[0], "state": after}
        if s["call"] == "infer":
            return {"y": y, "state": after}
        du = s["dout"].float() * _silu_slope(u)
        dfull = torch.zeros_like(full)
        dw = torch.empty_like(weight)
        for j in range(k):
            dfull[j:j + t] += weight[:, j] * du * there[j]
            dw[:, j] = (du * full[j:j + t] * there[j]).sum((0, 1))
        res = {"y": y, "state_n": after, "dx": dfull[k - 1:].to(dt), "dweight": dw, "dbias": du.sum((0, 1))}
        if state is not None:
            res["dstate"] = dfull[:k - 1].transpose(0, 1).to(dt)
        return res


def _same_sequence(t, b, k, reset):
    """[k][t, b, 1]: 1 where the input of tap j (k-1-j steps before) is of the step's own sequence."""
    there = [torch.ones(t, b, 1, device=DEV) for _ in range(k)]
    if reset is not None:
        begun = torch.cumsum(reset.long(), 0)
        begun = torch.cat((torch.zeros(k - 1, b, dtype=torch.long, device=DEV), begun))
        for j in range(k):
            there[j] = (begun[j:j + t] == begun[k - 1:]).float()[..., None]
    return there


def _last_sequence(t, b, k, reset):
    """[k-1, b, 1]: 1 where the input that the state keeps is of the last step's sequence."""
    if reset is None:
        return torch.ones(k - 1, b, 1, device=DEV)
    begun = torch.cat((torch.zeros(k - 1, b, dtype=torch.long, device=DEV), torch.cumsum(reset.long(), 0)))
    return (begun[t:] == begun[-1]).float()[..., None]


def _maps(a, h):
    """h_t = a_t h_{t-1} + h'_t for every t, h_{-1} = 0, in log2(T) passes: after the pass of distance
    k, (a_t, h_t) is the map of the steps t-2k+1 .. t.  Overwrites a and h."""
    k, t = 1, a.shape[0]
    while k < t:
        h[k:] += a[k:] * h[:-k]
        a[k:] = a[k:] * a[:-k]
        k *= 2
    return h


def _run_scan(s):
    x, reset, h0, z = s["x"], s["reset"], s["h0"], s["z"]
    if own:
        import prlstm_amd
        args = [s[k] for k in ("x", "delta", "a", "b", "c")]
        rest = dict(d=s["d"], z=z, delta_bias=s["delta_bias"], reset=reset)
        if s["call"] == "step":
            y, h = prlstm_amd.selective_scan_step(*args, h0, **rest)
            return {"y": y, "h": h}
        y, h = prlstm_amd.selective_scan(*args, h0=h0, **rest)
        if s["call"] == "infer":
            return {"y": y, "h": h}
        names = [k for k in ("x", "delta", "a", "b", "c", "d", "delta_bias", "z", "h0") if s[k] is not None]
        grads = torch.autograd.grad((y, h), [s[k] for k in names], (s["dout"], s["dh_n"]))
        return {"y": y.detach(), "h": h.detach(), **{"grad_" + k: g for k, g in zip(names, grads)}}
    with torch.no_grad():
        lift = (lambda v: None if v is None else v[None]) if s["call"] == "step" else (lambda v: v)
        x, delta, b, c, z, reset = (lift(s[k]) for k in ("x", "delta", "b", "c", "z", "reset"))
        dtype, a, skip = x.dtype, s["a"], s["d"]
        t, nb, d = x.shape
        n = a.shape[1]
        u = delta.float() + s["delta_bias"]
        step = u.clamp_min(0) + torch.log1p(torch.exp(-u.abs()))
        some = max(1, (1 << 26) // (nb * d * n))  # steps whose states are held at once

        def decay(i, j):
            """exp(step a) of the steps i..j-1, 0 at a reset."""
            f = torch.exp(step[i:j, ..., None] * a)
            return f if reset is None else torch.where(reset[i:j, :, None, None], torch.zeros((), device=DEV), f)

        def states(i, j, h):
            f = decay(i, j)
            e = (step[i:j] * x[i:j].float())[..., None] * b[i:j, :, None, :].float()
            e[0] += f[0] * h
            return f, _maps(f.clone(), e)

        h = torch.zeros(nb, d, n, device=DEV) if h0 is None else h0.detach()
        before, ys = [], []
        for i in range(0, t, some):
            before.append(h)
            _, hs = states(i, min(t, i + some), h)
            ys.append((hs * c[i:i + some, :, None, :].float()).sum(-1))
            h = hs[-1].clone()
        y0 = torch.cat(ys) + skip * x.float()  # before the gate
        y = (y0 if z is None else y0 * z.float() * torch.sigmoid(z.float())).to(dtype)
        if s["call"] != "train":
            return {"y": y[0] if s["call"] == "step" else y, "h": h}
        h_n, dout = h, s["dout"].float()
        dy = dout if z is None else dout * z.float() * torch.sigmoid(z.float())
        back = s["dh_n"]  # the gradient of the state behind the steps that are left
        da, db, dc = torch.zeros_like(a), [], []
        dstep, dx = torch.empty_like(step), torch.empty_like(step)
        for i, h in reversed(list(zip(range(0, t, some), before))):
            j = min(t, i + some)
            f, hs = states(i, j, h)
            dc.append((hs * dy[i:j, ..., None]).sum(2))
            # G_t = c_t dy_t + f_{t+1} G_{t+1}, the same recurrence from the last step to the first
            e = c[i:j, :, None, :].float() * dy[i:j, ..., None]
            e[-1] += back
            nxt = torch.zeros_like(f)
            nxt[:-1] = f[1:]
            grad = _maps(nxt.flip(0), e.flip(0)).flip(0)
            back = f[0] * grad[0]
            prev = torch.cat((h[None], hs[:-1]))
            p = f * grad * prev
            da += (p * step[i:j, ..., None]).sum((0, 1))
            gb = (grad * b[i:j, :, None, :].float()).sum(-1)
            dstep[i:j] = (p * a).sum(-1) + gb * x[i:j].float()
            dx[i:j] = gb * step[i:j]
            db.append((grad * (step[i:j] * x[i:j].float())[..., None]).sum(2))
        ddelta = dstep * torch.sigmoid(u)
        res = {"y": y, "h": h_n, "grad_x": (dx + skip * dy).to(dtype), "grad_delta": ddelta.to(dtype), "grad_a": da,
               "grad_b": torch.cat(db[::-1]).to(dtype), "grad_c": torch.cat(dc[::-1]).to(dtype),
               "grad_d": (dy * x.float()).sum((0, 1)), "grad_delta_bias": ddelta.sum((0, 1))}
        if z is not None:
            res["grad_z"] = (dout * y0 * _silu_slope(z.float())).to(dtype)
        if h0 is not None:
            res["grad_h0"] = back
        return res


def _run_loss(s):
    x, weight, bias, targets = s["x"], s["weight"], s["bias"], s["targets"]
    if own:
        import prlstm_amd
        loss = prlstm_amd.linear_cross_entropy(x, weight, targets, bias=bias)
        if s["call"] == "infer":
            return {"loss": loss}
        names = [k for k in ("x", "weight", "bias") if s[k] is not None]
        grads = torch.autograd.grad(loss, [s[k] for k in names], s["dloss"])
        return {"loss": loss.detach(), **{"d" + k: g for k, g in zip(names, grads)}}
    with torch.no_grad():
        dt, w = x.dtype, weight.float()
        logits = x.float() @ w.t()
        if bias is not None:
            logits += bias
        m = logits.amax(1, keepdim=True)
        logits -= m
        there, at = targets >= 0, targets.clamp_min(0)[:, None]
        mine = logits.gather(1, at)[:, 0]
        p = torch.exp_(logits)
        total = p.sum(1)
        loss = torch.where(there, torch.log(total) - mine, torch.zeros((), device=DEV))
        if s["call"] == "infer":
            return {"loss": loss}
        g = torch.where(there, s["dloss"], torch.zeros((), device=DEV))
        p *= (g / total)[:, None]
        p.scatter_add_(1, at, -g[:, None])
        res = {"loss": loss, "dx": (p @ w).to(dt), "dweight": (p.t() @ x.float()).to(dt)}
        if bias is not None:
            res["dbias"] = p.sum(0)
        return res


def work(case):
    e, train = BYTES[case["dtype"]], case["call"] == "train"
    if case["op"] == "loss":
        n, v, d = case["N"], case["V"], case["D"]
        size = (n + v) * d * e + n * 12 + (v * 4 if case["bias"] else 0)
        if train:
            size += (n + v) * d * e + n * 4 + (v * 4 if case["bias"] else 0)
        return {"bytes": size, "flops": 2 * n * v * d * (3 if train else 1) + n * v * (5 if train else 3)}
    tb, d = case["T"] * case["B"], case["D"]
    stream = tb * d * e
    size = tb if case["reset"] else 0
    if case["op"] == "conv":
        k = case["K"]
        state = case["B"] * (k - 1) * d * e
        size += 2 * stream + d * (k + 1) * 4 + state * (2 if case["state"] else 1)
        if train:
            size += 2 * stream + d * (k + 1) * 4 + (state if case["state"] else 0)
        return {"bytes": size, "flops": tb * d * ((6 * k + 20) if train else (2 * k + 5))}
    n = case["N"]
    states = case["B"] * d * n * 4
    size += (3 + case["gate"]) * stream + 2 * tb * n * e + d * (n + 2) * 4 + states * (2 if case["state"] else 1)
    if train:
        size += (3 + case["gate"]) * stream + 2 * tb * n * e + d * (n + 2) * 4 + states * (2 if case["state"] else 1)
    return {"bytes": size, "flops": tb * d * (n * (24 if train else 7) + (40 if train else 12))}


def exact(case, seed):
    """What run() returns, in 64 bits, step by step from the definitions."""
    s = prepare(case, seed)
    with torch.no_grad():
        return {"conv": _exact_conv, "scan": _exact_scan, "loss": _exact_loss}[case["op"]](s)


def _exact_conv(s):
    one = s["call"] == "step"
    x = s["x"].detach().double()
    x = x[None] if one else x
    t, b, d = x.shape
    w, bias = s["weight"].double(), s["bias"].double()
    k = w.shape[1]
    reset = torch.zeros(t, b, dtype=torch.bool, device=DEV) if s["reset"] is None else s["reset"].reshape(t, b)
    window = torch.zeros(k, b, d, dtype=torch.float64, device=DEV)  # the inputs of the last k steps
    if s["state"] is not None:
        window[1:] = s["state"].detach().double().transpose(0, 1)
    us, windows = [], []
    for i in range(t):
        window = torch.cat((window[1:], x[i:i + 1]))
        window[:-1, reset[i]] = 0
        windows.append(window)
        us.append((w.t()[:, None, :] * window).sum(0) + bias)
    u = torch.stack(us)
    sig = 1 / (1 + torch.exp(-u))
    y, after = u * sig, window[1:].transpose(0, 1)
    if one:
        return {"y": y[0], "state": after}
    if s["call"] == "infer":
        return {"y": y, "state": after}
    du = s["dout"].double() * sig * (1 + u * (1 - sig))
    dw, dwindow = torch.zeros_like(w), torch.zeros(k, b, d, dtype=torch.float64, device=DEV)
    dx = torch.empty_like(x)
    for i in range(t - 1, -1, -1):
        dwindow = dwindow + w.t()[:, None, :] * du[i]
        dw += (windows[i] * du[i]).sum(1).t()
        dx[i] = dwindow[-1]
        dwindow[:-1, reset[i]] = 0
        dwindow = torch.cat((torch.zeros_like(dwindow[:1]), dwindow[:-1]))
    res = {"y": y, "state_n": after, "dx": dx, "dweight": dw, "dbias": du.sum((0, 1))}
    if s["state"] is not None:
        res["dstate"] = dwindow[1:].transpose(0, 1)
    return res


def _exact_scan(s):
    one = s["call"] == "step"
    wide = lambda v: None if v is None else (v.detach().double()[None] if one else v.detach().double())  # noqa: E731
    x, delta, b, c, z = (wide(s[k]) for k in ("x", "delta", "b", "c", "z"))
    a, skip, bias = s["a"].detach().double(), s["d"].detach().double(), s["delta_bias"].detach().double()
    t, nb, d = x.shape
    n = a.shape[1]
    keep = torch.ones(t, nb, 1, 1, dtype=torch.float64, device=DEV)
    if s["reset"] is not None:
        keep -= s["reset"].reshape(t, nb, 1, 1).double()
    u = delta + bias
    dt = torch.logaddexp(u, torch.zeros_like(u))
    hs = torch.zeros(t + 1, nb, d, n, dtype=torch.float64, device=DEV)
    if s["h0"] is not None:
        hs[0] = s["h0"].detach().double()
    y0 = torch.empty_like(x)
    for i in range(t):
        hs[i + 1] = torch.exp(dt[i, ..., None] * a) * keep[i] * hs[i] + (dt[i] * x[i])[..., None] * b[i, :, None, :]
        y0[i] = torch.matmul(hs[i + 1], c[i, ..., None])[..., 0] + skip * x[i]
    sig = None if z is None else 1 / (1 + torch.exp(-z))
    y = y0 if z is None else y0 * z * sig
    if s["call"] != "train":
        return {"y": y[0] if one else y, "h": hs[-1]}
    dout, grad = s["dout"].double(), s["dh_n"].double()
    dy = dout if z is None else dout * z * sig
    da, dx, ddt, db, dc = torch.zeros_like(a), skip * dy, torch.empty_like(x), torch.empty_like(b), torch.empty_like(c)
    for i in range(t - 1, -1, -1):
        f = torch.exp(dt[i, ..., None] * a) * keep[i]
        grad = grad + c[i, :, None, :] * dy[i, ..., None]
        dc[i] = torch.matmul(dy[i, :, None, :], hs[i + 1])[:, 0]
        through = grad * f * hs[i]
        da += (through * dt[i, ..., None]).sum(0)
        into = torch.matmul(grad, b[i, ..., None])[..., 0]
        dx[i] += into * dt[i]
        ddt[i] = into * x[i] + (through * a).sum(-1)
        db[i] = torch.matmul((dt[i] * x[i])[:, None, :], grad)[:, 0]
        grad = grad * f
    ddelta = ddt / (1 + torch.exp(-u))
    res = {"y": y, "h": hs[-1], "grad_x": dx, "grad_delta": ddelta, "grad_a": da, "grad_b": db, "grad_c": dc,
           "grad_d": (dy * x).sum((0, 1)), "grad_delta_bias": ddelta.sum((0, 1))}
    if z is not None:
        res["grad_z"] = dout * y0 * sig * (1 + z * (1 - sig))
    if s["h0"] is not None:
        res["grad_h0"] = grad
    return res


def _exact_loss(s):
    x, w, targets = s["x"].detach().double(), s["weight"].detach().double(), s["targets"]
    logits = torch.mm(x, w.t())
    if s["bias"] is not None:
        logits += s["bias"].detach().double()
    lse = torch.logsumexp(logits, 1)
    scored = (targets >= 0).nonzero()[:, 0]
    loss = torch.zeros(len(targets), dtype=torch.float64, device=DEV)
    loss[scored] = lse[scored] - logits[scored, targets[scored]]
    if s["call"] == "infer":
        return {"loss": loss}
    g = torch.zeros(len(targets), dtype=torch.float64, device=DEV)
    g[scored] = s["dloss"].double()[scored]
    dl = logits.sub_(lse[:, None]).exp_().mul_(g[:, None])
    dl[scored, targets[scored]] -= g[scored]
    res = {"loss": loss, "dx": torch.mm(dl, w), "dweight": torch.mm(dl.t(), x)}
    if s["bias"] is not None:
        res["dbias"] = dl.sum(0)
    return res
