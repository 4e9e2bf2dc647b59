"""The selective layers' formulas in 64 bits, step by step, with the size of what each result sums.

``scan`` and ``conv`` return the results and the gradients; given the absolute values of everything
that enters linearly (``magnitude=True``), they return the sum of the absolute values of each
result's terms, against which a result's rounding errors are measured.
"""

import torch


def silu(z):
    return z * torch.sigmoid(z)


def silu_slope(z, magnitude=False):
    """The derivative; with `magnitude`, of its two terms' sizes (they cancel near z = -1.28, so that an
    error of either counts in full there)."""
    s = torch.sigmoid(z)
    return s + (z.abs() if magnitude else z) * s * (1 - s)


def scan(x, delta, a, b, c, d=None, z=None, delta_bias=None, h0=None, reset=None, softplus=True, dout=None, dh_n=None,
         magnitude=False):
    """A dict of y, h and the gradients (where dout or dh_n is given)."""
    up = lambda t: None if t is None else t.detach().double().cpu()  # noqa: E731
    x, delta, a, b, c, d, z, delta_bias, h0, dout, dh_n = map(up, (x, delta, a, b, c, d, z, delta_bias, h0, dout, dh_n))
    T, B, D = x.shape
    N = a.shape[1]
    u = delta if delta_bias is None else delta + delta_bias
    dt = torch.logaddexp(u, torch.zeros_like(u)) if softplus else u
    sig = torch.sigmoid(u) if softplus else torch.ones_like(u)
    gate = None if z is None else silu(z)
    slope = None if z is None else silu_slope(z, magnitude)
    factor = a
    if magnitude:
        ab = lambda t: None if t is None else t.abs()  # noqa: E731
        x, b, c, d, h0, dout, dh_n, gate, factor = map(ab, (x, b, c, d, h0, dout, dh_n, gate, factor))
    keep = torch.ones(T, B, dtype=torch.bool) if reset is None else ~reset.cpu().bool()
    h = torch.zeros(B, D, N, dtype=torch.float64) if h0 is None else h0
    before, hs, f = [], [], []
    for t in range(T):
        h = torch.where(keep[t, :, None, None], h, torch.zeros_like(h))
        before.append(h)
        f.append(torch.exp(dt[t, ..., None] * a))
        h = f[t] * h + (dt[t] * x[t])[..., None] * b[t, :, None, :]
        hs.append(h)
    skip = torch.zeros(D, dtype=torch.float64) if d is None else d
    y0 = torch.stack([(hs[t] * c[t, :, None, :]).sum(-1) + skip * x[t] for t in range(T)]) if T else x.clone()
    res = {"y": y0 if gate is None else y0 * gate, "h": h}
    if dout is None and dh_n is None:
        return res
    dout = torch.zeros_like(x) if dout is None else dout
    G = torch.zeros_like(h) if dh_n is None else dh_n
    dy = dout if gate is None else dout * gate
    dx, ddt, db, dc, da = skip * dy, torch.empty_like(x), torch.empty_like(b), torch.empty_like(c), torch.zeros_like(a)
    for t in range(T - 1, -1, -1):
        G = G + c[t, :, None, :] * dy[t, ..., None]
        dc[t] = (hs[t] * dy[t, ..., None]).sum(1)
        db[t] = (G * (dt[t] * x[t])[..., None]).sum(1)
        gb = (G * b[t, :, None, :]).sum(-1)
        p = G * f[t] * before[t]
        da += (p * dt[t, ..., None]).sum(0)
        dx[t] += gb * dt[t]
        ddt[t] = gb * x[t] + (p * factor).sum(-1)
        G = torch.where(keep[t, :, None, None], G * f[t], torch.zeros_like(G))
    ddelta = ddt * sig
    res.update(x=dx, delta=ddelta, a=da, b=db, c=dc, h0=G, delta_bias=ddelta.sum((0, 1)), d=(dy * x).sum((0, 1)))
    if gate is not None:
        res["z"] = dout * y0 * slope
    return res


def conv(x, weight, bias=None, state=None, reset=None, act=True, dout=None, dstate_n=None, magnitude=False):
    """A dict of y, state_n and the gradients (where dout or dstate_n is given)."""
    up = lambda t: None if t is None else t.detach().double().cpu()  # noqa: E731
    x, weight, bias, state, dout, dstate_n = map(up, (x, weight, bias, state, dout, dstate_n))
    T, B, D = x.shape
    K = weight.shape[1]
    bias = torch.zeros(D, dtype=torch.float64) if bias is None else bias
    full = torch.cat((torch.zeros(K - 1, B, D, dtype=torch.float64) if state is None else state.transpose(0, 1), x))
    # begun[i]: which sequence row i of full belongs to; row t + K - 1 is step t
    begun = torch.zeros(T + K - 1, B, dtype=torch.long)
    if reset is not None and T:
        begun[K - 1:] = reset.cpu().long().cumsum(0)

    def tap(t, j):
        """Step t's input at tap j, 0 where it is of another sequence."""
        return torch.where((begun[t + j] == begun[t + K - 1])[:, None], full[t + j], torch.zeros_like(full[0]))

    u = torch.stack([bias + sum(weight[:, j] * tap(t, j) for j in range(K)) for t in range(T)]) if T else x.clone()
    size = u
    if magnitude:
        weight, bias, full = weight.abs(), bias.abs(), full.abs()
        size = torch.stack([bias + sum(weight[:, j] * tap(t, j) for j in range(K)) for t in range(T)]) if T else x
    y = (torch.sigmoid(u) * size if act else size) if magnitude else (silu(u) if act else u)
    last = begun[T + K - 2] if T + K > 1 else None
    state_n = [torch.where((begun[T + j] == last)[:, None], full[T + j], torch.zeros_like(full[0]))
               for j in range(K - 1)]
    res = {"y": y, "state_n": torch.stack(state_n, 1) if K > 1 else torch.zeros(B, 0, D, dtype=torch.float64)}
    if dout is None and dstate_n is None:
        return res
    dout = torch.zeros_like(x) if dout is None else dout
    slope = silu_slope(u, magnitude) if act else torch.ones_like(u)
    if magnitude:
        dout = dout.abs()
        dstate_n = None if dstate_n is None else dstate_n.abs()
    du = dout * slope
    dfull, dw = torch.zeros_like(full), torch.zeros_like(weight)
    for t in range(T):
        for j in range(K):
            same = (begun[t + j] == begun[t + K - 1])[:, None]
            dfull[t + j] += torch.where(same, weight[:, j] * du[t], torch.zeros_like(du[t]))
            dw[:, j] += (du[t] * tap(t, j)).sum(0)
    if dstate_n is not None:
        for j in range(K - 1):
            dfull[T + j] += torch.where((begun[T + j] == last)[:, None], dstate_n[:, j], torch.zeros_like(dfull[0]))
    res.update(x=dfull[K - 1:], weight=dw, bias=du.sum((0, 1)), state=dfull[:K - 1].transpose(0, 1))
    return res
