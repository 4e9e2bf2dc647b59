"""The layers of a selective state space model, on the HIP kernels of libhsl.

* ``causal_conv(x, weight, bias)``: a short causal convolution of every channel over time, with SiLU,
  and ``causal_conv_step`` for one token of each of a batch of streams.
* ``selective_scan(x, delta, a, b, c)``: ``h_t = exp(dt_t a) h_{t-1} + dt_t x_t b_t``,
  ``y_t = c_t h_t + d x_t`` with N states per channel, and ``selective_scan_step``.

Streams are [T, B, ...] in bf16, fp16 or fp32 (all streams of a call in one type); weights, states
and their gradients are fp32.  Streams of any time and batch strides are read as they are (a
transposed [B, T, ...] too), and outputs and gradients take x's order in memory.  As in
``prlstm_amd.lm``, every call runs on the current HIP stream, can be captured in a graph, is
differentiable once, and raises ``RuntimeError`` for operands that do not fit.
"""

import torch
from torch.autograd.graph import increment_version

from . import _lib
from .lm import _first_order, _fits, _fmt, _launch, _like_order, _no_tangents, _size, _unit_inner, _ws

MAX_TAPS = 4     # of causal_conv
MAX_STATES = 64  # of a channel of selective_scan


def _strided(t):
    """Pointer and outer strides of a [T, B, ...] stream, of a [B, ...] step, or of none."""
    if t is None:
        return None, 0, 0
    s = t.stride()
    return t.data_ptr(), s[0] if len(s) == 3 else 0, s[-2]


def _reset_args(reset):
    if reset is None:
        return None, 0, 0
    s = reset.stride()
    return reset.data_ptr(), s[0] if len(s) == 2 else 0, s[-1]


def _check_reset(reset, lead, device):
    if reset is None:
        return
    if reset.shape != lead:
        raise RuntimeError(f"reset must have shape {tuple(lead)}, got {tuple(reset.shape)}")
    if reset.device != device or reset.dtype not in (torch.bool, torch.uint8):
        raise RuntimeError(f"reset must be a bool or uint8 tensor on {device}, got {reset.dtype} on {reset.device}")


def _check_like(name, t, shape, x):
    """A stream of the call beside x."""
    if tuple(t.shape) != shape or t.dtype is not x.dtype or t.device != x.device:
        raise RuntimeError(f"{name} must be {x.dtype} {shape} on {x.device}, got {t.dtype} {tuple(t.shape)} on "
                           f"{t.device}")


def _weight(name, t, shape, x):
    """A weight or state in fp32, dense."""
    if t is None or (t.dtype is torch.float32 and t.shape == shape and t.device == x.device and t.is_contiguous()):
        return t
    if tuple(t.shape) != shape or t.device != x.device or not t.dtype.is_floating_point:
        raise RuntimeError(f"{name} must be a floating-point tensor {shape} on {x.device}, got {t.dtype} "
                           f"{tuple(t.shape)} on {t.device}")
    return t.float().contiguous()


def _check_out(name, out, source):
    """An output that the caller gives: it may be the operand it replaces, but not a part of it."""
    p, q, size = out.data_ptr(), 0 if source is None else source.data_ptr(), out.nbytes
    if p != q and q - size < p < q + size:
        raise RuntimeError(f"{name} overlaps the state that it is computed from")


def _needs_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---- causal convolution --------------------------------------------------------------------


def _conv_check(x, weight, bias, state, reset, activation, dims):
    lead = ("T", "B")[2 - dims:]
    if x.dim() != dims + 1:
        raise RuntimeError(f"x must be [{', '.join(lead)}, D], got shape {tuple(x.shape)}")
    fmt = _fmt("x", x)
    _fits("x", x)
    _no_tangents(x, weight, bias, state)
    if activation not in ("silu", None):
        raise RuntimeError(f"activation must be 'silu' or None, got {activation!r}")
    b, d = x.shape[-2:]
    if weight.dim() != 2 or not 1 <= weight.shape[1] <= MAX_TAPS:
        raise RuntimeError(f"weight must be [D, K] with K in 1..{MAX_TAPS}, got shape {tuple(weight.shape)}")
    k = weight.shape[1]
    weight, bias = _weight("weight", weight, (d, k), x), _weight("bias", bias, (d,), x)
    if state is not None:
        _check_like("state", state, (b, k - 1, d), x)
    _check_reset(reset, x.shape[:-1], x.device)
    return fmt, weight, bias, k, 0 if activation is None else 1


def _conv_fwd(x, weight, bias, state, reset, silu, fmt):
    t, b, d = x.shape
    k = weight.shape[1]
    y, state_n = _like_order(x, t, b, d), x.new_empty(b, k - 1, d)
    P = _lib.ptr
    _launch(x.device, "hsl_conv_fwd", *_strided(x), P(weight), P(bias), P(state), *_reset_args(reset), *_strided(y),
            P(state_n), silu, t, b, d, k, fmt)
    return y, state_n


class CausalConvFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, reset, silu, fmt):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, state, reset)
        ctx.meta = (silu, fmt)
        return _conv_fwd(x, weight, bias, state, reset, silu, fmt)

    @staticmethod
    @_first_order
    def backward(ctx, dy, dstate_n):
        if dy is None and dstate_n is None:
            return (None,) * 7
        x, weight, bias, state, reset = ctx.saved_tensors
        silu, fmt = ctx.meta
        t, b, d = x.shape
        k = weight.shape[1]
        dy = None if dy is None else _unit_inner(dy)
        dstate_n = None if dstate_n is None else dstate_n.contiguous()
        dx, dw = _like_order(x, t, b, d), torch.empty_like(weight)
        dbias = None if bias is None else torch.empty_like(bias)
        dstate = None if state is None or not ctx.needs_input_grad[3] else torch.empty_like(state)
        nbytes = _size("hsl_conv_ws_bytes", t, b, d, k)
        ws = _ws(nbytes, x)
        P = _lib.ptr
        _launch(x.device, "hsl_conv_bwd", *_strided(x), P(weight), P(bias), P(state), *_reset_args(reset),
                *_strided(dy), P(dstate_n), *_strided(dx), P(dw), P(dbias), P(dstate), silu, P(ws), nbytes, t, b, d, k,
                fmt)
        return dx, dw, dbias, dstate, None, None, None


def causal_conv(x, weight, bias=None, state=None, reset=None, activation="silu"):
    """``y_t = act(bias + sum_j weight[:, j] x_{t-K+1+j})`` for every channel of x [T, B, D], with
    weight [D, K], K at most 4, and act SiLU (``activation=None``: none).  Returns (y, state_n).

    ``state`` [B, K-1, D] in x's dtype holds the inputs before the first step, the oldest first (None:
    zeros), and ``state_n`` is what the next call takes.  Where ``reset`` [T, B] is set a new sequence
    begins: no input from before that step passes it, forward or backward, nor does its NaN or
    infinity.  All of x, weight, bias and state have gradients.
    """
    fmt, weight, bias, _, silu = _conv_check(x, weight, bias, state, reset, activation, 2)
    x = _unit_inner(x)
    state = None if state is None else state.contiguous()
    if _needs_grad(x, weight, bias, state):
        return CausalConvFn.apply(x, weight, bias, state, reset, silu, fmt)
    return _conv_fwd(x, weight, bias, state, reset, silu, fmt)


def causal_conv_step(x, state, weight, bias=None, reset=None, activation="silu", state_out=None):
    """One step of ``causal_conv`` without gradients, for serving: x [B, D], state [B, K-1, D] (None:
    zeros), reset [B].  Returns (y [B, D], the new state); ``state_out`` receives the state where it is
    given; it may be state itself, and shares no memory with the other operands.
    """
    fmt, weight, bias, k, silu = _conv_check(x, weight, bias, state, reset, activation, 1)
    b, d = x.shape
    for name, t in (("state", state), ("state_out", state_out)):
        if t is not None and not t.is_contiguous():
            raise RuntimeError(f"{name} must be contiguous, got strides {t.stride()}")
    given = state_out is not None
    if given:
        _check_like("state_out", state_out, (b, k - 1, d), x)
        _check_out("state_out", state_out, state)
    else:
        state_out = x.new_empty(b, k - 1, d)
    x = _unit_inner(x)
    y = x.new_empty(b, d)
    P = _lib.ptr
    _launch(x.device, "hsl_conv_fwd", *_strided(x), P(weight), P(bias), P(state), *_reset_args(reset), *_strided(y),
            P(state_out), silu, 1, b, d, k, fmt)
    if given:
        increment_version(state_out)  # for a backward pass that has saved it
    return y, state_out


# ---- selective scan ------------------------------------------------------------------------


def _scan_check(x, delta, a, b, c, d, z, delta_bias, h0, reset, dims):
    """fmt and the fp32 weights."""
    lead = ("T", "B")[2 - dims:]
    if x.dim() != dims + 1:
        raise RuntimeError(f"x must be [{', '.join(lead)}, D], got shape {tuple(x.shape)}")
    fmt = _fmt("x", x)
    _fits("x", x)
    _no_tangents(x, delta, a, b, c, d, z, delta_bias, h0)
    width = x.shape[-1]
    if a.dim() != 2 or not 1 <= a.shape[1] <= MAX_STATES:
        raise RuntimeError(f"a must be [D, N] with N in 1..{MAX_STATES}, got shape {tuple(a.shape)}")
    n, shape = a.shape[1], tuple(x.shape)
    _check_like("delta", delta, shape, x)
    if z is not None:
        _check_like("z", z, shape, x)
    narrow = (*shape[:-1], n)
    _check_like("b", b, narrow, x)
    _check_like("c", c, narrow, x)
    _check_reset(reset, x.shape[:-1], x.device)
    return (fmt, _weight("a", a, (width, n), x), _weight("d", d, (width,), x),
            _weight("delta_bias", delta_bias, (width,), x))


def _scan_fwd(x, delta, a, b, c, d, z, delta_bias, h0, reset, softplus, fmt, keep):
    """(y, h_n, the states that the backward starts from, or None)."""
    t, bsz, width = x.shape
    n = a.shape[1]
    sizes = (t, bsz, width, n)
    y = _like_order(x, t, bsz, width)
    f32 = dict(dtype=torch.float32, device=x.device)
    h_n = torch.empty(bsz, width, n, **f32)
    ck = torch.empty(_size("hsl_selective_ck_floats", *sizes), **f32) if keep else None
    nbytes = _size("hsl_selective_fwd_ws_bytes", *sizes)
    ws = _ws(nbytes, x)
    P = _lib.ptr
    _launch(x.device, "hsl_selective_fwd", *_strided(x), *_strided(delta), P(a), *_strided(b), *_strided(c), P(d),
            *_strided(z), P(delta_bias), P(h0), *_reset_args(reset), *_strided(y), P(h_n), P(ck), softplus, P(ws),
            nbytes, *sizes, fmt)
    return y, h_n, ck


class SelectiveScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, delta, a, b, c, d, z, delta_bias, h0, reset, softplus, fmt):
        ctx.set_materialize_grads(False)
        y, h_n, ck = _scan_fwd(x, delta, a, b, c, d, z, delta_bias, h0, reset, softplus, fmt, True)
        ctx.save_for_backward(x, delta, a, b, c, d, z, delta_bias, reset, ck)
        ctx.meta = (softplus, fmt)
        return y, h_n

    @staticmethod
    @_first_order
    def backward(ctx, dout, dh_n):
        if dout is None and dh_n is None:
            return (None,) * 12
        x, delta, a, b, c, d, z, delta_bias, reset, ck = ctx.saved_tensors
        softplus, fmt = ctx.meta
        t, bsz, width = x.shape
        n = a.shape[1]
        sizes = (t, bsz, width, n)
        dout = None if dout is None else _unit_inner(dout)
        dh_n = None if dh_n is None else dh_n.contiguous()
        dx, ddelta = (_like_order(x, t, bsz, width) for _ in range(2))
        db, dc = (_like_order(x, t, bsz, n) for _ in range(2))
        dz = None if z is None else _like_order(x, t, bsz, width)
        da = torch.empty_like(a)
        dd, dbias = (None if w is None else torch.empty_like(w) for w in (d, delta_bias))
        dh0 = torch.empty(bsz, width, n, dtype=torch.float32, device=x.device) if ctx.needs_input_grad[8] else None
        nbytes = _size("hsl_selective_bwd_ws_bytes", *sizes)
        ws = _ws(nbytes, x)
        P = _lib.ptr
        _launch(x.device, "hsl_selective_bwd", *_strided(x), *_strided(delta), P(a), *_strided(b), *_strided(c), P(d),
                *_strided(z), P(delta_bias), *_reset_args(reset), P(ck), *_strided(dout), P(dh_n), *_strided(dx),
                *_strided(ddelta), P(da), *_strided(db), *_strided(dc), P(dd), *_strided(dz), P(dbias), P(dh0),
                softplus, P(ws), nbytes, *sizes, fmt)
        return dx, ddelta, da, db, dc, dd, dz, dbias, dh0, None, None, None


def selective_scan(x, delta, a, b, c, d=None, z=None, delta_bias=None, h0=None, reset=None, softplus=True):
    """``h_t = exp(dt_t a) h_{t-1} + dt_t x_t b_t`` with N states for every channel,
    ``y_t = sum_n c_t[n] h_t[n] + d x_t``, times ``z_t sigmoid(z_t)`` where z is given, and
    ``dt_t = log(1 + exp(delta_t + delta_bias))`` (``softplus=False``: ``delta_t + delta_bias``).

    x, delta and z are [T, B, D], b and c [T, B, N] (N at most 64) in one dtype; a [D, N] (negative
    where states shall fade), d and delta_bias [D].  Returns (y [T, B, D] in x's dtype, h_n [B, D, N]
    in fp32).  ``h0`` [B, D, N] is the state before the first step (None: zeros).  Where ``reset``
    [T, B] is set a new sequence begins: nothing of the state before that step passes it, forward or
    backward, nor does its NaN or infinity.  Everything but reset has a gradient; those of a, b, c, d
    and delta_bias are summed in a fixed order.
    """
    fmt, a, d, delta_bias = _scan_check(x, delta, a, b, c, d, z, delta_bias, h0, reset, 2)
    h0 = _weight("h0", h0, (x.shape[1], x.shape[2], a.shape[1]), x)
    x, delta, b, c = _unit_inner(x), _unit_inner(delta), _unit_inner(b), _unit_inner(c)
    z = None if z is None else _unit_inner(z)
    softplus = 1 if softplus else 0
    if _needs_grad(x, delta, a, b, c, d, z, delta_bias, h0):
        return SelectiveScanFn.apply(x, delta, a, b, c, d, z, delta_bias, h0, reset, softplus, fmt)
    return _scan_fwd(x, delta, a, b, c, d, z, delta_bias, h0, reset, softplus, fmt, False)[:2]


def selective_scan_step(x, delta, a, b, c, h, d=None, z=None, delta_bias=None, reset=None, softplus=True, h_out=None):
    """One step of ``selective_scan`` without gradients, for serving: x, delta and z [B, D], b and c
    [B, N], the state h [B, D, N] in fp32 (None: zeros), reset [B].  Returns (y [B, D] in x's dtype,
    the new state in fp32); ``h_out`` receives the state where it is given; it may be h itself, and
    shares no memory with the other operands.
    """
    fmt, a, d, delta_bias = _scan_check(x, delta, a, b, c, d, z, delta_bias, h, reset, 1)
    bsz, width = x.shape
    n = a.shape[1]
    state = (bsz, width, n)
    for name, t in (("h", h), ("h_out", h_out)):
        if t is not None and (t.dtype is not torch.float32 or tuple(t.shape) != state or t.device != x.device
                              or not t.is_contiguous()):
            raise RuntimeError(f"{name} must be a contiguous float32 tensor {state} on {x.device}, got {t.dtype} "
                               f"{tuple(t.shape)} on {t.device}")
    given = h_out is not None
    if given:
        _check_out("h_out", h_out, h)
    else:
        h_out = torch.empty(state, dtype=torch.float32, device=x.device)
    x, delta, b, c = _unit_inner(x), _unit_inner(delta), _unit_inner(b), _unit_inner(c)
    z = None if z is None else _unit_inner(z)
    y = x.new_empty(bsz, width)
    P = _lib.ptr
    _launch(x.device, "hsl_selective_fwd", *_strided(x), *_strided(delta), P(a), *_strided(b), *_strided(c), P(d),
            *_strided(z), P(delta_bias), P(h), *_reset_args(reset), *_strided(y), P(h_out), None,
            1 if softplus else 0, None, 0, 1, bsz, width, n, fmt)
    if given:
        increment_version(h_out)  # for a backward pass that has saved it
    return y, h_out
