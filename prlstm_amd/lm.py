"""Operators of a language model around the recurrent layers, on the HIP kernels of libhsl.

* ``embedding(ids, weight, scale)``: rows of a table, times a scale, and the table's gradient.
* ``gated_recurrence(zv, h0, reset)``: ``h_t = f_t h_{t-1} + (1 - f_t) v_t`` with ``f = sigmoid(z)``
  over sequences, and ``gated_recurrence_step`` for one token of each of a batch of streams.
* ``token_logprobs(logits, tokens, top)``: log probabilities of given tokens, the entropy and the
  best alternatives of each row.

Tensors are bf16, fp16 or fp32; states, statistics and log probabilities are fp32 whatever the
streams are.  Every call runs on the current HIP stream of its tensors' device, allocates only
through torch's caching allocator and synchronises nothing, so it can be captured in a graph.
Operands that do not fit raise ``RuntimeError``; CPU tensors are rejected.  The gradients are not
differentiable themselves, and forward-mode derivatives are refused (``NotImplementedError``).
"""

import functools
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _lib

_FMT = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_IDS = (torch.int64, torch.int32)
MAX_TOP = 32  # alternatives of a row that token_logprobs gives at most


@functools.lru_cache(maxsize=None)
def _entry(name):
    return getattr(_lib.load(), name)


@functools.lru_cache(maxsize=4096)
def _size(name, *args):
    """A size query of the library (they depend on nothing but their arguments)."""
    return _entry(name)(*args)


def _launch(device, name, *args):
    """The C entry point on the device's current stream, with that device current.  (The raw handle:
    a Stream object takes 3 us of the host, most of a small call.)"""
    index = device.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _launch(device, name, *args)
    if _entry(name)(*args, torch._C._cuda_getCurrentRawStream(index)):
        raise RuntimeError(f"{name} failed: {_lib.load().hsl_last_error().decode(errors='replace')}")


def _no_tangents(*tensors):
    """The kernels compute no forward-mode derivative; a launch alone would pass on one of zero."""
    if forward_ad._current_level >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("the operators of prlstm_amd.lm have no forward-mode derivatives")


def _first_order(backward):
    """``once_differentiable``, whose wrapping costs a small step some microseconds, only where a
    graph of the gradient is asked for."""
    checked = once_differentiable(backward)

    @functools.wraps(backward)
    def run(ctx, *grads):
        _no_tangents(*grads)
        return checked(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run


def _fmt(name, t):
    fmt = _FMT.get(t.dtype)
    if fmt is None:
        raise RuntimeError(f"{name} must be bfloat16, float16 or float32, got {t.dtype}")
    if not t.is_cuda:
        raise RuntimeError(f"prlstm_amd runs on ROCm devices only: {name} is on {t.device} (move it to the GPU)")
    return fmt


def _ids(name, t, device):
    if t.dtype not in _IDS:
        raise RuntimeError(f"{name} must be int64 or int32, got {t.dtype}")
    if t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, the other operands on {device}")
    return 1 if t.dtype is torch.int64 else 0


def _fits(name, t):
    """Sizes pass to the library in 32 bits, where 2^32 + 5 would be 5."""
    n = t.numel()
    if (n >= 1 << 31 or n == 0) and max(t.shape) >= 1 << 31:
        raise RuntimeError(f"{name} {tuple(t.shape)} has a size of 2^31 or more")


def _unit_inner(t):
    """t with its last dimension dense (a copy where it is not)."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _ws(nbytes, like):
    return like.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


# ---- embedding -----------------------------------------------------------------------------


def _scale(scale):
    if isinstance(scale, torch.Tensor):
        _no_tangents(scale)
        if scale.is_cuda or (scale.requires_grad and torch.is_grad_enabled()):
            raise RuntimeError(f"scale must be a number (it has no gradient and is not read from the GPU), got a "
                               f"tensor on {scale.device} with requires_grad={scale.requires_grad}")
    return float(scale)


def _embed_check(ids, weight, padding_idx):
    if weight.dim() != 2:
        raise RuntimeError(f"weight must be [V, D], got shape {tuple(weight.shape)}")
    fmt = _fmt("weight", weight)
    _fits("weight", weight)
    _no_tangents(weight)
    if padding_idx is not None and not 0 <= padding_idx < weight.shape[0]:
        raise RuntimeError(f"padding_idx {padding_idx} is not a row of weight {tuple(weight.shape)}")
    return fmt, _ids("ids", ids, weight.device)


def _embed_fwd(ids, weight, scale, fmt, ids64):
    v, d = weight.shape
    out = weight.new_empty((*ids.shape, d))
    _launch(weight.device, "hsl_embed_fwd", ids.data_ptr(), ids64, weight.data_ptr(), weight.stride(0), scale,
            out.data_ptr(), ids.numel(), v, d, fmt)
    return out


class EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx, fmt, ids64):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(ids)
        ctx.meta = (weight.shape, scale, -1 if padding_idx is None else padding_idx, fmt, ids64)
        return _embed_fwd(ids, weight, scale, fmt, ids64)

    @staticmethod
    @_first_order
    def backward(ctx, dout):
        if dout is None:
            return (None,) * 6
        ids, = ctx.saved_tensors
        (v, d), scale, padding, fmt, ids64 = ctx.meta
        n = ids.numel()
        dout = _unit_inner(dout if dout.dim() == 2 else dout.reshape(n, d))
        dw = dout.new_empty((v, d))
        nbytes = _size("hsl_embed_bwd_ws_bytes", n, v, d)
        ws = _ws(nbytes, dw)
        _launch(dw.device, "hsl_embed_bwd", ids.data_ptr(), ids64, dout.data_ptr(), dout.stride(0), scale, padding,
                dw.data_ptr(), _lib.ptr(ws), nbytes, n, v, d, fmt)
        return None, dw, None, None, None, None


def embedding(ids, weight, scale=1.0, padding_idx: Optional[int] = None):
    """``scale * weight[ids]`` in weight's dtype: ids of any shape (int64 or int32), weight [V, D].

    A negative id is a position without a token: a row of zeros, no gradient.  An id at or beyond V
    gives a row of NaN and raises the device word that ``prlstm_amd.check_errors`` reports.  The
    gradient of weight is dense and sums each row's positions in fp32 in a fixed order;
    ``padding_idx`` is a row that gets none.  scale is a number and has no gradient.
    """
    fmt, ids64 = _embed_check(ids, weight, padding_idx)
    ids, weight, scale = ids.contiguous(), _unit_inner(weight), scale if type(scale) is float else _scale(scale)
    if weight.requires_grad and torch.is_grad_enabled():
        return EmbeddingFn.apply(ids, weight, scale, padding_idx, fmt, ids64)
    return _embed_fwd(ids, weight, scale, fmt, ids64)


# ---- gated recurrence ----------------------------------------------------------------------


def _like_order(zv, t, b, n):
    """An empty [t, b, n] whose outer of time and batch in memory is zv's.  (No view of another tensor:
    torch allows no change in place to a view that a Function returns.)"""
    if zv.stride(0) >= zv.stride(1):
        return zv.new_empty(t, b, n)
    return zv.new_empty_strided((t, b, n), (n, t * n, 1))


def _gated_check(zv, h0, reset, dims):
    lead = ("T", "B")[2 - dims:]
    if zv.dim() != dims + 1 or zv.shape[-1] % 2:
        raise RuntimeError(f"zv must be [{', '.join(lead)}, 2H], got shape {tuple(zv.shape)}")
    fmt = _fmt("zv", zv)
    _fits("zv", zv)
    _no_tangents(zv, h0)
    state = (zv.shape[-2], zv.shape[-1] // 2)
    if h0 is not None:
        if tuple(h0.shape) != state:
            raise RuntimeError(f"h0 must have shape {state}, got {tuple(h0.shape)}")
        if h0.device != zv.device or not h0.dtype.is_floating_point:
            raise RuntimeError(f"h0 must be a floating-point tensor on {zv.device}, got {h0.dtype} on {h0.device}")
    if reset is not None:
        if reset.shape != zv.shape[:-1]:
            raise RuntimeError(f"reset must have shape {tuple(zv.shape[:-1])}, got {tuple(reset.shape)}")
        if reset.device != zv.device or reset.dtype not in (torch.bool, torch.uint8):
            raise RuntimeError(f"reset must be a bool or uint8 tensor on {zv.device}, got {reset.dtype} on "
                               f"{reset.device}")
    return fmt


def _gated_fwd(zv, h0, reset, fmt, keep):
    """(out, h_n, the states that the backward starts from, or None)."""
    t, b, n = zv.shape
    h = n // 2
    out = _like_order(zv, t, b, h)
    f32 = dict(dtype=torch.float32, device=zv.device)
    h_n = torch.empty(b, h, **f32)
    ck = torch.empty(_size("hsl_gated_ck_rows", t), b, h, **f32) if keep else None
    nbytes = _size("hsl_gated_ws_bytes", t, b, h)
    ws = _ws(nbytes, zv)
    rp, rt, rb = (None, 0, 0) if reset is None else (reset.data_ptr(), *reset.stride())
    _launch(zv.device, "hsl_gated_fwd", zv.data_ptr(), zv.stride(0), zv.stride(1), _lib.ptr(h0), rp, rt, rb,
            out.data_ptr(), out.stride(0), out.stride(1), h_n.data_ptr(), _lib.ptr(ck), _lib.ptr(ws), nbytes, t, b, h,
            fmt)
    return out, h_n, ck


class GatedRecurrenceFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, zv, h0, reset, fmt):
        ctx.set_materialize_grads(False)
        out, h_n, ck = _gated_fwd(zv, h0, reset, fmt, True)
        ctx.save_for_backward(zv, reset, ck)
        ctx.fmt = fmt
        return out, h_n

    @staticmethod
    @_first_order
    def backward(ctx, dout, dh_n):
        zv, reset, ck = ctx.saved_tensors
        if dout is None and dh_n is None:
            return None, None, None, None
        t, b, n = zv.shape
        h = n // 2
        dout = None if dout is None else _unit_inner(dout)
        dh_n = None if dh_n is None else dh_n.contiguous()
        dzv = _like_order(zv, t, b, n)
        dh0 = torch.empty(b, h, dtype=torch.float32, device=zv.device) if ctx.needs_input_grad[1] else None
        nbytes = _size("hsl_gated_ws_bytes", t, b, h)
        ws = _ws(nbytes, zv)
        rp, rt, rb = (None, 0, 0) if reset is None else (reset.data_ptr(), *reset.stride())
        dp, dt, db = (None, 0, 0) if dout is None else (dout.data_ptr(), dout.stride(0), dout.stride(1))
        _launch(zv.device, "hsl_gated_bwd", zv.data_ptr(), zv.stride(0), zv.stride(1), rp, rt, rb, ck.data_ptr(), dp,
                dt, db, _lib.ptr(dh_n), dzv.data_ptr(), dzv.stride(0), dzv.stride(1), _lib.ptr(dh0), _lib.ptr(ws),
                nbytes, t, b, h, ctx.fmt)
        return dzv, dh0, None, None


def gated_recurrence(zv, h0=None, reset=None):
    """``h_t = f_t h_{t-1} + (1 - f_t) v_t``, ``f = sigmoid(z)``, over [T, B, 2H] with z in the first
    and v in the last H channels; returns (out [T, B, H] in zv's dtype, h_n [B, H] in fp32).

    ``h0`` [B, H] is the state before the first step (None: zeros).  Where ``reset`` [T, B] is set a
    new sequence begins: nothing of the state before that step passes it, forward or backward, and
    neither does its NaN or infinity.  Any strides of time and batch are read as they are (a
    transposed [B, T, 2H] too); out and the gradient take zv's order in memory.
    """
    fmt = _gated_check(zv, h0, reset, 2)
    zv = _unit_inner(zv)
    h0 = None if h0 is None else h0.float().contiguous()
    if torch.is_grad_enabled() and (zv.requires_grad or (h0 is not None and h0.requires_grad)):
        return GatedRecurrenceFn.apply(zv, h0, reset, fmt)
    return _gated_fwd(zv, h0, reset, fmt, False)[:2]


def gated_recurrence_step(zv, h, reset=None, h_out=None):
    """One step of ``gated_recurrence`` without gradients, for serving: zv [B, 2H], the state h
    [B, H] in fp32 (None: zeros), reset [B].  Returns (out [B, H] in zv's dtype, the new state in
    fp32); ``h_out`` receives the state where it is given, and may be h itself.
    """
    fmt = _gated_check(zv, h, reset, 1)
    b, n = zv.shape
    state = (b, n // 2)
    for name, t in (("h", h), ("h_out", h_out)):
        if t is not None and (t.dtype is not torch.float32 or tuple(t.shape) != state or t.device != zv.device
                              or not t.is_contiguous()):
            raise RuntimeError(f"{name} must be a contiguous float32 tensor {state} on {zv.device}, got {t.dtype} "
                               f"{tuple(t.shape)} on {t.device}")
    zv = _unit_inner(zv)
    out = zv.new_empty(state)
    given = h_out is not None
    if not given:
        h_out = torch.empty(state, dtype=torch.float32, device=zv.device)
    rp, rb = (None, 0) if reset is None else (reset.data_ptr(), reset.stride(0))
    _launch(zv.device, "hsl_gated_fwd", zv.data_ptr(), 0, zv.stride(0), _lib.ptr(h), rp, 0, rb, out.data_ptr(), 0,
            n // 2, h_out.data_ptr(), None, None, 0, 1, b, n // 2, fmt)
    if given:
        increment_version(h_out)  # for a backward pass that has saved it
    return out, h_out


# ---- log probabilities ---------------------------------------------------------------------


class TokenLogprobs(NamedTuple):
    """fp32 log probabilities and entropies, shaped as the rows of logits; the alternatives have a
    last dimension of ``top`` (None where it is 0)."""

    logp: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_logp: Optional[torch.Tensor]
    top_ids: Optional[torch.Tensor]


def _logprob_fwd(x, tokens, top, fmt, ids64):
    n, v = x.shape
    f32 = dict(dtype=torch.float32, device=x.device)
    logp = None if tokens is None else torch.empty(n, **f32)
    entropy, stats = torch.empty(n, **f32), torch.empty(n, 2, **f32)
    top_logp = torch.empty(n, top, **f32) if top else None
    top_ids = torch.empty(n, top, dtype=torch.int64, device=x.device) if top else None
    nbytes = _size("hsl_logprob_fwd_ws_bytes", n, v, top)
    ws = _ws(nbytes, x)
    P = _lib.ptr
    _launch(x.device, "hsl_logprob_fwd", x.data_ptr(), x.stride(0), P(tokens), ids64, P(logp), entropy.data_ptr(),
            stats.data_ptr(), P(top_logp), P(top_ids), P(ws), nbytes, n, v, top, fmt)
    return logp, entropy, top_logp, top_ids, stats


class TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, tokens, top, fmt, ids64):
        ctx.set_materialize_grads(False)
        logp, entropy, top_logp, top_ids, stats = _logprob_fwd(x, tokens, top, fmt, ids64)
        ctx.save_for_backward(x, tokens, top_ids, stats, entropy)
        ctx.meta = (top, fmt, ids64)
        if top:
            ctx.mark_non_differentiable(top_ids)
        return logp, entropy, top_logp, top_ids

    @staticmethod
    @_first_order
    def backward(ctx, dlogp, dent, dtop, _):
        x, tokens, top_ids, stats, entropy = ctx.saved_tensors
        top, fmt, ids64 = ctx.meta
        if dlogp is None and dent is None and dtop is None:
            return None, None, None, None, None
        n, v = x.shape
        dlogp, dent, dtop = (None if g is None else g.contiguous() for g in (dlogp, dent, dtop))
        dx = x.new_empty(n, v)
        P = _lib.ptr
        _launch(x.device, "hsl_logprob_bwd", x.data_ptr(), x.stride(0), P(tokens), ids64, P(top_ids), stats.data_ptr(),
                entropy.data_ptr(), P(dlogp), P(dent), P(dtop), dx.data_ptr(), v, n, v, top, fmt)
        return dx, None, None, None, None


def token_logprobs(logits, tokens=None, top=0):
    """Log probabilities under the softmax of logits [..., V]: of ``tokens`` [...] (int64 or int32),
    of the ``top`` (at most 32) best alternatives of each row, and the rows' entropies.

    ``-inf`` masks a token; a row of nothing else has log probability ``-inf`` for every token,
    entropy 0 and no gradient.  A negative token is a position that is not scored: log probability
    0, no gradient through it.  A token at or beyond V gives NaN and raises the device word that
    ``prlstm_amd.check_errors`` reports.  Alternatives are ordered by logit (NaN first), the lowest
    id first among equals.  Rows of any stride are read as they are (logits cut from a wider
    projection); logp, entropy and top_logp are differentiable.
    """
    if logits.dim() < 1:
        raise RuntimeError("logits must be [..., V]")
    fmt = _fmt("logits", logits)
    _no_tangents(logits)
    lead, v = logits.shape[:-1], logits.shape[-1]
    _fits("logits", logits)
    top = int(top)
    if not 0 <= top <= min(MAX_TOP, v):
        raise RuntimeError(f"top must be in 0..{min(MAX_TOP, v)}, got {top}")
    ids64 = 0
    if tokens is not None:
        ids64 = _ids("tokens", tokens, logits.device)
        if tokens.shape != lead:
            raise RuntimeError(f"tokens must have shape {tuple(lead)}, got {tuple(tokens.shape)}")
        tokens = tokens.contiguous()
    x = _unit_inner(logits if len(lead) == 1 else logits.reshape(lead.numel(), v))
    if torch.is_grad_enabled() and logits.requires_grad:
        logp, entropy, top_logp, top_ids = TokenLogprobsFn.apply(x, tokens, top, fmt, ids64)
    else:
        logp, entropy, top_logp, top_ids, _ = _logprob_fwd(x, tokens, top, fmt, ids64)
    if len(lead) != 1:
        logp = None if logp is None else logp.reshape(lead)
        entropy = entropy.reshape(lead)
        if top:
            top_logp, top_ids = top_logp.reshape(*lead, top), top_ids.reshape(*lead, top)
    return TokenLogprobs(logp, entropy, top_logp, top_ids)
