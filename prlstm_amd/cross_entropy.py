"""``linear_cross_entropy(x, weight, targets, bias)``: the cross entropy of a projection on the vocabulary,
which the HIP kernels of libhsl compute without keeping the logits, in either direction.

The same streams, graphs, errors and derivatives as ``prlstm_amd.lm``; ``token_logprobs`` there works on
logits that are kept.
"""

import torch

from . import _lib
from .lm import _first_order, _fits, _fmt, _ids, _launch, _no_tangents, _size, _unit_inner, _ws
from .selective import _needs_grad, _weight


def _rows(t):
    """(t with dense rows that do not overlap, the elements between them).  16-bit rows that the kernels could read
    in place but for where they begin are copied."""
    t = _unit_inner(t)
    n, d = t.shape
    ld = t.stride(0) if n > 1 else d
    if ld < d:
        t, ld = t.contiguous(), d
    if d % 8 == 0 and t.dtype is not torch.float32 and (ld % 8 or ld >= 1 << 21 or t.data_ptr() % 16):
        t, ld = t.clone(memory_format=torch.contiguous_format), d
    return t, ld


def _xent_fwd(x, weight, bias, targets, fmt, ids64, keep):
    """(loss, the rows' statistics for the backward, or None)."""
    (x, ldx), (weight, ldw) = _rows(x), _rows(weight)
    n, d = x.shape
    v = weight.shape[0]
    f32 = dict(dtype=torch.float32, device=x.device)
    loss, stats = torch.empty(n, **f32), torch.empty(n, 2, **f32) if keep else None
    nbytes = _size("hsl_xent_ws_bytes", n, v, d, fmt, 0)
    ws = _ws(nbytes, x)
    P = _lib.ptr
    _launch(x.device, "hsl_xent_fwd", P(x), ldx, P(weight), ldw, P(bias), P(targets), ids64, P(loss), P(stats), P(ws),
            nbytes, n, v, d, fmt)
    return loss, stats


class LinearCrossEntropyFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, targets, fmt, ids64):
        ctx.set_materialize_grads(False)
        loss, stats = _xent_fwd(x, weight, bias, targets, fmt, ids64, True)
        ctx.save_for_backward(x, weight, bias, targets, stats)
        ctx.meta = (fmt, ids64)
        return loss

    @staticmethod
    @_first_order
    def backward(ctx, dloss):
        if dloss is None:
            return (None,) * 6
        x, weight, bias, targets, stats = ctx.saved_tensors
        fmt, ids64 = ctx.meta
        (x, ldx), (weight, ldw) = _rows(x), _rows(weight)
        (n, d), v = x.shape, weight.shape[0]
        dloss = dloss.contiguous()
        needs = ctx.needs_input_grad
        dx = x.new_empty(n, d) if needs[0] else None
        dw = weight.new_empty(v, d) if needs[1] else None
        dbias = torch.empty_like(bias) if bias is not None and needs[2] else None
        nbytes = _size("hsl_xent_ws_bytes", n, v, d, fmt, 1)
        ws = _ws(nbytes, x)
        P = _lib.ptr
        _launch(x.device, "hsl_xent_bwd", P(x), ldx, P(weight), ldw, P(bias), P(targets), ids64, P(stats), P(dloss),
                P(dx), P(dw), P(dbias), P(ws), nbytes, n, v, d, fmt)
        return dx, dw, dbias, None, None, None


def linear_cross_entropy(x, weight, targets, bias=None):
    """``-log softmax(x weight^T + bias)`` at ``targets``, in fp32 and shaped as targets: x [..., D] and
    weight [V, D] in one dtype, targets [...] (int64 or int32), bias [V].

    A negative target is a position that is not scored: loss 0, no gradient, and nothing that its row of
    x holds (NaN, infinities) reaches those of weight and bias.  One at or beyond V gives NaN, no gradient,
    and raises the device word that ``prlstm_amd.check_errors`` reports.  A bias of ``-inf`` masks a token
    whose logits are finite without it, and which then has no gradient; a masked target has loss ``inf``,
    and a row of nothing but masks has no gradient at all.  x, weight and bias have gradients; with 16-bit
    operands those of the logits are rounded to 16 bits before they are multiplied (up to 128 bf16 and 512
    fp16 rows: kept as two 16-bit numbers), and every sum is fp32.
    """
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise RuntimeError(f"x must be [..., D] and weight [V, D], got shapes {tuple(x.shape)} and "
                           f"{tuple(weight.shape)}")
    fmt = _fmt("x", x)
    _fits("x", x)
    _fits("weight", weight)
    _no_tangents(x, weight, bias)
    if weight.dtype is not x.dtype or weight.device != x.device:
        raise RuntimeError(f"weight must be {x.dtype} on {x.device}, got {weight.dtype} on {weight.device}")
    v, d = weight.shape
    if v == 0 or d == 0:
        raise RuntimeError(f"weight must not be empty, got shape {tuple(weight.shape)}")
    lead = x.shape[:-1]
    ids64 = _ids("targets", targets, x.device)
    if targets.shape != lead:
        raise RuntimeError(f"targets must have shape {tuple(lead)}, got {tuple(targets.shape)}")
    bias = _weight("bias", bias, (v,), x)
    targets = targets.contiguous()
    flat = x if len(lead) == 1 else x.reshape(lead.numel(), d)
    if _needs_grad(x, weight, bias):
        loss = LinearCrossEntropyFn.apply(flat, weight, bias, targets, fmt, ids64)
    else:
        loss, _ = _xent_fwd(flat, weight, bias, targets, fmt, ids64, False)
    return loss if len(lead) == 1 else loss.reshape(lead)
