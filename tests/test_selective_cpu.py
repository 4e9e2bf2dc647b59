"""The selective layers' reference against differences and autograd, and what the operators refuse
(no GPU)."""

import pytest
import torch
from torch.autograd import forward_ad

import prlstm_amd
import selective_reference as ref
from prlstm_amd import _lib


def _inputs(reset):
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    T, B, D, N = 5, 2, 3, 2
    s = dict(x=r(T, B, D), delta=r(T, B, D), a=-r(D, N).abs(), b=r(T, B, N), c=r(T, B, N), d=r(D), z=r(T, B, D),
             delta_bias=r(D), h0=r(B, D, N), reset=torch.rand(T, B, generator=g) < reset)
    return s, r(T, B, D), r(B, D, N)


def _differences(fn, leaves, outs, grads, eps=1e-6):
    """Central differences of <outs, their gradients> against the gradients in `grads`."""
    total = lambda: sum((fn()[k] * g).sum() for k, g in outs.items())  # noqa: E731
    for name, t in leaves.items():
        flat = t.view(-1)
        for i in range(flat.numel()):
            old = flat[i].item()
            flat[i] = old + eps
            hi = total()
            flat[i] = old - eps
            lo = total()
            flat[i] = old
            assert abs((hi - lo).item() / (2 * eps) - grads[name].reshape(-1)[i].item()) < 1e-7, (name, i)


@pytest.mark.parametrize("reset", [0.0, 0.4])
def test_reference_scan_against_differences(reset):
    s, dout, dh_n = _inputs(reset)
    grads = ref.scan(**s, dout=dout, dh_n=dh_n)
    _differences(lambda: ref.scan(**s), {k: v for k, v in s.items() if k != "reset"}, {"y": dout, "h": dh_n}, grads)


@pytest.mark.parametrize("act", [True, False])
def test_reference_conv_against_differences(act):
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    T, B, D, K = 6, 2, 3, 4
    s = dict(x=r(T, B, D), weight=r(D, K), bias=r(D), state=r(B, K - 1, D), reset=torch.rand(T, B, generator=g) < 0.3)
    dout, dn = r(T, B, D), r(B, K - 1, D)
    grads = ref.conv(**s, act=act, dout=dout, dstate_n=dn)
    _differences(lambda: ref.conv(**s, act=act), {k: v for k, v in s.items() if k != "reset"},
                 {"y": dout, "state_n": dn}, grads)


def test_cpu_tensors_are_rejected():
    z = torch.zeros
    for call in (lambda: prlstm_amd.causal_conv(z(4, 2, 3), z(3, 4)),
                 lambda: prlstm_amd.causal_conv_step(z(2, 3), None, z(3, 4)),
                 lambda: prlstm_amd.selective_scan(z(4, 2, 3), z(4, 2, 3), z(3, 5), z(4, 2, 5), z(4, 2, 5)),
                 lambda: prlstm_amd.selective_scan_step(z(2, 3), z(2, 3), z(3, 5), z(2, 5), z(2, 5), None)):
        with pytest.raises(RuntimeError, match="ROCm devices only"):
            call()


def _refused(rc, code, text):
    assert rc == code and text in _lib.load().hsl_last_error(), (rc, _lib.load().hsl_last_error())


def _conv_fwd(T=4, B=2, D=3, K=4, fmt=0, p=None):
    return _lib.load().hsl_conv_fwd(p, 0, 0, p, p, p, None, 0, 0, p, 0, 0, p, 1, T, B, D, K, fmt, None)


def _conv_bwd(T=4, B=2, D=3, K=4, fmt=0, p=None):
    return _lib.load().hsl_conv_bwd(p, 0, 0, p, p, p, None, 0, 0, p, 0, 0, p, p, 0, 0, p, p, p, 1, None, 0, T, B, D, K,
                                    fmt, None)


def _scan_fwd(T=4, B=2, D=3, N=4, fmt=0, p=None):
    return _lib.load().hsl_selective_fwd(p, 0, 0, p, 0, 0, p, p, 0, 0, p, 0, 0, p, p, 0, 0, p, p, None, 0, 0, p, 0, 0,
                                         p, None, 1, None, 0, T, B, D, N, fmt, None)


def _scan_bwd(T=4, B=2, D=3, N=4, fmt=0, p=None):
    return _lib.load().hsl_selective_bwd(p, 0, 0, p, 0, 0, p, p, 0, 0, p, 0, 0, p, p, 0, 0, p, None, 0, 0, p, p, 0, 0,
                                         p, p, 0, 0, p, 0, 0, p, p, 0, 0, p, 0, 0, p, p, 0, 0, p, p, 1, None, 0, T, B,
                                         D, N, fmt, None)


@pytest.mark.parametrize("call,last", [(_conv_fwd, "K"), (_conv_bwd, "K"), (_scan_fwd, "N"), (_scan_bwd, "N")])
def test_entry_points_refuse_bad_arguments(call, last):
    _refused(call(fmt=3), 1, b"format 3")
    _refused(call(T=-1), 1, b"negative size")
    _refused(call(B=-1), 1, b"negative size")
    _refused(call(**{last: 0}), 1, b"must be 1..")
    _refused(call(**{last: 65}), 1, b"must be 1..")
    _refused(call(), 1, b"null pointer")
    _refused(call(T=1 << 30), 2, b"index range")
    _refused(call(B=1 << 20, D=1 << 7), 2, b"index range")


def test_entry_points_refuse_small_workspaces():
    """The pointers are not looked at before the sizes."""
    _refused(_conv_bwd(p=1), 1, b"workspace 0 bytes")
    _refused(_scan_bwd(p=1), 1, b"workspace 0 bytes")
    _refused(_scan_fwd(T=4096, D=64, p=1), 1, b"workspace 0 bytes")  # in segments
    _refused(_scan_fwd(B=1 << 25, D=1, p=1), 2, b"index range")  # more threads than a launch has
    _refused(_conv_fwd(T=(1 << 30) - 1, B=1 << 10, D=1, p=1), 2, b"index range")


def test_size_queries():
    lib = _lib.load()
    assert lib.hsl_selective_ck_floats(0, 2, 3, 4) == 0
    assert lib.hsl_selective_ck_floats(17, 2, 3, 5) == 2 * 2 * 3 * 8
    assert lib.hsl_selective_ck_floats(17, 2, 3, 33) == 3 * 2 * 3 * 64
    for f in (lib.hsl_selective_fwd_ws_bytes, lib.hsl_selective_bwd_ws_bytes, lib.hsl_selective_ck_floats):
        assert f(-1, 2, 3, 4) == 0 and f(1 << 30, 2, 3, 4) == 0 and f(100, 1 << 20, 1 << 20, 4) == 0
        assert f(100, 2, 3, 65) == 0 and f(100, 0, 3, 4) == 0 and f(100, 2, 0, 4) == 0
    assert lib.hsl_selective_fwd_ws_bytes(1, 2, 64, 16) == 0 and lib.hsl_selective_fwd_ws_bytes(4096, 2, 64, 16) > 0
    assert lib.hsl_conv_ws_bytes(-1, 2, 3, 4) == 0 and lib.hsl_conv_ws_bytes(10, 2, 3, 5) == 0
    assert lib.hsl_conv_ws_bytes(4096, 16, 1024, 4) >= 5 * 1024 * 4


def test_empty_calls_do_nothing():
    assert _conv_fwd(B=0) == 0 and _conv_fwd(D=0) == 0 and _scan_fwd(B=0) == 0 and _scan_fwd(D=0) == 0
