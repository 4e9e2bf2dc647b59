"""linear_cross_entropy without a GPU: what the library refuses, and its size queries."""

import pytest
import torch

import prlstm_amd
from prlstm_amd import _lib


def _fwd(N=4, V=5, D=8, fmt=0, ld=8, p=None):
    return _lib.load().hsl_xent_fwd(p, ld, p, ld, p, p, 0, p, p, None, 0, N, V, D, fmt, None)


def _bwd(N=4, V=5, D=8, fmt=0, ld=8, p=None, out=None):
    return _lib.load().hsl_xent_bwd(p, ld, p, ld, p, p, 0, p, p, out, out, out, None, 0, N, V, D, fmt, None)


def _refused(rc, code, text):
    assert rc == code and text in _lib.load().hsl_last_error(), (rc, _lib.load().hsl_last_error())


@pytest.mark.parametrize("call", [_fwd, _bwd])
def test_refusals(call):
    _refused(call(fmt=3), 1, b"format 3")
    _refused(call(N=-1), 1, b"negative size")
    _refused(call(V=0), 1, b"empty projection")
    _refused(call(D=0), 1, b"empty projection")
    _refused(call(), 1, b"null pointer")
    _refused(call(p=1, ld=7), 1, b"row strides")
    _refused(call(p=1, ld=1 << 31), 1, b"row strides")
    _refused(call(p=1), 1, b"workspace 0 bytes")
    _refused(call(D=1 << 20), 2, b"beyond one launch")
    _refused(call(N=1 << 24, V=1 << 20), 2, b"beyond one launch")
    _refused(call(N=(1 << 31) - 1, V=1), 2, b"beyond one launch")


def test_rows_that_cannot_be_read_in_place():
    """Where D is a multiple of 8, 16-bit rows are read 16 bytes at a time; the pointers are not read before."""
    lib, room = _lib.load(), 1 << 40
    for x, ldx, w, ldw in ((2, 8, 16, 8), (16, 12, 16, 8), (16, 8, 16, 1 << 21), (16, 8, 24, 8)):
        rest = (16, 16, 0, 16, 16)
        _refused(lib.hsl_xent_fwd(x, ldx, w, ldw, *rest, 16, room, 4, 5, 8, 0, None), 1, b"multiples of 16 bytes")
        _refused(lib.hsl_xent_bwd(x, ldx, w, ldw, *rest, 16, 16, 16, 16, room, 4, 5, 8, 1, None), 1,
                 b"multiples of 16 bytes")


@pytest.mark.parametrize("call", [_fwd, _bwd])
def test_more_rows_than_a_launch_has(call):
    """A workgroup of 256 threads a row: 2^24 rows would be 2^32 threads, which wrap."""
    for fmt in (0, 1, 2):
        _refused(call(N=1 << 24, V=1, fmt=fmt, p=1), 2, b"beyond one launch")
        assert _lib.load().hsl_xent_ws_bytes(1 << 24, 1, 8, fmt, 1) == 0
        _refused(call(N=(1 << 24) - 1, V=1, fmt=fmt, p=1), 1, b"workspace 0 bytes")


def test_a_piece_is_no_wider_than_its_offsets():
    """256 rows of a piece's dl lie within 2^31 bytes, so few rows do not make it wider than 2^21 tokens."""
    f = _lib.load().hsl_xent_ws_bytes
    more = [f(3, 1 << e, 8, 0, 1) - f(3, 1 << e, 8, 0, 0) for e in (21, 22, 24)]  # dl, beside what both keep
    assert more[0] >= 3 * 2 << 21 and more[1] <= more[0] and more[2] <= more[0]


def test_calls_without_positions_do_nothing():
    assert _fwd(N=0) == 0 and _bwd(N=0) == 0


def test_size_queries():
    f = _lib.load().hsl_xent_ws_bytes
    assert f(0, 5, 8, 0, 1) == 0 and f(-1, 5, 8, 0, 1) == 0 and f(4, 0, 8, 0, 1) == 0 and f(4, 5, 8, 7, 0) == 0
    assert f(1 << 40, 5, 8, 0, 1) == 0
    for fmt in (0, 1, 2):
        # neither direction has room for all the logits
        assert 0 < f(8192, 131072, 1024, fmt, 0) < 8192 * 131072 * 2
        assert 0 < f(8192, 131072, 1024, fmt, 1) < 8192 * 131072 * 2
        for n, v, d in ((1, 1, 1), (1, 131072, 2048), (100000, 3, 5), (257, 511, 33)):
            assert f(n, v, d, fmt, 0) > 0 and f(n, v, d, fmt, 1) > 0


def test_cpu_tensors_are_rejected():
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        prlstm_amd.linear_cross_entropy(torch.zeros(3, 4), torch.zeros(5, 4), torch.zeros(3, dtype=torch.int64))
