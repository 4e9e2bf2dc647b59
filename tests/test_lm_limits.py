"""The ends of the sizes that the language-model operators take, as the host refuses them (no GPU)."""

from prlstm_amd import _lib

UNSUPPORTED = 2


def _refused(rc, text):
    assert rc == UNSUPPORTED and text in _lib.load().hsl_last_error(), (rc, _lib.load().hsl_last_error())


def test_embedding_gradients_beyond_one_launch_are_refused():
    """The sort has 1024 threads for 512 tokens, the sums 256 for 16 kB of the gradient; a launch holds
    fewer than 2^32 threads.  (The pointers are not looked at before the sizes.)"""
    bwd = _lib.load().hsl_embed_bwd
    for v, d, fmt in (((1 << 30) + 1, 1, 0), (1 << 28, 512, 0), (1 << 28, 264, 1), (1 << 28, 256, 2)):
        _refused(bwd(1, 0, 1, d, 1.0, -1, 1, 1, 0, 8, v, d, fmt, None), b"beyond one launch")
    # the last sizes that are taken get as far as the workspace
    for v, d, fmt in ((1 << 30, 1, 0), ((1 << 28) - 64, 512, 0), (1 << 28, 256, 0)):
        assert bwd(1, 0, 1, d, 1.0, -1, 1, 1, 0, 8, v, d, fmt, None) == 1
        assert b"workspace 0 bytes" in _lib.load().hsl_last_error()


def test_size_queries_of_refused_sizes():
    """They end, and say 0, whatever they are asked."""
    lib = _lib.load()
    most = (1 << 63) - 1
    for n in (0x7FFF0001, 1 << 43, 1 << 60, most):
        assert lib.hsl_embed_bwd_ws_bytes(n, 5, 5) == 0
    for t, b, h in ((4096, 1 << 20, 1 << 18), (4096, 1 << 30, 1 << 30), (0x7FFFFFFF, 1, 64), (1 << 20, 0x7FFFFFFF, 1)):
        assert lib.hsl_gated_ws_bytes(t, b, h) == 0
    for n in (1 << 40, most):
        assert lib.hsl_logprob_fwd_ws_bytes(n, 0x7FFF0000, 1) == 0
    assert lib.hsl_embed_bwd_ws_bytes(0x7FFF0000, 0x7FFF0000, 1) > 0
    assert lib.hsl_gated_ws_bytes((1 << 30) - 1, 1, 64) > 0


def test_channels_of_the_gated_recurrence():
    """It has no weight whose elements could pass 2^31: any width is taken up to 2^27 channels in all."""
    fwd = _lib.load().hsl_gated_fwd
    call = lambda t, b, h: fwd(None, 0, 0, None, None, 0, 0, None, 0, 0, None, None, None, 0, t, b, h, 0, None)  # noqa: E731
    for t, b, h in ((1, 2, 40001), (3, 1, (1 << 27) - 1), ((1 << 30) - 1, 1000, 1000)):
        assert call(t, b, h) == 1 and b"null pointer" in _lib.load().hsl_last_error()
    for t, b, h in ((3, 1, 1 << 27), (3, 1 << 20, 1 << 10), (1 << 30, 1, 1), (1, 0x7FFFFFFF, 0x7FFFFFFF)):
        _refused(call(t, b, h), b"index range")


def test_checkpoint_rows():
    """One state for each 16 steps that begin."""
    rows = _lib.load().hsl_gated_ck_rows
    assert [rows(t) for t in (-1, 0, 1, 15, 16, 17, 32, 33, 4096, 4097)] == [0, 0, 1, 1, 1, 2, 2, 3, 256, 257]
