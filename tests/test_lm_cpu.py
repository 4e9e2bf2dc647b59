"""Host-side checks of the language-model operators that need no GPU."""

import pytest
import torch

import prlstm_amd
from prlstm_amd import _lib


def test_entry_points_refuse_bad_arguments():
    lib = _lib.load()

    def refused(rc, code, text):
        assert rc == code and text in lib.hsl_last_error(), (rc, lib.hsl_last_error())

    n = None
    refused(lib.hsl_embed_fwd(n, 0, n, 4, 1.0, n, 3, 5, 4, 9, n), 1, b"format 9")
    refused(lib.hsl_embed_fwd(n, 0, n, 4, 1.0, n, -3, 5, 4, 0, n), 1, b"negative size")
    refused(lib.hsl_embed_fwd(n, 0, n, 4, 1.0, n, 3, 5, 4, 0, n), 1, b"null pointer")
    refused(lib.hsl_embed_fwd(n, 0, n, 4, 1.0, n, 1 << 31, 5, 4, 0, n), 2, b"2^31")
    refused(lib.hsl_embed_bwd(n, 0, n, 4, 1.0, -1, n, n, 0, 3, 5, 4, 0, n), 1, b"null pointer")
    refused(lib.hsl_embed_bwd(1, 0, 1, 4, 1.0, -1, 1, n, 0, 3, 5, 4, 0, n), 1, b"workspace 0 bytes")
    refused(lib.hsl_gated_fwd(n, 0, 0, n, n, 0, 0, n, 0, 0, n, n, n, 0, 4, 2, 3, 0, n), 1, b"null pointer")
    refused(lib.hsl_gated_fwd(n, 0, 0, n, n, 0, 0, n, 0, 0, n, n, n, 0, 4, -2, 3, 0, n), 1, b"negative")
    refused(lib.hsl_gated_fwd(n, 0, 0, n, n, 0, 0, n, 0, 0, n, n, n, 0, 4, 2, 3, 3, n), 1, b"format 3")
    refused(lib.hsl_gated_fwd(n, 0, 0, n, n, 0, 0, n, 0, 0, n, n, n, 0, 1 << 30, 2, 3, 0, n), 2, b"index range")
    refused(lib.hsl_gated_bwd(n, 0, 0, n, 0, 0, n, n, 0, 0, n, n, 0, 0, n, n, 0, 4, 2, 3, 0, n), 1, b"null pointer")
    refused(lib.hsl_logprob_fwd(n, 5, n, 0, n, n, n, n, n, n, 0, 2, 5, 6, 0, n), 1, b"top=6")
    refused(lib.hsl_logprob_fwd(n, 5, n, 0, n, n, n, n, n, n, 0, 2, 50, 33, 0, n), 1, b"top=33")
    refused(lib.hsl_logprob_fwd(n, 5, n, 0, n, n, n, n, n, n, 0, 2, 5, 2, 0, n), 1, b"null pointer")
    refused(lib.hsl_logprob_bwd(n, 5, n, 0, n, n, n, n, n, n, n, 5, 2, 5, 0, 0, n), 1, b"null pointer")
    refused(lib.hsl_logprob_bwd(n, 5, n, 0, n, n, n, n, n, n, n, 5, -2, 5, 0, 0, n), 1, b"negative size")


def test_empty_calls_do_nothing():
    lib = _lib.load()
    n = None
    assert lib.hsl_embed_fwd(n, 0, n, 4, 1.0, n, 0, 5, 4, 0, n) == 0
    assert lib.hsl_embed_bwd(n, 0, n, 4, 1.0, -1, n, n, 0, 3, 0, 4, 0, n) == 0
    assert lib.hsl_gated_fwd(n, 0, 0, n, n, 0, 0, n, 0, 0, n, n, n, 0, 4, 0, 3, 0, n) == 0
    assert lib.hsl_logprob_fwd(n, 5, n, 0, n, n, n, n, n, n, 0, 0, 5, 0, 0, n) == 0
    assert lib.hsl_logprob_bwd(n, 5, n, 0, n, n, n, n, n, n, n, 5, 0, 5, 0, 0, n) == 0


def test_size_queries():
    lib = _lib.load()
    assert lib.hsl_embed_bwd_ws_bytes(-1, 5, 5) == 0
    assert lib.hsl_embed_bwd_ws_bytes(1000, 5, 8) >= 1000 * 4  # the positions by token
    assert lib.hsl_gated_ck_rows(0) == 0 and lib.hsl_gated_ck_rows(1) == 1
    assert lib.hsl_gated_ck_rows(4096) < 4096 and lib.hsl_gated_ck_rows(4097) > lib.hsl_gated_ck_rows(4096) - 1
    for f in (lib.hsl_gated_ws_bytes,):
        assert f(-1, 1, 1) == 0 and f(100, 0, 5) == f(100, 5, 0) == 0


def test_cpu_tensors_are_rejected():
    ids = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        prlstm_amd.embedding(ids, torch.zeros(4, 6))
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        prlstm_amd.gated_recurrence(torch.zeros(5, 2, 8))
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        prlstm_amd.gated_recurrence_step(torch.zeros(2, 8), torch.zeros(2, 4))
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        prlstm_amd.token_logprobs(torch.zeros(3, 6), ids)
