"""Refusals of the training-step operators that are made before any CUDA call."""
import ctypes

import numpy as np
import torch

from suika_b200 import _lib as L
from suika_b200 import vocab as V

FAKE = 1 << 20  # an address that no check dereferences


def test_shard_gradient_entry_checks_the_vocabulary():
    lib = L.load()

    def call(first, end, lo=16, cols=8, sharded=1):
        o = L.RsLogprobOpts(4, cols, 8, lo, 0, 1, 0, sharded)
        return lib.rs_token_logprobs_shard_grad(ctypes.byref(o), first, end, FAKE, FAKE, FAKE, FAKE, None, None, None, FAKE, 8, 0, None)
    for first, end in ((17, 24), (0, 23), (24, 16), (-(1 << 63), 0)):
        assert call(first, end) == L.RS_ERR_ARG and b"vocabulary" in lib.rs_last_error(), (first, end)
    assert call(0, 24, sharded=0) == L.RS_ERR_ARG and b"sharded" in lib.rs_last_error()
    assert call(16, 24) == L.RS_ERR_ARG and b"NULL" in lib.rs_last_error()  # the rest as in the entry without a range
    assert lib.rs_token_logprobs_shard_grad(None, 0, 8, *[FAKE] * 8, 8, 0, None) == L.RS_ERR_ARG


def test_record_entry_checks_its_index_base():
    lib = L.load()

    def call(base, cols=8):
        return lib.rs_token_record_at(ctypes.byref(L.RsLogprobOpts(4, cols, 8, 0, 0, 1, 2, 1)), base, FAKE, None, FAKE, 0, None)
    assert call(-1) == L.RS_ERR_ARG and b"negative" in lib.rs_last_error()
    for base in ((1 << 31) - 8, 1 << 31, (1 << 63) - 1):
        assert call(base) == L.RS_ERR_CAPACITY, base
    assert call((1 << 31) - 9) == L.RS_ERR_ARG and b"NULL" in lib.rs_last_error()


def _rows_meet(rows, n, pitch, width, out, size):
    return any(rows + i * pitch < out + size and out < rows + i * pitch + width for i in range(n)) and width > 0 and size > 0


def test_embedding_gradient_entry_refuses_its_own_input():
    """Every place of a small output about a few rows, with gaps, without, and on top of one another, against a search."""
    lib = L.load()
    for n, stride, hidden in ((1, 8, 8), (3, 8, 8), (3, 12, 8), (3, 0, 8), (4, 6, 8)):
        for out_rows in (1, 2):
            for at in range(-24, 60):
                rows, out = FAKE, FAKE + 4 * at
                o = L.RsEmbedOpts(n, out_rows, hidden, 0, hidden, stride, 1.0, L.RS_F32, L.RS_F32, 1, 0, 0)
                rc = lib.rs_embed_grad(ctypes.byref(o), FAKE * 2, rows, out, None, 0, 0, None)
                meet = _rows_meet(rows, n, 4 * stride, 4 * hidden, out, 4 * hidden * out_rows)
                assert rc == (L.RS_ERR_ARG if meet else L.RS_ERR_CAPACITY), (n, stride, out_rows, at, lib.rs_last_error())  # no workspace was given
                if meet:
                    assert b"overlaps" in lib.rs_last_error()


def test_embedding_gradient_of_long_batches_refuses_its_own_input():
    whole = torch.zeros(200)
    for n, stride, hidden in ((1, 8, 8), (3, 8, 8), (3, 12, 8), (3, 0, 8), (4, 6, 8), (5, 1, 1)):
        g = whole[40:].as_strided((n, hidden), (stride, 1), 40)
        for out_rows in (1, 2):
            for at in range(0, 150):
                out = whole[at:at + out_rows * hidden].view(out_rows, hidden)
                meet = _rows_meet(40, n, stride, hidden, at, out_rows * hidden)
                assert V._touches(g, out) == meet, (n, stride, hidden, out_rows, at)
    assert not V._touches(whole[:0].view(0, 4), whole[:8].view(2, 4)) and not V._touches(whole[:8].view(2, 4), whole[:0].view(0, 4))


def test_entries_refuse_misaligned_addresses():
    """Statistics, results and workspaces are 4 or 8 bytes wide: an address between two of them would fault on the device."""
    lib = L.load()
    span = np.array([(FAKE, 4, L.RS_F32, 0)], dtype=L.GRAD_SPAN_DTYPE)
    assert lib.rs_grad_sumsq(span.ctypes.data, 1, FAKE + 4, 1 << 20, FAKE, 0, None) == L.RS_ERR_CAPACITY
    assert lib.rs_grad_sumsq(span.ctypes.data, 1, FAKE, 1 << 20, FAKE + 4, 0, None) == L.RS_ERR_ARG
    assert lib.rs_grad_clip(span.ctypes.data, 1, FAKE + 4, 1.0, FAKE, 0, None) == L.RS_ERR_ARG
    assert lib.rs_grad_clip(span.ctypes.data, 1, FAKE, 1.0, FAKE + 2, 0, None) == L.RS_ERR_ARG
    adam = np.array([(FAKE,) * 6 + (4, 0.0, 0, 0, 0)], dtype=L.ADAMW_TENSOR_DTYPE)
    opts = L.RsAdamwOpts(1e-3, 0.9, 0.99, 1e-8, 1.0)
    for sumsq, norm in ((FAKE + 4, FAKE), (FAKE, FAKE + 2)):
        assert lib.rs_adamw_step(adam.ctypes.data, 1, ctypes.byref(opts), sumsq, norm, FAKE, 1 << 20, 0, None) == L.RS_ERR_ARG
        assert b"misaligned" in lib.rs_last_error()
    o = L.RsLogprobOpts(4, 8, 8, 0, L.RS_F32, 1, 2, 0)
    outs = [FAKE] * 5
    for i in range(5):
        bad = list(outs)
        bad[i] += 2 if i < 4 else 4
        assert lib.rs_token_logprobs(ctypes.byref(o), FAKE, FAKE, *bad, 0, None) == L.RS_ERR_ARG and b"aligned" in lib.rs_last_error()
        starts = np.zeros(1, np.int64)
        assert lib.rs_token_merge(FAKE, starts.ctypes.data, 1, 4, 2, *bad, 0, None) == L.RS_ERR_ARG and b"aligned" in lib.rs_last_error()
    assert lib.rs_token_merge(FAKE + 2, starts.ctypes.data, 1, 4, 2, *outs, 0, None) == L.RS_ERR_ARG
    assert lib.rs_token_record(ctypes.byref(o), FAKE, FAKE, FAKE + 2, 0, None) == L.RS_ERR_ARG
    for i in range(5):
        bad = list(outs)
        bad[i] += 2
        assert lib.rs_token_logprobs_grad(ctypes.byref(o), FAKE, FAKE, *bad, FAKE, 8, 0, None) == L.RS_ERR_ARG and b"aligned" in lib.rs_last_error()
