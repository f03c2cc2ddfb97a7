"""Refusals of the training-step operators that are made before any CUDA call."""
import ctypes

from suika_b200 import _lib as L

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
