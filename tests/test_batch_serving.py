"""CPU checks of the batched-serving entry points: what they refuse, what counts as no work, the scratch they ask for,
and the plain page plan that the GPU tests hold the kernel to."""
import ctypes as C

import numpy as np
import pytest

from __graft_entry__ import load_device
from batch_util import PAGE, pages_of, plan, slots_of

dev = load_device()
P = 0x1000      # a non-null, 16-byte aligned stand-in; never dereferenced by these calls


def plan_call(**change):
    a = dict(new_lens=P, cache_lens=P + 64, n_seqs=4, tables=P, max_pages=8, free=P, n_free=P, lens_out=P + 128,
             row_starts=P, positions=P, slots=P, max_rows=16, n_free_out=P + 192, counts=P + 256,
             stream=None)
    a.update(change)
    return dev.vv_kv_page_plan_dev(*a.values())


def append_call(**change):
    a = dict(q=P, k=P, v=P, q_bias=None, k_bias=None, v_bias=None, positions=P, slots=P, q_out=P, k_store=P, v_store=P,
             n_rows=3, n_q_heads=4, n_kv_heads=2, head_dim=128, n_pages=4, kv_format=0, theta=1e6, stream=None)
    a.update(change)
    return dev.vv_rope_kv_append_dev(*a.values())


def attend_call(view=None, **change):
    v = dict(k=P, v=P, k_meta=None, v_meta=None, page_table=P, format=0, n_kv_heads=2, head_dim=128)
    v.update(view or {})
    kv = dev.KvView(**v)
    a = dict(backend=2, q=P, kv=C.addressof(kv), out=P, n_q_heads=4, n_seqs=3, cache_lens=P, max_pages=8, n_pages=4,
             scratch=P, scratch_bytes=1 << 40, stream=None)
    a.update(change)
    return dev.vv_attn_decode_batch(*a.values())


@pytest.mark.parametrize("name", ["new_lens", "cache_lens", "tables", "free", "n_free", "lens_out", "row_starts",
                                  "positions", "slots", "counts"])
def test_plan_null(name):
    assert plan_call(**{name: None}) == dev.VV_ERR_NULL_PTR


def test_plan_refusals():
    assert plan_call(n_seqs=0) == dev.VV_OK
    assert plan_call(n_seqs=-1) == dev.VV_OK
    assert plan_call(max_pages=0) == dev.VV_ERR_INVALID_ARG
    assert plan_call(max_rows=-1) == dev.VV_ERR_INVALID_ARG
    assert plan_call(lens_out=P) == dev.VV_ERR_INVALID_ARG            # the lengths over the request they follow from
    assert plan_call(counts=P) == dev.VV_ERR_INVALID_ARG              # the counts over the number of free pages
    assert plan_call(counts=P + 192) == dev.VV_ERR_INVALID_ARG        # or over what is left of them
    assert plan_call(max_rows=(1 << 30) + 1) == dev.VV_ERR_UNSUPPORTED


@pytest.mark.parametrize("name", ["q", "k", "v", "positions", "slots", "q_out", "k_store", "v_store"])
def test_append_null(name):
    assert append_call(**{name: None}) == dev.VV_ERR_NULL_PTR


def test_append_refusals():
    assert append_call(n_rows=0) == dev.VV_OK
    for name in ("n_q_heads", "n_kv_heads", "head_dim", "n_pages"):
        assert append_call(**{name: 0}) == dev.VV_ERR_INVALID_ARG
    assert append_call(head_dim=127) == dev.VV_ERR_UNSUPPORTED
    assert append_call(head_dim=258) == dev.VV_ERR_UNSUPPORTED
    for fmt in (3, 4, 5, 6, 9, -1):
        assert append_call(kv_format=fmt) == dev.VV_ERR_UNSUPPORTED
    for fmt in (1, 2):
        assert append_call(kv_format=fmt, head_dim=64) == dev.VV_ERR_UNSUPPORTED
        for name in ("q", "k", "v", "q_out", "q_bias", "k_bias", "v_bias"):
            assert append_call(kv_format=fmt, **{name: P + 2}) == dev.VV_ERR_UNSUPPORTED
        assert append_call(kv_format=fmt, k_store=P + 4) == dev.VV_ERR_UNSUPPORTED


@pytest.mark.parametrize("name", ["q", "kv", "out", "cache_lens", "scratch"])
def test_attend_null(name):
    assert attend_call(**{name: None}) == dev.VV_ERR_NULL_PTR


def test_attend_refusals():
    assert attend_call(n_seqs=0) == dev.VV_OK
    for name in ("k", "v", "page_table"):
        assert attend_call({name: None}) == dev.VV_ERR_NULL_PTR
    for fmt in (3, 4, 5, 6, 9, -1):
        assert attend_call({"format": fmt}) == dev.VV_ERR_UNSUPPORTED
    assert attend_call({"format": 1, "head_dim": 64}) == dev.VV_ERR_UNSUPPORTED
    assert attend_call({"format": 1, "k": P + 8}) == dev.VV_ERR_UNSUPPORTED
    assert attend_call({"head_dim": 258}) == dev.VV_ERR_UNSUPPORTED
    assert attend_call({"head_dim": 0}) == dev.VV_ERR_UNSUPPORTED
    assert attend_call({"n_kv_heads": 3}) == dev.VV_ERR_UNSUPPORTED
    assert attend_call(n_q_heads=0) == dev.VV_ERR_UNSUPPORTED
    assert attend_call(n_q_heads=16386) == dev.VV_ERR_UNSUPPORTED
    for name in ("max_pages", "n_pages"):
        assert attend_call(**{name: 0}) == dev.VV_ERR_INVALID_ARG
    assert attend_call(max_pages=1 << 25) == dev.VV_ERR_UNSUPPORTED             # positions past 32 bits
    assert attend_call(n_seqs=1 << 16, max_pages=1 << 15) == dev.VV_ERR_UNSUPPORTED
    assert attend_call(n_seqs=(1 << 21) + 1, max_pages=1) == dev.VV_ERR_UNSUPPORTED     # rows past a launch
    need = dev.vv_attn_decode_batch_scratch_bytes(3, 4, 2, 128)
    assert attend_call(scratch_bytes=need - 1) == dev.VV_ERR_INVALID_ARG
    assert attend_call(scratch=P + 4) == dev.VV_ERR_INVALID_ARG


def test_scratch_grows_with_the_sequences_by_their_count_alone():
    size = dev.vv_attn_decode_batch_scratch_bytes
    assert size(0, 4, 2, 128) == size(3, 4, 3, 128) == size(3, 0, 2, 128) == size(3, 4, 2, 0) == 0
    one = size(1, 28, 4, 128)
    assert 0 < one < 64 << 20
    assert one <= size(100, 28, 4, 128) <= one + 100 * 4 * 8 + 256
    assert size(1, 40, 2, 128) >= size(1, 20, 2, 128)


def test_the_plain_plan_hands_out_pages_like_a_stack():
    tables = np.array([[5, -1, -1], [-1, -1, -1], [7, 8, -1]], np.int32)
    got = plan([1, 65, 1], [64, 0, 127], tables, [20, 21, 22, 23], 4, 70)
    assert got["tables"].tolist() == [[5, 23, -1], [22, 21, -1], [7, 8, -1]]
    assert got["lens"].tolist() == [65, 65, 128] and got["counts"].tolist() == [1, 67, 0]
    assert got["n_free"] == 1
    assert got["row_starts"].tolist() == [0, 1, 66, 67]
    assert got["slots"][0] == 23 * PAGE and got["slots"][1] == 22 * PAGE and got["slots"][65] == 21 * PAGE
    assert got["slots"][66] == 8 * PAGE + 63 and (got["slots"][67:] == -1).all()
    assert got["positions"][[0, 1, 65, 66]].tolist() == [64, 0, 64, 127]
    assert slots_of(got["tables"][1], 65)[64] == 21 * PAGE
    # too few pages: the second is refused, and the third, which needs one, does not overtake it; the fourth needs none
    tables = np.array([[5, -1], [-1, -1], [6, -1], [7, -1]], np.int32)
    got = plan([1, 128, 1, 1], [64, 0, 64, 3], tables, [20, 21], 2, 200)
    assert got["lens"].tolist() == [65, 0, 64, 4] and got["n_free"] == 1
    assert got["counts"].tolist() == [-2, 131, 2]        # 2 less the 1 + 2 + 1 asked for up to the last one served
    assert (got["slots"][1:130] == -1).all() and got["slots"][130] == 7 * PAGE + 3
    assert pages_of(0) == 0 and pages_of(1) == 1 and pages_of(64) == 1 and pages_of(65) == 2


def test_counts_past_what_a_launch_or_32_bits_hold_are_refused():
    assert plan_call(n_seqs=(1 << 30) + 1) == dev.VV_ERR_UNSUPPORTED
    assert plan_call(max_pages=1 << 25) == dev.VV_ERR_UNSUPPORTED                # 2^31 positions
    # rows of 28 + 2 * 4 heads of 8 items run 320 threads: floor((2^32 - 1) / 320) of them fit a launch
    wide = dict(n_q_heads=28, n_kv_heads=4)
    assert append_call(n_rows=(2**32 - 1) // 320 + 1, **wide) == dev.VV_ERR_UNSUPPORTED
    assert append_call(n_rows=(2**32 - 1) // 256 + 1, head_dim=126) == dev.VV_ERR_UNSUPPORTED
