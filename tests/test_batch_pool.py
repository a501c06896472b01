"""CPU checks of what the batched-serving tests rest on: the bounds that attention is held to reject an answer that lost a
page, a tail or a single position, and a slot of a fixed pool that stands by keeps its row."""
import numpy as np
import pytest

from __graft_entry__ import load_device
from batch_util import PAGE, attend, attend_bound_lifted, census, census_bound, pages_of, plan, slots_of

dev = load_device()


def test_a_slot_that_stands_by_keeps_its_row():
    """A negative length with one row asked for: refused, so it gets no page and keeps its length, but its row stays its
    own; every other slot's row is its index."""
    tables = np.array([[4, -1], [-1, -1], [5, -1], [6, -1]], np.int32)
    got = plan([1, 1, 1, 1], [10, -1, -1 - 20, 63], tables, [1, 2], 2, 4)
    assert got["row_starts"].tolist() == [0, 1, 2, 3, 4]
    assert got["lens"].tolist() == [11, -1, -21, 64] and got["counts"].tolist() == [2, 4, 2]
    assert got["slots"].tolist() == [4 * PAGE + 10, -1, -1, 6 * PAGE + 63]
    assert np.array_equal(got["tables"], tables) and got["n_free"] == 2


def test_no_sequences_are_no_work():
    """VV_OK, and nothing is written: positions, slots and the rest keep what they held (host memory here: no launch)."""
    held = [np.full(8, -77, np.int64) for _ in range(6)]
    lens, starts, positions, slots, left, counts = (x.ctypes.data for x in held)
    for n in (0, -1):
        assert dev.vv_kv_page_plan_dev(lens, lens, n, lens, 4, lens, left, lens, starts, positions, slots, 8, left, counts,
                                       None) == dev.VV_OK
    assert all((x == -77).all() for x in held)


def draw(n, nq, nkv, hd, rng, sharp=2.0):
    """Inputs of the distribution that the GPU tests' pools have."""
    q = rng.normal(size=(nq, hd)) * sharp * 2 * hd ** -0.25
    k = rng.normal(size=(n, nkv, hd)) * 2 * hd ** -0.25
    return tuple(x.astype(np.float16).astype(np.float64) for x in (q, k, rng.normal(size=(n, nkv, hd))))


def worst(got, ref, mag, n, v):
    return (np.abs(got - ref) / attend_bound_lifted(ref, mag, n, np.abs(v).max())).max()


@pytest.mark.parametrize("n", [1000, 14449, 20000])
def test_the_bound_sees_a_lost_page_and_a_lost_tail(n):
    rng = np.random.default_rng(n)
    q, k, v = draw(n, 4, 2, 128, rng)
    ref, mag = attend(q, k, v)
    for page in rng.integers(0, n // PAGE, 4):
        drop = np.arange(page * PAGE, (page + 1) * PAGE)
        assert worst(attend(q, np.delete(k, drop, 0), np.delete(v, drop, 0))[0], ref, mag, n, v) > 1.0
    assert worst(attend(q, k[:-17], v[:-17])[0], ref, mag, n, v) > 1.0
    assert worst(ref.astype(np.float16).astype(np.float64), ref, mag, n, v) <= 1.0


@pytest.mark.parametrize("n", [4, 64, 190])
def test_the_bound_sees_another_answer(n):
    """Zeros, the other sign, the heads in reverse, uniform weights and another query's answer, at the lengths and of the
    distribution that the serving loops have."""
    q, k, v = draw(n, 8, 2, 128, np.random.default_rng(n))
    ref, mag = attend(q, k, v)
    for wrong in (np.zeros_like(ref), -ref, ref[::-1], np.repeat(v.mean(0), 4, 0), attend(q[::-1], k, v)[0]):
        assert worst(wrong, ref, mag, n, v) > 1.0


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,lost", [(65, 1), (14449, 1), (20000, 1), (1 << 20, PAGE)])
def test_the_census_sees_what_is_lost_or_counted_twice(n, lost, hd):
    rng = np.random.default_rng(n)
    pages = rng.integers(0, 300, pages_of(n))
    want = census(pages, n, hd)
    at = slots_of(pages.astype(np.int32), n) // PAGE % hd
    assert np.array_equal(want, np.bincount(at, minlength=hd) / n)
    for begin in rng.integers(0, n // lost, 4) * lost:
        some = at[begin:begin + lost]
        for wrong in (np.bincount(np.delete(at, np.arange(begin, begin + lost)), minlength=hd) / (n - lost),
                      np.bincount(np.append(at, some), minlength=hd) / (n + lost)):
            assert (np.abs(wrong - want) > census_bound(want)).any()
