"""Plain restatements, in Python integers and 64-bit floats, of the batched-serving operators (vv_kv_page_plan_dev,
vv_rope_kv_append_dev, vv_attn_decode_batch), for the tests on the CPU and on the GPU."""
import numpy as np

PAGE = 64


def pages_of(n):
    return -(-n // PAGE)


def plan(new_lens, cache_lens, tables, free, n_free, max_rows):
    """One sequence after another, as the header words it. Returns a dict of the call's outputs."""
    n, max_pages = tables.shape
    tables = tables.copy()
    starts, lens = [0], list(cache_lens)
    positions, slots = np.zeros(max_rows, np.int32), np.full(max_rows, -1, np.int64)
    asked_pages = taken = refused = asked_by_served = 0
    n_free = max(n_free, 0)
    for i in range(n):
        new, held = max(int(new_lens[i]), 0), int(cache_lens[i])
        begin, end = starts[-1], starts[-1] + new
        starts.append(end)
        if new == 0:
            continue
        if held < 0 or held + new > max_pages * PAGE or end > max_rows:
            refused += 1
            continue
        need = pages_of(held + new) - pages_of(held)
        asked_pages += need
        if need and asked_pages > n_free:
            refused += 1
            continue
        for j in range(need):
            tables[i, pages_of(held) + j] = free[n_free - 1 - taken - j]
        taken += need
        asked_by_served = asked_pages
        lens[i] = held + new
        for r in range(new):
            p = held + r
            page = int(tables[i, p // PAGE])
            positions[begin + r] = p
            slots[begin + r] = page * PAGE + p % PAGE if page >= 0 else -1
    starts = np.minimum(np.array(starts, np.int64), max_rows).astype(np.int32)
    return {"tables": tables, "lens": np.array(lens, np.int32), "row_starts": starts, "positions": positions,
            "slots": slots, "n_free": n_free - taken,
            "counts": np.array([n_free - asked_by_served, starts[-1], refused], np.int32)}


def slots_of(table_row, length):
    t = np.arange(length)
    return table_row[t // PAGE].astype(np.int64) * PAGE + t % PAGE


def attend(q, k, v):
    """q [nq][hd], k, v [n][nkv][hd] (float64) -> (out [nq][hd], weighted mean of |v| [nq][hd])."""
    nq, hd = q.shape
    group = nq // k.shape[1]
    out, mag = np.zeros((nq, hd)), np.zeros((nq, hd))
    if k.shape[0] == 0:
        return out, mag
    for h in range(nq):
        s = k[:, h // group] @ q[h] / np.sqrt(hd)
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h] = p @ v[:, h // group]
        mag[h] = p @ np.abs(v[:, h // group])
    return out, mag


def attend_bound(ref, mag, n, vmax):
    """What the kernel may be off. The probabilities of the second product are rounded to FP16: half a step, 2^-11 of
    each, or 2^-25 of the largest one where they are subnormal - n of those at most, each times a value. The scores'
    FP32 sums, the exponential and the sums of the join: below 2^-14 of a probability at these sizes (scores up to
    about 100, each off by some ten half steps of FP32, 2^-24). Then the one rounding of the result.

    The kernels form probabilities on a lifted scale, so the second term is 2^10 times what they can be off: at some 10^4
    positions it hides a lost page. attend_bound_lifted is without that slack."""
    with np.errstate(over="ignore"):
        ulp = np.spacing(np.abs(ref).astype(np.float16)).astype(np.float64)
    return mag * (2.0 ** -11 + 2.0 ** -14) + n * 2.0 ** -25 * vmax + 0.5 * ulp + 1e-12


def attend_bound_lifted(ref, mag, n, vmax):
    """attend_bound for the matrix kernels as they form a probability: 2^10 times it, on the scale of its row's maximum.
    FP16 is then off by half a step, 2^-11 of it, or, below 2^-14 on the lifted scale, by half of the smallest subnormal,
    2^-25 there: 2^-35 of the largest probability, for n of them at most, each times a value (the row's sum is at least
    that largest probability; a maximum that was still rising only makes the error smaller when it is scaled down). The
    other terms are attend_bound's."""
    with np.errstate(over="ignore"):
        ulp = np.spacing(np.abs(ref).astype(np.float16)).astype(np.float64)
    return mag * (2.0 ** -11 + 2.0 ** -14) + n * 2.0 ** -35 * vmax + 0.5 * ulp + 1e-12


def census(pages, length, hd):
    """What attention answers where every score is alike and the values of page p are 1 in channel p % hd, 0 elsewhere:
    each channel's share of the first `length` positions behind `pages`. One position lost or counted twice shows up to
    some 10^5 positions, one page up to 10^6."""
    held = np.full(len(pages), PAGE, np.int64)
    if len(pages):
        held[-1] = length - PAGE * (len(pages) - 1)
    return np.bincount(np.asarray(pages) % hd, weights=held, minlength=hd) / max(length, 1)


def census_bound(want):
    """The probabilities are all 2^10, which FP16 holds exactly (a step of FP32 in the exponential is 2^-23 of the row's
    sum), sums of up to 2^24 of them are exact, and the reciprocal is off by 2^-23; then the one rounding."""
    ulp = np.spacing(want.astype(np.float16)).astype(np.float64)
    return want * 2.0 ** -20 + 0.5 * ulp
