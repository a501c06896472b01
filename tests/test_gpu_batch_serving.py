"""GPU tests of the batched-serving operators through the C ABI: the page plan against a plain restatement, the rotary
append against the separate calls it replaces (bit for bit) and the closed form, decode attention over a paged pool
against 64-bit sums, and the three of them together as a serving loop runs them, also captured and replayed.

What a pool holds where no position lies is NaN here: a kernel that lets any of it into a result shows."""
import ctypes as C

import numpy as np
import pytest
import torch

import oracle
from batch_util import PAGE, attend, attend_bound, pages_of, plan, slots_of
from gpu_util import bits_of, dev, ok, stream, to_dev

pytestmark = pytest.mark.gpu
FP16, E4M3, E5M2 = 0, 1, 2
TORCH_FP8 = {E4M3: torch.float8_e4m3fn, E5M2: torch.float8_e5m2}


def ints(values, dtype=torch.int32):
    return torch.tensor(np.asarray(values), dtype=dtype, device="cuda")


# ── the page plan ────────────────────────────────────────────────────────────

def run_plan(new, lens, tables, free, n_free, max_rows, in_place=False, pad=7):
    n, max_pages = tables.shape
    d = dict(new=ints(new), lens=ints(lens), tables=ints(tables), free=ints(free if len(free) else [0]),
             counts=torch.full((3,), -77, dtype=torch.int32, device="cuda"))
    d["n_free"] = ints([n_free])
    d["n_free_out"] = d["n_free"] if in_place else ints([-77])
    d["lens_out"] = d["lens"] if in_place else torch.full((n,), -77, dtype=torch.int32, device="cuda")
    d["starts"] = torch.full((n + 1 + pad,), -77, dtype=torch.int32, device="cuda")
    d["positions"] = torch.full((max_rows + pad,), -77, dtype=torch.int32, device="cuda")
    d["slots"] = torch.full((max_rows + pad,), -77, dtype=torch.int64, device="cuda")
    ok(dev.vv_kv_page_plan_dev(d["new"].data_ptr(), d["lens"].data_ptr(), n, d["tables"].data_ptr(), max_pages,
                               d["free"].data_ptr(), d["n_free"].data_ptr(), d["lens_out"].data_ptr(),
                               d["starts"].data_ptr(), d["positions"].data_ptr(), d["slots"].data_ptr(), max_rows,
                               d["n_free_out"].data_ptr(), d["counts"].data_ptr(), stream()))
    torch.cuda.synchronize()
    assert (d["starts"][n + 1:] == -77).all() and (d["positions"][max_rows:] == -77).all() and \
        (d["slots"][max_rows:] == -77).all(), "written past the end"
    return {"tables": d["tables"].cpu().numpy(), "lens": d["lens_out"].cpu().numpy(),
            "row_starts": d["starts"][:n + 1].cpu().numpy(), "positions": d["positions"][:max_rows].cpu().numpy(),
            "slots": d["slots"][:max_rows].cpu().numpy(), "counts": d["counts"].cpu().numpy(),
            "n_free": int(d["n_free_out"])}


def check_plan(new, lens, max_pages, n_free, max_rows, seed, in_place=False):
    rng = np.random.default_rng(seed)
    n = len(new)
    tables = np.full((n, max_pages), -1, np.int32)
    held = sum(pages_of(max(x, 0)) for x in lens)
    perm = rng.permutation(held + max(n_free, 0) + 3).astype(np.int32)
    at = 0
    for i, x in enumerate(lens):
        m = min(pages_of(max(x, 0)), max_pages)
        tables[i, :m] = perm[at:at + m]
        at += m
    free = perm[at:at + max(n_free, 0)]
    want = plan(new, lens, tables, free, n_free, max_rows)
    got = run_plan(new, lens, tables, free, n_free, max_rows, in_place)
    for name in want:
        assert np.array_equal(got[name], want[name]), name
    return want


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,top,chunk,rows,free", [
    (1, 0, 1, 1, 1), (1, 64, 1, 1, 0), (1, 0, 4097, 4097, 65), (64, 1000, 1, 64, 64), (64, 1000, 1, 80, 3),
    (65, 300, 2, 200, 40), (193, 2000, 9, 700, 30), (256, 90, 40, 3000, 100), (257, 90, 40, 9000, 1000),
    (1024, 700, 1, 1024, 1024), (1025, 200, 3, 2100, 100), (2600, 130, 5, 9000, 3000), (31, 3000, 900, 20000, 400)])
def test_plan(n, top, chunk, rows, free, in_place):
    rng = np.random.default_rng(n + rows)
    new = rng.integers(0, chunk + 1, n) if chunk > 1 else np.ones(n, int)
    lens = rng.integers(0, top + 1, n)
    check_plan(new, lens, pages_of(top + chunk) + 1, free, rows, n, in_place)


def test_plan_refuses_one_at_a_time():
    # refused: a negative length, 120 + 10 > 128 positions, 0 + 200 > 128; a negative request asks for nothing
    want = check_plan([2, 1, -5, 10, 200, 3, 1], [63, -1, 5, 120, 0, 1, 64], 2, 3, 300, 1)
    assert want["counts"].tolist() == [1, 217, 3] and want["n_free"] == 1 and want["lens"].tolist() == [65, -1, 5, 120, 0, 4, 65]
    check_plan([0, 0, 0], [5, 0, 64], 2, 0, 4, 2)                       # nothing asked
    check_plan([1, 1], [5, 7], 1, 0, 0, 3)                              # no rows at all
    check_plan([1, 1], [64, 7], 2, -4, 3, 4)                            # a pool that is overdrawn already
    check_plan([2 ** 31 - 1, 1, 2 ** 31 - 1, 1], [5, 7, 2 ** 31 - 1, 9], 3, 9, 40, 5)      # sums past 32 bits


def test_plan_captured_advances_itself():
    """In place under a graph: every replay appends one position to each sequence, as a decode loop does."""
    n, max_pages, pool = 37, 4, 37 * 4
    rng = np.random.default_rng(7)
    lens = rng.integers(0, 130, n).astype(np.int32)
    tables = np.full((n, max_pages), -1, np.int32)
    perm = rng.permutation(pool).astype(np.int32)
    at = 0
    for i, x in enumerate(lens):
        tables[i, :pages_of(x)] = perm[at:at + pages_of(x)]
        at += pages_of(x)
    free, n_free = perm[at:], pool - at
    d_new, d_lens, d_tables, d_free = ints(np.ones(n)), ints(lens), ints(tables), ints(free)
    d_n_free, counts = ints([n_free]), ints([0, 0, 0])
    starts = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    positions = torch.zeros(n, dtype=torch.int32, device="cuda")
    slots = torch.zeros(n, dtype=torch.int64, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    h = C.c_void_p()
    ok(dev.vv_dev_graph_begin(s.cuda_stream))
    ok(dev.vv_kv_page_plan_dev(d_new.data_ptr(), d_lens.data_ptr(), n, d_tables.data_ptr(), max_pages,
                               d_free.data_ptr(), d_n_free.data_ptr(), d_lens.data_ptr(), starts.data_ptr(),
                               positions.data_ptr(), slots.data_ptr(), n, d_n_free.data_ptr(), counts.data_ptr(),
                               s.cuda_stream))
    ok(dev.vv_dev_graph_end(s.cuda_stream, C.byref(h)))
    for _ in range(70):
        want = plan(np.ones(n, int), lens, tables, free, n_free, n)
        ok(dev.vv_dev_graph_launch(h, s.cuda_stream))
        ok(dev.vv_dev_stream_sync(s.cuda_stream))
        lens, tables, n_free = want["lens"], want["tables"], want["n_free"]
        assert int(d_n_free) == n_free
        assert np.array_equal(d_lens.cpu().numpy(), lens) and np.array_equal(d_tables.cpu().numpy(), tables)
        assert np.array_equal(slots.cpu().numpy(), want["slots"]) and np.array_equal(counts.cpu().numpy(),
                                                                                     want["counts"])
    dev.vv_dev_graph_destroy(h)


# ── bias, rotation, append ───────────────────────────────────────────────────

def new_store(n_pages, nkv, hd, fmt):
    if fmt == FP16:
        return torch.full((n_pages * PAGE, nkv, hd), float("nan"), dtype=torch.float16, device="cuda")
    return torch.full((n_pages * PAGE, nkv, hd), 0x7F, dtype=torch.uint8, device="cuda")


def raw(t):
    torch.cuda.synchronize()
    return t.contiguous().view(torch.uint8).cpu().numpy()


def separate_calls(q, k, v, biases, positions, slots, n_pages, fmt):
    """The same rows one at a time through the entry points that serve one sequence."""
    rows, nq, hd = q.shape
    nkv = k.shape[1]
    q, k, v = q.clone(), k.clone(), v.clone()
    for x, b in zip((q, k, v), biases):
        if b is not None:
            ok(dev.vv_bias_add_dev(x.data_ptr(), b.data_ptr(), rows, x.shape[1] * hd, stream()))
    ks, vs = new_store(n_pages, nkv, hd, fmt), new_store(n_pages, nkv, hd, fmt)
    out = torch.full_like(q, float("nan"))
    for r in range(rows):
        if not 0 <= slots[r] < n_pages * PAGE:
            continue
        ok(dev.vv_rope_qk_dev(q[r].data_ptr(), k[r].data_ptr(), 1, nq, nkv, hd, int(positions[r]), None, 1e6, stream()))
        ok(dev.vv_kv_store_dev(k[r].data_ptr(), v[r].data_ptr(), ks.data_ptr(), vs.data_ptr(), None, None, None, False,
                               nkv, hd, int(slots[r]), None, 1, fmt, None, stream()))
        out[r] = q[r]
    return out, ks, vs


APPEND = [(1, 28, 4, 128, FP16), (17, 28, 4, 128, FP16), (70, 12, 2, 128, FP16), (33, 14, 2, 64, FP16),
          (9, 1, 1, 128, FP16), (9, 3, 3, 64, FP16), (6, 40, 8, 128, FP16), (300, 2, 1, 128, FP16),
          (21, 28, 4, 128, E4M3), (21, 12, 2, 128, E5M2), (5, 6, 3, 96, FP16), (5, 4, 2, 256, FP16), (4, 3, 1, 2, FP16),
          (4, 2, 2, 66, FP16)]


@pytest.mark.parametrize("biased", [True, False])
@pytest.mark.parametrize("rows,nq,nkv,hd,fmt", APPEND)
def test_append_against_the_separate_calls(rows, nq, nkv, hd, fmt, biased):
    n_pages, seed = pages_of(rows) + 2, rows * nq
    rng = np.random.default_rng(seed)
    q, k, v = (to_dev(oracle.normal_f16((rows, n, hd), seed + i, std=2.0)) for i, n in enumerate((nq, nkv, nkv)))
    biases = [to_dev(oracle.normal_f16((n, hd), seed + 5 + i)) if biased and i != rows % 3 else None
              for i, n in enumerate((nq, nkv, nkv))]
    positions = rng.integers(0, 32768, rows)
    positions[0] = 0
    slots = rng.permutation(n_pages * PAGE)[:rows].astype(np.int64)
    if rows > 4:
        slots[[1, 3, 4]] = [-1, n_pages * PAGE, 2 ** 40]              # skipped whole
    want_q, want_k, want_v = separate_calls(q, k, v, biases, positions, slots, n_pages, fmt)
    d_pos, d_slots = ints(positions), ints(slots, torch.int64)
    ks, vs = new_store(n_pages, nkv, hd, fmt), new_store(n_pages, nkv, hd, fmt)
    before = [raw(x) for x in (q, k, v)]

    def call(out):
        ok(dev.vv_rope_kv_append_dev(q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                     *(b.data_ptr() if b is not None else None for b in biases), d_pos.data_ptr(),
                                     d_slots.data_ptr(), out.data_ptr(), ks.data_ptr(), vs.data_ptr(), rows, nq, nkv,
                                     hd, n_pages, fmt, 1e6, stream()))

    out = torch.full_like(q, float("nan"))
    call(out)
    assert np.array_equal(raw(vs), raw(want_v)), "values"
    live = (slots >= 0) & (slots < n_pages * PAGE)
    if not any(b is not None for b in biases[:2]):
        assert np.array_equal(raw(out), raw(want_q)) and np.array_equal(raw(ks), raw(want_k)), "q, keys"
    else:
        # the separate calls round x + bias to FP16 before they turn it, 2^-11 of each of a pair; then both sides round
        # (2^-11 each, of values that differ by that much), and an FP8 pool once more
        def pair(x, b):
            y = x.double().abs() + (b.double().abs() if b is not None else 0.0)
            y = y[..., :hd // 2] + y[..., hd // 2:]
            return torch.cat([y, y], -1)

        at = torch.from_numpy(slots[live]).cuda()
        on = torch.from_numpy(np.flatnonzero(live)).cuda()
        code = {FP16: (0.0, 0.0), E4M3: (2.0 ** -4, 2.0 ** -9), E5M2: (2.0 ** -3, 2.0 ** -16)}[fmt]
        for got, want, mag, low in ((out[on], want_q[on], pair(q, biases[0])[on], (0.0, 0.0)),
                                    (ks[at], want_k[at], pair(k, biases[1])[on], code)):
            if got.dtype == torch.uint8:
                got, want = (t.view(TORCH_FP8[fmt]).float() for t in (got, want))
            want = want.double()
            off = mag * 2.0 ** -11 + (want.abs() + mag * 2.0 ** -11) * 2.0 ** -10 + 2.0 ** -24
            off = off + 2.0 * low[0] * (want.abs() + off) + low[1]
            assert ((got.double() - want).abs() <= off).all()
        untouched = torch.ones(ks.shape[0], dtype=torch.bool, device="cuda")
        untouched[at] = False
        assert np.array_equal(raw(ks[untouched]), raw(want_k[untouched])), "rows that no slot names"
    assert all(np.array_equal(raw(x), b) for x, b in zip((q, k, v), before)), "an input was written"
    # in place: the rows of skipped slots keep q as it was
    call(q)
    at = torch.from_numpy(np.flatnonzero(live)).cuda()
    assert np.array_equal(raw(q[at]), raw(out[at]))
    rest = np.flatnonzero(~live)
    assert np.array_equal(raw(q)[rest], before[0][rest])


@pytest.mark.parametrize("fmt", [FP16, E4M3, E5M2])
def test_append_against_the_formula(fmt):
    """In 64 bits. The angle is FP32(position) * FP32(theta^(-2i/hd)): off by half a step of the product and by the
    frequency's own rounding (powf: 1 step), 2^-24 + 2^-23 of the angle, and sincosf and the FP32 products by some 2^-21
    of the pair; one rounding to FP16 (2^-11), then to the pool's type (E4M3 2^-4, E5M2 2^-3, or half a step of its
    subnormals, 2^-10 and 2^-17)."""
    rows, nq, nkv, hd, n_pages = 40, 4, 2, 128, 3
    q, k, v = (oracle.normal_f16((rows, n, hd), 50 + i) for i, n in enumerate((nq, nkv, nkv)))
    bias = [oracle.normal_f16((n, hd), 60 + i) for i, n in enumerate((nq, nkv, nkv))]
    rng = np.random.default_rng(3)
    positions, slots = rng.integers(0, 16384, rows), rng.permutation(n_pages * PAGE)[:rows]
    d = [to_dev(x) for x in (q, k, v, *bias)]
    d_pos, d_slots = ints(positions), ints(slots, torch.int64)
    out, ks, vs = torch.zeros_like(d[0]), new_store(n_pages, nkv, hd, fmt), new_store(n_pages, nkv, hd, fmt)
    ok(dev.vv_rope_kv_append_dev(*(x.data_ptr() for x in d), d_pos.data_ptr(), d_slots.data_ptr(), out.data_ptr(),
                                 ks.data_ptr(), vs.data_ptr(), rows, nq, nkv, hd, n_pages, fmt, 1e6, stream()))
    x = [oracle.widen(a).astype(np.float64) + oracle.widen(b) for a, b in zip((q, k, v), bias)]
    angle = positions[:, None] * 1e6 ** (-2.0 * np.arange(hd // 2) / hd)
    angle = np.concatenate([angle, angle], -1)[:, None, :]
    half = 2.0 ** -11

    def rope(a):
        lo, hi = a[..., :hd // 2], a[..., hd // 2:]
        c, s = np.cos(angle[..., :hd // 2]), np.sin(angle[..., :hd // 2])
        mag = np.abs(lo) + np.abs(hi)
        mag = np.concatenate([mag, mag], -1)
        return np.concatenate([lo * c - hi * s, lo * s + hi * c], -1), mag * (angle * (2.0 ** -24 + 2.0 ** -23) + 2.0 ** -21)

    def held(store):
        t = store if fmt == FP16 else store.view(TORCH_FP8[fmt])
        return t.float().cpu().numpy().astype(np.float64)[slots]

    store_half, store_low = {FP16: (0.0, 0.0), E4M3: (2.0 ** -4, 2.0 ** -10), E5M2: (2.0 ** -3, 2.0 ** -17)}[fmt]
    for name, got, (want, off), packed in (("q", out.float().cpu().numpy(), rope(x[0]), False),
                                           ("k", held(ks), rope(x[1]), True), ("v", held(vs), (x[2], 0.0), True)):
        off = off + half * np.abs(want) * 1.01 + 2.0 ** -25
        if packed:
            off = off + store_half * (np.abs(want) + off) + store_low
        assert (np.abs(got - want) <= off).all(), name


@pytest.mark.parametrize("fmt", [E4M3, E5M2])
def test_append_codes_of_every_half(fmt):
    """All 65536 FP16 patterns as values: the codes are those of vv_kv_store_dev."""
    rows, nkv, hd, n_pages = 128, 4, 128, 2
    v = torch.arange(65536, dtype=torch.int32, device="cuda").to(torch.int16).view(torch.float16).view(rows, nkv, hd)
    q, k, out = (torch.zeros(rows, n, hd, dtype=torch.float16, device="cuda") for n in (4, nkv, 4))
    want, got = new_store(n_pages, nkv, hd, fmt), new_store(n_pages, nkv, hd, fmt)
    wk, gk = new_store(n_pages, nkv, hd, fmt), new_store(n_pages, nkv, hd, fmt)
    ok(dev.vv_kv_store_dev(k.data_ptr(), v.data_ptr(), wk.data_ptr(), want.data_ptr(), None, None, None, False, nkv, hd, 0,
                           None, rows, fmt, None, stream()))
    pos, slots = ints(np.arange(rows)), ints(np.arange(rows), torch.int64)
    ok(dev.vv_rope_kv_append_dev(q.data_ptr(), k.data_ptr(), v.data_ptr(), None, None, None, pos.data_ptr(),
                                 slots.data_ptr(), out.data_ptr(), gk.data_ptr(), got.data_ptr(), rows, 4, nkv, hd, n_pages,
                                 fmt, 1e6, stream()))
    # (the keys, zeros, were stored there without a rotation, which may turn the sign of a zero)
    assert np.array_equal(raw(got), raw(want)) and np.array_equal(raw(gk) & 0x7F, raw(wk))


@pytest.mark.parametrize("which", range(7))
def test_append_unaligned(which):
    """Any one FP16 tensor off 16 bytes: the 2-byte kernel, the same bits."""
    rows, nq, nkv, hd, n_pages = 5, 4, 2, 128, 2
    rng = np.random.default_rng(which)
    sizes = [(rows, nq, hd), (rows, nkv, hd), (rows, nkv, hd), (nq, hd), (nkv, hd), (nkv, hd)]
    x = [to_dev(oracle.normal_f16(s, 30 + i)) for i, s in enumerate(sizes)]
    for bias in x[3:5]:
        bias.zero_()                                        # q and K are then the separate calls' bits
    positions, slots = rng.integers(0, 9000, rows), rng.permutation(n_pages * PAGE)[:rows]
    want = separate_calls(*x[:3], x[3:], positions, slots, n_pages, FP16)
    if which < 6:
        wide = torch.zeros(x[which].numel() + 1, dtype=torch.float16, device="cuda")
        wide[1:] = x[which].flatten()
        x[which] = wide[1:]
    row = nkv * hd
    ks, vs = (torch.full((n_pages * PAGE * row + 1,), float("nan"), dtype=torch.float16, device="cuda") for _ in "kv")
    shift = 1 if which == 6 else 0
    out, d_pos, d_slots = torch.full_like(want[0], float("nan")), ints(positions), ints(slots, torch.int64)
    ok(dev.vv_rope_kv_append_dev(*(t.data_ptr() for t in x), d_pos.data_ptr(), d_slots.data_ptr(), out.data_ptr(),
                                 ks.data_ptr() + 2 * shift, vs.data_ptr(), rows, nq, nkv, hd, n_pages, FP16, 1e6,
                                 stream()))
    assert np.array_equal(raw(out), raw(want[0]))
    assert np.array_equal(raw(ks[shift:shift + n_pages * PAGE * row]), raw(want[1]).reshape(-1))
    assert np.array_equal(raw(vs[:n_pages * PAGE * row]), raw(want[2]).reshape(-1))


# ── attention ────────────────────────────────────────────────────────────────

class Pool:
    """Sequences of the given lengths in a shuffled pool; NaN (0x7F codes) where no position lies."""

    def __init__(self, lens, nq, nkv, hd, fmt=FP16, seed=0, max_pages=None, first_page=0, sharp=2.0, spare=3):
        rng = np.random.default_rng(seed)
        self.lens, self.nq, self.nkv, self.hd, self.fmt = list(lens), nq, nkv, hd, fmt
        self.max_pages = max_pages or max(1, max(pages_of(n) for n in lens))
        total = sum(pages_of(n) for n in lens)
        self.n_pages = first_page + total + spare
        perm = rng.permutation(total + spare)[:total].astype(np.int32) + first_page
        self.tables = np.full((len(lens), self.max_pages), -1, np.int32)
        at = 0
        for i, n in enumerate(lens):
            self.tables[i, :pages_of(n)] = perm[at:at + pages_of(n)]
            at += pages_of(n)
        g = torch.Generator(device="cuda").manual_seed(seed + 1)
        normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.q = (normal(len(lens), nq, hd) * sharp * hd ** -0.25 * 2).half()
        held = [normal(sum(lens), nkv, hd) * (hd ** -0.25 * 2 if i == 0 else 1) for i in range(2)]
        slots = np.concatenate([slots_of(self.tables[i], n) for i, n in enumerate(lens)] + [np.zeros(0, np.int64)])
        self.store = []
        for x in held:
            s = new_store(self.n_pages, nkv, hd, fmt)
            x = x.half() if fmt == FP16 else x.to(TORCH_FP8[fmt])
            s[torch.from_numpy(slots).cuda()] = x if fmt == FP16 else x.view(torch.uint8)
            self.store.append(s)
        self.scratch = None

    def values(self, i, n=None):
        """Sequence i's keys and values in 64 bits."""
        at = torch.from_numpy(slots_of(self.tables[i], self.lens[i] if n is None else n)).cuda()
        x = [s[at] if self.fmt == FP16 else s[at].view(TORCH_FP8[self.fmt]) for s in self.store]
        return [t.float().cpu().numpy().astype(np.float64) for t in x]

    def call(self, lens=None, tables=None, stream_=None, q=None, n=None, scratch_fill=0xFF, in_place=False):
        n = len(self.lens) if n is None else n
        q = self.q if q is None else q
        d_lens, d_tables = ints(self.lens if lens is None else lens), ints(self.tables if tables is None else tables)
        out = torch.full((n + 1, self.nq, self.hd), float("nan"), dtype=torch.float16, device="cuda")
        if in_place:
            out[:n] = q
            q = out
        size = dev.vv_attn_decode_batch_scratch_bytes(n, self.nq, self.nkv, self.hd)
        scratch = torch.full((size + 64,), scratch_fill, dtype=torch.uint8, device="cuda")      # NaN unless written
        view = dev.KvView(k=self.store[0].data_ptr(), v=self.store[1].data_ptr(), k_meta=None, v_meta=None,
                          page_table=d_tables.data_ptr(), format=self.fmt, n_kv_heads=self.nkv, head_dim=self.hd)
        torch.cuda.synchronize()
        ok(dev.vv_attn_decode_batch(2, q.data_ptr(), C.addressof(view), out.data_ptr(), self.nq, n, d_lens.data_ptr(),
                                    self.max_pages, self.n_pages, scratch.data_ptr(), size, stream_ or stream()))
        torch.cuda.synchronize()
        assert torch.isnan(out[n]).all(), "the row behind the last sequence was written"
        assert (scratch[size:] == scratch_fill).all(), "written past the scratch"
        return out[:n]

    def check(self, out, rows=None, values=None):
        got, q = out.float().cpu().numpy().astype(np.float64), self.q.float().cpu().numpy().astype(np.float64)
        for i in rows if rows is not None else range(len(self.lens)):
            k, v = values(i) if values else self.values(i)
            want, mag = attend(q[i], k, v)
            off = attend_bound(want, mag, k.shape[0], np.abs(v).max(initial=0.0))
            worst = np.abs(got[i] - want) / off
            assert (worst <= 1.0).all(), f"sequence {i} of {k.shape[0]} positions: {worst.max():.2f}x the bound"


EDGES = [1, 0, 15, 16, 17, 63, 64, 65, 127, 128, 129, 191, 192, 193, 0, 300, 1000, 2]
HEADS = [(28, 4, 128), (12, 2, 128), (1, 1, 128), (5, 5, 128), (16, 1, 128), (17, 1, 128), (40, 1, 128), (66, 2, 128),
         (14, 2, 64), (8, 8, 64), (3, 1, 64), (34, 2, 64)]


@pytest.mark.parametrize("nq,nkv,hd", HEADS)
def test_attend_edges(nq, nkv, hd):
    p = Pool(EDGES, nq, nkv, hd, seed=nq)
    out = p.call()
    p.check(out)
    assert (out[1] == 0).all() and (out[14] == 0).all()
    assert np.array_equal(raw(p.call(scratch_fill=0)), raw(out)), "another answer the second time"
    assert np.array_equal(raw(p.call(in_place=True)), raw(out)), "another answer over the query"


@pytest.mark.parametrize("fmt", [E4M3, E5M2])
@pytest.mark.parametrize("nq,nkv", [(28, 4), (4, 4), (20, 1)])
def test_attend_packed(fmt, nq, nkv):
    p = Pool(EDGES, nq, nkv, 128, fmt=fmt, seed=nq + fmt)
    p.check(p.call())
    # a bad page in either place of a pair, and both
    tables = p.tables.copy()
    tables[15, 1] = -1
    tables[16, [2, 3, 6]] = p.n_pages
    drop = {15: [*range(64, 128)], 16: [*range(128, 256), *range(384, 448)]}

    def values(i):
        return [np.delete(x, drop[i], 0) for x in p.values(i)]
    p.check(p.call(tables=tables), rows=[15, 16], values=values)


@pytest.mark.parametrize("fmt", [E4M3, E5M2])
def test_attend_every_code(fmt):
    """One position a sequence: the result is its value, for every finite code, exactly; and its key counts as that
    value too: two positions whose keys differ in one channel's code alone share the weight as the codes say."""
    codes = torch.arange(256, dtype=torch.uint8, device="cuda")
    value = codes.view(TORCH_FP8[fmt]).float()
    finite = codes[torch.isfinite(value)]
    n = finite.numel()
    p = Pool([2] * n, 2, 1, 128, fmt=fmt, seed=21)
    at = torch.from_numpy(np.stack([slots_of(t, 2) for t in p.tables])).cuda()
    p.store[0][:] = 0
    p.store[1][:] = 0
    p.store[1][at[:, 0]] = finite[:, None, None]
    out = p.call(lens=[1] * n)
    want = finite.view(TORCH_FP8[fmt]).half()
    assert torch.equal(out, want[:, None, None].expand(n, 2, 128))       # as numbers: +0 + -0 is +0
    p.store[0][at[:, 0], 0, 37] = finite
    p.q[:] = 0
    p.q[:, :, 37] = 2.0 ** -6 if fmt == E4M3 else 2.0 ** -13          # scores of either sign, up to 1
    p.check(p.call())


@pytest.mark.parametrize("nq,nkv,hd", [(6, 3, 96), (4, 2, 256), (2, 1, 80), (4, 4, 1), (3, 1, 65)])
def test_attend_other_head_dims(nq, nkv, hd):
    p = Pool(EDGES[:12], nq, nkv, hd, seed=hd)
    p.check(p.call())


def test_attend_unaligned_query():
    p = Pool([70, 0, 3], 4, 2, 128, seed=8)
    wide = torch.zeros(p.q.numel() + 1, dtype=torch.float16, device="cuda")
    wide[1:] = p.q.flatten()
    p.check(p.call(q=wide[1:]))


@pytest.mark.parametrize("lens", [[14449], [5000, 1, 9000, 64], [64] * 300, [1] * 1500, list(range(700)),
                                  [0] * 1100 + [77], [9000] + [60] * 39,
                                  [60] * 150 + [20000] + [60] * 149,
                                  [3] * 300 + [6000] + [0] * 300])
def test_attend_many_and_long(lens):
    """One long sequence over all workgroups, more sequences than threads, than workgroups, mostly empty ones."""
    p = Pool(lens, 4, 2, 128, seed=len(lens))
    out = p.call()
    p.check(out, rows=sorted(set(range(0, len(lens), max(1, len(lens) // 12))) | {len(lens) - 1}))
    assert np.array_equal(raw(p.call(in_place=True)), raw(out)), "another answer over the query"
    empty = [i for i, n in enumerate(lens) if n == 0]
    assert (out[empty] == 0).all()


def test_attend_is_vv_attn_decode_for_one_sequence():
    p = Pool([3000], 28, 4, 128, seed=5)
    view = dev.KvView(k=p.store[0].data_ptr(), v=p.store[1].data_ptr(), k_meta=None, v_meta=None,
                      page_table=None, format=FP16, n_kv_heads=4, head_dim=128)
    d_table = ints(p.tables)
    view.page_table = d_table.data_ptr()
    one = torch.empty_like(p.q)
    scratch = torch.empty(dev.vv_attn_scratch_bytes(28, 4, 128), dtype=torch.uint8, device="cuda")
    ok(dev.vv_attn_decode(2, p.q.data_ptr(), C.addressof(view), one.data_ptr(), 28, 3000, None, scratch.data_ptr(),
                          stream()))
    p.check(p.call())
    p.check(one)


def test_attend_odd_lengths_and_pages():
    p = Pool([200, 130, 64, 500, 10], 8, 2, 128, seed=9, max_pages=8)
    base = p.call()
    # negative: nothing; past the table: the table's positions (the last page's are all in use there)
    lens = [200, -3, 64, 500, 10]
    out = p.call(lens=lens)
    assert (out[1] == 0).all()
    p.check(out, rows=[0, 2, 3, 4])
    full = Pool([128, 512, 3], 8, 2, 128, seed=10, max_pages=8)
    out = full.call(lens=[128, 2 ** 31 - 1, 3])
    full.check(out)
    # a page id outside the pool: its positions are masked; all of them: zeros
    for bad in (-1, p.n_pages, 2 ** 31 - 1, -2 ** 31):
        tables = p.tables.copy()
        tables[0, 1] = bad
        tables[2, 0] = bad
        tables[3, 7] = bad
        out = p.call(tables=tables)
        assert (out[2] == 0).all()

        def values(i):
            k, v = p.values(i)
            drop = {0: range(64, 128), 3: range(448, 500)}.get(i, [])
            return np.delete(k, list(drop), 0), np.delete(v, list(drop), 0)
        p.check(out, rows=[0, 1, 3, 4], values=values)
        assert np.array_equal(raw(out[4]), raw(base[4]))


@pytest.mark.parametrize("hd", [64, 128, 96])
def test_attend_infinities_and_nan(hd):
    p = Pool([70, 65, 64, 90], 4, 2, hd, seed=11)
    last = int(slots_of(p.tables[0], 70)[-1])
    p.store[1][last, 0, 3] = float("inf")                      # the last value: its masked neighbours must not meet it
    at = int(slots_of(p.tables[1], 65)[10])
    p.store[0][at, 1] = float("-inf")
    p.q[1].abs_()                                              # every score of that key is -inf: it takes no part
    at3 = int(slots_of(p.tables[3], 90)[20])
    p.store[0][at3, 0, 0] = float("nan")                       # a key in use: NaN, for the heads that read it
    out = p.call().float().cpu().numpy()
    assert (out[0, :2, 3] == np.inf).all()
    assert np.isfinite(np.delete(out[0, :2], 3, axis=1)).all() and np.isfinite(out[0, 2:]).all()
    assert np.isnan(out[3, :2]).all() and np.isfinite(out[3, 2:]).all()
    p.check(torch.from_numpy(out), rows=[2])
    k, v = p.values(1)
    keep = np.delete(np.arange(65), 10)
    want, mag = attend(p.q[1, 2:].float().cpu().numpy().astype(np.float64), k[keep, 1:], v[keep, 1:])
    assert (np.abs(out[1, 2:] - want) <= attend_bound(want, mag, 65, np.abs(v).max())).all()


def test_attend_nan_query():
    """A query that is NaN gives NaN for its head, short rows and rows that many workgroups share, and for no other."""
    p = Pool([5000, 70, 0, 3000], 4, 2, 128, seed=22)
    p.q[0, 1, 5] = float("nan")
    p.q[1, 2, 0] = float("nan")
    out = p.call()
    bad = torch.isnan(out).all(-1).cpu().numpy()
    assert bad.tolist() == [[False, True, False, False], [False, False, True, False], [False] * 4, [False] * 4]
    assert torch.isfinite(out[torch.from_numpy(~bad).cuda()]).all()
    p.check(out, rows=[3])


@pytest.mark.parametrize("scale", [1e-3, 30.0])
def test_attend_flat_and_sharp(scale):
    """All scores alike (a mean of the values), and one key far above the rest."""
    p = Pool([4000, 4000, 130], 7, 1, 128, seed=12, sharp=scale)
    p.check(p.call())


def test_attend_rising_scores():
    """Each key above the one before it: the softmax's reference moves all the way."""
    p = Pool([1000, 37], 4, 1, 128, seed=13)
    at = torch.from_numpy(slots_of(p.tables[0], 1000)).cuda()
    p.q[0] = 1.0
    p.store[0][at] = (torch.arange(1000, device="cuda").float() / 100).half()[:, None, None]
    p.check(p.call())
    p.store[0][at] = (torch.arange(1000, 0, -1, device="cuda").float() / 100).half()[:, None, None]
    p.check(p.call())


def test_attend_far_pages():
    """A pool whose rows lie past 2^31 elements (and 2^32 bytes) from its start."""
    far = 2 ** 31 // (PAGE * 4 * 128) + 5
    n_pages = far + 12
    rows = [torch.empty(n_pages * PAGE, 4, 128, dtype=torch.float16, device="cuda") for _ in "kv"]
    p = Pool([300, 70], 8, 4, 128, seed=14)
    tables = np.where(p.tables >= 0, p.tables + far, -1).astype(np.int32)
    for wide, s in zip(rows, p.store):
        wide[far * PAGE:(far + p.n_pages) * PAGE] = s
    small = p.call()
    p.check(small)
    p.store, p.n_pages = rows, n_pages
    assert np.array_equal(raw(p.call(tables=tables)), raw(small))
    # and the append to those rows
    q, k, v = (to_dev(oracle.normal_f16((3, n, 128), n)) for n in (8, 4, 4))
    slots = np.array([far * PAGE + 700, 5, n_pages * PAGE - 1])
    pos, out = ints([0, 0, 0]), torch.empty_like(q)
    d_slots = ints(slots, torch.int64)
    ok(dev.vv_rope_kv_append_dev(q.data_ptr(), k.data_ptr(), v.data_ptr(), None, None, None, pos.data_ptr(),
                                 d_slots.data_ptr(), out.data_ptr(), rows[0].data_ptr(), rows[1].data_ptr(), 3, 8, 4, 128,
                                 n_pages, FP16, 1e6, stream()))
    assert np.array_equal(raw(rows[0][torch.from_numpy(slots).cuda()]), raw(k))       # position 0 turns nothing
    assert np.array_equal(raw(rows[1][torch.from_numpy(slots).cuda()]), raw(v))


def test_attend_on_two_streams_at_once():
    a, b = Pool([3000, 5, 700], 28, 4, 128, seed=15), Pool([64] * 40 + [2000], 12, 2, 128, seed=16)
    want = [raw(a.call()), raw(b.call())]
    outs = []
    for x in (a, b):
        st = torch.cuda.Stream()
        n = len(x.lens)
        size = dev.vv_attn_decode_batch_scratch_bytes(n, x.nq, x.nkv, x.hd)
        keep = [ints(x.lens), ints(x.tables), torch.empty(size, dtype=torch.uint8, device="cuda"), torch.empty_like(x.q)]
        view = dev.KvView(k=x.store[0].data_ptr(), v=x.store[1].data_ptr(), k_meta=None, v_meta=None,
                          page_table=keep[1].data_ptr(), format=FP16, n_kv_heads=x.nkv, head_dim=x.hd)
        outs.append((x, st, keep, view, n, size))
    torch.cuda.synchronize()
    for _ in range(20):
        for x, st, (lens, _, scratch, out), view, n, size in outs:
            ok(dev.vv_attn_decode_batch(2, x.q.data_ptr(), C.addressof(view), out.data_ptr(), x.nq, n, lens.data_ptr(),
                                        x.max_pages, x.n_pages, scratch.data_ptr(), size, st.cuda_stream))
    torch.cuda.synchronize()
    for w, (_, _, keep, _, _, _) in zip(want, outs):
        assert np.array_equal(raw(keep[3]), w)


# ── the three together ───────────────────────────────────────────────────────

@pytest.mark.parametrize("fmt", [FP16, E4M3])
@pytest.mark.parametrize("captured", [False, True])
def test_serving_loop(fmt, captured):
    """Requests at every stage, padded to a fixed number of rows: plan, append, attend, step after step, against dense
    attention over everything appended so far. One request outgrows its table, one finds the pool empty; both keep
    what they had. Captured, the same launches are replayed with new inputs and lengths in place."""
    nq, nkv, hd, n, max_pages, steps, theta = 8, 2, 128, 6, 3, 12, 1e4
    pool_pages, max_rows = 9, 8
    k_store, v_store = new_store(pool_pages, nkv, hd, fmt), new_store(pool_pages, nkv, hd, fmt)
    lens, n_free, counts = torch.zeros(n, dtype=torch.int32, device="cuda"), ints([pool_pages]), ints([0, 0, 0])
    tables = torch.full((n, max_pages), -1, dtype=torch.int32, device="cuda")
    free = ints(np.random.default_rng(0).permutation(pool_pages))
    new = torch.ones(n, dtype=torch.int32, device="cuda")
    view = dev.KvView(k=k_store.data_ptr(), v=v_store.data_ptr(), k_meta=None, v_meta=None,
                      page_table=tables.data_ptr(), format=fmt, n_kv_heads=nkv, head_dim=hd)
    size = dev.vv_attn_decode_batch_scratch_bytes(n, nq, nkv, hd)
    scratch = torch.empty(size, dtype=torch.uint8, device="cuda")

    def buffers(rows):
        return dict(q=torch.zeros(rows, nq, hd, dtype=torch.float16, device="cuda"),
                    k=torch.zeros(rows, nkv, hd, dtype=torch.float16, device="cuda"),
                    v=torch.zeros(rows, nkv, hd, dtype=torch.float16, device="cuda"),
                    qr=torch.zeros(rows, nq, hd, dtype=torch.float16, device="cuda"),
                    positions=torch.zeros(rows, dtype=torch.int32, device="cuda"),
                    slots=torch.zeros(rows, dtype=torch.int64, device="cuda"),
                    starts=torch.zeros(n + 1, dtype=torch.int32, device="cuda"),
                    out=torch.zeros(n, nq, hd, dtype=torch.float16, device="cuda"))

    def launch(b, rows, st):
        ok(dev.vv_kv_page_plan_dev(new.data_ptr(), lens.data_ptr(), n, tables.data_ptr(), max_pages, free.data_ptr(),
                                   n_free.data_ptr(), lens.data_ptr(), b["starts"].data_ptr(),
                                   b["positions"].data_ptr(), b["slots"].data_ptr(), rows, n_free.data_ptr(),
                                   counts.data_ptr(), st))
        ok(dev.vv_rope_kv_append_dev(b["q"].data_ptr(), b["k"].data_ptr(), b["v"].data_ptr(), None, None, None,
                                     b["positions"].data_ptr(), b["slots"].data_ptr(), b["qr"].data_ptr(),
                                     k_store.data_ptr(), v_store.data_ptr(), rows, nq, nkv, hd, pool_pages, fmt, theta, st))
        ok(dev.vv_attn_decode_batch(2, b["qr"].data_ptr(), C.addressof(view), b["out"].data_ptr(), nq, n,
                                    lens.data_ptr(), max_pages, pool_pages, scratch.data_ptr(), size, st))

    st = torch.cuda.Stream()
    # the prompts: rows per request, run eagerly through plan and append (their attention is prefill's business)
    prompts = [3, 63, 64, 130, 0, 191]
    big = buffers(sum(prompts))
    rng = np.random.default_rng(1)
    state = dict(history=[[] for _ in range(n)], lens=np.zeros(n, np.int32), tables=tables.cpu().numpy(),
                 n_free=pool_pages)

    def fill(b, rows):
        x = {}
        for name, h in (("q", nq), ("k", nkv), ("v", nkv)):
            x[name] = rng.normal(size=(rows, h, hd)).astype(np.float16)
            b[name].copy_(torch.from_numpy(x[name]))
        return x

    def expect(ask, x, rows):
        want = plan(ask, state["lens"], state["tables"], free.cpu().numpy(), state["n_free"], rows)
        state.update(lens=want["lens"], tables=want["tables"], n_free=want["n_free"])
        turn = theta ** (-2.0 * np.arange(hd // 2) / hd)
        for i in range(n):
            for r in range(want["row_starts"][i], want["row_starts"][i + 1]):
                if want["slots"][r] < 0:
                    continue
                z = np.exp(1j * want["positions"][r] * turn)
                kz = (x["k"][r, :, :hd // 2] + 1j * x["k"][r, :, hd // 2:].astype(np.float64)) * z
                state["history"][i].append((np.concatenate([kz.real, kz.imag], -1), x["v"][r].astype(np.float64)))
        return want

    new.copy_(ints(prompts))
    x = fill(big, sum(prompts))
    torch.cuda.synchronize()
    launch(big, sum(prompts), st.cuda_stream)
    torch.cuda.synchronize()
    want = expect(prompts, x, sum(prompts))
    assert np.array_equal(tables.cpu().numpy(), want["tables"]) and np.array_equal(lens.cpu().numpy(), want["lens"])

    small, graph = buffers(max_rows), C.c_void_p()
    if captured:
        torch.cuda.synchronize()
        ok(dev.vv_dev_graph_begin(st.cuda_stream))
        launch(small, max_rows, st.cuda_stream)
        ok(dev.vv_dev_graph_end(st.cuda_stream, C.byref(graph)))
    refused = 0
    for step in range(steps):
        ask = np.ones(n, int) if step % 4 else np.array([1, 1, 0, 1, 1, 1])
        new.copy_(ints(ask))
        x = fill(small, max_rows)
        small["qr"].fill_(float("nan"))
        torch.cuda.synchronize()
        if captured:
            ok(dev.vv_dev_graph_launch(graph, st.cuda_stream))
        else:
            launch(small, max_rows, st.cuda_stream)
        torch.cuda.synchronize()
        want = expect(ask, x, max_rows)
        refused += int(want["counts"][2])
        assert np.array_equal(counts.cpu().numpy(), want["counts"]) and int(n_free) == want["n_free"]
        assert np.array_equal(small["slots"].cpu().numpy(), want["slots"])
        assert np.array_equal(tables.cpu().numpy(), want["tables"]) and np.array_equal(lens.cpu().numpy(), want["lens"])
        # attention reads row i of qr for sequence i; the requests that asked nothing shift the rows, so hold the
        # operator to the rows as they lie
        qr = small["qr"].float().cpu().numpy().astype(np.float64)
        out = small["out"].float().cpu().numpy().astype(np.float64)
        for i in range(n):
            if not np.isfinite(qr[i]).all() or not state["history"][i]:
                continue
            k, v = (np.stack(t) for t in zip(*state["history"][i]))
            ref, mag = attend(qr[i], k, v)
            if fmt == FP16:        # K and V went through one rounding to FP16, as did q: 2^-11 of |q||k| in a score
                spread = 2.0 ** -10 * np.abs(qr[i]).sum(-1).max() * np.abs(k).max() / np.sqrt(hd)
                off = attend_bound(ref, mag, len(k), np.abs(v).max()) + mag * (np.expm1(2 * spread) + 2.0 ** -11)
            else:                  # E4M3: half a step is 2^-4 of each key and value
                spread = 2.0 ** -4 * np.abs(qr[i]).sum(-1).max() * np.abs(k).max() / np.sqrt(hd)
                off = mag * (np.expm1(2 * min(spread, 1.0)) + 2.0 ** -4) + 2.0 ** -9
            assert (np.abs(out[i] - ref) <= off).all(), f"step {step} sequence {i}"
    assert refused > 0
    if captured:
        dev.vv_dev_graph_destroy(graph)


@pytest.mark.parametrize("fmt", [FP16, E5M2])
def test_step_with_a_prompt(fmt):
    """Decoding requests first, a prompt's chunk behind them: one plan, one append, batched attention for the former and
    the paged prefill for the latter, all on one pool."""
    nq, nkv, hd, max_pages, theta = 8, 2, 128, 4, 1e6
    p = Pool([100, 63, 1, 200, 90], nq, nkv, hd, fmt=fmt, seed=31, max_pages=max_pages, spare=8)
    n_dec, chunk = 4, 70
    held = [p.values(i) for i in range(5)]
    free = np.setdiff1d(np.arange(p.n_pages), p.tables)
    new, n_free = [1] * n_dec + [chunk], len(free)
    rows = sum(new)
    x = [to_dev(oracle.normal_f16((rows, n, hd), 70 + i)) for i, n in enumerate((nq, nkv, nkv))]
    d = dict(new=ints(new), lens=ints(p.lens), tables=ints(p.tables), free=ints(free), n_free=ints([n_free]),
             starts=ints([0] * 6), pos=ints([0] * rows), slots=ints([0] * rows, torch.int64), counts=ints([0] * 3))
    at = {k: t.data_ptr() for k, t in d.items()}
    ok(dev.vv_kv_page_plan_dev(at["new"], at["lens"], 5, at["tables"], max_pages, at["free"], at["n_free"], at["lens"],
                               at["starts"], at["pos"], at["slots"], rows, at["n_free"], at["counts"], stream()))
    ok(dev.vv_rope_kv_append_dev(*(t.data_ptr() for t in x), None, None, None, at["pos"], at["slots"], x[0].data_ptr(),
                                 p.store[0].data_ptr(), p.store[1].data_ptr(), rows, nq, nkv, hd, p.n_pages, fmt, theta,
                                 stream()))
    view = dev.KvView(k=p.store[0].data_ptr(), v=p.store[1].data_ptr(), k_meta=None, v_meta=None,
                      page_table=at["tables"], format=fmt, n_kv_heads=nkv, head_dim=hd)
    size = dev.vv_attn_decode_batch_scratch_bytes(n_dec, nq, nkv, hd)
    scratch, out = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.full_like(x[0], float("nan"))
    ok(dev.vv_attn_decode_batch(2, x[0].data_ptr(), C.addressof(view), out.data_ptr(), nq, n_dec, at["lens"], max_pages,
                                p.n_pages, scratch.data_ptr(), size, stream()))
    one = dev.KvView(k=p.store[0].data_ptr(), v=p.store[1].data_ptr(), k_meta=None, v_meta=None,
                     page_table=at["tables"] + 4 * 4 * max_pages, format=fmt, n_kv_heads=nkv, head_dim=hd)
    step = n_dec * nq * hd * 2
    ok(dev.vv_attn_prefill(2, x[0].data_ptr() + step, C.addressof(one), out.data_ptr() + step, nq, chunk, 90, 90 + chunk,
                           True, None, stream()))
    torch.cuda.synchronize()
    # 101, 64, 2 and 201 positions fit the pages that 100, 63, 1 and 200 have; 160 need one more than 90
    assert d["counts"].tolist() == [n_free - 1, rows, 0] and d["lens"].tolist() == [101, 64, 2, 201, 160]
    p.tables, p.lens = d["tables"].cpu().numpy(), d["lens"].tolist()
    now = [p.values(i) for i in range(5)]
    for i in range(5):                                                   # what was cached is untouched
        assert all(np.array_equal(a, b[:len(a)]) for a, b in zip(held[i], now[i]))
    q, got = (t.float().cpu().numpy().astype(np.float64) for t in (x[0], out))
    for r in range(rows):
        i = min(r, 4)
        n = p.lens[i] if i < 4 else 90 + r - 4 + 1
        k, v = (t[:n] for t in now[i])
        want, mag = attend(q[r], k, v)
        assert (np.abs(got[r] - want) <= attend_bound(want, mag, n, np.abs(v).max())).all(), f"row {r}"
