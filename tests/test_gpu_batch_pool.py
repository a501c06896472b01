"""A fixed pool of slots served step after step as one captured (or eager) plan, append and attention: some slots decode,
some stand by, some are refused, requests come and go between steps. Each request is held to its own query and to what
the pool stores for it, at the pool's own precision."""
import ctypes as C

import numpy as np
import pytest
import torch

from batch_util import PAGE, attend, attend_bound_lifted, pages_of, plan, slots_of
from gpu_util import dev, ok
from test_gpu_batch_serving import E4M3, E5M2, FP16, TORCH_FP8, ints, new_store, raw

pytestmark = pytest.mark.gpu

NQ, NKV, HD, MAX_PAGES, THETA = 8, 2, 128, 3, 1e4
HALF = {FP16: (0.0, 0.0), E4M3: (2.0 ** -4, 2.0 ** -10), E5M2: (2.0 ** -3, 2.0 ** -17)}   # half a step; of the subnormals


def turned(x, position):
    """x [heads][hd] (FP16 values) rotated in 64 bits, and what the kernel's FP16 result may be off: the angle is an FP32
    product (2^-24) with a frequency off by a step (2^-23), sincosf and the FP32 products by some 2^-21 of the pair, one
    rounding to FP16."""
    x = x.astype(np.float64)
    lo, hi = x[:, :HD // 2], x[:, HD // 2:]
    angle = position * THETA ** (-2.0 * np.arange(HD // 2) / HD)
    c, s = np.cos(angle), np.sin(angle)
    want = np.concatenate([lo * c - hi * s, lo * s + hi * c], -1)
    mag = np.tile(np.abs(lo) + np.abs(hi), 2) * (np.tile(angle, 2) * (2.0 ** -24 + 2.0 ** -23) + 2.0 ** -21)
    return want, mag + 2.0 ** -11 * np.abs(want) * 1.01 + 2.0 ** -25


def stored(want, off, fmt):
    """The same once it lies in the pool."""
    half, low = HALF[fmt]
    return off + half * (np.abs(want) + off) + low


def values(store, fmt):
    t = store if fmt == FP16 else store.view(TORCH_FP8[fmt])
    return t.float().cpu().numpy().astype(np.float64)


class Slots:
    """The pool, its slots, and the plain restatement that follows them on the host."""

    def __init__(self, n, pool_pages, fmt, seed):
        self.n, self.fmt, self.pages, self.rng = n, fmt, pool_pages, np.random.default_rng(seed)
        self.k, self.v = new_store(pool_pages, NKV, HD, fmt), new_store(pool_pages, NKV, HD, fmt)
        self.lens, self.tables = np.full(n, -1, np.int32), np.full((n, MAX_PAGES), -1, np.int32)
        self.free, self.n_free = self.rng.permutation(pool_pages).astype(np.int32), pool_pages
        self.d = dict(new=ints(np.ones(n)), lens=ints(self.lens), tables=ints(self.tables), free=ints(self.free),
                      n_free=ints([pool_pages]), counts=ints([0] * 3), starts=ints([0] * (n + 1)))
        size = dev.vv_attn_decode_batch_scratch_bytes(n, NQ, NKV, HD)
        self.scratch = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")
        self.view = dev.KvView(k=self.k.data_ptr(), v=self.v.data_ptr(), k_meta=None, v_meta=None,
                               page_table=self.d["tables"].data_ptr(), format=fmt, n_kv_heads=NKV, head_dim=HD)

    def rows(self, rows):
        new = lambda *s, t=torch.float16: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
        return dict(q=new(rows, NQ, HD), k=new(rows, NKV, HD), v=new(rows, NKV, HD), qr=new(rows, NQ, HD),
                    positions=new(rows, t=torch.int32), slots=new(rows, t=torch.int64), out=new(self.n + 1, NQ, HD))

    def push(self):
        """What a host changes between steps: lengths, tables, the stack of free pages."""
        for name in ("lens", "tables", "free"):
            self.d[name].copy_(torch.from_numpy(getattr(self, name)))
        self.d["n_free"].fill_(self.n_free)

    def launch(self, b, rows, st, attention=True):
        at = {k: t.data_ptr() for k, t in {**self.d, **b}.items()}
        ok(dev.vv_kv_page_plan_dev(at["new"], at["lens"], self.n, at["tables"], MAX_PAGES, at["free"], at["n_free"],
                                   at["lens"], at["starts"], at["positions"], at["slots"], rows, at["n_free"],
                                   at["counts"], st))
        ok(dev.vv_rope_kv_append_dev(at["q"], at["k"], at["v"], None, None, None, at["positions"], at["slots"], at["qr"],
                                     self.k.data_ptr(), self.v.data_ptr(), rows, NQ, NKV, HD, self.pages, self.fmt,
                                     THETA, st))
        if attention:
            ok(dev.vv_attn_decode_batch(2, at["qr"], C.addressof(self.view), at["out"], NQ, self.n, at["lens"], MAX_PAGES,
                                        self.pages, self.scratch.data_ptr(), self.scratch.numel(), st))

    def fill(self, b):
        x = {}
        for name in "qkv":
            x[name] = self.rng.normal(size=tuple(b[name].shape)).astype(np.float16)
            b[name].copy_(torch.from_numpy(x[name]))
        b["qr"].fill_(float("nan"))
        b["out"].fill_(float("nan"))
        return x

    def check_append(self, b, x, want, before):
        """The pool after the append: the rows of the step hold this step's keys and values, all others what they held."""
        live = np.flatnonzero(want["slots"] >= 0)
        at = want["slots"][live]
        k, v, qr = values(self.k, self.fmt), values(self.v, self.fmt), values(b["qr"], FP16)
        for r, slot in zip(live, at):
            position = int(want["positions"][r])
            ref, off = turned(x["q"][r], position)
            assert (np.abs(qr[r] - ref) <= off).all(), f"query of row {r}"
            ref, off = turned(x["k"][r], position)
            assert (np.abs(k[slot] - ref) <= stored(ref, off, self.fmt)).all(), f"key of row {r}"
            ref = x["v"][r].astype(np.float64)
            assert (np.abs(v[slot] - ref) <= stored(ref, 0.0, self.fmt)).all(), f"values of row {r}"
        rest = np.setdiff1d(np.arange(self.pages * PAGE), at)
        assert all(np.array_equal(raw(s)[rest], old[rest]) for s, old in zip((self.k, self.v), before))
        skipped = np.setdiff1d(np.arange(len(want["slots"])), live)
        assert np.isnan(qr[skipped]).all(), "a row without a slot was written"

    def check_attention(self, b, want, live):
        """Every slot that was served against its own query over what the pool stores for it; zeros where none is held."""
        out, q = values(b["out"], FP16), values(b["qr"], FP16)
        assert np.isnan(out[self.n]).all(), "the row behind the last slot was written"
        k, v = values(self.k, self.fmt), values(self.v, self.fmt)
        for i in range(self.n):
            if self.lens[i] <= 0:
                assert (out[i] == 0).all(), f"slot {i} holds nothing"
            elif i in live:
                at = slots_of(self.tables[i], self.lens[i])
                ref, mag = attend(q[i], k[at], v[at])
                worst = np.abs(out[i] - ref) / attend_bound_lifted(ref, mag, len(at), np.abs(v[at]).max())
                assert (worst <= 1.0).all(), f"slot {i} of {len(at)} positions: {worst.max():.2f}x the bound"

    def step(self, b, rows, ask, x, run, attention=True):
        """One step on the device and on the host, compared."""
        self.d["new"].copy_(ints(ask))
        before = [raw(self.k), raw(self.v)]
        torch.cuda.synchronize()
        run()
        torch.cuda.synchronize()
        want = plan(ask, self.lens, self.tables, self.free, self.n_free, rows)
        self.lens, self.tables, self.n_free = want["lens"], want["tables"], want["n_free"]
        for name, t in (("lens", self.d["lens"]), ("tables", self.d["tables"]), ("row_starts", self.d["starts"]),
                        ("counts", self.d["counts"]), ("positions", b["positions"]), ("slots", b["slots"])):
            assert np.array_equal(t.cpu().numpy(), want[name]), name
        assert int(self.d["n_free"]) == self.n_free
        self.check_append(b, x, want, before)
        if attention:
            self.check_attention(b, want, set(np.flatnonzero(want["slots"][:self.n] >= 0)))
        return want


@pytest.mark.parametrize("fmt", [FP16, E4M3, E5M2])
@pytest.mark.parametrize("captured", [False, True])
def test_slots_decode_stand_by_and_are_refused(fmt, captured):
    """Slots 0 .. 6: a row each, whatever they do. A slot without a request has length -1; one that waits holds -1 less
    its length; the others ask for one position. Pages run out on the way, and come back when a request ends."""
    n = 7
    s = Slots(n, 9, fmt, seed=fmt)
    # four requests start with prompts (their attention is prefill's business); slots 2, 4 and 6 have none
    prompts = np.array([3, 63, 0, 130, 0, 64, 0])
    s.lens[prompts > 0] = 0
    s.push()
    rows = int(prompts.sum())
    big = s.rows(rows)
    st = torch.cuda.Stream()
    s.step(big, rows, prompts, s.fill(big), lambda: s.launch(big, rows, st.cuda_stream, attention=False), attention=False)
    assert s.lens.tolist() == [3, 63, -1, 130, -1, 64, -1] and s.n_free == 9 - 1 - 1 - 3 - 1
    small, graph, ask, refused, waited = s.rows(n), C.c_void_p(), np.ones(n, int), 0, 0
    if captured:
        torch.cuda.synchronize()
        ok(dev.vv_dev_graph_begin(st.cuda_stream))
        s.launch(small, n, st.cuda_stream)
        ok(dev.vv_dev_graph_end(st.cuda_stream, C.byref(graph)))

    def run():
        if captured:
            ok(dev.vv_dev_graph_launch(graph, st.cuda_stream))
        else:
            s.launch(small, n, st.cuda_stream)

    for step in range(14):
        if step in (3, 9):
            s.lens[0] = -1 - s.lens[0]                   # waits
        if step in (6, 12):
            s.lens[0] = -1 - s.lens[0]                   # goes on where it was
        if step in (2, 4, 5):
            s.lens[{2: 2, 4: 4, 5: 6}[step]] = 0         # a request starts in an idle slot; the last finds no page
        if step == 10:                                   # one ends: its pages go back on the stack, its slot is idle
            gone = pages_of(s.lens[3])
            s.free[s.n_free:s.n_free + gone] = s.tables[3, :gone]
            s.n_free += gone
            s.lens[3] = -1
        s.push()
        idle = (s.lens < 0).sum()
        want = s.step(small, n, ask, s.fill(small), run)
        assert want["row_starts"].tolist() == list(range(n + 1))
        assert want["counts"][2] >= idle
        refused += int(want["counts"][2] - idle)
        waited += int(s.lens[0] < -1)
    assert refused > 0 and waited == 6 and (s.lens > 0).sum() == 6
    if captured:
        dev.vv_dev_graph_destroy(graph)


@pytest.mark.parametrize("fmt", [FP16, E4M3, E5M2])
@pytest.mark.parametrize("captured", [False, True])
def test_every_slot_decodes(fmt, captured):
    """All slots decode from the first step on, from prompts that end at and around a page's end; two fill their tables
    and are refused from there on."""
    prompts = np.array([3, 63, 64, 130, 1, 191])
    n, rows = len(prompts), int(prompts.sum())
    s = Slots(n, 3 * n, fmt, seed=50 + fmt)
    s.lens[:] = 0
    s.push()
    big, st = s.rows(rows), torch.cuda.Stream()
    s.step(big, rows, prompts, s.fill(big), lambda: s.launch(big, rows, st.cuda_stream, attention=False), attention=False)
    small, graph = s.rows(n), C.c_void_p()
    if captured:
        torch.cuda.synchronize()
        ok(dev.vv_dev_graph_begin(st.cuda_stream))
        s.launch(small, n, st.cuda_stream)
        ok(dev.vv_dev_graph_end(st.cuda_stream, C.byref(graph)))
    for step in range(66):
        x = s.fill(small)
        s.step(small, n, np.ones(n, int), x, (lambda: ok(dev.vv_dev_graph_launch(graph, st.cuda_stream))) if captured
               else (lambda: s.launch(small, n, st.cuda_stream)))
    assert s.lens.tolist() == [69, 129, 130, 192, 67, 192]
    if captured:
        dev.vv_dev_graph_destroy(graph)
