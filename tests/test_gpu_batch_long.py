"""Batched decode attention over long caches, to bounds that see one lost page, and the kernel forms that only large or
many rows run: workers with several lists of pages, every fold, the streaming and the several-round rotary append."""
import ctypes as C

import numpy as np
import pytest
import torch

from batch_util import PAGE, attend, attend_bound_lifted, census, census_bound, pages_of, slots_of
from gpu_util import dev, ok, stream
from test_gpu_batch_serving import E4M3, E5M2, FP16, TORCH_FP8, Pool, ints, raw
from test_gpu_batch_serving import test_append_against_the_separate_calls as append_against_the_separate_calls

pytestmark = pytest.mark.gpu


def check_lifted(p, out, rows):
    got, q = out.float().cpu().numpy().astype(np.float64), p.q.float().cpu().numpy().astype(np.float64)
    for i in rows:
        k, v = p.values(i)
        want, mag = attend(q[i], k, v)
        worst = np.abs(got[i] - want) / attend_bound_lifted(want, mag, k.shape[0], np.abs(v).max(initial=0.0))
        assert (worst <= 1.0).all(), f"sequence {i} of {k.shape[0]} positions: {worst.max():.2f}x the bound"


@pytest.mark.parametrize("fmt,hd", [(FP16, 128), (FP16, 64), (E4M3, 128), (E5M2, 128)])
@pytest.mark.parametrize("lens", [[14449], [60] * 150 + [20000] + [60] * 149, [14449, 0, 12345, 700, 1, 20000]])
def test_attend_long_to_the_lifted_bound(lens, fmt, hd):
    p = Pool(lens, 4, 2, hd, fmt=fmt, seed=len(lens) + hd)
    check_lifted(p, p.call(), sorted({0, len(lens) // 2, len(lens) - 1, int(np.argmax(lens))}))


def one(fmt):
    return 1.0 if fmt == FP16 else int(torch.tensor(1.0).to(TORCH_FP8[fmt]).view(torch.uint8))


@pytest.mark.parametrize("nq,nkv,hd,fmt", [(4, 2, 128, FP16), (28, 4, 128, FP16), (4, 2, 64, FP16), (3, 1, 96, FP16),
                                           (4, 2, 128, E4M3), (20, 1, 128, E5M2)])
@pytest.mark.parametrize("lens", [[14449], [14449 - 64 * i - i for i in range(0, 24, 5)], [20000, 0, 65, 1],
                                  [64] * 1030 + [9000, 3], [90000]])
def test_attend_counts_every_position_once(lens, nq, nkv, hd, fmt):
    """Scores all alike and values that say which page they lie in: the shares of the pages, to a bound that one position
    passes. Sequences share the pages of a small pool."""
    if hd == 96 and max(lens) > 20000:
        lens = [20001]                                           # a wave walks all of it there
    n_pages, rng = 300, np.random.default_rng(len(lens) + hd)
    tables = rng.integers(0, n_pages, (len(lens), max(pages_of(n) for n in lens))).astype(np.int32)
    p = Pool([64], nq, nkv, hd, fmt=fmt, spare=n_pages - 1)
    p.lens, p.tables, p.max_pages = list(lens), tables, tables.shape[1]
    p.q = torch.zeros(len(lens), nq, hd, dtype=torch.float16, device="cuda")
    p.store[0][:] = 0
    p.store[1][:] = 0
    page = torch.arange(n_pages, device="cuda")
    p.store[1].view(n_pages, PAGE, nkv, hd)[page, :, :, page % hd] = one(fmt)
    got = p.call().float().cpu().numpy().astype(np.float64)
    for i, n in enumerate(lens):
        want = census(tables[i, :pages_of(n)], n, hd)
        assert (np.abs(got[i] - want) <= census_bound(want)).all(), f"sequence {i} of {n} positions"


@pytest.mark.parametrize("hd,fmt", [(128, FP16), (64, FP16), (128, E4M3)])
def test_attend_workers_with_several_lists_of_pages(hd, fmt):
    """Over 256 pages a workgroup: its list of pages is filled again in the middle of a row. Five sequences of 2^20
    positions, on pages of a small pool that they share (a slot's weight counts as often as the tables name it)."""
    n, nq, nkv, n_pages = 1 << 20, 4, 2, 200
    lens = [n, n - 1, n - 64, n - 100, n, 77]
    rng = np.random.default_rng(hd)
    tables = rng.integers(0, n_pages, (len(lens), n // PAGE)).astype(np.int32)
    assert sum(pages_of(x) for x in lens) * nkv > 512 * 256 + 512
    p = Pool([n_pages * PAGE], nq, nkv, hd, fmt=fmt, seed=hd, spare=0)
    p.lens, p.tables, p.max_pages = lens, tables, n // PAGE
    g = torch.Generator(device="cuda").manual_seed(hd)
    p.q = (torch.randn(len(lens), nq, hd, generator=g, device="cuda") * 4 * hd ** -0.25).half()
    got = p.call().float().cpu().numpy().astype(np.float64)
    k, v = (s if fmt == FP16 else s.view(TORCH_FP8[fmt]) for s in p.store)
    k, v = (x.float().cpu().numpy().astype(np.float64) for x in (k, v))
    q = p.q.float().cpu().numpy().astype(np.float64)
    for i, x in enumerate(lens):
        times = np.bincount(slots_of(tables[i], x), minlength=n_pages * PAGE)
        for h in range(nq):
            s = k[:, h // (nq // nkv)] @ q[i, h] / np.sqrt(hd)
            w = times * np.exp(s - s[times > 0].max())
            w /= w.sum()
            want, mag = w @ v[:, h // (nq // nkv)], w @ np.abs(v[:, h // (nq // nkv)])
            # a workgroup's share of a row is 320 blocks a wave: their FP32 sums add 320 * 4 half steps at most
            off = attend_bound_lifted(want, mag, x, np.abs(v).max()) + mag * 1280 * 2.0 ** -24
            assert (np.abs(got[i, h] - want) <= off).all(), f"sequence {i}, head {h}"
    # and every position once
    p.q.zero_()
    p.store[1][:] = 0
    page = torch.arange(n_pages, device="cuda")
    p.store[1].view(n_pages, PAGE, nkv, hd)[page, :, :, page % hd] = one(fmt)
    got = p.call().float().cpu().numpy().astype(np.float64)
    for i, x in enumerate(lens):
        want = census(tables[i, :pages_of(x)], x, hd)
        assert (np.abs(got[i] - want) <= census_bound(want)).all(), f"shares of sequence {i}"


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens", [[5000, 300], [3000, 0, 64, 65, 2000, 1, 700, 12], [900] * 17, [64] * 600 + [7000] + [3] * 50,
                                  [20] * 520 + [4000, 0, 5]])
def test_attend_every_fold(lens, hd):
    """At most 16 rows, at most 1024, and more, some of them cut over many workgroups; two and three heads a row."""
    for nq in (4, 6):
        p = Pool(lens, nq, 2, hd, seed=len(lens) + nq)
        out = p.call()
        check_lifted(p, out, sorted({0, len(lens) // 2, len(lens) - 1, int(np.argmax(lens))}))
        assert np.array_equal(raw(p.call()), raw(out)), "another answer the second time"


@pytest.mark.parametrize("biased", [True, False])
@pytest.mark.parametrize("rows,nq,nkv,hd,fmt", [
    (300, 28, 4, 128, FP16), (300, 28, 4, 128, E4M3), (301, 28, 4, 128, E5M2), (600, 12, 2, 128, FP16),    # streaming stores
    (400, 28, 4, 64, FP16),
    (3, 100, 16, 128, FP16), (3, 100, 16, 128, E4M3), (6, 260, 4, 64, FP16), (600, 100, 16, 128, FP16),   # over 1024 items a row
    (700, 14, 2, 64, FP16)])                                                                         # several rows a workgroup
def test_append_of_many_and_of_wide_rows(rows, nq, nkv, hd, fmt, biased):
    append_against_the_separate_calls(rows, nq, nkv, hd, fmt, biased)


def test_two_captured_steps_share_a_scratch():
    """Two graphs of different batches over one scratch, replayed in turn on one stream, with eager work between."""
    a, b = Pool([3000, 5, 700], 28, 4, 128, seed=40), Pool([64] * 40 + [2000], 12, 2, 128, seed=41)
    want = [raw(x.call()) for x in (a, b)]
    sizes = [dev.vv_attn_decode_batch_scratch_bytes(len(x.lens), x.nq, x.nkv, x.hd) for x in (a, b)]
    scratch = torch.full((max(sizes),), 0xFF, dtype=torch.uint8, device="cuda")
    st, held = torch.cuda.Stream(), []
    torch.cuda.synchronize()
    for x in (a, b):
        lens, tables, out, graph = ints(x.lens), ints(x.tables), torch.empty_like(x.q), C.c_void_p()
        view = dev.KvView(k=x.store[0].data_ptr(), v=x.store[1].data_ptr(), k_meta=None, v_meta=None,
                          page_table=tables.data_ptr(), format=FP16, n_kv_heads=x.nkv, head_dim=x.hd)
        torch.cuda.synchronize()
        ok(dev.vv_dev_graph_begin(st.cuda_stream))
        ok(dev.vv_attn_decode_batch(2, x.q.data_ptr(), C.addressof(view), out.data_ptr(), x.nq, len(x.lens),
                                    lens.data_ptr(), x.max_pages, x.n_pages, scratch.data_ptr(), max(sizes), st.cuda_stream))
        ok(dev.vv_dev_graph_end(st.cuda_stream, C.byref(graph)))
        held.append((lens, tables, out, graph, view))
    for _ in range(5):
        for _, _, out, _, _ in held:
            out.fill_(float("nan"))
        torch.cuda.synchronize()
        for _, _, _, graph, _ in held:
            ok(dev.vv_dev_graph_launch(graph, st.cuda_stream))
        torch.cuda.synchronize()
        for w, (_, _, out, _, _), x in zip(want, held, (a, b)):
            assert np.array_equal(raw(out), w)
            assert np.array_equal(raw(x.call()), w)
    for _, _, _, graph, _ in held:
        dev.vv_dev_graph_destroy(graph)


@pytest.mark.parametrize("nq,nkv,hd,fmt", [(28, 4, 128, FP16), (14, 2, 64, FP16), (28, 4, 128, E4M3), (6, 3, 96, FP16)])
def test_attend_into_an_output_off_any_alignment(nq, nkv, hd, fmt):
    """Only q, the stores and the scratch have an alignment to keep: out at two bytes, lengths and tables at four."""
    p = Pool([3000, 0, 65, 700, 1], nq, nkv, hd, fmt=fmt, seed=44)
    want, n = raw(p.call()), len(p.lens)
    lens, tables = (torch.cat([ints([-5]), ints(x).flatten()]) for x in (p.lens, p.tables))
    out = torch.full((n * nq * hd + 2,), float("nan"), dtype=torch.float16, device="cuda")
    size = dev.vv_attn_decode_batch_scratch_bytes(n, nq, nkv, hd)
    scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
    view = dev.KvView(k=p.store[0].data_ptr(), v=p.store[1].data_ptr(), k_meta=None, v_meta=None,
                      page_table=tables.data_ptr() + 4, format=fmt, n_kv_heads=nkv, head_dim=hd)
    torch.cuda.synchronize()
    ok(dev.vv_attn_decode_batch(2, p.q.data_ptr(), C.addressof(view), out.data_ptr() + 2, nq, n, lens.data_ptr() + 4,
                                p.max_pages, p.n_pages, scratch.data_ptr(), size, stream()))
    assert np.array_equal(raw(out[1:-1]).reshape(want.shape), want)
    assert torch.isnan(out[0]) and torch.isnan(out[-1])
