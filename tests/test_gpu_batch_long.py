"""Batched decode attention over long caches, to bounds that see one lost page or position."""
import numpy as np
import pytest
import torch

from batch_util import PAGE, attend, attend_bound_lifted, census, census_bound, pages_of
from test_gpu_batch_serving import E4M3, E5M2, FP16, TORCH_FP8, Pool

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
