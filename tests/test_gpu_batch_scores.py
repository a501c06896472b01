"""Batched decode attention at the ends of its number formats: scores of any size that FP16 queries can give."""
import numpy as np
import pytest
import torch

from batch_util import attend, slots_of
from test_gpu_batch_serving import E4M3, E5M2, FP16, TORCH_FP8, Pool

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nq,nkv,hd,fmt", [(8, 2, 128, FP16), (8, 2, 64, FP16), (6, 2, 96, FP16), (8, 2, 128, E4M3),
                                           (8, 2, 128, E5M2)])
def test_attend_huge_scores(nq, nkv, hd, fmt):
    """Keys that are one number c in every channel, queries that are one power of two: every product and partial sum of
    a score is exact in FP32 (c has eleven bits at most, 128 of them seven more). Distinct c differ by 2^-11 of the
    largest or more, thousands of exponents at these scores, so the result is the mean of the values whose key is the
    largest: their weights are one number, 2^10 in FP16, exactly; their FP32 sums are off by half a step, 2^-24, at each of
    up to 256 blocks that a wave adds; then the one rounding of the result."""
    lens = [1, 5, 64, 70, 130, 300, 1000, 4000]
    p = Pool(lens, nq, nkv, hd, fmt=fmt, seed=fmt + hd)
    rng = np.random.default_rng(hd + fmt)
    power = rng.permutation(np.arange(len(lens) * nq) % 5 + 11).reshape(len(lens), nq)      # 2^11 .. 2^15
    p.q = torch.from_numpy(np.repeat((2.0 ** power).astype(np.float16)[..., None], hd, -1)).cuda()
    low, high = (2.0 ** 13, 2.0 ** 15) if fmt != E4M3 else (256.0, 448.0)
    for i, n in enumerate(lens):
        c = torch.from_numpy(rng.uniform(low, high, (n, nkv, 1)).astype(np.float16)).cuda().expand(n, nkv, hd)
        if fmt != FP16:
            c = c.float().to(TORCH_FP8[fmt]).view(torch.uint8)
        p.store[0][torch.from_numpy(slots_of(p.tables[i], n)).cuda()] = c
    got = p.call().float().cpu().numpy().astype(np.float64)
    q = p.q.float().cpu().numpy().astype(np.float64)
    for i in range(len(lens)):
        want, mag = attend(q[i], *p.values(i))
        ulp = np.spacing(np.abs(want).astype(np.float16)).astype(np.float64)
        worst = np.abs(got[i] - want) / (mag * 2.0 ** -16 + 0.5 * ulp)
        assert (worst <= 1.0).all(), f"{lens[i]} positions: {np.nanmax(worst)} of the bound, {np.isnan(worst).sum()} NaN"
