"""Batched decode attention at the ends of its number formats: scores of any size that FP16 queries can give,
and the FP8 codes that stand for no number."""
import ctypes as C

import numpy as np
import pytest
import torch

from batch_util import attend, slots_of
from gpu_util import dev, ok, stream
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


@pytest.mark.parametrize("fmt", [E4M3, E5M2])
def test_codes_that_are_no_number(fmt):
    """What no store of this library writes: E4M3's 0x7F and 0xFF and E5M2's 0x7D .. 0x7F are NaN here, in a value and in
    a key, and E5M2's 0x7C is infinity. One position a sequence."""
    codes = np.array([0x7F, 0xFF] if fmt == E4M3 else [0x7C, 0xFC, 0x7D, 0x7F, 0xFE], np.uint8)
    p = Pool([1] * len(codes), 2, 1, 128, fmt=fmt, seed=3)
    at = torch.from_numpy(np.concatenate([slots_of(t, 1) for t in p.tables])).cuda()
    p.store[0][at] = 0
    p.store[1][at] = 0
    p.store[1][at, 0, 5] = torch.from_numpy(codes).cuda()
    out = p.call().float().cpu().numpy()
    want = torch.from_numpy(codes).view(TORCH_FP8[fmt]).float().numpy()
    assert np.array_equal(out[:, :, 5], np.repeat(want[:, None], 2, 1), equal_nan=True)
    assert (np.delete(out, 5, 2) == 0).all()
    p.store[1][at] = 0
    p.store[0][at, 0, 5] = torch.from_numpy(codes).cuda()
    p.q[:] = 1
    nan = np.isnan(p.call().float().cpu().numpy()).all(-1).all(-1)
    assert nan[np.isnan(want)].all()
    if fmt == E4M3:                       # where one sequence is decoded and where a store is unpacked they are numbers
        held = torch.from_numpy(np.repeat(codes, 32 * 128)).cuda().view(64, 1, 128)
        wide = torch.zeros(64, 1, 128, dtype=torch.float16, device="cuda")
        ok(dev.vv_kv_dequant_dev(held.data_ptr(), None, None, wide.data_ptr(), 1, 128, 64, fmt, stream()))
        assert (wide[:32] == 480.0).all() and (wide[32:] == -480.0).all()
        zero, one = torch.zeros_like(held), torch.zeros(2, 128, dtype=torch.float16, device="cuda")
        scratch = torch.empty(dev.vv_attn_scratch_bytes(2, 1, 128), dtype=torch.uint8, device="cuda")
        view = dev.KvView(k=zero.data_ptr(), v=held.data_ptr(), k_meta=None, v_meta=None, page_table=None, format=fmt,
                          n_kv_heads=1, head_dim=128)
        ok(dev.vv_attn_decode(2, p.q.data_ptr(), C.addressof(view), one.data_ptr(), 2, 1, None, scratch.data_ptr(), stream()))
        assert (one == 480.0).all()
