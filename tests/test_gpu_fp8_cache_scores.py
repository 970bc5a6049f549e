"""Attention over an e4m3 cache where scores are far from zero, against the definition in 64 bits. Softmax does not change
when all scores move together: rows whose scores are all far below zero, or are so over a stretch of the keys, are as
ordinary as others (keys with a common part, a first token that draws all attention). Tolerances: test_gpu_fp8_cache.py's."""

import math

import pytest
import torch

import fp8_cache_reference as ref
from kvx import ops
from test_gpu_fp8_cache import NAN, Setup, check_attention, fp8

pytestmark = pytest.mark.gpu


def lowered(gpu, lens, q_lens, heads, per_kv, hd, dtype, level, near=()):
    """A Setup whose scores lie within a few units of one value below -level, but for the groups of 16 keys in `near`
    (sequence, group), whose scores are near 0: queries near -1, keys near 1 under one scale, or a tiny one."""
    s = Setup(gpu, lens, q_lens, heads, per_kv, hd, 64, 16, dtype, unused=NAN)
    g = torch.Generator().manual_seed(7)
    s.q = (-1.0 - 0.1 * torch.randn(s.q.shape, generator=g)).to(dtype)
    used = s.k != NAN
    s.k = torch.where(used, torch.randint(0x36, 0x39, s.k.shape, generator=g, dtype=torch.uint8), s.k)  # 0.875 to 1
    s.ks.fill_(2.0 ** math.ceil(math.log2(level / (0.85 * hd ** 0.5))))
    for b, group in near:
        s.ks[int(s.tables[b, group * 16 // 64]), group * 16 % 64 // 16] = 2.0 ** -9
    return s


def check(s):
    want, want_lse, bound = s.want()
    check_attention(*s.run(), want, want_lse, bound, s.dtype, s.hd, 2.0 ** -8)
    # The weights that this lse gives, as tests of the weights bound them.
    where, how = s.batch()
    lse = want_lse.float()
    got = ops.attention_weights_fp8(s.q.to(s.gpu), lse.to(s.gpu), fp8(s.k, s.gpu), s.ks.to(s.gpu), *where, s.scale, **how)
    total = ref.weights(s.q, lse, s.k, s.ks, s.tables, s.lens, s.ranges, s.scale, got.shape[2])
    score = max(b[1] for b in bound.values())
    top = float(lse[lse.isfinite()].abs().max())
    terms = max(b - a for a, b in s.ranges) * s.q.shape[1] // s.k.shape[2]
    off = 2 * ((s.hd + 8) * 2.0 ** -24 * score + (top + score) * 2.0 ** -22 + (terms + 8) * 2.0 ** -24)
    assert ((got.cpu().double() - total).abs() <= total * off + 2.0 ** -100).all()
    return want_lse


@pytest.mark.parametrize("level", [100, 400])
@pytest.mark.parametrize("hd,per_kv,dtype", [(64, 4, torch.bfloat16), (128, 4, torch.bfloat16), (256, 2, torch.bfloat16),
                                             (128, 8, torch.float16)])
@pytest.mark.parametrize("rows", [None, 1, 4])
def test_all_scores_of_few_rows_far_below_zero(gpu, hd, per_kv, dtype, level, rows):
    # Contexts of one token, of one key more than a step, of several steps a wave, of several splits.
    lens = [1, 33, 300, 2100, 0]
    q_lens = None if rows is None else [1, rows, rows, rows, 0]
    lse = check(lowered(gpu, lens, q_lens, 1, per_kv, hd, dtype, level))
    assert (lse[lse.isfinite()] < -89).all()  # exp() of it is no normal fp32 number


@pytest.mark.parametrize("near", [0, 1, 2, 17, 70, 131])
@pytest.mark.parametrize("hd,rows", [(128, 1), (128, 6), (256, 5)])
def test_few_rows_with_one_stretch_near_zero(gpu, hd, rows, near):
    check(lowered(gpu, [2100, 300], [rows, 1], 1, 4, hd, torch.bfloat16, 200, [(0, near)]))


@pytest.mark.parametrize("hd", [64, 128])
def test_few_rows_with_low_scores_in_later_splits_alone(gpu, hd):
    check(lowered(gpu, [2100], None, 1, 4, hd, torch.bfloat16, 300, [(0, group) for group in range(64)]))


@pytest.mark.parametrize("level", [100, 400])
@pytest.mark.parametrize("hd,per_kv,dtype", [(64, 2, torch.bfloat16), (128, 2, torch.bfloat16), (96, 4, torch.float16),
                                             (256, 1, torch.bfloat16)])
def test_all_scores_of_chunks_far_below_zero(gpu, hd, per_kv, dtype, level):
    # A whole prompt, chunks behind prefixes of less than a pass and of several, one row, more rows than tokens.
    lens, q_lens = [40, 71, 700, 1, 3], [40, 33, 50, 1, 5]
    lse = check(lowered(gpu, lens, q_lens, 1, per_kv, hd, dtype, level))
    assert (lse[lse.isfinite()] < -89).all()


@pytest.mark.parametrize("near", [0, 1, 2, 9, 70, 129])
@pytest.mark.parametrize("hd,dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (128, torch.float16)])
def test_chunks_with_one_stretch_near_zero(gpu, hd, dtype, near):
    # 2,100 keys in several splits; rows 0 to 35 of the chunk do not see the last groups.
    check(lowered(gpu, [2100, 300], [40, 1], 1, 4, hd, dtype, 200, [(0, near)]))


@pytest.mark.parametrize("hd", [64, 128])
def test_chunks_with_low_scores_in_later_splits_alone(gpu, hd):
    check(lowered(gpu, [2100], [40], 1, 4, hd, torch.bfloat16, 300, [(0, group) for group in range(64)]))
