"""Packed attention where softmax weights are far apart, through every way that a call can take: row tiles, row tiles cut
along the keys, key chunks of one launch and divided ones."""
import math

import pytest
import torch

import idolq_lib as L
from test_gpu_attention_packed import BF16, DEV, FP16, check, offsets, oracle

pytestmark = pytest.mark.gpu

WAYS = {  # lq, lk, max_q, max_k: one sequence each
    "tile": (260, 260, 0, 0), "cut tiles": (150, 2600, 0, 2600), "short": (2, 900, 2, 900),
    "divided": (1, 9000, 1, 9000), "long": (3, 40000, 3, 40000)}


def call(q, k, v, way, **kw):
    lq, lk, mq, mk = WAYS[way]
    return L.attention_packed(q, k, v, offsets([lq]).to(DEV), offsets([lk]).to(DEV), 1, 1, q.shape[1], max_q=mq, max_k=mk,
                              **kw)


def rows(n, hd, seed, std=0.0):
    return torch.randn((n, hd), generator=torch.Generator().manual_seed(seed)) * std


@pytest.mark.parametrize("way", list(WAYS))
@pytest.mark.parametrize("power", [10, 20, 24, 27, 28, 29, 30, 33])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_large_scores_that_tie(way, power, dtype):
    # every key's score is 2^power exactly (and rounds alike for all keys in base 2): all weights are the same
    lq, lk = WAYS[way][:2]
    q, k, v = torch.zeros((lq, 64)), torch.zeros((lk, 64)), rows(lk, 64, 4, 1.0)
    q[:, 3], k[:, 3] = 2.0 ** 10, 2.0 ** 10
    q, k, v = (t.to(dtype).to(DEV) for t in (q, k, v))
    want = v.double().cpu().mean(0).expand(lq, 64)
    check(call(q, k, v, way, scale=2.0 ** (power - 20)), want, v.double().cpu().abs().mean(0).expand(lq, 64), dtype)


@pytest.mark.parametrize("way", list(WAYS))
@pytest.mark.parametrize("power", [3, 19, 22, 25, 27])
def test_large_scores_that_tie_over_values_near_the_largest(way, power):
    # bf16 sums stay finite: hundreds of values of an eighth of the largest with the same weight
    lq, lk = WAYS[way][:2]
    q, k, v = torch.zeros((lq, 64)), torch.zeros((lk, 64)), 1 + rows(lk, 64, 11, 0.1).clamp(-0.5, 0.5)
    q[:, 3], k[:, 3] = 2.0 ** 10, 2.0 ** 10
    q, k, v = q.to(BF16).to(DEV), k.to(BF16).to(DEV), (v * (torch.finfo(BF16).max / 8)).to(BF16).to(DEV)
    want = v.double().cpu().mean(0).expand(lq, 64)
    check(call(q, k, v, way, scale=2.0 ** (power - 20)), want, want, BF16)


@pytest.mark.parametrize("way", list(WAYS))
@pytest.mark.parametrize("gap", [12.0, 15.0, 17.5, 19.0])
@pytest.mark.parametrize("dtype,hd", [(FP16, 64), (FP16, 128), (BF16, 64)])
def test_small_weights_next_to_a_dominant_key(way, gap, dtype, hd):
    # The first key stands `gap` above the others, its values are 0: the output is the small weights' alone. fp16 weights are
    # multiples of 2^-24 where the largest is 2^8 or more, so each is off by at most 2^-25 / 2^8 = 2^-33 of the row's sum,
    # beside the relative roundings that check() counts.
    lq, lk = WAYS[way][:2]
    q, k, v = rows(lq, hd, 1, 0.3), rows(lk, hd, 2, 0.3), 1 + rows(lk, hd, 3, 0.25)
    q[:, 0], k[:, 0], k[0, 0] = 4.0, 0.0, gap * math.sqrt(hd) / 4
    v[0] = 0
    q, k, v = (t.to(dtype).to(DEV) for t in (q, k, v))
    o, big = oracle(q, k, v, [lq], [lk], 1, 1, hd, False)
    if dtype == FP16:
        # check() allows 2^-13 of `big` among others: what the multiples add is counted as that much more of it
        big = big + 2.0 ** 13 * 2.0 ** -33 * v.double().cpu().abs().sum(0)
    check(call(q, k, v, way), o, big, dtype)


@pytest.mark.parametrize("way", list(WAYS))
@pytest.mark.parametrize("level", [-100.0, -12.0, 0.0, 100.0])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_first_keys_with_scores_of_minus_infinity(way, level, dtype):
    # keys whose score is -inf have no weight, wherever they are: the first keys of every tile, wave or chunk walk, and
    # more; the others' scores are near `level`
    lq, lk = WAYS[way][:2]
    q, k, v = rows(lq, 64, 5, 0.3), rows(lk, 64, 6, 0.3), rows(lk, 64, 7, 1.0)
    q[:, 0], k[:, 0], q[:, 1], k[:, 1] = 1.0, 0.0, 32.0, level / 4
    k[:min(lk - 60, 700), 0] = -math.inf
    q, k, v = (t.to(dtype).to(DEV) for t in (q, k, v))
    got = call(q, k, v, way, causal=False)
    o, big = oracle(q, k, v, [lq], [lk], 1, 1, 64, False)
    # scores up to 2^8: their fp32 sums are off by up to 2^-15 of them, 2^-7 in the exponent (12: 2^-11; and 2^-13 for the
    # first finite ones, which are taken 2^12 above the row's reference point)
    err, u = (got.double().cpu() - o).abs(), torch.finfo(dtype).eps / 2
    assert (err <= u * o.abs() + (u + (2.0 ** -7 if abs(level) > 12 else 2.0 ** -10)) * (big + o.abs())).all()
    k[:, 0] = -math.inf
    assert (call(q, k, v, way) == 0).all()     # nothing has weight


@pytest.mark.parametrize("way", ["cut tiles", "short", "divided", "long"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_a_value_that_is_no_number_is_seen_behind_any_weight(way, bad, dtype):
    # the keys from 384 on have scores 200 below the others, so whole waves and parts have no weight in the sum
    lq, lk = WAYS[way][:2]
    q, k, v = rows(lq, 64, 8, 0.3), rows(lk, 64, 9, 0.3), rows(lk, 64, 10, 1.0)
    q[:, 0], k[:, 0] = 16.0, 0.0
    k[384:, 0] = -100.0
    q, k, v = (t.to(dtype).to(DEV) for t in (q, k, v))
    clean = call(q, k, v, way)
    v[lk * 2 // 3 if lk > 1000 else 390, 5] = bad
    got = call(q, k, v, way)
    assert not torch.isfinite(got[:, 5]).any()
    others = [c for c in range(64) if c != 5]
    assert torch.equal(got[:, others], clean[:, others]) and torch.isfinite(clean).all()
