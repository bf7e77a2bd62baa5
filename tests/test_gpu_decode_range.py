"""The decode step's attention at the ends of its range, every variant against the float64
reference."""

from __future__ import annotations

import math

import pytest
import torch

import test_gpu_decode as base
from kernelpilot_b200 import specs_decode as sd
from kernelpilot_b200.specs import randn

pytestmark = pytest.mark.gpu

DEV = base.DEV
VARIANTS = base.VARIANTS


def rows_of(B, Hq, Hkv, D, n, dtype, seed):
    """q, and keys and values in fp32 as (B, Hkv, n, D)."""
    g = base.generator(seed)
    q = randn((B, Hq, D), dtype, DEV, g)
    k, v = (randn((B, Hkv, n, D), torch.float32, DEV, g) for _ in range(2))
    return q, k, v


def cache_of(rows, page, dtype, e4m3):
    """(B, Hkv, n, D) rows into pages of their own: (cache, scales or None, table)."""
    B, H, n, D = rows.shape
    per = -(-n // page)
    pool = torch.zeros(B, H, per * page, D, device=DEV)
    pool[:, :, :n] = rows
    pool = pool.view(B, H, per, page, D).transpose(1, 2).reshape(B * per, H, page, D)
    table = torch.arange(B * per, dtype=torch.int32, device=DEV).view(B, per)
    if not e4m3:
        return pool.to(dtype), None, table
    codes, scale = sd.e4m3_rows(pool)
    return codes, scale.float(), table


def inputs(q, k, v, dtype, e4m3, page=16):
    kc, ks, table = cache_of(k, page, dtype, e4m3)
    vc, vs, _ = cache_of(v, page, dtype, e4m3)
    lens = torch.full((q.shape[0],), k.shape[2], dtype=torch.int32, device=DEV)
    return q, kc, vc, table, lens, ks, vs


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("dtype", base.DTYPES)
@pytest.mark.parametrize("gap", [15, 30, 45, 60])
@pytest.mark.parametrize("n,best,at", [(40, 3, 20), (40, 20, 3), (300, 3, 250), (300, 250, 3)])
def test_infinite_values_under_small_weights(n, best, at, gap, dtype, variant):
    # every key but `best` is `gap` nats below it; two elements of key `at` are infinite. The
    # weight is e^-gap, not zero, so the outputs are the infinities
    for D in (64, 128):
        q, k, v = rows_of(2, 4, 1, D, n, dtype, 1)
        q.zero_()[..., 0] = 1.0
        k[..., 0] = -float(gap)
        k[:, :, best, 0] = 0.0
        clean = inputs(q, k, v, dtype, 0)
        v[:, :, at, 9], v[:, :, at, 5] = float("inf"), float("-inf")
        ins = inputs(q, k, v, dtype, 0)
        got = base.run_paged(ins, variant, 1.0)
        (want,) = sd.paged_attention_reference(*ins, 1.0)
        assert torch.all(got[..., 9] == float("inf")) and torch.all(got[..., 5] == float("-inf"))
        live = torch.tensor([i for i in range(D) if i not in (5, 9)], device=DEV)
        base.check(got[..., live], want[..., live], base.attention_limit(*clean, 1.0))


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Hq,D", [(4, 64), (4, 128), (12, 128), (4, 256), (12, 96)])
def test_zero_rows_among_tiny_values(Hq, D, dtype, variant):
    # a row of zeros has the scale 1, whatever the others' are; here those lie near 2^-38.
    # fp16 is left out: the results are far below its smallest number
    q, k, v = rows_of(5, Hq, 1, D, 300, dtype, 2)
    v *= 1e-9
    v[0, :, 7] = 0.0         # one in the middle of a tile
    v[1, :, :40] = 0.0       # the first tiles whole
    v[2, :, 250:] = 0.0      # the last ones
    v[3, :, ::2] = 0.0       # every other
    v[4, :, 1:] = 0.0        # all but one
    ins = inputs(q, k, v, dtype, 1)
    for n in (300, 40, 1):
        ins[4].fill_(n)
        base.check_paged(ins, variant)


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("dtype,ratio", [(torch.bfloat16, 12), (torch.bfloat16, 20),
                                         (torch.bfloat16, 24), (torch.float16, 20),
                                         (torch.float32, 20)], ids=str)
@pytest.mark.parametrize("Hq,D", [(4, 64), (12, 128), (4, 256)])
def test_queries_with_one_large_channel(Hq, D, dtype, ratio, variant):
    # the large channel meets zeros in every key, so the scores are the other channels' alone.
    # e4m3 products take q as fp16 with the head's largest element at 2^14: the smallest here,
    # 2^29 below, lies at 2^-15 and keeps a bf16's eight bits (fp16: 2^25 below, eleven bits),
    # so that 16-bit queries are exact; an fp32 one is off by 2^-25, half of fp16's smallest
    # number, which is 2^-39 of the largest element
    q, k, v = rows_of(3, Hq, 1, D, 200, dtype, 3)
    low = 2.0 ** -8 if dtype == torch.float16 else 1.0
    q.copy_(torch.clamp(q.float().abs(), min=0.05) * q.float().sign() * low)
    q[..., 0] = low * 2.0 ** ratio
    k[..., 0] = 0.0
    ins = inputs(q, k, v, dtype, 1)
    scale = 1.0 / (math.sqrt(D) * low)
    lim = base.attention_limit(*ins, scale)
    if dtype == torch.float32 and variant == 1:
        # each of D channels off by 2^-39 of the largest element: the score by that times the
        # sum of |k|, a weight by twice it
        kk = sd._values(ins[1], ins[5], torch.arange(ins[1].shape[0], device=DEV)[:, None],
                        torch.arange(16, device=DEV), torch.float64)
        off = 2.0 ** (ratio - 39) * float(kk.abs().sum(-1).max()) * scale
        lim = lim + 2 * off * float(v.abs().max())
    got = base.run_paged(ins, variant, scale)
    (want,) = sd.paged_attention_reference(*ins, scale)
    base.check(got, want, lim)


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("e4m3", [0, 1])
@pytest.mark.parametrize("size", [115, -118])
def test_very_large_and_very_small_values(size, e4m3, dtype, variant):
    # 700 weights of at most 1 over values of up to 6 * 2^115 sum to less than 2^128; the small
    # ones are far above fp32's smallest normal number, 2^-126
    for Hq, D in ((4, 64), (4, 128), (12, 128), (4, 256)):
        q, k, v = rows_of(2, Hq, 1, D, 700, dtype, 4)
        v *= 2.0 ** size
        ins = inputs(q, k, v, dtype, e4m3)
        for n in (700, 16):  # joined from parts, and not
            ins[4].fill_(n)
            base.check_paged(ins, variant)


def weight_error(dtype, e4m3, variant):
    """What a weight may be off by beside fp32's roundings, relative to itself: where weights
    enter the products as two 16-bit parts, what the two leave. bf16: the first is cut to 8
    bits (2^-7 left), the second rounded to 2^-8 of that. fp16 values: cut to 11 bits (2^-10),
    2^-11 of that; e4m3 values, as fp16: rounded (2^-11), 2^-11 of that."""
    if variant == 0 or (dtype == torch.float32 and not e4m3):
        return 0.0
    if e4m3:
        return 2.0 ** -22
    return 2.0 ** -15 if dtype == torch.bfloat16 else 2.0 ** -21


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("dtype", base.DTYPES)
@pytest.mark.parametrize("e4m3", [0, 1])
@pytest.mark.parametrize("n", [2, 3, 5])
def test_weights_keep_the_bits_of_their_path(n, e4m3, dtype, variant):
    # one channel of q and k makes the scores, of at most 4 and exact but for the roundings of
    # one product (16-bit q) or of q's two fp16 parts (2^-22, fp32 q on e4m3), the scale and
    # the change to powers of two: 4 * 2^-24 of 4 and 2^-22 of 4. The maximum's subtraction is
    # off by 2^-24 of 4 too, 2^x by 2^-22 (twice: above and below the division); up to n + 6
    # roundings of the sums, the division and the products, and 2^-23 for each of the four tensor
    # core products, whose sums are cut
    B, Hq, D = 32, 4, 64
    q, k, v = rows_of(B, Hq, 1, D, n, dtype, 5)
    top = 1.0 + torch.rand(B, Hq, generator=base.generator(6), device=DEV)
    q.zero_()[..., 0] = top.to(dtype)
    k.zero_()[..., 0] = torch.randint(0, 16, k.shape[:3], generator=base.generator(7),
                                      device=DEV) / 8.0
    ins = inputs(q, k, v, dtype, e4m3)
    got = base.run_paged(ins, variant, 1.0)
    (want,) = sd.paged_attention_reference(*ins, 1.0)
    # sum of w |v| per output element
    absolute = (*ins[:2], ins[2].float().abs().to(ins[2].dtype), *ins[3:])
    (av,) = sd.paged_attention_reference(*absolute, 1.0)
    score = 4 * (5 * base.U24 + (2.0 ** -22 if e4m3 and dtype == torch.float32 else 0.0))
    rel = 2 * score + 2 * 2.0 ** -22 + (n + 14) * base.U24 + 2 * weight_error(dtype, e4m3, variant)
    base.check(got, want, rel * av)


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("e4m3", [0, 1])
@pytest.mark.parametrize("size", [124, 60, -60, -110, -122])
def test_queries_of_any_size(size, e4m3, dtype, variant):
    # the score's scale brings them back; the smallest elements are fp32's subnormals (a bf16's
    # too), exact in the inputs
    q, k, v = rows_of(2, 4, 1, 64, 90, dtype, 8)
    ins = inputs((q.float() * 2.0 ** size).to(dtype), k, v, dtype, e4m3)
    if size == 124 and dtype == torch.bfloat16 and not e4m3 and variant == 1:
        # outside what kp_b200.h allows: 16-bit products are summed before the scale, and sums of
        # 64 products of values near 2^124 and 1 pass fp32's largest number
        sums = ins[0].double().abs() @ ins[1].double().abs().amax(0)[0].transpose(0, 1)
        assert float(sums.max()) > torch.finfo(torch.float32).max
        return
    base.check_paged(ins, variant, scale=2.0 ** -size / 8)


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("dtype", base.DTYPES)
def test_e4m3_rows_and_queries_that_are_not_finite(dtype, variant):
    # a key or value row that was not finite has the scale NaN: its sequence's heads are NaN; so
    # is a head whose query holds an infinity or NaN, and no other
    q, k, v = rows_of(4, 4, 1, 64, 90, dtype, 9)
    q[2, 1, 3], q[2, 2, 60] = float("inf"), float("nan")
    k[0, 0, 50, 7] = float("inf")
    v[1, 0, 3, 9] = float("nan")
    ins = inputs(q, k, v, dtype, 1)
    got = base.run_paged(ins, variant)
    (want,) = sd.paged_attention_reference(*ins)
    assert torch.isnan(got[:2]).all() and torch.isnan(want[:2]).all()
    assert torch.isnan(got[2, 1:3]).all() and torch.isnan(want[2, 1:3]).all()
    clean = (q.nan_to_num(posinf=0.0), *ins[1:])
    lim = base.attention_limit(*clean)
    for at in ((2, slice(0, 1)), (2, slice(3, 4)), (3, slice(0, 4))):
        base.check(got[at], want[at], lim[at])
