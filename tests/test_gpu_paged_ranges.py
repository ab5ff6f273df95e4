"""Attention over the paged cache at the ends of its ranges, against the definitions in 64 bits (paged_reference.py).

Tolerances, per output row, with A = sum p |v| / sum p, as in test_gpu_paged_kv.py: half a step of the result's type; for
each score (D + 8) 2^-24 of sum |q k| <= S, once in the sum over V and once in the sum of the weights; 2^-20 for
exponentials and their arguments; (n / 16 + 16) 2^-24 for the sums over n keys; 2^-11 for a weight rounded to fp16, and
2^-25 of the row's largest weight times scale, times 448, for what fp16 cannot hold of each.  The floor is half of
the type's smallest step, so results of any size are compared."""
import math

import pytest
import torch

import paged_reference as P
import rdna4_sage
from rdna4_sage import _attention
from test_gpu_paged_kv import DEV, filled, handle, ints, queries, trees

pytestmark = pytest.mark.gpu


def compare(q, cache, table, lens, mask=None, sm_scale=None, lost=2.0 ** -25):
    """Result and log-sum-exp within the bounds above; returns the results of both sides."""
    o, lse = rdna4_sage.attention_paged_kv(q, handle(cache), table, ints(lens), mask, None, "NHD", sm_scale, True)
    _attention.check_status(torch.device("cuda", 0))
    want, want_lse, mean, S, top = P.attention(q, cache, table, lens, mask, None, sm_scale)
    n, D, info = max(lens) + q.shape[1], q.shape[-1], torch.finfo(q.dtype)
    weight = 2 * ((D + 8) * 2.0 ** -24 * S + 2.0 ** -22 * want_lse.transpose(1, 2).abs().nan_to_num(0, 0, 0) +
                  2.0 ** -20 + (n / 16 + 16) * 2.0 ** -24)
    tol = info.eps / 2 * want.abs() + mean * (2.0 ** -11 + weight[..., None]) + (n * lost * 448 * top)[..., None] + \
        info.smallest_normal * info.eps / 2
    off = (o.double() - want).abs()
    assert torch.equal(o.isnan(), want.isnan())
    assert bool((off <= tol)[~want.isnan()].all()), float((off / tol).nan_to_num(0).max())
    seen = want_lse > -math.inf
    assert torch.equal(lse > -math.inf, seen)
    ltol = (weight.transpose(1, 2) + 2.0 ** -23 * want_lse.abs())[seen]
    lo = (lse.double() - want_lse).abs()[seen]
    assert bool((lo <= ltol).all()), float((lo / ltol).max())
    return o, lse


SHAPES = [(64, 1, 2), (96, 2, 8), (128, 1, 8), (128, 4, 16), (256, 1, 8), (256, 3, 8),     # D, T, H over 2 kv heads: few rows
          (64, 24, 8), (128, 40, 4), (96, 33, 4), (256, 17, 4)]                            # many


@pytest.mark.parametrize("D,T,H", SHAPES)
@pytest.mark.parametrize("power", [-101, -97, -80, -40, 60, 75, 84, 124])
def test_v_rows_of_the_smallest_and_largest_size(D, T, H, power):
    # scales near 2^-108 and 2^117, the ends of what append writes, and between them, on either side of where one exponential
    # no longer serves both sums: neither the weights' sum nor a result is lost
    lens = [5000, 70]
    cache, table = filled(lens, T, 32, 2, D, seed=D + T)
    cache["vs"].mul_(2.0 ** power)
    for size in (0.3, 3.0):
        compare(queries(2, T, H, D, size=size), cache, table, lens, trees(2, T) if T > 2 else None)


@pytest.mark.parametrize("D,T,H", SHAPES)
def test_v_rows_of_both_ends_in_one_context(D, T, H):
    lens = [1500, 200]
    cache, table = filled(lens, T, 64, 2, D, seed=D)
    plain, lse = compare(queries(2, T, H, D), cache, table, lens)
    for b in range(2):
        p, r = P.place(cache, table, b, range(0, lens[b], 2))
        cache["vs"][p, :, r] *= 2.0 ** 110
        p, r = P.place(cache, table, b, range(1, lens[b], 2))
        cache["vs"][p, :, r] *= 2.0 ** -95
        p, r = P.place(cache, table, b, range(0, lens[b], 50))
        cache["vs"][p, :, r] = 0.0
        cache["v8"].view(torch.uint8)[p, :, r] = 0
    compare(queries(2, T, H, D), cache, table, lens)


@pytest.mark.parametrize("D,T,H", SHAPES)
def test_v_rows_that_are_zero_up_to_the_last(D, T, H):
    # zero rows count in the weights' sum only, whatever came before and comes after them
    lens = [900, 130]
    cache, table = filled(lens, T, 16, 2, D, seed=T)
    for b in range(2):
        p, r = P.place(cache, table, b, range(0, lens[b] - 3))
        cache["vs"][p, :, r] = 0.0
        cache["v8"].view(torch.uint8)[p, :, r] = 0
    cache["vs"].mul_(2.0 ** -60)
    compare(queries(2, T, H, D), cache, table, lens)


@pytest.mark.parametrize("D,T,H", SHAPES)
@pytest.mark.parametrize("at", [0, 100, 803])
def test_a_v_row_with_nan_leaves_the_log_sum_exp(D, T, H, at):
    # as append writes it: scale NaN, codes 0.  The result of a row that sees it is NaN, its log-sum-exp is that of its scores
    lens = [804, 77]
    cache, table = filled(lens, T, 32, 2, D, seed=at)
    q = queries(2, T, H, D)
    a, la = compare(q, cache, table, lens)
    p, r = P.place(cache, table, 0, [at])
    cache["vs"][p, :, r] = math.nan
    cache["v8"].view(torch.uint8)[p, :, r] = 0
    b, lb = compare(q, cache, table, lens)
    assert bool(b[0].isnan().all()) and torch.equal(b[1], a[1]) and torch.equal(lb[1], la[1])


@pytest.mark.parametrize("D,T,H,B", [(64, 1, 8, 600), (128, 2, 8, 320), (256, 1, 4, 320), (64, 24, 4, 150), (128, 17, 4, 150)])
@pytest.mark.parametrize("x", [3.78125, 2.953125, 2.53125])
def test_one_dominating_key_over_a_long_context(D, T, H, B, x):
    """A key at the front with score 20, hundreds of thousands of others at x: 2^-23.4 to 2^-25.2 of its weight each, 1 to 4
    percent of the result together, and all of them rounded alike.  A row's largest weight is held at 2^7 or more, so what
    fp16 cannot hold of a weight (half of its smallest step, 2^-25) is 2^-32 of that.  As many sequences over the same pages
    as there are CTAs, so that a CTA works through all of the keys."""
    n = 400000
    cache, table = filled([n], T, 256, 1, D, seed=1)
    g = torch.Generator(device=DEV).manual_seed(D)
    k = torch.zeros((1, n + T, 1, D), device=DEV)
    k[..., 0] = x
    k[:, 0, :, 0] = 20.0
    P.append(cache, k.bfloat16(), (1 + 0.5 * torch.rand(k.shape, device=DEV, generator=g)).bfloat16(), table, [0])
    q = torch.zeros((1, T, H, D), device=DEV, dtype=torch.float16)
    q[..., 0] = 1
    o, lse = compare(q, cache, table, [n], sm_scale=1.0, lost=2.0 ** -32)
    want, want_lse, mean, S, top = P.attention(q, cache, table, [n], sm_scale=1.0)
    got, got_lse = rdna4_sage.attention_paged_kv(q.expand(B, -1, -1, -1), handle(cache), table.expand(B, -1), ints([n] * B),
                                                 None, None, "NHD", 1.0, True)
    # The tensor cores take four keys at a time and cut the sum towards zero at the accumulator's last place (seen with +1,
    # small terms, -1: four terms of 0.9985 last places leave 3, those of 0.5 leave 1): less than 2^-23 of it each time, so
    # 2^-25 for a key.  With few rows four warps share the keys.  The sum of the weights is rounded, by 2^-24 for 16 keys.
    keys = n / 4 if T * H <= (16 if D == 256 else 32) else n
    weight = 2 * ((D + 8) * 2.0 ** -24 * S.max() + 2.0 ** -22 * want_lse.max() + 2.0 ** -20) + (keys / 16 + 16) * 2.0 ** -24
    tol = 2.0 ** -11 * want + mean * (2.0 ** -11 + weight + keys * 2.0 ** -25) + (n * 2.0 ** -32 * 448 * top)[..., None]
    assert bool(((got.double() - want).abs() <= tol).all()), float(((got.double() - want).abs() / tol).max())
    assert bool(((got_lse.double() - want_lse).abs() <= weight + 2.0 ** -23 * want_lse).all())


@pytest.mark.parametrize("D,T,H", SHAPES)
@pytest.mark.parametrize("big", [3e38, 2.0 ** 127, 1.2e38])
def test_queries_of_the_largest_size(D, T, H, big):
    # One channel of each query near the end of bf16's range and small codes of K under it, the others a thousandth of that:
    # scores of a few units with the smallest sm_scale that fp32 holds well.
    lens = [300, 41]
    cache, table = filled(lens, T, 32, 2, D, seed=D)
    g = torch.Generator(device=DEV).manual_seed(T)
    cache["k8"][..., 0] = torch.randint(-2, 3, cache["k8"].shape[:3], device=DEV, generator=g).to(torch.int8)
    cache["ks"].copy_(torch.rand(cache["ks"].shape, device=DEV, generator=g) + 0.5)
    q = queries(2, T, H, D, size=1e35)
    q[..., 0] = torch.where(q[..., 0] > 0, big, -big)
    o, lse = compare(q, cache, table, lens, sm_scale=2.0 ** -125)
    assert float(lse.std()) > 0.5                        # the scores are no zeros


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scales_are_the_quotients_rounded_once(dtype):
    """Every finite largest value of a row that the type has.  a / 127 and a / 448, rounded to fp32: the reference divides in
    64 bits and rounds again, which is the same, since a quotient with a 11-bit numerator and a 7-bit odd divisor lies on a
    border between two floats or at least 2^-32 of itself away from it."""
    x = torch.arange(2 ** 15 - 1, dtype=torch.int16, device=DEV).view(dtype)
    x = x[torch.isfinite(x)]
    k = torch.zeros((1, x.numel(), 1, 64), device=DEV, dtype=dtype)
    k[0, :, 0, 3] = x
    page = 256
    table = torch.arange((x.numel() + page - 1) // page, dtype=torch.int32, device=DEV)[None]
    got, want = (P.new_cache(table.numel(), page, 1, 64, DEV) for _ in range(2))
    P.append(want, k, -k, table, [0])
    rdna4_sage.paged_kv_append(handle(got), k, -k, table, ints([0]), tensor_layout="NHD")
    for name in ("ks", "vs", "k8"):
        assert torch.equal(got[name], want[name]), name
    assert torch.equal(got["v8"].view(torch.uint8), want["v8"].view(torch.uint8))


@pytest.mark.parametrize("D,T,H", SHAPES)
@pytest.mark.parametrize("power", [8, 17, 18, 19, 21, 26, 40, 80])
def test_scores_far_beyond_the_fraction_of_fp32(D, T, H, power):
    """Scores 2^power times a whole number up to 100, exact in fp32, in one channel: each row's largest belongs to one key, by
    2^power or more, and the result is that key's V row.  One row of V is 2^40 times smaller than the others, so that the
    references of scores and of weights lie apart."""
    lens = [700, 45]
    cache, table = filled(lens, T, 32, 2, D, seed=T)
    cache["ks"].fill_(1.0)
    cache["k8"].zero_()
    g = torch.Generator(device=DEV).manual_seed(power)
    for b in range(2):
        at = torch.arange(lens[b] + T, device=DEV)
        p, r = P.place(cache, table, b, at)
        for head in range(2):
            code = torch.randint(-90, 91, (lens[b] + T,), device=DEV, generator=g)
            order = torch.randperm(lens[b], device=DEV, generator=g)
            code[order[0]], code[order[1]] = 100, -100
            cache["k8"][p, head, r, 0] = code.to(torch.int8)
        p, r = P.place(cache, table, b, order[2:3])
        cache["vs"][p, :, r] *= 2.0 ** -40
    q = torch.zeros((2, T, H, D), device=DEV, dtype=torch.bfloat16)
    q[..., 0] = 2.0 ** power * torch.where(torch.rand((2, T, H), device=DEV, generator=g) < 0.5, -1.0, 1.0)
    o, lse = rdna4_sage.attention_paged_kv(q, handle(cache), table, ints(lens), None, None, "NHD", 1.0, True)
    want, want_lse, *_ = P.attention(q, cache, table, lens, sm_scale=1.0)
    # the other keys' weights are below exp(-2^8) each: nothing.  e4m3 times a scale, weight times scale in fp16, one rounding
    assert bool(((o.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -20) * want.abs()).all())
    assert bool(((lse.double() - want_lse).abs() <= 2.0 ** -22 * want_lse.abs()).all())
