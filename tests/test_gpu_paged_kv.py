"""The paged K/V cache and attention over it on the GPU, against their definitions in 64 bits (paged_reference.py).

Codes and scales are compared exactly (scales to one rounding): the roundings have no undecided cases for 16-bit rows.
Attention tolerances, per output row, with A = sum p |v| / sum p:
  - the result is rounded once: half a step of its type, eps / 2 |o|;
  - a weight may be rounded to fp16 (2^-11) before the product with V, and what fp16 cannot hold of it is below
    2^-25 of the row's largest weight times scale, times 448, for each of the n keys;
  - a score is a sum of D products (and three factors) in fp32: off by (D + 8) 2^-24 of sum |q k| <= S, which is
    the relative error of a weight, once in the sum over V and once in the sum of the weights; exp2, its argument
    (|s| 2^-23) and the sums over n keys add 2^-20 + (n / 16 + 16) 2^-24 A."""
import math

import pytest
import torch

import paged_reference as P
import rdna4_sage
from rdna4_sage import _attention

pytestmark = pytest.mark.gpu
DEV = "cuda"


def tables(lens, new, page, spare=2, seed=0, extra=0):
    need = [max(0, (n + new + page - 1) // page) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).int()
    table = torch.full((len(lens), max(1, max(need)) + extra), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table.to(DEV), sum(need) + spare


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def handle(cache):
    return rdna4_sage.PagedKV(**cache)


def same_cache(a, b):
    for name in ("k8", "v8"):
        torch.testing.assert_close(a[name].view(torch.uint8), b[name].view(torch.uint8), rtol=0, atol=0)
    for name in ("ks", "vs"):
        torch.testing.assert_close(a[name], b[name], rtol=2.0 ** -22, atol=0, equal_nan=True)


def filled(lens, new, page, Hkv, D, seed=0, fill=0xff, spread=False):
    """A cache with random rows at every position of each sequence, and garbage elsewhere (NaN codes and scales)."""
    table, pages = tables(lens, new, page, seed=seed)
    cache = P.new_cache(pages, page, Hkv, D, DEV, fill)
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    for b, n in enumerate(lens):
        if n + new == 0:
            continue
        k, v = (torch.randn((1, n + new, Hkv, D), device=DEV, generator=g) for _ in range(2))
        if spread:   # rows of very different size
            v = v * torch.exp(6 * torch.randn((1, n + new, Hkv, 1), device=DEV, generator=g))
        P.append(cache, k.bfloat16(), v.bfloat16(), table[b:b + 1], [0])
    return cache, table


# ------------------------------------------------------------------------------------------------ append, read, keep
def special_rows(x):
    """Rows that test the rules: zeros, ties, one value, tiny, NaN, infinities (as many as there are rows)."""
    flat = x.view(-1, x.shape[-1])
    t = torch.arange(x.shape[-1], device=DEV) % 255 - 127
    rows = [torch.zeros_like(flat[0]), t.to(x.dtype) * 0.5, torch.where(t == 0, 2.0, 1.0).to(x.dtype), flat[0] * 1e-3]
    if x.dtype == torch.bfloat16:
        rows += [flat[0] * 1e-33, (t.to(x.dtype) * 1e30)]
    else:
        rows += [(t.to(x.dtype) * 6e-8), t.to(x.dtype) * 500]
    nan, inf = flat[0].clone(), flat[0].clone()
    nan[-1], inf[0] = math.nan, -math.inf
    for i, r in enumerate(rows + [nan, inf]):
        if i < flat.shape[0]:
            flat[i] = r
    return x


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype,layout,page,S,Hkv,lens,counts", [
    (torch.bfloat16, "NHD", 16, 1, 1, [0], None),
    (torch.float16, "HND", 16, 5, 3, [0, 13, 31], None),
    (torch.bfloat16, "HND", 64, 70, 2, [1, 63, 200], [70, 0, 33]),
    (torch.float16, "NHD", 256, 33, 4, [250, 5], [1, 33]),
    (torch.bfloat16, "NHD", 32, 257, 5, [16, 0], [257, 31])])
def test_append(D, dtype, layout, page, S, Hkv, lens, counts):
    g = torch.Generator(device=DEV).manual_seed(D + S)
    k, v = (special_rows(torch.randn((len(lens), S, Hkv, D), device=DEV, generator=g).to(dtype)) for _ in range(2))
    table, pages = tables(lens, S, page)
    want, got = (P.new_cache(pages, page, Hkv, D, DEV, 0x35) for _ in range(2))
    P.append(want, k, v, table, lens, counts)
    if layout == "HND":
        k, v = k.transpose(1, 2), v.transpose(1, 2).contiguous()
    rdna4_sage.paged_kv_append(handle(got), k, v, table, ints(lens), None if counts is None else ints(counts), layout)
    _attention.check_status(torch.device("cuda", 0))
    same_cache(got, want)


def test_every_rounding_of_a_row():
    # all pairs (value, largest value) of 8-bit fractions: codes from the rational numbers themselves, in integers
    D, a = 128, torch.arange(128, 256)
    x = torch.zeros((1, 128 * 10, 1, D), device=DEV)
    for shift in range(10):
        x[0, shift * 128:(shift + 1) * 128, 0, :] = torch.arange(128, 256, device=DEV)[None] * 2.0 ** -shift
    x[..., 0] = a.repeat(10).to(DEV).float()[None, :, None]
    for shift in range(10):                                        # no value above the row's first
        part = x[0, shift * 128:(shift + 1) * 128, 0]
        part[:] = torch.minimum(part, part[:, :1])
    table, pages = tables([0], x.shape[1], 64)
    want, got = (P.new_cache(pages, 64, 1, D, DEV) for _ in range(2))
    for dtype in (torch.bfloat16, torch.float16):
        P.append(want, x.to(dtype), -x.to(dtype), table, [0])
        rdna4_sage.paged_kv_append(handle(got), x.to(dtype), -x.to(dtype), table, ints([0]), tensor_layout="NHD")
        same_cache(got, want)
        k, _ = P.rows(got, table, 0, x.shape[1])
        p, r = P.place(got, table, 0, range(x.shape[1]))
        xi = (x[0, :, 0].double() * 2 ** 9).long()
        top = xi[:, :1]
        tie_away = (2 * 127 * xi + top) // (2 * top)               # floor(127 x / a + 1/2), x >= 0
        assert torch.equal(got["k8"][p, 0, r].long(), tie_away)


@pytest.mark.parametrize("D,page,dtype,layout,lens,n", [
    (64, 16, torch.bfloat16, "HND", [0, 1, 40], 40), (96, 32, torch.float16, "NHD", [77, 5], 80),
    (128, 64, torch.bfloat16, "NHD", [130, 64, 63, 0], 130), (256, 128, torch.float16, "HND", [300], 257)])
def test_read(D, page, dtype, layout, lens, n):
    cache, table = filled(lens, 0, page, 3, D)
    k, v = rdna4_sage.paged_kv_read(handle(cache), table, ints(lens), n, dtype, layout)
    assert k.is_contiguous() and k.dtype == dtype and k.shape == v.shape
    k, v = (x if layout == "NHD" else x.transpose(1, 2) for x in (k, v))
    for b, held in enumerate(lens):
        held = min(held, n)
        want = P.rows(cache, table, b, held) if held else (k[b, :0].double(),) * 2
        for got, w in zip((k[b], v[b]), want):
            # code * scale is rounded to fp32 (2^-24) and then to 16 bits (half a step, fp16 not below 2^-25)
            tol = (torch.finfo(dtype).eps / 2 + 2.0 ** -23) * w.abs() + 2.0 ** -25
            assert bool(((got[:held].double() - w).abs() <= tol).all())
            assert not bool(got[held:].any())


@pytest.mark.parametrize("D,page,Hkv", [(64, 16, 2), (96, 32, 3), (128, 16, 8), (256, 64, 1)])
def test_keep(D, page, Hkv):
    T, lens = 50, [0, 15, 100, 7]
    cache, table = filled(lens, T, page, Hkv, D)
    keep = torch.stack([torch.randperm(T, generator=torch.Generator().manual_seed(b))[:40].sort().values for b in range(4)])
    keep[3] = torch.arange(40)                                     # stays where it is
    counts = [40, 1, 0, 33]
    want = {n: x.clone() for n, x in cache.items()}
    for b, n in enumerate(counts):
        for i in range(n):
            (p0, r0), (p1, r1) = P.place(cache, table, b, [lens[b] + int(keep[b, i])]), P.place(cache, table, b, [lens[b] + i])
            for name in cache:
                w, c = (x.view(torch.uint8) if name == "v8" else x for x in (want[name], cache[name]))
                w[p1, :, r1] = c[p0, :, r0]
    rdna4_sage.paged_kv_keep(handle(cache), table, ints(lens), keep.int().to(DEV), ints(counts))
    same_cache(cache, want)
    wide = torch.full((4, 60), -5, dtype=torch.int32, device=DEV)  # strided rows, no counts
    wide[:, :3] = ints([[0, 2, 4]] * 4)
    for b in range(4):
        for i, j in enumerate((0, 2, 4)):
            (p0, r0), (p1, r1) = P.place(want, table, b, [lens[b] + j]), P.place(want, table, b, [lens[b] + i])
            for name in want:
                w = want[name].view(torch.uint8) if name == "v8" else want[name]
                w[p1, :, r1] = w[p0, :, r0]
    rdna4_sage.paged_kv_keep(handle(cache), table, ints(lens), wide[:, :3])
    same_cache(cache, want)


# ------------------------------------------------------------------------------------------------ attention
def check_attention(q, cache, table, lens, mask=None, counts=None, layout="NHD", sm_scale=None):
    x = q if layout == "NHD" else q.transpose(1, 2).contiguous()
    o, lse = rdna4_sage.attention_paged_kv(x, handle(cache), table, ints(lens), mask,
                                           None if counts is None else ints(counts), layout, sm_scale, True)
    _attention.check_status(torch.device("cuda", 0))
    assert o.shape == x.shape and o.dtype == q.dtype
    got = (o if layout == "NHD" else o.transpose(1, 2)).double()
    want, want_lse, mean, S, top = P.attention(q, cache, table, lens, mask, counts, sm_scale)
    n, D = max(lens) + q.shape[1], q.shape[-1]
    weight = 2 * ((D + 8) * 2.0 ** -24 * S + 2.0 ** -22 * want_lse.transpose(1, 2).abs().nan_to_num(0, 0, 0) +
                  2.0 ** -20 + (n / 16 + 16) * 2.0 ** -24)
    tol = torch.finfo(q.dtype).eps / 2 * want.abs() + mean * (2.0 ** -11 + weight[..., None]) + \
        (n * 2.0 ** -25 * 448 * top)[..., None] + 2.0 ** -25
    off = (got - want).abs()
    # the computed value lies within tol of want, and what reaches the type's largest value and half a step more
    # (its step there is max eps / (2 - eps)) rounds to infinity
    info = torch.finfo(q.dtype)
    over = want.abs() + tol >= info.max * (1 + info.eps / 2 / (2 - info.eps))
    off = torch.where(over & (got == torch.copysign(torch.full_like(want, math.inf), want)), 0.0, off)
    assert bool((off <= tol).all()), (float((off / tol).max()), float(off.max()))
    empty = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    ltol = (weight.transpose(1, 2) + 2.0 ** -23 * want_lse.abs())[~empty]
    assert bool(((lse.double() - want_lse).abs()[~empty] <= ltol).all())
    assert torch.equal(rdna4_sage.attention_paged_kv(x, handle(cache), table, ints(lens), mask,
                                                     None if counts is None else ints(counts), layout, sm_scale), o)
    return got, lse


def queries(B, T, H, D, dtype=torch.bfloat16, seed=3, size=1.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (size * torch.randn((B, T, H, D), device=DEV, generator=g)).to(dtype)


def trees(B, T, seed=5):
    g = torch.Generator().manual_seed(seed)
    mask = torch.zeros((B, T, T), dtype=torch.bool)
    for b in range(B):
        for i in range(T):
            up = int(torch.randint(-1, i, (1,), generator=g)) if i else -1
            if up >= 0:
                mask[b, i] = mask[b, up]
            mask[b, i, i] = True
    return mask.to(DEV)


ATT = [  # T, H, Hkv, page, lens, counts, tree
    (1, 1, 1, 16, [0], None, False),
    (1, 8, 8, 16, [0, 1, 15, 16, 17, 200], None, False),
    (1, 32, 8, 64, [63, 64, 65, 1000], None, False),
    (1, 40, 2, 32, [127, 3], None, False),
    (5, 6, 2, 16, [0, 11, 333], [5, 0, 3], False),
    (13, 4, 4, 32, [19, 700], None, True),
    (33, 16, 2, 128, [0, 100, 129], [33, 17, 1], True),
    (64, 8, 1, 64, [64, 1, 500], None, True),
    (100, 10, 5, 256, [77, 256], None, True),
    (150, 3, 1, 16, [40], None, False),
]


@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (96, torch.float16), (128, torch.bfloat16),
                                     (128, torch.float16), (256, torch.bfloat16)])
@pytest.mark.parametrize("c", ATT)
def test_attention(c, D, dtype):
    T, H, Hkv, page, lens, counts, tree = c
    cache, table = filled(lens, T, page, Hkv, D, seed=T)
    q = queries(len(lens), T, H, D, dtype)
    check_attention(q, cache, table, lens, trees(len(lens), T) if tree else None, counts,
                    layout="HND" if T % 2 else "NHD", sm_scale=None if T > 1 else 0.07)


def test_masks_that_leave_nothing_and_shared_masks():
    T, lens = 20, [0, 5]
    cache, table = filled(lens, T, 16, 2, 128)
    q = queries(2, T, 8, 128)
    mask = trees(1, T)[0]
    mask[3] = False
    mask[17] = False
    a, lse = check_attention(q, cache, table, lens, mask)                        # [T, T], shared
    assert not bool(a[0, [3, 17]].any()) and bool((lse[0, :, [3, 17]] == -math.inf).all())
    assert bool(a[1, 3].any())                                                   # it has a context
    for m in (mask[None], mask.expand(2, T, T), torch.stack((mask, mask)), mask.t().contiguous().t()):
        b, _ = check_attention(q, cache, table, lens, m)
        assert torch.equal(a, b)
    check_attention(q, cache, table, lens, torch.zeros_like(mask))
    check_attention(q, cache, table, lens, torch.ones_like(mask))                # drafts may see what comes after them


@pytest.mark.parametrize("H", [2, 4, 16])                               # 24, 48 and 192 rows of a kv head
def test_masked_rows_may_hold_anything(H):
    # NaN and infinities at drafts that nothing sees, and behind the last token, stay where they are
    T, lens, page = 24, [37, 0], 16
    cache, table = filled(lens, T, page, 2, 64)
    mask = trees(2, T)
    dead = 9
    mask[:, :, dead] = False
    q = queries(2, T, H, 64)
    a, _ = check_attention(q, cache, table, lens, mask)
    for junk in (math.nan, math.inf, -math.inf, -1e-40, 1e-40, -3.0, 0.0, 3e38):
        for b in range(2):
            p, r = P.place(cache, table, b, [lens[b] + dead])
            for name in ("ks", "vs"):
                cache[name][p, :, r] = junk
            cache["v8"].view(torch.uint8)[p, :, r] = 0x7f
        # behind the last token too, in the rest of the page
        p, r = P.place(cache, table, 1, range(T, 2 * page))
        cache["vs"][p, :, r] = junk
        b_, _ = check_attention(q, cache, table, lens, mask)
        assert torch.equal(a, b_), junk
    # a visible NaN reaches the rows that see it, and only those
    p, r = P.place(cache, table, 0, [lens[0] + 2])
    cache["ks"][p, :, r] = math.nan
    o = rdna4_sage.attention_paged_kv(q, handle(cache), table, ints(lens), mask, None, "NHD")
    hit = mask[0, :, 2]
    assert bool(o[0, hit].isnan().all()) and torch.equal(o[0, ~hit].double(), a[0, ~hit]) and torch.equal(o[1].double(), a[1])


def test_rows_of_very_different_size():
    # weights times scales over many orders of magnitude, all-zero V rows among them
    for D, T in ((128, 1), (64, 17)):
        lens = [300, 2000]
        cache, table = filled(lens, T, 32, 2, D, seed=8, spread=True)
        p, r = P.place(cache, table, 1, range(0, 2000, 3))
        cache["vs"][p, :, r] = 0.0
        cache["v8"].view(torch.uint8)[p, :, r] = 0
        for size in (0.02, 1.0, 6.0):
            check_attention(queries(2, T, 8, D, torch.float16, size=size), cache, table, lens)
        check_attention(queries(2, T, 8, D, size=1e-20), cache, table, lens)
        check_attention(queries(2, T, 8, D, size=1e20), cache, table, lens, sm_scale=2e-21)
    cache["vs"].zero_()
    cache["v8"].view(torch.uint8).zero_()
    o, _ = check_attention(queries(2, T, 8, D), cache, table, lens)
    assert not bool(o.any())


def test_long_context_split_over_the_gpu():
    for B, H, Hkv, D, page, n in ((1, 8, 1, 128, 64, 70001), (3, 4, 4, 64, 16, 9999), (1, 16, 2, 256, 128, 30011)):
        lens = [n] + [n // 3 + 7] * (B - 1)
        cache, table = filled(lens, 1, page, Hkv, D, seed=n)
        check_attention(queries(B, 1, H, D, size=0.5), cache, table, lens)


def test_many_sequences():
    lens = [(37 * i) % 211 for i in range(300)]
    cache, table = filled(lens, 2, 16, 2, 64)
    check_attention(queries(300, 2, 4, 64), cache, table, lens)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_row_tiles_without_live_rows(D):
    # 800 query rows of a kv head in several row tiles, some of which hold no token of a padded batch's short sequences
    T, lens, counts = 200, [70, 1, 500, 0], [200, 3, 0, 64]
    cache, table = filled(lens, T, 32, 2, D, seed=4)
    q = queries(4, T, 8, D)
    a, lse = check_attention(q, cache, table, lens, None, counts)
    for b, n in enumerate(counts):
        assert not bool(a[b, n:].any()) and bool((lse[b, :, n:] == -math.inf).all())
    check_attention(q, cache, table, lens, trees(4, T), counts, layout="HND")


@pytest.mark.parametrize("T", [1, 12])
def test_more_sequences_than_threads(T):
    lens = [(53 * i) % 97 for i in range(700)]
    cache, table = filled(lens, T, 16, 1, 64)
    check_attention(queries(700, T, 4, 64), cache, table, lens, trees(1, T)[0] if T > 1 else None)


def test_offsets_past_32_bits():
    # a pool of 2^31 + codes a tensor: the sequences sit in its last and its first pages
    page, Hkv, D = 256, 8, 256
    pages = 2 ** 31 // (page * Hkv * D) + 3
    cache = dict(k8=torch.zeros((pages, Hkv, page, D), dtype=torch.int8, device=DEV),
                 v8=torch.zeros((pages, Hkv, page, D), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn),
                 ks=torch.zeros((pages, Hkv, page), device=DEV), vs=torch.zeros((pages, Hkv, page), device=DEV))
    table, lens, T = ints([[pages - 1, 0], [pages - 2, pages - 3]]), [200, 300], 40
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randn((2, 340, Hkv, D), device=DEV, generator=g).bfloat16() for _ in range(2))
    counts = [240, 340]
    rdna4_sage.paged_kv_append(handle(cache), k, v, table, ints([0, 0]), ints(counts), "NHD")
    want = {n: cache[n][[0, pages - 3, pages - 2, pages - 1]].clone() for n in ("k8", "ks", "vs")}
    small = P.new_cache(4, page, Hkv, D, DEV)
    P.append(small, k, v, ints([[3, 0], [2, 1]]), [0, 0], counts)
    for n, x in want.items():
        torch.testing.assert_close(x, small[n], rtol=2.0 ** -22, atol=0)
    check_attention(queries(2, T, 8, D), cache, table, lens)
    rk, _ = rdna4_sage.paged_kv_read(handle(cache), table, ints(counts), 340, tensor_layout="NHD")
    sk, _ = rdna4_sage.paged_kv_read(handle(small), ints([[3, 0], [2, 1]]), ints(counts), 340, tensor_layout="NHD")
    assert torch.equal(rk, sk)
    rdna4_sage.paged_kv_keep(handle(cache), table, ints(lens), ints([[5, 9], [3, 30]]))
    p, r = P.place(cache, table, 0, [200, 205, 201, 209])
    # rows 205 and 209 are where 200 and 201 are now
    assert torch.equal(cache["k8"][p[0], :, r[0]], cache["k8"][p[1], :, r[1]])
    assert torch.equal(cache["k8"][p[2], :, r[2]], cache["k8"][p[3], :, r[3]])


# ------------------------------------------------------------------------------------------------ a run of steps
def test_steps_of_a_drafted_run_and_the_same_as_a_graph():
    """Prompt, then steps of rotary + append + tree attention + keep, eager and as one captured graph replayed with
    new inputs, against the 64-bit forms."""
    B, T, H, Hkv, D, page = 3, 9, 8, 2, 128, 16
    g = torch.Generator(device=DEV).manual_seed(11)
    start, room = [20, 3, 47], 200
    table, pages = tables([0] * B, room, page)
    rope = rdna4_sage.Rotary(D)
    ref = P.new_cache(pages, page, Hkv, D, DEV)
    cache = {n: x.clone() for n, x in ref.items()}
    kv, lens = handle(cache), ints(start)
    prompt = [torch.randn((B, max(start), Hkv, D), device=DEV, generator=g).bfloat16() for _ in range(2)]
    rdna4_sage.paged_kv_append(kv, *prompt, table, ints([0] * B), ints(start), "NHD")
    P.append(ref, *prompt, table, [0] * B, start)
    same_cache(cache, ref)
    x = {n: torch.zeros((B, T, h, D), device=DEV, dtype=torch.bfloat16) for n, h in (("q", H), ("k", Hkv), ("v", Hkv))}
    depth, mask = torch.zeros((B, T), dtype=torch.int32, device=DEV), torch.zeros((B, T, T), dtype=torch.bool, device=DEV)
    accepted, counts = torch.zeros((B, 4), dtype=torch.int32, device=DEV), torch.zeros(B, dtype=torch.int32, device=DEV)

    def step():
        q, k = rdna4_sage.rotary(x["q"], x["k"], lens[:, None] + depth, rope, "NHD")
        rdna4_sage.paged_kv_append(kv, k, x["v"], table, lens, tensor_layout="NHD")
        o = rdna4_sage.attention_paged_kv(q, kv, table, lens, mask, tensor_layout="NHD")
        rdna4_sage.paged_kv_keep(kv, table, lens, accepted, counts)
        lens.add_(counts)
        return q, k, o

    graph, out = None, None
    for n in range(6):
        for t in x.values():
            t.copy_(torch.randn(t.shape, device=DEV, generator=g))
        m = trees(B, T, seed=n)
        mask.copy_(m)
        depth.copy_(m.sum(-1) - 1)
        for b in range(B):                                          # accept the start of the path to some draft
            path = m[b, (2 * n + b) % T].nonzero()[:4, 0]
            accepted[b, :len(path)] = path.int()
            counts[b] = len(path)
        before = lens.tolist()
        if n == 3:
            keep_state = {name: t.clone() for name, t in cache.items()}, lens.clone()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step()
            assert lens.tolist() == before                          # captured, not run
            assert all(torch.equal(t.view(torch.uint8), keep_state[0][name].view(torch.uint8)) for name, t in cache.items())
        if graph is None:
            out = step()
        else:
            graph.replay()
        q, k, o = out
        want_k = P.rotary(x["k"], torch.tensor(before, device=DEV)[:, None] + depth, rope.frequencies, 1.0, D, False)
        assert bool(((k.double() - want_k).abs() <= 2.0 ** -8 * want_k.abs() + 2.0 ** -16).all())
        P.append(ref, k, x["v"], table, before)
        want, _, mean, S, _ = P.attention(q, ref, table, before, mask)
        tol = 2.0 ** -8 * want.abs() + mean * (2.0 ** -11 + 2 * (136 * 2.0 ** -24 * S[..., None] + 2.0 ** -18)) + 2.0 ** -25
        assert bool(((o.double() - want).abs() <= tol).all()), n
        for b in range(B):
            for i in range(int(counts[b])):
                (p0, r0), (p1, r1) = (P.place(ref, table, b, [before[b] + j]) for j in (int(accepted[b, i]), i))
                for name in ref:
                    w = ref[name].view(torch.uint8) if name == "v8" else ref[name]
                    w[p1, :, r1] = w[p0, :, r0]
        same_cache(cache, ref)
        assert lens.tolist() == [s + int(c) for s, c in zip(before, counts)]
    _attention.check_status(torch.device("cuda", 0))
    # the context read back goes through the dense kernels as any K and V
    n = int(lens.min())
    rk, rv = rdna4_sage.paged_kv_read(kv, table, lens, n, tensor_layout="NHD")
    dense = rdna4_sage.attention(q[:, :1].contiguous(), rk, rv, "NHD")
    assert dense.shape == (B, 1, H, D) and bool(torch.isfinite(dense).all())


def test_side_stream_and_two_calls_at_once():
    lens, T = [500, 90, 1300], 7
    cache, table = filled(lens, T, 32, 4, 128)
    q = queries(3, T, 16, 128)
    q2 = queries(3, T, 16, 128, seed=9)
    L, kv = ints(lens), handle(cache)
    want, want2 = (rdna4_sage.attention_paged_kv(x, kv, table, L, tensor_layout="NHD") for x in (q, q2))
    graphs = []
    for x in (q, q2):                                               # two graphs whose replays overlap
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            y = rdna4_sage.attention_paged_kv(x, kv, table, L, tensor_layout="NHD")
        graphs.append((gr, y))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for (gr, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want2)
    outs = []
    for x, st in zip((q, q2) * 10, streams * 10):
        with torch.cuda.stream(st):
            outs.append(rdna4_sage.attention_paged_kv(x, kv, table, L, tensor_layout="NHD"))
    torch.cuda.synchronize()
    assert all(torch.equal(o, (want, want2)[i % 2]) for i, o in enumerate(outs))


# ------------------------------------------------------------------------------------------------ bad lengths and pages
def test_bad_pages_and_lengths_are_reported_and_not_touched():
    lens, T, page = [30, 40, 10], 4, 16
    cache, table = filled(lens, T, page, 2, 64)
    kv, q, dev = handle(cache), queries(3, T, 4, 64), torch.device("cuda", 0)
    pages = cache["k8"].shape[0]
    k = queries(3, T, 2, 64)
    good = rdna4_sage.attention_paged_kv(q, kv, table, ints(lens), tensor_layout="NHD")
    rk, _ = rdna4_sage.paged_kv_read(kv, table, ints(lens), 40, tensor_layout="NHD")
    before = {n: x.clone() for n, x in cache.items()}
    capacity = table.shape[1] * page
    for what, t, n, c in [("page", (1, 1, pages), lens, None), ("page", (1, 1, -1), lens, None),
                          ("lens", None, [30, -1, 10], None), ("lens", None, [30, capacity + 100, 10], None),
                          ("counts", None, lens, [4, T + 1, 4]), ("counts", None, lens, [4, -1, 4])]:
        tb = table.clone()
        if t is not None:
            tb[t[0], t[1]] = t[2]
        cc = None if c is None else ints(c)
        o = rdna4_sage.attention_paged_kv(q, kv, tb, ints(n), None, cc, "NHD")
        with pytest.raises(RuntimeError, match="invalid argument"):
            _attention.check_status(dev)
        assert torch.equal(o[0], good[0]) and torch.equal(o[2], good[2]), (what, t, n, c)
        if c is None:
            r, _ = rdna4_sage.paged_kv_read(kv, tb, ints(n), 40, tensor_layout="NHD")
            assert torch.equal(r[0], rk[0]) and torch.equal(r[2], rk[2])
            with pytest.raises(RuntimeError, match="invalid argument"):
                _attention.check_status(dev)
    # append: only the other sequences change
    for n, c in (([30, capacity, 10], None), ([30, -T, 10], None), (lens, [0, -3, 0])):
        rdna4_sage.paged_kv_append(kv, k, k, table, ints(n), None if c is None else ints(c), "NHD")
        with pytest.raises(RuntimeError, match="invalid argument"):
            _attention.check_status(dev)
        want = {m: x.clone() for m, x in before.items()}
        if c is None:
            P.append(want, k[[0, 2]], k[[0, 2]], table[[0, 2]], [30, 10])
            before = want
        same_cache(cache, want)
    # keep: rows that do not increase leave their sequence alone
    for row in ([0, 2, 2], [1, 0, 3], [-1, 0, 1]):
        rdna4_sage.paged_kv_keep(kv, table, ints(lens), ints([[0, 1, 2], row, [0, 1, 2]]))
        with pytest.raises(RuntimeError, match="invalid argument"):
            _attention.check_status(dev)
        same_cache(cache, before)
    # without a check, the next call on the device raises
    rdna4_sage.paged_kv_keep(kv, table, ints(lens), ints([[1, 0]] * 3))
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="paged K/V"):
        rdna4_sage.paged_kv_keep(kv, table, ints(lens), ints([[0, 1]] * 3))
    rdna4_sage.paged_kv_keep(kv, table, ints(lens), ints([[0, 1]] * 3))
    _attention.check_status(dev)


def test_empty_batches():
    cache, table = filled([10], 2, 16, 2, 64)
    kv = handle(cache)
    empty = torch.zeros((0, 2, 4, 64), device=DEV, dtype=torch.bfloat16)
    none, t0 = torch.zeros(0, dtype=torch.int32, device=DEV), table[:0]
    assert rdna4_sage.attention_paged_kv(empty, kv, t0, none, tensor_layout="NHD").shape == empty.shape
    rdna4_sage.paged_kv_append(kv, empty[:, :, :2], empty[:, :, :2], t0, none, tensor_layout="NHD")
    q = torch.zeros((1, 0, 4, 64), device=DEV, dtype=torch.bfloat16)
    assert rdna4_sage.attention_paged_kv(q, kv, table, ints([10]), tensor_layout="NHD").shape == q.shape
    rdna4_sage.paged_kv_append(kv, q[:, :, :2], q[:, :, :2], table, ints([10]), tensor_layout="NHD")
    assert rdna4_sage.paged_kv_read(kv, table, ints([10]), 0)[0].shape == (1, 2, 0, 64)
    rdna4_sage.paged_kv_keep(kv, table, ints([10]), torch.zeros((1, 0), dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("T", [2, 17])                                  # 8 and 68 rows of a kv head
def test_every_page_size(D, page, T):
    lens = [page - 1, 2 * page, 5]
    cache, table = filled(lens, T, page, 2, D, seed=page + T)
    check_attention(queries(3, T, 8, D, seed=T), cache, table, lens, trees(3, T), [T, T - 1, 1])


@pytest.mark.parametrize("T", [3, 40])
@pytest.mark.parametrize("layout", ["NHD", "HND"])
def test_views_of_a_projection_bytes_of_v_and_shared_pages(T, layout):
    """q, k and v as views of one tensor, both aligned and not, and one that all heads share; V's codes as bytes; two
    sequences whose context lies in the same pages."""
    H, Hkv, D, page, lens = 8, 2, 128, 16, [32, 32]
    cache, table = filled(lens, T, page, Hkv, D, seed=T)
    table[1, :2] = table[0, :2]
    g = torch.Generator(device=DEV).manual_seed(T)
    for pad in (0, 8, 3):                                               # channels in front of q
        x = torch.randn((2, T, pad + (H + 2 * Hkv) * D), device=DEV, generator=g).bfloat16()
        q, k, v = (t.unflatten(-1, (-1, D)) for t in x[..., pad:].split([H * D, Hkv * D, Hkv * D], -1))
        k = k[:, :, :1].expand(-1, -1, Hkv, -1)
        want = {n: t.clone() for n, t in cache.items()}
        P.append(want, k, v, table, lens)
        turn = (lambda t: t.transpose(1, 2)) if layout == "HND" else (lambda t: t)
        kv = rdna4_sage.PagedKV(cache["k8"], cache["ks"], cache["v8"].view(torch.uint8), cache["vs"])
        rdna4_sage.paged_kv_append(kv, turn(k), turn(v), table, ints(lens), tensor_layout=layout)
        same_cache(cache, want)
        plain, _ = check_attention(q.contiguous(), cache, table, lens)
        got = rdna4_sage.attention_paged_kv(turn(q), kv, table, ints(lens), tensor_layout=layout)
        assert torch.equal(turn(got).double(), plain)


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("T,H", [(1, 4), (2, 8), (4, 8), (8, 16)])      # 2, 8, 16 and 64 rows of a kv head
def test_row_tiles_of_one_key_tile(D, T, H):
    """A CTA walks many row tiles that end with the key tile they begin with: the parts of one must not be overtaken by
    the next one's.  Every run gives the same bits."""
    lens = [(29 * i) % (63 - T) for i in range(400)]
    cache, table = filled(lens, T, 16, 2, D, seed=D)
    q = queries(400, T, H, D, seed=T)
    want, lse = check_attention(q, cache, table, lens)
    kv, at = handle(cache), ints(lens)
    for _ in range(30):
        o, l2 = rdna4_sage.attention_paged_kv(q, kv, table, at, tensor_layout="NHD", return_lse=True)
        assert torch.equal(o.double(), want) and torch.equal(l2, lse)
