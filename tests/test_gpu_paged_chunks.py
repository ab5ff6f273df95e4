"""Chunks of a prompt over a cached context (hundreds of new tokens: many row tiles and many key tiles of the step's own), and a
step under torch.compile."""
import pytest
import torch

import rdna4_sage
from test_gpu_paged_kv import DEV, check_attention, filled, handle, ints, queries, tables, trees

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (96, torch.bfloat16), (128, torch.bfloat16), (256, torch.float16)])
@pytest.mark.parametrize("T,counts", [(1100, None), (515, [515, 257, 0])])
def test_chunk_of_a_prompt(D, dtype, T, counts):
    lens = [0, 700, 61]
    cache, table = filled(lens, T, 64, 2, D, seed=D)
    check_attention(queries(3, T, 4, D, dtype), cache, table, lens, None, counts)


def test_chunk_with_any_mask():
    # a mask of random bytes: rows that see later tokens, and one that sees nothing of the step
    T, lens = 400, [0, 130]
    cache, table = filled(lens, T, 32, 1, 128, seed=7)
    g = torch.Generator(device=DEV).manual_seed(3)
    mask = torch.rand((2, T, T), device=DEV, generator=g) < 0.3
    mask[:, 77] = False
    check_attention(queries(2, T, 2, 128), cache, table, lens, mask)


def test_a_chunk_is_its_tokens_one_by_one():
    T, lens = 130, [50]
    cache, table = filled(lens, T, 16, 2, 128, seed=2)
    q = queries(1, T, 8, 128)
    whole = rdna4_sage.attention_paged_kv(q, handle(cache), table, ints(lens), tensor_layout="NHD")
    for i in (0, 1, 63, 129):
        one = rdna4_sage.attention_paged_kv(q[:, i:i + 1], handle(cache), table, ints([50 + i]), tensor_layout="NHD")
        # both are roundings to bf16 of numbers 2^-10 of the row's values apart at the most: weights in fp16, sums in another order
        tol = 2.0 ** -8 * whole[:, i:i + 1].abs().float() + 2.0 ** -10 * 4
        assert bool(((one.float() - whole[:, i:i + 1].float()).abs() <= tol).all()), i


def test_compiled_step():
    B, T, H, Hkv, D, page = 2, 5, 4, 2, 64, 16
    table, pages = tables([0] * B, 100, page)
    rope = rdna4_sage.Rotary(D)
    q, k, v = (queries(B, T, h, D, seed=h) for h in (H, Hkv, Hkv))
    mask, lens = trees(B, T), ints([9, 30])
    depth = mask.sum(-1) - 1

    def step(kv, q, k, v):
        q, k = rdna4_sage.rotary(q, k, lens[:, None] + depth, rope, "NHD")
        rdna4_sage.paged_kv_append(kv, k, v, table, lens, tensor_layout="NHD")
        return rdna4_sage.attention_paged_kv(q, kv, table, lens, mask, tensor_layout="NHD") * 2
    caches = [rdna4_sage.PagedKV.empty(pages, page, Hkv, D) for _ in range(2)]
    for kv in caches:
        rdna4_sage.paged_kv_append(kv, *(queries(B, 30, Hkv, D, seed=s) for s in (8, 9)), table, ints([0, 0]), lens, "NHD")
    want = step(caches[0], q, k, v)
    compiled = torch.compile(step)
    for _ in range(2):
        assert torch.equal(compiled(caches[1], q, k, v), want)
    for a, b in zip((caches[0].k8, caches[0].ks, caches[0].v8), (caches[1].k8, caches[1].ks, caches[1].v8)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    x = q.clone().requires_grad_()
    turn = torch.compile(lambda x: (rdna4_sage.rotary(x, None, lens[:, None] + depth, rope, "NHD") * 3).float().sum())
    turn(x).backward()
    g, = torch.autograd.grad(rdna4_sage.rotary(x, None, lens[:, None] + depth, rope, "NHD"), x, torch.full_like(x, 3.0))
    assert torch.equal(x.grad, g)
