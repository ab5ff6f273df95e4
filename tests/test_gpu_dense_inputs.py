"""Dense calls on tensors that are contiguous but not aligned, and captured behind an eager call whose status is under way."""
import pytest
import torch

import rdna4_sage

pytestmark = pytest.mark.gpu


def qkv(shape, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(shape, device="cuda", generator=g).to(dtype) for _ in range(3)]


def shifted(x, by):
    """The same numbers `by` elements behind an aligned address, contiguous."""
    y = torch.empty(x.numel() + by, device=x.device, dtype=x.dtype)[by:].view(x.shape).copy_(x)
    assert y.is_contiguous() and y.data_ptr() % 16 == 2 * by % 16
    return y


@pytest.mark.parametrize("layout,shape", [("HND", (1, 4, 300, 64)), ("NHD", (2, 130, 3, 128)), ("HND", (1, 1, 257, 96))])
@pytest.mark.parametrize("by", [1, 4])
def test_contiguous_tensors_off_alignment(layout, shape, by):
    q, k, v = qkv(shape)
    want = rdna4_sage.attention(q, k, v, layout)
    kv = rdna4_sage.quantize_kv(k, v, layout)
    want_kv = rdna4_sage.attention_quantized_kv(q, kv, layout)
    a, b, c = (shifted(x, by) for x in (q, k, v))
    for x, y, z in ((a, k, v), (q, b, v), (q, k, c), (a, b, c)):
        assert torch.equal(rdna4_sage.attention(x, y, z, layout), want)
    assert torch.equal(rdna4_sage.attention_quantized_kv(a, rdna4_sage.quantize_kv(b, c, layout), layout), want_kv)


def test_axes_of_one_with_odd_strides():
    q, k, v = qkv((1, 2, 200, 64))
    want = rdna4_sage.attention(q, k, v, "HND")
    odd = [x.as_strided(x.shape, (7, *x.stride()[1:])) for x in (q, k, v)]
    assert torch.equal(rdna4_sage.attention(*odd, "HND"), want)


def test_captured_behind_an_eager_call():
    q, k, v = qkv((1, 8, 4096, 128))
    x = torch.zeros_like(q)
    want = rdna4_sage.attention(q, k, v, "HND")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rdna4_sage.attention(x, k, v, "HND")
        y = rdna4_sage.attention(x, k, v, "HND")
    x.copy_(q)
    for _ in range(2):
        rdna4_sage.attention(q, k, v, "HND")
        graph.replay()
    assert torch.equal(y, want)
