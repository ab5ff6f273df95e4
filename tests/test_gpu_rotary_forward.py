"""Forward-mode derivatives of rotary positions on the GPU (the logic itself: test_paged_derivatives_cpu.py)."""
import pytest
import torch
import torch.autograd.forward_ad as fw

import rdna4_sage
from rdna4_sage import Unsupported
from test_gpu_paged_kv import filled, handle, ints, queries
from test_gpu_rotary import CASES, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("c", CASES[:5])
def test_tangents(c):
    q, k, pos, rope, layout, _ = make(c)
    tq, tk = torch.randn_like(q), torch.randn_like(k)
    plain, want = (rdna4_sage.rotary(*x, pos, rope, layout) for x in ((q, k), (tq, tk)))
    back = rdna4_sage.rotary(tq, None, -pos, rope, layout)
    with fw.dual_level():
        out = rdna4_sage.rotary(fw.make_dual(q, tq), fw.make_dual(k, tk), pos, rope, layout)
        for y, p, w in zip(out, plain, want):
            primal, tangent = fw.unpack_dual(y)
            assert torch.equal(primal, p) and torch.equal(tangent, w)
        x = q.clone().requires_grad_()
        g, = torch.autograd.grad(rdna4_sage.rotary(x, None, pos, rope, layout), x, fw.make_dual(tq, tq))
        primal, tangent = fw.unpack_dual(g)
        assert torch.equal(primal, back) and torch.equal(tangent, back)


def test_a_model_in_forward_mode():
    # elementwise operations around the op: the tangent of sum(rotary(w x)^2) against that of the gradient
    q, _, pos, rope, layout, _ = make(CASES[4])
    w, t = torch.randn_like(q), torch.randn_like(q)

    def loss(w):
        return (rdna4_sage.rotary(w * q, None, pos, rope, layout).float() ** 2).sum()
    with fw.dual_level():
        tangent = fw.unpack_dual(loss(fw.make_dual(w, t))).tangent
    x = w.clone().requires_grad_()
    g, = torch.autograd.grad(loss(x), x)
    # five 16-bit roundings on either side (of w q, its turn, the gradient's, their tangents and products), 2^-9 each, of sums
    # whose terms have up to the size of |g| |t|
    assert abs(float(tangent) - float((g.double() * t.double()).sum())) <= 10 * 2.0 ** -9 * float((g.double() * t.double()).abs().sum())


def test_the_cache_refuses_tangents():
    cache, table = filled([10], 2, 16, 2, 64)
    q = queries(1, 2, 4, 64)
    with fw.dual_level():
        with pytest.raises(Unsupported, match="derivative"):
            rdna4_sage.attention_paged_kv(fw.make_dual(q, q), handle(cache), table, ints([10]), tensor_layout="NHD")
        rdna4_sage.attention_paged_kv(q, handle(cache), table, ints([10]), tensor_layout="NHD")
