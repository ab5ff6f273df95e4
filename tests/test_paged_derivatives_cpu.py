"""Forward-mode derivatives (dual tensors) of the step calls, without a GPU: rotary carries them, the cache refuses them."""
import pytest
import torch
import torch.autograd.forward_ad as fw

import paged_reference as P
import rdna4_sage
from rdna4_sage import Unsupported, _rotary


def turned(q, k, positions, rope, layout, backward):
    """_rotary._launch from the definition, in the inputs' type."""
    def one(x):
        if x is None:
            return None
        x = x.detach().transpose(1, 2) if layout == "HND" else x.detach()
        y = P.rotary(x, positions.expand(x.shape[0], -1), rope.frequencies, rope.magnitude, rope.rotary_dim, rope.interleaved,
                     backward).to(x.dtype)
        return y.transpose(1, 2) if layout == "HND" else y
    return one(q), one(k)


@pytest.fixture
def on_cpu(monkeypatch):
    monkeypatch.setattr(_rotary, "_launch", turned)
    monkeypatch.setattr(_rotary, "step", lambda *tensors: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return rdna4_sage.Rotary(64, device="cpu"), torch.arange(5)


def tensors(seed, n):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn((2, 5, h, 64), generator=g).bfloat16() for h in [4, 2, 4, 2][:n]]


@pytest.mark.parametrize("dual", [(True, False), (False, True), (True, True)])
@pytest.mark.parametrize("layout", ["NHD", "HND"])
def test_tangent_is_the_turned_tangent(on_cpu, dual, layout):
    rope, at = on_cpu
    q, k, tq, tk = (x.transpose(1, 2) if layout == "HND" else x for x in tensors(1, 4))
    plain = rdna4_sage.rotary(q, k, at, rope, layout)
    want = rdna4_sage.rotary(tq, tk, at, rope, layout)
    with fw.dual_level():
        out = rdna4_sage.rotary(fw.make_dual(q, tq) if dual[0] else q, fw.make_dual(k, tk) if dual[1] else k, at, rope, layout)
        for y, p, w, d in zip(out, plain, want, dual):
            primal, tangent = fw.unpack_dual(y)
            assert torch.equal(primal, p)
            assert (tangent is not None) == d and (not d or torch.equal(tangent, w))
        if dual[0]:
            y = rdna4_sage.rotary(fw.make_dual(q, tq), None, at, rope, layout)
            assert torch.equal(fw.unpack_dual(y).tangent, want[0])


def test_tangent_through_the_gradient(on_cpu):
    # forward over reverse: the gradient of sum(dy f(x)) in x is f^T(dy); its tangent along dy is f^T of that
    rope, at = on_cpu
    q, k, dq, dk = tensors(2, 4)
    t = torch.randn_like(dq)
    with fw.dual_level():
        x = q.clone().requires_grad_()
        y = rdna4_sage.rotary(x, k, at, rope, "NHD")[0]
        g, = torch.autograd.grad(y, x, fw.make_dual(dq, t))
        primal, tangent = fw.unpack_dual(g)
    assert torch.equal(primal, turned(dq, None, at, rope, "NHD", True)[0])
    assert torch.equal(tangent, turned(t, None, at, rope, "NHD", True)[0])
    with fw.dual_level():                                          # both at once: a dual leaf that requires its gradient
        x = q.clone().requires_grad_()
        y = rdna4_sage.rotary(fw.make_dual(x, t), k, at, rope, "NHD")[0]
        p, ty = fw.unpack_dual(y)
        assert torch.equal(ty, turned(t, None, at, rope, "NHD", False)[0])
        g, = torch.autograd.grad(p, x, dq)
    assert torch.equal(g, turned(dq, None, at, rope, "NHD", True)[0])


def test_the_cache_refuses_dual_tensors():
    kv = rdna4_sage.PagedKV(**P.new_cache(4, 16, 2, 64))
    table, lens = torch.zeros((2, 2), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    q, k, *_ = tensors(3, 4)
    v = k.clone()
    with fw.dual_level():
        dual = lambda x: fw.make_dual(x, torch.ones_like(x))  # noqa: E731
        for no_grad in (False, True):
            with torch.set_grad_enabled(not no_grad):
                for args in ((dual(k), v), (k, dual(v))):
                    with pytest.raises(Unsupported, match="derivative"):
                        rdna4_sage.paged_kv_append(kv, *args, table, lens, tensor_layout="NHD")
                with pytest.raises(Unsupported, match="derivative"):
                    rdna4_sage.attention_paged_kv(dual(q), kv, table, lens, tensor_layout="NHD")
        with pytest.raises(Unsupported, match="CUDA GPU"):           # a plain tensor at a dual level goes on
            rdna4_sage.attention_paged_kv(q, kv, table, lens, tensor_layout="NHD")


def test_a_refused_capture_leaves_the_mark_of_an_earlier_one():
    """A graph captured on stream 7 is alive: a capture on 8 is refused, another one on 7 still is not."""
    x = torch.randn(3, requires_grad=True)
    node = _rotary._accumulator(x, 7)
    y = x * 2
    del node
    with pytest.raises(Unsupported, match="outside the capture"):
        _rotary._accumulator(x, 8)
    _rotary._accumulator(x, 7)
    with pytest.raises(Unsupported, match="outside the capture"):
        _rotary._accumulator(x, 8)
    y.sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, 2.0))
