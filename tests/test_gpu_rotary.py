"""Rotary positions on the GPU against the formula in 64 bits, and their gradient against the formula and differences.

Tolerance: y = m (x1 c -+ x2 s).  The angle is off by at most 2^-25 half turns (the fraction of a turn rounded to a
float) = 9.4e-8, sincospi by 2 units of 2^-24, the factor m, the two products and the sum round by 2^-24 each: together
below 2^-20 of m (|x1| + |x2|).  Here and in the formula in 64 bits a frequency is known to 2^-53, which an angle of
p positions multiplies: p 2^-52 more.  Then the result is rounded once, by half a step of its type (fp16: at least 2^-25)."""
import math

import pytest
import torch

import paged_reference as P
import rdna4_sage

pytestmark = pytest.mark.gpu


def close(got, want, x, m, far=0):
    """`x`: the turned input, whose row's largest pair bounds |x1| + |x2|."""
    size = 2 * m * x.double().abs().amax(-1, keepdim=True)
    tol = torch.finfo(got.dtype).eps / 2 * want.abs() + (2.0 ** -20 + far * 2.0 ** -52) * size + 2.0 ** -25
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


def nhd(x, layout):
    return x if layout == "NHD" else x.transpose(1, 2)


CASES = [  # B, S, H, Hkv, D, R, interleaved, scaling, start, dtype, layout
    (1, 1, 1, 1, 64, 64, False, None, 0, torch.bfloat16, "NHD"),
    (3, 7, 5, 1, 64, 32, True, "linear", 5, torch.float16, "HND"),
    (2, 130, 8, 2, 96, 96, False, "ntk", 1000, torch.bfloat16, "HND"),
    (2, 33, 4, 4, 96, 16, True, "ramp", 70000, torch.float16, "NHD"),
    (5, 1, 32, 8, 128, 128, False, "ramp", 10 ** 6, torch.bfloat16, "NHD"),
    (1, 257, 12, 4, 128, 64, True, None, -300, torch.bfloat16, "HND"),
    (2, 19, 3, 3, 256, 256, False, "linear", 2 ** 32, torch.float16, "NHD"),
    (1, 65, 16, 2, 256, 128, True, "ntk", 12345, torch.bfloat16, "NHD"),
]


def make(c):
    B, S, H, Hkv, D, R, inter, scaling, start, dtype, layout = c
    g = torch.Generator(device="cuda").manual_seed(S * D + R)
    more = dict(factor=8.0, original_len=4096, ramp=(1.0, 32.0)) if scaling == "ramp" else dict(factor=8.0)
    rope = rdna4_sage.Rotary(D, rotary_dim=R, interleaved=inter, scaling=scaling, **(more if scaling else {}))
    shape = (lambda h: (B, S, h, D)) if layout == "NHD" else (lambda h: (B, h, S, D))
    q, k = (torch.randn(shape(h), device="cuda", generator=g).to(dtype) for h in (H, Hkv))
    pos = start + torch.randint(0, 500, (B, S), device="cuda", generator=g)
    pos = pos if abs(start) > 2 ** 31 else pos.int()
    ref = lambda x, back=False: nhd(P.rotary(nhd(x.detach(), layout), pos, rope.frequencies, rope.magnitude, R,  # noqa: E731
                                             inter, back), layout)
    return q, k, pos, rope, layout, ref


@pytest.mark.parametrize("c", CASES)
def test_forward_and_gradient(c):
    q, k, pos, rope, layout, ref = make(c)
    got_q, got_k = rdna4_sage.rotary(q, k, pos, rope, layout)
    assert got_q.shape == q.shape and got_k.dtype == k.dtype
    far = abs(c[8])
    close(got_q, ref(q), q, rope.magnitude, far)
    close(got_k, ref(k), k, rope.magnitude, far)
    only = rdna4_sage.rotary(q, None, pos, rope, layout)
    assert torch.equal(only, got_q)
    q1, k1 = q.clone().requires_grad_(), k.clone().requires_grad_()
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    out = rdna4_sage.rotary(q1, k1, pos, rope, layout)
    assert torch.equal(out[0], got_q) and torch.equal(out[1], got_k)
    gq, gk = torch.autograd.grad(out, (q1, k1), (dq, dk))
    close(gq, ref(dq, True), dq, rope.magnitude, far)
    close(gk, ref(dk, True), dk, rope.magnitude, far)


def test_gradient_against_differences():
    # the op is linear: <dy, f(x + h) - f(x)> = <gradient, h>.  Each of the three tensors is rounded by half a step of
    # its size, independent signs are not assumed: the sums of the bounds are the tolerance
    q, k, pos, rope, layout, _ = make(CASES[6])
    eps = torch.finfo(q.dtype).eps / 2 + 2.0 ** -19
    x, h, dy = q.clone().requires_grad_(), torch.randn_like(q), torch.randn_like(q)
    moved = (x.detach() + h)
    y0, y1 = rdna4_sage.rotary(x.detach(), None, pos, rope, layout), rdna4_sage.rotary(moved, None, pos, rope, layout)
    g, = torch.autograd.grad(rdna4_sage.rotary(x, None, pos, rope, layout), x, dy)
    step = moved.double() - x.detach().double()
    lhs, rhs = (dy.double() * (y1.double() - y0.double())).sum(), (g.double() * step).sum()
    size = lambda t: 2 * t.double().abs().amax(-1, keepdim=True)  # noqa: E731
    tol = eps * ((dy.double().abs() * (size(y1) + size(y0))).sum() + (size(g) * step.abs()).sum())
    assert abs(float(lhs - rhs)) <= float(tol)


def test_gradients_of_one_input_and_of_broadcast_inputs():
    q, k, pos, rope, layout, ref = make(CASES[4])
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    k1 = k.clone().requires_grad_()
    out = rdna4_sage.rotary(q, k1, pos, rope, layout)
    assert torch.equal(torch.autograd.grad(out, k1, (dq, dk))[0], rdna4_sage.rotary(dk, None, -pos, rope, layout))
    q1 = q.clone().requires_grad_()
    out = rdna4_sage.rotary(q1, k1, pos, rope, layout)
    g = torch.autograd.grad(out[0], (q1, k1), dq, allow_unused=True)      # k's output unused
    close(g[0], ref(dq, True), dq, rope.magnitude)
    assert g[1] is None or not bool(g[1].any())
    # one head for all: the gradient is the sum over the heads
    one = k[:, :, :1].clone().requires_grad_()
    wide = one.expand_as(k)
    g, = torch.autograd.grad(rdna4_sage.rotary(wide, None, pos, rope, layout), one, dk)
    want = rdna4_sage.rotary(dk, None, -pos, rope, layout).double().sum(2, keepdim=True)
    # torch sums the eight 16-bit rows in fp32 and rounds once
    tol = torch.finfo(g.dtype).eps / 2 * want.abs() + 2.0 ** -20 * dk.double().abs().sum(2, keepdim=True) * 2 + 2.0 ** -25
    assert bool(((g.double() - want).abs() <= tol).all())
    # second derivatives: the gradient of <gradient, x> in dy is the op on x
    x, dy = q.clone().requires_grad_(), dq.clone().requires_grad_()
    g, = torch.autograd.grad(rdna4_sage.rotary(x, None, pos, rope, layout), x, dy, create_graph=True)
    gg, = torch.autograd.grad(g, dy, q)
    assert torch.equal(gg, rdna4_sage.rotary(q, None, pos, rope, layout))


def test_strides_alignment_and_positions():
    q, k, pos, rope, layout, ref = make(CASES[5])               # HND
    want_q, want_k = rdna4_sage.rotary(q, k, pos, rope, layout)
    packed = torch.randn((*q.shape[:3], 3 * q.shape[3]), device="cuda").to(q.dtype)
    packed[..., 128:256] = q
    odd = torch.empty(q.numel() + 1, device="cuda", dtype=q.dtype)[1:].view(q.shape).copy_(q)    # 2 bytes off
    for x in (q.transpose(1, 2).contiguous().transpose(1, 2), packed[..., 128:256], odd,
              q.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)):
        assert torch.equal(rdna4_sage.rotary(x, k, pos, rope, layout)[0], want_q)
    every = torch.arange(q.shape[2], device="cuda")
    a = rdna4_sage.rotary(q, k, every, rope, layout)
    for p in (every.int(), every[None], every.expand(q.shape[0], -1), torch.stack((every, every), 1)[:, 0]):
        b = rdna4_sage.rotary(q, k, p, rope, layout)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # no tokens, no sequences
    assert rdna4_sage.rotary(q[:, :, :0], k[:, :, :0], every[:0], rope, layout)[1].shape == k[:, :, :0].shape
    assert rdna4_sage.rotary(q[:0], None, every, rope, layout).shape[0] == 0


def test_streams_graph_and_compile_free_use():
    q, k, pos, rope, layout, ref = make(CASES[2])
    want = rdna4_sage.rotary(q, k, pos, rope, layout)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rdna4_sage.rotary(q, k, pos, rope, layout)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros_like(q)
    with torch.cuda.graph(graph):
        y = rdna4_sage.rotary(x, k, pos, rope, layout)
    x.copy_(q)
    graph.replay()
    assert torch.equal(y[0], want[0])
    # infinities and NaN stay in their own pairs
    bad = q.clone()
    bad[0, 0, 3, 5] = math.inf
    y = rdna4_sage.rotary(bad, None, pos, rope, layout)
    hit = torch.zeros_like(q, dtype=torch.bool)
    hit[0, 0, 3, 5] = hit[0, 0, 3, 5 + 48] = True
    assert torch.equal(y[~hit], want[0][~hit]) and not bool(torch.isfinite(y[hit]).any())


def leaves(seed=3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k = (torch.randn(2, 5, h, 128, device="cuda", generator=g).bfloat16() for h in (8, 2))
    dq, dk = (torch.randn(2, 5, h, 128, device="cuda", generator=g).bfloat16() for h in (8, 2))
    return q.requires_grad_(), k.requires_grad_(), dq, dk, torch.arange(5, device="cuda"), rdna4_sage.Rotary(128)


def test_captured_gradient():
    """Two calls on the same leaves in one capture, replayed with other gradients and positions."""
    q, k, dq, dk, pos, rope = leaves()

    def run():
        a, b = rdna4_sage.rotary(q, k, pos, rope, "NHD")
        c = rdna4_sage.rotary(q, None, pos, rope, "NHD")
        return torch.autograd.grad((a, b, c), (q, k), (dq, dk, dq))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for turn in range(3):
        dq.mul_(-0.5)
        pos.add_(100 * turn)
        graph.replay()
        want = run()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_captured_gradient_of_a_leaf_in_another_graph_is_refused():
    q, k, dq, dk, pos, rope = leaves()
    alive = rdna4_sage.rotary(q, k, pos, rope, "NHD")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x = torch.zeros_like(dq)
        with pytest.raises(rdna4_sage.Unsupported, match="outside the capture"):
            rdna4_sage.rotary(q, k, pos, rope, "NHD")
        with torch.no_grad():
            y = rdna4_sage.rotary(q, k, pos, rope, "NHD")   # without a gradient there is nothing to refuse
    graph.replay()
    assert torch.equal(y[0], alive[0]) and torch.equal(y[1], alive[1]) and not bool(x.any())
    got = torch.autograd.grad(alive, (q, k), (dq, dk))        # the graph that was alive still answers
    want = torch.autograd.grad(rdna4_sage.rotary(q, k, pos, rope, "NHD"), (q, k), (dq, dk))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
