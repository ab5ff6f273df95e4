"""Rotary positions for q and k: the frequencies a model keeps (Rotary) and the op (rotary), with its gradient.

The reference leaves positions to its callers; here they sit in front of attention() and of the paged K/V cache, which
stores keys already turned.
"""
from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from . import _lib
from ._attention import DTYPES, HEAD_DIMS, Unsupported, forward_mode, launch, step, step_rows

SCALINGS = (None, "linear", "ntk", "ramp")


class Rotary:
    """The frequencies of rotary positions on one GPU.

    Channels 0 .. rotary_dim - 1 of each head (default: all of them; a multiple of 16) are turned in pairs: channel i
    with i + rotary_dim / 2, or 2 i with 2 i + 1 when `interleaved`.  Pair i has frequency w_i = base^(-2 i / rotary_dim)
    radians per position, scaled for contexts longer than the trained one by
      scaling="linear"  w_i / factor
      scaling="ntk"     base * factor^(rotary_dim / (rotary_dim - 2)) in place of base
      scaling="ramp"    w_i (g / 1 + (1 - g) / factor), where g rises from 0 to 1 as the number of turns within
                        original_len positions, r_i = original_len w_i / (2 pi), rises from ramp[0] to ramp[1]
                        (programs that let g rise with i between the two have other frequencies: give those themselves)
    `magnitude` multiplies the turned channels (default 1; for "ramp" 0.1 ln(factor) + 1).  `frequencies`: a tensor or
    list of rotary_dim / 2 radians per position in place of all this.
    """

    def __init__(self, head_dim, rotary_dim=None, base=10000.0, interleaved=False, scaling=None, factor=1.0,
                 original_len=None, ramp=(1.0, 32.0), magnitude=None, frequencies=None, device=None):
        R = head_dim if rotary_dim is None else rotary_dim
        if head_dim not in HEAD_DIMS:
            raise Unsupported(f"head_dim {head_dim} (supported {HEAD_DIMS})")
        if R < 16 or R > head_dim or R % 16:
            raise Unsupported(f"rotary_dim {R} (a multiple of 16 up to head_dim {head_dim} required)")
        if frequencies is not None:
            if scaling is not None:
                raise ValueError("give frequencies or a scaling, not both")
            w = torch.as_tensor(frequencies, dtype=torch.float64, device="cpu").detach()
            if w.shape != (R // 2,) or not bool(torch.isfinite(w).all()):
                raise ValueError(f"frequencies: {R // 2} finite numbers required")
        else:
            w = _frequencies(R, base, scaling, factor, original_len, ramp)
        if magnitude is None:
            magnitude = 0.1 * math.log(factor) + 1.0 if scaling == "ramp" else 1.0
        self.head_dim, self.rotary_dim, self.interleaved, self.magnitude = head_dim, R, bool(interleaved), float(magnitude)
        self.frequencies = w
        # turns per position as 64-bit fixed-point fractions, in (-1/2, 1/2] of a turn
        turns = w / (2 * math.pi)
        turns = [int(round((t - round(t)) * 2.0 ** 64)) for t in turns.tolist()]
        self.turns = torch.tensor([min(max(t, -2 ** 63), 2 ** 63 - 1) for t in turns], dtype=torch.int64,
                                  device="cuda" if device is None else device)


def _frequencies(R, base, scaling, factor, original_len, ramp):
    if scaling not in SCALINGS:
        raise ValueError(f"scaling {scaling!r} (one of {SCALINGS})")
    if not (base > 1.0 and math.isfinite(base) and factor > 0.0 and math.isfinite(factor)):
        raise ValueError(f"base {base} (above 1) and factor {factor} (above 0) must be finite")
    i = torch.arange(0, R, 2, dtype=torch.float64)
    if scaling == "ntk":
        base = base * factor ** (R / (R - 2))
    w = base ** (-i / R)
    if scaling == "linear":
        return w / factor
    if scaling == "ramp":
        lo, hi = ramp
        if original_len is None or original_len <= 0 or not lo < hi:
            raise ValueError('scaling="ramp" needs original_len > 0 and ramp[0] < ramp[1]')
        g = ((original_len * w / (2 * math.pi) - lo) / (hi - lo)).clamp(0.0, 1.0)
        return w * (g + (1.0 - g) / factor)
    return w


def _check(q, k, positions, rope, layout):
    """Raise Unsupported with the reason if the kernel cannot run these inputs (devices aside)."""
    if layout not in ("HND", "NHD"):
        raise Unsupported(f"layout {layout!r}")
    s_ax = 2 if layout == "HND" else 1
    shape = q.shape
    if q.dtype not in DTYPES or len(shape) != 4 or shape[3] != rope.head_dim:
        _refuse(q, q, rope)
    if k is not None:
        other = k.shape
        if k.dtype != q.dtype or len(other) != 4 or other[3] != rope.head_dim:
            _refuse(q, k, rope)
        if other[0] != shape[0] or other[s_ax] != shape[s_ax]:
            raise Unsupported("q and k must hold the same tokens")
    if positions.dtype not in (torch.int32, torch.int64):
        raise Unsupported(f"positions {positions.dtype} (int32 or int64 required)")
    B, S, at = shape[0], shape[s_ax], positions.shape
    if at != (B, S) and at != (S,) and at != (1, S):
        raise Unsupported(f"positions {tuple(at)}: (S,) or (B, S) of ({B}, {S}) tokens required")


def _refuse(q, x, rope):
    if x.dtype not in DTYPES or x.dtype != q.dtype:
        raise Unsupported(f"dtype {x.dtype} (fp16 or bf16, one for q and k, required)")
    raise Unsupported(f"4D tensors with head_dim {rope.head_dim} required")


def _launch(q, k, positions, rope, layout, backward):
    """(q, k) turned, new tensors in the inputs' layout (k may be None)."""
    if q.numel() == 0 or k is not None and k.numel() == 0:
        if q.numel() != 0 or k is not None and k.numel() != 0:
            raise Unsupported("q and k must both hold heads")
        return torch.empty_like(q), None if k is None else torch.empty_like(k)
    q, qp, qs = step_rows(q, layout)
    q_out = torch.empty_like(q)   # of a tensor that the kernels take, so it is one too
    _, qop, qos = step_rows(q_out, layout)
    if layout == "HND":
        B, H, S, D = q.shape
    else:
        B, S, H, D = q.shape
    if k is None:
        k_out, Hkv, kp, kop, ks, kos = None, 0, 0, 0, (0, 0, 0), (0, 0, 0)
    else:
        k, kp, ks = step_rows(k, layout)
        k_out = torch.empty_like(k)
        _, kop, kos = step_rows(k_out, layout)
        Hkv = k.shape[1 if layout == "HND" else 2]
    ps = positions.stride()
    pb = ps[0] if len(ps) == 2 and positions.shape[0] > 1 else 0
    args = _lib.PACK_ROTARY(qp, kp, qop, kop, positions.data_ptr(), rope.turns.data_ptr(), *qs, *ks, *qos, *kos, pb, ps[-1],
                            DTYPES[q.dtype], B, S, H, Hkv, D, rope.rotary_dim, rope.interleaved,
                            32 if positions.dtype == torch.int32 else 64, rope.magnitude, backward)
    launch(q.get_device(), "sage_rotary", _lib.lib().sage_rotary, args)
    return q_out, k_out


class _RotaryFunction(torch.autograd.Function):
    """The gradient of a turn is the turn by the negative angle, so the backward pass is the op itself again."""

    @staticmethod
    def forward(ctx, q, k, positions, rope, layout, backward):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions)
        ctx.rope, ctx.layout, ctx.turn_back = rope, layout, not backward
        q_out, k_out = _launch(q, k, positions, rope, layout, backward)
        return q_out if k is None else (q_out, k_out)

    @staticmethod
    def backward(ctx, dq, dk=None):
        positions, = ctx.saved_tensors
        dq = dq if ctx.needs_input_grad[0] else None
        dk = dk if ctx.needs_input_grad[1] else None
        args = (positions, ctx.rope, ctx.layout, ctx.turn_back)
        if dq is not None:
            dq, dk = _turn(dq, dk, *args)
        elif dk is not None:
            dk, _ = _turn(dk, None, *args)
        return dq, dk, None, None, None, None


def _turn(q, k, positions, rope, layout, backward):
    """(q, k) turned (k may be None), with the derivatives that the inputs ask for."""
    if forward_mode():
        # the op is linear: the tangent of a result is the op on the tangent
        (q, tq), (k, tk) = forward_ad.unpack_dual(q), (None, None) if k is None else forward_ad.unpack_dual(k)
        if tq is not None or tk is not None:
            out = _turn(q, k, positions, rope, layout, backward)
            if tq is not None and tk is not None:
                tangents = _turn(tq, tk, positions, rope, layout, backward)
            else:
                tangents = [None if t is None else _turn(t, None, positions, rope, layout, backward)[0] for t in (tq, tk)]
            return tuple(y if t is None else forward_ad.make_dual(y, t) for y, t in zip(out, tangents))
    if (q.requires_grad or k is not None and k.requires_grad) and torch.is_grad_enabled():
        out = _RotaryFunction.apply(q, k, positions, rope, layout, backward)
        return (out, None) if k is None else out
    return _launch(q, k, positions, rope, layout, backward)


_MARK = "rdna4_sage capture"


def _accumulator(x, stream):
    """The node that adds up the gradient of leaf `x`, for a graph recorded while `stream` is captured.  A leaf has one
    node, tied to the stream where the oldest graph alive made it; from another stream's, a captured backward pass would
    wait for work outside the capture, which breaks the capture off.  Autograd does not tell a node's stream, but a mark
    outlives the last reference held here only if another graph holds the node."""
    edge = torch.autograd.graph.get_gradient_edge
    node = edge(x).node
    before = node.metadata.get(_MARK)
    if before == stream:   # an earlier call of this capture
        return node
    node.metadata[_MARK] = stream
    del node
    node = edge(x).node
    if _MARK in node.metadata:
        if before is None:
            del node.metadata[_MARK]
        else:
            node.metadata[_MARK] = before
        raise Unsupported("a graph of this leaf from outside the capture is alive, so its gradient cannot be captured: "
                          "release that graph first (or pass a view of the leaf if it was recorded on this stream)")
    node.metadata[_MARK] = stream
    return node


def rotary(q, k, positions, rope, tensor_layout="HND"):
    """q and k turned to their positions: (B, H, S, D) and (B, Hkv, S, D) for "HND", (B, S, H, D) and (B, S, Hkv, D) for
    "NHD", fp16 or bf16; new tensors of the same shapes and types (rounded once).  k may be None: the result is q
    alone.  positions: int32 or int64 of any value, (S,) for all sequences or (B, S), on the GPU.  rope: a Rotary.
    Differentiable in q and k, in reverse and in forward mode (dual tensors).  A backward pass can be captured into a CUDA graph if no other graph of the same leaves is
    alive then; a leaf q or k that breaks this is refused, leaves further back are the caller's.  Raises Unsupported for
    inputs the kernel does not take."""
    _check(q, k, positions, rope, tensor_layout)
    if k is None:
        step(q, positions, rope.turns)
    else:
        step(q, k, positions, rope.turns)
    if (q.requires_grad or k is not None and k.requires_grad) and torch.is_grad_enabled():
        if torch.cuda.is_current_stream_capturing():   # the nodes are held until the graph below holds them
            at = torch.cuda.current_stream(q.device).cuda_stream
            held = [_accumulator(x, at) for x in (q, k) if x is not None and x.requires_grad and x.is_leaf]  # noqa: F841
    q_out, k_out = _turn(q, k, positions, rope, tensor_layout, False)
    return q_out if k is None else (q_out, k_out)
