"""The paged K/V cache (int8 K, e4m3 V, one scale per row) of a growing context, and attention over it.

quantize_kv() holds a context that is there as a whole; this cache grows by the tokens of each step, in pages that a
page table deals to the sequences.  One serving step of a batch, with `lens` the context lengths before it:

    q, k = rotary(q, k, lens[:, None] + depth, rope)               # depth: position of each draft in its tree
    paged_kv_append(kv, k, v, page_table, lens)                    # the step's tokens: positions lens, lens + 1, ...
    o = attention_paged_kv(q, kv, page_table, lens, tree_mask)     # sees the context and the drafts of the mask
    paged_kv_keep(kv, page_table, lens, accepted, counts)          # the accepted drafts move to the front
    lens += counts

No call waits for the GPU or reads its tensors on the host, so a step can be captured into a CUDA graph.  Lengths and
page numbers are checked on the device: what lies outside the cache or the table is not touched, and a later call on
the device (or check_status) raises RuntimeError.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _attention, _lib
from ._attention import (DTYPES, HEAD_DIMS, Unsupported, _current_device, _raw_stream, forward_mode, launch, step,
                         step_rows)

_alloc = getattr(torch._C, "_cuda_cudaCachingAllocator_raw_alloc", None)   # absent from a torch built without CUDA
_free = getattr(torch._C, "_cuda_cudaCachingAllocator_raw_delete", None)

PAGE_SIZES = (16, 32, 64, 128, 256)


class PagedKV:
    """The buffers of a paged cache: k8 [num_pages, kv_heads, page_size, head_dim] int8, v8 the same in
    float8_e4m3fn (or its bytes), ks and vs [num_pages, kv_heads, page_size] fp32 scales."""

    def __init__(self, k8, ks, v8, vs):
        if k8.dim() != 4 or k8.dtype != torch.int8 or v8.shape != k8.shape or \
                v8.dtype not in (torch.float8_e4m3fn, torch.uint8):
            raise Unsupported("k8 (int8) and v8 (float8_e4m3fn or uint8) must be [pages, kv_heads, page_size, head_dim]")
        if any(s.shape != k8.shape[:3] or s.dtype != torch.float32 for s in (ks, vs)):
            raise Unsupported("ks and vs must be float32 [pages, kv_heads, page_size]")
        if k8.shape[2] not in PAGE_SIZES or k8.shape[3] not in HEAD_DIMS or 0 in k8.shape:
            raise Unsupported(f"page_size {k8.shape[2]} (supported {PAGE_SIZES}), head_dim {k8.shape[3]} "
                              f"(supported {HEAD_DIMS}), at least one page and head")
        for t in (k8, ks, v8, vs):
            if not t.is_contiguous() or t.device != k8.device:
                raise Unsupported("cache buffers must be contiguous tensors on one device")
        if any(t.data_ptr() % 16 for t in (k8, ks, v8, vs)):
            raise Unsupported("cache buffers must be 16-byte aligned")
        self.k8, self.ks, self.v8, self.vs = k8, ks, v8, vs
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = k8.shape
        # error word of the device: allocated here rather than by a first call under graph capture
        self._word = _attention.host_word(k8.device) if k8.is_cuda else 0

    @classmethod
    def empty(cls, num_pages, page_size, kv_heads, head_dim, device="cuda"):
        """A cache of num_pages pages with nothing written."""
        shape = (num_pages, kv_heads, page_size, head_dim)
        return cls(torch.zeros(shape, dtype=torch.int8, device=device), torch.zeros(shape[:3], device=device),
                   torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
                   torch.zeros(shape[:3], device=device))

    @property
    def device(self):
        return self.k8.device

    def _args(self, table, lens, counts, B):
        """The cache part of a call's arguments."""
        return (self.k8.data_ptr(), self.ks.data_ptr(), self.v8.data_ptr(), self.vs.data_ptr(), table.data_ptr(),
                lens.data_ptr(), 0 if counts is None else counts.data_ptr(), self._word, table.stride(0), self.num_pages,
                self.page_size, self.kv_heads, self.head_dim, table.shape[1], B)


def _check_table(page_table, lens, counts, B):
    shape = page_table.shape
    if len(shape) != 2 or page_table.dtype != torch.int32 or shape[0] != B or shape[1] == 0 or page_table.stride(1) != 1:
        raise Unsupported(f"page_table must be int32 [{B}, pages] with contiguous rows")
    if lens.dtype != torch.int32 or lens.shape != (B,) or not lens.is_contiguous():
        raise Unsupported(f"lens must be contiguous int32 [{B}]")
    if counts is not None and (counts.dtype != torch.int32 or counts.shape != (B,) or not counts.is_contiguous()):
        raise Unsupported(f"counts must be contiguous int32 [{B}]")


def _check_rows(kv, x, layout, heads=None):
    """(B, S, heads) of step tensors in `layout`."""
    if layout not in ("HND", "NHD"):
        raise Unsupported(f"layout {layout!r}")
    if x.dtype not in DTYPES:
        raise Unsupported(f"dtype {x.dtype} (fp16 or bf16 required)")
    shape = x.shape
    if len(shape) != 4 or shape[3] != kv.head_dim:
        raise Unsupported(f"4D tensors with head_dim {kv.head_dim} required")
    B, H, S = shape[:3] if layout == "HND" else (shape[0], shape[2], shape[1])
    if H % kv.kv_heads or H == 0 or (heads is not None and H != heads):
        raise Unsupported(f"heads {H} do not fit the cache's {kv.kv_heads} kv heads")
    _no_grad(x)
    return B, S, H


def _no_grad(x):
    if x.requires_grad and torch.is_grad_enabled():
        raise Unsupported("the paged cache has no backward pass: call it under torch.no_grad()")
    if forward_mode() and forward_ad.unpack_dual(x).tangent is not None:
        raise Unsupported("the paged cache has no derivatives: pass the primal of a dual tensor")


def paged_kv_append(kv, k, v, page_table, lens, counts=None, tensor_layout="HND"):
    """Quantise and write the step's k, v: (B, Hkv, S, D) for "HND" or (B, S, Hkv, D) for "NHD", token i of sequence b at
    position lens[b] + i.  counts (int32 [B], 0..S): the tokens of each sequence in a padded batch; the cache keeps
    what it held behind them."""
    B, S, Hkv = _check_rows(kv, k, tensor_layout, kv.kv_heads)
    if v.shape != k.shape or v.dtype != k.dtype:
        raise Unsupported("k and v must match in shape and dtype")
    _no_grad(v)
    _check_table(page_table, lens, counts, B)
    if counts is None:
        dev = step(kv.k8, k, v, page_table, lens)
    else:
        dev = step(kv.k8, k, v, page_table, lens, counts)
    if B == 0 or S == 0:
        return
    k, kp, ks = step_rows(k, tensor_layout)
    v, vp, vs = step_rows(v, tensor_layout)
    launch(dev.index, "sage_paged_append", _lib.lib().sage_paged_append,
           _lib.PACK_ROWS(*kv._args(page_table, lens, counts, B), kp, vp, *ks, *vs, DTYPES[k.dtype], S))


def paged_kv_read(kv, page_table, lens, max_len, dtype=torch.bfloat16, tensor_layout="HND"):
    """k, v of positions 0 .. max_len - 1 in 16 bits, (B, Hkv, max_len, D) for "HND" or (B, max_len, Hkv, D) for "NHD",
    contiguous; positions from lens[b] on are zero.  For a dense attention() call on a context held in the cache."""
    if tensor_layout not in ("HND", "NHD"):
        raise Unsupported(f"layout {tensor_layout!r}")
    if dtype not in DTYPES:
        raise Unsupported(f"dtype {dtype} (fp16 or bf16 required)")
    if max_len < 0:
        raise ValueError(f"max_len {max_len}")
    B = lens.shape[0] if lens.dim() == 1 else -1
    _check_table(page_table, lens, None, B)
    dev = step(kv.k8, page_table, lens)
    Hkv, D = kv.kv_heads, kv.head_dim
    shape = (B, Hkv, max_len, D) if tensor_layout == "HND" else (B, max_len, Hkv, D)
    k = torch.empty(shape, device=dev, dtype=dtype)
    v = torch.empty_like(k)
    if 0 in shape:
        return k, v
    _, kp, st = step_rows(k, tensor_layout)
    launch(dev.index, "sage_paged_read", _lib.lib().sage_paged_read,
           _lib.PACK_ROWS(*kv._args(page_table, lens, None, B), kp, v.data_ptr(), *st, *st, DTYPES[dtype], max_len))
    return k, v


def paged_kv_keep(kv, page_table, lens, keep, counts=None):
    """Drop rejected drafts: the token at position lens[b] + keep[b, i] moves to lens[b] + i, for i < counts[b] (all N
    without counts).  keep: int32 [B, N], strictly increasing in each row (the accepted path of a tree whose parents
    come before their children); entries from counts[b] on are not read."""
    B = lens.shape[0] if lens.dim() == 1 else -1
    _check_table(page_table, lens, counts, B)
    if keep.dim() != 2 or keep.shape[0] != B or keep.dtype != torch.int32 or (keep.shape[1] > 1 and keep.stride(1) != 1):
        raise Unsupported(f"keep must be int32 [{B}, N] with contiguous rows")
    if counts is None:
        dev = step(kv.k8, page_table, lens, keep)
    else:
        dev = step(kv.k8, page_table, lens, keep, counts)
    if keep.numel() == 0:
        return
    launch(dev.index, "sage_paged_keep", _lib.lib().sage_paged_keep,
           _lib.PACK_KEEP(*kv._args(page_table, lens, counts, B), keep.data_ptr(), keep.stride(0), keep.shape[1]))


def attention_paged_kv(q, kv, page_table, lens, tree_mask=None, counts=None, tensor_layout="HND", sm_scale=None,
                       return_lse=False):
    """Attention of the step's T tokens over the cache, which already holds their K and V: q (B, H, T, D) for "HND" or
    (B, T, H, D) for "NHD".  Token i of sequence b sees the context (positions before lens[b]) and of the step's own
    tokens those t <= i, or with tree_mask (bool [T, T] or [B, T, T]) those with tree_mask[b, i, t].  counts (int32 [B],
    0..T): the tokens of each sequence in a padded batch.  sm_scale: factor of the scores (default, and for values up to
    0: 1 / sqrt(D)).  Returns the result in q's layout and dtype, and with return_lse also the (B, H, T) fp32 log-sum-exp;
    tokens from counts[b] on, and rows that see nothing, are zero with log-sum-exp -inf."""
    B, T, H = _check_rows(kv, q, tensor_layout)
    _check_table(page_table, lens, counts, B)
    tensors = [kv.k8, q, page_table, lens]
    if counts is not None:
        tensors.append(counts)
    mask, mask_b, mask_i = 0, 0, 0
    if tree_mask is not None:
        shape = tree_mask.shape
        if tree_mask.dtype != torch.bool or shape != (B, T, T) and shape != (T, T) and shape != (1, T, T):
            raise Unsupported(f"tree_mask must be bool [{T}, {T}] or [{B}, {T}, {T}]")
        tensors.append(tree_mask)
        st = tree_mask.stride()
        if st[-1] != 1:
            tree_mask = tree_mask.contiguous()
            st = tree_mask.stride()
        mask, mask_i = tree_mask.data_ptr(), st[-2]
        mask_b = st[0] if len(st) == 3 and shape[0] == B else 0
    dev = step(*tensors)
    q, qp, qs = step_rows(q, tensor_layout)
    out = torch.empty_like(q)   # of a tensor that the kernels take, so it is one too
    lse = q.new_empty((B, H, T), dtype=torch.float32) if return_lse else None
    if B and T:
        _, op, os = step_rows(out, tensor_layout)
        L, index = _lib.lib(), dev.index
        ws_bytes = L.sage_paged_attention_workspace_bytes(B, T, H, kv.kv_heads, kv.head_dim)
        # for the call alone: back with the stream's allocator as soon as the kernels are enqueued
        stream = _raw_stream(index)
        ws = _alloc(ws_bytes, stream) if _current_device() == index else None
        hold = torch.empty(ws_bytes, device=dev, dtype=torch.uint8) if ws is None else None
        try:
            launch(index, "sage_paged_attention", L.sage_paged_attention,
                   _lib.PACK_ATTENTION(*kv._args(page_table, lens, counts, B), qp, op, lse.data_ptr() if return_lse else 0,
                                       mask, ws if hold is None else hold.data_ptr(), ws_bytes, *qs, *os, mask_b, mask_i,
                                       float(sm_scale or 0.0), DTYPES[q.dtype], T, H))
        finally:
            if hold is None:
                _free(ws)
    return (out, lse) if return_lse else out
