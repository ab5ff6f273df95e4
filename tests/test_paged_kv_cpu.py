"""Refusals and host arithmetic of rotary positions and the paged K/V cache, without a GPU."""
import ctypes
import math
import os
import struct
import subprocess

import pytest
import torch

import paged_reference as P
import rdna4_sage
from rdna4_sage import Unsupported, _lib


def cache(pages=4, page=16, Hkv=2, D=64):
    return rdna4_sage.PagedKV(**P.new_cache(pages, page, Hkv, D))


def step(B=2, T=3, H=4, D=64, dtype=torch.bfloat16):
    return torch.zeros((B, T, H, D), dtype=dtype)


TABLE = torch.zeros((2, 2), dtype=torch.int32)
LENS = torch.zeros(2, dtype=torch.int32)


@pytest.mark.parametrize("change,match", [
    (dict(page=17), "page_size 17"), (dict(page=512), "page_size 512"), (dict(D=80), "head_dim 80"),
    (dict(pages=0), "at least one page"), (dict(Hkv=0), "at least one page")])
def test_cache_shapes_refused(change, match):
    with pytest.raises(Unsupported, match=match):
        cache(**change)


def test_cache_buffers_refused():
    c = P.new_cache(4, 16, 2, 64)
    for name, bad, match in [("k8", c["k8"].float(), "k8"), ("v8", c["v8"][:3], "v8"), ("ks", c["ks"].double(), "float32"),
                             ("vs", c["vs"][:, :1], "float32"),
                             ("k8", c["k8"].transpose(1, 2).contiguous().transpose(1, 2), "contiguous")]:
        with pytest.raises(Unsupported, match=match):
            rdna4_sage.PagedKV(**{**c, name: bad})
    kv = rdna4_sage.PagedKV(**{**c, "v8": c["v8"].view(torch.uint8)})     # bytes are taken for v8
    assert (kv.num_pages, kv.kv_heads, kv.page_size, kv.head_dim) == (4, 2, 16, 64)
    assert rdna4_sage.PagedKV.empty(3, 32, 2, 96, device="cpu").k8.shape == (3, 2, 32, 96)


@pytest.mark.parametrize("args,kw,match", [
    ((step(H=2, dtype=torch.float32),), {}, "dtype"),
    ((step(H=2, D=128),), {}, "head_dim 64"),
    ((step(H=4),), {}, "heads 4"),
    ((step(H=2),), dict(tensor_layout="BSHD"), "layout"),
    ((step(H=2),), dict(v=step(H=2, T=4)), "match"),
    ((step(H=2),), dict(table=TABLE.long()), "page_table"),
    ((step(H=2),), dict(table=TABLE[:1]), "page_table"),
    ((step(H=2),), dict(table=TABLE.t().contiguous().t()), "page_table"),
    ((step(H=2),), dict(lens=LENS.long()), "lens"),
    ((step(H=2),), dict(lens=LENS[:1]), "lens"),
    ((step(H=2),), dict(counts=torch.zeros(3, dtype=torch.int32)), "counts"),
    ((step(H=2),), {}, "CUDA GPU")])
def test_append_refused(args, kw, match):
    kw = dict(kw)
    kw.setdefault("tensor_layout", "NHD")
    k = args[0]
    with pytest.raises(Unsupported, match=match):
        rdna4_sage.paged_kv_append(cache(), k, kw.pop("v", k), kw.pop("table", TABLE), kw.pop("lens", LENS), **kw)


@pytest.mark.parametrize("kw,match", [
    (dict(q=step(H=3)), "heads 3"), (dict(q=step(D=96)), "head_dim 64"), (dict(q=step().float()), "dtype"),
    (dict(tree_mask=torch.ones((4, 4), dtype=torch.bool)), "tree_mask"),
    (dict(tree_mask=torch.ones((3, 3))), "tree_mask"),
    (dict(tree_mask=torch.ones((3, 3, 3), dtype=torch.bool)), "tree_mask"),
    (dict(q=step().requires_grad_()), "no backward"),
    (dict(), "CUDA GPU")])
def test_attention_refused(kw, match):
    kw = dict(kw)
    with pytest.raises(Unsupported, match=match):
        rdna4_sage.attention_paged_kv(kw.pop("q", step()), cache(), TABLE, LENS, tensor_layout="NHD", **kw)


def test_read_and_keep_refused():
    with pytest.raises(Unsupported, match="dtype"):
        rdna4_sage.paged_kv_read(cache(), TABLE, LENS, 5, dtype=torch.float32)
    with pytest.raises(ValueError, match="max_len"):
        rdna4_sage.paged_kv_read(cache(), TABLE, LENS, -1)
    with pytest.raises(Unsupported, match="page_table"):
        rdna4_sage.paged_kv_read(cache(), TABLE, LENS[None], 5)
    for keep in (torch.zeros(2, dtype=torch.int32), torch.zeros((2, 3)), torch.zeros((1, 3), dtype=torch.int32),
                 torch.zeros((3, 2), dtype=torch.int32).t()):
        with pytest.raises(Unsupported, match="keep"):
            rdna4_sage.paged_kv_keep(cache(), TABLE, LENS, keep)
    with pytest.raises(Unsupported, match="CUDA GPU"):
        rdna4_sage.paged_kv_keep(cache(), TABLE, LENS, torch.zeros((2, 3), dtype=torch.int32))


def test_rotary_refused():
    rope = rdna4_sage.Rotary(64, device="cpu")
    at = torch.arange(3)
    for q, k, pos, layout, match in [
            (step(), step(H=2), at, "BSHD", "layout"), (step(), step(H=2, dtype=torch.float16), at, "NHD", "dtype"),
            (step(D=128), None, at, "NHD", "head_dim 64"), (step(), step(T=2), at, "NHD", "same tokens"),
            (step(), None, at.float(), "NHD", "positions"), (step(), None, at[:2], "NHD", "positions"),
            (step(), None, at[None].expand(3, 3), "NHD", "positions"), (step(), step(), at, "NHD", "CUDA GPU")]:
        with pytest.raises(Unsupported, match=match):
            rdna4_sage.rotary(q, k, pos, rope, tensor_layout=layout)
    for kw in (dict(head_dim=80), dict(head_dim=64, rotary_dim=24), dict(head_dim=64, rotary_dim=80),
               dict(head_dim=64, rotary_dim=0)):
        with pytest.raises(Unsupported):
            rdna4_sage.Rotary(device="cpu", **kw)
    for kw in (dict(scaling="other"), dict(scaling="ramp", factor=2.0), dict(base=0.5), dict(factor=0.0),
               dict(scaling="ramp", factor=2.0, original_len=64, ramp=(4.0, 4.0)), dict(frequencies=[1.0]),
               dict(frequencies=[math.inf] * 32), dict(frequencies=[1.0] * 32, scaling="linear")):
        with pytest.raises(ValueError):
            rdna4_sage.Rotary(64, device="cpu", **kw)


def test_rotary_frequencies():
    R = 64
    i = torch.arange(R // 2, dtype=torch.float64)
    w = 10000.0 ** (-2 * i / R)
    make = lambda **kw: rdna4_sage.Rotary(128, rotary_dim=R, device="cpu", **kw)  # noqa: E731
    torch.testing.assert_close(make().frequencies, w, rtol=1e-14, atol=0)
    torch.testing.assert_close(make(scaling="linear", factor=8.0).frequencies, w / 8, rtol=1e-14, atol=0)
    torch.testing.assert_close(make(scaling="ntk", factor=8.0).frequencies[-1], w[-1] / 8, rtol=1e-12, atol=0)
    r = make(scaling="ramp", factor=8.0, original_len=4096, ramp=(1.0, 4.0))
    turns = 4096 * w / (2 * math.pi)
    torch.testing.assert_close(r.frequencies[turns >= 4], w[turns >= 4], rtol=1e-14, atol=0)
    torch.testing.assert_close(r.frequencies[turns <= 1], w[turns <= 1] / 8, rtol=1e-14, atol=0)
    mid = (turns > 1) & (turns < 4)
    assert bool(mid.any()) and bool(((r.frequencies[mid] < w[mid]) & (r.frequencies[mid] > w[mid] / 8)).all())
    assert r.magnitude == pytest.approx(0.1 * math.log(8.0) + 1.0) and make().magnitude == 1.0
    # the fixed-point turns: the fraction of a turn at a far position is right to 2^-53 * position
    for pos in (1, 1000, 2 ** 20 + 3):
        for f, t in zip(r.frequencies.tolist(), r.turns.tolist()):
            got = (pos * t) % 2 ** 64 / 2.0 ** 64
            want = math.fmod(pos * f / (2 * math.pi), 1.0)
            d = abs(got - want)
            assert min(d, 1 - d) <= pos * 2.0 ** -52, (pos, f)
    # any frequency is taken: whole turns fall away (the product and the quotient by 2 pi each round by 2^-53 of 3.25,
    # together at most 2^-50 of a turn)
    own = rdna4_sage.Rotary(64, device="cpu", frequencies=[2 * math.pi * 3.25] * 32)  # held in 64 bits
    assert abs(int(own.turns[0]) - 2 ** 62) <= 2 ** 14


def test_c_entries_check_their_arguments_without_gpu():
    L = _lib.lib()
    p, st = 256, [8, 8, 8]
    bad, unsupported = _lib.SAGE_ERR_INVALID, _lib.SAGE_ERR_UNSUPPORTED

    def rot(q=p, k=p, turns=p, D=64, R=64, bits=32):
        return L.sage_rotary(_lib.PACK_ROTARY(q, k, p, p, p, turns, *st * 4, 3, 1, 0, 1, 3, 2, 1, D, R, 0, bits, 1.0, 0), None)
    assert rot(D=80) == unsupported and rot(R=24) == unsupported and rot(bits=16) == unsupported
    assert rot(q=8) == bad and rot(k=0) == bad and rot(turns=0) == bad and L.sage_rotary(None, None) == bad

    def kv(k8=p, ks=p, table=p, lens=p, pages=4, page=16, Hkv=2, D=64, most=2):
        return k8, ks, p, p, table, lens, 0, p, 2, pages, page, Hkv, D, most, 2

    def rows(entry, k=p, S=3, dtype=0, **kw):
        return getattr(L, entry)(_lib.PACK_ROWS(*kv(**kw), k, p, *st * 2, dtype, S), None)
    for entry in ("sage_paged_append", "sage_paged_read"):
        assert rows(entry, D=80) == unsupported and b"head_dim 80" in L.sage_last_error()
        assert rows(entry, k=8) == bad and rows(entry, S=0) == unsupported and rows(entry, dtype=2) == unsupported
        assert rows(entry, page=24) == unsupported and b"page_size 24" in L.sage_last_error()
        assert rows(entry, pages=0) == unsupported and rows(entry, k8=8) == bad and rows(entry, ks=0) == bad
        assert rows(entry, table=0) == bad and rows(entry, lens=0) == bad and rows(entry, ks=260) == bad
        assert getattr(L, entry)(None, None) == bad

    def keep(keep=p, N=3, **kw):
        return L.sage_paged_keep(_lib.PACK_KEEP(*kv(**kw), keep, 3, N), None)
    assert keep(keep=0) == bad and keep(N=0) == unsupported and keep(page=8) == unsupported

    def att(q=p, H=4, T=3, ws=p, ws_bytes=0, **kw):
        return L.sage_paged_attention(_lib.PACK_ATTENTION(*kv(**kw), q, p, 0, 0, ws, ws_bytes, *st * 2, 0, 0, 0.0, 0, T, H), None)
    assert att(H=3) == unsupported and att(q=8) == bad and att(T=0) == unsupported and L.sage_paged_attention(None, None) == bad
    assert att(most=2 ** 27) == unsupported and b"positions must fit 32 bits" in L.sage_last_error()
    assert att(pages=2 ** 27) == unsupported and b"cache rows must fit 32 bits" in L.sage_last_error()
    need = L.sage_paged_attention_workspace_bytes(2, 3, 4, 2, 64)
    assert need > 0 and att(ws_bytes=need - 1) == bad and b"workspace" in L.sage_last_error()
    assert att(ws=0, ws_bytes=need) == bad and att(ws=264, ws_bytes=need) == bad
    for shape in ((0, 3, 4, 2, 64), (2, 3, 3, 2, 64), (2, 3, 4, 2, 80)):
        assert L.sage_paged_attention_workspace_bytes(*shape) == 0


def test_argument_structs_match_the_header(tmp_path):
    # the formats that Python packs, against the compiler's layout of the structs
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    fields = {"sage_rotary_args": ("positions", "q_st", "position_st", "dtype", "magnitude", "backward"),
              "sage_paged_rows_args": ("k", "k_st", "v_st", "dtype", "S"), "sage_paged_keep_args": ("keep", "keep_stride", "N"),
              "sage_paged_attention_args": ("q", "workspace_bytes", "mask_st", "sm_scale", "dtype", "H")}
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "sage_b200.h"\nint main(void) {\n' + "".join(
        f'printf("%zu ", offsetof({s}, {f}));\n' for s, fs in fields.items() for f in fs) + "return 0; }\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    size = struct.calcsize
    kv = _lib.PAGED_KV
    want = [size("4P"), size("6P"), size("6P12q"), size("6P14q"), size("6P14q9i"), size("6P14q9if"),
            size(kv), size(kv + "2P"), size(kv + "2P3q"), size(kv + "2P6q"), size(kv + "2P6qi"),
            size(kv), size(kv + "P"), size(kv + "Pq"),
            size(kv), size(kv + "5P"), size(kv + "5P7q"), size(kv + "5P9q"), size(kv + "5P9qd"), size(kv + "5P9qd2i")]
    assert got == want


def test_reference_codes_by_hand():
    # 64-bit rules of the cache that the GPU tests hold the kernels to: ties away from zero, special rows
    c, s = P.codes(torch.tensor([[2.0, 1.0, -1.0, 0.0], [0.0] * 4, [1.0, math.inf, 0, 0], [1e-37, 0, 0, 0]]), 127)
    assert c[0].tolist() == [127, 64, -64, 0] and s[0] == torch.tensor(2.0 / 127)
    assert c[1:].abs().sum() == 0 and s[1] == 0 and bool(s[2].isnan()) and s[3] == 0
    c, _ = P.codes(torch.tensor([[448.0, 17.0, -17.0, 0.0009765625]]), 448)
    assert c[0].tolist() == [448, 18, -18, 0.001953125]     # 17 lies between 16 and 18; 2^-10 between 0 and 2^-9
    assert ctypes.sizeof(ctypes.c_int) == 4


def test_a_leaf_of_an_older_graph_is_told_from_a_free_one():
    """The check of a captured gradient, which needs no GPU: `stream` is only compared."""
    from rdna4_sage import _rotary
    x = torch.randn(3, requires_grad=True)
    node = _rotary._accumulator(x, 7)                  # free
    assert _rotary._accumulator(x, 7) is node          # again in the same capture
    with pytest.raises(rdna4_sage.Unsupported, match="outside the capture"):
        _rotary._accumulator(x, 8)
    del node
    _rotary._accumulator(x, 8)
    y = x * 2
    for _ in range(2):                                 # a refusal leaves no mark that would let the next call through
        with pytest.raises(rdna4_sage.Unsupported, match="outside the capture"):
            _rotary._accumulator(x, 7)
    y.sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, 2.0))
    del y
    _rotary._accumulator(x, 7)
