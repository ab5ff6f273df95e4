"""Lengths and counts outside their range leave a sequence of the paged cache as it was, whole: no token of it lands in its
context.  (test_gpu_paged_kv.py has those for which every position is outside.)"""
import pytest
import torch

import paged_reference as P
import rdna4_sage
from rdna4_sage import _attention
from test_gpu_paged_kv import filled, handle, ints, queries, same_cache

pytestmark = pytest.mark.gpu
LENS = [30, 40, 10]


def raises():
    with pytest.raises(RuntimeError, match="invalid argument"):
        _attention.check_status(torch.device("cuda", 0))


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("lens,counts", [([30, -1, 10], None), ([30, -3, 10], None), ([30, -2, 10], [4, 4, 4]),
                                         ([30, -2 ** 31, 10], None), (LENS, [4, 5, 4]), (LENS, [4, 2 ** 31 - 1, 4]),
                                         (LENS, [4, -1, 4]), ([30, -1, 10], [4, 5, 4])])
def test_append_of_a_bad_sequence_writes_none_of_it(D, lens, counts):
    T = 4
    cache, table = filled(LENS, T, 16, 2, D)
    k, v = queries(3, T, 2, D), queries(3, T, 2, D, seed=8)
    want = {n: x.clone() for n, x in cache.items()}
    P.append(want, k[[0, 2]], v[[0, 2]], table[[0, 2]], [30, 10])
    rdna4_sage.paged_kv_append(handle(cache), k, v, table, ints(lens), None if counts is None else ints(counts), "NHD")
    raises()
    same_cache(cache, want)


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("length,counts", [(-1, None), (-2, None), (-1, [3, 2, 3]), (-2 ** 31, None)])
def test_keep_of_a_bad_length_moves_nothing(D, length, counts):
    cache, table = filled(LENS, 4, 16, 2, D)
    want = {n: x.clone() for n, x in cache.items()}
    for b in (0, 2):
        for i, j in enumerate((1, 2, 3)):
            (p0, r0), (p1, r1) = P.place(want, table, b, [LENS[b] + j]), P.place(want, table, b, [LENS[b] + i])
            for name in want:
                w = want[name].view(torch.uint8) if name == "v8" else want[name]
                w[p1, :, r1] = w[p0, :, r0]
    rdna4_sage.paged_kv_keep(handle(cache), table, ints([30, length, 10]), ints([[1, 2, 3]] * 3),
                             None if counts is None else ints(counts))
    raises()
    same_cache(cache, want)
