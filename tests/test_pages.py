"""Page management: what the host decides, on the CPU (refusals of the C entries and of PagePool)."""
import ctypes

import pytest
import torch

from ffa_mi355x import _native as N
from ffa_mi355x.pages import PagePool
from ffa_mi355x.paged import PagedQ2Cache


def _pages(ptrs=(4096, 8192), sizes=(64, 32), **kw):
    p = (ctypes.c_void_p * len(ptrs))(*ptrs)
    b = (ctypes.c_size_t * len(sizes))(*sizes)
    pg = N.Pages(ctypes.addressof(p), ctypes.addressof(b), len(ptrs), 16, 4096)
    for k, v in kw.items():
        setattr(pg, k, v)
    pg._keep = (p, b)
    return pg


X = 4096  # an address that no refused call reads


@pytest.mark.parametrize("pg,rc", [
    (dict(npools=0), -1), (dict(pools=None), -1), (dict(page_bytes=None), -1), (dict(num_pages=0), -1),
    (dict(num_pages=(1 << 28) + 1), -2), (dict(refs=None), -1), (dict(refs=4100), -1), (dict(ptrs=(4096, 0)), -1),
    (dict(ptrs=(4096, 4104)), -1), (dict(sizes=(64, 0)), -1), (dict(sizes=(64, 40)), -1), (dict(sizes=(64, 1 << 31)), -2),
])
def test_pools_refused(pg, rc):
    L, p = N.lib(), ctypes.byref(_pages(**pg))
    assert L.ffa_pages_copy(p, X, X, 1, None) == rc
    assert L.ffa_pages_fork(p, X, 4, 1, X, X, 1, 2 * X, X, X, None) == rc
    assert L.ffa_pages_extend(p, X, 4, 1, X, 1, X, X, None) == rc
    assert L.ffa_pages_count(p, X, 4, 1, X, 1, X, X, None) == rc
    assert L.ffa_pages_compact(p, None, None, 0, X, None) == rc


def test_calls_refused():
    L, pg = N.lib(), _pages()
    p = ctypes.byref(pg)
    assert L.ffa_pages_copy(p, None, X, 1, None) == -1
    assert L.ffa_pages_copy(p, X, X, -1, None) == -1
    assert L.ffa_pages_copy(p, None, None, 0, None) == 0  # nothing to do, nothing launched
    for kw, rc in ((dict(table=None), -1), (dict(cols=0), -1), (dict(lens=None), -1), (dict(rows=0), -1), (dict(err=None), -1),
                   (dict(rows=65536), -2), (dict(cols=(1 << 24) + 1), -2)):
        a = dict(table=X, cols=4, lens=X, rows=2, err=X) | kw
        assert L.ffa_pages_fork(p, a["table"], a["cols"], 1, a["lens"], X, a["rows"], 2 * X, X, a["err"], None) == rc
        assert L.ffa_pages_extend(p, a["table"], a["cols"], a["rows"], a["lens"], 1, X, a["err"], None) == rc
        assert L.ffa_pages_count(p, a["table"], a["cols"], a["rows"], a["lens"], 1, X, a["err"], None) == rc
    assert L.ffa_pages_fork(p, X, 4, 0, X, X, 1, 2 * X, X, X, None) == -1
    assert L.ffa_pages_fork(p, X, 4, 1, X, None, 1, 2 * X, X, X, None) == -1
    assert L.ffa_pages_fork(p, X, 4, 1, X, X, 1, X, X, X, None) == -1  # children into the parents' table
    assert L.ffa_pages_extend(p, X, 4, 1, X, -1, X, X, None) == -1
    assert L.ffa_pages_extend(p, X, 1 << 24, 65535, X, 1 << 30, X, X, None) == -2  # more pages than the ranks count
    assert L.ffa_pages_count(p, X, 4, 1, X, 2, X, X, None) == -1
    assert L.ffa_pages_count(p, X, 4, 1, X, 1, None, X, None) == -1
    assert L.ffa_pages_compact(p, None, None, 1, X, None) == -1
    assert L.ffa_pages_compact(p, None, None, 0, None, None) == -1
    t = (ctypes.c_void_p * 9)(*[X] * 9)
    n = (ctypes.c_size_t * 9)(*[1] * 9)
    assert L.ffa_pages_compact(p, ctypes.addressof(t), ctypes.addressof(n), 9, X, None) == -2


def test_scratch_words():
    L = N.lib()
    assert [L.ffa_pages_alloc_scratch(*x) for x in ((1, 0), (5, 1), (5, 64), (5, 65), (0, 1), (1, -1))] == [3, 12, 12, 17, 0, 0]
    assert L.ffa_pages_alloc_scratch(1, 2 ** 31 - 1) == 2 + (2 ** 31 + 62) // 64 + 1
    assert [L.ffa_pages_compact_scratch(x) for x in (0, 1, 64)] == [0, 5, 132]


def test_pool_needs_gpu_caches():
    with pytest.raises(ValueError):
        PagePool([])
    with pytest.raises(ValueError):
        PagePool([PagedQ2Cache(2, 1, "cpu")])


def test_argument_struct_matches_header(tmp_path):
    from test_native_abi import test_ctypes_argument_structs_match_header as check

    check(tmp_path, "ffa_pages", "Pages")
    assert torch.int32.itemsize == 4
