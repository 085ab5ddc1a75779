"""Exact attention over the paged caches: what the host decides, on the CPU (plans of shared pages, refusals)."""
import ctypes

import pytest
import torch

from ffa_mi355x import _native as N
from ffa_mi355x.attend import SharedPrefix

I = torch.int32


def test_shared_prefix_plan():
    table = torch.tensor([[5, 6, 7, 1], [5, 6, 8, 2], [5, 9, 7, 3], [4, 6, 7, 1]], dtype=I)
    lens = torch.tensor([200, 200, 200, 200], dtype=I)
    plan = SharedPrefix(table, lens)
    assert plan.sizes == [3, 1] and plan.pages == [1, 0]
    plan = SharedPrefix(table, lens, group_sizes=[2, 2])
    assert plan.pages == [2, 0]
    assert plan._dev.tolist() == [0, 2, 4, 2, 0, 0, 0, 1, 1]
    # shared pages lie wholly inside every member
    assert SharedPrefix(table, torch.tensor([200, 127, 200, 64], dtype=I), group_sizes=[2, 2]).pages == [1, 0]
    # ids past the lengths are not data: rows of equal padding do not belong together
    assert SharedPrefix(torch.zeros((3, 2), dtype=I), torch.tensor([0, 0, 10], dtype=I)).sizes == [1, 1, 1]
    one = SharedPrefix(table[:1], lens[:1])
    assert one.sizes == [1] and one.pages == [0] and len(one) == 1


@pytest.mark.parametrize("sizes", [[3], [5], [4, 0], [2, -1, 3], []])
def test_shared_prefix_refuses(sizes):
    with pytest.raises(ValueError):
        SharedPrefix(torch.zeros((4, 2), dtype=I), torch.full((4,), 100, dtype=I), group_sizes=sizes)


def test_shared_prefix_refuses_shapes():
    with pytest.raises(ValueError):
        SharedPrefix(torch.zeros(4, dtype=I), torch.zeros(4, dtype=I))
    with pytest.raises(ValueError):
        SharedPrefix(torch.zeros((4, 2), dtype=I), torch.zeros(3, dtype=I))
    with pytest.raises(ValueError):
        SharedPrefix(torch.zeros((0, 2), dtype=I), torch.zeros(0, dtype=I))


def _args(**kw):
    a = N.AttendArgs()
    a.q = a.k = a.k_scale = a.k_zero = a.k_residual = a.v = a.block_table = a.out = 4096
    a.q_dtype, a.v_dtype, a.res_dtype, a.format = N.DT_BF16, N.DT_F16, N.DT_FP8_E4M3, N.PAGES_Q2
    a.B, a.T, a.L, a.HQ, a.HKV, a.bt_stride, a.num_pages, a.scale = 2, 128, 1, 8, 2, 2, 4, 1.0
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw", [
    dict(B=0), dict(T=0), dict(L=0), dict(HQ=0), dict(HKV=0), dict(HQ=7), dict(T=129), dict(bt_stride=0),
    dict(num_pages=0), dict(q_dtype=N.DT_F32), dict(v_dtype=N.DT_F32), dict(format=3), dict(format=-1),
    dict(res_dtype=N.DT_F16), dict(q=None), dict(k=None), dict(k_scale=None), dict(k_zero=None), dict(k_residual=None),
    dict(v=None), dict(block_table=None), dict(out=None), dict(q=4098), dict(out=4104), dict(v=4100), dict(ngroups=-1),
    dict(ngroups=3), dict(ngroups=1), dict(scratch_bytes=0, T=12800, bt_stride=200),
])
def test_c_entry_refuses(kw):
    rc = N.lib().ffa_paged_attend(ctypes.byref(_args(**kw)), None)
    assert rc == -1, N.lib().ffa_last_error()


@pytest.mark.parametrize("kw", [dict(B=65536), dict(HKV=65536, HQ=65536), dict(T=(1 << 30) + 64, bt_stride=1 << 25), dict(L=1 << 29, HQ=8)])
def test_c_entry_unsupported(kw):
    a = _args(**kw)
    assert N.lib().ffa_paged_attend(ctypes.byref(a), None) == -2


@pytest.mark.parametrize("start,pages", [([0, 1, 3], [1, 1]), ([1, 2, 2], [1, 1]), ([0, 0, 2], [1, 1]), ([0, 1, 2], [3, 0]),
                                         ([0, 1, 2], [-1, 0])])
def test_c_entry_refuses_groups(start, pages):
    s, p = (ctypes.c_int32 * 3)(*start), (ctypes.c_int32 * 2)(*pages)
    a = _args(ngroups=2, group_start=4096, group_pages=4096, seq_group=4096, group_start_host=ctypes.addressof(s),
              group_pages_host=ctypes.addressof(p))
    assert N.lib().ffa_paged_attend(ctypes.byref(a), None) == -1
    assert N.lib().ffa_paged_attend_scratch(ctypes.byref(a)) == 0


def test_scratch_sizes():
    L = N.lib()
    assert L.ffa_paged_attend_scratch(ctypes.byref(_args())) == 0  # one range of pages a row: no partials
    long = _args(T=64 * 4000, bt_stride=4000)
    need = L.ffa_paged_attend_scratch(ctypes.byref(long))
    assert need > 0 and need % (2 * 8 * 130 * 4) == 0
    assert L.ffa_paged_attend_scratch(None) == 0


def test_argument_struct_matches_header(tmp_path):
    from test_native_abi import test_ctypes_argument_structs_match_header as check

    check(tmp_path, "ffa_paged_attend_args", "AttendArgs")
