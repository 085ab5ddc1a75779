"""The cache of keys and values in 4 bits and rotary positions with several axes: what the host decides, on the CPU."""
import ctypes

import numpy as np
import pytest
import torch

import mxfp4_ref as R
from ffa_mi355x import _native as N
from ffa_mi355x.paged_mxfp4 import PagedMXFP4Cache
from ffa_mi355x.rope_axes import AxisRope, strided_rows

I = torch.int32


def test_pairs_of_axes():
    r = AxisRope((16, 24, 24), device="cpu")
    assert r.axis == [0] * 16 + [1] * 24 + [2] * 24 and r.axes == 3
    r = AxisRope((24, 20, 20), device="cpu", order="cycled")
    assert r.axis == [0, 1, 2] * 20 + [0] * 4
    r = AxisRope((62, 1, 1), device="cpu", order="cycled")
    assert r.axis == [0, 1, 2] + [0] * 61
    r = AxisRope((64,), base=500.0, device="cpu")
    assert r.inv_freq[0] == 1.0 and abs(r.inv_freq[32] - 500.0 ** -0.5) < 1e-16
    turns = r.table[:, 0].view(torch.float64)
    assert torch.allclose(turns * 2 * np.pi, torch.tensor(r.inv_freq, dtype=torch.float64), rtol=1e-15)
    assert r.table[:, 1].tolist() == [0] * 64
    f = torch.rand(64)
    assert AxisRope((64,), device="cpu", inv_freq=f).inv_freq == f.double().tolist()


@pytest.mark.parametrize("args,kw", [
    (((16, 24, 23),), {}), (((65,),), {}), ((()  ,), {}), (((70, -6),), {}), (((64,),), dict(pairs="both")),
    (((64,),), dict(order="mixed")), (((64,),), dict(base=0.0)), (((64,),), dict(inv_freq=[1.0] * 32)),
])
def test_rope_refuses(args, kw):
    with pytest.raises(ValueError):
        AxisRope(*args, device="cpu", **kw)


def test_positions():
    r = AxisRope((32, 32), device="cpu")
    cpu = torch.device("cpu")
    p = torch.arange(2 * 3 * 5).view(2, 3, 5)
    got, a, b = r._positions(p, 3, 5, cpu)
    assert got is p and (a, b) == (15, 5)
    got, a, b = r._positions(p[:, 1], 3, 5, cpu)  # for every sequence
    assert b == 0 and torch.equal(got, p[:, 1:2].expand(2, 3, 5))
    got, a, b = r._positions(p.transpose(1, 2).contiguous().transpose(1, 2), 3, 5, cpu)  # tokens apart: copied
    assert got.stride(2) == 1 and torch.equal(got, p)
    got, _, _ = AxisRope((64,), device="cpu")._positions(p[0], 3, 5, cpu)
    assert torch.equal(got[0], p[0])
    for bad in (p.float(), p[:1], p[:, :2], p[..., :4], p[0]):
        with pytest.raises(ValueError):
            r._positions(bad, 3, 5, cpu)


def test_strided_rows():
    x = torch.zeros(2, 7, 3, 512)
    a, s = strided_rows(x[..., 128:256])
    assert a.data_ptr() == x[..., 128:].data_ptr() and s == (7 * 3 * 512, 3 * 512, 512)
    a, s = strided_rows(x[:, :1, :, :128])  # one token: its stride does not count
    assert s == (7 * 3 * 512, 0, 512)
    a, s = strided_rows(x[..., 2:130])  # not a multiple of 16 bytes
    assert a.data_ptr() % 16 == 0 and a.is_contiguous()
    a, s = strided_rows(x[..., ::4])
    assert a.is_contiguous()
    a, s = strided_rows(torch.zeros(2, 7, 3, 130)[..., :128])
    assert a.is_contiguous() and s == (7 * 3 * 128, 3 * 128, 128)
    a, s = strided_rows(torch.zeros(2, 1, 3, 128).expand(2, 7, 3, 128))
    assert s == (3 * 128, 0, 128)


def test_reference_values():
    """The definition against values worked out by hand, so that the other tests compare with the right thing."""
    x = np.zeros((1, 128))
    x[0, :8] = [7, 3.5, -2.5, 0.25, 0.75, 1.25, 1.75, 5]
    x[0, 32], x[0, 33] = 7.0001, 1.0
    x[0, 64] = 2.0 ** -40
    x[0, 96:98] = 1e30, -40000.0
    code, byte = R.quantize(x)
    assert byte.tolist() == [[127, 128, 105, 140]]
    assert R.values(code, byte)[0, :8].tolist() == [6, 4, -2, 0, 1, 1, 2, 4]
    assert R.values(code, byte)[0, [32, 33, 64]].tolist() == [8, 1, 0]
    assert R.values(code, byte)[0, 96:98].tolist() == [49152, -32768]  # on the midpoint of 4 and 6: the even code
    x[0, 5] = np.nan
    x[0, 70] = -np.inf
    code, byte = R.quantize(x)
    assert byte.tolist() == [[255, 128, 255, 140]] and (code[0, :32] == 0).all()
    assert np.isnan(R.held(x)[0, :32]).all() and np.isfinite(R.held(x)[0, 32:64]).all()
    # every place of a page once
    for b, h in ((R.K_BYTE, R.K_HALF), (R.V_BYTE, R.V_HALF)):
        assert sorted((2 * b + h).ravel().tolist()) == list(range(8192))


def test_layout_matches_the_kernels(tmp_path):
    """mx_k_off / mx_v_off of csrc/mxfp4.h give the places of the definition."""
    import re
    import shutil
    import subprocess
    from pathlib import Path

    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host compiler")
    text = (Path(__file__).resolve().parents[1] / "ffa-speedtest_amd" / "csrc" / "mxfp4.h").read_text()
    fns = re.findall(r"__host__ __device__ (constexpr uint32_t mx_[kv]_off\(.*?\n\})", text, flags=re.S)
    assert len(fns) == 2
    src = tmp_path / "o.cpp"
    src.write_text("#include <cstdint>\n#include <cstdio>\n" + "\n".join(fns) + """
int main() {
  for (int t = 0; t < 64; ++t) for (int c = 0; c < 128; ++c) printf("%u %u\\n", mx_k_off(t, c / 8) + c % 8 / 2, mx_v_off(c, t));
}""")
    subprocess.run([cxx, "-std=c++17", str(src), "-o", str(tmp_path / "o")], check=True)
    got = np.array([list(map(int, l.split())) for l in subprocess.run([str(tmp_path / "o")], check=True, capture_output=True,
                                                                       text=True).stdout.splitlines()]).reshape(64, 128, 2)
    assert (got[..., 0] == R.K_BYTE).all() and (got[..., 1] == R.V_BYTE).all()


def test_argument_structs_match_header(tmp_path):
    from test_native_abi import test_ctypes_argument_structs_match_header as check

    check(tmp_path, "ffa_rope_axes_args", "RopeAxesArgs")
    check(tmp_path, "ffa_mxfp4_append_args", "MXFP4AppendArgs")


def _rope_args(**kw):
    a = N.RopeAxesArgs()
    a.q = a.q_out = a.k = a.k_out = a.pairs = a.positions = 4096
    a.dtype, a.B, a.T, a.HQ, a.HKV, a.axes = N.DT_BF16, 2, 3, 8, 2, 3
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw", [
    dict(B=0), dict(T=0), dict(HQ=0), dict(HKV=-1), dict(axes=0), dict(q=None), dict(q_out=None), dict(k=None),
    dict(k_out=None), dict(pairs=None), dict(positions=None), dict(dtype=N.DT_FP8_E4M3), dict(dtype=-1), dict(q=4104),
    dict(k_out=4098), dict(q_token=4), dict(k_out_head=1), dict(dtype=N.DT_F32, q_batch=2),
])
def test_rope_entry_refuses(kw):
    assert N.lib().ffa_rope_axes(ctypes.byref(_rope_args(**kw)), None) == -1, N.lib().ffa_last_error()


def test_rope_entry_unsupported():
    assert N.lib().ffa_rope_axes(ctypes.byref(_rope_args(HQ=1 << 21)), None) == -2
    assert N.lib().ffa_rope_axes(None, None) == -1


def test_calls_beyond_a_grid():
    """More workgroups than a grid of 2^32 threads holds."""
    assert N.lib().ffa_rope_axes(ctypes.byref(_rope_args(B=1 << 14, T=1 << 15)), None) == -2
    assert N.lib().ffa_mxfp4_append(ctypes.byref(_append_args(B=1 << 25, T=1)), None) == -2
    assert N.lib().ffa_mxfp4_append(ctypes.byref(_append_args(B=1 << 18, T=1 << 13, pairs=None, HQ=0, q=None)), None) == -2
    assert N.lib().ffa_mxfp4_dequant(4096, 4096, 4096, 4096, 4096, 2, 4, None, 1 << 24, 64, 2, 4096, 4096, N.DT_F16, None) == -2


def _append_args(**kw):
    a = N.MXFP4AppendArgs()
    a.k = a.v = a.q = a.pairs = a.pos = a.block_table = a.k_pages = a.k_scale = a.v_pages = a.v_scale = a.q_out = 4096
    a.k_values = a.v_values = 4096
    a.dtype, a.B, a.T, a.HKV, a.HQ, a.bt_stride, a.num_pages = N.DT_F16, 2, 3, 2, 8, 2, 4
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw", [
    dict(B=0), dict(T=0), dict(HKV=0), dict(HQ=-1), dict(bt_stride=0), dict(num_pages=0), dict(k=None), dict(pos=None),
    dict(block_table=None), dict(k_pages=None), dict(k_scale=None), dict(v_pages=None), dict(v_scale=None), dict(q=None),
    dict(q_out=None), dict(pairs=None), dict(positions=4096, axes=0), dict(v=None), dict(dtype=N.DT_NONE), dict(k=4100),
    dict(v_values=4104), dict(k_pages=4097), dict(v_token=3), dict(dtype=N.DT_F32, q_head=6),
])
def test_append_entry_refuses(kw):
    assert N.lib().ffa_mxfp4_append(ctypes.byref(_append_args(**kw)), None) == -1, N.lib().ffa_last_error()


@pytest.mark.parametrize("kw", [dict(T=(1 << 30) + 1), dict(HKV=1 << 17), dict(HQ=1 << 21), dict(B=1 << 20, T=1 << 20)])
def test_append_entry_unsupported(kw):
    assert N.lib().ffa_mxfp4_append(ctypes.byref(_append_args(**kw)), None) == -2


@pytest.mark.parametrize("kw,rc", [
    (dict(B=0), -1), (dict(T=0), -1), (dict(T=65), -1), (dict(HKV=0), -1), (dict(bt=1), -1), (dict(P=0), -1), (dict(dt=5), -1),
    (dict(k=None), -1), (dict(vo=None), -1), (dict(ko=4104), -1), (dict(HKV=1 << 16), -2), (dict(B=1 << 30), -2),
])
def test_dequant_entry_refuses(kw, rc):
    a = dict(k=4096, ko=4096, vo=4096, bt=2, P=4, B=2, T=128, HKV=2, dt=N.DT_F16, **{})
    a.update(kw)
    assert N.lib().ffa_mxfp4_dequant(a["k"], 4096, 4096, 4096, 4096, a["bt"], a["P"], None, a["B"], a["T"], a["HKV"], a["ko"],
                                     a["vo"], a["dt"], None) == rc


def _attend_args(**kw):
    a = N.AttendArgs()
    a.q = a.k = a.k_scale = a.v = a.block_table = a.out = 4096
    a.q_dtype, a.v_dtype, a.res_dtype, a.format = N.DT_BF16, N.DT_NONE, N.DT_NONE, N.PAGES_MXFP4
    a.B, a.T, a.L, a.HQ, a.HKV, a.bt_stride, a.num_pages, a.scale = 2, 128, 1, 8, 2, 2, 4, 1.0
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw", [
    dict(B=0), dict(T=129), dict(HQ=7), dict(q_dtype=N.DT_F32), dict(v_dtype=N.DT_F16), dict(format=N.PAGES_Q2),
    dict(format=4), dict(res_dtype=N.DT_FP8_E4M3), dict(k_zero=4096), dict(k_residual=4096), dict(v=None), dict(v=4100),
    dict(scratch_bytes=0, T=12800, bt_stride=200), dict(ngroups=1),
])
def test_attend_entry_refuses(kw):
    assert N.lib().ffa_mxfp4_attend(ctypes.byref(_attend_args(**kw)), 4096, None) == -1, N.lib().ffa_last_error()


def test_attend_entries_keep_to_their_formats():
    """The other formats' entry takes no mxfp4 pages, nor this one a call without V's scales."""
    L, a = N.lib(), _attend_args(v_dtype=N.DT_F16)
    assert L.ffa_paged_attend(ctypes.byref(a), None) == -1
    assert L.ffa_mxfp4_attend(ctypes.byref(_attend_args()), None, None) == -1
    assert L.ffa_mxfp4_attend(ctypes.byref(_attend_args()), 4100, None) == -1
    assert L.ffa_mxfp4_attend_scratch(ctypes.byref(_attend_args()), None) == 0
    long = _attend_args(T=64 * 4000, bt_stride=4000)
    need = L.ffa_mxfp4_attend_scratch(ctypes.byref(long), 4096)
    assert need > 0 and need % (2 * 8 * 130 * 4) == 0


def test_cache_refuses_on_the_cpu():
    cache = PagedMXFP4Cache(4, 2, "cpu")
    assert cache.nbytes_per_page() == 2 * 64 * 136 and [t.shape[0] for t in cache.pools()] == [4] * 4
    k = torch.zeros(1, 3, 2, 128)
    pos, table = torch.zeros(1, dtype=I), torch.zeros(1, 2, dtype=I)
    for bad in (k[..., :64], k[:, :, :1], k[0]):
        with pytest.raises(ValueError):
            cache.append(bad, bad, pos, table)
    with pytest.raises(ValueError):
        cache.append(k, k[:, :2], pos, table)
    with pytest.raises(NotImplementedError):
        cache.append(k.double(), k.double(), pos, table)
    with pytest.raises(ValueError):  # no CPU path
        cache.append(k, k, pos, table)
    with pytest.raises(ValueError):
        cache.dequantize(table, 64)
    with pytest.raises(NotImplementedError):
        cache.dequantize(table, 64, out_dtype=torch.float64)
    with pytest.raises(ValueError):
        cache.attend(k.half()[:, :1], table, torch.ones(1, dtype=I))
    with pytest.raises(ValueError):
        AxisRope((64,), device="cpu").rotate(torch.zeros(1, 1, 3, dtype=I), k)
