"""The paged caches' keys and values in 64 bits, exact attention over them, and how far an output may be off."""
import numpy as np
import torch

from ffa_mi355x.paged import (CODES_ORDER, GSCALE_ORDER, K4_ORDER, PAGE, RES_ORDER, VT_ORDER, PagedQ2Cache, scale_pos,
                              to_logical)
from ffa_mi355x.paged_kfmt import PagedKfmtCache
from oracle import formats as OF

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative


def make_cache(fmt, P, HKV, dev, res=torch.float8_e4m3fn, v=torch.float16, seed=0):
    """A cache whose pools hold random bytes (NaN patterns among them) until pages are filled."""
    cache = (PagedQ2Cache(P, HKV, dev, res_dtype=res, v_dtype=v) if fmt == "q2"
             else PagedKfmtCache(fmt, P, HKV, dev, res_dtype=res, v_dtype=v))
    g = torch.Generator().manual_seed(seed + 100)
    for t in cache.pools():
        t.view(torch.uint8).copy_(torch.randint(0, 256, t.view(torch.uint8).shape, generator=g, dtype=torch.uint8))
    return cache


def fill(cache, k, v, table_row, start=0):
    """Append k, v [T, HKV, 128] of one sequence at position start."""
    dev = cache.v.device
    cache.append(k[None].to(dev), v[None].to(dev), torch.tensor([start], dtype=torch.int32, device=dev),
                 table_row[None].to(dev))


def _f8(t):
    return t.float().cpu().double().numpy()


def logical_kv(cache, fmt, pages, residual=True):
    """K, V [64 len(pages), HKV, 128] of the pages in 64 bits."""
    with np.errstate(invalid="ignore"):  # slots past the sequences hold anything
        return _logical_kv(cache, fmt, [int(p) for p in pages], residual)


def _logical_kv(cache, fmt, pages, residual):
    H = cache.HKV
    n = len(pages)
    if fmt == "q2":
        codes = to_logical(cache.k_q[pages].cpu().numpy(), CODES_ORDER, 8)  # [n, H, 4, 64, 8]
        c = ((codes[..., None] >> np.array([0, 2, 4, 6], dtype=np.uint8)) & 3).reshape(n, H, 4, PAGE, 32)
        sp = np.array([scale_pos(t) for t in range(PAGE)])
        s = to_logical(cache.k_scale[pages].cpu().numpy(), GSCALE_ORDER)[..., sp].astype(np.float64)
        z = to_logical(cache.k_zero[pages].cpu().numpy(), GSCALE_ORDER)[..., sp].astype(np.float64)
        k = (c * s[..., None] + z[..., None]).transpose(0, 3, 1, 2, 4).reshape(n * PAGE, H, 128)
    else:
        packed = to_logical(cache.k[pages].cpu().numpy(), K4_ORDER)  # [n, H, 64, 64]
        c = np.stack([packed & 15, packed >> 4], -1).reshape(n, H, PAGE, 128)
        s = _f8(cache.k_scale[pages].to(torch.float32))
        if fmt == "nvfp4":
            lv = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
            val = np.where(c & 8, -lv[c & 7], lv[c & 7])
        else:
            val = OF.NF4_CODEBOOK.astype(np.float64)[c]
        k = (val * np.repeat(s, 128 // s.shape[-1], axis=-1)).transpose(0, 2, 1, 3).reshape(n * PAGE, H, 128)
    if residual:
        r8 = to_logical(cache.k_res[pages].view(torch.uint8).cpu().numpy(), RES_ORDER)
        r = _f8(torch.from_numpy(r8.copy()).view(cache.k_res.dtype))
        k = k + r.transpose(0, 2, 1, 3).reshape(n * PAGE, H, 128)
    vt = to_logical(cache.v[pages].float().cpu().numpy(), VT_ORDER)  # [n, H, 128, 64]
    v = vt.transpose(0, 3, 1, 2).reshape(n * PAGE, H, 128).astype(np.float64)
    return k, v


def reference(q, k, v, T, ql, scale, tokens=None):
    """q [L, HQ, 128] (torch), k, v [>= T, HKV, 128] f64 -> (o, bound) [L, HQ, 128] f64; rows past ql are zeros.
    tokens: the query tokens to compute (default all; the others stay zeros).

    bound, by element, in units of the operands' arithmetic: each k is rounded once to fp16 (2^-11 relative, or
    2^-25 of the smallest normal), so a score is off by at most d = scale sum_c |q_c k_c| (2^-11 + 2^-17), the second
    part for 128 fp32 additions and products; weights change by a factor within e^(2 d), and their rounding to fp16
    by 2^-11 more (2^-20: the exponential, the sums and the stale maximum's 2^-25 absolute steps over the tokens)."""
    L, HQ, _ = q.shape
    G = HQ // k.shape[1]
    o = np.zeros((L, HQ, 128))
    bound = np.zeros((L, HQ, 128))
    qf = q.double().cpu().numpy()
    for i in range(min(ql, L)) if tokens is None else tokens:
        n = T - ql + i + 1
        if n <= 0:
            continue
        for h in range(HQ):
            kk, vv = k[:n, h // G], v[:n, h // G]
            s = scale * (kk @ qf[i, h])
            with np.errstate(invalid="ignore", over="ignore"):
                w = np.exp(s - s.max())
                w = w / w.sum()
                o[i, h] = w @ vv
                d = abs(scale) * (np.abs(kk) @ np.abs(qf[i, h])).max() * (2.0 ** -11 + 2.0 ** -17) + n * 2.0 ** -25
                bound[i, h] = (np.expm1(2 * d) + 2.0 ** -11 + 2.0 ** -20) * (w @ np.abs(vv)) + n * 2.0 ** -25 * 2.0 ** -8
    return o, bound


def assert_close(out, o, bound, dtype, what=""):
    got = out.double().cpu().numpy()
    limit = bound + U[dtype] * (np.abs(o) + bound) + 2.0 ** -25
    same = (np.isnan(o) & np.isnan(got)) | (np.isinf(o) & (o == got))
    with np.errstate(invalid="ignore"):
        bad = ~same & ~(np.abs(got - o) <= limit)
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} beyond the bound, first at {np.argwhere(bad)[0]}, "
                           f"got {got[bad][0]} want {o[bad][0]} +- {limit[bad][0]}")
