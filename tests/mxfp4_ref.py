"""The MXFP4 cache's definition in 64 bits: the values that blocks are held as, the pages' order, rotary positions."""
import numpy as np
import torch

from ffa_mi355x.paged_mxfp4 import PAGE, PagedMXFP4Cache

LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
VALUES = np.concatenate([LEVELS, -LEVELS])
LOW, HIGH, NAN = 105, 140, 255

_t, _c = np.arange(PAGE)[:, None], np.arange(128)[None, :]
# byte of token t, channel c in a (page, KV head) block, and which half of the byte
K_BYTE = ((_t % 4 * 4 + _c // 32) * 16 + _t // 4) * 16 + _c % 32 // 2
K_HALF = np.broadcast_to(_c % 2, K_BYTE.shape)
V_BYTE = ((_c // 32 * 4 + _t // 16) * 16 + _c % 16) * 16 + _c // 16 % 2 * 8 + _t % 16 // 2
V_HALF = np.broadcast_to(_t % 2, V_BYTE.shape)


def quantize(x):
    """x [..., 128] (numpy, any float) -> codes [..., 128], scale bytes [..., 4]."""
    b = np.asarray(x, dtype=np.float64).reshape(x.shape[:-1] + (4, 32))
    with np.errstate(invalid="ignore"):
        top = np.abs(b).max(-1)
    byte = np.full(top.shape, LOW)
    for e in range(LOW, HIGH):  # the smallest power of two of which the largest magnitude is at most seven
        byte = np.where(top > 7 * 2.0 ** (e - 127), e + 1, byte)
    bad = ~np.isfinite(b).all(-1)
    byte = np.where(bad, NAN, byte)
    y = np.where(bad[..., None], 0, np.where(bad[..., None], 0, b) / 2.0 ** (np.where(bad, 127, byte)[..., None] - 127.0))
    code = np.zeros(y.shape, dtype=np.int64)
    for i in range(7):  # past a midpoint; on it to the even code
        mid = (LEVELS[i] + LEVELS[i + 1]) / 2
        code = np.where((np.abs(y) >= mid) if i % 2 else (np.abs(y) > mid), i + 1, code)
    code = code + 8 * np.signbit(y)
    return code.reshape(x.shape), byte


def values(code, byte):
    s = np.where(byte == NAN, np.nan, 2.0 ** (byte.astype(np.float64) - 127))
    return VALUES[code] * np.repeat(s, 32, axis=-1)


def held(x):
    return values(*quantize(x))


def codes_of(pools, pages):
    """Codes [n 64, HKV, 128] and scale bytes [n 64, HKV, 4] of K and of V in the pages: pools in numpy."""
    out = []
    for name, at, half in (("k", K_BYTE, K_HALF), ("v", V_BYTE, V_HALF)):
        raw = pools[name][pages].reshape(len(pages), -1, 4096)  # [n, H, 4096]
        code = (raw[:, :, at] >> (4 * half)) & 15  # [n, H, 64, 128]
        byte = pools[name + "_scale"][pages]  # [n, H, 4, 64]
        H = raw.shape[1]
        out.append((code.transpose(0, 2, 1, 3).reshape(-1, H, 128).astype(np.int64),
                    byte.transpose(0, 3, 1, 2).reshape(-1, H, 4).astype(np.int64)))
    return out


def write(pools, page, t, name, code, byte):
    """Token t of a page: code [HKV, 128] and byte [HKV, 4] into the numpy pools."""
    at, half = (K_BYTE[t], K_HALF[t]) if name == "k" else (V_BYTE[t], V_HALF[t])
    flat = pools[name][page].reshape(-1, 4096)
    for c in range(128):
        keep = 0xF0 if half[c] == 0 else 0x0F
        flat[:, at[c]] = (flat[:, at[c]] & keep) | (code[:, c] << (4 * half[c])).astype(np.uint8)
    pools[name + "_scale"][page][:, :, t] = byte


def to_numpy(cache):
    return {n: getattr(cache, n).cpu().numpy().copy() for n in ("k", "k_scale", "v", "v_scale")}


def make_cache(P, HKV, dev, seed=0, scales=True):
    """A cache whose pools hold random bytes (blocks of NaN among them) until pages are filled."""
    cache = PagedMXFP4Cache(P, HKV, dev)
    g = torch.Generator().manual_seed(seed + 100)
    for t in cache.pools():
        t.copy_(torch.randint(0, 256, t.shape, generator=g, dtype=torch.uint8))
    return cache


def logical_kv(cache, pages):
    (kc, kb), (vc, vb) = codes_of(to_numpy(cache), [int(p) for p in pages])
    with np.errstate(over="ignore"):
        return values(kc, kb), values(vc, vb)


def rotate(x, positions, axis, freq, adjacent, inverse=False):
    """x [B, T, H, 128] turned in 64 bits; positions [axes, B, T]."""
    x = np.asarray(x, dtype=np.float64)
    out = np.empty_like(x)
    for j in range(64):
        a = np.asarray(positions[axis[j]], dtype=np.float64) * freq[j]
        a = -a if inverse else a
        c, s = np.cos(a)[..., None], np.sin(a)[..., None]
        m, n = (2 * j, 2 * j + 1) if adjacent else (j, j + 64)
        out[..., m] = x[..., m] * c - x[..., n] * s
        out[..., n] = x[..., n] * c + x[..., m] * s
    return out


def turn_bound(x, adjacent):
    """How far the turn may leave an element from the 64-bit one: sine and cosine are rounded to fp32 once (2^-25; before
    that they are within 2^-40, and the angle, at positions up to 2^20, within 2^-30), the two products and their sum once
    each (2^-24 of |a| + |b| for the products together, and as much for the sum)."""
    a = np.abs(np.asarray(x, dtype=np.float64))
    if adjacent:
        s = np.repeat(a[..., ::2] + a[..., 1::2], 2, axis=-1)
    else:
        s = np.concatenate([a[..., :64] + a[..., 64:]] * 2, -1)
    return s * (2.0 ** -25 + 2.0 ** -23 + 2.0 ** -29)
