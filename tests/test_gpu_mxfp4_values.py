"""Exact attention over mxfp4 pages: V whose powers of two lie far apart counts in full, whichever kernel takes the rows.

Keys are signs and queries are signs, so that every score is a whole number of log2 units that all of the arithmetic holds
exactly, and what is left are the weights' rounding and the sums.
"""
import math

import numpy as np
import pytest
import torch

import mxfp4_ref as R
from attend_ref import U, assert_close, reference
from ffa_mi355x.attend import SharedPrefix
from ffa_mi355x.paged_mxfp4 import PagedMXFP4Cache

pytestmark = pytest.mark.gpu
LN2 = math.log(2)
# query tokens, heads of the one KV head, and copies of the sequence: 4 rows, 20 by sixteens and as they are, 300 by sixteens (or
# 64), 40, 100 and 300 rows as they are
KERNELS = [(1, 4, 1), (5, 4, 1), (5, 4, 300), (150, 2, 1), (40, 1, 300), (100, 1, 150), (150, 2, 60)]


def _signs(g, *shape):
    return torch.where(torch.rand(shape, generator=g) < 0.5, -1.0, 1.0)


def _cache(g, k, v, dev, copies):
    """A cache of one sequence k, v [n, 1, 128] on scattered pages, its table and length as often as said."""
    n = k.shape[0]
    pages = -(-n // 64)
    cache = R.make_cache(pages + 2, 1, dev, seed=7)
    table = torch.randperm(pages + 2, generator=g)[:pages].to(torch.int32)[None].to(dev)
    cache.append(k[None].to(dev), v[None].to(dev), torch.zeros(1, dtype=torch.int32, device=dev), table)
    return cache, table.repeat(copies, 1), torch.full((copies,), n, dtype=torch.int32, device=dev)


def _bound(w, v):
    """Of weights w (in 64 bits, their sum one) and v [n, 128]: each weight is rounded to fp16 (2^-11 of it; below fp16's normal
    numbers half a step, 2^-25, where the largest weight is 2^8 or more, and no more than the weight itself), the sum of them
    as they are rounded stands below the fraction bar; 2^-13 for exponentials of arguments up to 2^9 in fp32 and the sums."""
    steps = np.minimum(w, 2.0 ** -33)
    a = np.abs(v)
    return (2.0 ** -10 + 2.0 ** -13) * (w @ a) + steps @ a + steps.sum() * (w @ a)


def _close(got, k, q, v, limit, dtype, scale):
    """got [128] against attention of q [128] over the first `limit` of k, v (numpy)."""
    s = scale * (k[:limit] @ q)
    w = np.exp(s - s.max())
    w /= w.sum()
    o, b = w @ v[:limit], _bound(w, v[:limit])
    assert (np.abs(o) > 2 * b).mean() > 0.5  # zeros would not pass
    low = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -100
    off = np.abs(got.double().cpu().numpy() - o) - (b + U[dtype] * (np.abs(o) + b) + low)
    assert (off <= 0).all(), (float(off.max()), o[off.argmax()], got[int(off.argmax())])


def _rows(L, copies):
    return [(b, i) for b in sorted({0, copies // 2, copies - 1}) for i in sorted({0, L // 2, L - 1})]


@pytest.mark.parametrize("L,HQ,copies", KERNELS)
@pytest.mark.parametrize("dtype,gap", [("fp16", 10), ("fp16", 14), ("fp16", 18), ("bf16", 22), ("bf16", 24), ("bf16", 28), ("bf16", 33)])
@pytest.mark.parametrize("at", [3, 60])
def test_one_large_value_of_no_weight(gpu, L, HQ, copies, dtype, gap, at):
    """In every page a key with half of the weight, tens of keys 2^-5.6 below it, and one of no weight whose V is 2^gap times the
    others'."""
    g = torch.Generator().manual_seed(gap)
    dt = {"fp16": torch.float16, "bf16": torch.bfloat16}[dtype]
    n, u, scale = 5000, _signs(g, 128), 0.94 * LN2
    k = u.repeat(n, 1, 1)
    k[:, 0, :3] *= -1  # q . k = 122
    k[5::64, 0] = u
    k[at::64, 0] = -2 * u  # 361 log2 units below
    small = 2.0 ** (13 - gap)
    v = torch.arange(128).float().remainder(3).add(1).repeat(n, 1, 1) * small
    v[5::64] *= -0.5
    v[at::64] = _signs(g, 128) * 2.0 ** 13
    cache, table, lens = _cache(g, k, v, gpu, copies)
    q = u.to(dt).to(gpu).expand(copies, L, HQ, 128).contiguous()
    out = cache.attend(q, table, lens, scale=scale)
    kk, vv = (x[:, 0] for x in R.logical_kv(cache, table[0].tolist()))
    for b, i in _rows(L, copies):
        for h in (0, HQ - 1):
            _close(out[b, i, h], kk, u.double().numpy(), vv, n - L + i + 1, dt, scale)


@pytest.mark.parametrize("L,HQ,copies", KERNELS)
@pytest.mark.parametrize("gap", [24, 33])
def test_one_large_block_of_channels(gpu, L, HQ, copies, gap):
    """V's first 32 channels are 2^gap times the others in every token, and the next 32 zero."""
    g = torch.Generator().manual_seed(gap)
    n, u = 3300, _signs(g, 128)
    k = u.repeat(n, 1, 1)
    k[:, 0, :5] *= -1
    k[100::400, 0] = u
    v = _signs(g, n, 1, 128) + 2
    v[..., :32] *= 2.0 ** 11
    v[..., 32:64] = 0
    v[..., 64:] *= 2.0 ** (11 - gap)
    cache, table, lens = _cache(g, k, v, gpu, copies)
    q = u.bfloat16().to(gpu).expand(copies, L, HQ, 128).contiguous()
    out = cache.attend(q, table, lens, scale=LN2)
    kk, vv = (x[:, 0] for x in R.logical_kv(cache, table[0].tolist()))
    assert (out[..., 32:64] == 0).all()
    for b, i in _rows(L, copies):
        _close(out[b, i, 0], kk, u.double().numpy(), vv, n - L + i + 1, torch.bfloat16, LN2)


@pytest.mark.parametrize("L,HQ,copies", [x for x in KERNELS if x[0] > 1])
def test_values_that_a_row_does_not_see(gpu, L, HQ, copies):
    """The V of the newest token changes nothing, bit for bit, in the rows before it."""
    g = torch.Generator().manual_seed(1)
    n = 3300
    k, v = _signs(g, n, 1, 128), torch.randn(n, 1, 128, generator=g) * 2.0 ** -18
    q = torch.randn(1, L, HQ, 128, generator=g).bfloat16().to(gpu).repeat(copies, 1, 1, 1)
    cache, table, lens = _cache(g, k, v, gpu, copies)
    want = cache.attend(q, table, lens)
    for power in (0, 13):
        cache.append(k[None, -1:].to(gpu), torch.full((1, 1, 1, 128), 2.0 ** power, device=gpu),
                     torch.full((1,), n - 1, dtype=torch.int32, device=gpu), table[:1])
        got = cache.attend(q, table, lens)
        assert torch.equal(got[:, :-1], want[:, :-1]) and not torch.equal(got[:, -1], want[:, -1])


@pytest.mark.parametrize("L,HQ,copies", KERNELS)
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_every_value_of_the_format(gpu, L, HQ, copies, dtype):
    """All of the weight on one key: the row is that token's V, exactly, for every power of two and code.  (Where a page range
    without weight is joined, its sum, at most 3350 tokens x 2^15 x 49152 < 2^43, counts 2^-126, so that an infinity of it would
    stay one; over the largest weight, 2^8 or more, that is below 2^-91 beside a zero, and nothing beside 2^-23 or more.)"""
    g = torch.Generator().manual_seed(5)
    dt = {"fp16": torch.float16, "bf16": torch.bfloat16}[dtype]
    n = 3200 + L
    k = _signs(g, n, 1, 128)
    levels = torch.tensor([6.0] + R.VALUES.tolist() + [-6.0])
    v = levels[torch.randint(0, 18, (n, 1, 128), generator=g)]
    v[..., ::32] = 6  # the blocks' powers of two are what they are made of
    power = (torch.arange(n)[:, None] * 7 + torch.arange(4) * 11) % 36 - 22
    v = (v.view(n, 4, 32) * 2.0 ** power[..., None].float()).view(n, 1, 128)
    cache, table, lens = _cache(g, k, v, gpu, copies)
    for start in range(0, 36 * 4, L * HQ):
        find = (start + torch.arange(L * HQ)) % (36 * 4)
        q = k[find, 0].view(1, L, HQ, 128).to(dt).to(gpu).repeat(copies, 1, 1, 1)
        out = cache.attend(q, table, lens, scale=8 * LN2)  # none of the other keys agrees in more than 124 signs, 64 log2 units below
        want = v[find, 0].view(L, HQ, 128).to(dt).to(gpu)
        for b in sorted({0, copies // 2, copies - 1}):
            assert ((out[b] == want) | (want == 0) & (out[b].abs() < 2.0 ** -91)).all()


@pytest.mark.parametrize("power", [-21, -8, 12])
@pytest.mark.parametrize("L,HQ,copies", KERNELS)
def test_keys_of_every_size(gpu, L, HQ, copies, power):
    """Keys from the smallest to the largest powers of two, and a scale that makes up for it.  (fp16 numbers below 2^-14 have down to
    three bits: what the sum of their products may lose beside larger ones', 2^-17, is in the reference's bound.)"""
    g = torch.Generator().manual_seed(9)
    n, scale = 700, 2.0 ** (-4 - power)
    k, v = _signs(g, n, 1, 128) * torch.randint(1, 4, (n, 1, 1), generator=g), torch.randn(n, 1, 128, generator=g)
    q = torch.randn(1, L, HQ, 128, generator=g).half().to(gpu).repeat(copies, 1, 1, 1)
    cache, table, lens = _cache(torch.Generator().manual_seed(2), k * 2.0 ** power, v, gpu, copies)
    out = cache.attend(q, table, lens, scale=scale)
    kk, vv = R.logical_kv(cache, table[0].tolist())
    assert np.array_equal(kk[:n], k.double().numpy() * 2.0 ** power)
    some = sorted({0, L // 2, L - 1})
    o, bound = reference(q[0], kk, vv, n, L, scale, some)
    assert_close(out[copies // 2][some], o[some], bound[some], q.dtype)


@pytest.mark.parametrize("HQ", [8, 24])
def test_large_values_behind_shared_pages(gpu, HQ):
    """Shared pages for many rows and own ones for few: a large V of no weight in the own pages of some."""
    g = torch.Generator().manual_seed(3)
    B, shared, own = 40, 640, 300
    u = _signs(g, 128)
    tail = u.clone()
    tail[:6] *= -1
    pages = shared // 64 + B * 5
    cache = R.make_cache(pages + 1, 1, gpu, seed=11)
    ids = torch.randperm(pages + 1, generator=g).to(torch.int32)
    table = torch.cat([ids[:10].repeat(B, 1), ids[10:10 + 5 * B].view(B, 5)], 1).to(gpu)
    zero = torch.zeros(1, dtype=torch.int32, device=gpu)
    k, v = tail.repeat(shared, 1, 1), _signs(g, shared, 1, 128) * 2.0 ** -16
    k[5] = u
    cache.append(k[None].to(gpu), v[None].to(gpu), zero, table[:1])
    for b in range(B):
        k, v = tail.repeat(own, 1, 1), (_signs(g, own, 1, 128) + 2) * 2.0 ** -16
        k[70] = u
        if b % 2:
            k[11], v[11] = -2 * u, 2.0 ** 12
        cache.append(k[None].to(gpu), v[None].to(gpu), zero + shared, table[b:b + 1])
    lens = torch.full((B,), shared + own, dtype=torch.int32, device=gpu)
    q = u.bfloat16().to(gpu).expand(B, 1, HQ, 128).contiguous()
    out = cache.attend(q, table, lens, scale=LN2, shared=SharedPrefix(table, lens))
    for b in (0, 1, 20, B - 1):
        kk, vv = (x[:, 0] for x in R.logical_kv(cache, table[b].tolist()))
        _close(out[b, 0, HQ - 1], kk, u.double().numpy(), vv, shared + own, torch.bfloat16, LN2)


@pytest.mark.parametrize("L,HQ,copies", KERNELS)
def test_pages_without_values(gpu, L, HQ, copies):
    """Keys appended alone to a new cache: its V is zeros, whose bytes are below the format's powers of two."""
    g = torch.Generator().manual_seed(13)
    n = 3300
    cache = PagedMXFP4Cache(54, 1, gpu)
    table = torch.randperm(54, generator=g)[:52].to(torch.int32)[None].to(gpu)
    cache.append(_signs(g, 1, n, 1, 128).to(gpu), None, torch.zeros(1, dtype=torch.int32, device=gpu), table)
    q = torch.randn(1, L, HQ, 128, generator=g).half().to(gpu).repeat(copies, 1, 1, 1)
    lens = torch.full((copies,), n, dtype=torch.int32, device=gpu)
    assert (cache.attend(q, table.repeat(copies, 1), lens) == 0).all()
    v = torch.ones(1, 64, 1, 128, device=gpu)  # one page of values: what it weighs
    cache.append(v, v, torch.full((1,), 128, dtype=torch.int32, device=gpu), table)
    out = cache.attend(q, table.repeat(copies, 1), lens)
    kk, vv = R.logical_kv(cache, table[0].tolist())
    some = sorted({0, L // 2, L - 1})
    o, bound = reference(q[0], kk, vv, n, L, 1 / math.sqrt(128), some)
    assert_close(out[copies // 2][some], o[some], bound[some], q.dtype)
