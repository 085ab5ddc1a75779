"""Exact attention over the paged caches on the GPU against a plain implementation in 64 bits.

Lengths around pages and page ranges, query tokens from one to several row tiles, groups of 1 to 16 rows, every
format, residual and V type, padded batches, empty rows, infinities and NaN where a row must not see them, and
groups of sequences that share leading pages (whose result is that of the call without them).
"""
import math

import numpy as np
import pytest
import torch

from attend_ref import assert_close, fill, logical_kv, make_cache, reference
from ffa_mi355x.attend import SharedPrefix

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(128)


def _rand(g, *shape):
    return torch.randn(shape, generator=g)


def _batch(fmt, lens, HQ, HKV, L, dtype, seed, dev, heavy=True, **kw):
    """A cache of sequences with pages in random order, and queries that look for some keys."""
    g = torch.Generator().manual_seed(seed)
    npg = [-(-n // 64) for n in lens]
    P = sum(npg) + 2
    ids = torch.randperm(P, generator=g)
    cache = make_cache(fmt, P, HKV, dev, seed=seed, **kw)
    table = torch.zeros((len(lens), max(npg) + 1), dtype=torch.int32)
    q = _rand(g, len(lens), L, HQ, 128).to(dtype)
    at = 0
    for b, n in enumerate(lens):
        table[b, :npg[b]] = ids[at:at + npg[b]]
        at += npg[b]
        if n == 0:
            continue
        k, v = _rand(g, n, HKV, 128), _rand(g, n, HKV, 128)
        if heavy:
            for h in range(HKV):
                t = int(torch.randint(0, n, (1,), generator=g))
                x = q[b, -1, h * (HQ // HKV)].float()
                k[t, h] = 0.8 * x / x.norm() * math.sqrt(128) + 0.6 * k[t, h]
        fill(cache, k, v, table[b])
    return cache, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), q.to(dev)


def _check(cache, fmt, table, lens, q, out, q_lens=None, residual=True, scale=SCALE):
    B, L = q.shape[:2]
    for b in range(B):
        n = int(lens[b])
        ql = L if q_lens is None else int(q_lens[b])
        if n == 0:
            assert (out[b] == 0).all()
            continue
        k, v = logical_kv(cache, fmt, table[b, :-(-n // 64)].tolist(), residual)
        o, bound = reference(q[b], k[:n], v[:n], n, ql, scale)
        assert_close(out[b], o, bound, q.dtype, f"sequence {b}")


@pytest.mark.parametrize("fmt", ["q2", "nvfp4", "nf4"])
@pytest.mark.parametrize("lens,HQ,HKV,L", [
    ([1], 4, 4, 1),                      # one token
    ([1, 63, 64, 65, 0], 8, 2, 1),       # around a page, an empty sequence
    ([700, 255, 257], 32, 8, 1),         # several pages a wave
    ([130, 40], 14, 2, 3),               # groups of 7 rows, 21 rows: two tiles
    ([200, 5], 16, 1, 5),                # 80 rows: several row blocks; fewer keys than rows of a tile
    ([90, 64], 12, 4, 33),               # 99 rows of a chunk
])
def test_lengths(gpu, fmt, lens, HQ, HKV, L):
    cache, table, sl, q = _batch(fmt, lens, HQ, HKV, L, torch.bfloat16, 3, gpu)
    out = cache.attend(q, table, sl)
    _check(cache, fmt, table, lens, q, out)


@pytest.mark.parametrize("fmt", ["q2", "nvfp4", "nf4"])
@pytest.mark.parametrize("res", [torch.float8_e4m3fn, torch.float8_e5m2])
@pytest.mark.parametrize("v", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_types(gpu, fmt, res, v, dtype):
    lens = [150, 333]
    cache, table, sl, q = _batch(fmt, lens, 8, 2, 2, dtype, 5, gpu, res=res, v=v)
    _check(cache, fmt, table, lens, q, cache.attend(q, table, sl))
    _check(cache, fmt, table, lens, q, cache.attend(q, table, sl, use_fp8_residual=False), residual=False)


def test_long_and_scale(gpu):
    """Page ranges split over many workgroups; a scale of the caller's; T above every length."""
    lens = [9000, 4097]
    cache, table, sl, q = _batch("q2", lens, 8, 2, 1, torch.float16, 7, gpu)
    table = torch.cat([table, torch.full((2, 300), -1, dtype=torch.int32, device=gpu)], 1)
    out = cache.attend(q, table, sl, T=20000, scale=0.03)
    _check(cache, "q2", table, lens, q, out, scale=0.03)


@pytest.mark.parametrize("L,HQ", [(1, 4), (40, 8)])
@pytest.mark.parametrize("scale", [-0.05, 0.0, 2.0])
def test_other_scales(gpu, scale, L, HQ):
    """Negative scales (the least product weighs most), 0 (a mean over the keys), scores far apart."""
    cache, table, sl, q = _batch("nf4", [150], HQ, 1, L, torch.float16, 73, gpu)
    _check(cache, "nf4", table, [150], q, cache.attend(q, table, sl, scale=scale), scale=scale)


def test_empty_batch_of_sequences(gpu):
    cache, table, _, q = _batch("q2", [64, 64], 4, 1, 2, torch.float16, 79, gpu)
    for kw in (dict(seq_lens=torch.zeros(2, dtype=torch.int32, device=gpu)), dict(T=0),
               dict(seq_lens=torch.full((2,), 64, device=gpu), T=0)):
        out = torch.full_like(q, 7)
        assert cache.attend(q, table, out=out, **kw) is out and (out == 0).all()
    sl = torch.tensor([-3, 64], device=gpu)  # clamped
    assert (cache.attend(q, table, sl)[0] == 0).all()


def test_three_dimensions_out_and_strides(gpu):
    """[B, HQ, 128] queries, a strided view of them, int64 tables, a given output."""
    lens = [100, 77]
    cache, table, sl, q = _batch("q2", lens, 8, 2, 1, torch.bfloat16, 9, gpu)
    want = cache.attend(q, table, sl)
    wide = torch.zeros((2, 8, 256), dtype=q.dtype, device=gpu)
    wide[..., :128] = q[:, 0]
    got = cache.attend(wide[..., :128], table.long(), sl.long())
    assert got.shape == (2, 8, 128) and torch.equal(got, want[:, 0])
    buf = torch.empty_like(got)
    assert cache.attend(q[:, 0], table, sl, out=buf) is buf and torch.equal(buf, got)
    odd = torch.empty(2 * 8 * 128 + 1, dtype=q.dtype, device=gpu)[1:].view(2, 8, 128)  # not a multiple of 16 bytes
    odd.copy_(q[:, 0])
    assert torch.equal(cache.attend(odd, table, sl), got)


def test_padded_batch(gpu):
    """q_lens: query tokens past a sequence's own give zeros, also where NaN lies in them; more query tokens than keys."""
    lens, ql = [130, 64, 2, 0], [5, 1, 5, 0]
    cache, table, sl, q = _batch("nvfp4", lens, 8, 2, 5, torch.bfloat16, 11, gpu)
    for b, n in enumerate(ql):
        q[b, n:] = float("nan")
    out = cache.attend(q, table, sl, q_lens=torch.tensor(ql, device=gpu))
    _check(cache, "nvfp4", table, lens, q, out, q_lens=ql)
    assert (out[2, :3] == 0).all() and (out[2, 3:] != 0).any()


@pytest.mark.parametrize("L,HQ", [(70, 4), (9, 16), (5, 2)])
def test_hidden_infinities(gpu, L, HQ):
    """An infinity or NaN in V at a token counts for the rows that see it and for no other."""
    n = 200
    cache, table, sl, q = _batch("q2", [n], HQ, 1, L, torch.float16, 13, gpu)
    v = torch.randn((2, 1, 128))
    v[0, 0, 5], v[1, 0, 7], v[1, 0, 9] = float("inf"), float("nan"), float("-inf")
    k = torch.randn((2, 1, 128))
    fill(cache, k, v, table[0], n - 4)  # tokens n - 4, n - 3: seen by the last 4 and 3 query tokens only
    out = cache.attend(q, table, sl)
    assert torch.isfinite(out[0, :L - 4]).all()
    assert torch.isinf(out[0, L - 4, :, 5]).all() and torch.isfinite(out[0, L - 4, :, 7]).all()
    assert torch.isnan(out[0, L - 3:, :, 7]).all()
    _check(cache, "q2", table, [n], q, out)


def test_large_queries(gpu):
    """bf16 queries beyond fp16's range and tiny ones: rows are scaled by a power of two."""
    cache, table, sl, q = _batch("q2", [80], 8, 2, 1, torch.bfloat16, 17, gpu)
    for f in (2.0 ** 30, 2.0 ** -40):
        _check(cache, "q2", table, [80], q * f, cache.attend(q * f, table, sl, scale=SCALE / f), scale=SCALE / f)


def test_bad_pages_read_page_zero(gpu):
    g = torch.Generator().manual_seed(19)
    cache = make_cache("q2", 5, 1, gpu, seed=19)
    good = torch.tensor([[3, 0, 2]], dtype=torch.int32)
    fill(cache, _rand(g, 192, 1, 128), _rand(g, 192, 1, 128), good[0])
    q = _rand(g, 1, 1, 4, 128).half().to(gpu)
    sl = torch.tensor([130], dtype=torch.int32, device=gpu)
    want = cache.attend(q, good.to(gpu), sl)
    for bad in (-1, 2 ** 31 - 1, -2 ** 31, cache.P):
        t = good.clone()
        t[0, 1] = bad
        assert torch.equal(cache.attend(q, t.to(gpu), sl), want)


def _forked(fmt, sizes, prefix, own, HQ, HKV, L, dtype, seed, dev, **kw):
    """Groups whose members hold the same leading pages; own[b]: tokens past the prefix."""
    g = torch.Generator().manual_seed(seed)
    lens, b = [], 0
    for n, p in zip(sizes, prefix):
        lens += [p + x for x in own[b:b + n]]
        b += n
    P = sum(-(-x // 64) + 1 for x in lens) + sum(-(-p // 64) for p in prefix)
    ids = torch.randperm(P, generator=g).tolist()
    cache = make_cache(fmt, P, HKV, dev, seed=seed, **kw)
    table = torch.full((len(lens), max(-(-x // 64) for x in lens) + 2), -1, dtype=torch.int32)
    b = 0
    for n, p in zip(sizes, prefix):
        sp = p // 64
        shared = [ids.pop() for _ in range(sp)]
        kp, vp = _rand(g, p, HKV, 128), _rand(g, p, HKV, 128)
        for i in range(b, b + n):
            table[i, :sp] = torch.tensor(shared, dtype=torch.int32)
            for j in range(sp, -(-lens[i] // 64)):
                table[i, j] = ids.pop()
            k = torch.cat([kp, _rand(g, own[i], HKV, 128)])
            v = torch.cat([vp, _rand(g, own[i], HKV, 128)])
            if lens[i]:
                fill(cache, k, v, table[i])
        b += n
    q = _rand(g, len(lens), L, HQ, 128).to(dtype)
    return cache, table.to(dev), lens, torch.tensor(lens, dtype=torch.int32, device=dev), q.to(dev)


@pytest.mark.parametrize("fmt", ["q2", "nvfp4", "nf4"])
@pytest.mark.parametrize("sizes,prefix,HQ,HKV,L", [
    ([4], [200], 8, 2, 1),                     # a partial page at the prefix's end, 16 rows
    ([3, 1, 5], [640, 100, 64], 8, 2, 1),      # a group of one, a prefix of one page
    ([2, 9], [63, 130], 16, 2, 1),             # a prefix below a page, 72 rows
    ([6], [3000], 14, 2, 3),                   # groups of 7 rows, 126 rows, three drafted tokens
    ([40], [1000], 8, 1, 1),                   # 320 rows
])
def test_shared_prefix(gpu, fmt, sizes, prefix, HQ, HKV, L):
    B = sum(sizes)
    own = [(37 * b) % 150 + L for b in range(B)]
    cache, table, lens, sl, q = _forked(fmt, sizes, prefix, own, HQ, HKV, L, torch.bfloat16, 23, gpu)
    plan = SharedPrefix(table, sl, group_sizes=sizes)
    assert plan.pages == [p // 64 if n > 1 else 0 for n, p in zip(sizes, prefix)]
    out = cache.attend(q, table, sl, shared=plan)
    _check(cache, fmt, table, lens, q, out)


@pytest.mark.parametrize("fmt,v", [("q2", torch.float16), ("nvfp4", torch.bfloat16), ("nf4", torch.float16)])
@pytest.mark.parametrize("sizes,prefix,HQ,HKV,L", [
    ([40], [700], 8, 1, 1),            # 320 rows over two workgroups, 8 own rows
    ([17, 3, 30], [900, 64, 320], 16, 2, 3),  # uneven groups, drafts: 24 own rows; one group's rows fill a part
])
def test_shared_and_own_pages_in_one_launch(gpu, fmt, v, sizes, prefix, HQ, HKV, L):
    """Own parts of several pages: both kinds of workgroup in one grid; some sequences end before the others' ranges."""
    own = [L + (211 * b) % 700 for b in range(sum(sizes))]
    cache, table, lens, sl, q = _forked(fmt, sizes, prefix, own, HQ, HKV, L, torch.bfloat16, 61, gpu, v=v)
    plan = SharedPrefix(table, sl, group_sizes=sizes)
    out = cache.attend(q, table, sl, shared=plan)
    some = range(0, sum(sizes), 5)
    _check(cache, fmt, table[list(some)], [lens[b] for b in some], q[list(some)], out[list(some)])
    # without the plan, and with a capacity for T: other ranges of the same sums
    for other in (cache.attend(q, table, sl), cache.attend(q, table, sl, T=64 * table.shape[1], shared=plan)):
        assert torch.allclose(out.float(), other.float(), atol=2.0 ** -6, rtol=2.0 ** -7)


@pytest.mark.parametrize("n,L,HQ,HKV", [
    (3300, 150, 8, 2),    # 600 rows over 52 pages: 256-row workgroups, split ranges
    (3200, 140, 64, 4),   # 8960 rows: the join by a wave per row
    (1500, 300, 32, 4),   # few pages, many rows: smaller workgroups, ranges not split
    (700, 100, 4, 4),     # 100 rows of each head: a workgroup's waves with two tiles, one and none
])
def test_chunks(gpu, n, L, HQ, HKV):
    cache, table, sl, q = _batch("q2", [n], HQ, HKV, L, torch.float16, 67, gpu)
    out = cache.attend(q, table, sl)
    k, v = logical_kv(cache, "q2", table[0, :-(-n // 64)].tolist())
    tokens = sorted({0, 1, 63, L // 2, L - 64, L - 2, L - 1} & set(range(L)))
    o, bound = reference(q[0], k[:n], v[:n], n, L, SCALE, tokens)
    assert_close(out[0, tokens], o[tokens], bound[tokens], q.dtype)
    for i in range(0, L, 7):  # every part of the chunk against the same rows as short chunks of their own
        part = cache.attend(q[:, i:i + 7].contiguous(), table, torch.tensor([n - L + min(i + 7, L)], device=gpu))
        assert torch.allclose(part.float(), out[:, i:i + 7].float(), atol=2.0 ** -8, rtol=2.0 ** -8)


def test_hidden_infinities_of_long_chunks(gpu):
    """The same as test_hidden_infinities where 256 rows are a workgroup's and the ranges are split."""
    n, L, HQ = 3200, 200, 4
    cache, table, sl, q = _batch("nvfp4", [n], HQ, 1, L, torch.bfloat16, 71, gpu, v=torch.bfloat16)
    v, k = torch.randn((3, 1, 128)), torch.randn((3, 1, 128))
    v[0, 0, 5], v[1, 0, 7], v[2, 0, 9] = float("inf"), float("nan"), 3e38  # beyond the fp16 operand: an infinity
    fill(cache, k, v, table[0], n - 100)
    out = cache.attend(q, table, sl)[0].float()
    first = L - 100  # the first query token that sees token n - 100
    assert torch.isfinite(out[:first]).all()
    assert torch.isinf(out[first:, :, 5]).all() and torch.isfinite(out[first, :, 7]).all()
    assert torch.isnan(out[first + 1:, :, 7]).all() and torch.isfinite(out[first + 1, :, 9]).all()
    assert torch.isinf(out[first + 2:, :, 9]).all()
    rest = [c for c in range(128) if c not in (5, 7, 9)]
    assert torch.isfinite(out[..., rest]).all()


def test_shared_whole_pages_and_drafts(gpu):
    """Sequences of shared pages only: drafted tokens inside the shared pages, causal there."""
    cache, table, lens, sl, q = _forked("q2", [3], [128], [0, 0, 0], 8, 2, 4, torch.float16, 29, gpu)
    plan = SharedPrefix(table, sl)
    assert plan.sizes == [3] and plan.pages == [2]
    _check(cache, "q2", table, lens, q, cache.attend(q, table, sl, shared=plan))


def test_shared_after_a_cut(gpu):
    """Lengths that later fall below the shared pages (a sequence cut short, an emptied one): the plan still holds."""
    cache, table, lens, sl, q = _forked("q2", [4], [300], [10, 20, 30, 40], 8, 2, 2, torch.bfloat16, 31, gpu)
    plan = SharedPrefix(table, sl)
    cut = [310, 70, 0, 1]
    out = cache.attend(q, table, torch.tensor(cut, device=gpu), T=340, shared=plan)
    _check(cache, "q2", table, cut, q, out)


def test_graph_replays(gpu):
    """A captured call replayed with new queries and grown lengths equals the eager call, with eager work between."""
    cache, table, lens, sl, q = _forked("q2", [4], [500], [1, 2, 3, 4], 8, 2, 1, torch.bfloat16, 37, gpu)
    plan = SharedPrefix(table, sl)
    T = table.shape[1] * 64
    sl = sl - 2
    cache.attend(q, table, sl, T=T, shared=plan)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attend(q, table, sl, T=T, shared=plan)
        plain = cache.attend(q, table, sl, T=T)
    for step in range(4):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(step)).to(q.dtype))
        if step:
            sl += step % 2
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, cache.attend(q, table, sl, T=T, shared=plan))
        assert torch.equal(plain, cache.attend(q, table, sl, T=T))
        _check(cache, "q2", table, sl.tolist(), q, out)


def test_another_stream(gpu):
    cache, table, sl, q = _batch("q2", [1000, 300], 8, 2, 1, torch.bfloat16, 41, gpu)
    want = cache.attend(q, table, sl, T=1000)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = cache.attend(q, table, sl, T=1000)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(want, got)


def test_two_streams_and_two_graphs(gpu):
    """Calls that overlap on two streams, and two captured calls replayed in turn, do not share partials."""
    sets = [_batch("q2", [4000, 900], 8, 2, 1, torch.bfloat16, 83 + i, gpu) for i in range(2)]
    want = [c.attend(q, t, sl, T=4000) for c, t, sl, q in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, (c, t, sl, q) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                outs[i].append(c.attend(q, t, sl, T=4000))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in outs[i])
    graphs, caught = [], []
    for c, t, sl, q in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            caught.append(c.attend(q, t, sl, T=4000))
        graphs.append(g)
    for order in ((0, 1), (1, 0), (0, 0, 1)):
        for o in caught:
            o.zero_()
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(caught[0], want[0]) and torch.equal(caught[1], want[1])


def test_repeatable(gpu):
    """The same bits every time (no order of atomics in them)."""
    cache, table, lens, sl, q = _forked("nf4", [5], [2000], [9] * 5, 8, 2, 1, torch.float16, 43, gpu)
    plan = SharedPrefix(table, sl)
    first = cache.attend(q, table, sl, shared=plan)
    for _ in range(3):
        assert torch.equal(first, cache.attend(q, table, sl, shared=plan))


def test_against_the_pruned_decode_that_keeps_all(gpu):
    """One token: the pruned decode with every block kept computes the same (within its own fp16 steps)."""
    lens = [700, 130]
    cache, table, sl, q = _batch("q2", lens, 8, 2, 1, torch.bfloat16, 47, gpu)
    out = cache.attend(q, table, sl)[:, 0]
    ws = cache.decode(q, table, sl, precomputed_threshold=torch.full((2, 8), -1e30, device=gpu))
    assert int(ws.mask_buf[0].min()) == 1
    for b, n in enumerate(lens):
        k, v = logical_kv(cache, "q2", table[b, :-(-n // 64)].tolist())
        o, bound = reference(q[b], k[:n], v[:n], n, 1, SCALE)
        assert_close(ws.o[b][None], o, 2 * bound, q.dtype)
        assert_close(out[b][None], o, bound, q.dtype)


def test_refusals_on_the_gpu(gpu):
    cache, table, sl, q = _batch("q2", [64], 4, 2, 1, torch.bfloat16, 53, gpu)
    with pytest.raises(NotImplementedError):
        cache.attend(q.float(), table, sl)
    with pytest.raises(ValueError):
        cache.attend(q, table, sl, T=10 ** 6)
    with pytest.raises(ValueError):
        cache.attend(q[:, :, :3], table, sl)
    with pytest.raises(ValueError):
        cache.attend(q, table, sl, out=torch.empty((1, 4, 128), dtype=q.dtype, device=gpu))
    with pytest.raises(ValueError):
        cache.attend(q, table.repeat(2, 1), sl)
    with pytest.raises(ValueError):
        cache.attend(q, table, sl, shared=SharedPrefix(table.repeat(2, 1), sl.repeat(2)))
    with pytest.raises(ValueError):
        cache.attend(q.cpu(), table, sl)
    with pytest.raises(ValueError):
        cache.attend(q, table)
    assert np.isfinite(cache.attend(q, table, sl).float().cpu().numpy()).all()


def _opposed(cache, table, b, n, HKV, at, depth, g):
    """Keys of sequence b along one direction u, that at `at` against it: with queries along u and the returned scale its
    score lies about `depth` log2 units below the others.  Its V holds an infinity, another key's a NaN."""
    u = torch.sign(_rand(g, 128))
    k, v = 0.5 * u + 0.05 * _rand(g, n, HKV, 128), _rand(g, n, HKV, 128)
    k[at] = -u
    v[at, :, 5], v[at, :, 6], v[at + 1, :, 7] = float("inf"), float("-inf"), float("nan")
    fill(cache, k, v, table[b])
    return u, depth * math.log(2) / 192


@pytest.mark.parametrize("depth", [40, 200])  # below fp16's least weight, and below fp32's
@pytest.mark.parametrize("fmt,v", [("q2", torch.float16), ("nf4", torch.bfloat16)])
@pytest.mark.parametrize("n,L,HQ,HKV,at", [
    (200, 1, 4, 1, 10), (200, 1, 4, 1, 190),      # a page that every row sees, and the last one
    (200, 6, 8, 2, 10),                           # two tiles of rows
    (200, 40, 2, 1, 70), (400, 100, 8, 2, 3),     # operands in LDS
    (9000, 1, 8, 2, 700), (9000, 1, 8, 2, 8990),  # ranges of pages, joined
    (3300, 150, 8, 2, 70), (3200, 140, 64, 4, 1), # ranges of a chunk
])
def test_infinities_of_small_weight(gpu, depth, fmt, v, n, L, HQ, HKV, at):
    """A visible infinity counts whatever its weight, also one that rounds to 0 (0 * inf would be a NaN), in the page that
    a row sees in part, in one that all rows see, and joined with ranges of far larger scores."""
    g = torch.Generator().manual_seed(89)
    cache, table, sl, _ = _batch(fmt, [n], HQ, HKV, 1, torch.float16, 89, gpu, v=v)
    u, scale = _opposed(cache, table, 0, n, HKV, at, depth, g)
    q = (u + 0.05 * _rand(g, 1, L, HQ, 128)).half().to(gpu)
    out = cache.attend(q, table, sl, scale=scale)
    sees = [i for i in range(L) if n - L + i >= at]
    last = [i for i in range(L) if n - L + i >= at + 1]
    assert (out[0, sees, :, 5] == float("inf")).all() and (out[0, sees, :, 6] == float("-inf")).all()
    assert torch.isnan(out[0, last, :, 7]).all()
    rest = [c for c in range(128) if c not in (5, 6, 7)]
    assert torch.isfinite(out[..., rest]).all() and torch.isfinite(out[0, [i for i in range(L) if i not in sees]]).all()
    some = sorted({0, L // 2, L - 1})
    k, vv = logical_kv(cache, fmt, table[0, :-(-n // 64)].tolist())
    o, bound = reference(q[0], k[:n], vv[:n], n, L, scale, some)
    assert_close(out[0, some], o[some], bound[some], q.dtype)


@pytest.mark.parametrize("own", [[30, 1, 60, 7], [300, 170, 500, 90]])
@pytest.mark.parametrize("members,L,HQ", [(4, 1, 8), (4, 5, 64), (40, 1, 8)])
def test_infinities_of_small_weight_in_shared_pages(gpu, members, L, HQ, own):
    """The same in pages that sequences share: the call without the plan gives the same infinities."""
    own = [own[b % 4] + L for b in range(members)]
    cache, table, lens, sl, _ = _forked("q2", [members], [640], own, HQ, 1, L, torch.bfloat16, 97, gpu)
    g = torch.Generator().manual_seed(97)
    q = None
    for b, n in enumerate(lens):  # the shared pages are written by every member, with the same values
        u, scale = _opposed(cache, table, b, n, 1, 130, 40, torch.Generator().manual_seed(97))
        q = q if q is not None else (u + 0.05 * _rand(g, members, L, HQ, 128)).bfloat16().to(gpu)
    plan = SharedPrefix(table, sl)
    assert plan.pages == [10]
    a, b = cache.attend(q, table, sl, scale=scale, shared=plan), cache.attend(q, table, sl, scale=scale)
    for out in (a, b):
        assert (out[..., 5] == float("inf")).all() and (out[..., 6] == float("-inf")).all() and torch.isnan(out[..., 7]).all()
    rest = [c for c in range(128) if c not in (5, 6, 7)]
    assert torch.isfinite(a[..., rest]).all() and torch.isfinite(b[..., rest]).all()
    assert torch.allclose(a[..., rest].float(), b[..., rest].float(), atol=2.0 ** -6, rtol=2.0 ** -7)


@pytest.mark.parametrize("fmt", ["q2", "nvfp4", "nf4"])
@pytest.mark.parametrize("n,L,HQ", [
    (2000, 1, 4), (2000, 4, 8),     # one and two tiles of rows
    (2000, 40, 1), (2000, 30, 4),   # operands in LDS
    (9000, 1, 8), (3300, 150, 4),   # ranges of pages, joined
])
def test_constant_values(gpu, fmt, n, L, HQ):
    """V of ones gives ones, whatever the weights round to: the sum below the fraction bar is that of the weights that are
    multiplied.  (Both sums are chains of at most 52 pages x 32 fp32 additions, off by 52 x 32 x 2^-24 < 2^-13 each; half a
    step of fp16 below 1 is 2^-12.)"""
    g = torch.Generator().manual_seed(101)
    cache, table, sl, _ = _batch(fmt, [n], HQ, 1, 1, torch.float16, 101, gpu)
    u = torch.sign(_rand(g, 128))
    k = (-u).repeat(n, 1, 1)
    k[3::64] = u  # one key of every page above the others, which have one score
    fill(cache, k, torch.ones(n, 1, 128), table[0])
    q = u.expand(1, L, HQ, 128).half().contiguous().to(gpu)
    for step in range(24):  # 2 to 4 log2 units below: weights that round by up to half a step either way
        out = cache.attend(q, table, sl, scale=(2 + step / 12) * math.log(2) / 256)
        assert (out == 1).all(), (step, out.float().min(), out.float().max())


@pytest.mark.parametrize("fmt,v", [("q2", torch.float16), ("nvfp4", torch.bfloat16), ("nf4", torch.float16)])
@pytest.mark.parametrize("depth", [20, 25, 27, 30])
@pytest.mark.parametrize("n,L,HQ", [(2000, 1, 4), (2000, 4, 8), (2000, 30, 4), (9000, 1, 8), (3300, 150, 4)])
def test_many_small_weights(gpu, fmt, v, depth, n, L, HQ):
    """Keys far below the largest score, which together weigh something: their weights are not lost below fp16's steps."""
    g = torch.Generator().manual_seed(103)
    cache, table, sl, _ = _batch(fmt, [n], HQ, 1, 1, torch.float16, 103, gpu, v=v)
    u = torch.sign(_rand(g, 128))
    k, vv = (-u).repeat(n, 1, 1), torch.ones(n, 1, 128)
    k[3], vv[3] = u, 0
    fill(cache, k, vv, table[0])
    q = u.expand(1, L, HQ, 128).half().contiguous().to(gpu)
    scale = depth * math.log(2) / 256
    out = cache.attend(q, table, sl, scale=scale)
    k, vv = logical_kv(cache, fmt, table[0, :-(-n // 64)].tolist())
    some = sorted({0, L // 2, L - 1})
    o, bound = reference(q[0], k[:n], vv[:n], n, L, scale, some)
    assert_close(out[0, some], o[some], bound[some], q.dtype)
