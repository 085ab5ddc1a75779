"""Page management on the GPU against a plain model of it: counts, tables and every byte of every pool; and the calls
together as a sampler uses them (prompt, fork, append, attention with the shared pages, free, compact)."""
import math

import pytest
import torch

from attend_ref import assert_close, fill, logical_kv, make_cache, reference
from ffa_mi355x.attend import SharedPrefix
from ffa_mi355x.pages import PagePool

pytestmark = pytest.mark.gpu
I = torch.int32


class Model:
    """The same pool in plain lists; page contents as one tag per page."""

    def __init__(self, P):
        self.P, self.refs, self.tag = P, [0] * P, list(range(P))

    def take(self, n):
        free = [p for p in range(self.P) if self.refs[p] == 0][:n]
        return free if len(free) == n else None

    def fork(self, table, lens, parents):
        need = sum(1 for c in parents if lens[c] % 64)
        new = self.take(need)
        rows = []
        if new is None:
            return [[-1] * len(table[0]) for _ in parents]
        for c in parents:
            full = lens[c] // 64
            row = table[c][:full] + [-1] * (len(table[0]) - full)
            for p in row[:full]:
                self.refs[p] += 1
            if lens[c] % 64:
                row[full] = new.pop(0)
                self.refs[row[full]] = 1
                self.tag[row[full]] = self.tag[table[c][full]]
            rows.append(row)
        return rows

    def extend(self, table, lens, n):
        need = [(r, j) for r, x in enumerate(lens) for j in range(-(-x // 64), -(-(x + n) // 64))]
        new = self.take(len(need))
        if new is None or any(j >= len(table[0]) for _, j in need):
            return
        for (r, j), p in zip(need, new):
            table[r][j] = p
            self.refs[p] = 1

    def count(self, table, lens, step):
        for row, x in zip(table, lens):
            for p in row[:-(-x // 64)]:
                self.refs[p] = max(0, self.refs[p] + step)

    def compact(self, *tables):
        n = sum(r > 0 for r in self.refs)
        holes = [p for p in range(n) if self.refs[p] == 0]
        moves = [p for p in range(n, self.P) if self.refs[p] > 0]
        to = dict(zip(moves, holes))
        for a, b in to.items():
            self.refs[b], self.refs[a], self.tag[b] = self.refs[a], 0, self.tag[a]
        for t in tables:
            for row in t:
                row[:] = [to.get(p, p) for p in row]
        return n


def _pool(dev, P, fmts=("q2", "nf4", "nvfp4"), HKV=2):
    caches = [make_cache(f, P, HKV, dev, seed=i) for i, f in enumerate(fmts)]
    pool = PagePool(caches)
    before = [t.view(torch.uint8).view(P, -1).clone() for c in caches for t in c.pools()]
    return pool, before


def _same(pool, before, m):
    assert pool.refs.tolist() == m.refs
    tag = torch.tensor(m.tag, device=pool.device)
    for t, b in zip((t for c in pool.caches for t in c.pools()), before):
        assert torch.equal(t.view(torch.uint8).view(pool.P, -1), b[tag])


def _dev(x, dev):
    return torch.tensor(x, dtype=I, device=dev)


@pytest.mark.parametrize("HKV", [1, 3, 8])
def test_copy(gpu, HKV):
    pool, before = _pool(gpu, 40, HKV=HKV)
    m = Model(40)
    src, dst = [5, 5, 39, 0], [6, 1, 2, 38]
    for a, b in zip(src, dst):
        m.tag[b] = m.tag[a]
    pool.copy(torch.tensor(src), _dev(dst, gpu))
    _same(pool, before, m)
    pool.copy(_dev([], gpu), _dev([], gpu))
    pool.copy(_dev([40, -1, 3], gpu), _dev([7, 8, 40], gpu), check=False)  # outside the pool: left out
    _same(pool, before, m)
    for s, d in (([1], [1]), ([1, 2], [3, 3]), ([1, 2], [2, 4]), ([40], [1]), ([1], [-1]), ([1, 2], [3])):
        with pytest.raises(ValueError):
            pool.copy(_dev(s, gpu), _dev(d, gpu))
    _same(pool, before, m)


@pytest.mark.parametrize("P", [17, 400, 20000])
def test_random_life(gpu, P):
    """Extend, fork, free and compact in a random order, counts and contents checked after every call."""
    g = torch.Generator().manual_seed(P)
    r = lambda a, b: int(torch.randint(a, b + 1, (1,), generator=g))  # noqa: E731
    pool, before = _pool(gpu, P, fmts=("nf4",), HKV=1)
    m, cols = Model(P), 6
    busy = [p for p in range(P) if P > 1000 and p % 5]  # a large pool that is mostly held
    for p in busy:
        m.refs[p] = 3
    pool.refs.copy_(_dev(m.refs, gpu))
    rows, lens = [], []
    for step in range(25):
        op = r(0, 3) if rows else 0
        if op == 0:
            n, add = r(1, 3), r(1, 200)
            t = [[-1] * cols for _ in range(n)]
            td = _dev(t, gpu)
            ok = m.take(n * -(-add // 64)) is not None
            if ok:
                pool.extend(td, _dev([0] * n, gpu), add)
            else:
                with pytest.raises(RuntimeError):
                    pool.extend(td, _dev([0] * n, gpu), add)
            m.extend(t, [0] * n, add)
            assert td.tolist() == t
            if ok:
                rows += t
                lens += [add] * n
        elif op == 1:
            parents = [r(0, len(rows) - 1) for _ in range(r(1, 4))]
            ok = m.take(sum(1 for c in parents if lens[c] % 64)) is not None
            child = m.fork(rows, lens, parents)
            if ok:
                got = pool.fork(_dev(rows, gpu), _dev(lens, gpu), _dev(parents, gpu))
            else:
                with pytest.raises(RuntimeError):
                    pool.fork(_dev(rows, gpu), _dev(lens, gpu), _dev(parents, gpu))
                got = pool.fork(_dev(rows, gpu), _dev(lens, gpu), _dev(parents, gpu), check=False)
            assert got.tolist() == child
            if ok:
                rows += child
                lens += [lens[c] for c in parents]
        elif op == 2:
            k = r(0, len(rows) - 1)
            m.count([rows[k]], [lens[k]], -1)
            pool.free(_dev([rows[k]], gpu), _dev([lens[k]], gpu))
            del rows[k], lens[k]
        else:
            td = _dev(rows, gpu)
            assert pool.compact(td) == m.compact(rows)
            assert td.tolist() == rows
        _same(pool, before, m)


def test_extend_partial_pages(gpu):
    """Tokens that fit the last page take none; rows at a page's end, of no tokens, several pages at once."""
    pool, before = _pool(gpu, 30, fmts=("q2",))
    m = Model(30)
    t, lens = [[-1] * 8 for _ in range(4)], [0, 0, 0, 0]
    td = _dev(t, gpu)
    for add in (1, 62, 1, 1, 130, 0):
        pool.extend(td, _dev(lens, gpu), add)
        m.extend(t, lens, add)
        lens = [x + add for x in lens]
        assert td.tolist() == t
        _same(pool, before, m)
    td2 = td.clone()
    with pytest.raises(ValueError):  # beyond the row
        pool.extend(td2, _dev([0, 0, 8 * 64, 0], gpu), 1)
    with pytest.raises(ValueError):
        pool.extend(td2, _dev([0, -1, 0, 0], gpu), 1)
    with pytest.raises(RuntimeError):  # not enough pages: none is taken
        pool.extend(td2, _dev([0] * 4, gpu), 8 * 64)
    assert torch.equal(td, td2)
    _same(pool, before, m)
    assert pool.num_free() == sum(r == 0 for r in m.refs)


def test_fork_refusals(gpu):
    pool, before = _pool(gpu, 30, fmts=("q2",))
    m = Model(30)
    t, lens = [[-1] * 4 for _ in range(2)], [0, 0]
    td = _dev(t, gpu)
    pool.extend(td, _dev(lens, gpu), 100)
    m.extend(t, lens, 100)
    lens = _dev([100, 100], gpu)
    for parents in ([2], [-1], [0, 1, 2 ** 31 - 1]):
        with pytest.raises(ValueError):
            pool.fork(td, lens, _dev(parents, gpu))
        assert (pool.fork(td, lens, _dev(parents, gpu), check=False) == -1).all()
    for bad in ([257, 100], [-5, 100]):
        with pytest.raises(ValueError):
            pool.fork(td, _dev(bad, gpu), _dev([0], gpu))
    wrong = td.clone()
    wrong[0, 1] = 29  # the partial page is one that nobody holds
    with pytest.raises(ValueError):
        pool.fork(wrong, lens, _dev([0], gpu))
    wrong[0, 1] = 30
    with pytest.raises(ValueError):
        pool.fork(wrong, lens, _dev([0], gpu))
    _same(pool, before, m)
    assert int(pool.errors.item()) == 2
    wrong = td.clone()
    wrong[0, 0] = -7  # a whole page outside the pool: not shared, reported
    with pytest.raises(ValueError):
        pool.fork(wrong, lens, _dev([0], gpu))
    assert pool.fork(td, lens, _dev([], gpu)).shape == (0, 4)
    for bad in (dict(block_table=td[0]), dict(seq_lens=lens[:1]), dict(parents=td)):
        with pytest.raises(ValueError):
            pool.fork(**{**dict(block_table=td, seq_lens=lens, parents=_dev([0], gpu)), **bad})


def test_free_twice(gpu):
    """A page freed twice stays free; the same row twice in one call counts twice."""
    pool, _ = _pool(gpu, 10, fmts=("nvfp4",))
    t = _dev([[-1] * 3], gpu)
    pool.extend(t, _dev([0], gpu), 150)
    pool.hold(t, _dev([150], gpu))
    assert pool.refs.tolist() == [2, 2, 2] + [0] * 7
    pool.free(t.repeat(2, 1), _dev([150, 64], gpu))
    assert pool.refs.tolist() == [0, 1, 1] + [0] * 7
    with pytest.raises(ValueError):
        pool.free(t, _dev([150], gpu))
    assert pool.refs.tolist() == [0] * 10
    for bad in ([[-1, 0, 0]], [[10, 0, 0]]):
        with pytest.raises(ValueError):
            pool.hold(_dev(bad, gpu), _dev([1], gpu))
    with pytest.raises(ValueError):
        pool.hold(t, _dev([1000], gpu))


def test_compact_several_tables(gpu):
    """Counts above one, entries that name no page, a table given twice, an empty and a full pool."""
    pool, before = _pool(gpu, 50)
    m = Model(50)
    assert pool.compact() == 0
    for p, c in ((49, 2), (3, 1), (7, 1), (30, 4), (31, 1)):
        m.refs[p] = c
    pool.refs.copy_(_dev(m.refs, gpu))
    a, b = [[49, 3, -1], [30, 49, 10]], [[7, 31, 2 ** 31 - 1, 30]]
    ad, bd = _dev(a, gpu), _dev(b, gpu)
    assert pool.compact(ad, bd, ad) == m.compact(a, b)
    assert ad.tolist() == a and bd.tolist() == b
    _same(pool, before, m)
    pool.refs.fill_(1)
    m.refs = [1] * 50
    assert pool.compact(ad) == 50 and ad.tolist() == a
    _same(pool, before, m)
    with pytest.raises(ValueError):
        pool.compact(ad.long())
    with pytest.raises(ValueError):
        pool.compact(ad.t())
    with pytest.raises(NotImplementedError):
        pool.compact(*[ad] * 9)


def test_many_layers(gpu):
    """More pools than one launch takes (32 layers of five)."""
    pool, before = _pool(gpu, 6, fmts=("q2",) * 32, HKV=1)
    m = Model(6)
    t = [[-1, -1]]
    td = _dev(t, gpu)
    pool.extend(td, _dev([0], gpu), 70)
    m.extend(t, [0], 70)
    assert pool.fork(td, _dev([70], gpu), _dev([0, 0], gpu)).tolist() == m.fork(t, [70], [0, 0])
    _same(pool, before, m)
    pool.copy(_dev([0], gpu), _dev([5], gpu))
    m.tag[5] = m.tag[0]
    pool.free(td, _dev([70], gpu))
    m.count(t, [70], -1)
    _same(pool, before, m)
    assert pool.compact() == m.compact()
    _same(pool, before, m)


def test_pool_refusals(gpu):
    with pytest.raises(ValueError):
        PagePool([make_cache("q2", 4, 1, gpu), make_cache("q2", 5, 1, gpu)])
    with pytest.raises(ValueError):
        PagePool([])


def test_captured_fork(gpu):
    """Fork and free in a graph, replayed with other parents; equal to eager calls on an equal pool."""
    pool, before = _pool(gpu, 60, fmts=("q2", "nf4"))
    m = Model(60)
    t, lens = [[-1] * 5 for _ in range(3)], [0] * 3
    td, ld, pd = _dev(t, gpu), _dev(lens, gpu), _dev([0, 1, 2, 0], gpu)
    pool.extend(td, ld, 200)
    m.extend(t, lens, 200)
    ld.fill_(200)
    pool.free(pool.fork(td, ld, pd, check=False), ld[pd.long()], check=False)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        child = pool.fork(td, ld, pd, check=False)
        clens = ld[pd.long()]
        held = pool.refs.clone()
        pool.free(child, clens, check=False)
    for parents in ([0, 1, 2, 0], [2, 2, 2, 2], [1, 0, 1, 0]):
        pd.copy_(_dev(parents, gpu))
        graph.replay()
        torch.cuda.synchronize()
        rows = m.fork(t, [200] * 3, parents)
        assert child.tolist() == rows and held.tolist() == m.refs
        m.count(rows, [200] * 4, -1)
        _same(pool, before, m)
        assert int(pool.errors.item()) == 0


@pytest.mark.parametrize("fmt", ["q2", "nvfp4", "nf4"])
def test_samples_of_prompts(gpu, fmt):
    """Two prompts, three samples each, two layers: prompt pages, fork, tokens appended to every sample, attention
    with the shared pages, prompts freed, compaction, and the same attention again; all against 64 bits."""
    HQ, HKV, cols = 8, 2, 12
    g = torch.Generator().manual_seed(3)
    layers = [make_cache(fmt, 60, HKV, gpu, seed=i) for i in range(2)]
    pool = PagePool(layers)
    plens = [200, 333]
    table = torch.full((2, cols), -1, dtype=I, device=gpu)
    for b, n in enumerate(plens):  # prompts of different lengths, one by one
        pool.extend(table[b:b + 1], _dev([0], gpu), n)
        for cache in layers:
            fill(cache, torch.randn((n, HKV, 128), generator=g), torch.randn((n, HKV, 128), generator=g), table[b])
    lens = _dev(plens, gpu)
    parents = _dev([0, 0, 0, 1, 1, 1], gpu)
    child, clens = pool.fork(table, lens, parents), lens[parents.long()]
    pool.free(table, lens)
    plan = SharedPrefix(child, clens)
    assert plan.sizes == [3, 3] and plan.pages == [3, 5]
    for step, n in enumerate((1, 70, 1)):
        pool.extend(child, clens, n)
        for cache in layers:
            cache.append(torch.randn((6, n, HKV, 128), generator=g).to(gpu), torch.randn((6, n, HKV, 128), generator=g).to(gpu),
                         clens, child, ragged=True)
        clens = clens + n
        q = torch.randn((6, min(n, 5), HQ, 128), generator=g).to(torch.bfloat16).to(gpu)
        outs = [cache.attend(q, child, clens, shared=plan) for cache in layers]
        for cache, out in zip(layers, outs):
            for b in range(6):
                x = int(clens[b])
                k, v = logical_kv(cache, fmt, child[b, :-(-x // 64)].tolist())
                o, bound = reference(q[b], k[:x], v[:x], x, q.shape[1], 1 / math.sqrt(128))
                assert_close(out[b], o, bound, q.dtype, f"step {step} sequence {b}")
    first = [cache.attend(q, child, clens, shared=plan) for cache in layers]
    pool.free(child[4:], clens[4:])
    held = pool.compact(child)
    assert held == int((pool.refs > 0).sum()) == int(pool.refs.nonzero().max()) + 1
    plan = SharedPrefix(child[:4], clens[:4])
    for cache, out in zip(layers, first):  # the groups' sizes changed, so the page ranges may
        again = cache.attend(q[:4], child[:4], clens[:4], shared=plan)
        assert torch.allclose(again.float(), out[:4].float(), atol=2.0 ** -7, rtol=2.0 ** -7)


@pytest.mark.parametrize("cols", [6, 9000])  # the check within the ranking, and by a launch of its own
def test_fork_of_bad_whole_pages_changes_nothing(gpu, cols):
    """A parent's whole page that is free (the next one to be given out, too) or outside the pool: no child, no count, no
    copy, whichever child is the bad one's."""
    pool, before = _pool(gpu, 40, fmts=("q2", "nf4"))
    m = Model(40)
    t, lens = [[-1] * cols for _ in range(2)], [0, 0]
    td = _dev(t, gpu)
    pool.extend(td, _dev(lens, gpu), 300)
    m.extend(t, lens, 300)
    lens = _dev([300, 300], gpu)
    _same(pool, before, m)
    for col in (0, 3):
        for bad in (10, 39, 40, -1, 2 ** 31 - 1):  # 10: the lowest free page
            wrong = td.clone()
            wrong[1, col] = bad
            for parents in ([1], [0, 1, 0]):
                pool.errors.zero_()
                with pytest.raises(ValueError):
                    pool.fork(wrong, lens, _dev(parents, gpu))
                assert (pool.fork(wrong, lens, _dev(parents, gpu), check=False) == -1).all()
                assert int(pool.errors.item()) == 4
                _same(pool, before, m)
            child = pool.fork(wrong, lens, _dev([0], gpu))  # the other sequence is served
            assert child.tolist() == m.fork(t, [300, 300], [0])
            pool.free(child, lens[:1])
            m.count(child.tolist(), [300], -1)
            _same(pool, before, m)
    wrong = td.clone()
    wrong[0, 0], wrong[1, 4] = 39, 39  # a whole page and a partial one
    pool.errors.zero_()
    pool.fork(wrong, lens, _dev([0, 1], gpu), check=False)
    assert int(pool.errors.item()) == 6
    _same(pool, before, m)


@pytest.mark.parametrize("children,cols", [(70, 30), (600, 90)])
def test_fork_of_many_rows(gpu, children, cols):
    """More children than one pass of the ranking workgroup's waves, by both ways of the check."""
    pool, before = _pool(gpu, 2000, fmts=("nf4",), HKV=1)
    m = Model(2000)
    t, lens = [[-1] * cols for _ in range(3)], [0] * 3
    td = _dev(t, gpu)
    pool.extend(td, _dev(lens, gpu), 64 * cols - 7)
    m.extend(t, lens, 64 * cols - 7)
    lens = [64 * cols - 7, 64 * 11, 64 * 17 + 1]
    parents = [(5 * c) % 3 for c in range(children)]
    assert pool.fork(td, _dev(lens, gpu), _dev(parents, gpu)).tolist() == m.fork(t, lens, parents)
    _same(pool, before, m)
    wrong = td.clone()
    wrong[2, 16] = 1999
    with pytest.raises(ValueError):
        pool.fork(wrong, _dev(lens, gpu), _dev(parents[:-2] + [2, 0], gpu))
    _same(pool, before, m)


@pytest.mark.parametrize("bad", [4, 29, 30, -1, -2 ** 31, 2 ** 31 - 1])  # 4: the lowest free page
@pytest.mark.parametrize("tokens", [0, 1, 100])
def test_extend_refuses_bad_partial_pages(gpu, bad, tokens):
    """A last page, partly filled, that is free or outside the pool: no row gets pages (a free one could be given out as a
    new page, its tokens beside others')."""
    pool, before = _pool(gpu, 30, fmts=("q2",))
    m = Model(30)
    t, lens = [[-1] * 6 for _ in range(2)], [0, 0]
    td = _dev(t, gpu)
    pool.extend(td, _dev(lens, gpu), 100)
    m.extend(t, lens, 100)
    for row in (0, 1):
        wrong = td.clone()
        wrong[row, 1] = bad
        given = wrong.clone()
        pool.errors.zero_()
        with pytest.raises(ValueError):
            pool.extend(given, _dev([100, 100], gpu), tokens)
        pool.extend(given, _dev([100, 100], gpu), tokens, check=False)
        assert torch.equal(given, wrong) and int(pool.errors.item()) == 2
        _same(pool, before, m)
    at_end = td.clone()
    at_end[:, 1] = bad  # past whole pages: written, not read
    pool.extend(at_end, _dev([64, 64], gpu), tokens)
    m.extend(t, [64, 64], tokens)
    assert pool.refs.tolist() == m.refs
    assert tokens == 0 or at_end.tolist() == t
