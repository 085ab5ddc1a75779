"""The Hugging Face cache layer's batch operations on the CPU, with plain stand-ins for the pages and their counts: what
every sequence reads through its block table, and through the plan of shared pages, is its own tokens."""
import importlib.util
from pathlib import Path

import pytest
import torch

E2E = Path(__file__).resolve().parents[1] / "ffa-speedtest_amd" / "ffa-q2fp8" / "e2e" / "q2fp8_cache.py"


class Cache:
    """One number per token, taken from its key."""

    def __init__(self, num_pages, HKV, device, res_dtype=None, v_dtype=None):
        self.P, self.HKV, self.res_dtype, self.v_dtype = num_pages, HKV, res_dtype, v_dtype
        self.data = torch.full((num_pages, 64), -1.0)

    def pools(self):
        return [self.data]

    def append(self, k, v, pos, table):
        assert k.shape[3] == 128 and len(pos) == len(table)
        for b in range(k.shape[0]):
            for n in range(k.shape[1]):
                t = int(pos[b]) + n
                page = int(table[b, t // 64])
                assert 0 <= page < self.P
                self.data[page, t % 64] = k[b, n, 0, 0]


class Pool:
    """ffa_mi355x.pages.PagePool's calls by its documentation."""

    def __init__(self, caches):
        self.caches, self.P = caches, caches[0].P
        self.refs = torch.zeros(self.P, dtype=torch.int32)

    def _new(self):
        page = int((self.refs == 0).nonzero()[0])
        self.refs[page] = 1
        return page

    def hold(self, table, lens, check=True):
        for row, n in zip(table, lens):
            for j in range(-(-int(n) // 64)):
                self.refs[row[j]] += 1

    def free(self, table, lens, check=True):
        for row, n in zip(table, lens):
            for j in range(-(-int(n) // 64)):
                assert self.refs[row[j]] > 0
                self.refs[row[j]] -= 1

    def extend(self, table, lens, tokens, check=True):
        for row, n in zip(table, lens.tolist()):
            for j in range(-(-n // 64), -(-(n + tokens) // 64)):
                row[j] = self._new()

    def fork(self, table, lens, parents, check=True):
        child = torch.full((len(parents), table.shape[1]), -1, dtype=torch.int32)
        for r, p in enumerate(parents.tolist()):
            n = int(lens[p])
            child[r, :n // 64] = table[p, :n // 64]
            self.hold(child[r:r + 1], [n // 64 * 64])
            if n % 64:
                child[r, n // 64] = self._new()
                self.caches[0].data[child[r, n // 64]] = self.caches[0].data[table[p, n // 64]]
        return child


class Both:
    """A layer and each sequence's numbers."""

    def __init__(self, monkeypatch, B, max_batch, cap=640):
        spec = importlib.util.spec_from_file_location("q2fp8_cache_pages_cpu", E2E)
        C = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(C)
        monkeypatch.setattr(C, "PagedQ2Cache", Cache)
        monkeypatch.setattr(C, "PagePool", Pool)
        self.layer = C.Q2FP8PagedLayer(max_batch, cap, page_seed=1)
        self.rows, self.next = [[] for _ in range(B)], 0

    def update(self, n, B=None):
        if B is not None:
            self.rows = [[] for _ in range(B)]
        new = self.next + torch.arange(len(self.rows) * n).float().view(len(self.rows), n)
        self.next += new.numel()
        k = new[:, None, :, None].expand(-1, 1, -1, 128)
        self.layer.update(k, k)
        self.rows = [r + x.tolist() for r, x in zip(self.rows, new)]

    def repeat(self, n):
        self.layer.batch_repeat_interleave(n)
        self.rows = [list(r) for r in self.rows for _ in range(n)]

    def crop(self, n, keep):
        self.layer.crop(n)
        self.rows = [r[:keep] for r in self.rows]

    def check(self):
        y = self.layer
        assert y.seq_lens.tolist() == [len(r) for r in self.rows] and y.seq_len == len(self.rows[0])
        table = y.block_table.clone()
        for plan in (False, True):
            if plan and y.shared is not None:  # a group's shared columns are read from its first row
                assert y.shared.B == len(self.rows)
                at = 0
                for size, pages in zip(y.shared.sizes, y.shared.pages):
                    table[at:at + size, :pages] = table[at, :pages].clone()
                    at += size
            for row, want in zip(table, self.rows):
                got = y.pool.data[row[:-(-len(want) // 64)].long()].reshape(-1)[:len(want)]
                assert got.tolist() == want
        if y.pages is not None:
            held = torch.bincount(y.block_table[:, :-(-y.seq_len // 64)].reshape(-1).long(), minlength=y.pages.P)
            assert torch.equal(held.int(), y.pages.refs)


@pytest.mark.parametrize("keep", [0, 1, 64, 100, 128, 192, 200, 209])
@pytest.mark.parametrize("negative", [False, True])
def test_crop_of_samples(monkeypatch, keep, negative):
    """Shortened inside and at the end of shared pages, to nothing, and by less than the samples' own tokens; the
    samples then go on apart, into new pages."""
    x = Both(monkeypatch, 1, 6)
    x.update(200)
    x.repeat(3)
    x.update(10)
    x.check()
    if keep == 0 and not negative:
        return  # crop(0) removes nothing
    x.crop(keep - 210 if negative else keep, keep)
    x.check()
    for n in (1, 99, 130):
        x.update(n)
        x.check()


def test_crop_of_two_groups_twice(monkeypatch):
    x = Both(monkeypatch, 2, 4)
    x.update(256)
    x.repeat(2)
    for keep in (192, 64):
        x.crop(keep, keep)
        assert x.layer.shared.sizes == [2, 2] and x.layer.shared.pages == [keep // 64] * 2
        x.update(128)
        x.check()
    x.crop(-192, 0)
    x.check()


@pytest.mark.parametrize("empty", [lambda y: y.reset(), lambda y: y.crop(-10 ** 6)])
def test_other_batches_after_an_empty_cache(monkeypatch, empty):
    """One prompt, samples of it, emptied: the next prompt's batch is its own."""
    x = Both(monkeypatch, 1, 5)
    x.update(200)
    x.repeat(3)
    x.update(70)
    for B in (1, 4, 5, 3):
        empty(x.layer)
        x.update(130, B)
        x.check()
        x.update(1)
        x.check()
        with pytest.raises(ValueError):  # with tokens cached the batch stands
            x.layer.update(torch.zeros(B - 1 or 2, 1, 1, 128), torch.zeros(B - 1 or 2, 1, 1, 128))
        x.check()
    x.layer.batch_select_indices(torch.tensor([2, 0]))
    x.rows = [x.rows[2], x.rows[0]]
    x.check()
    x.layer.reset()
    for B in (0, 6):
        with pytest.raises(ValueError):
            x.layer.update(torch.zeros(B, 1, 1, 128), torch.zeros(B, 1, 1, 128))


def test_empty_selections_are_refused(monkeypatch):
    """No sequence selected: refused before anything changes."""
    x = Both(monkeypatch, 2, 4)
    x.update(100)
    for counted in (False, True):
        for call in (lambda y: y.batch_repeat_interleave(0), lambda y: y.batch_select_indices(torch.zeros(len(x.rows), dtype=torch.bool)),
                     lambda y: y.batch_select_indices(torch.tensor([], dtype=torch.long)),
                     lambda y: y.reorder_cache(torch.tensor([], dtype=torch.long))):
            with pytest.raises(ValueError):
                call(x.layer)
            x.check()
        assert (x.layer.pages is not None) == counted
        x.repeat(2 - counted)
        x.update(30)
        x.check()


def test_refused_tokens_take_no_pages(monkeypatch):
    """An append that is refused (here: a head dimension that the cache does not hold) after its pages were taken."""
    x = Both(monkeypatch, 1, 3)
    x.update(60)
    x.repeat(3)
    for n in (1, 300):  # inside the last page, and past it
        for _ in range(3):
            with pytest.raises(AssertionError):
                x.layer.update(torch.zeros(3, 1, n, 64), torch.zeros(3, 1, n, 64))
            x.check()
    x.update(500)
    x.check()
