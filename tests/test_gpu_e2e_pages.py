"""The Hugging Face cache's batch operations on shared pages, and exact steps over the pages themselves.

A layer after any sequence of operations holds, bit for bit, what a layer holds that was given each sequence's own K
and V from the start; exact attention with paged_exact is within the arithmetic's bound of 64 bits.
"""
import importlib.util
import math
from pathlib import Path

import pytest
import torch

from attend_ref import assert_close, logical_kv, reference

pytestmark = pytest.mark.gpu
E2E = Path(__file__).resolve().parents[1] / "ffa-speedtest_amd" / "ffa-q2fp8" / "e2e" / "q2fp8_cache.py"


def _load():
    spec = importlib.util.spec_from_file_location("q2fp8_cache_pages", E2E)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


class Both:
    """A layer under test and each sequence's K and V."""

    def __init__(self, C, B, max_batch, dev, cap=640):
        self.C, self.dev, self.cap, self.g = C, dev, cap, torch.Generator().manual_seed(B * 100 + cap)
        self.layer = C.Q2FP8PagedLayer(max_batch, cap, page_seed=3)
        self.rows = [[torch.zeros(2, 0, 128), torch.zeros(2, 0, 128)] for _ in range(B)]

    def update(self, n):
        B = len(self.rows)
        k, v = (torch.randn((B, 2, n, 128), generator=self.g).bfloat16() for _ in range(2))
        self.layer.update(k.to(self.dev), v.to(self.dev))
        self.rows = [[torch.cat([r[0], k[i].float()], 1), torch.cat([r[1], v[i].float()], 1)] for i, r in enumerate(self.rows)]

    def select(self, idx):
        self.rows = [list(self.rows[i]) for i in idx]

    def cut(self, n):
        self.rows = [[r[0][:, :n], r[1][:, :n]] for r in self.rows]

    def check(self):
        S, B = self.rows[0][0].shape[1], len(self.rows)
        assert self.layer.get_seq_length() == S and self.layer.block_table.shape[0] == B
        assert self.layer.seq_lens.tolist() == [S] * B
        want = self.C.Q2FP8PagedLayer(B, self.cap)
        k, v = (torch.stack([r[j] for r in self.rows]).bfloat16().to(self.dev) for j in range(2))
        want.update(k, v)
        got = self.layer.pool.dequantize(self.layer.block_table, S, self.layer.seq_lens)
        for a, b in zip(got, want.pool.dequantize(want.block_table, S, want.seq_lens)):
            assert torch.equal(a, b)
        pages = self.layer.pages
        if pages is not None:
            assert int(pages.errors.item()) == 0
            held = torch.bincount(self.layer.block_table[:, : -(-S // 64)].reshape(-1).long(), minlength=pages.P)
            assert torch.equal(held.int(), pages.refs)


def test_samples_beams_and_crops(gpu):
    x = Both(_load(), 2, 6, gpu)
    x.update(200)
    x.check()
    x.layer.batch_repeat_interleave(3)
    x.select([0, 0, 0, 1, 1, 1])
    x.check()
    assert x.layer.shared.sizes == [3, 3] and x.layer.shared.pages == [3, 3]
    for n in (1, 60, 1):
        x.update(n)
        x.check()
    for beams in ([1, 0, 0, 5, 4, 3], [0] * 6, [5, 4, 3, 2, 1, 0]):
        x.layer.reorder_cache(torch.tensor(beams, device=gpu))
        x.select(beams)
        x.update(1)
        x.check()
    x.layer.batch_select_indices(torch.tensor([4, -1, 0], device=gpu))
    x.select([4, 5, 0])
    x.check()
    x.update(130)
    x.check()
    x.layer.crop(-200)  # into the pages that the samples share
    x.cut(x.rows[0][0].shape[1] - 200)
    x.check()
    x.update(70)
    x.check()
    x.layer.crop(128)  # the length to keep, a page's end
    x.cut(128)
    x.update(3)
    x.check()
    x.layer.crop(-10 ** 6)
    x.cut(0)
    x.update(65)
    x.check()
    x.layer.reset()
    x.cut(0)
    x.update(300)
    x.check()


def test_full_cache_reorders(gpu):
    """Every page held, all last pages partial: the spare pages serve the copies."""
    x = Both(_load(), 4, 4, gpu, cap=128)
    x.update(127)
    for beams in ([3, 2, 1, 0], [0, 0, 1, 1]):
        x.layer.reorder_cache(torch.tensor(beams, device=gpu))
        x.select(beams)
        x.check()
    x.update(1)
    x.check()
    with pytest.raises(ValueError):
        x.update(1)


def test_crop_without_sharing(gpu):
    x = Both(_load(), 2, 2, gpu)
    x.update(300)
    x.layer.crop(-77)
    x.cut(223)
    x.update(5)
    x.check()
    assert x.layer.pages is None


def test_refusals(gpu):
    x = Both(_load(), 2, 4, gpu)
    x.layer.batch_repeat_interleave(2)  # nothing cached yet: nothing to repeat
    x.layer.reorder_cache(torch.tensor([1, 0]))
    x.update(100)
    with pytest.raises(ValueError):
        x.layer.batch_repeat_interleave(3)
    with pytest.raises(IndexError):
        x.layer.batch_select_indices(torch.tensor([2]))
    x.layer.batch_select_indices(torch.tensor([True, False]))
    x.select([0])
    x.check()


def test_llama_samples_with_paged_exact(gpu):
    """A model's prompt, repeated for samples, decoded and extended by exact attention over the pages."""
    from transformers import LlamaConfig, LlamaForCausalLM

    C = _load()
    cfg = LlamaConfig(vocab_size=512, hidden_size=1024, intermediate_size=1536, num_hidden_layers=2,
                      num_attention_heads=8, num_key_value_heads=2, head_dim=128, max_position_embeddings=8192,
                      rope_theta=500000.0)
    torch.manual_seed(0)
    model = LlamaForCausalLM(cfg).to(device=gpu, dtype=torch.bfloat16).eval()
    cache = C.Q2FP8Cache(num_layers=2, max_batch_size=8, max_cache_len=512, page_seed=5)
    seen = []

    def on_exact(i, q, o, layer):
        S, L = layer.seq_len, q.shape[2]
        for b in (0, q.shape[0] - 1):
            k, v = logical_kv(layer.pool, "q2", layer.block_table[b, : -(-S // 64)].tolist())
            want, bound = reference(q[b].transpose(0, 1), k[:S], v[:S], S, L, 1 / math.sqrt(128))
            assert_close(o[b], want, bound, q.dtype, f"layer {i} S={S} L={L} b={b}")
        seen.append((i, q.shape[0], L, layer.shared is not None))

    C.enable_ffa_q2fp8(model, use_ffa_decode=False, paged_exact=True, on_exact=on_exact)
    g = torch.Generator().manual_seed(2)
    ids = lambda *s: torch.randint(0, 512, s, generator=g).to(gpu)  # noqa: E731
    with torch.no_grad():
        model(input_ids=ids(2, 150), past_key_values=cache, use_cache=True)
        cache.batch_repeat_interleave(4)
        for n in (1, 1, 7):
            out = model(input_ids=ids(8, n), past_key_values=cache, use_cache=True)
        cache.reorder_cache(torch.tensor([7, 0, 0, 1, 2, 3, 3, 3], device=gpu))
        out = model(input_ids=ids(8, 1), past_key_values=cache, use_cache=True)
    assert torch.isfinite(out.logits.float()).all() and cache.get_seq_length() == 160
    assert seen == [(i, b, n, s) for b, n, s in ((2, 150, False), (8, 1, True), (8, 1, True), (8, 7, True), (8, 1, False))
                    for i in range(2)]


def test_generate_with_beams(gpu):
    """transformers' own beam search over the cache."""
    from transformers import LlamaConfig, LlamaForCausalLM

    C = _load()
    cfg = LlamaConfig(vocab_size=64, hidden_size=256, intermediate_size=256, num_hidden_layers=1, num_attention_heads=2,
                      num_key_value_heads=1, head_dim=128, max_position_embeddings=512)
    torch.manual_seed(1)
    model = LlamaForCausalLM(cfg).to(device=gpu, dtype=torch.bfloat16).eval()
    C.enable_ffa_q2fp8(model, paged_exact=True)
    ids = torch.randint(0, 64, (2, 70), generator=torch.Generator().manual_seed(3)).to(gpu)
    cache = C.Q2FP8Cache(num_layers=1, max_batch_size=6, max_cache_len=256)
    with torch.no_grad():
        out = model.generate(ids, past_key_values=cache, max_new_tokens=6, num_beams=3, do_sample=False, pad_token_id=0,
                             eos_token_id=None)
    assert out.shape == (2, 76) and torch.equal(out[:, :70], ids)
    assert cache.layers[0].pages is not None and int(cache.layers[0].pages.errors.item()) == 0


@pytest.mark.parametrize("keep", [0, 64, 128])
def test_attention_after_a_crop_to_a_page(gpu, keep):
    """Samples that share three pages, cut to a page's end (or to nothing) and continued apart: attention with the
    layer's plan of shared pages is every sample's own."""
    x = Both(_load(), 1, 3, gpu)
    x.update(200)
    x.layer.batch_repeat_interleave(3)
    x.select([0, 0, 0])
    x.update(10)
    x.layer.crop(keep - 210)
    x.cut(keep)
    for n in (1, 90):
        x.update(n)
        x.check()
        S = x.layer.seq_len
        assert x.layer.shared.sizes == [3] and x.layer.shared.pages == [keep // 64]
        q = torch.randn((3, n, 8, 128), generator=x.g).bfloat16().to(gpu)
        out = x.layer.pool.attend(q, x.layer.block_table, x.layer.seq_lens, T=S, shared=x.layer.shared)
        for b in range(3):
            k, v = logical_kv(x.layer.pool, "q2", x.layer.block_table[b, : -(-S // 64)].tolist())
            want, bound = reference(q[b], k[:S], v[:S], S, n, 1 / math.sqrt(128))
            assert_close(out[b], want, bound, q.dtype, f"S={S} b={b}")


def test_a_new_prompt_after_samples(gpu):
    """One prompt, samples, reset, prompts of other batches; decoded by the pruned kernel as a fresh layer's."""
    C = _load()
    x = Both(C, 1, 4, gpu)
    x.update(200)
    x.layer.batch_repeat_interleave(4)
    x.select([0] * 4)
    x.update(70)
    for B in (1, 3):
        x.layer.reset()
        x.rows = [[torch.zeros(2, 0, 128), torch.zeros(2, 0, 128)] for _ in range(B)]
        x.update(150)
        x.check()
        x.update(1)
        x.check()
        fresh = C.Q2FP8PagedLayer(B, x.cap)
        fresh.update(*(torch.stack([r[j] for r in x.rows]).bfloat16().to(gpu) for j in range(2)))
        q = torch.randn((B, 8, 128), generator=x.g).bfloat16().to(gpu)
        outs = [y.pool.decode(q, y.block_table, y.seq_lens, T=y.capacity, workspace=y.workspace(8, 64, 64, q.dtype)).o
                for y in (x.layer, fresh)]
        assert torch.equal(*outs)


def _copying(C):
    """The cache with every sequence's pages its own: batch operations copy them."""

    class Layer(C.Q2FP8PagedLayer):
        def _select(self, indices, check):
            if not self.is_initialized:
                return
            old, table, idx = self.pool, self.block_table, indices.reshape(-1).cpu()
            npg = table.shape[1]
            self.pool = type(old)(len(idx) * npg, old.HKV, self.device, res_dtype=old.res_dtype, v_dtype=old.v_dtype)
            source = table[idx.to(table.device)].reshape(-1).long()
            for new, t in zip(self.pool.pools(), old.pools()):
                new.view(torch.uint8).copy_(t.view(torch.uint8)[source])
            self.block_table = torch.arange(len(idx) * npg, dtype=torch.int32, device=self.device).view(-1, npg)
            self.seq_lens = torch.full((len(idx),), self.seq_len, dtype=torch.int32, device=self.device)

    def cache(layers, batch, length):
        made = C.Q2FP8Cache(num_layers=layers, max_batch_size=batch, max_cache_len=length)
        made.layers = [Layer(batch, length, page_seed=i) for i in range(layers)]
        return made

    return cache


@pytest.mark.parametrize("ffa_decode", [True, False])
def test_beams_are_those_of_copied_caches(gpu, ffa_decode):
    """transformers' beam search over shared pages: the same tokens and scores, bit for bit, as over caches that copy."""
    from transformers import LlamaConfig, LlamaForCausalLM

    C = _load()
    cfg = LlamaConfig(vocab_size=96, hidden_size=512, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=128, max_position_embeddings=512)
    torch.manual_seed(4)
    model = LlamaForCausalLM(cfg).to(device=gpu, dtype=torch.bfloat16).eval()
    C.enable_ffa_q2fp8(model, use_ffa_decode=ffa_decode, paged_exact=True)
    ids = torch.randint(0, 96, (2, 120), generator=torch.Generator().manual_seed(5)).to(gpu)
    runs = []
    for make in (lambda *a: C.Q2FP8Cache(num_layers=a[0], max_batch_size=a[1], max_cache_len=a[2]), _copying(C)):
        cache = make(2, 8, 256)
        with torch.no_grad():
            out = model.generate(ids, past_key_values=cache, max_new_tokens=30, num_beams=4, num_return_sequences=4,
                                 do_sample=False, pad_token_id=0, eos_token_id=None, return_dict_in_generate=True,
                                 output_scores=True)
        runs.append((out.sequences, out.sequences_scores, out.beam_indices))
        assert cache.get_seq_length() == 149
    assert runs[0][0].shape == (8, 150) and torch.equal(runs[0][0][:, :120], ids.repeat_interleave(4, 0))
    assert len({tuple(r) for r in runs[0][0].tolist()}) == 8
    moved = runs[0][2][:, 1:30] - runs[0][2][:, :29]
    assert (moved != 0).any()  # beams changed places
    for a, b in zip(*runs):
        assert torch.equal(a, b)
