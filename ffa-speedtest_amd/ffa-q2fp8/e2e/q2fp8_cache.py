"""Hugging Face integration of the q2fp8 pruned decode: a paged KV cache and a decode attention hook.

The reference integrates its fp8fp8 kernel into a copied Llama (ffa-fp8fp8/e2e/fp8fp8_cache.py:183-224,
ffa-fp8fp8/e2e/modeling_llama.py:293-321): a `Cache` subclass stores the quantized K, and the attention
forward calls the FFA decode when a step has one query token.  Its cache rebuilds a dequantized copy of
all keys on every update (fp8fp8_cache.py:60-69) and grows by `torch.cat`.

Here, for q2fp8, on the MI355X library:

* `Q2FP8Cache` / `Q2FP8PagedLayer`: every layer keeps a `PagedQ2Cache` (64-token pages, g32 2-bit codes +
  fp8 residual K, V^T pages) sized once for `max_batch_size` x `max_cache_len`, with a seeded page table.
  `update()` g32-quantizes and appends the new (already rotated) K and V in one kernel
  (`ffa_q2_quantize_g32_append`) and never dequantizes the cache.
* `ffa_q2fp8_attention`: registered with transformers' attention registry as "ffa_q2fp8", so an
  unmodified `LlamaForCausalLM` (or any model whose attention goes through `ALL_ATTENTION_FUNCTIONS`)
  uses it once `enable_ffa_q2fp8(model, ...)` is called.  As in the reference's hook
  (modeling_llama.py:281-337, settings from `config.attn_settings`, e2e/bench_llama_fp8fp8.py:179-189):
  a step with one query token per sequence, `use_ffa_decode` set and the layer in `pattern_layers`
  (default: every layer) runs the pruned decode over the paged cache (BS, SBS, delta,
  use_fp8_residual); every other step -- the prompt, a later multi-token chunk, decode steps of layers
  outside `pattern_layers` or with `use_ffa_decode=False` -- runs exact causal attention over the
  cache's own keys and values dequantized by `ffa_q2_paged_dequant` (the reference attends with
  FlashAttention to the keys its cache returns dequantized from every update, fp8fp8_cache.py:60-69,
  84-89).  The exact attention itself is fp32 torch matmuls, as the reference's is a library call; with
  `paged_exact=True` those steps of fp16 / bf16 models run `PagedQ2Cache.attend` instead, which reads the
  quantized pages themselves, and the pages that samples of a prompt share once (after `reorder_cache`, which
  reads nothing back, every beam's pages for it alone).
* Batch operations of transformers' caches (`batch_repeat_interleave`: samples of a prompt,
  `batch_select_indices`, `reorder_cache`: beams, `crop`) fork and free pages (`ffa_mi355x.pages`) instead of
  copying caches: whole pages are shared, partial last pages copied.  Every layer counts its own pages.

The HF models apply RoPE (their half-split `rotate_half`) before `Cache.update`, so the cache receives
rotated K and appends it with the quantize-append entry point; the fused K-projection + RoPE producer
follows the reference producer's interleaved-pair RoPE instead and serves the benchmark path.

Limits: all sequences of a batch have the same length (no padding).
"""
from __future__ import annotations

import math
import sys
import threading
from pathlib import Path
from typing import Any, Callable, Optional

import torch
from transformers import AttentionInterface
from transformers.cache_utils import Cache, CacheLayerMixin

sys.path.insert(0, str(Path(__file__).resolve().parents[2]))  # ffa-speedtest_amd/
from ffa_mi355x.attend import SharedPrefix  # noqa: E402
from ffa_mi355x.decode import DecodeWorkspace  # noqa: E402
from ffa_mi355x.paged import PAGE, PagedQ2Cache  # noqa: E402
from ffa_mi355x.pages import PagePool  # noqa: E402

__all__ = ["Q2FP8Cache", "Q2FP8PagedLayer", "ffa_q2fp8_attention", "enable_ffa_q2fp8"]

ATTN_NAME = "ffa_q2fp8"
DEFAULT_SETTINGS = dict(use_ffa_decode=True, BS=64, SBS=64, delta=5.0, use_fp8_residual=True, pattern_layers=None,
                        paged_exact=False)
# (layer index, layer) of the update() that ran last on this thread; the attention of that layer
# takes it (and clears it), so a model run without a Q2FP8Cache cannot pick up a stale layer
_current = threading.local()


class Q2FP8PagedLayer(CacheLayerMixin):
    """One layer's paged q2fp8 cache (pools allocated on the first update)."""

    is_sliding = False

    def __init__(self, max_batch_size: int, max_cache_len: int, res_dtype=torch.float8_e4m3fn, page_seed: int = 0):
        super().__init__()
        self.max_batch_size = int(max_batch_size)
        self.max_cache_len = int(max_cache_len)
        self.res_dtype = res_dtype
        self.page_seed = page_seed
        self.pool: Optional[PagedQ2Cache] = None
        self.block_table: Optional[torch.Tensor] = None
        self.seq_lens: Optional[torch.Tensor] = None
        self.seq_len = 0
        self._workspace: Optional[DecodeWorkspace] = None
        self.pages: Optional[PagePool] = None  # from the first batch operation on: pages are shared and counted
        self.shared: Optional[SharedPrefix] = None

    @property
    def capacity(self) -> int:
        return self.block_table.shape[1] * PAGE

    def lazy_initialization(self, key_states: torch.Tensor, value_states: torch.Tensor) -> None:
        B, HKV, _, D = key_states.shape
        if D != 128:
            raise NotImplementedError(f"head_dim {D}: the q2fp8 decode implements 128")
        if B > self.max_batch_size:
            raise ValueError(f"batch {B} exceeds max_batch_size {self.max_batch_size}")
        self.dtype, self.device = key_states.dtype, key_states.device
        npg = -(-self.max_cache_len // PAGE)
        # V pages hold fp16(V): the decode's P.V operand, converted once per token at append
        self.pool = PagedQ2Cache(B * npg, HKV, self.device, res_dtype=self.res_dtype, v_dtype=torch.float16)
        # a seeded permutation of the pool: sequences' pages are scattered as in a serving cache
        perm = torch.randperm(B * npg, generator=torch.Generator().manual_seed(self.page_seed))
        self.block_table = perm.view(B, npg).to(torch.int32).to(self.device)
        self.seq_lens = torch.zeros(B, dtype=torch.int32, device=self.device)
        self.seq_len = 0
        self.is_initialized = True

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, *args, **kwargs):
        """Append K / V [B, HKV, Tn, 128] (rotated) at the current length; returns them unchanged."""
        if not self.is_initialized:
            self.lazy_initialization(key_states, value_states)
        B, HKV, Tn, D = key_states.shape
        if self.pages is not None and self.seq_len == 0 and 0 < B <= self.max_batch_size:
            self._empty_rows(B)
        if B != self.block_table.shape[0] or HKV != self.pool.HKV:
            raise ValueError("key_states do not match the cache's batch / KV heads")
        if self.seq_len + Tn > self.capacity:
            raise ValueError(f"cache holds {self.capacity} tokens, {self.seq_len + Tn} requested")
        pos = torch.full((B,), self.seq_len, dtype=torch.int32, device=self.device)
        first, end = -(-self.seq_len // PAGE), -(-(self.seq_len + Tn) // PAGE)
        if self.pages is not None and end > first:
            self.pages.extend(self.block_table, self.seq_lens, Tn)
        try:
            self.pool.append(key_states.transpose(1, 2).contiguous(), value_states.transpose(1, 2).contiguous(), pos,
                             self.block_table)
        except Exception:  # refused: the new pages hold nothing
            self._drop_pages(first, end)
            raise
        self.seq_len += Tn
        self.seq_lens.fill_(self.seq_len)
        self.last_query_len = Tn
        return key_states, value_states

    def workspace(self, HQ: int, BS: int, SBS: int, dtype) -> DecodeWorkspace:
        B = self.block_table.shape[0]
        ws = self._workspace
        if ws is None or not ws.matches(B, HQ, self.pool.HKV, self.capacity, BS, SBS, self.device, dtype):
            ws = self._workspace = DecodeWorkspace(B, HQ, self.pool.HKV, self.capacity, BS, SBS, self.device, dtype)
        return ws

    def get_mask_sizes(self, query_length: int) -> tuple[int, int]:
        return self.seq_len + query_length, 0

    def get_seq_length(self) -> int:
        return self.seq_len

    def get_max_length(self) -> int:
        return self.max_cache_len

    def reset(self) -> None:
        self.seq_len = 0
        self.shared = None
        if self.seq_lens is not None:
            self.seq_lens.zero_()
        if self.pages is not None:
            self.pages.refs.zero_()
            self.block_table.fill_(-1)

    # ------------------------------------------------------------------ batch operations
    def _empty_rows(self, B: int) -> None:
        """Rows for a batch of B, where no row holds a page: a new prompt may have another batch than the samples and
        beams before it."""
        if B != self.block_table.shape[0]:
            self.block_table = torch.full((B, self.block_table.shape[1]), -1, dtype=torch.int32, device=self.device)
            self.seq_lens = torch.zeros(B, dtype=torch.int32, device=self.device)
            self.shared = None

    def _count_pages(self) -> PagePool:
        """From fixed rows of pages to counted ones, in a pool that holds max_batch_size whole sequences and the copies
        of their last pages that a fork makes before the parents go."""
        if self.pages is None:
            old, npg = self.pool, self.block_table.shape[1]
            self.pool = PagedQ2Cache(self.max_batch_size * (npg + 1), old.HKV, self.device, res_dtype=old.res_dtype,
                                     v_dtype=old.v_dtype)
            for new, t in zip(self.pool.pools(), old.pools()):
                new[: old.P].view(torch.uint8).copy_(t.view(torch.uint8))
            self.block_table[:, -(-self.seq_len // PAGE):] = -1
            self.pages = PagePool([self.pool])
            self.pages.hold(self.block_table, self.seq_lens)
        return self.pages

    def _drop_pages(self, first: int, end: int) -> None:
        """Free the pages of columns [first, end) of every row."""
        if self.pages is not None and first < end:
            tail = self.block_table[:, first:end].contiguous()
            self.pages.free(tail, torch.full_like(self.seq_lens, tail.shape[1] * PAGE))
            self.block_table[:, first:end] = -1

    def _select(self, indices: torch.Tensor, check: bool) -> None:
        if not self.is_initialized:
            return
        n = int(indices.numel())
        if not 0 < n <= self.max_batch_size:
            raise ValueError(f"a batch of {n}: the cache holds 1 to {self.max_batch_size} sequences")
        pages = self._count_pages()
        child = pages.fork(self.block_table, self.seq_lens, indices.reshape(-1), check=check)
        pages.free(self.block_table, self.seq_lens, check=check)
        self.block_table = child
        self.seq_lens = torch.full((n,), self.seq_len, dtype=torch.int32, device=self.device)
        self.shared = None

    def batch_repeat_interleave(self, repeats: int) -> None:
        """Every sequence `repeats` times (samples of a prompt); the copies share its whole pages."""
        if self.is_initialized:
            self._select(torch.arange(self.block_table.shape[0]).repeat_interleave(repeats), True)
            self.shared = SharedPrefix(self.block_table, self.seq_lens)

    def batch_select_indices(self, indices: torch.Tensor) -> None:
        """Sequences `indices` (a boolean mask or indices, from the end where negative) in this order."""
        if self.is_initialized:
            rows = torch.arange(self.block_table.shape[0])[indices.cpu()]
            self._select(rows, True)
            self.shared = SharedPrefix(self.block_table, self.seq_lens)

    def reorder_cache(self, beam_idx: torch.LongTensor) -> None:
        """Beam search: beam i continues beam beam_idx[i] (within the batch).  Does not synchronise, and makes no plan
        of the shared pages (a read of the table): exact steps then read every beam's pages for it alone."""
        self._select(beam_idx, False)

    def crop(self, tokens_to_remove: int) -> None:
        """Remove the newest -tokens_to_remove tokens (or, where positive, those past that length)."""
        if not self.is_initialized or tokens_to_remove == 0:
            return
        length = min(tokens_to_remove, self.seq_len) if tokens_to_remove > 0 else max(self.seq_len + tokens_to_remove, 0)
        first, end = -(-length // PAGE), -(-self.seq_len // PAGE)
        self._drop_pages(first, end)
        cut = length < self.seq_len
        self.seq_len = length
        self.seq_lens.fill_(length)
        if self.pages is None or not cut:
            return
        shared = self.shared
        if length % PAGE:  # the last page may be one that others share: tokens are appended to a copy
            self._select(torch.arange(self.block_table.shape[0]), True)
        if shared is not None:  # pages that are gone are shared no more, also where the length is a page's end
            self.shared = SharedPrefix(self.block_table, self.seq_lens, group_sizes=shared.sizes)

    def offload(self):
        raise NotImplementedError("offloading is not supported by the paged q2fp8 cache")

    def prefetch(self):
        pass


class Q2FP8Cache(Cache):
    """Paged q2fp8 KV cache for a whole model (one Q2FP8PagedLayer per decoder layer)."""

    def __init__(self, num_layers: int, max_batch_size: int, max_cache_len: int, res_dtype=torch.float8_e4m3fn,
                 page_seed: int = 0):
        layers = [Q2FP8PagedLayer(max_batch_size, max_cache_len, res_dtype, page_seed + i) for i in range(num_layers)]
        super().__init__(layers=layers)

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, layer_idx: int, *args, **kwargs):
        out = self.layers[layer_idx].update(key_states, value_states)
        _current.entry = (layer_idx, self.layers[layer_idx])  # taken by ffa_q2fp8_attention of that layer
        return out


def exact_attention(query: torch.Tensor, layer: Q2FP8PagedLayer, scaling: float) -> torch.Tensor:
    """Causal attention of the L newest query tokens [B, HQ, L, D] over the whole cache (positions
    seq_len - L .. seq_len - 1 see the keys up to their own position), on the keys and values the
    cache holds, dequantized in the model dtype (fp32 arithmetic, contiguous operands).  Returns
    [B, L, HQ, D]."""
    B, HQ, L, D = query.shape
    S = layer.seq_len
    k, v = layer.pool.dequantize(layer.block_table, S, layer.seq_lens, out_dtype=layer.dtype)
    G = HQ // layer.pool.HKV
    k = k[:, :S].float().transpose(1, 2).repeat_interleave(G, dim=1).contiguous()  # [B, HQ, S, D]
    v = v[:, :S].float().transpose(1, 2).repeat_interleave(G, dim=1).contiguous()
    s = torch.matmul(query.float().contiguous(), k.transpose(2, 3).contiguous()) * scaling
    qpos = torch.arange(S - L, S, device=s.device)[:, None]
    s = s.masked_fill(torch.arange(S, device=s.device)[None, :] > qpos, float("-inf"))
    p = torch.softmax(s, dim=-1)
    return torch.matmul(p, v).to(query.dtype).transpose(1, 2).contiguous()


def ffa_q2fp8_attention(module, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, attention_mask,
                        scaling: Optional[float] = None, dropout: float = 0.0, **kwargs):
    """Attention of one layer (the transformers attention-function signature); query [B, HQ, L, D] rotated.

    L == 1 with use_ffa_decode and the layer in pattern_layers: the pruned q2fp8 decode over the
    layer's paged cache (modeling_llama.py:293-321's branch); otherwise exact causal attention over
    the cache's keys and values (:322-337), dequantized, or with paged_exact as they lie in the pages."""
    settings = dict(DEFAULT_SETTINGS)
    settings.update(getattr(module.config, "attn_settings", None) or {})
    entry = getattr(_current, "entry", None)
    _current.entry = None
    if entry is None or not isinstance(entry[1], Q2FP8PagedLayer):
        raise RuntimeError("ffa_q2fp8 attention needs a Q2FP8Cache passed as past_key_values (with use_cache)")
    layer_idx, layer = entry
    if getattr(module, "layer_idx", layer_idx) != layer_idx:
        raise RuntimeError(f"ffa_q2fp8 attention of layer {module.layer_idx} after the cache update of layer "
                           f"{layer_idx}")
    B, HQ, L, D = query.shape
    scale = scaling if scaling is not None else 1.0 / math.sqrt(D)
    pattern = settings.get("pattern_layers")
    if pattern is not None and not isinstance(pattern, (list, tuple)):
        raise TypeError("pattern_layers must be a list of layer indices")
    if L == 1 and settings["use_ffa_decode"] and (pattern is None or layer_idx in pattern):
        ws = layer.workspace(HQ, settings["BS"], settings["SBS"], query.dtype)
        layer.pool.decode(query[:, :, 0, :].contiguous(), layer.block_table, layer.seq_lens, T=layer.capacity,
                          scale=scale, BS=settings["BS"], SBS=settings["SBS"], delta=settings["delta"],
                          use_fp8_residual=settings["use_fp8_residual"], workspace=ws)
        out = ws.o.unsqueeze(1)  # [B, 1, HQ, D]
        hook: Optional[Callable] = settings.get("on_decode")
        if hook is not None:
            hook(layer_idx, query[:, :, 0, :], out[:, 0], layer)
        return out, None
    if settings["paged_exact"] and query.dtype in (torch.float16, torch.bfloat16):
        out = layer.pool.attend(query.transpose(1, 2).contiguous(), layer.block_table, layer.seq_lens, T=layer.seq_len,
                                scale=scale, shared=layer.shared)
    else:
        out = exact_attention(query, layer, scale)
    hook = settings.get("on_exact")
    if hook is not None:
        hook(layer_idx, query, out, layer)
    return out, None


def enable_ffa_q2fp8(model, **attn_settings: Any) -> None:
    """Route the model's attention through ffa_q2fp8_attention (registered once) with these settings
    (BS, SBS, delta, use_fp8_residual, use_ffa_decode, pattern_layers, paged_exact; optional
    on_decode(layer_idx, q, o, cache_layer) and on_exact(layer_idx, q, o, cache_layer) observers)."""
    AttentionInterface.register(ATTN_NAME, ffa_q2fp8_attention)
    cfg = model.config
    cfg.attn_settings = {**DEFAULT_SETTINGS, **attn_settings}
    if hasattr(model, "set_attn_implementation"):
        model.set_attn_implementation(ATTN_NAME)
    else:
        cfg._attn_implementation = ATTN_NAME
