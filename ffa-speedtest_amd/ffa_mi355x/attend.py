"""Exact attention over the paged caches (no pruning), with shared leading pages read once per group.

The reference attends to its cache's dequantized keys with a library call whenever it does not prune
(ffa-fp8fp8/e2e/modeling_llama.py:322-337).  Here the kernel reads the quantized pages themselves: L query
tokens per sequence (a decode step, drafted tokens, a prompt's chunk), causal at the sequence's end.
`PagedQ2Cache.attend` and `PagedKfmtCache.attend` call `run_attend`.
"""
from __future__ import annotations

import ctypes
import math
from contextlib import nullcontext

import torch

from . import _native as N
from .decode import HEAD_DIM

PAGE = 64
_SCALE = 1.0 / math.sqrt(HEAD_DIM)
_FORMATS = {"q2": N.PAGES_Q2, "nvfp4": N.PAGES_NVFP4, "nf4": N.PAGES_NF4}


class SharedPrefix:
    """Which sequences of a batch share leading pages: consecutive sequences whose block tables start with the
    same page ids (forked from one prompt).

    group_sizes: sequences per group, in batch order (their sum is the batch); by default a sequence belongs to
    the group before it if its first page is that group's.  A group's shared pages are the longest run of equal
    leading page ids that lie wholly inside every member (seq_lens): one level, so requests behind one short system
    prompt and each with samples of its own are better given as groups of samples (group_sizes).  Reads block_table and seq_lens on the host
    (once: make it when sequences are forked, not per step).  It stays valid while the members keep those pages;
    their own pages and lengths may change, so it serves every step until a fork, free or compaction."""

    def __init__(self, block_table: torch.Tensor, seq_lens: torch.Tensor, group_sizes=None):
        if block_table.ndim != 2 or tuple(seq_lens.shape) != (block_table.shape[0],):
            raise ValueError("block_table must be [B, n] and seq_lens [B]")
        B, cols = block_table.shape
        if B == 0 or cols == 0:
            raise ValueError("empty block table")
        table, lens = block_table.cpu().tolist(), seq_lens.cpu().tolist()
        if group_sizes is None:
            group_sizes = []
            for b in range(B):
                if b and table[b][0] == table[b - 1][0] and min(lens[b], lens[b - 1]) >= PAGE:
                    group_sizes[-1] += 1
                else:
                    group_sizes.append(1)
        sizes = [int(n) for n in group_sizes]
        if any(n <= 0 for n in sizes) or sum(sizes) != B:
            raise ValueError("group_sizes must be positive and sum to the batch")
        start, pages, group = [0], [], []
        for g, n in enumerate(sizes):
            b = start[-1]
            members = table[b:b + n]
            most = max(0, min(min(lens[b:b + n]) // PAGE, cols)) if n > 1 else 0
            same = 0
            while same < most and all(row[same] == members[0][same] for row in members):
                same += 1
            pages.append(same)
            group += [g] * n
            start.append(b + n)
        self.B, self.sizes, self.pages = B, sizes, pages
        self.device = block_table.device
        self._start_host = (ctypes.c_int32 * len(start))(*start)
        self._pages_host = (ctypes.c_int32 * len(pages))(*pages)
        dev = torch.tensor(start + pages + group, dtype=torch.int32).to(self.device)
        self._dev = dev
        self.most = max(pages)
        at = dev.data_ptr()
        self._args = (len(sizes), at, at + 4 * len(start), at + 4 * (len(start) + len(pages)),
                      ctypes.addressof(self._start_host), ctypes.addressof(self._pages_host),
                      sum(max(-(-n // PAGE) - pages[g], 0) for n, g in zip(lens, group)))

    def __len__(self) -> int:
        return len(self.sizes)


def _int32(t: torch.Tensor, device: torch.device) -> torch.Tensor:
    if t.dtype is torch.int32 and t.device == device and t.is_contiguous():
        return t
    return t.to(device=device, dtype=torch.int32).contiguous()


def _on(device: torch.device):
    """The device's context, where another one is current."""
    return nullcontext() if device.index in (None, torch.cuda.current_device()) else torch.cuda.device(device)


def _call(a: N.AttendArgs, dev: torch.device) -> int:
    lib, ref = N.lib(), ctypes.byref(a)
    need = lib.ffa_paged_attend_scratch(ref)
    if need:
        scratch = torch.empty(need, dtype=torch.uint8, device=dev)
        a.scratch, a.scratch_bytes = scratch.data_ptr(), need
    return lib.ffa_paged_attend(ref, N.stream_of(dev))


def run_attend(fmt, q, k, k_scale, k_zero, k_res, v, block_table, seq_lens=None, *, T=None, q_lens=None, scale=None,
               use_fp8_residual=True, shared: SharedPrefix | None = None, out=None) -> torch.Tensor:
    """Exact attention of q [B, L, HQ, 128] (or [B, HQ, 128]) over the page pools of one format.

    Query token i of sequence b sits at position seq_lens[b] - q_lens[b] + i and sees the keys up to its own;
    query tokens i >= q_lens[b] (padding of a batch of uneven chunks) and rows that see no key give zeros.
    seq_lens counts the query tokens, which are in the cache already.  T: the largest length (read from the
    device when not given); a capacity serves, and lets a captured graph's sequences grow.
    Returns out (allocated unless given) in q's shape and type."""
    if q.ndim not in (3, 4):
        raise ValueError(f"q must be [B, L, HQ, 128] or [B, HQ, 128], got {tuple(q.shape)}")
    shape = q.shape
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise NotImplementedError(f"attend computes on fp16 operands: q must be fp16 or bf16, got {q.dtype}")
    if shape[-1] != HEAD_DIM:
        raise NotImplementedError(f"head_dim {shape[-1]} is not supported (this build implements {HEAD_DIM})")
    B, HQ = shape[0], shape[-2]
    L = shape[1] if q.ndim == 4 else 1
    P, HKV = v.shape[0], v.shape[1]
    if B == 0 or L == 0 or HQ == 0 or HQ % HKV:
        raise ValueError(f"q {tuple(shape)} needs sequences, query tokens and a multiple of {HKV} heads")
    dev = q.device
    if dev.type != "cuda" or v.device != dev:
        raise ValueError(f"q is on {dev}, the cache on {v.device}: both must be on one GPU")
    q = q.contiguous()
    if q.data_ptr() % 16:
        q = q.clone()
    if block_table.ndim != 2 or block_table.shape[0] != B:
        raise ValueError("block_table must be [B, >= ceil(T/64)]")
    block_table = _int32(block_table, dev)
    if seq_lens is not None:
        if seq_lens.shape != (B,):
            raise ValueError("seq_lens must be [B]")
        if T is None:
            T = int(seq_lens.max().item())
        seq_lens = _int32(seq_lens, dev)
    elif T is None:
        raise ValueError("give T or seq_lens")
    if q_lens is not None:
        if q_lens.shape != (B,):
            raise ValueError("q_lens must be [B]")
        q_lens = _int32(q_lens, dev)
    T, cols = int(T), block_table.shape[1]
    if cols * PAGE < T:
        raise ValueError("block_table must be [B, >= ceil(T/64)]")
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != shape or out.dtype != q.dtype or out.device != dev or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor of q's shape, type and device")
    if T <= 0:  # a batch of empty sequences
        return out.zero_()
    res = k_res if use_fp8_residual else None
    groups = (0, None, None, None, None, None, 0)
    if shared is not None:
        if shared.B != B or shared.device != dev:
            raise ValueError("shared was made for another batch")
        if shared.most > cols:
            raise ValueError("shared pages exceed the block table")
        groups = shared._args
    a = N.AttendArgs(  # in the order of the fields: one call instead of thirty assignments
        q.data_ptr(), N.dtype_code(q.dtype), _FORMATS[fmt], k.data_ptr(), k_scale.data_ptr(), N.ptr(k_zero), N.ptr(res),
        N.DT_NONE if res is None else N.dtype_code(res.dtype), v.data_ptr(), N.dtype_code(v.dtype), block_table.data_ptr(),
        cols, P, N.ptr(seq_lens), N.ptr(q_lens), B, T, L, HQ, HKV, _SCALE if scale is None else float(scale), *groups,
        out.data_ptr(), None, 0)
    if dev.index == torch.cuda.current_device():
        rc = _call(a, dev)
    else:
        with torch.cuda.device(dev):
            rc = _call(a, dev)
    N.check(rc, "ffa_paged_attend")
    return out
