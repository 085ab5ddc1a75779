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
_FORMATS = {"q2": N.PAGES_Q2, "nvfp4": N.PAGES_NVFP4, "nf4": N.PAGES_NF4}


class SharedPrefix:
    """Which sequences of a batch share leading pages: consecutive sequences whose block tables start with the
    same page ids (forked from one prompt).

    group_sizes: sequences per group, in batch order (their sum is the batch); by default a sequence belongs to
    the group before it if its first page is that group's.  A group's shared pages are the longest run of equal
    leading page ids that lie wholly inside every member (seq_lens).  Reads block_table and seq_lens on the host
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
        self._ptrs = (dev.data_ptr(), dev.data_ptr() + 4 * len(start), dev.data_ptr() + 4 * (len(start) + len(pages)))

    def __len__(self) -> int:
        return len(self.sizes)


def _on(device: torch.device):
    """The device's context, where another one is current."""
    return nullcontext() if device.index in (None, torch.cuda.current_device()) else torch.cuda.device(device)


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
    block_table = block_table.to(device=dev, dtype=torch.int32).contiguous()
    if seq_lens is not None:
        if tuple(seq_lens.shape) != (B,):
            raise ValueError("seq_lens must be [B]")
        if T is None:
            T = int(seq_lens.max().item())
        seq_lens = seq_lens.to(device=dev, dtype=torch.int32).contiguous()
    elif T is None:
        raise ValueError("give T or seq_lens")
    if q_lens is not None:
        if tuple(q_lens.shape) != (B,):
            raise ValueError("q_lens must be [B]")
        q_lens = q_lens.to(device=dev, dtype=torch.int32).contiguous()
    T = max(int(T), 1)  # a batch of empty sequences
    if block_table.shape[1] * PAGE < T:
        raise ValueError("block_table must be [B, >= ceil(T/64)]")
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=dev)
    elif out.shape != shape or out.dtype != q.dtype or out.device != dev or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor of q's shape, type and device")
    a = N.AttendArgs()
    a.q, a.q_dtype = q.data_ptr(), N.dtype_code(q.dtype)
    a.format = _FORMATS[fmt]
    a.k, a.k_scale, a.k_zero = k.data_ptr(), k_scale.data_ptr(), N.ptr(k_zero)
    if use_fp8_residual:
        a.k_residual, a.res_dtype = k_res.data_ptr(), N.dtype_code(k_res.dtype)
    else:
        a.res_dtype = N.DT_NONE
    a.v, a.v_dtype = v.data_ptr(), N.dtype_code(v.dtype)
    a.block_table, a.bt_stride, a.num_pages = block_table.data_ptr(), block_table.shape[1], P
    a.seq_lens, a.q_lens = N.ptr(seq_lens), N.ptr(q_lens)
    a.B, a.T, a.L, a.HQ, a.HKV = B, T, L, HQ, HKV
    a.scale = 1.0 / math.sqrt(HEAD_DIM) if scale is None else float(scale)
    if shared is not None:
        if shared.B != B or shared.device != dev:
            raise ValueError("shared was made for another batch")
        if max(shared.pages) > block_table.shape[1]:
            raise ValueError("shared pages exceed the block table")
        a.ngroups = len(shared)
        a.group_start, a.group_pages, a.seq_group = shared._ptrs
        a.group_start_host = ctypes.addressof(shared._start_host)
        a.group_pages_host = ctypes.addressof(shared._pages_host)
    a.out = out.data_ptr()
    lib = N.lib()
    with _on(dev):
        need = lib.ffa_paged_attend_scratch(ctypes.byref(a))
        scratch = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        a.scratch, a.scratch_bytes = N.ptr(scratch), need
        rc = lib.ffa_paged_attend(ctypes.byref(a), N.stream_of(dev))
    N.check(rc, "ffa_paged_attend")
    return out
