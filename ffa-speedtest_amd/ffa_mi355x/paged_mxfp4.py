"""Paged KV cache that holds keys and values in 4 bits (MXFP4; 64-token pages; no reference counterpart).

The other paged caches keep a key's residual in 8 bits and values in 16 (432-456 bytes a token and KV head); this one
keeps both as e2m1 codes with a power of two per 32 channels of a token, 136 bytes:

    k        [P, HKV, 64, 64]   u8  K codes, two channels a byte, in the order of the matrix operands
    k_scale  [P, HKV, 4, 64]    u8  powers of two of the blocks of 32 channels, token by token
    v        [P, HKV, 128, 32]  u8  V codes, two tokens a byte
    v_scale  [P, HKV, 4, 64]    u8

The values that codes and scales stand for, and the codes' places, are stated in include/ffa_mi355x.h; every value is
exact in fp16 and bf16.  block_table[b, i] is the pool page of tokens [64 i, 64 i + 64) of sequence b.
"""
from __future__ import annotations

import ctypes

import torch

from . import _native as N
from .attend import _int32, _on
from .decode import HEAD_DIM
from .paged import PAGE, check_append_fits
from .rope_axes import _NO_STRIDES, AxisRope, _launch, rows_like, strided_rows

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


class PagedMXFP4Cache:
    """Page pools of keys and values in MXFP4, with append (quantize + write), read-back and exact attention."""

    def __init__(self, num_pages, HKV, device):
        self.P, self.HKV = int(num_pages), int(HKV)
        self.device = torch.device(device)
        P, H = self.P, self.HKV
        self.k = torch.zeros((P, H, PAGE, HEAD_DIM // 2), dtype=torch.uint8, device=device)
        self.k_scale = torch.zeros((P, H, 4, PAGE), dtype=torch.uint8, device=device)
        self.v = torch.zeros((P, H, HEAD_DIM, PAGE // 2), dtype=torch.uint8, device=device)
        self.v_scale = torch.zeros((P, H, 4, PAGE), dtype=torch.uint8, device=device)

    def nbytes_per_page(self) -> int:
        return sum(t[0].numel() for t in self.pools())

    def pools(self) -> list[torch.Tensor]:
        """The pools, one page of each per page id."""
        return [self.k, self.k_scale, self.v, self.v_scale]

    # ------------------------------------------------------------------ writes
    def append(self, k: torch.Tensor, v: torch.Tensor | None, pos: torch.Tensor, block_table: torch.Tensor,
               ragged: bool = False, *, values: bool = False, check: bool = True):
        """Quantize k and v [B, Tn, HKV, 128] (fp16, bf16, fp32) and write them at positions pos[b] + n.  ragged: rows
        of the table hold no pages past their own last position (as PagePool leaves them).  values: return
        (k, v) [B, Tn, HKV, 128] as the cache holds them, in k's type.  check=False leaves out the bounds check, which
        reads the table on the host: tokens outside it are then not written.  Results carry no gradients or tangents."""
        got = self._append(None, k, v, pos, block_table, None, None, ragged, values, check)
        return tuple(got[1:]) if values else None

    def append_rotary(self, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor | None, pos: torch.Tensor,
                      block_table: torch.Tensor, rope: AxisRope, positions: torch.Tensor | None = None,
                      ragged: bool = False, *, values: bool = False, check: bool = True):
        """append of k turned by `rope` (in fp32: k is not rounded between), with q [B, Tn, HQ, 128] turned beside it.
        positions [axes, B, Tn] (or [axes, Tn]): by default pos[b] + n on every axis.  Returns q turned (None without
        q), or with values (q, k, v), none of them with gradients or tangents: `rope.rotate` gives a q that has them."""
        got = self._append(q, k, v, pos, block_table, rope, positions, ragged, values, check)
        return tuple(got) if values else got[0]

    def _append(self, q, k, v, pos, block_table, rope, positions, ragged, values, check):
        shape = k.shape
        if len(shape) != 4 or shape[2] != self.HKV or shape[3] != HEAD_DIM:
            raise ValueError("k shape does not match the cache")
        B, Tn, HKV, _ = shape
        if v is not None and v.shape != shape:
            raise ValueError("v must have the shape of k")
        dev = self.k.device
        for x in (k, v, q):
            if x is None:
                continue
            if x.dtype not in _DTYPES:
                raise NotImplementedError(f"rows must be fp16, bf16 or fp32, got {x.dtype}")
            if x.device != dev or not x.is_cuda:
                raise ValueError(f"rows are on {x.device}, the cache on {dev}: both must be on one GPU")
        HQ = 0
        if rope is not None and rope.table.device != dev:
            raise ValueError(f"the rotation is on {rope.table.device}, the cache on {dev}")
        if q is not None:
            shape = q.shape
            if len(shape) != 4 or shape[0] != B or shape[1] != Tn or shape[3] != HEAD_DIM or q.dtype != k.dtype:
                raise ValueError("q must be [B, Tn, HQ, 128] of k's type")
            HQ = shape[2]
        if pos.shape != (B,) or block_table.ndim != 2 or block_table.shape[0] != B:
            raise ValueError("pos must be [B] and block_table [B, n]")
        out_type = k.dtype
        if v is not None and v.dtype != k.dtype:  # fp32 holds both
            k, v = k.float(), v.float()
            q = None if q is None else q.float()
        q_out = None if q is None else rows_like(q)
        k_values = rows_like(k) if values else None
        v_values = rows_like(v) if values and v is not None else None
        if k.numel():
            pos, block_table = _int32(pos, dev), _int32(block_table, dev)
            if check:
                check_append_fits(pos, Tn, block_table, self.P, ragged)
            k, ks = strided_rows(k)
            v, vs = (None, _NO_STRIDES) if v is None else strided_rows(v)
            q, qs = strided_rows(q) if HQ else (None, _NO_STRIDES)
            p, p_axis, p_batch, axes = None, 0, 0, 0
            if rope is not None:
                axes = rope.axes
                if positions is not None:
                    p, p_axis, p_batch = rope._positions(positions, B, Tn, dev)
            a = N.MXFP4AppendArgs(
                k.data_ptr(), N.ptr(v), N.ptr(q), N.dtype_code(k.dtype), B, Tn, HKV, HQ, *ks, *vs, *qs,
                None if rope is None else rope.table.data_ptr(), N.ptr(p), p is not None and p.dtype is torch.int64, axes,
                p_axis, p_batch, rope is not None and rope.adjacent, pos.data_ptr(), block_table.data_ptr(),
                block_table.shape[1], self.P, self.k.data_ptr(), self.k_scale.data_ptr(), self.v.data_ptr(),
                self.v_scale.data_ptr(), N.ptr(q_out), N.ptr(k_values), N.ptr(v_values))
            N.check(_launch(N.lib().ffa_mxfp4_append, a, dev), "ffa_mxfp4_append")
        if k.dtype is not out_type:
            return [x if x is None else x.to(out_type) for x in (q_out, k_values, v_values)]
        return [q_out, k_values, v_values]

    # ------------------------------------------------------------------ reads
    def dequantize(self, block_table: torch.Tensor, T: int, seq_lens: torch.Tensor | None = None,
                   out_dtype: torch.dtype = torch.float32):
        """K and V [B, T', HKV, 128] of the first T tokens of every sequence (T' = T rounded up to a page), exact in
        out_dtype; tokens at or past seq_lens[b] are zeros."""
        if out_dtype not in _DTYPES:
            raise NotImplementedError(f"out_dtype must be fp16, bf16 or fp32, got {out_dtype}")
        dev = self.k.device
        if dev.type != "cuda":
            raise ValueError(f"the cache is on {dev}: it must be on a GPU")
        if block_table.ndim != 2:
            raise ValueError("block_table must be [B, n]")
        block_table = _int32(block_table, dev)
        B = block_table.shape[0]
        Tp = -(-int(T) // PAGE) * PAGE
        if Tp < 0 or Tp > block_table.shape[1] * PAGE:
            raise ValueError("T exceeds the block table")
        if seq_lens is not None:
            if seq_lens.shape != (B,):
                raise ValueError("seq_lens must be [B]")
            seq_lens = _int32(seq_lens, dev)
        k = torch.empty((B, Tp, self.HKV, HEAD_DIM), dtype=out_dtype, device=dev)
        v = torch.empty_like(k)
        if k.numel():
            with _on(dev):
                rc = N.lib().ffa_mxfp4_dequant(
                    self.k.data_ptr(), self.k_scale.data_ptr(), self.v.data_ptr(), self.v_scale.data_ptr(),
                    block_table.data_ptr(), block_table.shape[1], self.P, N.ptr(seq_lens), B, Tp, self.HKV, k.data_ptr(),
                    v.data_ptr(), N.dtype_code(out_dtype), N.stream_of(dev))
            N.check(rc, "ffa_mxfp4_dequant")
        return k, v

    def attend(self, q, block_table, seq_lens=None, **kw) -> torch.Tensor:
        """Exact causal attention of the newest L tokens' q [B, L, HQ, 128] (fp16 or bf16) over the cache: T, q_lens,
        scale, shared (SharedPrefix), out as in attend.run_attend."""
        from .attend import run_attend

        return run_attend("mxfp4", q, self.k, self.k_scale, None, None, self.v, block_table, seq_lens,
                          v_scale=self.v_scale, **kw)
