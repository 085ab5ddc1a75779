"""Rotary positions with several axes (time, height and width of video; height and width of images; plain text).

The reference rotates keys by cos / sin tables of one axis (ffa-q2fp8/fused_kproj_rope_q2fp8.py:10-37, here
`rope.py`).  `AxisRope` keeps the frequency and the axis of each of the 64 pairs of channels; `rotate` turns given
queries and keys (both in one launch), and `PagedMXFP4Cache.append_rotary` turns while it stores.
"""
from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd import forward_ad

from . import _native as N
from .attend import _on
from .decode import HEAD_DIM

PAIRS = HEAD_DIM // 2
_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
_NO_STRIDES = (0, 0, 0)


def _launch(fn, args: ctypes.Structure, device: torch.device) -> int:
    if device.index == torch.cuda.current_device():
        return fn(ctypes.byref(args), N.stream_of(device))
    with _on(device):
        return fn(ctypes.byref(args), N.stream_of(device))


def _strides(x: torch.Tensor) -> tuple[int, int, int]:
    """Strides of [B, T, H] (elements), 0 where a dimension has one entry: torch keeps any number there, contiguous or not."""
    (b, t, h, _), (sb, st, sh, _) = x.shape, x.stride()
    return (sb if b > 1 else 0, st if t > 1 else 0, sh if h > 1 else 0)


def _dense(shape) -> tuple[int, int, int]:
    """The same of contiguous rows."""
    b, t, h, _ = shape
    return (HEAD_DIM * h * t if b > 1 else 0, HEAD_DIM * h if t > 1 else 0, HEAD_DIM if h > 1 else 0)


def strided_rows(x: torch.Tensor) -> tuple[torch.Tensor, tuple[int, int, int]]:
    """x [B, T, H, 128] and its strides (elements; 0 where a dimension has one entry) as the kernels take rows: 128
    contiguous channels, every address a multiple of 16 bytes.  Others are copied."""
    if x.is_contiguous() and x.data_ptr() % 16 == 0:
        return x, _dense(x.shape)
    step = 16 // x.element_size()
    strides = _strides(x)
    if x.stride(3) == 1 and not (strides[0] % step or strides[1] % step or strides[2] % step or x.data_ptr() % 16):
        return x, strides
    return x.clone(memory_format=torch.contiguous_format), _dense(x.shape)


def rows_like(x: torch.Tensor) -> torch.Tensor:
    """Contiguous rows of x's shape and type (empty_like: a third of empty's time on the host)."""
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _nested(extent: int, dims) -> bool:
    """Whether pieces of `extent` bytes repeated along (stride, entries) lie apart because each stride spans all of the
    smaller ones."""
    for stride, n in sorted(dims):
        if stride < extent:
            return False
        extent += stride * (n - 1)
    return True


def _side_by_side(q: torch.Tensor, k: torch.Tensor) -> bool:
    """Whether q and k are two blocks of memory, or lie one behind the other in each token, as rows_overlap would find out (a
    fifth of its 10 us on the host)."""
    es = q.element_size()
    apart = (k.data_ptr() - q.data_ptr()) // es
    if q.is_contiguous() and k.is_contiguous():
        return apart >= q.numel() or -apart >= k.numel()
    (B, T, HQ, _), HK = q.shape, k.shape[2]
    (qb, qt, qh, _), (kb, kt, kh, _) = q.stride(), k.stride()
    if qh < HEAD_DIM or kh < HEAD_DIM:
        return False
    q_end, k_end = (HQ - 1) * qh + HEAD_DIM, (HK - 1) * kh + HEAD_DIM
    token = apart + k_end if apart >= q_end else q_end - apart
    if apart < q_end and -apart < k_end or (T > 1 and (qt != kt or qt < token)):
        return False
    return B == 1 or (qb == kb and qb >= (qt * (T - 1) if T > 1 else 0) + token)


def rows_overlap(*xs: torch.Tensor) -> bool:
    """Whether any two rows of one tensor or two, [B, T, H, 128] with contiguous channels, have a byte in common."""
    xs = sorted((x for x in xs if x.numel()), key=lambda x: x.data_ptr())
    if not xs:
        return False
    es = xs[0].element_size()
    row = HEAD_DIM * es
    dims = [[(s * es, n) for s, n in zip(_strides(x), x.shape)] for x in xs]
    if all(_nested(row, [d for d in ds if d[1] > 1]) for ds in dims):
        if len(xs) == 1:
            return False
        apart = xs[1].data_ptr() - xs[0].data_ptr()
        # one behind the other as a whole, or, as in a joined projection, within each sequence, token or both
        for outer in ((), (0,), (1,), (0, 1)):
            if any(dims[0][i] != dims[1][i] for i in outer):
                continue
            ends = [row + sum(s * (n - 1) for i, (s, n) in enumerate(ds) if i not in outer) for ds in dims]
            if apart >= ends[0] and _nested(apart + ends[1], [dims[0][i] for i in outer if dims[0][i][1] > 1]):
                return False
    starts = []  # of every row
    for x, ds in zip(xs, dims):
        b, t, h = (torch.arange(n) * s for s, n in ds)
        starts.append((x.data_ptr() + b[:, None, None] + t[:, None] + h).reshape(-1))
    return bool((torch.cat(starts).sort().values.diff() < row).any())


class AxisRope:
    """Rotary positions of 128 channels: pair j of a token turns by positions[axis of j] * frequency j.

    sections: pairs of each axis, 64 in all.  order: "blocks" gives axis 0 the first sections[0] pairs, axis 1 the
    next ones, ...; "cycled" gives the pairs to the axes in turn while they have pairs left.
    pairs: "half" turns channels (j, j + 64), as transformers' rotate_half; "adjacent" (2 j, 2 j + 1).
    base: frequency j is base^(-j / 64); inv_freq [64] gives other ones (scaled or stretched).
    """

    def __init__(self, sections, base: float = 10000.0, device="cuda", *, pairs: str = "half", order: str = "blocks",
                 inv_freq=None):
        sections = [int(n) for n in sections]
        if not sections or min(sections) < 0 or sum(sections) != PAIRS:
            raise ValueError(f"sections must sum to {PAIRS} pairs, got {sections}")
        if pairs not in ("half", "adjacent"):
            raise ValueError('pairs must be "half" or "adjacent"')
        if order not in ("blocks", "cycled"):
            raise ValueError('order must be "blocks" or "cycled"')
        if inv_freq is None:
            if not base > 0:
                raise ValueError("base must be positive")
            freq = [float(base) ** (-j / PAIRS) for j in range(PAIRS)]
        else:
            freq = torch.as_tensor(inv_freq).detach().double().reshape(-1).tolist()
            if len(freq) != PAIRS:
                raise ValueError(f"inv_freq must hold {PAIRS} frequencies, got {len(freq)}")
        if order == "blocks":
            axis = [a for a, n in enumerate(sections) for _ in range(n)]
        else:
            axis, left = [], list(sections)
            while len(axis) < PAIRS:
                for a in range(len(sections)):
                    if left[a]:
                        axis.append(a)
                        left[a] -= 1
        self.sections, self.axes, self.axis = sections, len(sections), axis
        self.inv_freq = freq
        self.adjacent = pairs == "adjacent"
        self.device = torch.device(device)
        turns = torch.tensor([f / (2 * math.pi) for f in freq], dtype=torch.float64)
        # ffa_rope_pair: {double turns; int64 axis}
        self.table = torch.stack([turns.view(torch.int64), torch.tensor(axis)], 1).contiguous().to(self.device)

    def _positions(self, positions: torch.Tensor, B: int, T: int, dev) -> tuple[torch.Tensor, int, int]:
        """positions [axes, B, T], [axes, T] for every sequence, or [B, T] of one axis -> (them, strides)."""
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
        if positions.device != dev:
            raise ValueError(f"positions are on {positions.device}, the rows on {dev}")
        shape = tuple(positions.shape)
        if shape == (self.axes, B, T):
            if positions.is_contiguous():
                return positions, B * T, T
            p = positions
        elif shape == (self.axes, T):
            p = positions[:, None].expand(self.axes, B, T)
        elif self.axes == 1 and shape == (B, T):
            p = positions[None]
        else:
            raise ValueError(f"positions must be [{self.axes}, {B}, {T}] or [{self.axes}, {T}], got {shape}")
        if T > 1 and p.stride(2) != 1:
            p = p.contiguous()
        return p, p.stride(0), p.stride(1)

    def _check(self, x: torch.Tensor, what: str) -> torch.Size:
        shape = x.shape
        if len(shape) != 4 or shape[3] != HEAD_DIM:
            raise ValueError(f"{what} must be [B, T, H, {HEAD_DIM}], got {tuple(shape)}")
        if x.dtype not in _DTYPES:
            raise NotImplementedError(f"{what} must be fp16, bf16 or fp32, got {x.dtype}")
        if self.table.device != x.device or not x.is_cuda:
            raise ValueError(f"{what} is on {x.device}, the rotation on {self.table.device}: both must be on one GPU")
        return shape

    @staticmethod
    def _rows(x: torch.Tensor, inplace: bool):
        """What the kernel reads and writes for x: input, strides, output, strides."""
        src, st = strided_rows(x)
        if not inplace:
            return src, st, rows_like(x), _dense(x.shape)
        if src is not x:
            raise ValueError("rows turned in place must have contiguous channels and 16-byte aligned strides")
        if not x.is_inference():
            torch.autograd.graph.increment_version(x)  # a graph that saved x must not use it turned
        return x, st, x, st

    def _run(self, positions, q, k, inverse, inplace):
        dev, dtype = q.device, q.dtype
        B, T, HQ, _ = q.shape
        pos, pos_axis, pos_batch = self._positions(positions, B, T, dev)
        q_in, qs, q_out, qo = self._rows(q, inplace)
        HKV, k_in, ks, k_out, ko = 0, None, _NO_STRIDES, None, _NO_STRIDES
        if k is not None:
            HKV = k.shape[2]
            k_in, ks, k_out, ko = self._rows(k, inplace)
        outs = (q_out,) if k is None else (q_out, k_out)
        if B == 0 or T == 0 or HQ + HKV == 0:
            return outs
        if HQ == 0:  # k alone, in q's place
            q_in, qs, q_out, qo, HQ, HKV = k_in, ks, k_out, ko, HKV, 0
        a = N.RopeAxesArgs(
            q_in.data_ptr(), q_out.data_ptr(), N.ptr(k_in), N.ptr(k_out), N.dtype_code(dtype), B, T, HQ, HKV, *qs, *qo, *ks, *ko,
            self.table.data_ptr(), pos.data_ptr(), pos.dtype is torch.int64, self.axes, pos_axis, pos_batch, self.adjacent,
            inverse)
        N.check(_launch(N.lib().ffa_rope_axes, a, dev), "ffa_rope_axes")
        return outs

    def rotate(self, positions: torch.Tensor, q: torch.Tensor, k: torch.Tensor | None = None, *, inverse: bool = False,
               inplace: bool = False):
        """q [B, T, H, 128] (and k, with heads of its own) turned by positions [axes, B, T] (or [axes, T] for every
        sequence; int32 or int64), angles in 64 bits, one rounding to the rows' type.  inverse: turned back, which is
        also the gradient; `rotate` records it where q or k needs one, and turns tangents of forward mode with them.  inplace: into q and k themselves, no two rows of
        which may overlap.
        Returns q, or (q, k) where k is given."""
        B, T, _, _ = self._check(q, "q")
        if k is not None:
            Bk, Tk, _, _ = self._check(k, "k")
            if Bk != B or Tk != T or k.dtype != q.dtype:
                raise ValueError("q and k must have the same sequences, tokens and type")
        if inplace and (rows_overlap(q) if k is None else not _side_by_side(q, k) and rows_overlap(q, k)):
            raise ValueError("rows turned in place must not overlap (expanded ones, or q and k in each other's memory)")
        if _differentiated(q) or (k is not None and _differentiated(k)):
            if inplace:
                raise ValueError("rows that need gradients are not turned in place")
            got = _Rotate.apply(self, positions, inverse, q, k)
        else:
            got = self._run(positions, q, k, inverse, inplace)
        return got[0] if k is None else got


def _differentiated(x: torch.Tensor) -> bool:
    """Whether x's gradient is recorded, or x has a tangent (forward mode)."""
    if x.requires_grad and torch.is_grad_enabled():
        return True
    # (asked outside of forward mode's levels, which torch keeps to itself, unpack_dual costs half a us and says the same)
    return getattr(forward_ad, "_current_level", 0) >= 0 and forward_ad.unpack_dual(x).tangent is not None


class _Rotate(torch.autograd.Function):
    """rotate with its derivatives: of its gradient the rotation back (linear, so the gradient's own is the rotation again), of
    tangents the rotation."""

    @staticmethod
    def forward(ctx, rope, positions, inverse, q, k):
        ctx.rope, ctx.inverse, ctx.two = rope, inverse, k is not None
        ctx.save_for_backward(positions)
        ctx.save_for_forward(positions)
        return rope._run(positions, q, k, inverse, False)

    @staticmethod
    def backward(ctx, gq, gk=None):
        (positions,) = ctx.saved_tensors
        got = _Rotate.apply(ctx.rope, positions, not ctx.inverse, gq, gk)
        return None, None, None, got[0], got[1] if ctx.two else None

    @staticmethod
    def jvp(ctx, _rope, _positions, _inverse, tq, tk=None):
        (positions,) = ctx.saved_tensors
        return _Rotate.apply(ctx.rope, positions, ctx.inverse, tq, tk if ctx.two else None)
