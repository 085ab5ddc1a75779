"""Exact attention over mxfp4 pages of batches with padded query tokens: zeros for those, and for the others what they give
without padding, whatever the padding holds."""
import math

import numpy as np
import pytest
import torch

import mxfp4_ref as R
from attend_ref import assert_close, reference

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(128)


# query tokens, heads of the one KV head, copies of the batch: few rows by sixteens, two row tiles, 64, 128 and 256 rows
@pytest.mark.parametrize("L,HQ,copies", [(4, 4, 1), (5, 4, 1), (5, 4, 200), (12, 4, 100), (25, 4, 60), (60, 4, 30)])
@pytest.mark.parametrize("lens", [[700, 130, 64, 900], [4000, 3300, 100, 5000]])
def test_padding_does_not_count(gpu, L, HQ, copies, lens):
    g = torch.Generator().manual_seed(L)
    B = len(lens)
    ql = [L, max(L // 2, 1), 1, L - 1]
    npg = [-(-n // 64) for n in lens]
    cache = R.make_cache(sum(npg) + 1, 1, gpu, seed=L)
    ids = torch.randperm(sum(npg) + 1, generator=g).to(torch.int32)
    table, at = torch.full((B, max(npg)), -1, dtype=torch.int32), 0
    for b, n in enumerate(lens):
        table[b, :npg[b]] = ids[at:at + npg[b]]
        at += npg[b]
        x = torch.randn(2, 1, n, 1, 128, generator=g).to(gpu)
        cache.append(x[0], x[1], torch.zeros(1, dtype=torch.int32, device=gpu), table[b:b + 1].to(gpu), True)
    q = torch.randn(B, L, HQ, 128, generator=g).bfloat16()
    args = [t.to(gpu).repeat(copies, *[1] * (t.ndim - 1)) for t in (q, table, torch.tensor(lens), torch.tensor(ql))]
    outs = []
    for pad in (0.0, float("nan"), float("inf"), 1e30, 3.0):
        x = args[0].clone()
        for b, n in enumerate(ql):
            x.view(copies, B, L, HQ, 128)[:, b, n:] = pad
        outs.append(cache.attend(x, args[1], args[2], q_lens=args[3]))
        assert torch.equal(outs[-1], outs[0])
    for c in sorted({0, copies - 1}):
        for b, n in enumerate(ql):
            out = outs[0].view(copies, B, L, HQ, 128)[c, b]
            assert (out[n:] == 0).all()
            kk, vv = R.logical_kv(cache, table[b, :npg[b]].tolist())
            rows = sorted({0, n // 2, n - 1})
            o, bound = reference(q[b], kk, vv, lens[b], n, SCALE, rows)
            assert_close(out[rows], o[rows], bound[rows], q.dtype, f"sequence {b}")
    # no query token of a whole batch
    assert (cache.attend(args[0], args[1], args[2], q_lens=torch.zeros_like(args[3])) == 0).all()
