"""Rows of unusual strides through the rotary and mxfp4 kernels."""
import pytest
import torch

import mxfp4_ref as R
from ffa_mi355x.rope_axes import AxisRope
from test_mxfp4_rows import _odd_batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_one_sequence_of_a_batch_at_an_odd_stride(gpu, dtype):
    q, k = _odd_batch(5, 4, dtype).to(gpu), _odd_batch(5, 2, dtype)
    base = torch.empty(2, 5 * 2 * 128 + 1, dtype=dtype, device=gpu)
    base[:, :-1] = k.reshape(1, -1).to(gpu)
    k = base[:, :-1].view(2, 5, 2, 128)[:1]
    assert k.is_contiguous() and k.stride(0) % 8 == 1
    plain = [x.clone(memory_format=torch.contiguous_format).view(-1).clone().view(x.shape) for x in (q, k)]
    rope, pos = AxisRope((64,), device=gpu), torch.arange(5, device=gpu)[None] + 100
    want = rope.rotate(pos, *plain)
    for a, b in zip(rope.rotate(pos, q, k), want):
        assert torch.equal(a, b)
    table, at = torch.zeros(1, 1, dtype=torch.int32, device=gpu), torch.full((1,), 3, dtype=torch.int32, device=gpu)
    pages = []
    for qq, kk in ((q, k), plain):
        cache = R.make_cache(1, 2, gpu)
        got = cache.append_rotary(qq, kk, kk, at, table, rope, values=True)
        pages.append((*got, *cache.pools()))
    assert all(torch.equal(a, b) for a, b in zip(*pages))
    a, b = rope.rotate(pos, q, k, inplace=True)
    assert a is q and b is k and torch.equal(q, want[0]) and torch.equal(k, want[1])
