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


def test_in_place_where_rows_overlap(gpu):
    """Refused, and nothing is turned; rows side by side in one projection are turned."""
    rope, pos = AxisRope((64,), device=gpu), torch.arange(5, device=gpu)[None]
    joined = torch.randn(2, 5, 10, 128, device=gpu)
    before = joined.clone()
    wide = torch.as_strided(joined, (1, 9, 1, 128), (0, 64, 0, 1))
    for q, k in ((joined[:, :, :8], joined[:, :, 6:]), (joined[:, :, 6:], joined[:, :, :8]), (joined[:, :, :4], joined[:, :, :4]),
                 (joined[:, :, :1].expand(2, 5, 4, 128), None), (joined[:, :1].expand(2, 5, 10, 128), None)):
        with pytest.raises(ValueError):
            rope.rotate(pos, q, k, inplace=True)
    with pytest.raises(ValueError):
        rope.rotate(torch.arange(9, device=gpu)[None], wide, inplace=True)
    assert torch.equal(joined, before)
    want = rope.rotate(pos, joined[:, :, :6].clone(), joined[:, :, 6:8].clone())
    rope.rotate(pos, joined[:, :, :6], joined[:, :, 6:8], inplace=True)
    assert torch.equal(joined[:, :, :6], want[0]) and torch.equal(joined[:, :, 6:8], want[1])
    assert torch.equal(joined[:, :, 8:], before[:, :, 8:])
    rope.rotate(pos, joined[:, :, 1::2], joined[:, :, ::2], inplace=True)  # every other head
    assert torch.equal(joined[:, :, 9], rope.rotate(pos, before[:, :, 9:])[:, :, 0])
