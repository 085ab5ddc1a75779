"""Rows as the rotary and mxfp4 kernels take them: what the host decides, on the CPU."""
import random

import pytest
import torch

from ffa_mi355x.rope_axes import _side_by_side, rows_overlap, strided_rows


def _odd_batch(T=5, H=2, dtype=torch.float16):
    """One sequence out of a batch whose sequences lie an odd number of elements apart: contiguous, with that stride."""
    x = torch.randn(2, T * H * 128 + 1).to(dtype)
    return x[:, :-1].view(2, T, H, 128)[:1]


def test_strides_of_single_entries_do_not_count():
    x = _odd_batch()
    assert x.is_contiguous() and x.stride(0) % 8 == 1
    a, s = strided_rows(x)
    assert a is x and s == (0, 256, 128)
    a, s = strided_rows(torch.empty_like(x))  # keeps the strides
    assert s == (0, 256, 128)
    y = torch.as_strided(torch.zeros(2000), (3, 1, 1, 128), (128, 7, 9, 1))
    a, s = strided_rows(y)
    assert a is y and s == (128, 0, 0)


@pytest.mark.parametrize("T", [1, 5])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_rows_that_start_elsewhere_are_copied(T, dtype):
    x = torch.randn(T * 2 * 128 + 4).to(dtype)[1:T * 256 + 1].view(1, T, 2, 128)
    a, s = strided_rows(x)
    assert a.data_ptr() % 16 == 0 and torch.equal(a, x) and all(n % (16 // x.element_size()) == 0 for n in s)
    step = torch.randn(1, T, 2, 130).to(dtype)[..., :128]
    a, s = strided_rows(step)
    assert torch.equal(a, step) and all(n % (16 // x.element_size()) == 0 for n in s) and a.stride(3) == 1


def _bytes(x):
    at = torch.arange(x.shape[3]) * x.element_size()
    for n, s in zip(x.shape[2::-1], x.stride()[2::-1]):
        at = (torch.arange(n)[:, None] * s * x.element_size() + at.reshape(1, -1)).reshape(-1)
    return (x.data_ptr() + at[:, None] + torch.arange(x.element_size())).reshape(-1)


def test_overlap_of_rows_as_models_lay_them_out():
    joined = torch.zeros(2, 5, 10 * 128)
    q, k, v = joined[..., :768].view(2, 5, 6, 128), joined[..., 768:1024].view(2, 5, 2, 128), joined[..., 1024:].view(2, 5, 2, 128)
    for a, b in ((q, k), (k, q), (k, v), (q, v)):
        assert not rows_overlap(a, b)
    heads = torch.zeros(2, 10, 5, 128).transpose(1, 2)  # [B, T, H, 128], heads before tokens in memory
    assert not rows_overlap(heads[:, :, :6], heads[:, :, 6:8]) and rows_overlap(heads[:, :, :6], heads[:, :, 5:8])
    tokens = torch.zeros(5, 2, 10, 128).transpose(0, 1)
    assert not rows_overlap(tokens[:, :, :6], tokens[:, :, 6:]) and rows_overlap(tokens[:, :, 2:6], tokens[:, :, :3])
    assert not rows_overlap(joined[:1, :, :128].unsqueeze(2), joined[1:, :, :128].unsqueeze(2))
    full = joined.view(2, 5, 10, 128)
    assert not rows_overlap(full[:, :, ::2], full[:, :, 1::2])  # every other head
    assert rows_overlap(full[:, :, :8], full[:, :, 6:])
    assert rows_overlap(joined[..., :768].view(2, 5, 6, 128), joined[..., 704:960].view(2, 5, 2, 128))  # by half of a row
    assert rows_overlap(full[:, :1].expand(2, 5, 10, 128)) and not rows_overlap(full[:, :0], full)
    assert rows_overlap(torch.as_strided(joined, (1, 9, 1, 128), (0, 64, 0, 1)))  # windows
    assert not rows_overlap(torch.as_strided(joined, (2, 3, 2, 128), (256, 512, 128, 1)))
    assert _side_by_side(q, k) and _side_by_side(k, q) and not _side_by_side(q, q) and _side_by_side(q.clone(), k.clone())
    assert not rows_overlap(q) and not rows_overlap(full[:, :, :0]) and rows_overlap(q, q)


def test_overlap_of_rows_at_random():
    r = random.Random(3)
    base, seen = torch.zeros(20000, dtype=torch.float16), [0, 0]
    for _ in range(1500):
        xs = []
        same = r.random() < 0.5
        strides = [r.choice([64, 128, 136, 256, 384, 512, 640, 1024]) for _ in range(3)]
        for _ in range(r.choice([1, 2, 2])):
            shape = [2, r.randint(1, 2), r.randint(1, 3)] if same else [r.randint(1, 3) for _ in range(3)]
            st = strides if same else [r.choice([0, 64, 128, 256, 384, 512, 1024]) for _ in range(3)]
            xs.append(torch.as_strided(base, (*shape, 128), (*st, 1), 8 * r.randint(0, 800)))
        used = torch.cat([_bytes(x) for x in xs])
        want = used.unique().numel() < used.numel()
        assert rows_overlap(*xs) == want, [(x.shape, x.stride(), x.storage_offset()) for x in xs]
        if len(xs) == 2 and xs[0].shape[:2] == xs[1].shape[:2]:
            assert not (_side_by_side(*xs) and want), [(x.shape, x.stride(), x.storage_offset()) for x in xs]
        seen[want] += 1
    assert min(seen) > 200
