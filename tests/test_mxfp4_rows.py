"""Rows as the rotary and mxfp4 kernels take them: what the host decides, on the CPU."""
import pytest
import torch

from ffa_mi355x.rope_axes import strided_rows


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
