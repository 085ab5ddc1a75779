"""The appends' bounds check on the host: with ragged each row counts up to its own last position."""
import pytest
import torch

from ffa_mi355x.paged import check_append_fits

I = torch.int32


@pytest.mark.parametrize("cols", [4, 70000])
def test_rows_up_to_their_own_positions(cols):
    table = torch.full((2, cols), -1, dtype=I)
    table[0, :1] = 5
    table[1, :3] = torch.tensor([0, 1, 9], dtype=I)
    check_append_fits(torch.tensor([10, 180], dtype=I), 12, table, 10, ragged=True)
    with pytest.raises(ValueError):  # as ever without it
        check_append_fits(torch.tensor([10, 180], dtype=I), 12, table, 10)
    check_append_fits(torch.tensor([63, 191], dtype=I), 1, table, 10, ragged=True)
    for pos, n in (([63, 180], 2), ([10, 191], 2), ([64, 0], 1), ([-1, 0], 1), ([0, cols * 64], 1)):
        with pytest.raises(ValueError):
            check_append_fits(torch.tensor(pos, dtype=I), n, table, 10, ragged=True)
    with pytest.raises(ValueError):
        check_append_fits(torch.tensor([10, 180], dtype=I), 1, table, 9, ragged=True)
    table[1, 0] = -1  # a page before the new tokens
    with pytest.raises(ValueError):
        check_append_fits(torch.tensor([10, 180], dtype=I), 1, table, 10, ragged=True)
