"""Layer norm with several times more rows than its kernels have slots: every slot of the rings is filled again, with rows
that start at other places within 16 bytes, and the blocks that share a row exchange their sums row after row."""
import pytest
import torch

from test_layer_norm_gpu import PAIRS, check, inputs

pytestmark = pytest.mark.gpu


# Rows above groups x slots of any type on 148 SMs: warps 3552 x 8, two warps 1776 x 8, four 888 x 8, eight 444 x 8,
# sixteen 148 x 8 (forward; backward has fewer).
@pytest.mark.parametrize("dtype, par", PAIRS)
@pytest.mark.parametrize("rows, d", [(60000, 301), (20000, 1003), (9000, 2001), (6000, 4001), (3000, 8001)])
def test_odd_rows_in_slots_that_are_filled_again(rows, d, dtype, par):
    check(*inputs(rows, d, dtype, par, seed=d))


# Rows above teams x slots: 74 x 8, 74 x 8, 29 x 8, 18 x 8.
@pytest.mark.parametrize("dtype, par", PAIRS)
@pytest.mark.parametrize("rows, d", [(1500, 16384), (1500, 8193), (600, 40001), (300, 65001)])
def test_rows_shared_by_blocks_one_after_the_other(rows, d, dtype, par):
    check(*inputs(rows, d, dtype, par, seed=d))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows, d", [(60000, 299), (20000, 1002), (6000, 4001), (1500, 8195)])
def test_rows_and_gradients_at_places_of_their_own(rows, d, dtype):
    """x and the upstream gradient start at different places within 16 bytes, other ones in every row."""
    x, w, b, dy = inputs(rows, d, dtype, torch.float32, seed=d)
    wide, up = torch.empty(rows, d + 7, device="cuda", dtype=dtype), torch.empty(rows, d + 4, device="cuda", dtype=dtype)
    x, dy = wide[:, 1:d + 1].copy_(x), up[:, 2:d + 2].copy_(dy)
    check(x, w, b, dy)
