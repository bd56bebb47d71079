"""Calls of the 8-bit operators that are refused, and that nothing else depends on: without a GPU."""
import pytest
import torch

from block_transformer_amd import ops
from block_transformer_amd._lib import BtError


def weight(columns, rows=8):
    w = torch.zeros(rows, (columns + 15) // 16 * 16, dtype=torch.int8), torch.zeros(rows)
    w[0].columns = columns                # as quantize_rows leaves it
    return w


def test_linear_q8_of_another_number_of_columns():
    """515 and 520 columns both take 528 codes: their product would mean nothing."""
    with pytest.raises(BtError, match="x has 515 columns, the weight 520"):
        ops.linear_q8(torch.zeros(3, 515), weight(520))
    with pytest.raises(BtError, match="x has 515 columns, the weight 520"):
        ops.linear_q8(weight(515, 3), weight(520), dtype=torch.float32)
    with pytest.raises(BtError, match="GPU memory"):      # (refused for the device alone)
        ops.linear_q8(torch.zeros(3, 520), weight(520))
    with pytest.raises(BtError, match="GPU memory"):
        ops.linear_q8(weight(520, 3), weight(520), dtype=torch.float32)
    with pytest.raises(BtError, match="GPU memory"):      # codes that do not say
        ops.linear_q8(torch.zeros(3, 515), (torch.zeros(8, 528, dtype=torch.int8), torch.zeros(8)))
