"""Windows, sinks and budgets that are no whole numbers: refused as arguments,
whatever they are."""

import numpy as np
import pytest
import torch

from naivllm_amd.layers.attention import Attention, _int_arg


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan"), None, "4", "many", 2.5, -1, [4], np.inf])
def test_refused(value):
    with pytest.raises(ValueError, match="window must be an integer of at least 0"):
        Attention(4, 64, window=value)


@pytest.mark.parametrize("value", [4, 4.0, np.int64(4), np.float32(4), torch.tensor(4), True + 3])
def test_taken(value):
    assert _int_arg(value, "window", 1) == 4


def test_beyond_every_table_is_no_bound():
    assert _int_arg(1 << 40, "window", 1) == _int_arg(2.0 ** 50, "window", 1) == 1 << 30
