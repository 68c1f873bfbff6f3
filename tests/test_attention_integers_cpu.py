"""Whole-number arguments of the attention block's operators: nothing is cut to one."""
import numpy as np
import pytest

import torch_rs

F = torch_rs.nn.functional


@pytest.mark.parametrize("bad", [2.5, np.float32(1.5), float("nan"), float("inf"), "2", [2]], ids=repr)
def test_what_is_no_whole_number_is_refused(bad):
    x, table = torch_rs.zeros((1, 1, 2, 4)), torch_rs.zeros((2, 2))
    with pytest.raises(TypeError, match="'window' must be int"):
        F.window_attention(x, x, x, window=bad)
    with pytest.raises(TypeError, match="'sinks' must be int"):
        F.window_attention(x, x, x, sinks=bad)
    with pytest.raises(TypeError, match="'start' must be int"):
        F.head_norm_rope(x, x, None, None, table, table, start=bad)


@pytest.mark.parametrize("good", [2, 2.0, np.int64(2), np.uint8(2), np.float32(2)], ids=repr)
def test_whole_numbers_of_any_type_reach_the_device_check(good):
    x, table = torch_rs.zeros((1, 1, 2, 4)), torch_rs.zeros((2, 2))
    for call in (lambda: F.window_attention(x, x, x, window=good, sinks=good), lambda: F.head_norm_rope(x, x, None, None, table, table, start=good)):
        with pytest.raises(RuntimeError):  # host tensors
            call()
