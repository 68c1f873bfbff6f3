"""Argument checks of the attention block's operators that need no device."""
import ctypes

import numpy as np
import pytest

import torch_rs
from trs_backend import abi

F = torch_rs.nn.functional


def test_dropout_takes_a_mask_or_a_seed_and_checks_both_words():
    x = torch_rs.zeros((2, 3))
    with pytest.raises(ValueError, match="a mask or a seed"):
        F.dropout(x, 0.5, mask=np.ones((2, 3), np.uint8), seed=1)
    for kw in ({"seed": 1.5}, {"seed": True}, {"seed": "1"}, {"seed": 1, "offset": None}):
        with pytest.raises(TypeError, match="must be int"):
            F.dropout(x, 0.5, **kw)
    for kw in ({"seed": -1}, {"seed": 1 << 64}, {"seed": 1, "offset": -1}):
        with pytest.raises(ValueError, match="2\\*\\*64"):
            F.dropout(x, 0.5, **kw)
    with pytest.raises(NotImplementedError, match="inplace"):
        F.dropout(x, 0.5, inplace=True, seed=1)
    with pytest.raises(NotImplementedError, match="does not support sampling"):
        F.dropout(x, 0.5)  # as before: no seed, no mask
    assert F.dropout(x, 0.5, False, seed=1) is x
    with pytest.raises(RuntimeError):
        F.dropout(x, 0.5, seed=1)  # a host tensor


def test_attention_arguments():
    x = torch_rs.zeros((1, 1, 2, 4))
    with pytest.raises(TypeError, match="'key' must be Tensor"):
        F.window_attention(x, None, x)
    with pytest.raises(ValueError, match="window"):
        F.window_attention(x, x, x, window=0)
    with pytest.raises(ValueError, match="sinks"):
        F.window_attention(x, x, x, sinks=-1)
    with pytest.raises(RuntimeError):
        F.window_attention(x, x, x)  # host tensors
    with pytest.raises(TypeError, match="'cos' must be Tensor"):
        F.head_norm_rope(x, None, None, None, None, None)
    with pytest.raises(RuntimeError):
        F.head_norm_rope(x, x, None, None, torch_rs.zeros((2, 2)), torch_rs.zeros((2, 2)))
    with pytest.raises(TypeError, match="integers"):
        F.index_buffer([1.5])
    with pytest.raises(ValueError, match="32 bits"):
        F.index_buffer([1 << 31])


def test_the_abi_refuses_before_it_looks_for_a_device():
    lay = abi.layout_of((2, 3))
    one = ctypes.c_void_p(4096)
    E = abi.TRS_E_INVALID_ARGUMENT
    assert abi.lib.trs_dropout_f32(one, ctypes.byref(lay), 1.5, 0, 0, one, ctypes.byref(lay)) == E
    assert abi.lib.trs_dropout_f32(None, ctypes.byref(lay), 0.5, 0, 0, one, ctypes.byref(lay)) == E
    assert abi.lib.trs_dropout_f32(one, None, 0.5, 0, 0, one, ctypes.byref(lay)) == E
    q = abi.layout_of((1, 1, 2, 4))
    args = [one, ctypes.byref(q)] * 3
    assert abi.lib.trs_window_attention_f32(*args, None, 0, 0, 1.0, ctypes.c_void_p(65536), ctypes.byref(q), None) == E
    assert abi.lib.trs_window_attention_f32(*args, None, 4, 0, 1.0, one, ctypes.byref(q), None) == E  # the output is the query
    assert abi.lib.trs_head_norm_rope_f32(3, None, None, None, 1e-6, None, None, ctypes.byref(lay), 0, None, 0, None, None) == E
