"""Axes of a rotation's pairs through torch_rs: an empty list is no axes for 0 pairs, not the default for all of them."""
import numpy as np
import pytest

import torch_rs
from attention_util import rotation_tables

pytestmark = pytest.mark.gpu
F = torch_rs.nn.functional


def device(*shape):
    return torch_rs.tensor(np.ones(shape, np.float32), device="cuda")


def test_axes_for_no_pairs():
    x, cache = device(1, 1, 2, 4), F.paged_cache(1, 1, 4, 4)
    cos, sin = (torch_rs.tensor(t, device="cuda") for t in rotation_tables(3, 4))
    for axes in ([], ()):
        with pytest.raises(RuntimeError, match="rope_axes has axes for 0 pairs, and tables of 2"):
            F.rope_axes(x, None, cos, sin, pair_axes=axes)
        with pytest.raises(RuntimeError, match="paged_append has axes for 0 pairs, and tables of 2"):
            F.paged_append(cache, [[0]], [2], x, x, cos, sin, pair_axes=axes, positions=np.zeros((2, 1, 2), int))
    # Tables of no pairs turn nothing, and have that many axes.
    none = torch_rs.tensor(np.ones((3, 0), np.float32), device="cuda")
    assert np.array_equal(F.rope_axes(x, None, none, none, pair_axes=[]).numpy(), x.numpy())
