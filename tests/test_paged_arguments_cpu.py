"""Arguments of the paged cache's operators that say nothing, or not what was meant, are refused rather than dropped."""
import pytest

import torch_rs

F = torch_rs.nn.functional


def zeros(*shape):
    return torch_rs.zeros(shape)


@pytest.mark.parametrize("name,value", [("positions", [[0, 1]]), ("pair_axes", [0, 0]), ("pair_axes", []), ("interleaved", True)])
def test_appending_without_tables_takes_nothing_of_a_rotation(name, value):
    x = zeros(1, 1, 2, 4)
    with pytest.raises(ValueError, match=f"{name} without tables"):
        F.paged_append(None, [[0]], [2], x, x, **{name: value})
    with pytest.raises(ValueError, match=f"{name} without tables"):
        F.paged_append(None, [[0]], [2], x, x, None, None, query=x, **{name: value})


def test_no_axes_for_pairs_that_there_are():
    """An empty list is no axes for 0 pairs, not the default for all of them."""
    x, tables = zeros(1, 1, 2, 4), zeros(3, 2)
    with pytest.raises(RuntimeError, match="device"):  # host tensors, and nothing before that
        F.rope_axes(x, None, zeros(3, 0), zeros(3, 0), pair_axes=[])
    for axes in ([], ()):
        with pytest.raises(RuntimeError, match="rope_axes has axes for 0 pairs, and tables of 2"):
            F.rope_axes(x, None, tables, tables, pair_axes=axes)
