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
