"""Argument checks of the paged cache's operators that need no device."""
import ctypes

import pytest

import torch_rs
from trs_backend import abi

F = torch_rs.nn.functional
E, M, O = abi.TRS_E_INVALID_ARGUMENT, abi.TRS_E_SHAPE_MISMATCH, -2
PAGE = 1 << 20  # operands that no check takes for one another


def at(i):
    return ctypes.c_void_p(PAGE * (i + 1))


def cache(pages=4, heads=2, page=16, dim=8, width=3, **kw):
    lay = abi.layout_of((pages, heads, page, dim))
    fields = dict(k=at(0).value, v=at(1).value, lk=lay, lv=lay, type=abi.PAGES_F32, table=at(2).value, table_width=width, lengths=at(3).value)
    fields.update(kw)
    return abi.PagedCache(**fields)


def test_layout_struct_matches_header_size():
    assert ctypes.sizeof(abi.PagedCache) == 2 * 8 + 2 * ctypes.sizeof(abi.Layout) + 8 + 3 * 8


def append(c, k=(1, 2, 3, 8), v=None, q=None, q_out=None, table=None, axes=1, pair_axes=None, at_k=4, at_v=5, at_out=7):
    def arg(shape, i):
        return (None, None) if shape is None else (at(i), ctypes.byref(abi.layout_of(shape)))

    tab = (None, None, None) if table is None else (at(8), at(9), ctypes.byref(abi.layout_of(table)))
    return abi.lib.trs_paged_append_f32(ctypes.byref(c) if c else None, *arg(k, at_k), *arg(v or k, at_v), *arg(q, 6), *arg(q_out, at_out), *tab, 0, axes,
                                        pair_axes, None)


def attention(c, q=(1, 4, 3, 8), out=None, shared=0, window=5, sinks=0, scale=1.0, at_out=7, stride=None):
    lo = abi.layout_of(out or q, stride)
    return abi.lib.trs_paged_attention_f32(at(6), ctypes.byref(abi.layout_of(q)), ctypes.byref(c) if c else None, shared, window, sinks, scale, at(at_out),
                                           ctypes.byref(lo), None)


@pytest.mark.parametrize("call,batch", [(append, 1), (attention, 1)])
def test_caches_that_are_refused(call, batch):
    lay = abi.layout_of
    assert call(None) == E
    assert call(cache(type=2)) == E and call(cache(type=-1)) == E
    assert call(cache(table=None)) == E and call(cache(lengths=None)) == E and call(cache(k=None)) == E and call(cache(v=None)) == E
    assert call(cache(table_width=-1)) == E and call(cache(pages=0)) == E and call(cache(page=0)) == E
    assert call(cache(table_width=1 << 27)) == O and call(cache(lk=lay((4, 2, 1 << 31, 8), (0, 0, 0, 1)), lv=lay((4, 2, 1 << 31, 8), (0, 0, 0, 1)))) == O
    assert call(cache(lv=lay((4, 2, 16, 7)))) == M and call(cache(lk=lay((4, 2, 16)))) == E
    assert call(cache(lk=lay((4, 2, 16, 8), (256, 128, 8, 2)))) == E
    assert call(cache(lk=lay((1 << 32, 2, 16, 8), (0, 0, 8, 1)), lv=lay((1 << 32, 2, 16, 8), (0, 0, 8, 1)))) == O
    assert call(cache(dim=9)) == M
    for strides in ((1 << 31, 128, 8, 1), (256, 128, 1 << 31, 1)):
        assert call(cache(lk=lay((4, 2, 16, 8), strides))) == O and call(cache(lv=lay((4, 2, 16, 8), strides))) == O


def test_appending_refuses_before_it_looks_for_a_device():
    c = cache()
    assert append(c, k=(1, 3, 3, 8)) == M and append(c, v=(1, 2, 2, 8)) == M and append(c, k=(2, 3, 8)) == E
    assert append(c, q=(1, 4, 3, 8)) == E and append(c, q_out=(1, 4, 3, 8)) == E and append(c, q=(1, 4, 2, 8), q_out=(1, 4, 2, 8)) == M
    assert append(c, q=(1, 4, 3, 8), q_out=(1, 4, 3, 7)) == M
    assert append(c, table=(5, 5)) == M and append(c, table=(5,)) == E and append(c, table=(5, 4), axes=0) == E and append(c, table=(5, 4), axes=5) == E
    assert append(c, table=(5, 4), axes=2, pair_axes=bytes([0, 1, 2, 0])) == E
    assert append(c, at_k=0) == E and append(c, at_v=1) == E  # the pools are read
    assert append(c, q=(1, 4, 3, 8), q_out=(1, 4, 3, 8), at_out=1) == E and append(c, q=(1, 4, 3, 8), q_out=(1, 4, 3, 8), at_out=5) == E
    assert append(cache(v=at(0).value)) == E  # one pool twice
    assert append(cache(lk=abi.layout_of((4, 2, 16, 8), (0, 128, 8, 1)))) == E  # pages on one another
    both = abi.layout_of((4, 2, 16, 8), (512, 128, 8, 1))
    for size, kind in ((4, abi.PAGES_F32), (2, abi.PAGES_BF16)):  # one buffer for both passes this check (and asks for a device), one entry further in does not
        assert append(cache(lk=both, lv=both, v=at(0).value + 256 * size, type=kind), table=(5, 5)) == M
        assert append(cache(lk=both, lv=both, v=at(0).value + 255 * size, type=kind)) == E


def test_attention_refuses_before_it_looks_for_a_device():
    c = cache()
    assert attention(c, window=0) == E and attention(c, sinks=-1) == E and attention(c, shared=-1) == E
    assert attention(c, scale=float("inf")) == E and attention(c, scale=float("nan")) == E
    assert attention(c, q=(1, 3, 3, 8)) == M and attention(c, q=(4, 3, 8)) == E and attention(c, out=(1, 4, 3, 9)) == M
    assert attention(c, at_out=6) == E and attention(c, at_out=0) == E and attention(c, at_out=3) == E
    assert attention(c, stride=(192, 48, 16, 2)) == E and attention(c, stride=(96, 0, 8, 1)) == E
    wide = cache(dim=257)
    assert attention(wide, q=(1, 4, 3, 257)) == E


def test_rotations_refuse_before_they_look_for_a_device():
    one = abi.layout_of((1, 2, 3, 8))
    two = (abi.Layout * 2)(one, abi.layout_of((1, 2, 4, 8)))
    same = (abi.Layout * 2)(one, one)

    def call(n=1, lx=same, lo=same, axes=1, pair_axes=None, table=(5, 4), start=0, x=(0, 1), y=(2, 3)):
        ptrs = [(ctypes.c_void_p * 2)(*(at(i).value for i in ids)) for ids in (x, y)]
        return abi.lib.trs_rope_axes_f32(n, ptrs[0], lx, at(8), at(9), ctypes.byref(abi.layout_of(table)), 0, axes, pair_axes, None, start, 0, ptrs[1], lo)

    assert call(n=0) == E and call(n=3) == E and call(n=2, lx=two, lo=two) == M and call(lo=(abi.Layout * 2)(abi.layout_of((1, 2, 3, 7)), one)) == M
    assert call(axes=5) == E and call(axes=0) == E and call(axes=3, pair_axes=bytes([0, 3, 0, 0])) == E
    assert call(table=(5, 5)) == M and call(table=(5,)) == E and call(start=3) == E and call(start=-1) == E
    assert call(n=2, y=(2, 2)) == E and call(n=2, y=(1, 3)) == E and call(y=(8, 3)) == E


def test_python_arguments():
    x = torch_rs.zeros((1, 1, 2, 4))
    with pytest.raises(TypeError, match="'cos' must be Tensor"):
        F.rope_axes(x, x, None, None)
    with pytest.raises(TypeError, match="'key' must be Tensor"):
        F.rope_axes(x, 1, x, x)
    with pytest.raises(ValueError, match="pair_axes"):
        F.rope_axes(x, x, x, x, pair_axes=[-1, 0])
    with pytest.raises(ValueError, match="1 to 4 axes"):
        F.rope_axes(x, x, x, x, pair_axes=[0, 4])
    with pytest.raises(TypeError, match="start"):
        F.rope_axes(x, x, x, x, start=0.5)
    with pytest.raises(RuntimeError):
        F.rope_axes(x, None, torch_rs.zeros((2, 2)), torch_rs.zeros((2, 2)))  # host tensors
    with pytest.raises(TypeError, match="dtype"):
        F.paged_cache(4, 2, 16, 8, "float16")
    with pytest.raises(TypeError, match="pages"):
        F.paged_cache(4.5, 2, 16, 8)
    with pytest.raises(RuntimeError, match="device"):
        F.paged_cache(4, 2, 16, 8, device="cpu")
    with pytest.raises(TypeError, match="PagedCache"):
        F.paged_append(None, [[0]], [1], x, x)
    with pytest.raises(ValueError, match="both tables"):
        F.paged_append(None, [[0]], [1], x, x, x)
    with pytest.raises(TypeError, match="PagedCache"):
        F.paged_attention(x, x, [[0]], [1])
    with pytest.raises(TypeError, match="'query' must be Tensor"):
        F.paged_attention(None, x, [[0]], [1])
