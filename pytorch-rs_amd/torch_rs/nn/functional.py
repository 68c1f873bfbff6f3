"""Functional interface."""
# torch_rs.nn.functional: relu and the dropout family, as the reference's
# python/torch_rs/nn/functional.py:1-265 and src/python_nn_functional.rs:13-200.
# The module docstring, relu's docstring and signature are the reference's.

import math
import sys as _sys
import warnings

import numpy as _np

from .._native import native as _C


def relu(input: _C.Tensor, inplace: bool = False) -> _C.Tensor:
    if inplace:
        raise NotImplementedError("torch_rs.nn.functional.relu does not support inplace=True")
    return input.relu()


relu.__doc__ = ("relu(input, inplace=False) -> Tensor\n\n"
                "Applies the rectified linear unit function element-wise. See\n"
                ":class:`~torch.nn.ReLU` for more details.\n") if _sys.version_info >= (3, 13) else (
    """relu(input, inplace=False) -> Tensor

    Applies the rectified linear unit function element-wise. See
    :class:`~torch.nn.ReLU` for more details.
    """)


def _autograd_suffix(t) -> str:
    name = t._grad_fn_name
    if name is not None:
        return f", grad_fn=<{name}>"
    return ", requires_grad=True" if t.requires_grad else ""


def _format_single_element(t, value: float) -> str:
    """A one-element tensor as PyTorch prints it in this diagnostic
    (python/torch_rs/_diagnostics.py:9-43): integral values as `2.`, others
    with 4 decimals, scientific outside [1e-4, 1e8]; one bracket per dim."""
    finite = math.isfinite(value)
    if finite and value != 0.0:
        integral = value == math.ceil(value)
        scientific = abs(value) > 1.0e8 or abs(value) < 1.0e-4
    else:
        integral, scientific = True, False
    if scientific:
        text = f"{value:.4e}"
    elif integral:
        text = f"{value:.0f}" + ("." if finite else "")
    else:
        text = f"{value:.4f}"
    for _ in range(len(t.shape)):
        text = f"[{text}]"
    return f"tensor({text}{_autograd_suffix(t)})"


def _validate_probability(p):
    """_validate_dropout_probability (python/torch_rs/nn/functional.py:14-24, 86-105)."""
    shown = p
    if isinstance(p, _C.Tensor):
        n = p.numel()
        if n == 0:
            raise RuntimeError("Boolean value of Tensor with no values is ambiguous")
        if n != 1:
            raise RuntimeError("Boolean value of Tensor with more than one value is ambiguous")
        value = p.item()
        shown = value if len(p.shape) == 0 else _format_single_element(p, value)
        p = value
    if p < 0.0 or p > 1.0:
        raise ValueError(f"dropout probability has to be between 0 and 1, but got {shown}")


def _type_name(x) -> str:
    t = type(x)
    return t.__name__ if t.__module__ == "builtins" else f"{t.__module__}.{t.__name__}"


# The reference's dropout family (src/python_nn_functional.rs:13-62): public
# name -> (operation, in-place operation, scalar-tensor p allowed, p == 1
# allowed, input ranks allowed or None).
_DROPOUT_KINDS = {
    "dropout": ("dropout", "dropout_", True, True, None),
    "alpha_dropout": ("alpha_dropout", "alpha_dropout_", False, False, None),
    "feature_alpha_dropout": ("feature_alpha_dropout", "feature_alpha_dropout_", True, True, None),
    "dropout1d": ("feature_dropout", "feature_dropout_", True, False, (2, 3)),
    "dropout2d": ("feature_dropout", "feature_dropout_", True, False, (3, 4)),
    "dropout3d": ("feature_dropout", "feature_dropout_", True, True, (5,)),
}


def _float_like(p, op):
    """parse_float_like_argument (src/python_argument_schema.rs:51-89)."""
    if isinstance(p, _C.Tensor):
        if len(p.shape) == 0 and not p.requires_grad:
            return float(p.item())
        raise TypeError(f"{op}(): argument 'p' (position 2) must be float, not Tensor")
    if isinstance(p, (int, float)):
        return float(p)
    if isinstance(p, _np.bool_):
        return 1.0 if p else 0.0
    if isinstance(p, (_np.integer, _np.floating)):
        return float(p)
    raise TypeError(f"{op}(): argument 'p' (position 2) must be float, not {_type_name(p)}")


def _dropout_bridge(kind, input, p, training, inplace, mask=None, counter=None):
    """_nn_functional_dropout (src/python_nn_functional.rs:117-200): schema
    checks, then identity when not training, p == 0 or the input is empty;
    ``input * 0.0`` for p == 1 where the kind allows it; sampling is
    unsupported."""
    op_name, inplace_name, tensor_p, p_one, ranks = _DROPOUT_KINDS[kind]
    op = inplace_name if inplace else op_name
    if not isinstance(input, _C.Tensor):
        raise TypeError(f"{op}(): argument 'input' (position 1) must be Tensor, not {_type_name(input)}")
    if not tensor_p and isinstance(p, _C.Tensor):
        raise TypeError(f"{op}(): argument 'p' (position 2) must be float, not Tensor")
    prob = _float_like(p, op)
    if type(training) is not bool:
        raise TypeError(f"{op}(): argument 'train' (position 3) must be bool, not {_type_name(training)}")
    if not 0.0 <= prob <= 1.0:
        if math.isnan(prob):
            shown = "-nan" if math.copysign(1.0, prob) < 0 else "nan"
        else:
            shown = format(prob, ".6g")
        raise RuntimeError(f"dropout probability has to be between 0 and 1, but got {shown}")
    rank = len(input.shape)
    if ranks is not None and rank not in ranks:
        allowed = " or ".join(f"rank-{r}" for r in ranks)
        raise NotImplementedError(f"torch_rs.nn.functional.{kind} only supports {allowed} inputs")
    unbatched_1d = kind == "dropout1d" and rank == 2
    if unbatched_1d and inplace:
        raise NotImplementedError(
            "torch_rs.nn.functional.dropout1d does not support inplace=True for rank-2 inputs")
    if not training or prob == 0.0 or input.numel() == 0:
        # PyTorch runs an unbatched input through unsqueeze(0) and squeeze(0),
        # so even the identity returns a new view with a SqueezeBackward1 edge.
        return input._unsqueeze_front().squeeze(0) if unbatched_1d else input
    if counter is not None:
        if inplace:
            raise NotImplementedError(f"torch_rs.nn.functional.{kind} does not support inplace=True")
        return _C.dropout_counter(input, prob, *counter)
    if mask is not None:
        if inplace:
            raise NotImplementedError(f"torch_rs.nn.functional.{kind} does not support inplace=True")
        if not isinstance(mask, _C.ByteBuffer):
            mask = keep_mask(mask, input.device)
        return _C.mask_apply(input, mask, _np.float32(1.0 / (1.0 - prob)) if prob < 1.0 else _np.float32(0.0))
    if p_one and not inplace and prob == 1.0:
        return input * 0.0
    raise NotImplementedError(f"torch_rs.nn.functional.{kind} does not support sampling")


def _word64(name, value) -> int:
    """An int taken modulo nothing: it has to fit an unsigned 64-bit word."""
    if isinstance(value, bool) or not isinstance(value, (int, _np.integer)):
        raise TypeError(f"dropout(): argument '{name}' must be int, not {_type_name(value)}")
    if not 0 <= int(value) < 1 << 64:
        raise ValueError(f"dropout {name} has to be between 0 and 2**64 - 1, but got {int(value)}")
    return int(value)


def dropout(input, p: float = 0.5, training: bool = True, inplace: bool = False, *, mask=None, seed=None, offset: int = 0):
    """The reference's dropout (python/torch_rs/nn/functional.py:14-31, 121-143):
    the Python range check, then the native bridge.

    ``mask`` (this backend's addition) is a precomputed keep-mask -- a uint8
    array (or a device byte buffer from ``keep_mask``) of the input's shape
    with 1 = keep -- applied as ``(input * mask) * f32(1/(1-p))``, the
    reference composition ``mul`` then ``mul_scalar``, with the mask read as
    one byte per element.

    ``seed`` (this backend's addition) samples on the device instead, from a
    counter-based generator (``trs_dropout_f32``): element i in row-major order is
    kept by word i % 4 of counter ``offset + i // 4``, and nothing is stored for
    backward.  A call uses ``ceil(numel / 4)`` counters: advance ``offset`` by that
    much, or change the seed, for another mask."""
    _validate_probability(p)
    counter = None
    if seed is not None:
        if mask is not None:
            raise ValueError("dropout takes a mask or a seed, not both")
        counter = _word64("seed", seed), _word64("offset", offset)
    return _dropout_bridge("dropout", input, p, training, inplace, mask, counter)


def dropout1d(input, p: float = 0.5, training: bool = True, inplace: bool = False):
    """python/torch_rs/nn/functional.py:34-40, 146-171."""
    _validate_probability(p)
    input.dim()  # the reference validates the input before the bridge
    return _dropout_bridge("dropout1d", input, p, training, inplace)


def dropout2d(input, p: float = 0.5, training: bool = True, inplace: bool = False):
    """python/torch_rs/nn/functional.py:43-60, 174-199."""
    _validate_probability(p)
    if input.dim() == 3:
        warnings.warn(
            "dropout2d: Received a 3D input to dropout2d and assuming that channel-wise 1D dropout behavior is "
            "desired - input is interpreted as shape (N, C, L), where C is the channel dim. This behavior will "
            "change in a future release to interpret the input as one without a batch dimension, i.e. shape "
            "(C, H, W). To maintain the 1D channel-wise dropout behavior, please switch to using dropout1d "
            "instead.", stacklevel=2)
    return _dropout_bridge("dropout2d", input, p, training, inplace)


def dropout3d(input, p: float = 0.5, training: bool = True, inplace: bool = False):
    """python/torch_rs/nn/functional.py:63-69, 202-227."""
    _validate_probability(p)
    input.dim()
    return _dropout_bridge("dropout3d", input, p, training, inplace)


def alpha_dropout(input, p: float = 0.5, training: bool = False, inplace: bool = False):
    """python/torch_rs/nn/functional.py:72-76, 230-245."""
    _validate_probability(p)
    return _dropout_bridge("alpha_dropout", input, p, training, inplace)


def feature_alpha_dropout(input, p: float = 0.5, training: bool = False, inplace: bool = False):
    """python/torch_rs/nn/functional.py:79-87, 248-265."""
    _validate_probability(p)
    return _dropout_bridge("feature_alpha_dropout", input, p, training, inplace)


def keep_mask(mask, device="cuda"):
    """Upload a uint8 keep-mask (1 = keep) to the device once, for reuse across steps."""
    from .. import _device_str
    arr = _np.asarray(mask, dtype=_np.uint8, order="C")
    return _C.bytes_from_numpy(arr, _device_str(device, "keep_mask"))


def index_buffer(values, device="cuda"):
    """Upload integers (positions, key lengths) to the device once, as int32, for reuse across calls."""
    from .. import _device_str
    arr = _np.asarray(values)
    if arr.size and arr.dtype.kind not in "iu":
        raise TypeError(f"index_buffer(): values must be integers, not {arr.dtype}")
    if arr.size and (arr.min() < -(1 << 31) or arr.max() >= 1 << 31):
        raise ValueError("index_buffer(): values must fit 32 bits")
    return _C.indices_from_numpy(_np.ascontiguousarray(arr, dtype=_np.int32).reshape(arr.shape), _device_str(device, "index_buffer"))


def _indices(values, like):
    if values is None or isinstance(values, _C.IndexBuffer):
        return values
    return index_buffer(values, like.device)


def _integer(op, name, value) -> int:
    """A whole number of any type; nothing is cut to one."""
    if not isinstance(value, (int, float, _np.integer, _np.floating)) or value != value // 1 or math.isinf(value):
        raise TypeError(f"{op}(): argument '{name}' must be int, not {value!r}")
    return int(value)


def _tensor_arguments(op, **tensors):
    for name, t in tensors.items():
        if not isinstance(t, _C.Tensor):
            raise TypeError(f"{op}(): argument '{name}' must be Tensor, not {_type_name(t)}")


def head_norm_rope(query, key, query_weight, key_weight, cos, sin, *, eps: float = 1e-6, start: int = 0, positions=None,
                   interleaved: bool = False):
    """The norm of every head's vector with the rotation by its position, of
    queries and keys [batch, head, token, dim] in one launch; returns both.

    Per row: ``y = R(position) (x * weight / sqrt(mean(x**2) + eps))``.  ``cos`` and
    ``sin`` are tables [positions, pairs]: row t turns the pairs (i, i + pairs) or,
    ``interleaved``, (2i, 2i + 1) of the first 2 * pairs entries.  Token t stands at
    ``start + t``, or where ``positions`` ([batch, token] integers, or an
    ``index_buffer``) says.  A weight may be None (ones); ``key`` may be None, and the
    query alone is returned then.  Gradients reach queries, keys and weights."""
    _tensor_arguments("head_norm_rope", query=query, cos=cos, sin=sin)
    xs, ws = [query], [query_weight]
    if key is not None:
        _tensor_arguments("head_norm_rope", key=key)
        xs.append(key)
        ws.append(key_weight)
    for name, w in zip(("query_weight", "key_weight"), ws):
        if w is not None:
            _tensor_arguments("head_norm_rope", **{name: w})
            if len(w.shape) != 1:
                raise RuntimeError(f"head_norm_rope weight has {len(w.shape)} dims, expected 1")
    start = _integer("head_norm_rope", "start", start)
    out = _C.head_norm_rope(xs, ws, cos, sin, float(eps), bool(interleaved), start, _indices(positions, query))
    return out[0] if key is None else tuple(out)


def window_attention(query, key, value, *, window=None, sinks: int = 0, scale=None, key_lengths=None):
    """Causal attention with a sliding window and first tokens that stay visible.

    ``query`` [batch, heads, tokens, dim], ``key`` and ``value`` [batch, key heads,
    keys, dim]; each key head serves heads / key heads consecutive query heads.
    The last query stands at the last key's place, and a query at place p sees key
    j where ``j <= p and (p - j < window or j < sinks)`` (``window`` None: all up to
    p).  ``scale`` is 1/sqrt(dim) by default.  ``key_lengths`` ([batch] integers, or
    an ``index_buffer``) are the keys that each sequence of a cache has.  A query
    that sees nothing gives 0.  Gradients reach queries, keys and values."""
    _tensor_arguments("window_attention", query=query, key=key, value=value)
    window = None if window is None else _integer("window_attention", "window", window)
    sinks = _integer("window_attention", "sinks", sinks)
    if window is not None and window < 1:
        raise ValueError(f"window_attention window has to be at least 1, but got {window}")
    if sinks < 0:
        raise ValueError(f"window_attention sinks have to be at least 0, but got {sinks}")
    if scale is None:
        scale = 1.0 / math.sqrt(query.shape[-1]) if len(query.shape) and query.shape[-1] else 1.0
    every = (1 << 63) - 1
    return _C.window_attention(query, key, value, every if window is None else min(window, every), min(sinks, every),
                               float(scale), _indices(key_lengths, query))


def _pair_axes(op, positions, pair_axes, tables):
    """The number of axes, and the axis of every pair as bytes (none: axis 0)."""
    axes = None
    if positions is not None:
        axes = positions.shape[0] if len(positions.shape) == 3 else 1
    if pair_axes is None:
        return axes or 1, []
    pair_axes = [_integer(op, "pair_axes", a) for a in pair_axes]
    if not pair_axes and len(tables.shape) == 2 and tables.shape[1]:  # (other numbers are the engine's to compare)
        raise RuntimeError(f"{op} has axes for 0 pairs, and tables of {tables.shape[1]}")
    axes = axes or max(pair_axes, default=0) + 1
    if not 1 <= axes <= 4:
        raise ValueError(f"{op} positions have 1 to 4 axes, but got {axes}")
    for a in pair_axes:
        if not 0 <= a < axes:
            raise ValueError(f"{op} pair_axes have to be between 0 and {axes - 1}, but got {a}")
    return axes, pair_axes


def rope_axes(query, key, cos, sin, *, positions=None, pair_axes=None, start: int = 0, interleaved: bool = False):
    """The rotation of queries and keys [batch, head, token, dim] by positions of
    several axes (time, height, width), in one launch; returns both.

    ``cos`` and ``sin`` are tables [positions, pairs]: the pairs (j, j + pairs) or,
    ``interleaved``, (2j, 2j + 1) of the first 2 * pairs entries turn by entry j of row
    ``positions[pair_axes[j]][batch][token]``.  ``positions`` are [axes, batch, token]
    integers, or an ``index_buffer`` of that shape ([batch, token] for one axis), or None
    for ``start + token`` on every axis; ``pair_axes`` gives each pair's axis (None: 0 for all).
    ``key`` may be None, and the query alone is returned then.  Gradients reach queries and
    keys."""
    _tensor_arguments("rope_axes", query=query, cos=cos, sin=sin)
    xs = [query]
    if key is not None:
        _tensor_arguments("rope_axes", key=key)
        xs.append(key)
    start = _integer("rope_axes", "start", start)
    positions = _indices(positions, query)
    axes, pair_axes = _pair_axes("rope_axes", positions, pair_axes, cos)
    out = _C.rope_axes(xs, cos, sin, bool(interleaved), axes, pair_axes, start, positions)
    return out[0] if key is None else tuple(out)


def paged_cache(pages: int, kv_heads: int, page: int, dim: int, dtype: str = "float32", device="cuda"):
    """Pools of keys and values in ``pages`` pages of ``page`` tokens, zero at first; "float32" or "bfloat16"."""
    from .. import _device_str
    if dtype not in ("float32", "bfloat16"):
        raise TypeError(f"paged_cache(): dtype must be 'float32' or 'bfloat16', not {dtype!r}")
    sizes = [_integer("paged_cache", name, value) for name, value in (("pages", pages), ("kv_heads", kv_heads), ("page", page), ("dim", dim))]
    return _C.PagedCache(*sizes, dtype == "bfloat16", _device_str(device, "paged_cache"))


def _cache_arguments(op, cache, table, lengths, like):
    if not isinstance(cache, _C.PagedCache):
        raise TypeError(f"{op}(): argument 'cache' must be PagedCache, not {_type_name(cache)}")
    return _indices(table, like), _indices(lengths, like)


def paged_append(cache, table, lengths, key, value, cos=None, sin=None, *, query=None, positions=None, pair_axes=None, interleaved: bool = False):
    """Writes new tokens' keys and values [batch, key head, token, dim] to the pages that
    ``table`` ([batch, pages] integers, or an ``index_buffer``) gives, the keys turned on the
    way as ``rope_axes`` turns them (``cos`` and ``sin`` None: as they are, and no argument of
    a rotation is taken); returns the turned ``query`` [batch, head, token, dim], if there is one.

    ``lengths`` ([batch]) are the tokens that each sequence has with the new ones: token t
    stands at place ``lengths - tokens + t``, which is also its position on every axis
    where ``positions`` is None.  Tokens before place 0 are padding; neither they nor tokens
    behind the last place of the table's row are written.
    Records no gradient."""
    _tensor_arguments("paged_append", key=key, value=value)
    if (cos is None) != (sin is None):
        raise ValueError("paged_append takes both tables, cos and sin, or neither")
    for name, t in (("cos", cos), ("sin", sin), ("query", query)):
        if t is not None:
            _tensor_arguments("paged_append", **{name: t})
    if cos is None:
        for name, given in (("positions", positions is not None), ("pair_axes", pair_axes is not None), ("interleaved", interleaved)):
            if given:
                raise ValueError(f"paged_append takes no {name} without tables: nothing is turned")
    table, lengths = _cache_arguments("paged_append", cache, table, lengths, key)
    positions = _indices(positions, key)
    axes, pair_axes = _pair_axes("paged_append", positions, pair_axes, cos)
    return _C.paged_append(cache, table, lengths, key, value, query, cos, sin, bool(interleaved), axes, pair_axes, positions)


def paged_attention(query, cache, table, lengths, *, window=None, sinks: int = 0, scale=None, shared: int = 0):
    """``window_attention`` of ``query`` [batch, heads, tokens, dim] over a paged cache.

    The last query of a sequence stands at its last token, ``lengths`` of ``table``'s
    (see ``paged_append``).  The first ``shared`` tokens of every sequence, a prefix that
    all have in common, are read through the table's first row: once for the whole batch
    where that saves enough reading.  Records no gradient."""
    _tensor_arguments("paged_attention", query=query)
    table, lengths = _cache_arguments("paged_attention", cache, table, lengths, query)
    window = None if window is None else _integer("paged_attention", "window", window)
    sinks, shared = _integer("paged_attention", "sinks", sinks), _integer("paged_attention", "shared", shared)
    if window is not None and window < 1:
        raise ValueError(f"paged_attention window has to be at least 1, but got {window}")
    if sinks < 0 or shared < 0:
        raise ValueError(f"paged_attention sinks and shared have to be at least 0, but got {sinks} and {shared}")
    if scale is None:
        scale = 1.0 / math.sqrt(query.shape[-1]) if len(query.shape) and query.shape[-1] else 1.0
    every = (1 << 63) - 1
    return _C.paged_attention(query, cache, table, lengths, min(shared, every), every if window is None else min(window, every),
                              min(sinks, every), float(scale))
