"""Window caches with sinks and attention over them, on torch CUDA tensors.

Operators on one layer's state for programs that run their own layers beside the
runtime: the binding of ``st_cache_append``, ``st_cache_attention``,
``st_cache_unpack`` and ``st_window_attention`` (include/streaming_b200.h).

A cache is two plain tensors ``keys`` and ``values``, [streams, heads, slots,
head_dim] of float32, float16 or bfloat16. Its first ``sinks`` slots keep the
first positions of a stream for good, the other ``window = slots - sinks`` are a
ring: position t lives in slot t when t < sinks and in sinks + (t - sinks) %
window otherwise. A 4-bit cache is uint8 [streams, heads, slots, head_dim // 2]
with ``key_scales`` and ``value_scales``, bfloat16 [streams, heads, slots,
head_dim // 32, 2] (scale and lowest value of every 32 columns; see
``new_cache``).

A stream that starts with a backlog runs ``cache_append`` and
``window_attention`` over all its events at once, then ``cache_append`` and
``cache_attention`` for each further one:

    cache = new_cache(streams, heads, window, head_dim, sinks=4, mode="bf16")
    f = rotation_frequencies(head_dim)
    q, k = cache_append(q, k, v, *cache[:2], positions, f, sinks=4, starts=starts, rotated_keys=True)
    out = window_attention(q, k, v, window=window, sinks=4, starts=starts)
    ...
    q = cache_append(q, k, v, *cache[:2], positions, f, sinks=4)
    out = cache_attention(q, *cache[:2], positions)

Work is queued on the current stream of the tensors' device, which may be
another device than the current one; nothing waits. Positions and starts are
read on the device, so a captured CUDA graph replays with new ones. There is no
backward pass: a call with an input that requires a gradient raises while
gradients are on. Errors are ``StreamError`` with the C status, as the runtime's.
"""
from __future__ import annotations

import ctypes

import torch

from .runtime import StreamError, library

__all__ = ["cache_append", "cache_attention", "new_cache", "rotation_frequencies", "unpack_cache", "window_attention"]

INT4 = 3           # ST_CACHE_INT4
GROUP = 32         # ST_CACHE_GROUP
_MODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_MODE_NAMES = {"fp32": torch.float32, "mixed": torch.float16, "bf16": torch.bfloat16}
_INVALID = -1

_I, _L, _P, _F = ctypes.c_int, ctypes.c_int64, ctypes.c_void_p, ctypes.c_float


class _Cache(ctypes.Structure):
    _fields_ = [("device", _I), ("type", _I), ("streams", _I), ("heads", _I), ("head_dim", _I), ("sinks", _I),
                ("window", _I), ("stream_stride", _L), ("head_stride", _L), ("keys", _P), ("values", _P),
                ("key_scales", _P), ("value_scales", _P)]


class _Rows(ctypes.Structure):
    _fields_ = [("data", _P), ("row_stride", _L), ("head_stride", _L)]


class _Append(ctypes.Structure):
    _fields_ = [("mode", _I), ("heads", _I), ("rows", _L), ("q", _Rows), ("k", _Rows), ("v", _Rows),
                ("q_out", _Rows), ("k_out", _Rows), ("q_gain", _P), ("k_gain", _P), ("epsilon", _F), ("rotary", _I),
                ("frequencies", _P), ("positions", _P), ("starts", _P)]


class _Attend(ctypes.Structure):
    _fields_ = [("mode", _I), ("heads", _I), ("scale", _F), ("q", _Rows), ("out", _Rows), ("positions", _P),
                ("workspace", _P), ("workspace_bytes", ctypes.c_size_t)]


class _Window(ctypes.Structure):
    _fields_ = [("device", _I), ("mode", _I), ("heads", _I), ("kv_heads", _I), ("head_dim", _I), ("sequences", _I),
                ("rows", _L), ("window", _I), ("sinks", _I), ("scale", _F), ("q", _Rows), ("k", _Rows), ("v", _Rows),
                ("out", _Rows), ("starts", _P)]


_INT_MAX = 2 ** 31 - 1
_lib = None


def _library():
    global _lib
    if _lib is None:
        lib = library()
        C = ctypes.POINTER
        for name, args in {"st_cache_append": [C(_Cache), C(_Append), _P],
                           "st_cache_attention_workspace": [C(_Cache), _I, C(ctypes.c_size_t)],
                           "st_cache_attention": [C(_Cache), C(_Attend), _P],
                           "st_cache_unpack": [C(_Cache), _I, _P, _P, _P],
                           "st_window_attention": [C(_Window), _P]}.items():
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = _I, args
        lib.st_cache_error.restype = ctypes.c_char_p
        _lib = lib
    return _lib


def _raise(code: int):
    raise StreamError(code, _library().st_cache_error().decode())


def _refuse(message: str):
    raise StreamError(_INVALID, message)


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _no_gradient(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                _refuse("there is no backward pass: detach the inputs or call under torch.no_grad()")


def _rows(t: torch.Tensor, name: str, device, dtype, rows: int, heads: int, head_dim: int) -> _Rows:
    """[rows, heads, head_dim] with contiguous columns, any row and head strides."""
    if t.device != device or t.dtype != dtype:
        _refuse(f"{name}: expected {dtype} on {device}, got {t.dtype} on {t.device}")
    if t.shape != (rows, heads, head_dim):
        _refuse(f"{name}: expected shape {(rows, heads, head_dim)}, got {tuple(t.shape)}")
    s = t.stride()
    if s[2] != 1:
        _refuse(f"{name}: columns must be contiguous")
    return _Rows(t.data_ptr(), s[0] if rows > 1 else heads * head_dim, s[1] if heads > 1 else head_dim)


def _small(t: torch.Tensor, name: str, device, dtype, count: int) -> int:
    """A contiguous one-dimensional tensor of `count` values; its address."""
    if t.device != device or t.dtype != dtype:
        _refuse(f"{name}: expected {dtype} on {device}, got {t.dtype} on {t.device}")
    if t.shape != (count,) or (count > 1 and t.stride(0) != 1):
        _refuse(f"{name}: expected {count} contiguous values, got shape {tuple(t.shape)}")
    return t.data_ptr()


def _cache(keys, values, key_scales, value_scales, sinks: int) -> _Cache:
    if not 0 <= sinks <= _INT_MAX:
        _refuse(f"sinks: {sinks} is out of range")
    if not keys.is_cuda:
        _refuse(f"keys: expected a CUDA tensor, got {keys.device}")
    four = keys.dtype == torch.uint8
    if not four and keys.dtype not in _MODES:
        _refuse(f"keys: {keys.dtype} is no cache type")
    if keys.dim() != 4 or keys.shape[3] < 1 or keys.shape[0] < 1 or keys.shape[1] < 1:
        _refuse(f"keys: expected [streams, heads, slots, columns], got {tuple(keys.shape)}")
    streams, heads, slots, columns = keys.shape
    if slots > 1 << 30:
        _refuse("a cache has at most 2^30 slots")
    s = keys.stride()
    if (values.shape != keys.shape or values.dtype != keys.dtype or values.device != keys.device
            or (keys.numel() and values.stride() != s)):
        _refuse("values must have the keys' shape, strides, type and device")
    if s[3] != 1 or (slots > 1 and s[2] != columns):
        _refuse("the slots of a cache head must be contiguous")
    if (streams > 1 and s[0] % columns) or (heads > 1 and s[1] % columns):
        _refuse("cache strides must be whole rows")
    # a stride along a dimension of one element is never used
    stream_stride = s[0] // columns if streams > 1 else heads * slots
    head_stride = s[1] // columns if heads > 1 else slots
    if four != (key_scales is not None) or four != (value_scales is not None):
        _refuse("a 4-bit cache has scales, any other has none")
    head_dim = columns * 2 if four else columns
    if four:
        groups = head_dim // GROUP
        for name, t in (("key_scales", key_scales), ("value_scales", value_scales)):
            if t.dtype != torch.bfloat16 or t.device != keys.device or t.shape != (streams, heads, slots, groups, 2):
                _refuse(f"{name}: expected bfloat16 {(streams, heads, slots, groups, 2)} on {keys.device}")
            z = t.stride()
            if (z[4] != 1 or (groups > 1 and z[3] != 2) or (slots > 1 and z[2] != 2 * groups)
                    or (streams > 1 and z[0] != stream_stride * 2 * groups)
                    or (heads > 1 and z[1] != head_stride * 2 * groups)):
                _refuse(f"{name}: strides must be those of the rows")
    return _Cache(keys.device.index, INT4 if four else _MODES[keys.dtype], streams, heads, head_dim, sinks, slots - sinks,
                  stream_stride, head_stride, keys.data_ptr(), values.data_ptr(),
                  key_scales.data_ptr() if four else None, value_scales.data_ptr() if four else None)


def new_cache(streams: int, heads: int, window: int, head_dim: int, *, sinks: int = 0, mode: str = "bf16",
              device="cuda"):
    """An empty cache: (keys, values, key_scales, value_scales), zeroed. ``mode``
    is "fp32", "mixed" (fp16), "bf16" or "int4"; the scales are None unless "int4"."""
    rows = (int(streams), int(heads), int(sinks) + int(window))
    if min(rows) < 1 or sinks < 0 or window < 1 or head_dim < 8 or head_dim % (GROUP if mode == "int4" else 8):
        _refuse("invalid cache dimensions")
    if mode == "int4":
        def scales():
            return torch.zeros(*rows, head_dim // GROUP, 2, dtype=torch.bfloat16, device=device)

        def codes():
            return torch.zeros(*rows, head_dim // 2, dtype=torch.uint8, device=device)
        return codes(), codes(), scales(), scales()
    if mode not in _MODE_NAMES:
        _refuse(f"unknown cache mode {mode!r}")
    keys = torch.zeros(*rows, head_dim, dtype=_MODE_NAMES[mode], device=device)
    return keys, torch.zeros_like(keys), None, None


def rotation_frequencies(head_dim: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """Radians per position of each adjacent pair, base ** (-2 p / head_dim), in
    float64: what ``cache_append`` rotates by. Scaled variants are other tables."""
    p = torch.arange(0, head_dim, 2, dtype=torch.float64, device=device)
    return float(base) ** (p / -head_dim)


def cache_append(q, k, v, keys, values, positions, frequencies, *, sinks: int = 0, starts=None, q_gain=None, k_gain=None,
                 epsilon: float = 1e-6, key_scales=None, value_scales=None, rotated_keys: bool = False, out=None):
    """Norm, rotate and insert new rows (st_cache_append).

    q [rows, heads, head_dim], k and v [rows, cache heads, head_dim];
    ``positions`` int64 [streams], the position of each stream's first new row
    (negative: the stream is idle); ``starts`` int32 [streams + 1], the packed
    rows of each stream, or None for one row each. Per head, q and k are
    RMS-normed with ``q_gain`` and ``k_gain`` (float32 [head_dim]; None: no
    norm) and their pairs turned by position * ``frequencies`` (float64
    [up to head_dim / 2]); k and v enter the cache. Returns the rotated queries
    (written to ``out`` when given, which may be q), or with ``rotated_keys``
    the pair (queries, keys). Rows of idle streams come back as 0; rows of no
    stream are left as they were in ``out``, and undefined in a fresh tensor."""
    cache = _cache(keys, values, key_scales, value_scales, sinks)
    device, dtype = keys.device, q.dtype
    if dtype not in _MODES:
        _refuse(f"q: {dtype} is no row type")
    if q.dim() != 3:
        _refuse(f"q: expected [rows, heads, head_dim], got {tuple(q.shape)}")
    _no_gradient(q, k, v, q_gain, k_gain)
    rows, heads, head_dim = q.shape[0], q.shape[1], cache.head_dim
    args = _Append()
    args.mode, args.heads, args.rows = _MODES[dtype], heads, rows
    args.q = _rows(q, "q", device, dtype, rows, heads, head_dim)
    args.k = _rows(k, "k", device, dtype, rows, cache.heads, head_dim)
    args.v = _rows(v, "v", device, dtype, rows, cache.heads, head_dim)
    if out is None:
        out = torch.empty(rows, heads, head_dim, dtype=dtype, device=device)
    args.q_out = _rows(out, "out", device, dtype, rows, heads, head_dim)
    turned = None
    if rotated_keys:
        turned = torch.empty(rows, cache.heads, head_dim, dtype=dtype, device=device)
        args.k_out = _rows(turned, "k", device, dtype, rows, cache.heads, head_dim)
    if q_gain is not None:
        args.q_gain = _small(q_gain, "q_gain", device, torch.float32, head_dim)
    if k_gain is not None:
        args.k_gain = _small(k_gain, "k_gain", device, torch.float32, head_dim)
    args.epsilon = epsilon
    if frequencies.dim() != 1:
        _refuse("frequencies: expected one dimension")
    args.rotary = frequencies.shape[0]
    args.frequencies = _small(frequencies, "frequencies", device, torch.float64, args.rotary)
    args.positions = _small(positions, "positions", device, torch.int64, cache.streams)
    if starts is not None:
        args.starts = _small(starts, "starts", device, torch.int32, cache.streams + 1)
    code = _library().st_cache_append(cache, args, _stream(device))
    if code:
        _raise(code)
    return (out, turned) if rotated_keys else out


def cache_attention(q, keys, values, positions, *, key_scales=None, value_scales=None, scale: float | None = None,
                    out=None):
    """One query row per stream over its cache (st_cache_attention).

    q [streams, heads, head_dim], heads a multiple of the cache's;
    ``positions`` int64 [streams], the position of each stream's newest inserted
    row (negative: a row of zeros). Every slot up to min(position + 1, slots)
    is seen. ``scale`` defaults to head_dim ** -0.5."""
    cache = _cache(keys, values, key_scales, value_scales, 0)
    device, dtype = keys.device, q.dtype
    if dtype not in _MODES:
        _refuse(f"q: {dtype} is no row type")
    if q.dim() != 3:
        _refuse(f"q: expected [streams, heads, head_dim], got {tuple(q.shape)}")
    _no_gradient(q, keys, values)
    heads, head_dim = q.shape[1], cache.head_dim
    lib = _library()
    args = _Attend()
    args.mode, args.heads = _MODES[dtype], heads
    args.scale = head_dim ** -0.5 if scale is None else scale
    args.q = _rows(q, "q", device, dtype, cache.streams, heads, head_dim)
    if out is None:
        out = torch.empty(cache.streams, heads, head_dim, dtype=dtype, device=device)
    args.out = _rows(out, "out", device, dtype, cache.streams, heads, head_dim)
    args.positions = _small(positions, "positions", device, torch.int64, cache.streams)
    need = ctypes.c_size_t(0)
    code = lib.st_cache_attention_workspace(cache, heads, need)
    if code:
        _raise(code)
    if need.value:
        # from torch's stream-ordered allocator: calls on other streams, and captured graphs, get their own
        work = torch.empty(need.value, dtype=torch.uint8, device=device)
        args.workspace, args.workspace_bytes = work.data_ptr(), need.value
    code = lib.st_cache_attention(cache, args, _stream(device))
    if code:
        _raise(code)
    return out


def unpack_cache(keys, values, *, key_scales, value_scales, dtype=torch.bfloat16):
    """What the rows of a 4-bit cache stand for (st_cache_unpack): (keys, values)
    [streams, heads, slots, head_dim] of ``dtype``, every slot, written or not."""
    cache = _cache(keys, values, key_scales, value_scales, 0)
    if dtype not in _MODES:
        _refuse(f"{dtype} is no row type")
    shape = (*keys.shape[:3], cache.head_dim)
    outs = [torch.empty(shape, dtype=dtype, device=keys.device) for _ in range(2)]
    code = _library().st_cache_unpack(cache, _MODES[dtype], outs[0].data_ptr(), outs[1].data_ptr(), _stream(keys.device))
    if code:
        _raise(code)
    return outs[0], outs[1]


def window_attention(q, k, v, *, window: int, sinks: int = 0, starts=None, scale: float | None = None, out=None):
    """Causal attention of packed sequences with a window and sinks (st_window_attention).

    q [rows, heads, head_dim], k and v [rows, key heads, head_dim], heads a
    multiple of the key heads; ``starts`` int32 [sequences + 1], or None for one
    sequence. Row i of a sequence sees that sequence's rows j <= i with
    i - j < window or j < sinks. Rows of no sequence are left as they were in
    ``out``, and undefined in a fresh tensor."""
    if not q.is_cuda:
        _refuse(f"q: expected a CUDA tensor, got {q.device}")
    device, dtype = q.device, q.dtype
    if dtype not in _MODES:
        _refuse(f"q: {dtype} is no row type")
    if q.dim() != 3 or k.dim() != 3:
        _refuse("q, k and v: expected [rows, heads, head_dim]")
    _no_gradient(q, k, v)
    if window < 1 or sinks < 0:
        _refuse("window is at least 1 and sinks at least 0")
    # no sequence is longer than the largest int: a wider window sees as much
    window, sinks = min(window, _INT_MAX), min(sinks, _INT_MAX)
    rows, heads, head_dim = q.shape
    kv_heads = k.shape[1]
    args = _Window()
    args.device, args.mode, args.heads, args.kv_heads, args.head_dim = device.index, _MODES[dtype], heads, kv_heads, head_dim
    args.rows, args.window, args.sinks = rows, window, sinks
    args.scale = (head_dim ** -0.5 if head_dim else 0.0) if scale is None else scale
    args.q = _rows(q, "q", device, dtype, rows, heads, head_dim)
    args.k = _rows(k, "k", device, dtype, rows, kv_heads, head_dim)
    args.v = _rows(v, "v", device, dtype, rows, kv_heads, head_dim)
    if out is None:
        out = torch.empty(rows, heads, head_dim, dtype=dtype, device=device)
    args.out = _rows(out, "out", device, dtype, rows, heads, head_dim)
    if starts is None:
        args.sequences = 1
    else:
        if starts.dim() != 1 or starts.shape[0] < 1:
            _refuse("starts: expected [sequences + 1]")
        args.sequences = starts.shape[0] - 1
        args.starts = _small(starts, "starts", device, torch.int32, args.sequences + 1)
    code = _library().st_window_attention(args, _stream(device))
    if code:
        _raise(code)
    return out
