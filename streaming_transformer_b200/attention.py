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

    keys, values, _, _ = new_cache(streams, kv_heads, window, head_dim, sinks=4, mode="bf16")
    f = rotation_frequencies(head_dim)
    q, k = cache_append(q, k, v, keys, values, positions, f, sinks=4, starts=starts, rotated_keys=True)
    out = window_attention(q, k, v, window=window, sinks=4, starts=starts)
    positions += torch.where(positions >= 0, starts.diff(), 0)  # the next event's; a stream at a negative one is idle
    # then, for each further event of every stream
    q = cache_append(q, k, v, keys, values, positions, f, sinks=4)
    out = cache_attention(q, keys, values, positions)
    positions += positions >= 0

Work is queued on the current stream of the tensors' device, which may be
another device than the current one; nothing waits. Positions and starts are
read on the device, so a captured CUDA graph replays with new ones. There is no
backward pass: a call with an input (frequencies, gains and scales among them)
or a cache that requires a gradient raises while gradients are on, and one with
a forward-mode tangent always. Errors are ``StreamError`` with the C status, as the runtime's.
"""
from __future__ import annotations

import importlib.util

import torch

from .runtime import LIB_PATH, StreamError

__all__ = ["cache_append", "cache_attention", "new_cache", "rotation_frequencies", "unpack_cache", "window_attention"]

GROUP = 32         # ST_CACHE_GROUP
_MODES = {"fp32": torch.float32, "mixed": torch.float16, "bf16": torch.bfloat16}


def _load():
    path = LIB_PATH.with_name("attention_binding.so")
    if not path.exists():
        raise StreamError(-3, f"binding missing: {path} (run python -m streaming_transformer_b200.build)")
    spec = importlib.util.spec_from_file_location("attention_binding", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.set_error(StreamError)
    return module


_native = _load()
_TYPES = {t: torch.empty(0, dtype=t) for t in _MODES.values()}


def _refuse(message: str):
    raise StreamError(-1, message)


def new_cache(streams: int, heads: int, window: int, head_dim: int, *, sinks: int = 0, mode: str = "bf16",
              device="cuda"):
    """An empty cache: (keys, values, key_scales, value_scales), zeroed. ``mode``
    is "fp32", "mixed" (fp16), "bf16" or "int4"; the scales are None unless "int4"."""
    rows = (int(streams), int(heads), int(sinks) + int(window))
    if min(rows) < 1 or sinks < 0 or window < 1 or not 8 <= head_dim <= 256 or head_dim % (GROUP if mode == "int4" else 8):
        _refuse("invalid cache dimensions")
    if mode == "int4":
        def scales():
            return torch.zeros(*rows, head_dim // GROUP, 2, dtype=torch.bfloat16, device=device)

        def codes():
            return torch.zeros(*rows, head_dim // 2, dtype=torch.uint8, device=device)
        return codes(), codes(), scales(), scales()
    if mode not in _MODES:
        _refuse(f"unknown cache mode {mode!r}")
    keys = torch.zeros(*rows, head_dim, dtype=_MODES[mode], device=device)
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
    stream are left as they were in ``out``, and undefined in a fresh tensor.
    A row's mean square is an fp32 number: normed values stay below 2 ** 60, and
    the largest of a row above 2 ** -50 where epsilon is below 2 ** -60."""
    return _native.append(q, k, v, keys, values, positions, frequencies, sinks, starts, q_gain, k_gain, epsilon,
                          key_scales, value_scales, rotated_keys, out)


def cache_attention(q, keys, values, positions, *, key_scales=None, value_scales=None, scale: float | None = None,
                    out=None):
    """One query row per stream over its cache (st_cache_attention).

    q [streams, heads, head_dim], heads a multiple of the cache's;
    ``positions`` int64 [streams], the position of each stream's newest inserted
    row (negative: a row of zeros). Every slot up to min(position + 1, slots)
    is seen. ``scale`` defaults to head_dim ** -0.5; ``out`` may be q. Over a
    4-bit cache, value scales are 0 or 2 ** -56 to 2 ** 56 and queries below
    2 ** 120; seen values of any cache stay below 2 ** 127 / slots."""
    return _native.attend(q, keys, values, positions, key_scales, value_scales, scale, out)


def unpack_cache(keys, values, *, key_scales, value_scales, dtype=torch.bfloat16):
    """What the rows of a 4-bit cache stand for (st_cache_unpack): (keys, values)
    [streams, heads, slots, head_dim] of ``dtype``, every slot, written or not."""
    if dtype not in _TYPES:
        _refuse(f"{dtype} is no row type")
    return _native.unpack(keys, values, key_scales, value_scales, _TYPES[dtype])


def window_attention(q, k, v, *, window: int, sinks: int = 0, starts=None, scale: float | None = None, out=None):
    """Causal attention of packed sequences with a window and sinks (st_window_attention).

    q [rows, heads, head_dim], k and v [rows, key heads, head_dim], heads a
    multiple of the key heads; ``starts`` int32 [sequences + 1], or None for one
    sequence. Row i of a sequence sees that sequence's rows j <= i with
    i - j < window or j < sinks. Rows of no sequence are left as they were in
    ``out``, which may not overlap an input, and undefined in a fresh tensor."""
    return _native.window(q, k, v, window, sinks, starts, scale, out)
