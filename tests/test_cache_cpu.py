"""Refusals of the window-cache C entry points, all of them before any CUDA call
(no GPU, pointers that are never followed), and the binding's struct layouts."""
import ctypes

import pytest

from streaming_transformer_b200 import StreamError, library

_I, _L, _P, _F = ctypes.c_int, ctypes.c_int64, ctypes.c_void_p, ctypes.c_float


class Cache(ctypes.Structure):
    _fields_ = [("device", _I), ("type", _I), ("streams", _I), ("heads", _I), ("head_dim", _I), ("sinks", _I),
                ("window", _I), ("stream_stride", _L), ("head_stride", _L), ("keys", _P), ("values", _P),
                ("key_scales", _P), ("value_scales", _P)]


class Rows(ctypes.Structure):
    _fields_ = [("data", _P), ("row_stride", _L), ("head_stride", _L)]


class Append(ctypes.Structure):
    _fields_ = [("mode", _I), ("heads", _I), ("rows", _L), ("q", Rows), ("k", Rows), ("v", Rows),
                ("q_out", Rows), ("k_out", Rows), ("q_gain", _P), ("k_gain", _P), ("epsilon", _F), ("rotary", _I),
                ("frequencies", _P), ("positions", _P), ("starts", _P)]


class Attend(ctypes.Structure):
    _fields_ = [("mode", _I), ("heads", _I), ("scale", _F), ("q", Rows), ("out", Rows), ("positions", _P),
                ("workspace", _P), ("workspace_bytes", ctypes.c_size_t)]


class Window(ctypes.Structure):
    _fields_ = [("device", _I), ("mode", _I), ("heads", _I), ("kv_heads", _I), ("head_dim", _I), ("sequences", _I),
                ("rows", _L), ("window", _I), ("sinks", _I), ("scale", _F), ("q", Rows), ("k", Rows), ("v", Rows),
                ("out", Rows), ("starts", _P)]


def entry_points():
    lib, at = library(), ctypes.POINTER
    for name, args in {"st_cache_append": [at(Cache), at(Append), _P],
                       "st_cache_attention_workspace": [at(Cache), _I, at(ctypes.c_size_t)],
                       "st_cache_attention": [at(Cache), at(Attend), _P],
                       "st_cache_unpack": [at(Cache), _I, _P, _P, _P],
                       "st_window_attention": [at(Window), _P]}.items():
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = _I, args
    lib.st_cache_error.restype = ctypes.c_char_p
    return lib


P = 4096                      # a 16-byte aligned address that nothing reads
INVALID = -1


def cache(**change):
    c = Cache(0, 2, 4, 2, 64, 4, 28, 2 * 32, 32, P, P, None, None)
    for k, v in change.items():
        setattr(c, k, v)
    return c


FOUR = dict(type=3, key_scales=P, value_scales=P)


def rows(heads, dim=64):
    return Rows(P, heads * dim, dim)


def append(**change):
    a = Append()
    a.mode, a.heads, a.rows = 2, 4, 4
    a.q, a.k, a.v, a.q_out = rows(4), rows(2), rows(2), rows(4)
    a.epsilon, a.rotary, a.frequencies, a.positions = 1e-6, 32, P, P
    for k, v in change.items():
        setattr(a, k, v)
    return a


def attend(**change):
    a = Attend()
    a.mode, a.heads, a.scale, a.q, a.out, a.positions = 2, 4, 0.125, rows(4), rows(4), P
    for k, v in change.items():
        setattr(a, k, v)
    return a


def window(**change):
    a = Window()
    a.mode, a.heads, a.kv_heads, a.head_dim, a.sequences, a.rows, a.window, a.sinks, a.scale = 2, 4, 2, 64, 1, 10, 5, 1, 0.125
    a.q, a.k, a.v, a.out = rows(4), rows(2), rows(2), Rows(2 * P, 256, 64)
    for k, v in change.items():
        setattr(a, k, v)
    return a


def refused(code, match):
    assert code == INVALID
    assert match in entry_points().st_cache_error().decode()


CACHE = [
    (dict(device=-1), "device"), (dict(device=64), "device"), (dict(type=4), "cache type"), (dict(type=-1), "cache type"),
    (dict(streams=0), "streams and heads"), (dict(streams=65536), "streams and heads"), (dict(heads=0), "streams and heads"),
    (dict(head_dim=0), "head_dim"), (dict(head_dim=60), "head_dim"), (dict(head_dim=264), "head_dim"),
    (dict(FOUR, head_dim=80), "multiple of 32"), (dict(sinks=-1), "sinks"), (dict(window=0), "window"),
    (dict(window=2 ** 30), "2^30"), (dict(keys=None), "null"), (dict(values=None), "null"), (dict(keys=P + 8), "16-byte"),
    (dict(key_scales=P), "scales"), (dict(type=3), "scales"), (dict(FOUR, value_scales=P + 4), "16-byte"),
    (dict(stream_stride=-1), "strides"), (dict(head_stride=2 ** 41), "strides"),
]


@pytest.mark.parametrize("change,match", CACHE, ids=lambda v: str(v))
def test_cache_descriptors_that_are_refused(change, match):
    lib, need = entry_points(), ctypes.c_size_t()
    refused(lib.st_cache_append(cache(**change), append(), None), match)
    refused(lib.st_cache_attention(cache(**change), attend(), None), match)
    refused(lib.st_cache_attention_workspace(cache(**change), 4, need), match)


@pytest.mark.parametrize("change,match", [
    (dict(mode=3), "row mode"), (dict(mode=1), "cache's type"), (dict(heads=0), "query heads"), (dict(rows=-1), "rows are"),
    (dict(rows=2 ** 31), "rows are"), (dict(rows=5), "one row for each stream"), (dict(q=Rows(None, 256, 64)), "q: null"),
    (dict(k=Rows(P + 2, 128, 64)), "k: must start"), (dict(v=Rows(P, 128, 60)), "v: strides must be"),
    (dict(q=Rows(P, -256, 64)), "q: strides out"), (dict(q_out=Rows(P, 128, 64)), "q_out: strides let"),
    (dict(q_out=Rows(P, 0, 64)), "q_out: strides let"), (dict(k_out=Rows(P, 64, 64)), "k_out: strides let"),
    (dict(positions=None), "null positions"), (dict(epsilon=-1e-6), "epsilon"), (dict(epsilon=float("nan")), "epsilon"),
    (dict(epsilon=float("inf")), "epsilon"), (dict(rotary=33), "rotary"), (dict(rotary=-1), "rotary"),
    (dict(frequencies=None), "rotary"), (dict(q_gain=P + 4), "gains"),
    (dict(q=Rows(P, 256, 2 ** 34)), "q: head strides"), (dict(k_out=Rows(P, 128, 2 ** 34)), "k_out: head strides"),
], ids=lambda v: str(v))
def test_append_arguments_that_are_refused(change, match):
    refused(entry_points().st_cache_append(cache(), append(**change), None), match)


def test_overlapping_caches_are_read_but_not_written():
    lib, need = entry_points(), ctypes.c_size_t()
    for change in (dict(stream_stride=0), dict(head_stride=31), dict(stream_stride=32, head_stride=32)):
        refused(lib.st_cache_append(cache(**change), append(), None), "overlap")
        assert lib.st_cache_attention_workspace(cache(**change), 4, need) == 0


def test_null_arguments_and_types_across_caches():
    lib = entry_points()
    refused(lib.st_cache_append(None, append(), None), "null cache")
    refused(lib.st_cache_append(cache(), None, None), "null arguments")
    refused(lib.st_cache_attention(cache(), None, None), "null arguments")
    refused(lib.st_cache_attention_workspace(cache(), 4, None), "null pointer")
    refused(lib.st_window_attention(None, None), "null arguments")
    refused(lib.st_cache_append(cache(**FOUR), append(mode=0), None), "fp16 or bf16")
    refused(lib.st_cache_attention(cache(**FOUR), attend(mode=0), None), "fp16 or bf16")
    refused(lib.st_cache_unpack(cache(), 2, P, P, None), "only a 4-bit cache")
    refused(lib.st_cache_unpack(cache(**FOUR), 3, P, P, None), "row mode")
    refused(lib.st_cache_unpack(cache(**FOUR), 2, P, None, None), "null pointer")
    refused(lib.st_cache_unpack(cache(**FOUR), 2, P, P + 8, None), "16-byte")


@pytest.mark.parametrize("change,match", [
    (dict(mode=-1), "row mode"), (dict(heads=3), "multiple of the cache"), (dict(heads=65536), "multiple of the cache"),
    (dict(q=Rows(None, 256, 64)), "q: null"), (dict(out=Rows(P, 0, 64)), "out: strides let"),
    (dict(positions=None), "null positions"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
], ids=lambda v: str(v))
def test_attention_arguments_that_are_refused(change, match):
    refused(entry_points().st_cache_attention(cache(), attend(**change), None), match)


@pytest.mark.parametrize("change,match", [
    (dict(device=-1), "device"), (dict(mode=4), "row mode"), (dict(heads=3), "multiple of the key heads"), (dict(kv_heads=0), "key heads"),
    (dict(head_dim=68), "multiple of 8"), (dict(head_dim=512), "up to 256"), (dict(rows=2 ** 30 + 1), "rows are"), (dict(out=rows(4)), "may not be an input"),
    (dict(window=0), "window"), (dict(sinks=-1), "sinks"), (dict(sequences=2), "one sequence"),
    (dict(sequences=-1, starts=P), "one sequence"), (dict(scale=float("nan")), "scale"), (dict(q=Rows(P + 8, 256, 64)), "q: must start"),
    (dict(k=Rows(P, 128, 4)), "k: strides must be"), (dict(out=Rows(P, 256, 32)), "out: strides let"),
], ids=lambda v: str(v))
def test_window_arguments_that_are_refused(change, match):
    refused(entry_points().st_window_attention(window(**change), None), match)


def test_the_binding_needs_cuda_tensors():
    torch = pytest.importorskip("torch")
    from streaming_transformer_b200 import attention as ops
    keys = torch.zeros(1, 1, 4, 64)
    q = torch.zeros(1, 1, 64)
    for call in (lambda: ops.cache_attention(q, keys, keys, torch.zeros(1, dtype=torch.int64)), lambda: ops.window_attention(q, q, q, window=2)):
        with pytest.raises(StreamError, match="expected a CUDA tensor"):
            call()


def test_new_cache_shapes_and_refusals():
    pytest.importorskip("torch")
    from streaming_transformer_b200 import attention as ops
    k, v, ks, vs = ops.new_cache(2, 3, 5, 64, sinks=2, mode="int4", device="cpu")
    assert k.shape == v.shape == (2, 3, 7, 32) and ks.shape == vs.shape == (2, 3, 7, 2, 2)
    k, v, ks, vs = ops.new_cache(1, 1, 1, 8, mode="fp32", device="cpu")
    assert k.shape == (1, 1, 1, 8) and ks is None and vs is None
    for bad in (dict(window=0), dict(streams=0), dict(head_dim=12), dict(head_dim=264), dict(head_dim=80, mode="int4"), dict(sinks=-1), dict(mode="int8")):
        with pytest.raises(StreamError):
            ops.new_cache(**{**dict(streams=1, heads=1, window=4, head_dim=64, device="cpu"), **bad})
