"""Calls of the window-cache operators at the edges of what their documentation
allows, against their definitions in 64 bits (tests/cache_reference.py)."""
import ctypes
import re
import subprocess
import sys
import textwrap
from pathlib import Path

import pytest
import torch

import cache_reference as ref
from streaming_transformer_b200.runtime import StreamError
import test_cache_cpu as c_calls
from test_gpu_cache import TYPES, attend_reference, filled_cache, generator, normal, scales_of, starts_of, window_reference

pytestmark = pytest.mark.gpu

ops = pytest.importorskip("streaming_transformer_b200.attention")


@pytest.mark.parametrize("rows", [3, 40])
def test_more_sequences_than_half_of_the_integers(rows):
    # 2^30 + 2^27 sequences (4.8 GB of starts), all empty but two of the last ones
    sequences = 2 ** 30 + 2 ** 27
    starts = torch.zeros(sequences + 1, dtype=torch.int32, device="cuda")
    starts[sequences - 3:] = rows - 1
    starts[sequences] = rows
    g = generator(51)
    q, k, v = (normal(g, rows, h, 64, dtype=torch.bfloat16) for h in (4, 2, 2))
    got = ops.window_attention(q, k, v, window=7, sinks=1, starts=starts)
    for a, b, want, bound in window_reference(q, k, v, [0, rows - 1, rows], 7, 1, 0.125, torch.bfloat16):
        ref.check(got[a:b], want, bound, f"rows {a}..{b}")


def test_a_call_for_a_device_that_is_not_there_leaves_no_error_behind():
    lib, need, missing = c_calls.entry_points(), ctypes.c_size_t(), torch.cuda.device_count()
    cache, _ = filled_cache(generator(52), 1, 2, 9, 64, 0, "bf16")
    q = torch.ones(1, 4, 64, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([8], device="cuda")
    want = ops.cache_attention(q, *cache[:2], at)
    absent = c_calls.cache(device=missing)
    for call in (lambda: lib.st_cache_append(absent, c_calls.append(), None),
                 lambda: lib.st_cache_unpack(c_calls.cache(device=missing, **c_calls.FOUR), 2, c_calls.P, c_calls.P, None),
                 lambda: lib.st_cache_attention(absent, c_calls.attend(), None),
                 lambda: lib.st_window_attention(c_calls.window(device=missing), None)):
        assert call() == -3 and b"device" in lib.st_cache_error()
        assert torch.equal(ops.cache_attention(q, *cache[:2], at), want)
    lib.st_cache_attention_workspace(absent, 4, need)
    assert torch.equal(ops.cache_attention(q, *cache[:2], at), want)


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
@pytest.mark.parametrize("dim", [8, 128, 256])
def test_the_norm_at_the_ends_of_its_range(mode, dim):
    # the largest and least rows whose mean square is said to be held, without an epsilon and with one
    g = generator(53)
    dtype = TYPES[mode]
    exponents = [-50, -49, -40, -31, -29, 0, 30, 50, 57, 58]
    n = len(exponents)
    size = torch.tensor([2.0 ** e for e in exponents], dtype=torch.float64, device="cuda")[:, None, None]
    x = torch.randn(n, 2, dim, generator=g, device="cuda", dtype=torch.float64).clamp(-3, 3)
    x[:, :, 0] = 1.5
    x[:, 1, 1:] *= 2.0 ** -20                    # rows that one column outweighs
    x = (x * size).to(dtype)
    gain = 0.5 + torch.rand(dim, generator=g, device="cuda")
    at = torch.arange(n, device="cuda") * 1000
    f = ops.rotation_frequencies(dim)
    for epsilon in (0.0, 2.0 ** -80, 1e-6, 2.0 ** 122):
        cache = ops.new_cache(n, 2, 4, dim, mode=mode)
        q, k = ops.cache_append(x, x, x, *cache[:2], at, f, q_gain=gain, k_gain=gain, epsilon=epsilon, rotated_keys=True)
        want, bound = ref.rotated(x, at, f, gain, torch.tensor(epsilon, dtype=torch.float32).item(), dtype)
        ref.check(q, want, bound, f"epsilon {epsilon}")
        assert torch.equal(q, k)


def test_the_norm_of_rows_that_are_not_finite_or_zero():
    x = torch.ones(4, 1, 64, device="cuda")
    x[0, 0, 5] = float("inf")                    # x / inf: 0, and the infinite column is no number
    x[1, 0, 7] = float("nan")
    x[2] = 0
    gain = torch.ones(64, device="cuda")
    cache = ops.new_cache(4, 1, 4, 64, mode="fp32")
    at = torch.zeros(4, dtype=torch.int64, device="cuda")
    q = ops.cache_append(x, x, x, *cache[:2], at, ops.rotation_frequencies(64)[:0], q_gain=gain, k_gain=gain)
    assert torch.isnan(q[0, 0, 5]) and int(torch.isnan(q[0]).sum()) == 1 and int((q[0] == 0).sum()) == 63
    assert torch.isnan(q[1]).all() and not q[2].any() and torch.isfinite(q[3]).all()
    q = ops.cache_append(x, x, x, *cache[:2], at, ops.rotation_frequencies(64)[:0], q_gain=gain, k_gain=gain, epsilon=0.0)
    assert torch.isnan(q[2]).all()               # 0 / 0


@pytest.mark.parametrize("heads,kv,dim", [(2, 2, 64), (4, 1, 64), (16, 1, 64), (1, 1, 96), (4, 2, 128), (16, 1, 128), (2, 1, 32),
                                          (1, 1, 256), (3, 1, 160)])
def test_weights_of_fp16_rows_over_four_bits_keep_the_precision_of_fp16(heads, kv, dim):
    # Values of opposite sign at the ends of a group nearly cancel, so that what a weight loses shows. Keys are constant
    # rows (scale 0) and queries sum to about 1, so logits are small and exact. The bound is that of the reference with
    # a weight's rounding at 2^-16, two bf16 numbers (2^-8 twice), in place of one.
    g = generator(54)
    streams, slots = 40, 5
    k_scales, v_scales = (torch.zeros(streams, kv, slots, dim // 32, 2, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    k_scales[..., 1] = normal(g, streams, kv, slots, 1, dtype=torch.bfloat16)
    v_scales[..., 0] = 0.1328125
    v_scales[..., 1] = -7.5 * 0.1328125
    codes = (torch.arange(slots, device="cuda")[:, None] + torch.arange(dim, device="cuda") // 3) % 2 * 15
    v = ref.pack(codes.to(torch.uint8)).expand(streams, kv, -1, -1).contiguous()
    k = torch.zeros_like(v)
    q = (1 + 0.5 * normal(g, streams, heads, dim)).mul(2 / dim).to(torch.float16)
    at = torch.arange(streams, device="cuda") % slots
    got = ops.cache_attention(q, k, v, at, key_scales=k_scales, value_scales=v_scales, scale=1.0)
    group, u = heads // kv, ref.unit(torch.float16)
    see = torch.arange(slots, device="cuda") <= at[:, None]
    for s in range(streams):
        qs = q[s].double().unflatten(0, (kv, group))
        ks, vs = ref.unpack(k[s], k_scales[s]), ref.unpack(v[s], v_scales[s])
        sizes = [(15 * x[s, ..., 0].double() + x[s, ..., 1].double().abs()).repeat_interleave(32, -1) for x in (k_scales, v_scales)]
        mask = see[s].expand(kv, group, -1)
        want, bound = ref.attention(qs, ks, vs, mask, 1.0, torch.float16, sizes)
        size, _ = ref.attention(qs, ks, sizes[1], mask, 1.0, torch.float16, sizes)
        bound = bound - (1 + u) * (ref.unit(torch.bfloat16) - 2.0 ** -16) * size
        ref.check(got[s].unflatten(0, (kv, group)), want, bound, f"stream {s}")


def recipe(where):
    """The documented calls: (for the backlogs, for each further event)."""
    guides = (path.read_text() for path in Path(__file__).parents[1].glob("*.md"))
    text = ops.__doc__ if where == "module" else next(text for text in guides if "= new_cache(" in text)
    block = re.search(r"^ *keys, values.*= new_cache\(.*?(?=^ *```|^ *$)", text, re.M | re.S)[0]
    backlogs, events = re.split(r"^# then.*\n", textwrap.dedent(block), flags=re.M)
    return backlogs, events


@pytest.mark.parametrize("where", ["module", "guide"])
def test_the_documented_calls_give_the_attention_of_each_streams_history(where):
    # two streams with backlogs, one without, and one that stays idle
    g = generator(55)
    heads, kv, dim, window, sizes, more = 4, 2, 64, 24, [60, 0, 10, 0], 20
    backlogs, events = recipe(where)
    total = [n + more for n in sizes]
    history = [[normal(g, n, h, dim, dtype=torch.bfloat16) for h in (heads, kv, kv)] for n in total]
    gains = [0.5 + torch.rand(dim, generator=g, device="cuda") for _ in range(2)] if "gq" in events else [None, None]
    names = dict(vars(ops), streams=4, kv_heads=kv, window=window, head_dim=dim, starts=starts_of(sizes), gq=gains[0], gk=gains[1],
                 positions=torch.tensor([0, 0, 0, -1], device="cuda"))
    names.update(zip("qkv", (torch.cat([h[i][:n] for h, n in zip(history, sizes)]) for i in range(3))))
    exec(backlogs, names)
    got = [[names["out"][a:b]] for a, b in zip(names["starts"].tolist(), names["starts"].tolist()[1:])]
    for t in range(more):
        names.update(zip("qkv", (torch.stack([h[i][n + t] for h, n in zip(history, sizes)]) for i in range(3))))
        exec(events, names)
        for s in range(4):
            got[s].append(names["out"][s:s + 1])
    assert names["positions"].tolist() == [80, 20, 30, -1]
    assert not torch.cat(got[3]).any()
    for s in range(3):
        at = torch.arange(total[s], device="cuda")
        q, k = (ref.rotated(history[s][i], at, names["f"], gains[i], 1e-6, torch.bfloat16)[0] for i in range(2))
        for _, _, want, bound in window_reference(q, k, history[s][2], [0, total[s]], window, 4, dim ** -0.5, torch.bfloat16):
            # the operators see q and k rounded to the type: a logit moves by at most 2 u(T) sum|q k| scale, and a
            # weight by twice that, relative
            products = (q.abs().sum(-1).amax() * k.abs().amax()).item() * dim ** -0.5
            extra = 2 * 2 * 2 * (ref.unit(torch.bfloat16) + 24 * ref.F) * products * history[s][2].double().abs().amax()
            ref.check(torch.cat(got[s]), want, bound + extra, f"stream {s}")
            # and, as that bound is far from what happens: a norm that a wrong slot or angle would leave
            assert (torch.cat(got[s]).double() - want).norm() < 0.02 * want.norm()


def test_window_and_sinks_of_any_integer_type():
    import numpy as np
    q = normal(generator(56), 40, 2, 64, dtype=torch.bfloat16)
    want = ops.window_attention(q, q, q, window=9, sinks=2)
    assert torch.equal(ops.window_attention(q, q, q, window=np.int64(9), sinks=np.int32(2)), want)
    with pytest.raises(StreamError, match="window: expected an integer"):
        ops.window_attention(q, q, q, window=9.0)


@pytest.mark.parametrize("mode", ["mixed", "bf16"])
def test_a_stride_of_a_single_head_is_never_used(mode):
    # whatever it is, the call takes the way of its size, which the bits tell
    g, lib = generator(57), c_calls.entry_points()
    q, k, v = (normal(g, 200, 1, 64, dtype=TYPES[mode]) for _ in range(3))
    want = ops.window_attention(q, k, v, window=50, scale=0.125)
    for stride in (0, 64, 2 ** 40):
        out = torch.empty_like(q)
        a = c_calls.window(mode=1 if mode == "mixed" else 2, heads=1, kv_heads=1, rows=200, window=50, sinks=0, device=torch.cuda.current_device(),
                           q=c_calls.Rows(q.data_ptr(), 64, stride), k=c_calls.Rows(k.data_ptr(), 64, stride),
                           v=c_calls.Rows(v.data_ptr(), 64, stride), out=c_calls.Rows(out.data_ptr(), 64, 64))
        assert lib.st_window_attention(a, torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(out, want), f"head stride {stride}"


@pytest.mark.parametrize("mode", ["fp32", "mixed", "bf16"])
@pytest.mark.parametrize("dim", [64, 72, 128, 200])
def test_strides_of_every_order_take_the_way_of_their_size(mode, dim):
    # heads outermost, rows with a tail, rows whose stride is no multiple of the heads', rows and heads that overlap or
    # repeat: the same bits as of a copy in the usual order
    g = generator(58)
    n, heads, kv = 150, 4, 2
    q, out = normal(g, n, heads, dim, dtype=TYPES[mode]), torch.empty(n, heads, dim, dtype=TYPES[mode], device="cuda")
    pool = normal(g, 400000, dtype=TYPES[mode])
    for strides in ((dim, n * dim), (kv * dim + 8, dim), (dim + 8, n * (dim + 8) + 16), (8, 16), (16, 8), (0, dim), (dim, 0), (0, 0),
                    (kv * (dim + 8), dim + 8)):
        k, v = (pool[8 * i:].as_strided((n, kv, dim), (*strides, 1)) for i in range(2))
        got = ops.window_attention(q, k, v, window=40, sinks=2)
        assert torch.equal(got, ops.window_attention(q, k.contiguous(), v.contiguous(), window=40, sinks=2)), strides
    for strides in ((dim, n * dim), (heads * dim + 8, dim), (heads * (dim + 8), dim + 8)):
        wide = torch.full((400000,), 7.0, dtype=TYPES[mode], device="cuda")
        qs, to = pool.as_strided((n, heads, dim), (*strides, 1)), wide.as_strided((n, heads, dim), (*strides, 1))
        ops.window_attention(qs, q[:, :kv], q[:, kv:], window=40, sinks=2, out=to)
        assert torch.equal(to, ops.window_attention(qs.contiguous(), q[:, :kv], q[:, kv:], window=40, sinks=2, out=out)), strides
        assert int((wide != 7).sum()) == int((to != 7).sum())


@pytest.mark.parametrize("outside", [1e4, float("nan")])
@pytest.mark.parametrize("mode", ["fp32", "mixed", "bf16"])
@pytest.mark.parametrize("dim", [8, 16, 24, 32, 40, 64, 72, 80, 96, 120, 128, 136, 160, 192, 200, 248, 256])
def test_what_rows_of_no_sequence_hold_does_not_count(dim, mode, outside):
    # Large finite values reach the results of the tiles if a mask misses them; values that are not finite make the tiles
    # be done again row by row, so that each way is compared by itself.
    g = generator(59)
    dtype = TYPES[mode]
    for heads, kv, window, sinks, sizes in ((2, 1, 50, 3, [130, 1, 61]), (3, 3, 200, 0, [7, 161]), (1, 1, 33, 40, [97, 33])):
        before, n = 5, 5 + sum(sizes) + 40
        q, k, v = (normal(g, n, h, dim, dtype=dtype) for h in (heads, kv, kv))
        for x in (q, k, v):
            x[:before] = outside
            x[before + sum(sizes):] = outside
            x[before + sum(sizes)::2] *= -1
        starts = starts_of(sizes, before)
        got = torch.full((n, heads, dim), 7.0, dtype=dtype, device="cuda")
        ops.window_attention(q, k, v, window=window, sinks=sinks, starts=starts, out=got)
        for a, b, want, bound in window_reference(q, k, v, starts.tolist(), window, sinks, dim ** -0.5, dtype):
            ref.check(got[a:b], want, bound, f"{heads} heads, rows {a}..{b}")
        assert (got[:before] == 7).all() and (got[before + sum(sizes):] == 7).all()


@pytest.mark.parametrize("mode", ["fp32", "mixed", "bf16", "int4"])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 256])
def test_large_values_in_unseen_slots_do_not_count(mode, dim):
    # unlike NaN, which would show at once, they would only shift a result
    g = generator(60)
    dtype = TYPES.get(mode, torch.bfloat16)
    at = [0, 14, 31, 32, 77, 128]
    cache, held = filled_cache(g, len(at), 2, 140, dim, 0, mode)
    for s, p in enumerate(at):
        for t in cache[2:] if mode == "int4" else cache[:2]:
            t[s, :, p + 1:] = 1e4
    for heads in (2, 6, 24):
        q = normal(g, len(at), heads, dim, dtype=dtype)
        got = ops.cache_attention(q, *cache[:2], torch.tensor(at, device="cuda"), **scales_of(cache))
        want, bound = attend_reference(q, held, at, dim ** -0.5, dtype)
        ref.check(got, want, bound, f"{heads} heads")


@pytest.mark.parametrize("mode", ["fp32", "mixed", "bf16", "int4"])
def test_a_second_backlog_enters_a_full_cache(mode):
    # two appends of many rows, then single events: every slot holds the newest position that belongs there
    g = generator(61)
    dtype, kind = TYPES.get(mode, torch.bfloat16), mode
    heads, kv, dim, window, sinks = 4, 2, 64, 19, 3
    cache = ops.new_cache(3, kv, window, dim, sinks=sinks, mode=kind)
    f = ops.rotation_frequencies(dim)
    positions = torch.zeros(3, dtype=torch.int64, device="cuda")
    keys, values = ([[] for _ in range(3)] for _ in range(2))
    for sizes in ([30, 1, 20], [5, 44, 0], [1, 1, 1], [25, 2, 19], [1, 1, 1]):
        starts = starts_of(sizes)
        q, k, v = (normal(g, sum(sizes), h, dim, dtype=dtype) for h in (heads, kv, kv))
        q, k = ops.cache_append(q, k, v, *cache[:2], positions, f, sinks=sinks, starts=starts, rotated_keys=True, **scales_of(cache))
        for s, (a, b) in enumerate(zip(starts.tolist(), starts.tolist()[1:])):
            keys[s] += k[a:b]
            values[s] += v[a:b]
        positions += starts.diff()
        if sizes == [1, 1, 1]:
            held = [torch.zeros(3, kv, sinks + window, dim, dtype=dtype, device="cuda") for _ in range(2)]
            for s in range(3):
                for t in range(len(keys[s])):
                    if t < sinks or t >= len(keys[s]) - window:
                        slot = t if t < sinks else sinks + (t - sinks) % window
                        held[0][s, :, slot], held[1][s, :, slot] = keys[s][t], values[s][t]
            at = positions - 1
            if mode == "int4":
                stands = [ref.unpack(cache[i], cache[2 + i]) for i in range(2)]
                for x, h in zip(stands, held):    # the right rows: half a step of at most 10 / 15, and roundings to bf16
                    assert (x - h.double()).abs().amax() < 0.75
                sizes4 = [(15 * t[..., 0].double() + t[..., 1].double().abs()).repeat_interleave(32, -1) for t in cache[2:]]
                held = (*stands, *sizes4)
            else:
                assert torch.equal(cache[0], held[0]) and torch.equal(cache[1], held[1])
                held = [h.double() for h in held]
            got = ops.cache_attention(q, *cache[:2], at, **scales_of(cache))
            want, bound = attend_reference(q, held, at.tolist(), dim ** -0.5, dtype)
            ref.check(got, want, bound)


@pytest.mark.parametrize("q_size,k_size,v_scale", [(2.0 ** 119, 2.0 ** -118, 1.0), (1.0, 1.0, 2.0 ** 56), (1.0, 1.0, 2.0 ** -56),
                                                   (2.0 ** -100, 2.0 ** 100, 2.0 ** -20)])
@pytest.mark.parametrize("dim,heads", [(64, 2), (64, 8), (96, 2), (128, 8), (256, 4)])
def test_four_bit_attention_at_the_ends_of_its_range(dim, heads, q_size, k_size, v_scale):
    g = generator(62)
    codes, s, low = ref.quantise(normal(g, 2, 2, 90, dim) * k_size)
    k, ks = ref.pack(codes), torch.stack([s, low], -1)
    v = ref.pack(torch.randint(0, 16, (2, 2, 90, dim), generator=g, device="cuda").to(torch.uint8))
    vs = torch.tensor([v_scale, -7.5 * v_scale], dtype=torch.bfloat16, device="cuda").expand(2, 2, 90, dim // 32, 2).contiguous()
    held = [ref.unpack(k, ks), ref.unpack(v, vs)] + [(15 * x[..., 0].double() + x[..., 1].double().abs()).repeat_interleave(32, -1) for x in (ks, vs)]
    q = normal(g, 2, heads, dim).clamp(-1.9, 1.9).mul(q_size).to(torch.bfloat16)
    at = [89, 40]
    got = ops.cache_attention(q, k, v, torch.tensor(at, device="cuda"), key_scales=ks, value_scales=vs)
    want, bound = attend_reference(q, held, at, dim ** -0.5, torch.bfloat16)
    ref.check(got, want, bound)
    assert (got.double() - want).norm() < 0.01 * want.norm()


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
def test_attention_of_the_largest_values(mode):
    # every value next to 2^127 / slots: the sum stays a number
    g = generator(63)
    slots, dtype = 128, TYPES[mode]
    size = 2.0 ** 127 / slots * 0.99
    q, k = normal(g, 1, 4, 64, dtype=dtype), normal(g, 1, 2, slots, 64, dtype=dtype)
    v = torch.full((1, 2, slots, 64), size, device="cuda").to(dtype)
    got = ops.cache_attention(q, k, v, torch.tensor([slots - 1], device="cuda"))
    want, bound = attend_reference(q, (k.double(), v.double()), [slots - 1], 0.125, dtype)
    ref.check(got, want, bound)
    q, k = normal(g, slots, 4, 64, dtype=dtype), normal(g, slots, 2, 64, dtype=dtype)
    v = torch.full((slots, 2, 64), size, device="cuda").to(dtype)
    got = ops.window_attention(q, k, v, window=slots)
    for _, _, want, bound in window_reference(q, k, v, [0, slots], slots, 0, 0.125, dtype):
        ref.check(got, want, bound)


FIRST_CALLS = """
import sys
import torch
from streaming_transformer_b200 import attention as ops

def rows(*shape):
    return torch.arange(torch.tensor(shape).prod().item(), device="cuda").remainder(7).sub(3).view(shape).to(dtype)

mode = sys.argv[1]
dtype = {"fp32": torch.float32, "mixed": torch.float16}.get(mode, torch.bfloat16)
cache = ops.new_cache(2, 2, 3000, 64, mode=mode)
scales = dict(key_scales=cache[2], value_scales=cache[3])
q, k, v = (rows(2, h, 64) for h in (4, 2, 2))
many = [rows(300, h, 64) for h in (4, 2, 2)]
at, f = torch.tensor([5, 2999], device="cuda"), ops.rotation_frequencies(64)
calls = {
    "append": lambda: ops.cache_append(q, k, v, *cache[:2], at, f, **scales),
    "attend": lambda: ops.cache_attention(q, *cache[:2], at, **scales),
    "unpack": lambda: ops.unpack_cache(*cache[:2], **scales)[0],
    "window": lambda: ops.window_attention(*many, window=90),
}
side = torch.cuda.Stream()
for name in ("append", "attend") + (("unpack",) if mode == "int4" else ("window",)):
    graph = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        out = calls[name]()
    torch.cuda.current_stream().wait_stream(side)
    graph.replay()
    assert torch.equal(out, calls[name]()), name
"""


@pytest.mark.parametrize("mode", ["fp32", "bf16", "int4"])
def test_a_first_call_can_be_captured(mode):
    # in a process of its own, so that nothing has loaded the kernels before
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS, mode], cwd=Path(__file__).parents[1], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.parametrize("mode", ["fp32", "mixed", "bf16", "int4"])
def test_append_rotates_keys_in_place(mode):
    # the C call's q_out and k_out may be q and k themselves
    g, lib = generator(64), c_calls.entry_points()
    dtype, types = TYPES.get(mode, torch.bfloat16), {"fp32": 0, "mixed": 1, "bf16": 2, "int4": 3}
    streams, heads, kv, dim, window, sinks, sizes = 3, 6, 2, 96, 9, 2, [30, 0, 7]
    n = sum(sizes)
    q, k, v = (normal(g, n, h, dim, dtype=dtype) for h in (heads, kv, kv))
    gains = [0.5 + torch.rand(dim, generator=g, device="cuda") for _ in range(2)]
    at, starts, f = torch.tensor([3, 5, 1000], device="cuda"), starts_of(sizes), ops.rotation_frequencies(dim)
    caches = [ops.new_cache(streams, kv, window, dim, sinks=sinks, mode=mode) for _ in range(2)]
    want = ops.cache_append(q, k, v, *caches[0][:2], at, f, sinks=sinks, starts=starts, q_gain=gains[0], k_gain=gains[1], epsilon=1e-5,
                            rotated_keys=True, **scales_of(caches[0]))
    keys, values, ks, vs = caches[1]
    slots = sinks + window
    c = c_calls.cache(device=torch.cuda.current_device(), type=types[mode], streams=streams, heads=kv, head_dim=dim, sinks=sinks, window=window,
                      stream_stride=kv * slots, head_stride=slots, keys=keys.data_ptr(), values=values.data_ptr(),
                      key_scales=ks.data_ptr() if ks is not None else None, value_scales=vs.data_ptr() if vs is not None else None)
    rows = [c_calls.Rows(x.data_ptr(), x.stride(0), dim) for x in (q, k, v)]
    a = c_calls.append(mode=2 if mode == "int4" else types[mode], heads=heads, rows=n, q=rows[0], k=rows[1], v=rows[2], q_out=rows[0], k_out=rows[1],
                       q_gain=gains[0].data_ptr(), k_gain=gains[1].data_ptr(), epsilon=1e-5, rotary=dim // 2, frequencies=f.data_ptr(),
                       positions=at.data_ptr(), starts=starts.data_ptr())
    assert lib.st_cache_append(c, a, torch.cuda.current_stream().cuda_stream) == 0
    for x, y in zip((q, k, *caches[1]), (*want, *caches[0])):
        assert x is None or torch.equal(x, y)


@pytest.mark.parametrize("mode", ["fp32", "mixed", "bf16", "int4"])
def test_append_of_rows_that_repeat_or_lie_in_another_order(mode):
    g = generator(65)
    dtype = TYPES.get(mode, torch.bfloat16)
    n, heads, kv, dim = 40, 4, 2, 64
    pool = normal(g, 100000, dtype=dtype)
    at, starts, f = torch.tensor([7, 0], device="cuda"), starts_of([25, 15]), ops.rotation_frequencies(dim)
    for row, head in ((0, dim), (heads * dim, 0), (0, 0), (dim, n * dim), (8, 16), (heads * dim + 24, dim)):
        q, k, v = (pool[8 * i:].as_strided((n, h, dim), (row, head, 1)) for i, h in enumerate((heads, kv, kv)))
        caches = [ops.new_cache(2, kv, 11, dim, sinks=1, mode=mode) for _ in range(2)]
        results = [ops.cache_append(*x, *c[:2], at, f, sinks=1, starts=starts, rotated_keys=True, **scales_of(c))
                   for x, c in zip(((q, k, v), [t.contiguous() for t in (q, k, v)]), caches)]
        for x, y in zip((*results[0], *caches[0]), (*results[1], *caches[1])):
            assert x is None or torch.equal(x, y), (row, head)


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_sequences_whose_offsets_pass_32_bits(mode, dim):
    # rows 2^24 elements apart: the last ones lie past 2^31 elements, and 2^32 bytes
    g = generator(66)
    n, heads, kv, apart = 150, 2, 1, 2 ** 24
    buffer = torch.empty(n * apart, dtype=TYPES[mode], device="cuda")
    q, k, v, out = (buffer[4096 * i:].as_strided((n, h, dim), (apart, dim, 1)) for i, h in enumerate((heads, kv, kv, heads)))
    for x in (q, k, v):
        x.copy_(normal(g, *x.shape, dtype=TYPES[mode]))
    assert ops.window_attention(q, k, v, window=50, sinks=1, out=out) is out
    assert torch.equal(out, ops.window_attention(*(x.contiguous() for x in (q, k, v)), window=50, sinks=1))
    cache, f = ops.new_cache(1, kv, 30, dim, mode=mode), ops.rotation_frequencies(dim)
    at, starts = torch.tensor([11], device="cuda"), starts_of([n])
    want = ops.cache_append(*(x.contiguous() for x in (q, k, v)), *cache[:2], at, f, starts=starts)
    held = [t.clone() for t in cache[:2]]
    ops.cache_append(q, k, v, *cache[:2], at, f, starts=starts, out=q)
    assert torch.equal(q, want) and all(torch.equal(t, h) for t, h in zip(cache[:2], held))
