"""The window-cache operators on the GPU against their definitions in 64 bits
(tests/cache_reference.py has the formulas and derives the bounds)."""
import itertools

import pytest
import torch

import cache_reference as ref
from streaming_transformer_b200.runtime import StreamError

pytestmark = pytest.mark.gpu

ops = pytest.importorskip("streaming_transformer_b200.attention")

TYPES = {"fp32": torch.float32, "mixed": torch.float16, "bf16": torch.bfloat16}


def generator(seed):
    return torch.Generator("cuda").manual_seed(seed)


def normal(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def starts_of(sizes, offset=0):
    out = [offset]
    for n in sizes:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device="cuda")


def filled_cache(g, streams, heads, window, dim, sinks, mode, dtype=torch.bfloat16):
    """(keys, values, key_scales, value_scales) and the float64 values they stand for
    (4-bit: and the bounds of their sizes)."""
    rows = (streams, heads, sinks + window)
    if mode != "int4":
        k, v = (normal(g, *rows, dim, dtype=TYPES[mode]) for _ in range(2))
        return (k, v, None, None), (k.double(), v.double())
    packed, scales, held, sizes = [], [], [], []
    for _ in range(2):
        codes, s, low = ref.quantise(normal(g, *rows, dim))
        packed.append(ref.pack(codes))
        scales.append(torch.stack([s, low], -1))
        held.append(ref.unpack(packed[-1], scales[-1]))
        sizes.append((15 * s.double() + low.double().abs()).repeat_interleave(32, -1))
    return (*packed, *scales), (*held, *sizes)


def scales_of(cache):
    return dict(key_scales=cache[2], value_scales=cache[3])


# ---------------------------------------------------------------- append

APPEND = [
    # mode, heads, kv, dim, window, sinks, sizes (None: one row a stream), streams, rotary, gains
    ("fp32", 8, 8, 64, 128, 4, None, 1, 32, True),
    ("fp32", 3, 1, 8, 5, 0, None, 7, 4, True),
    ("fp32", 2, 2, 256, 7, 2, [3, 0, 21, 1], 4, 128, True),
    ("fp32", 4, 2, 40, 9, 3, [13, 2], 2, 13, True),
    ("mixed", 16, 4, 80, 33, 1, [1, 40, 0, 0, 5], 5, 40, True),
    ("mixed", 5, 5, 16, 6, 6, None, 300, 8, False),
    ("bf16", 16, 16, 64, 256, 4, None, 64, 32, True),
    ("bf16", 32, 8, 128, 20, 4, [57, 1, 0, 20, 24, 25], 6, 64, True),
    ("bf16", 7, 1, 96, 1, 0, [4, 1], 2, 0, True),
    ("bf16", 1, 1, 256, 3, 1, [600, 2], 2, 128, False),
    ("int4", 8, 8, 64, 19, 2, [30, 0, 3], 3, 32, True),
    ("int4", 32, 8, 128, 64, 4, None, 17, 64, True),
    ("int4", 4, 2, 32, 5, 0, [1, 9], 2, 16, False),
    ("int4", 6, 2, 96, 11, 1, [12, 12], 2, 40, True),
    ("int4", 2, 1, 256, 4, 0, [5], 1, 128, True),
    ("int4", 3, 3, 224, 9, 1, [14], 1, 112, True),
    ("bf16", 2, 1, 200, 12, 2, None, 3, 51, True),
    ("mixed", 40, 20, 128, 7, 1, None, 5, 64, True),       # more rows than a CTA's lanes hold at a time
    ("mixed", 2, 1, 16, 3, 1, [0, 2, 1] * 200, 600, 8, True),          # more streams than a CTA has threads
    ("fp32", 1, 1, 8, 2, 0, [0] * 255 + [1, 0, 3], 258, 4, True),
    # more rows than are resident at once: CTAs of 128 threads
    ("fp32", 3, 1, 40, 7, 2, [300, 0, 461], 3, 20, True),
    ("mixed", 20, 2, 128, 33, 1, [5, 800], 2, 64, True),
    ("bf16", 2, 1, 256, 9, 4, None, 750, 128, True),
    ("bf16", 5, 5, 16, 2, 0, [0, 2, 1] * 300, 900, 8, True),
    ("int4", 4, 2, 64, 19, 2, [790, 3], 2, 32, True),
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(map(str, c[:6])))
def test_append_matches_the_definition(case):
    mode, heads, kv, dim, window, sinks, sizes, streams, rotary, gains = case
    g = generator(7)
    dtype = TYPES.get(mode, torch.bfloat16)
    before = 3 if sizes else 0                       # rows of no stream, ahead of the first and behind the last
    rows = (before + sum(sizes) + 2) if sizes else streams
    starts = starts_of(sizes, before) if sizes else None
    q, k, v = (normal(g, rows, h, dim, dtype=dtype) for h in (heads, kv, kv))
    cache, held = filled_cache(g, streams, kv, window, dim, sinks, mode)
    old = [None if t is None else t.clone() for t in cache]
    # young, at the sinks' edge, far, and (from three streams on) one idle stream
    at = [(0, max(0, sinks - 1), (1 << 26) - 5, -1, 12345, 2 * window)[i % 6] for i in range(streams)]
    positions = torch.tensor(at, dtype=torch.int64, device="cuda")
    f = ops.rotation_frequencies(dim)[:rotary]
    gain = [0.5 + torch.rand(dim, generator=g, device="cuda") if gains else None for _ in range(2)]
    out = torch.full((rows, heads, dim), 7.0, dtype=dtype, device="cuda")
    _, turned = ops.cache_append(q, k, v, cache[0], cache[1], positions, f, sinks=sinks, starts=starts, q_gain=gain[0],
                                 k_gain=gain[1], epsilon=1e-5, rotated_keys=True, out=out, **scales_of(cache))
    edges = starts.tolist() if sizes else list(range(streams + 1))
    assert torch.equal(out[:edges[0]], torch.full_like(out[:edges[0]], 7)), "rows ahead of the first stream"
    assert torch.equal(out[edges[-1]:], torch.full_like(out[edges[-1]:], 7)), "rows behind the last stream"
    written = torch.zeros(streams, sinks + window, dtype=torch.bool, device="cuda")
    now = [ref.unpack(cache[i], cache[2 + i]) if mode == "int4" else cache[i] for i in range(2)]
    for s in range(streams):
        a, b = edges[s], edges[s + 1]
        if at[s] < 0:
            assert not out[a:b].any() and not turned[a:b].any()
            continue
        place = torch.arange(at[s], at[s] + b - a, device="cuda")
        for got, x, gn in ((out, q, gain[0]), (turned, k, gain[1])):
            want, bound = ref.rotated(x[a:b], place, f, gn, 1e-5, dtype)
            if b > a:
                ref.check(got[a:b], want, bound, f"stream {s}")
        slots = ref.slots_of(place.tolist(), at[s] + b - a - 1, sinks, window)
        keep = [i for i, t in enumerate(slots) if t is not None]
        if not keep:
            continue
        where = torch.tensor([slots[i] for i in keep], device="cuda")
        assert len(set(where.tolist())) == len(keep)
        written[s, where] = True
        rows_in = torch.tensor(keep, device="cuda") + a
        kw, kb = ref.rotated(k[rows_in], place[torch.tensor(keep, device="cuda")], f, gain[1], 1e-5, torch.float32)
        if mode == "int4":
            # v enters as it is: the stored words are those of the definition
            codes, sc, low = ref.quantise(v[rows_in])
            assert torch.equal(cache[1][s][:, where].transpose(0, 1), ref.pack(codes))
            assert torch.equal(cache[3][s][:, where].transpose(0, 1), torch.stack([sc, low], -1))
            # k is off by half a step, plus what bf16 takes from the scale (15 steps) and from the lowest value
            step = cache[2][s][:, where].double().transpose(0, 1)
            slack = (step[..., :1] * (0.5 + 15 * 2.0 ** -9 + 1e-4) + step[..., 1:].abs() * 2.0 ** -8).expand(*step.shape[:-1], 32)
            ref.check(now[0][s][:, where].transpose(0, 1), kw, slack.flatten(-2) + kb, f"4-bit keys of stream {s}")
        else:
            # one rounding, from the same fp32 value as the returned row
            assert torch.equal(cache[0][s][:, where].transpose(0, 1), turned[rows_in])
            assert torch.equal(cache[1][s][:, where].transpose(0, 1), v[rows_in])
    for t, o in zip(cache, old):
        if t is not None:
            left = ~written[:, None, :].expand(-1, kv, -1)
            assert torch.equal(t[left], o[left]), "slots that no row entered"


def test_append_in_place_and_strided():
    # q, k and v as the thirds of one projection, q rotated in place
    g = generator(3)
    n, heads, dim = 12, 4, 64
    qkv = normal(g, n, 3, heads, dim, dtype=torch.bfloat16)
    q, k, v = (qkv[:, i] for i in range(3))
    saved = qkv.clone()
    f = ops.rotation_frequencies(dim)
    big = torch.zeros(heads, n, 2, 9, dim, dtype=torch.bfloat16, device="cuda")   # [head][stream][k or v][slot]
    keys, values = (big[:, :, i].transpose(0, 1) for i in range(2))
    positions = torch.arange(n, device="cuda")
    out = ops.cache_append(q, k, v, keys, values, positions, f, sinks=1, out=q)
    assert out is q
    assert torch.equal(qkv[:, 1:], saved[:, 1:])
    want, bound = ref.rotated(saved[:, 0], positions, f, None, 0, torch.bfloat16)
    ref.check(q, want, bound)
    want, bound = ref.rotated(saved[:, 1], positions, f, None, 0, torch.bfloat16)
    for s in range(n):
        slot = s if s < 1 else 1 + (s - 1) % 8
        ref.check(keys[s, :, slot], want[s], bound[s])
        assert torch.equal(values[s, :, slot], saved[s, 2])
    assert int((big != 0).any(-1).sum()) == 2 * n * heads


def test_four_bit_groups_at_their_limits():
    # pass-through rows (no norm, no rotation): the stored words follow the definition, group by group
    dim, inf, nan = 32 * 8, float("inf"), float("nan")
    x = torch.zeros(1, 1, dim)
    x[..., :32] = torch.linspace(-1e-38, 1e-38, 32)       # the scale is below bf16's normal numbers
    x[..., 32:64] = 3.0                                   # constant: scale 0
    x[..., 64:96] = torch.linspace(-1e-40, 1e-40, 32)     # the range underflows bf16's normal numbers
    x[..., 96:128] = torch.linspace(-3e38, 3e38, 32)      # the range overflows fp32
    x[..., 128:160] = 1.0
    x[..., 131] = inf
    x[..., 160:192] = 1.0
    x[..., 191] = nan
    x[..., 192:224] = torch.linspace(1000, 1001, 32)      # far from zero: the lowest value is rounded
    x[..., 224:256] = torch.arange(32) % 16
    v = x.to(torch.bfloat16).cuda()
    cache = ops.new_cache(1, 1, 2, dim, mode="int4")
    f = ops.rotation_frequencies(dim)[:0]
    at = torch.zeros(1, dtype=torch.int64, device="cuda")
    ops.cache_append(v, v, v, cache[0], cache[1], at, f, **scales_of(cache))
    for got in ops.unpack_cache(*cache[:2], dtype=torch.float32, **scales_of(cache)):
        got = got[0, 0, 0]
        codes, s, low = ref.quantise(v[0, 0])
        want = ref.unpack(ref.pack(codes), torch.stack([s, low], -1)).float()
        bad = torch.zeros(dim, dtype=torch.bool, device="cuda")
        bad[96:192] = True
        assert torch.isnan(got[bad]).all()
        assert torch.equal(got[~bad], want[~bad])
        assert torch.equal(got[32:64], v[0, 0, 32:64].float())
        assert torch.equal(got[224:], v[0, 0, 224:].float())
    assert not ops.unpack_cache(*cache[:2], **scales_of(cache))[0][0, 0, 1].any(), "the slot that nothing entered"


@pytest.mark.parametrize("dtype", list(TYPES.values()), ids=list(TYPES))
def test_unpack_matches_the_definition(dtype):
    g = generator(11)
    cache, held = filled_cache(g, 3, 2, 37, 96, 1, "int4")
    for got, want in zip(ops.unpack_cache(*cache[:2], dtype=dtype, **scales_of(cache)), held[:2]):
        # lowest + scale * code: the product is exact in fp32 (8 + 4 bits), one rounding of the sum, one to the type
        ref.check(got, want, want.abs() * (ref.unit(dtype) + 2 * ref.F) + ref.TINY[dtype])


# ---------------------------------------------------------------- attention over a cache

ATTEND = [
    # mode, row type, heads, kv, dim, slots, positions
    ("fp32", None, 8, 8, 64, 132, [0, 131, 5000, 63, -1]),
    ("fp32", None, 6, 2, 40, 77, [76, 75, 31]),
    ("fp32", None, 24, 1, 256, 45, [44, 7]),
    ("fp32", None, 3, 3, 8, 1, [0, -5]),
    ("fp32", None, 32, 4, 128, 1111, [1110, 600]),
    ("mixed", None, 4, 4, 64, 260, [259, 15, 16, 17, -1, 0]),
    ("mixed", None, 14, 2, 80, 333, [10 ** 9, 300, 1]),
    ("mixed", None, 16, 1, 128, 2049, [2048, 1000]),
    ("bf16", None, 16, 16, 64, 256, [255, 31, 32, 33, 100]),
    ("bf16", None, 32, 8, 128, 700, [699, 0, -1, 350]),
    ("bf16", None, 21, 3, 96, 129, [128, 127]),
    ("bf16", None, 17, 1, 256, 97, [96, 40]),
    ("bf16", None, 40, 1, 32, 65, [64, 2]),
    ("bf16", None, 2, 1, 16, 50, [49]),
    ("bf16", None, 8, 1, 64, 20000, [30000]),
    ("int4", "bf16", 16, 16, 64, 260, [259, 31, 32, 33, 0, -1]),
    ("int4", "mixed", 16, 16, 64, 516, [515, 100]),
    ("int4", "bf16", 32, 8, 128, 1000, [999, 1, 500]),
    ("int4", "mixed", 14, 2, 96, 201, [200, 64]),
    ("int4", "bf16", 9, 1, 32, 65, [64, 3]),
    ("int4", "bf16", 20, 1, 256, 95, [94, 47]),
    ("int4", "bf16", 16, 1, 128, 30000, [29999]),
    ("bf16", None, 6, 2, 72, 100, [99, 31]),
    ("mixed", None, 3, 1, 136, 61, [60, 15]),
    ("bf16", None, 1, 1, 200, 40, [39]),
    ("bf16", None, 5, 5, 8, 33, [32, 5]),
    ("int4", "bf16", 4, 2, 160, 70, [69, 16]),
    ("int4", "mixed", 2, 2, 192, 35, [34]),
    ("int4", "bf16", 12, 1, 224, 130, [129, 64]),
    ("int4", "bf16", 3, 3, 32, 3000, [2999]),
    ("fp32", None, 5, 5, 24, 4100, [4099, 77]),
    ("bf16", None, 1, 1, 64, 500, [499]),          # 7 parts of one head: an odd number of statistics ahead of the sums
    ("fp32", None, 1, 1, 32, 450, [449]),
    ("int4", "bf16", 1, 1, 64, 460, [459, 100, 7]),
    ("mixed", None, 3, 3, 128, 450, [449]),
]


def attend_reference(q, held, positions, scale, dtype):
    outs, bounds = [], []
    for s, p in enumerate(positions):
        slots, kv = held[0].shape[2], held[0].shape[1]
        see = (torch.arange(slots, device="cuda") <= p)[None, None]
        group = q.shape[1] // kv
        sizes = (held[2][s], held[3][s]) if len(held) == 4 else None
        o, b = ref.attention(q[s].double().unflatten(0, (kv, group)), held[0][s], held[1][s], see.expand(kv, group, -1), scale, dtype, sizes)
        outs.append(o.flatten(0, 1))
        bounds.append(b.flatten(0, 1))
    return torch.stack(outs), torch.stack(bounds)


@pytest.mark.parametrize("case", ATTEND, ids=lambda c: "-".join(map(str, c[:6])))
def test_cache_attention_matches_the_definition(case):
    mode, rows, heads, kv, dim, slots, at = case
    g = generator(5)
    dtype = TYPES[rows or mode]
    cache, held = filled_cache(g, len(at), kv, slots, dim, 0, mode)
    q = normal(g, len(at), heads, dim, dtype=dtype)
    positions = torch.tensor(at, dtype=torch.int64, device="cuda")
    for scale in (None, 0.7, -0.2, 0.0):
        got = ops.cache_attention(q, *cache[:2], positions, scale=scale, **scales_of(cache))
        want, bound = attend_reference(q, held, at, dim ** -0.5 if scale is None else scale, dtype)
        ref.check(got, want, bound, f"scale {scale}")


@pytest.mark.parametrize("mode", ["fp32", "mixed", "bf16", "int4"])
def test_unseen_slots_do_not_count_whatever_they_hold(mode):
    g = generator(6)
    dtype = TYPES.get(mode, torch.bfloat16)
    at = [4, 16, 40, 99]
    cache, held = filled_cache(g, 4, 2, 150, 64, 0, mode)
    for s, p in enumerate(at):
        if mode == "int4":
            for t in cache[2:]:
                t[s, :, p + 1:] = float("nan")
        else:
            cache[0][s, :, p + 1:] = float("nan")
            cache[1][s, :, p + 1::2] = float("inf")
            cache[1][s, :, p + 2::2] = float("nan")
    q = normal(g, 4, 4, 64, dtype=dtype)
    got = ops.cache_attention(q, *cache[:2], torch.tensor(at, device="cuda"), **scales_of(cache))
    clean = [torch.where((torch.arange(150, device="cuda")[None, :] <= torch.tensor(at, device="cuda")[:, None])[:, None, :, None], h, 0.0) for h in held]
    want, bound = attend_reference(q, clean, at, 0.125, dtype)
    ref.check(got, want, bound)


@pytest.mark.parametrize("mode", ["fp32", "mixed", "bf16", "int4"])
def test_non_finite_rows_reach_their_own_heads_only(mode):
    # a NaN in a seen row makes its head NaN, an infinite value likewise infinite or NaN; no other head or stream
    g = generator(8)
    dtype = TYPES.get(mode, torch.bfloat16)
    cache, held = filled_cache(g, 3, 2, 70, 64, 0, mode)
    if mode == "int4":
        cache[2][1, 0, 20] = float("nan")
        cache[3][2, 1, 69] = float("nan")
    else:
        cache[0][1, 0, 20, 5] = float("nan")
        cache[1][2, 1, 69, :] = float("nan")
    q = normal(g, 3, 4, 64, dtype=dtype)
    at = [69, 69, 69]
    got = ops.cache_attention(q, *cache[:2], torch.tensor(at, device="cuda"), **scales_of(cache))
    want, bound = attend_reference(q, held, at, 0.125, dtype)
    assert torch.isnan(got[1, :2]).all() and torch.isnan(got[2, 2:]).all()
    for s, h in ((0, slice(0, 4)), (1, slice(2, 4)), (2, slice(0, 2))):
        ref.check(got[s, h], want[s, h], bound[s, h])


@pytest.mark.parametrize("mode", ["fp32", "mixed", "bf16"])
def test_large_and_equal_logits(mode):
    # logits near the type's limits: the maximum is taken out first. Keys alternate between +-big, so about half
    # of the weights are equal and the rest vanish; the result is the mean of the values of the larger side.
    g = generator(9)
    dtype = TYPES[mode]
    big = 200.0
    keys = torch.full((1, 1, 101, 64), big, device="cuda", dtype=dtype)
    keys[:, :, 1::2] = -big
    values = normal(g, 1, 1, 101, 64, dtype=dtype)
    q = torch.full((1, 2, 64), big, device="cuda", dtype=dtype)
    q[:, 1] = -big
    got = ops.cache_attention(q, keys, values, torch.tensor([100], device="cuda"))
    want = torch.stack([values[0, 0, 0::2].double().mean(0), values[0, 0, 1::2].double().mean(0)])[None]
    size = torch.stack([values[0, 0, 0::2].double().abs().mean(0), values[0, 0, 1::2].double().abs().mean(0)])[None]
    ref.check(got, want, (2 * ref.unit(dtype) + 200 * ref.F) * size + ref.TINY[dtype])


@pytest.mark.parametrize("rows", ["mixed", "bf16"])
@pytest.mark.parametrize("q_size,k_size,v_size", [(1e4, 1e-4, 1.0), (1e-4, 1e3, 1e-9), (3.0, 1.0, 1e4), (2.0 ** -14, 1.0, 1.0), (0.0, 1.0, 1.0)])
def test_four_bit_attention_over_a_range_of_sizes(rows, q_size, k_size, v_size):
    # queries are scaled by a power of two and values' scales folded into the weights: neither may lose small or large ones
    g = generator(21)
    dtype = TYPES[rows]
    packed, scales, held = [], [], []
    for size in (k_size, v_size):
        codes, s, low = ref.quantise(normal(g, 2, 2, 90, 64) * size)
        packed.append(ref.pack(codes))
        scales.append(torch.stack([s, low], -1))
        held.append(ref.unpack(packed[-1], scales[-1]))
        held.append((15 * s.double() + low.double().abs()).repeat_interleave(32, -1))
    held = (held[0], held[2], held[1], held[3])
    q = (normal(g, 2, 4, 64) * q_size).to(dtype)
    q[:, :, :8] *= 2.0 ** -10                       # and columns far below the largest
    at = [89, 40]
    got = ops.cache_attention(q, *packed, torch.tensor(at, device="cuda"), key_scales=scales[0], value_scales=scales[1])
    want, bound = attend_reference(q, held, at, 0.125, dtype)
    ref.check(got, want, bound)


def test_cache_attention_in_place():
    g = generator(22)
    for mode, slots in (("bf16", 100), ("bf16", 5000), ("fp32", 100)):
        dtype = TYPES[mode]
        cache, _ = filled_cache(g, 2, 2, slots, 64, 0, mode)
        q = normal(g, 2, 8, 64, dtype=dtype)
        at = torch.tensor([slots - 1, 40], device="cuda")
        want = ops.cache_attention(q, *cache[:2], at)
        assert ops.cache_attention(q, *cache[:2], at, out=q) is q
        assert torch.equal(q, want)


def test_append_past_the_last_position_stays_in_bounds():
    guard = torch.zeros(3, 2, 8, 64, dtype=torch.bfloat16, device="cuda")
    keys, values = guard[1:2], torch.zeros_like(guard)[1:2]
    x = torch.ones(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([2 ** 63 - 2], device="cuda")
    ops.cache_append(x, x, x, keys, values, at, ops.rotation_frequencies(64), starts=starts_of([4]))
    assert not guard[0].any() and not guard[2].any()


def test_cache_attention_over_strided_and_broadcast_caches():
    g = generator(10)
    S, kv, slots, dim = 3, 2, 90, 64
    big = normal(g, kv, S, 2, slots, dim, dtype=torch.bfloat16)     # [head][stream][k or v][slot]
    keys, values = (big[:, :, i].transpose(0, 1) for i in range(2))
    wide = normal(g, S, 3, 6, dim, dtype=torch.bfloat16)
    q = wide[:, 1]
    out = torch.zeros(S, 2, 6, dim, dtype=torch.bfloat16, device="cuda")
    at = [89, 12, 200]
    positions = torch.tensor(at, device="cuda")
    ops.cache_attention(q, keys, values, positions, out=out[:, 1])
    want, bound = attend_reference(q, (keys.double(), values.double()), at, 0.125, torch.bfloat16)
    ref.check(out[:, 1], want, bound)
    assert not out[:, 0].any()
    one = (keys[:1].expand(S, -1, -1, -1), values[:1].expand(S, -1, -1, -1))      # one prompt, seen by every stream
    got = ops.cache_attention(q, *one, positions)
    want, bound = attend_reference(q, (one[0].double(), one[1].double()), at, 0.125, torch.bfloat16)
    ref.check(got, want, bound)


def test_offsets_past_32_bits():
    # the second head's rows start 2^31 elements (4 GiB) into each buffer
    g = generator(12)
    slots, dim, apart = 300, 64, 2 ** 25
    buffers = [torch.empty((apart + slots) * dim, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    keys, values = (b.as_strided((1, 2, slots, dim), ((apart + slots) * dim, apart * dim, dim, 1)) for b in buffers)
    positions = torch.tensor([slots - 1], device="cuda")
    rows = normal(g, slots, 2, dim, dtype=torch.bfloat16)
    f = ops.rotation_frequencies(dim)[:0]
    begin = torch.zeros(1, dtype=torch.int64, device="cuda")
    ops.cache_append(rows, rows, rows, keys, values, begin, f, starts=starts_of([slots]))
    assert torch.equal(keys[0].transpose(0, 1), rows) and torch.equal(values[0].transpose(0, 1), rows)
    q = normal(g, 1, 4, dim, dtype=torch.bfloat16)
    got = ops.cache_attention(q, keys, values, positions)
    want, bound = attend_reference(q, (keys.double(), values.double()), [slots - 1], 0.125, torch.bfloat16)
    ref.check(got, want, bound)


@pytest.mark.parametrize("mode", ["fp32", "mixed", "bf16"])
def test_attention_over_a_snapshot_of_the_runtime_matches_its_step(mode):
    # a snapshot's layer is a cache without sinks: the same q over it gives the attention that the step traced
    import numpy as np

    from policy import check_state
    from streaming_transformer_b200 import Backend, ModelConfig, Runtime, RuntimeOptions, synthetic

    c = ModelConfig(2, 256, 4, 128, 40, 32, 1e-5)
    events = synthetic.make_events(57, 32, seed=12)
    with Runtime(synthetic.make_model(c, mode, seed=11), RuntimeOptions(backend=Backend.CUDA, blocks=0)) as rt:
        for e in events[:56]:          # past one full ring revolution
            rt.step(e)
        trace, snap = rt.trace_step(events[56]), rt.snapshot()
    positions = torch.tensor([snap.position - 1], dtype=torch.int64, device="cuda")
    for layer in range(c.layers):
        keys, values = (torch.from_numpy(np.ascontiguousarray(x[layer])).to(TYPES[mode])[None].cuda() for x in (snap.keys, snap.values))
        q = torch.from_numpy(trace[f"layers.{layer}.q"]).to(TYPES[mode]).view(1, c.heads, c.head_dim).cuda()
        got = ops.cache_attention(q, keys, values, positions).float().cpu().numpy().reshape(1, 1, -1)
        check_state(got, trace[f"layers.{layer}.attention"][None, None, :], mode, f"layer {layer}")


# ---------------------------------------------------------------- attention of packed sequences

WINDOW = [
    # mode, heads, kv, dim, window, sinks, sizes (None: one sequence of 150 rows)
    ("fp32", 4, 4, 64, 64, 2, None),
    ("fp32", 6, 2, 40, 17, 0, [1, 0, 130, 33]),
    ("fp32", 2, 1, 256, 1000, 4, [70, 65]),
    ("fp32", 3, 3, 8, 1, 1, [40]),
    # rows and heads for each size of the fp32 tiles
    ("fp32", 8, 2, 64, 100, 3, [300, 77]),
    ("fp32", 16, 16, 24, 70, 2, [600]),
    ("fp32", 6, 3, 96, 50, 1, [300, 1]),
    ("fp32", 8, 1, 128, 90, 4, [500, 3]),
    ("fp32", 1, 1, 128, 40, 2, [90]),
    ("mixed", 4, 4, 64, 100, 4, [301]),
    ("mixed", 7, 1, 80, 60, 1, [129, 127, 128, 1, 1, 300]),
    ("mixed", 2, 2, 128, 5, 200, [400, 3]),
    ("mixed", 4, 1, 256, 33, 2, [150]),
    ("bf16", 16, 16, 64, 256, 4, [511, 257, 13]),
    ("bf16", 8, 2, 256, 300, 5, [700, 1, 129]),
    ("mixed", 6, 3, 136, 90, 70, [31, 400, 2]),
    ("bf16", 2, 1, 192, 2 ** 33, 0, [260]),
    ("bf16", 3, 3, 248, 1, 1, [128, 64]),
    ("bf16", 32, 8, 128, 500, 16, [1200]),
    ("bf16", 8, 2, 96, 1, 0, [140]),
    ("bf16", 8, 1, 128, 130, 3, [0, 0, 260, 0, 100, 0]),
    ("bf16", 3, 1, 32, 128, 130, [513]),
    ("bf16", 5, 5, 16, 31, 7, [100] * 9),
    ("bf16", 12, 4, 64, 2 ** 40, 0, [385, 1]),
    ("bf16", 4, 4, 64, 300, 61, list(range(1, 40))),
]


def window_reference(q, k, v, edges, window, sinks, scale, dtype):
    kv, group = k.shape[1], q.shape[1] // k.shape[1]
    for a, b in itertools.pairwise(edges):
        if a == b:
            continue
        i = torch.arange(b - a, device="cuda")
        see = (i[None] <= i[:, None]) & ((i[:, None] - i[None] < window) | (i[None] < sinks))
        qs = q[a:b].double().transpose(0, 1)
        ks, vs = (x[a:b].double().transpose(0, 1).repeat_interleave(group, 0) for x in (k, v))
        o, bound = ref.attention(qs, ks, vs, see[None], scale, dtype)
        yield a, b, o.transpose(0, 1), bound.transpose(0, 1)


@pytest.mark.parametrize("case", WINDOW, ids=lambda c: "-".join(map(str, c[:6])))
def test_window_attention_matches_the_definition(case):
    mode, heads, kv, dim, window, sinks, sizes = case
    g = generator(13)
    dtype = TYPES[mode]
    before = 5 if sizes else 0
    n = before + sum(sizes) + 3 if sizes else 150
    q, k, v = (normal(g, n, h, dim, dtype=dtype) for h in (heads, kv, kv))
    if sizes:   # rows of no sequence hold anything
        for x in (q, k, v):
            x[:before] = float("nan")
            x[n - 3:] = float("inf")
    starts = starts_of(sizes, before) if sizes else None
    edges = starts.tolist() if sizes else [0, n]
    for scale in (None, 0.3, -0.2, 0.0):
        out = torch.full((n, heads, dim), 7.0, dtype=dtype, device="cuda")
        ops.window_attention(q, k, v, window=window, sinks=sinks, starts=starts, scale=scale, out=out)
        assert (out[:edges[0]] == 7).all() and (out[edges[-1]:] == 7).all(), "rows of no sequence"
        for a, b, want, bound in window_reference(q, k, v, edges, window, sinks, dim ** -0.5 if scale is None else scale, dtype):
            ref.check(out[a:b], want, bound, f"rows {a}..{b}")


@pytest.mark.parametrize("mode,heads,dim", [("fp32", 2, 64), ("fp32", 6, 64), ("fp32", 20, 64), ("mixed", 2, 64), ("bf16", 2, 64),
                                            ("bf16", 4, 64), ("bf16", 4, 128), ("mixed", 2, 192)])
@pytest.mark.parametrize("where", [140, 200, 259])
def test_non_finite_rows_reach_those_that_see_them_only(mode, heads, dim, where):
    g = generator(14)
    dtype = TYPES[mode]
    n, window = 420, 70
    sizes = [260, 160]
    q, k, v = (normal(g, n, h, dim, dtype=dtype) for h in (heads, 2, 2))
    v[where, 0] = float("nan")
    k[where, 1] = float("nan")
    out = ops.window_attention(q, k, v, window=window, sinks=1, starts=starts_of(sizes))
    hit = torch.zeros(n, dtype=torch.bool, device="cuda")
    hit[where:min(where + window, 260)] = True
    assert torch.isnan(out[hit]).all()
    clean = [torch.where(torch.isnan(x), 0.0, x.float()).to(dtype) for x in (k, v)]
    for a, b, want, bound in window_reference(q, *clean, [0, 260, 420], window, 1, dim ** -0.5, dtype):
        keep = ~hit[a:b]
        ref.check(out[a:b][keep], want[keep], bound[keep], f"rows {a}..{b}")


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
def test_window_attention_of_strided_rows(mode):
    g = generator(15)
    dtype = TYPES[mode]
    n, heads, dim = 200, 4, 64
    qkv = normal(g, n, 3, heads, dim, dtype=dtype)
    out = torch.zeros(heads, n, dim, dtype=dtype, device="cuda")
    q, k, v = (qkv[:, i] for i in range(3))
    shared = k[:, :1].expand(-1, heads, -1)          # one key head broadcast to all
    ops.window_attention(q, shared, v, window=50, sinks=3, out=out.transpose(0, 1))
    for a, b, want, bound in window_reference(q, shared, v, [0, n], 50, 3, 0.125, dtype):
        ref.check(out.transpose(0, 1)[a:b], want, bound)


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
def test_window_attention_of_one_repeated_key_row(mode):
    # a row stride of 0: every position has the same key and value, so every row is that value, to one rounding of it
    # and the weights' (u(T) each) and sums'
    g = generator(23)
    dtype = TYPES[mode]
    k, v = (normal(g, 1, 2, 64, dtype=dtype).expand(300, -1, -1) for _ in range(2))
    got = ops.window_attention(normal(g, 300, 2, 64, dtype=dtype), k, v, window=100, sinks=2)
    ref.check(got, v.double(), v.double().abs() * (2 * ref.unit(dtype) + 300 * ref.F) + ref.TINY[dtype])


@pytest.mark.parametrize("mode", ["fp32", "mixed", "bf16"])
def test_many_short_and_skipped_key_tiles(mode):
    # long gaps between a tile's sinks and its window: key tiles that one of a CTA's two query tiles needs and the
    # other does not, for an odd and an even number of heads a key head
    g = generator(24)
    dtype = TYPES[mode]
    for heads, kv, dim in ((3, 3, 64), (4, 2, 64), (3, 1, 128), (4, 1, 128)):
        sizes = [700, 1, 390, 133]
        n = sum(sizes)
        q, k, v = (normal(g, n, h, dim, dtype=dtype) for h in (heads, kv, kv))
        for window, sinks in ((20, 150), (3, 1), (129, 70)):
            got = ops.window_attention(q, k, v, window=window, sinks=sinks, starts=starts_of(sizes))
            for a, b, want, bound in window_reference(q, k, v, starts_of(sizes).tolist(), window, sinks, dim ** -0.5, dtype):
                ref.check(got[a:b], want, bound, f"{heads} heads, window {window}, rows {a}..{b}")


def test_a_captured_backlog_replays_with_other_starts():
    g = generator(25)
    n, window, sinks = 400, 90, 3
    q, k, v = (normal(g, n, h, 64, dtype=torch.bfloat16) for h in (4, 2, 2))
    starts = starts_of([100, 300, 0])
    ops.window_attention(q, k, v, window=window, sinks=sinks, starts=starts)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        out = ops.window_attention(q, k, v, window=window, sinks=sinks, starts=starts)
    torch.cuda.current_stream().wait_stream(side)
    for sizes in ([300, 40, 60], [1, 1, 398]):
        starts.copy_(starts_of(sizes))
        q.copy_(normal(g, *q.shape))
        graph.replay()
        assert torch.equal(out, ops.window_attention(q, k, v, window=window, sinks=sinks, starts=starts))
        for a, b, want, bound in window_reference(q, k, v, starts.tolist(), window, sinks, 0.125, torch.bfloat16):
            ref.check(out[a:b], want, bound)


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("mode", ["fp32", "mixed", "bf16"])
def test_a_backlog_then_single_events_match_one_long_sequence(mode):
    # three streams: a backlog each (one empty), then single events; every event's attention is the row of the
    # whole history's window attention, to the bounds of both
    g = generator(16)
    dtype = TYPES[mode]
    heads, kv, dim, window, sinks, more = 4, 2, 64, 24, 3, 30
    sizes = [60, 0, 10]
    total = [s + more for s in sizes]
    hist = [[normal(g, n, h, dim, dtype=dtype) for h in (heads, kv, kv)] for n in total]
    gains = [0.5 + torch.rand(dim, generator=g, device="cuda") for _ in range(2)]
    f = ops.rotation_frequencies(dim)
    cache = ops.new_cache(3, kv, window, dim, sinks=sinks, mode=mode)
    kw = dict(sinks=sinks, q_gain=gains[0], k_gain=gains[1])
    zero = torch.zeros(3, dtype=torch.int64, device="cuda")
    packed = [torch.cat([hist[s][i][:sizes[s]] for s in range(3)]) for i in range(3)]
    starts = starts_of(sizes)
    q, k = ops.cache_append(*packed, *cache[:2], zero, f, starts=starts, rotated_keys=True, **kw)
    first = ops.window_attention(q, k, packed[2], window=window, sinks=sinks, starts=starts)
    got = [[first[a:b]] for a, b in itertools.pairwise(starts.tolist())]
    positions = torch.tensor(sizes, device="cuda")
    for t in range(more):
        one = [torch.stack([hist[s][i][sizes[s] + t] for s in range(3)]) for i in range(3)]
        q = ops.cache_append(*one, *cache[:2], positions, f, **kw)
        out = ops.cache_attention(q, *cache[:2], positions)
        for s in range(3):
            got[s].append(out[s:s + 1])
        positions += 1
    for s in range(3):
        at = torch.arange(total[s], device="cuda")
        q, _ = ref.rotated(hist[s][0], at, f, gains[0], 1e-6, dtype)
        k, _ = ref.rotated(hist[s][1], at, f, gains[1], 1e-6, dtype)
        # the operators see q and k rounded to the type: a logit moves by at most 2 u(T) sum|q k| scale, and a
        # weight by twice that, relative
        for a, b, want, bound in window_reference(q, k, hist[s][2], [0, total[s]], window, sinks, dim ** -0.5, dtype):
            products = (q.abs().sum(-1).amax() * k.abs().amax()).item() * dim ** -0.5
            extra = 2 * 2 * 2 * (ref.unit(dtype) + 24 * ref.F) * products * hist[s][2].double().abs().amax()
            ref.check(torch.cat(got[s]), want, bound + extra, f"stream {s}")


def test_a_captured_step_replays_with_new_positions_and_on_another_stream():
    g = generator(17)
    S, heads, kv, dim, window, sinks = 4, 8, 2, 128, 3000, 2
    f = ops.rotation_frequencies(dim)
    caches = [ops.new_cache(S, kv, window, dim, sinks=sinks, mode="bf16") for _ in range(2)]
    noise = normal(g, S, kv, window + sinks, dim, dtype=torch.bfloat16)
    for c in caches:
        c[0].copy_(noise)
        c[1].copy_(noise)
    q, k, v = (normal(g, S, h, dim, dtype=torch.bfloat16) for h in (heads, kv, kv))
    positions = torch.tensor([0, 2999, 5, 100000], device="cuda")

    def step(c):
        turned = ops.cache_append(q, k, v, *c[:2], positions, f, sinks=sinks)
        return ops.cache_attention(turned, *c[:2], positions)

    step(caches[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for _ in range(2):      # two graphs of one step: each has its own intermediate memory
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(step(caches[0]))
            graphs.append(graph)
    torch.cuda.current_stream().wait_stream(side)
    for move in (1, 700):
        positions += move
        q.copy_(normal(g, *q.shape))
        graphs[0].replay()
        graphs[1].replay()
        caches[1][0].copy_(caches[0][0])
        caches[1][1].copy_(caches[0][1])
        want = step(caches[1])
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
        assert torch.equal(caches[0][0], caches[1][0])


@pytest.mark.parametrize("mode", ["fp32", "bf16", "int4"])
def test_calls_on_two_streams_at_once_and_repeated_calls_agree_bit_for_bit(mode):
    g = generator(18)
    dtype = TYPES.get(mode, torch.bfloat16)
    cache, _ = filled_cache(g, 2, 2, 9000, 128, 0, mode)
    positions = torch.tensor([8999, 4000], device="cuda")
    q = normal(g, 2, 8, 128, dtype=dtype)
    want = ops.cache_attention(q, *cache[:2], positions, **scales_of(cache))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(8):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ops.cache_attention(q, *cache[:2], positions, **scales_of(cache)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_refusals_of_the_binding():
    keys, values, _, _ = ops.new_cache(2, 2, 8, 64, mode="bf16")
    four = ops.new_cache(2, 2, 8, 64, mode="int4")
    at = torch.zeros(2, dtype=torch.int64, device="cuda")
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    kv = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    f = ops.rotation_frequencies(64)

    def refused(match, call):
        with pytest.raises(StreamError, match=match) as e:
            call()
        assert e.value.status == "INVALID"

    refused("cache's type", lambda: ops.cache_attention(q.float(), keys, values, at))
    refused("cache's type", lambda: ops.cache_attention(q.float(), *four[:2], at, **scales_of(four)))
    refused("has scales", lambda: ops.cache_attention(q, *four[:2], at))
    refused("has scales", lambda: ops.cache_attention(q, keys, values, at, **scales_of(four)))
    refused("multiple of the cache", lambda: ops.cache_attention(q[:, :3], keys, values, at))
    refused("expected shape", lambda: ops.cache_attention(q[:1], keys, values, at))
    refused("int64", lambda: ops.cache_attention(q, keys, values, at.int()))
    refused("2 contiguous", lambda: ops.cache_attention(q, keys, values, at[:1]))
    refused("columns must be contiguous", lambda: ops.cache_attention(q.transpose(1, 2).contiguous().transpose(1, 2), keys, values, at))
    refused("keys' shape", lambda: ops.cache_attention(q, keys, values[:, :, :4], at))
    refused("16-byte", lambda: ops.cache_attention(torch.zeros(2 * 4 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, 4, 64), keys, values, at))
    refused("backward", lambda: ops.cache_attention(q.clone().requires_grad_(), keys, values, at))
    refused("window >= 1", lambda: ops.cache_append(q, kv, kv, keys, values, at, f, sinks=8))
    refused("sinks", lambda: ops.cache_append(q, kv, kv, keys, values, at, f, sinks=-1))
    refused("overlap", lambda: ops.cache_append(q, kv, kv, keys[:1].expand(2, -1, -1, -1), values[:1].expand(2, -1, -1, -1), at, f))
    refused("rows overlap", lambda: ops.cache_append(q, kv, kv, keys, values, at, f, out=q[:1].expand(2, -1, -1)))
    refused("one row for each stream", lambda: ops.cache_append(q[:1], kv[:1], kv[:1], keys, values, at, f))
    refused("rotary", lambda: ops.cache_append(q, kv, kv, keys, values, at, ops.rotation_frequencies(128)))
    refused("epsilon", lambda: ops.cache_append(q, kv, kv, keys, values, at, f, epsilon=-1.0))
    refused("3 contiguous", lambda: ops.cache_append(q, kv, kv, keys, values, at, f, starts=torch.zeros(4, dtype=torch.int32, device="cuda")))
    refused("window is at least 1", lambda: ops.window_attention(q, kv, kv, window=0))
    refused("multiple of the key heads", lambda: ops.window_attention(q[:, :3], kv, kv, window=4))
    refused("multiple of 8", lambda: ops.window_attention(q[..., :12].contiguous(), kv[..., :12].contiguous(), kv[..., :12].contiguous(), window=4))
    refused("no row type", lambda: ops.window_attention(q.double(), kv.double(), kv.double(), window=4))
    with torch.no_grad():
        ops.cache_attention(q.clone().requires_grad_(), keys, values, at)


def test_empty_calls():
    keys, values, _, _ = ops.new_cache(2, 2, 8, 64, mode="bf16")
    none = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    at = torch.zeros(2, dtype=torch.int64, device="cuda")
    f = ops.rotation_frequencies(64)
    starts = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert ops.cache_append(none, none, none, keys, values, at, f, starts=starts).shape == (0, 2, 64)
    assert ops.window_attention(none, none, none, window=3).shape == (0, 2, 64)
    one = torch.ones(1, 2, 64, dtype=torch.bfloat16, device="cuda")
    out = torch.full_like(one, 5)
    ops.window_attention(one, one, one, window=3, starts=starts, out=out)        # a row of no sequence
    assert (out == 5).all()
    ops.cache_append(one, one, one, keys, values, at, f, starts=starts, out=out)
    assert (out == 5).all() and not keys.any()


def test_writes_are_seen_by_gradients():
    """A cache that takes part in a gradient is refused, and a tensor that a backward pass saved counts its writes."""
    keys, values, _, _ = ops.new_cache(2, 2, 8, 64, mode="fp32")
    at = torch.zeros(2, dtype=torch.int64, device="cuda")
    q, kv = torch.ones(2, 2, 64, device="cuda"), torch.ones(2, 2, 64, device="cuda")
    f = ops.rotation_frequencies(64)
    for side in (keys, values):
        side.requires_grad_()
        with pytest.raises(StreamError, match="backward"):
            ops.cache_append(q, kv, kv, keys, values, at, f)
        side.requires_grad_(False)
    with pytest.raises(StreamError, match="rotated_keys"):
        ops.cache_append(q, kv, kv, keys, values, at, f, rotated_keys=kv)
    w = torch.ones(2, 2, 8, 64, device="cuda", requires_grad=True)
    loss = (w * keys).sum()
    ops.cache_append(q, kv, kv, keys, values, at, f)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    for call in (lambda out: ops.cache_append(q, kv, kv, keys, values, at, f, out=out),
                 lambda out: ops.cache_attention(q, keys, values, at, out=out),
                 lambda out: ops.window_attention(q, kv, kv, window=3, out=out)):
        out = torch.empty_like(q)
        before = out._version
        call(out)
        assert out._version == before + 1
    with torch.inference_mode():
        ops.cache_attention(q, keys, values, at, out=torch.empty_like(q))


def test_columns_past_the_rotation_pass():
    """Whatever they hold: a lane that has the last rotated pair does not touch the pair beside it."""
    g = generator(41)
    f = ops.rotation_frequencies(40)
    for pairs in (0, 1, 3, 4, 13, 20):
        q, k, v = (normal(g, 2, 2, 40, dtype=torch.float32) for _ in range(3))
        for x in (q, k):
            x[:, 0, 2 * pairs:] = float("inf")
            x[:, 1, 2 * pairs + 1::2] = float("-inf")
        keys, values, _, _ = ops.new_cache(2, 2, 4, 40, mode="fp32")
        at = torch.tensor([5, 2], device="cuda")
        out = ops.cache_append(q, k, v, keys, values, at, f[:pairs])
        held = torch.stack([keys[0, :, 1], keys[1, :, 2]])
        for x, y in ((q, out), (k, held)):
            assert torch.equal(x[..., 2 * pairs:], y[..., 2 * pairs:])
            assert torch.isfinite(y[..., :2 * pairs]).all()


@pytest.mark.parametrize("mode", ["fp32", "mixed", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 2, 6, 7, 8])
def test_window_attention_of_a_few_rows(mode, dim, n):
    g = generator(43)
    dtype = TYPES[mode]
    q, k, v = (normal(g, n, h, dim, dtype=dtype) for h in (4, 2, 2))
    for sizes in (None, [n - 1, 0, 1]):
        starts, edges = (starts_of(sizes), starts_of(sizes).tolist()) if sizes else (None, [0, n])
        for window, sinks in ((1, 0), (3, 1), (100, 4)):
            out = ops.window_attention(q, k, v, window=window, sinks=sinks, starts=starts)
            for a, b, want, bound in window_reference(q, k, v, edges, window, sinks, dim ** -0.5, dtype):
                ref.check(out[a:b], want, bound, f"window {window}, rows {a}..{b}")
