"""What the cache and attention operators of streaming_transformer_b200.attention are measured on.

Three operators, for one layer of many streams:

* ``cache_append``: per-head RMS norm of the queries and keys, the position rotation of adjacent pairs in the same
  pass, and the insert of the keys and values into every stream's window cache. A cache has ``sinks`` slots that the
  first positions keep for good and a ring of ``window`` slots; it holds fp32, fp16, bf16 or 4-bit rows.
* ``cache_attention``: one query row per stream over the slots its cache holds (16-bit, fp32 or 4-bit rows).
* ``window_attention``: whole sequences, packed one after another, each row over the last ``window`` positions of its
  own sequence and that sequence's first ``sinks`` positions.

4-bit rows: every 32 values of a row share a bf16 scale and a bf16 lowest value, and a value stands for
``lowest + scale * code`` with a code of 0..15, two codes a byte, the even column in the low bits.

``run`` computes them with elementary torch operations where ``own`` is false and through the framework where it is true.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "mixed": torch.float16, "bf16": torch.bfloat16, "int4": torch.bfloat16}
EPSILON = 1e-6
GROUP = 32  # columns that share a scale in a 4-bit row


def listed():
    return [
        # One event of one stream at the Main shape: the step's own insert, where only latency counts.
        dict(name="append-one-main-fp32", op="append", type="fp32", streams=1, tokens=1, heads=8, kv_heads=8, head_dim=64, window=128, sinks=4),
        # One event of each of 256 Large streams.
        dict(name="append-256-large-bf16", op="append", type="bf16", streams=256, tokens=256, heads=16, kv_heads=16, head_dim=64, window=256, sinks=4),
        # A backlog of 16384 events of eight streams with shared key heads, quantised into 4-bit caches and read back.
        dict(name="append-backlog-int4", op="append", type="int4", streams=8, tokens=16384, heads=32, kv_heads=8, head_dim=128, window=512, sinks=4),
        # One event of one stream at the Main shape.
        dict(name="attend-one-main-fp32", op="attend", type="fp32", streams=1, heads=8, kv_heads=8, head_dim=64, window=128, sinks=4, ragged=False),
        # 256 Large streams, full windows.
        dict(name="attend-256-large-bf16", op="attend", type="bf16", streams=256, heads=16, kv_heads=16, head_dim=64, window=256, sinks=4, ragged=False),
        # Streams that joined at different times, some of them idle, with shared key heads.
        dict(name="attend-ragged-fp16", op="attend", type="mixed", streams=37, heads=32, kv_heads=8, head_dim=128, window=4096, sinks=4, ragged=True),
        # One stream with a long memory: the work has to be split over the slots.
        dict(name="attend-one-long-bf16", op="attend", type="bf16", streams=1, heads=32, kv_heads=8, head_dim=128, window=131072, sinks=4, ragged=False),
        # The same 256 streams on 4-bit caches of twice the window.
        dict(name="attend-256-large-int4", op="attend", type="int4", streams=256, heads=16, kv_heads=16, head_dim=64, window=512, sinks=4, ragged=False),
        # Long ragged 4-bit caches with shared key heads.
        dict(name="attend-ragged-int4", op="attend", type="int4", streams=9, heads=32, kv_heads=8, head_dim=128, window=65536, sinks=16, ragged=True),
        # A short odd history at the Small shape.
        dict(name="window-short-fp32", op="window", type="fp32", sequences=1, tokens=201, heads=4, kv_heads=4, head_dim=64, window=64, sinks=2),
        # The backlogs of 16 Large streams, of uneven lengths, in one call.
        dict(name="window-ragged-bf16", op="window", type="bf16", sequences=16, tokens=8109, heads=16, kv_heads=16, head_dim=64, window=256, sinks=4),
        # One long history with shared key heads and a wide window.
        dict(name="window-long-bf16", op="window", type="bf16", sequences=1, tokens=8192, heads=32, kv_heads=8, head_dim=128, window=4096, sinks=16),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "window"])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    heads = kv_heads * rng.choice([g for g in (1, 2, 3, 4, 7, 8, 16) if g * kv_heads <= 32])
    if op == "window":
        kind = rng.choice(["fp32", "mixed", "bf16", "bf16"])
        dim = rng.choice([32, 64, 80, 96, 128])
        case = dict(op=op, type=kind, sequences=_log(rng, 1, 24), tokens=_log(rng, 24, 6000 if kind != "fp32" else 2500), heads=heads, kv_heads=kv_heads,
                    head_dim=dim, window=_log(rng, 1, 6000), sinks=rng.choice([0, 1, 4, 16, 61]))
        while work(case)["flops"] > 2e11:
            case["window"] = max(1, case["window"] // 2)
        return case
    kind = rng.choice(["fp32", "mixed", "bf16", "int4", "int4"])
    dim = rng.choice([64, 96, 128] if kind == "int4" else [32, 64, 80, 96, 128])
    if op == "append":
        streams = _log(rng, 1, 256)
        case = dict(op=op, type=kind, streams=streams, tokens=streams if rng.random() < 0.5 else _log(rng, streams, 12000), heads=heads, kv_heads=kv_heads,
                    head_dim=dim, window=_log(rng, 1, 1500), sinks=rng.choice([0, 1, 4, 13]))
        while work(case)["bytes"] > 2e8 or _cache_bytes(case) > 1e9:
            case["window"] = max(1, case["window"] // 2)
            case["tokens"] = max(streams, case["tokens"] * 3 // 4)
        return case
    case = dict(op=op, type=kind, streams=_log(rng, 1, 256), heads=heads, kv_heads=kv_heads, head_dim=dim, window=_log(rng, 1, 100000), sinks=rng.choice([0, 1, 4, 13]),
                ragged=rng.random() < 0.5)
    while _cache_bytes(case) > 4.5e8:
        case["window"] = max(1, case["window"] * 2 // 3)
    return case


# ---- sizes that follow from a case

def _cut(total, parts):
    """`total` tokens in `parts` uneven sequences, none empty."""
    parts = min(parts, total)
    weight = [1 + (7 * i) % 11 for i in range(parts)]
    sizes = [1 + (total - parts) * w // sum(weight) for w in weight]
    sizes[-1] += total - sum(sizes)
    return sizes


def _visible(case):
    """How many slots each stream sees: all of them, or a spread from none to all."""
    slots, streams = case["sinks"] + case["window"], case["streams"]
    if not case["ragged"]:
        return [slots] * streams
    return [slots if streams == 1 else slots * i // (streams - 1) for i in range(streams)]


def _row_bytes(kind, dim):
    return dim // 2 + dim // GROUP * 4 if kind == "int4" else dim * DTYPES[kind].itemsize


def _cache_bytes(case):
    return 2 * case["streams"] * case["kv_heads"] * (case["sinks"] + case["window"]) * _row_bytes(case["type"], case["head_dim"])


def _pairs(case):
    """(query, key) pairs that see each other."""
    w, n = case["window"], 0
    for size in _cut(case["tokens"], case["sequences"]):
        full = min(size, w)
        n += full * (full + 1) // 2 + (size - full) * w
        late = size - full  # rows whose window no longer reaches the start: they see 1, 2, ... sinks more
        some = min(late, case["sinks"])
        n += some * (some + 1) // 2 + (late - some) * case["sinks"]
    return n


def work(case):
    elem, dim = DTYPES[case["type"]].itemsize, case["head_dim"]
    if case["op"] == "append":
        n, heads, kv = case["tokens"], case["heads"], case["kv_heads"]
        stay = sum(min(size, case["sinks"] + case["window"]) for size in _cut(n, case["streams"]))
        moved = n * (2 * heads + 2 * kv) * dim * elem + 2 * stay * kv * _row_bytes(case["type"], dim)
        if case["type"] == "int4":  # the caches are read and handed out as the values they stand for
            slots = case["streams"] * (case["sinks"] + case["window"])
            moved += _cache_bytes(case) + 2 * slots * kv * dim * elem
        return {"bytes": moved, "flops": n * (heads + kv) * dim * 7}
    if case["op"] == "attend":
        seen = sum(_visible(case))
        rows = 2 * case["streams"] * case["heads"] * dim * elem
        return {"bytes": 2 * seen * case["kv_heads"] * _row_bytes(case["type"], dim) + rows, "flops": 4 * seen * case["heads"] * dim}
    n = case["tokens"]
    return {"bytes": 2 * n * (case["heads"] + case["kv_heads"]) * dim * elem, "flops": 4 * _pairs(case) * case["heads"] * dim}


# ---- inputs

def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dtype, dim, heads, kv = DTYPES[case["type"]], case["head_dim"], case["heads"], case["kv_heads"]

    def normal(*shape, dtype=dtype):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    def even(*shape):
        return (torch.rand(shape, generator=g, device="cuda") * 4 - 2).to(dtype)

    s = dict(case)
    if case["op"] == "window":
        sizes = torch.tensor(_cut(case["tokens"], case["sequences"]))
        sizes = sizes[torch.randperm(len(sizes), generator=torch.Generator().manual_seed(seed))]
        s["starts"] = torch.cat([torch.zeros(1, dtype=torch.long), sizes.cumsum(0)]).to(torch.int32).cuda()
        s.update(q=normal(case["tokens"], heads, dim), k=normal(case["tokens"], kv, dim), v=normal(case["tokens"], kv, dim))
        return s
    streams, slots = case["streams"], case["sinks"] + case["window"]
    rows = (streams, kv, slots, dim)
    s["key_scales"] = s["value_scales"] = None
    if case["type"] == "int4":
        for name in ("key", "value"):
            s[name + "s"], s[name + "_scales"] = _pack(normal(*rows, dtype=torch.float32))
    else:
        s.update(keys=normal(*rows), values=normal(*rows))
    if case["op"] == "attend":
        seen = torch.tensor(_visible(case), dtype=torch.long)
        seen = seen[torch.randperm(streams, generator=torch.Generator().manual_seed(seed))].cuda()
        # A stream that sees all slots is anywhere past the fill; one that sees n is at position n - 1, and -1 is idle.
        later = torch.randint(0, 100000, (streams,), generator=g, device="cuda")
        s["positions"] = seen - 1 + torch.where(seen == slots, later, 0)
        s["q"] = normal(streams, heads, dim)
        return s
    n = case["tokens"]
    s["starts"] = None
    if n != streams:
        sizes = torch.tensor(_cut(n, streams))
        sizes = sizes[torch.randperm(streams, generator=torch.Generator().manual_seed(seed))]
        s["starts"] = torch.cat([torch.zeros(1, dtype=torch.long), sizes.cumsum(0)]).to(torch.int32).cuda()
    s["positions"] = torch.randint(0, 1 << 20, (streams,), generator=g, device="cuda")
    s["positions"][: streams // 3] %= 2 * slots  # some streams are young
    s["frequencies"] = 10000.0 ** (torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / -dim)
    for name in ("q_gain", "k_gain"):
        s[name] = 0.9 + 0.2 * torch.rand(dim, generator=g, device="cuda")
    s.update(q=even(n, heads, dim), k=even(n, kv, dim), v=even(n, kv, dim))
    return s


# ---- one pass

def run(s):
    if own:
        from streaming_transformer_b200 import attention as ops
        scales = {k: s[k] for k in ("key_scales", "value_scales") if k in s}
        if s["op"] == "append":
            q = ops.cache_append(s["q"], s["k"], s["v"], s["keys"], s["values"], s["positions"], s["frequencies"], sinks=s["sinks"], starts=s["starts"],
                                 q_gain=s["q_gain"], k_gain=s["k_gain"], epsilon=EPSILON, **scales)
            if s["type"] == "int4":
                keys, values = ops.unpack_cache(s["keys"], s["values"], dtype=s["q"].dtype, **scales)
                return {"q": q, "keys": keys, "values": values}
            return {"q": q, "keys": s["keys"], "values": s["values"]}
        if s["op"] == "attend":
            return ops.cache_attention(s["q"], s["keys"], s["values"], s["positions"], **scales)
        return ops.window_attention(s["q"], s["k"], s["v"], window=s["window"], sinks=s["sinks"], starts=s["starts"])
    return {"append": _append, "attend": _attend, "window": _window}[s["op"]](s)


# ---- the plain forms

def _pack(x):
    x = x.unflatten(-1, (-1, GROUP))
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale, low = ((high - low) * (1 / 15)).bfloat16(), low.bfloat16()
    step = scale.float()
    code = torch.where(step > 0, ((x - low.float()) / step).round().clamp(0, 15), torch.zeros_like(x)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, torch.cat([scale, low], -1)


def _unpack(codes, scales):
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, GROUP)).float()
    return (code * scales[..., :1].float() + scales[..., 1:].float()).flatten(-2)


def _tokens(s, n):
    """Each packed row's stream and its place in that stream's rows."""
    row = torch.arange(n, device="cuda")
    if s["starts"] is None:
        return row, torch.zeros_like(row)
    owner = torch.bucketize(row, s["starts"][1:].long(), right=True)
    return owner, row - s["starts"][owner]


def _append(s):
    n, sinks, window = s["tokens"], s["sinks"], s["window"]
    stream, place = _tokens(s, n)
    position = s["positions"][stream] + place
    count = torch.ones_like(s["positions"]) if s["starts"] is None else (s["starts"][1:] - s["starts"][:-1]).long()
    angle = position[:, None, None] * s["frequencies"]
    cos, sin = angle.cos().float(), angle.sin().float()

    def turn(x, gain):
        x = x.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPSILON) * gain
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)

    q, k, v = turn(s["q"], s["q_gain"]), turn(s["k"], s["k_gain"]), s["v"].float()
    last = s["positions"] + count - 1
    stay = (position < sinks) | (position > last[stream] - window)
    slot = torch.where(position < sinks, position, sinks + (position - sinks) % window)[stay]
    stream = stream[stay]
    if s["type"] != "int4":
        s["keys"][stream, :, slot] = k[stay].to(s["keys"].dtype)
        s["values"][stream, :, slot] = v[stay].to(s["keys"].dtype)
        return {"q": q.to(s["q"].dtype), "keys": s["keys"], "values": s["values"]}
    for name, x in (("key", k), ("value", v)):
        s[name + "s"][stream, :, slot], s[name + "_scales"][stream, :, slot] = _pack(x[stay])
    return {"q": q.to(s["q"].dtype), "keys": _unpack(s["keys"], s["key_scales"]).to(s["q"].dtype),
            "values": _unpack(s["values"], s["value_scales"]).to(s["q"].dtype)}


def _attend(s):
    keys, values = s["keys"], s["values"]
    if s["type"] == "int4":
        keys, values = _unpack(keys, s["key_scales"]), _unpack(values, s["value_scales"])
    keys, values = keys.float(), values.float()
    q = s["q"].float().unflatten(1, (s["kv_heads"], -1))
    seen = (torch.arange(keys.shape[2], device="cuda") <= s["positions"][:, None])[:, None, None]
    score = ((q @ keys.transpose(2, 3)) * s["head_dim"] ** -0.5).masked_fill(~seen, -math.inf)
    p = (score - score.amax(-1, keepdim=True).clamp_min(-1e30)).exp()
    total = p.sum(-1, keepdim=True)
    return ((p @ values) / torch.where(total > 0, total, 1)).flatten(1, 2).to(s["q"].dtype)


def _window(s):
    n, kv = s["tokens"], s["kv_heads"]
    sequence, place = _tokens(s, n)
    see = (sequence[:, None] == sequence) & (place <= place[:, None]) & ((place > place[:, None] - s["window"]) | (place < s["sinks"]))
    q = s["q"].float().unflatten(1, (kv, -1)).permute(1, 2, 0, 3)
    k, v = (s[x].float().permute(1, 0, 2)[:, None] for x in ("k", "v"))
    score = (q @ k.transpose(2, 3)).mul_(s["head_dim"] ** -0.5).masked_fill_(~see, -math.inf)
    p = score.sub_(score.amax(-1, keepdim=True)).exp_()
    return ((p @ v) / p.sum(-1, keepdim=True)).permute(2, 0, 1, 3).flatten(1, 2).to(s["q"].dtype)


# ---- the definitions in 64 bits, stream by stream

def _quantised(x):
    """What rows of 64-bit values stand for once they are held in 4 bits."""
    out = torch.empty_like(x)
    for c in range(0, x.shape[-1], GROUP):
        part = x[..., c:c + GROUP]
        low = part.min(-1, keepdim=True).values
        step = ((part.max(-1, keepdim=True).values - low) / 15).to(torch.bfloat16).double()
        low = low.to(torch.bfloat16).double()
        code = torch.clamp(torch.round((part - low) / torch.where(step > 0, step, torch.ones_like(step))), 0, 15)
        out[..., c:c + GROUP] = low + step * code
    return out


def _held(codes, scales):
    """The 64-bit values that 4-bit rows stand for."""
    out = torch.empty(*codes.shape[:-1], codes.shape[-1] * 2, dtype=torch.float64, device=codes.device)
    out[..., 0::2] = torch.remainder(codes, 16).double()
    out[..., 1::2] = torch.div(codes, 16, rounding_mode="floor").double()
    for c in range(scales.shape[-2]):
        out[..., c * GROUP:(c + 1) * GROUP] *= scales[..., c, 0:1].double()
        out[..., c * GROUP:(c + 1) * GROUP] += scales[..., c, 1:2].double()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    dim, kv, group = case["head_dim"], case["kv_heads"], case["heads"] // case["kv_heads"]
    if case["op"] == "attend":
        out = torch.zeros(case["streams"], case["heads"], dim, dtype=torch.float64, device="cuda")
        for i, at in enumerate(s["positions"].tolist()):
            n = min(at + 1, case["sinks"] + case["window"])
            if n <= 0:
                continue
            if case["type"] == "int4":
                keys, values = (_held(s[x + "s"][i, :, :n], s[x + "_scales"][i, :, :n]) for x in ("key", "value"))
            else:
                keys, values = s["keys"][i, :, :n].double(), s["values"][i, :, :n].double()
            for h in range(case["heads"]):
                p = torch.softmax(keys[h // group] @ s["q"][i, h].double() / math.sqrt(dim), 0)
                out[i, h] = p @ values[h // group]
        return out
    if case["op"] == "window":
        out = torch.empty(case["tokens"], case["heads"], dim, dtype=torch.float64, device="cuda")
        edges = s["starts"].tolist()
        for a, b in zip(edges[:-1], edges[1:]):
            i, j = torch.arange(b - a, device="cuda")[:, None], torch.arange(b - a, device="cuda")[None]
            hidden = (j > i) | ((i - j >= case["window"]) & (j >= case["sinks"]))
            for h in range(case["heads"]):
                score = s["q"][a:b, h].double() @ s["k"][a:b, h // group].double().T / math.sqrt(dim)
                out[a:b, h] = torch.softmax(torch.where(hidden, -math.inf, score), 1) @ s["v"][a:b, h // group].double()
        return out
    four, sinks, window = case["type"] == "int4", case["sinks"], case["window"]
    held = {x: _held(s[x + "s"], s[x + "_scales"]) if four else s[x + "s"].double() for x in ("key", "value")}
    edges = s["starts"].tolist() if s["starts"] is not None else list(range(case["tokens"] + 1))
    new = {}
    for name in ("q", "k"):
        x = s[name].double()
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / dim + EPSILON) * s[name + "_gain"].double()
        z = torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous())
        at = torch.cat([torch.arange(b - a, device="cuda") + p for a, b, p in zip(edges[:-1], edges[1:], s["positions"].tolist())])
        new[name] = torch.view_as_real(z * torch.exp(1j * at[:, None, None].double() * s["frequencies"])).flatten(-2)
    for i, (a, b, p) in enumerate(zip(edges[:-1], edges[1:], s["positions"].tolist())):
        first = max(0, b - a - window)
        for x, rows in (("key", new["k"][a:b]), ("value", s["v"][a:b].double())):
            rows = (_quantised(rows) if four else rows).transpose(0, 1)
            at = torch.arange(p, p + b - a, device="cuda")
            ring = torch.arange(first, b - a, device="cuda")
            ring = ring[at[ring] >= sinks]
            held[x][i][:, sinks + (at[ring] - sinks) % window] = rows[:, ring]
            early = torch.nonzero(at < sinks)[:, 0]
            held[x][i][:, at[early]] = rows[:, early]
    return {"q": new["q"], "keys": held["key"], "values": held["value"]}
