"""What is measured of the operators that serve a block token by token: the norm and rotation of queries
and keys in one pass, the cache held in 4 bits (write and read back) and the attention over it.

`run` computes each operator in its plain form, or, where `own` is true, through oct_b200.reactor.

The cache.  Keys and values of a (token, head) row are quantised in groups of 32 channels: with x
clamped to +-65504, z is the greatest float16 <= min x, s the least float16 with z + 15 s >= max x and
a code the nearest integer to (x - z) / s (ties to even).  Pages hold tiles of 16 tokens per head:
key codes [16][D/2], key (s, z) pairs [16][D/32], the same of the values.  In a row, the four codes of
channels 32 j + 4 g + 0..3 are the halfword g * (D/32) + j, the lowest code in the lowest bits.
"""
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZES = {"bf16": 2, "f16": 2, "f32": 4}
TILE = 16
GROUP = 32
F16_MAX = 65504.0


# ------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of the Gemma block: one token, 8 query heads and 1 key head of 256 channels
        {"name": "rotate 1 token 8+1x256", "op": "rotate", "type": "bf16", "tokens": 1, "heads": 8, "kv_heads": 1,
         "dim": 256, "rotary": 256, "axes": 1, "interleaved": False, "norm": True, "far": 131071},
        # the Gemma block's benchmark batch, 4 x 1024 tokens, in the framework's own fp32
        {"name": "rotate 4x1024 8+1x256", "op": "rotate", "type": "f32", "tokens": 4096, "heads": 8, "kv_heads": 1,
         "dim": 256, "rotary": 256, "axes": 1, "interleaved": False, "norm": True, "far": 1024},
        # the DiT block's benchmark batch, 2 x 4096 image tokens of 24 heads, positions with three axes
        {"name": "rotate 2x4096 24+24x128 3ax", "op": "rotate", "type": "bf16", "tokens": 8192, "heads": 24,
         "kv_heads": 24, "dim": 128, "rotary": 128, "axes": 3, "interleaved": True, "norm": True, "far": 64},
        # one decode step of 64 sequences: one new key and value row per sequence and head, written and read back
        {"name": "write+read 64x1 8x128", "op": "cache", "type": "bf16", "batch": 64, "least": 1, "most": 1,
         "before": 4000, "kv_heads": 8, "dim": 128, "page": 64, "write": True, "lengths": 1},
        # the prompts of the Gemma block's benchmark batch, in fp32
        {"name": "write+read 4x1024 1x256", "op": "cache", "type": "f32", "batch": 4, "least": 1024, "most": 1024,
         "before": 0, "kv_heads": 1, "dim": 256, "page": 64, "write": True, "lengths": 2},
        # 24 prompts of very different lengths appended behind what their sequences hold already
        {"name": "write+read 24 ragged 8x128", "op": "cache", "type": "bf16", "batch": 24, "least": 0, "most": 8191,
         "before": 999, "kv_heads": 8, "dim": 128, "page": 32, "write": True, "lengths": 3},
        # a cached prefix fetched for a sequence that moves elsewhere
        {"name": "read 1x777 4x64", "op": "cache", "type": "f16", "batch": 1, "least": 777, "most": 777,
         "before": 5, "kv_heads": 4, "dim": 64, "page": 16, "write": False, "lengths": 4},
        {"name": "read 8x16384 8x128", "op": "cache", "type": "bf16", "batch": 8, "least": 16000, "most": 16384,
         "before": 0, "kv_heads": 8, "dim": 128, "page": 128, "write": False, "lengths": 5},
        # the Gemma block's decode step over a thousand keys: latency counts
        {"name": "attend 1x1000 8/1x256", "op": "attend", "type": "bf16", "batch": 1, "least": 1000, "most": 1000,
         "queries": 1, "heads": 8, "kv_heads": 1, "dim": 256, "page": 64, "window": 0, "causal": True, "lengths": 6},
        # four tokens verified at once over a sliding window, fp32
        {"name": "attend 16x4 window 8/1x256", "op": "attend", "type": "f32", "batch": 16, "least": 300, "most": 9000,
         "queries": 4, "heads": 8, "kv_heads": 1, "dim": 256, "page": 16, "window": 512, "causal": True, "lengths": 7},
        # a decode step of one very long sequence: few rows, the keys have to be split
        {"name": "attend 1x131071 32/8x128", "op": "attend", "type": "f16", "batch": 1, "least": 131071,
         "most": 131071, "queries": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 256, "window": 0,
         "causal": True, "lengths": 8},
        # a full decode batch of ragged sequences
        {"name": "attend 64 ragged 32/8x128", "op": "attend", "type": "bf16", "batch": 64, "least": 0, "most": 16384,
         "queries": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "causal": True, "lengths": 9},
    ]


def _spread(rng, low, high):
    """A whole number of low..high, even over its logarithm."""
    return min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49))))))


def draw(rng):
    op = rng.choice(["rotate", "cache", "cache", "attend", "attend", "attend"])
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    dim = rng.choice([64, 128, 128, 256])
    if op == "rotate":
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        heads = _spread(rng, 1, 32)
        kv_heads = rng.choice([h for h in range(1, heads + 1) if heads % h == 0])
        tokens = _spread(rng, 1, max(1, min(16384, (8192 * 48 * 128 // 2) // ((heads + kv_heads) * dim))))
        axes = rng.choice([1, 1, 2, 3, 4])
        return {"op": op, "type": kind, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rotary": rng.choice([dim, dim, dim // 32 * 16]), "axes": axes, "interleaved": rng.random() < 0.4,
                "norm": rng.random() < 0.8, "far": _spread(rng, 100, 1000000)}
    kv_heads = rng.choice([1, 1, 2, 4, 8])
    page = rng.choice([16, 32, 64, 128, 256])
    lengths = rng.randrange(1 << 20)
    batch = _spread(rng, 1, 64)
    if op == "cache":
        room = 24 * 2000 * 8 * 128 // (batch * kv_heads * dim)
        most = _spread(rng, 1, max(1, min(16384, room)))
        return {"op": op, "type": kind, "batch": batch, "least": rng.choice([0, most // 2, most]), "most": most,
                "before": rng.choice([0, 1, 13, 500]), "kv_heads": kv_heads, "dim": dim, "page": page,
                "write": rng.random() < 0.6, "lengths": lengths}
    room = 64 * 5000 * 8 * 128 // (batch * kv_heads * dim)
    most = _spread(rng, 1, max(1, min(131072, room)))
    queries = rng.choice([1, 1, 1, 2, 3, 5, 8])
    return {"op": op, "type": kind, "batch": batch, "least": rng.choice([0, most // 2, most]), "most": most,
            "queries": queries, "heads": kv_heads * rng.choice([1, 2, 3, 4, 7, 8, 16]), "kv_heads": kv_heads,
            "dim": dim, "page": page, "window": rng.choice([0, 0, 0, 1, 100, 1000]), "causal": True,
            "lengths": lengths}


def _counts(case):
    """What each sequence brings (new tokens, or queries) and holds after it, from the case alone."""
    r = random.Random(case["lengths"])
    if case["op"] == "cache":
        new = [case["most"]] + [r.randint(case["least"], case["most"]) for _ in range(case["batch"] - 1)]
        return new, [n + (r.randint(0, case["before"]) if case["most"] != case["least"] else case["before"]) for n in new]
    held = [case["most"]] + [r.randint(case["least"], case["most"]) for _ in range(case["batch"] - 1)]
    return [case["queries"]] * case["batch"], held


def _tile_bytes(dim):
    return 2 * TILE * (dim // 2 + dim // GROUP * 4)


def work(case):
    size, dim = _SIZES[case["type"]], case["dim"]
    if case["op"] == "rotate":
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * dim
        return {"bytes": 2 * n * size + 4 * case["tokens"] * case["axes"], "flops": 8 * n}
    new, held = _counts(case)
    row = dim // 2 + dim // GROUP * 4
    if case["op"] == "cache":
        rows = 2 * sum(new) * case["kv_heads"]
        passes = 2 if case["write"] else 1
        return {"bytes": passes * rows * (dim * size + row), "flops": passes * 4 * rows * dim}
    seen = read = 0
    for n, h in zip(new, held):
        last = [max(0, h - n + i + 1) for i in range(n)]
        first = [max(0, e - case["window"]) if case["window"] else 0 for e in last]
        seen += sum(e - f for e, f in zip(last, first))
        read += max(last) - first[0]
    q = sum(new) * case["heads"]
    return {"bytes": 2 * read * case["kv_heads"] * row + q * (2 * dim * size + 4),
            "flops": 4 * dim * seen * case["heads"]}


# ------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator("cuda").manual_seed(seed * 7919 + 17)


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _int(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def _pages(case, g, held):
    """A page table over pages in no order, and how many pages there are."""
    page = case["page"]
    width = max(1, -(-max(held) // page))
    total = case["batch"] * width + 3
    order = torch.randperm(total, generator=g, device="cuda")[: case["batch"] * width]
    return order.to(torch.int32).reshape(case["batch"], width).contiguous(), total


def _rows_like(g, *shape):
    """Keys or values as a model gives them: some channels stand out by their size or an offset."""
    dim = shape[-1]
    gain = 1.0 + 4.0 * (torch.rand(dim, generator=g, device="cuda") < 0.05)
    shift = 2.0 * torch.randn(dim, generator=g, device="cuda") * (torch.rand(dim, generator=g, device="cuda") < 0.1)
    return _normal(g, *shape) * gain + shift


def prepare(case, seed):
    g = _generator(seed)
    dtype, dim = _TYPES[case["type"]], case["dim"]
    if case["op"] == "rotate":
        t, h, k = case["tokens"], case["heads"], case["kv_heads"]
        # queries, keys and values side by side, as the fused projection leaves them
        x = _normal(g, t, h + 2 * k, dim, dtype=dtype)
        pairs = case["rotary"] // 2
        axes = [pairs // case["axes"]] * case["axes"]
        axes[0] += pairs - sum(axes)
        within = torch.cat([torch.arange(n, device="cuda", dtype=torch.float64) / n for n in axes])
        return {"case": case, "q": x[:, :h], "k": x[:, h:h + k],
                "positions": torch.randint(0, case["far"] + 1, (t, case["axes"]), generator=g, device="cuda",
                                           dtype=torch.int32),
                "frequencies": torch.pow(10000.0, -within), "axes": axes,
                "q_weight": 1.0 + 0.2 * _normal(g, dim), "k_weight": 1.0 + 0.2 * _normal(g, dim),
                "q_out": torch.empty(t, h, dim, device="cuda", dtype=dtype),
                "k_out": torch.empty(t, k, dim, device="cuda", dtype=dtype)}
    new, held = _counts(case)
    table, total = _pages(case, g, held)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s = {"case": case, "table": table, "held": _int(held), "starts": _int(starts), "tokens": starts[-1],
         "most_new": max(new), "most_held": max(held)}
    shape = (total, case["kv_heads"], case["page"] // TILE, TILE, dim)
    if case["op"] == "cache":
        s["k"] = _rows_like(g, starts[-1], case["kv_heads"], dim).to(dtype)
        s["v"] = _rows_like(g, starts[-1], case["kv_heads"], dim).to(dtype)
        s["k_back"], s["v_back"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
        if case["write"]:
            s["data"] = torch.zeros(*shape[:3], _tile_bytes(dim), device="cuda", dtype=torch.uint8)
            return s
    else:
        s["q"] = _normal(g, starts[-1], case["heads"], dim, dtype=dtype)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(starts[-1], case["heads"], device="cuda", dtype=torch.float32)
    s["data"] = torch.cat([_packed(*_quantised(_rows_like(g, *shape))),
                           _packed(*_quantised(_rows_like(g, *shape)))], dim=-1)
    return s


# --------------------------------------------------------------------------------- the plain forms
def _f16_below(x):
    """The greatest float16 <= x."""
    h = x.half()
    bits = h.view(torch.int16).int() & 0xFFFF
    down = torch.where(bits == 0, 0x8001, torch.where(bits >= 0x8000, bits + 1, bits - 1))
    down = torch.where(bits == 0x8000, 0x8001, down)
    bits = torch.where(h.double() > x.double(), down, bits)
    return torch.where(bits >= 0x8000, bits - 0x10000, bits).to(torch.int16).view(torch.float16)


def _f16_above(x):
    """The least float16 >= x, for x >= 0."""
    h = x.half()
    bits = h.view(torch.int16).int()
    return torch.where(h.double() < x.double(), bits + 1, bits).to(torch.int16).view(torch.float16)


def _quantised(x):
    """Codes [..., D], scales and zeros [..., D/32]."""
    x = x.double().clamp(-F16_MAX, F16_MAX).unflatten(-1, (-1, GROUP))
    z = _f16_below(x.amin(-1))
    s = _f16_above((x.amax(-1) - z.double()) / 15)
    codes = torch.where(s[..., None] > 0, torch.round((x - z.double()[..., None]) / s.double()[..., None]), 0.0)
    return codes.to(torch.uint8).flatten(-2), s, z


def _packed(codes, s, z):
    """[..., 16, D] codes and their scales and zeros as bytes [..., half a tile]."""
    dim = codes.shape[-1]
    x = codes.unflatten(-1, (dim // GROUP, 8, 4)).transpose(-3, -2).flatten(-3)
    x = x[..., 0::2] | (x[..., 1::2] << 4)
    return torch.cat([x.flatten(-2), torch.stack([s, z], dim=-1).view(torch.uint8).flatten(-3)], dim=-1)


def _values(half, dim):
    """Half a tile's bytes [..., n] as values [..., 16, D] in 32 bits."""
    groups = dim // GROUP
    x = half[..., : TILE * dim // 2].unflatten(-1, (TILE, dim // 2))
    x = torch.stack([x & 15, x >> 4], dim=-1).flatten(-2).unflatten(-1, (8, groups, 4)).transpose(-3, -2)
    p = half[..., TILE * dim // 2:].contiguous().view(torch.float16).unflatten(-1, (TILE, groups, 2)).float()
    return (x.flatten(-2).float() * p[..., 0:1] + p[..., 1:2]).flatten(-2)


def _plain_rotate(s):
    case = s["case"]
    angle = s["positions"].double()[:, _axis_of_pair(s["axes"])] * s["frequencies"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    return [_plain_rotate_one(x, w, cos, sin, case) for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"]))]


def _axis_of_pair(axes):
    return torch.repeat_interleave(torch.arange(len(axes)), torch.tensor(axes)).to("cuda")


def _plain_rotate_one(x, w, cos, sin, case):
    y = x.float()
    if case["norm"]:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w
    turn, rest = y[..., : case["rotary"]], y[..., case["rotary"]:]
    if case["interleaved"]:
        a, b = turn[..., 0::2], turn[..., 1::2]
        turn = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = turn.chunk(2, dim=-1)
        turn = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turn, rest], dim=-1).to(x.dtype)


def _slots(s):
    """Page and place in it of every token that a call brings."""
    starts, held, page = s["starts"].long(), s["held"].long(), s["case"]["page"]
    new = starts[1:] - starts[:-1]
    seq = torch.repeat_interleave(torch.arange(new.numel(), device="cuda"), new, output_size=s["tokens"])
    at = held[seq] - new[seq] + torch.arange(s["tokens"], device="cuda") - starts[seq]
    return s["table"].long()[seq, at // page], at % page


def _plain_cache(s):
    case, dim = s["case"], s["case"]["dim"]
    pages, place = _slots(s)
    tile, row = place // TILE, place % TILE
    data, half = s["data"], _tile_bytes(dim) // 2
    codes = TILE * dim // 2
    by_codes = torch.arange(dim // 2, device="cuda")
    by_params = codes + torch.arange(dim // GROUP * 4, device="cuda")
    at = torch.cat([row[:, None] * (dim // 2) + by_codes, row[:, None] * (dim // GROUP * 4) + by_params], dim=1)
    place = (pages[:, None, None], torch.arange(case["kv_heads"], device="cuda")[None, :, None], tile[:, None, None])
    if case["write"]:
        data[(*place, at[:, None])] = _packed_rows(s["k"])
        data[(*place, half + at[:, None])] = _packed_rows(s["v"])
    return [_row_values(data[(*place, at[:, None] + off)], dim).to(s["k"].dtype) for off in (0, half)]


def _packed_rows(x):
    codes, s, z = _quantised(x)
    dim = codes.shape[-1]
    c = codes.unflatten(-1, (dim // GROUP, 8, 4)).transpose(-3, -2).flatten(-3)
    return torch.cat([c[..., 0::2] | (c[..., 1::2] << 4), torch.stack([s, z], dim=-1).view(torch.uint8).flatten(-2)], dim=-1)


def _row_values(row, dim):
    groups = dim // GROUP
    x = row[..., : dim // 2]
    x = torch.stack([x & 15, x >> 4], dim=-1).flatten(-2).unflatten(-1, (8, groups, 4)).transpose(-3, -2)
    p = row[..., dim // 2:].contiguous().view(torch.float16).unflatten(-1, (groups, 2)).float()
    return (x.flatten(-2).float() * p[..., 0:1] + p[..., 1:2]).flatten(-2)


def _plain_attend(s):
    case, dim, n = s["case"], s["case"]["dim"], s["case"]["queries"]
    half = _tile_bytes(dim) // 2
    b, kv = case["batch"], case["kv_heads"]
    data = s["data"][s["table"].long()]  # [b][pages][kv][tiles][bytes]
    k, v = (_values(data[..., at: at + half], dim).permute(0, 2, 1, 3, 4, 5).reshape(b, kv, -1, dim) for at in (0, half))
    q = s["q"].float().reshape(b, n, kv, -1, dim).permute(0, 2, 1, 3, 4).reshape(b, kv, -1, dim)
    last = s["held"].long()[:, None] - n + torch.arange(n, device="cuda")
    key = torch.arange(k.shape[2], device="cuda")
    seen = key <= last[..., None]
    if case["window"]:
        seen = seen & (key > last[..., None] - case["window"])
    seen = seen.repeat_interleave(case["heads"] // kv, dim=1)[:, None]
    scores = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(dim))
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / total.clamp_min(1e-38)
    lse = (top + torch.log(total)).squeeze(-1)
    back = lambda x, *d: x.reshape(b, kv, n, -1, *d).transpose(1, 2).reshape(b * n, case["heads"], *d)  # noqa: E731
    return [back(o, dim).to(s["q"].dtype), back(lse)]


# ------------------------------------------------------------------------------ the framework's own
_runtime = None


def _handle():
    global _runtime
    if _runtime is None:
        from oct_b200.reactor import Runtime
        _runtime = Runtime()
    return _runtime


def _own_cache(s):
    """The descriptors that a serving program makes once and keeps."""
    if "cache" not in s:
        from oct_b200.reactor import Kv4Batch, Kv4Cache
        case = s["case"]
        s["cache"] = Kv4Cache(s["data"], page_size=case["page"], kv_heads=case["kv_heads"], head_dim=case["dim"])
        s["batch"] = Kv4Batch(s["table"], s["held"], s["starts"], max_tokens=s["most_new"], max_kv_len=s["most_held"])
        if case["op"] == "attend":
            s["workspace"] = torch.empty(_handle().kv4_attention_workspace_bytes(s["cache"], s["batch"], s["q"]),
                                         device="cuda", dtype=torch.uint8)
    return s["cache"], s["batch"]


def _own_run(s):
    rt, case = _handle(), s["case"]
    if case["op"] == "rotate":
        rt.qk_norm_rope_device(s["q"], s["k"], s["q_out"], s["k_out"], s["positions"], s["frequencies"],
                               axis_pairs=s["axes"], interleaved=case["interleaved"], normalize=case["norm"],
                               q_weight=s["q_weight"] if case["norm"] else None,
                               k_weight=s["k_weight"] if case["norm"] else None, eps=1e-6)
        return [s["q_out"], s["k_out"]]
    cache, batch = _own_cache(s)
    if case["op"] == "attend":
        rt.kv4_attention_device(cache, batch, s["q"], s["out"], causal=case["causal"], window=case["window"],
                                lse=s["lse"], workspace=s["workspace"])
        return [s["out"], s["lse"]]
    if case["write"]:
        rt.kv4_store_device(cache, batch, s["k"], s["v"])
    rt.kv4_load_device(cache, batch, s["k_back"], s["v_back"])
    return [s["k_back"], s["v_back"]]


def run(state):
    if own:
        return _own_run(state)
    op = state["case"]["op"]
    return (_plain_rotate if op == "rotate" else _plain_cache if op == "cache" else _plain_attend)(state)


# ----------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"rotate": _exact_rotate, "cache": _exact_cache, "attend": _exact_attend}[case["op"]](s)


def _exact_rotate(s):
    case = s["case"]
    outs = []
    for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        y = x.double()
        if case["norm"]:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / case["dim"] + 1e-6) * w.double()
        z = y.clone()
        j = 0
        for axis, count in enumerate(s["axes"]):
            for _ in range(count):
                turn = (s["positions"][:, axis].double() * s["frequencies"][j])[:, None]
                a, b = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + case["rotary"] // 2)
                z[..., a] = y[..., a] * turn.cos() - y[..., b] * turn.sin()
                z[..., b] = y[..., a] * turn.sin() + y[..., b] * turn.cos()
                j += 1
        outs.append(z)
    return outs


def _channel_places(dim):
    """Where in a row's codes each channel stands: its byte and the power of 16 in it."""
    byte, high = [], []
    for c in range(dim):
        halfword = (c % 32) // 4 * (dim // 32) + c // 32
        byte.append(2 * halfword + c % 4 // 2)
        high.append(c % 2)
    return torch.tensor(byte, device="cuda"), torch.tensor(high, device="cuda")


def _exact_rows(data, dim, table, first, last, page, half):
    """The values of positions first..last-1 of a sequence, [tokens][kv heads][D], read code by code."""
    at = torch.arange(first, last, device="cuda")
    tiles = data[table.long()[at // page], :, at % page // 16]  # [tokens][kv heads][bytes]
    row = (at % 16)[:, None, None]
    byte, high = _channel_places(dim)
    index = (half + row * (dim // 2) + byte).expand(-1, tiles.shape[1], -1)
    codes = torch.gather(tiles, 2, index).long()
    codes = torch.where(high.bool(), codes // 16, codes % 16)
    where = half + 16 * (dim // 2) + row * (dim // 8) + 4 * (torch.arange(dim, device="cuda") // 32)
    word = [torch.gather(tiles, 2, (where + i).expand(-1, tiles.shape[1], -1)).int() for i in range(4)]
    s, z = ((lo + 256 * hi).to(torch.int32) for lo, hi in ((word[0], word[1]), (word[2], word[3])))
    s, z = (torch.where(u >= 32768, u - 65536, u).to(torch.int16).view(torch.float16).double() for u in (s, z))
    return z + s * codes


def _exact_quantised(x):
    """What a written row reads back as, from the definition: bounds searched among the float16 numbers."""
    grid = torch.arange(0x7C00, device="cuda", dtype=torch.int16).view(torch.float16).double()  # 0 and up
    both = torch.cat([-grid.flip(0)[:-1], grid])
    x = x.double().clamp(-F16_MAX, F16_MAX)
    y = x.reshape(*x.shape[:-1], -1, 32)
    low, high = y.min(-1).values, y.max(-1).values
    z = both[torch.searchsorted(both, low, right=True) - 1]
    s = grid[torch.searchsorted(grid * 15, high - z)]
    step = torch.where(s > 0, s, torch.ones_like(s))[..., None]
    code = ((y - z[..., None]) / step).round() * (s > 0)[..., None]
    return (z[..., None] + s[..., None] * code).reshape(x.shape)


def _exact_cache(s):
    case, dim = s["case"], s["case"]["dim"]
    if case["write"]:
        return [_exact_quantised(s["k"]), _exact_quantised(s["v"])]
    new, held = _counts(case)
    half = _tile_bytes(dim) // 2
    return [torch.cat([_exact_rows(s["data"], dim, s["table"][i], h - n, h, case["page"], at)
                       for i, (n, h) in enumerate(zip(new, held))]) for at in (0, half)]


def _exact_attend(s):
    case, dim, n = s["case"], s["case"]["dim"], s["case"]["queries"]
    half, share = _tile_bytes(dim) // 2, case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    lse = torch.full(out.shape[:2], -math.inf, device="cuda", dtype=torch.float64)
    _, held = _counts(case)
    for i, h in enumerate(held):
        begin = max(0, h - n + 1 - case["window"]) if case["window"] else 0
        if h <= 0:
            continue
        k, v = (_exact_rows(s["data"], dim, s["table"][i], begin, h, case["page"], at) for at in (0, half))
        for t in range(n):
            last = h - n + t + 1
            first = max(0, last - case["window"]) if case["window"] else 0
            if last <= first:
                continue
            kk, vv = k[first - begin: last - begin], v[first - begin: last - begin]
            q = s["q"][i * n + t].double().reshape(-1, share, dim)
            score = torch.einsum("hgd,lhd->hgl", q, kk) / math.sqrt(dim)
            lse[i * n + t] = torch.logsumexp(score, -1).reshape(-1)
            out[i * n + t] = torch.einsum("hgl,lhd->hgd", torch.softmax(score, -1), vv).reshape(-1, dim)
    return [out, lse]
