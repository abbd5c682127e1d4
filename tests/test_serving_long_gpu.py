"""The 4-bit cache attention where its blocks take equal runs of long keys: steps of many turns of a
warp's ring, cut items and their join, against a binary64 computation on the device.

Tolerances are those of test_serving_gpu.py, term by term.  A cache here is random codes with chosen
scales and zeros (any bits are codes), whose pages the sequences share, so that millions of keys need a
few thousand tokens of memory.
"""
from __future__ import annotations

import numpy as np
import pytest

from oct_b200 import reactor as R
from oracle import serving as O
from tests.test_serving_gpu import TYPES, _int, _ok, _torch

pytestmark = pytest.mark.gpu

RESIDENT = {True: 444, False: 296}  # blocks the GPU holds: 3 an SM where dim * row groups <= 128, else 2
ITEM_COST = 5


class Pool:
    """Pages of tokens, and sequences that name them in any order, some of them many times."""

    def __init__(self, rng, dim, kv_heads, page, pages, size=None, lift=None):
        """size [2][kv_heads][tokens], lift likewise: scale and middle of each token's values (2: keys, values)."""
        import torch
        self.dim, self.kv_heads, self.page, self.pages = dim, kv_heads, page, pages
        tokens, groups = pages * page, dim // 32
        if size is None:
            size = np.full((2, kv_heads, tokens), 0.25)
        if lift is None:
            lift = np.zeros((2, kv_heads, tokens))
        codes = rng.integers(0, 16, (2, kv_heads, tokens, dim), dtype=np.uint8)
        s = (size[..., None] * rng.uniform(0.5, 1.0, (2, kv_heads, tokens, groups))).astype(np.float16)
        z = (lift[..., None] - s.astype(np.float64) * rng.uniform(5.0, 10.0, s.shape)).astype(np.float16)
        byte, high = O._places(dim)
        packed = np.zeros((2, kv_heads, tokens, dim // 2), np.uint8)
        for odd in (0, 1):
            packed[..., byte[high == odd]] |= codes[..., high == odd] << (4 * odd)
        params = np.stack([s, z], axis=-1).reshape(2, kv_heads, tokens, -1).view(np.uint8)
        tiles = lambda x: x.reshape(2, kv_heads, pages, page // 16, -1).transpose(2, 1, 3, 0, 4)  # noqa: E731
        data = np.concatenate([tiles(packed), tiles(params)], axis=-1).reshape(pages, kv_heads, page // 16, -1)
        assert data.shape[-1] == O.tile_bytes(dim)
        self.cache = R.Kv4Cache(torch.from_numpy(np.ascontiguousarray(data)).cuda(), page_size=page, kv_heads=kv_heads,
                                head_dim=dim)
        s64, z64 = (np.repeat(x.astype(np.float64), 32, axis=-1) for x in (s, z))
        self.values = torch.from_numpy(z64 + s64 * codes).cuda()          # [2][kv_heads][tokens][dim]
        self.reach = torch.from_numpy(np.abs(z64) + 15.0 * s64).cuda()

    def batch(self, table, held, new, width=None):
        """A table of at least `width` pages a sequence; pages behind a sequence's last are none of the cache's."""
        full = np.full((len(held), max(width or 0, table.shape[1])), -1, np.int32)
        for b, h in enumerate(held):
            used = -(-h // self.page)
            full[b, :used] = table[b, :used]
        starts = np.concatenate([[0], np.cumsum(new)])
        return R.Kv4Batch(_int(full), _int(held), _int(starts), max_tokens=max(new), page_size=self.page)

    def random_table(self, rng, held):
        return rng.integers(0, self.pages, (len(held), max(1, -(-max(held) // self.page)))).astype(np.int32)


def _layout(pool, batch, q_heads, held, new, window, workspace):
    """(units, blocks, whether units are few, units of a block's run) of an attention call, restated."""
    share = q_heads // pool.kv_heads
    most = {64: 32, 128: 16, 256: 8}[pool.dim]
    tile = 8
    while tile < most and tile < max(new) * share:
        tile *= 2
    narrow = pool.dim * tile // 8 <= 128
    unit = 16 * 4 * (2 if narrow else 1)
    blocks = workspace // (2 * tile * (pool.dim * 4 + 8) + 32)
    total = items = 0
    for h, n in zip(held, new):
        for first in range(0, n * share, tile):
            last = min(n * share, first + tile) - 1
            hi0, hi1 = h - n + first // share, h - n + last // share
            lo = max(0, hi0 - window + 1) if window else 0
            tiles = hi1 // 16 + 1 - lo // 16 if hi1 >= 0 else 0
            total += max(1, -(-tiles // (unit // 16))) * pool.kv_heads
            items += pool.kv_heads
    few = total <= 4 * blocks and items <= blocks // 2
    run = total if few else total + ITEM_COST * items
    assert blocks <= RESIDENT[narrow]
    return total, blocks, few, -(-run // (blocks - items if few else blocks))


def _want(pool, table, h, q, scale, window):
    """Binary64 attention of one sequence's n rows q [n][heads][dim], and what its tolerance needs."""
    import torch
    n, heads, dim = q.shape
    share = heads // pool.kv_heads
    pos = torch.arange(h, device="cuda")
    at = torch.as_tensor(table, device="cuda", dtype=torch.int64)[pos // pool.page] * pool.page + pos % pool.page
    last = h - n + torch.arange(n, device="cuda").repeat_interleave(share)[:, None]
    seen = (pos <= last) & ((pos > last - window) if window else True)
    out, weight, lse, reach = [], [], [], []
    for head in range(pool.kv_heads):
        k, v = pool.values[0, head, at], pool.values[1, head, at]
        x = q[:, head * share:(head + 1) * share].double().reshape(n * share, dim)
        score = (x @ k.T * scale).masked_fill(~seen, -np.inf)
        top = score.amax(-1, keepdim=True) if h else score.new_full((n * share, 1), -np.inf)
        e = torch.exp(score - top.clamp_min(-1e300))
        total = e.sum(-1, keepdim=True)
        p = e / total.clamp_min(1e-300)
        out.append(p @ v)
        weight.append(p @ pool.reach[1, head, at])
        lse.append((top + total.log())[:, 0])
        m = (x.abs() @ pool.reach[0, head, at].T * abs(scale)).masked_fill(~seen, 0.0)
        reach.append(m.amax(-1) if h else lse[-1].new_zeros(n * share))
    back = lambda parts: torch.stack(parts).unflatten(1, (n, share)).transpose(0, 1).flatten(1, 2)  # noqa: E731
    return back(out), back(weight), back(lse), back(reach)


def _check(pool, kind, table, held, new, q, out, lse, window=0, scale=None):
    import torch
    u = TYPES[kind][1]
    scale = float(np.float32(1.0) / np.sqrt(np.float32(pool.dim))) if scale is None else float(np.float32(scale))
    start = 0
    for b, (h, n) in enumerate(zip(held, new)):
        sl = slice(start, start + n)
        start += n
        if n == 0:
            continue
        want, weight, want_lse, reach = _want(pool, table[b], h, q[sl], scale, window)
        pages = torch.as_tensor(table[b][: -(-h // pool.page)], device="cuda", dtype=torch.int64)
        largest = pool.reach[1].unflatten(1, (-1, pool.page))[:, pages].amax().item() if h else 0.0
        d = 2.0 ** -20 * reach + 2.0 ** -21
        sums = (h / 16 + 48) * 2.0 ** -24
        rel = 2 * d + 2.0 ** -21 + (2.0 ** -11 if kind == "bf16" else 2.0 ** -21) + sums
        tiny = (2.0 ** -25 if kind == "f16" else 0.0) + h * 2.0 ** -33 * largest ** 2 / 15
        off = (out[sl].double() - want).abs() - (u * want.abs() * 1.01 + rel[..., None] * weight + tiny)
        assert not (off > 0).any() and out[sl].isfinite().all(), (b, h, off.max().item())
        empty = want_lse == -np.inf
        assert torch.equal(lse[sl] == -np.inf, empty), (b, h)
        off = (lse[sl].double() - want_lse).abs() - (d + 2.0 ** -22 * want_lse.abs() + sums)
        assert not (off[~empty] > 0).any() and not lse[sl].isnan().any(), (b, h, off[~empty].max().item())
        assert (out[sl][empty] == 0).all()


def _run(runtime, pool, batch, q, window=0, scale=None, out=None):
    import torch
    need = runtime.kv4_attention_workspace_bytes(pool.cache, batch, q, window=window)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    out = torch.full_like(q, 7.0) if out is None else out
    lse = torch.full(q.shape[:2], 7.0, device="cuda")
    runtime.kv4_attention_device(pool.cache, batch, q, out, lse=lse, window=window, scale=scale, workspace=ws)
    return out, lse, need


# dim, query heads per key head, queries: every row tile of every dim
FORMS = [(64, 1, 1), (64, 4, 3), (64, 8, 4), (128, 4, 1), (128, 5, 3), (256, 8, 1), (256, 3, 5)]


def _ragged(rng, sequences, dim, rows, queries, runs):
    """Lengths, a quarter of them short or none, whose key tiles fill about `runs` units for each resident block."""
    tile = 8
    while tile < {64: 32, 128: 16, 256: 8}[dim] and tile < rows:
        tile *= 2
    narrow = dim * tile // 8 <= 128
    keys = RESIDENT[narrow] * runs * (128 if narrow else 64)
    mean = keys / (2 * sequences * -(-rows // tile))
    held = [int(x) for x in rng.uniform(0.4, 2.2, sequences) * mean]
    for i in rng.permutation(sequences)[: sequences // 4]:
        held[i] = int(rng.integers(0, 300))
    held[3], held[7], held[11] = 0, 1, queries - 1  # the last: its first query sees nothing
    return held


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("form", FORMS, ids=lambda f: "-".join(map(str, f)))
def test_long_ragged_sequences_in_equal_runs(runtime, kind, form):
    """A warp takes more than 32 steps of an item (a second look at the page table, its ring many times
    round), blocks end one cut item and begin another, empty and short sequences lie between."""
    import torch
    dim, share, queries = form
    rng = np.random.default_rng(dim + 10 * share + queries)
    sequences, page = 44, {64: 16, 128: 48, 256: 64}[dim]
    held = _ragged(rng, sequences, dim, share * queries, queries, 60)
    pool = Pool(rng, dim, 2, page, 3000 // page)
    table = pool.random_table(rng, held)
    new = [queries] * sequences
    batch = pool.batch(table, held, new)
    q = _torch(rng.standard_normal((sum(new), 2 * share, dim)), kind)
    out, lse, need = _run(runtime, pool, batch, q)
    total, blocks, few, per = _layout(pool, batch, 2 * share, held, new, 0, need)
    assert need > 0 and not few and per - ITEM_COST > 32
    again, lse2, _ = _run(runtime, pool, batch, q)
    _ok(runtime)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    _check(pool, kind, table, held, new, q, out, lse)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("form", FORMS, ids=lambda f: "-".join(map(str, f)))
def test_windows_and_cut_items(runtime, kind, form):
    """A window of many units, cut anywhere, over some sequences that are shorter than it."""
    dim, share, queries = form
    rng = np.random.default_rng(1 + dim + 10 * share + queries)
    sequences, page = 60, {64: 64, 128: 16, 256: 32}[dim]
    held = _ragged(rng, sequences, dim, share * queries, queries, 30)
    pool = Pool(rng, dim, 2, page, 3000 // page)
    table = pool.random_table(rng, held)
    new = [queries] * sequences
    batch = pool.batch(table, held, new)
    q = _torch(rng.standard_normal((sum(new), 2 * share, dim)), kind)
    window = int(np.median(held)) // 2 + 5
    out, lse, need = _run(runtime, pool, batch, q, window=window)
    total, blocks, few, per = _layout(pool, batch, 2 * share, held, new, window, need)
    assert need > 0 and not few and per > ITEM_COST
    _ok(runtime)
    _check(pool, kind, table, held, new, q, out, lse, window=window)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim, share", [(64, 2), (128, 8), (256, 8)])
def test_many_short_items_whose_cost_is_cut(runtime, kind, dim, share):
    """More items than half the blocks, most of one unit: runs end inside an item's cost, and leave
    parts without a key; rows behind the last sequence stay as they were."""
    rng = np.random.default_rng(2 + dim)
    held = [int(x) for x in rng.integers(0, 60, 260)]
    for i, h in ((0, 5000), (100, 2500), (101, 2500), (259, 4000)):
        held[i] = h
    pool = Pool(rng, dim, 2, 16, 200)
    table = pool.random_table(rng, held)
    new = [int(x) for x in rng.integers(0, 2, 260)]
    new[0] = new[100] = new[101] = new[259] = 1
    batch = pool.batch(table, held, new)
    q = _torch(rng.standard_normal((sum(new) + 3, 2 * share, dim)), kind)
    out, lse, need = _run(runtime, pool, batch, q)
    total, blocks, few, per = _layout(pool, batch, 2 * share, held, new, 0, need)
    assert need > 0 and not few and per <= ITEM_COST + 2
    _ok(runtime)
    _check(pool, kind, table, held, new, q, out, lse)
    assert (out[sum(new):] == 7.0).all() and (lse[sum(new):] == 7.0).all()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim, share", [(64, 4), (64, 32), (128, 4), (128, 16), (256, 4)])
def test_scores_and_values_that_move_along_the_keys(runtime, kind, dim, share):
    """Scores rise (key head 0) and fall (key head 1), fast, slowly and not at all by the query head;
    values come as zeros first and then grow (head 0), or shrink (head 1): the running maximum and the
    weights' scale are renewed many times within one block's run."""
    rng = np.random.default_rng(3 + dim + share)
    page, sequences = 64, 40
    narrow = dim * (8 if share <= 8 else 16 if share <= 16 else 32) // 8 <= 128
    longest = RESIDENT[narrow] * 45 * (128 if narrow else 64) // (2 * sequences) // page * page
    pages = longest // page
    at = np.arange(longest) / longest
    size, lift = np.full((2, 2, longest), 0.02), np.zeros((2, 2, longest))
    lift[0] = 12.0 * np.stack([at, 1.0 - at])
    size[1] = np.stack([np.where(at < 0.3, 0.0, 1e-5 * 3e5 ** at), 3.0 * 1e-5 ** at])
    pool = Pool(rng, dim, 2, page, pages, size, lift)
    # the first key's and the last one's, whole and short of it
    held = [longest - int(x) for x in rng.integers(0, longest // 8, sequences)]
    held[0] = longest
    table = np.tile(np.arange(pages, dtype=np.int32), (sequences, 1))
    new = [1] * sequences
    batch = pool.batch(table, held, new)
    # scores of sum(q) * lift: 250 over the whole length for the first query head, a tenth of that for the next
    towards = np.array([1.0, 0.1, 0.0, -1.0] * (share // 4) * 2)[None, :, None]
    q = _torch(rng.standard_normal((sequences, 2 * share, dim)) * 0.02 + towards, kind)
    scale = 250.0 / (12.0 * dim)
    out, lse, need = _run(runtime, pool, batch, q, scale=scale)
    total, blocks, few, per = _layout(pool, batch, 2 * share, held, new, 0, need)
    assert need > 0 and not few and per - ITEM_COST > 32
    _ok(runtime)
    _check(pool, kind, table, held, new, q, out, lse, scale=scale)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim, heads", [(64, 8), (128, 16), (256, 8)])
def test_one_long_sequence(runtime, kind, dim, heads):
    """Few units a block: no block has parts of two items, and an item has up to hundreds of parts."""
    rng = np.random.default_rng(4 + dim)
    pool = Pool(rng, dim, 1, 32, 100)
    for held in ([70001], [70001, 5, 0, 33]):
        table = pool.random_table(rng, held)
        new = [1] * len(held)
        batch = pool.batch(table, held, new)
        q = _torch(rng.standard_normal((len(held), heads, dim)), kind)
        out, lse, need = _run(runtime, pool, batch, q)
        _, _, few, per = _layout(pool, batch, heads, held, new, 0, need)
        assert need > 0 and few and per > 1
        _ok(runtime)
        _check(pool, kind, table, held, new, q, out, lse)


@pytest.mark.parametrize("kind", list(TYPES))
def test_a_spread_call_over_its_own_queries(runtime, kind):
    import torch
    rng = np.random.default_rng(5)
    held, new = [30000, 0, 700, 9000], [1, 1, 3, 2]
    pool = Pool(rng, 128, 2, 16, 300)
    table = pool.random_table(rng, held)
    batch = pool.batch(table, held, new)
    q = _torch(rng.standard_normal((7, 8, 128)), kind)
    out, lse, need = _run(runtime, pool, batch, q)
    own = q.clone()
    _, lse2, _ = _run(runtime, pool, batch, own, out=own)
    _ok(runtime)
    assert need > 0 and torch.equal(own, out) and torch.equal(lse, lse2)
    _check(pool, kind, table, held, new, q, out, lse)


def test_captured_spread_steps_follow_lengths_on_two_streams(runtime):
    """Two graphs with a workspace each, replayed at once while the lengths go from many units a block to
    few and back: both kernels of a call are captured, the second launched dependent on the first."""
    import torch
    rng = np.random.default_rng(6)
    sequences, dim, heads = 40, 64, 8
    pool = Pool(rng, dim, 2, 64, 60)
    longest = 444 * 20 * 128 // (2 * sequences)
    lengths = [[longest - 17 * i for i in range(sequences)], [int(x) for x in rng.integers(0, 200, sequences)],
               [longest if i == 5 else i for i in range(sequences)], [(longest * i) // sequences for i in range(sequences)]]
    table = pool.random_table(rng, [longest])
    table = np.concatenate([table] * sequences)
    new = [1] * sequences
    batch = pool.batch(table, [longest] * sequences, new)
    streams = [torch.cuda.Stream() for _ in range(2)]
    parts = []
    for s in streams:
        q = _torch(rng.standard_normal((sequences, heads, dim)), "bf16")
        need = runtime.kv4_attention_workspace_bytes(pool.cache, batch, q)
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        out, lse = torch.empty_like(q), torch.empty((sequences, heads), device="cuda")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            for _ in range(2):  # the second call's first kernel follows the first call's join
                runtime.kv4_attention_device(pool.cache, batch, q, out, lse=lse, workspace=ws, stream=s)
        parts.append((graph, q, ws, out, lse))
        assert need > 0
    kinds = set()
    for held in lengths:
        batch.kv_lens.copy_(_int(held))
        kinds.add(_layout(pool, batch, heads, held, new, 0, need)[2])
        torch.cuda.synchronize()
        for _ in range(5):
            for (graph, *_), s in zip(parts, streams):
                with torch.cuda.stream(s):
                    graph.replay()
        _ok(runtime)
        for _, q, _, out, lse in parts:
            _check(pool, "bf16", table, held, new, q, out, lse)
    assert kinds == {True, False}
    del graph, parts


def test_spread_calls_at_once_on_two_streams(runtime):
    import torch
    rng = np.random.default_rng(7)
    parts = []
    for i in range(2):
        pool = Pool(rng, 128, 1, 16, 200)
        held = [60000 + i, 7, 0, 2100]
        table = pool.random_table(rng, held)
        q = _torch(rng.standard_normal((4, 8, 128)), "f16")
        batch = pool.batch(table, held, [1] * 4)
        ws = torch.empty(runtime.kv4_attention_workspace_bytes(pool.cache, batch, q), dtype=torch.uint8, device="cuda")
        assert ws.numel() > 0
        parts.append((pool, table, held, batch, q, torch.full_like(q, 7.0), torch.full((4, 8), 7.0, device="cuda"), ws))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for (pool, _, _, batch, q, out, lse, ws), s in zip(parts, streams):
            runtime.kv4_attention_device(pool.cache, batch, q, out, lse=lse, workspace=ws, stream=s)
    _ok(runtime)
    for pool, table, held, _, q, out, lse, _ in parts:
        _check(pool, "f16", table, held, [1] * 4, q, out, lse)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim, ratio", [(64, 30), (64, 1000), (128, 100), (256, 30), (256, 1000)])
def test_queries_with_channels_that_stand_out(runtime, kind, dim, ratio):
    """One channel of every group of 32 is far larger than the others (of either sign, or all positive), so that the
    products of the others are small beside those they are added to."""
    rng = np.random.default_rng(8 + dim + ratio)
    held, new = [1500, 40000], [4, 1]
    pool = Pool(rng, dim, 1, 16, 200)
    table = pool.random_table(rng, held)
    batch = pool.batch(table, held, new)
    for positive in (False, True):
        x = rng.standard_normal((5, 8, dim))
        x = np.abs(x) if positive else x
        x[:, :, 5::32] *= ratio
        q = _torch(x, kind)
        scale = 8.0 / (2.0 * (ratio * dim / 32 + dim))
        out, lse, _ = _run(runtime, pool, batch, q, scale=scale)
        _ok(runtime)
        _check(pool, kind, table, held, new, q, out, lse, scale=scale)


def test_a_step_on_torchs_current_stream(runtime):
    """Norm and rotation, store, attention and status with the stream that torch's own operations of the step are
    on, then the same captured: what an inference loop under torch.cuda.stream or torch.cuda.graph does."""
    import torch
    heads, kv, dim, page, sequences = 8, 2, 64, 16, 3
    data = torch.zeros((3 * 20 * kv, R.kv4_tile_bytes(dim)), dtype=torch.uint8, device="cuda")
    cache = R.Kv4Cache(data, page_size=page, kv_heads=kv, head_dim=dim)
    table = torch.arange(60, dtype=torch.int32, device="cuda").view(sequences, 20)
    lens = torch.zeros(sequences, dtype=torch.int32, device="cuda")
    batch = R.Kv4Batch(table, lens, page_size=page)
    freq = torch.logspace(0, -4, dim // 2, dtype=torch.float64, device="cuda")
    w = torch.randn(dim, (heads + 2 * kv) * dim, generator=torch.Generator("cuda").manual_seed(1), device="cuda")
    first = torch.randn(sequences, dim, generator=torch.Generator("cuda").manual_seed(2), device="cuda")
    state = first.clone()
    ws = torch.empty(runtime.kv4_attention_workspace_bytes(cache, batch, torch.empty(sequences, heads, dim)),
                     dtype=torch.uint8, device="cuda")

    def step():
        s = torch.cuda.current_stream()
        x = (state @ w).view(sequences, heads + 2 * kv, dim)
        q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
        pos = lens.clone()
        lens.add_(1)
        runtime.qk_norm_rope_device(q, k, q, k, pos, freq, stream=s)
        runtime.kv4_store_device(cache, batch, k, v, stream=s)
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        runtime.kv4_attention_device(cache, batch, q, out, workspace=ws, stream=s)
        state.copy_(torch.tanh(out.mean(1)) + first)

    def run(once):
        data.zero_()
        lens.zero_()
        state.copy_(first)
        torch.cuda.synchronize()
        for _ in range(100):
            once()
        torch.cuda.synchronize()
        return state.clone()

    side = torch.cuda.Stream()

    def waiting():
        step()
        torch.cuda.synchronize()

    def beside():
        with torch.cuda.stream(side):
            step()

    want = run(waiting)
    assert runtime.sync_status().ok
    assert torch.equal(run(beside), want)
    with torch.cuda.stream(side):
        step()  # torch's own matrix product sets itself up before the capture
    assert runtime.sync_status(side).ok
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    assert torch.equal(run(graph.replay), want)
    assert runtime.sync_status().ok and (lens == 100).all()
    del graph
