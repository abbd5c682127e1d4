"""The token-by-token serving kernels against their binary64 oracle (oracle/serving.py).

Tolerances, derived from the arithmetic (u = half a step of the output type):
* head norm + rotation: the sum of squares, its root, the two products, the fp32 cosine and
  sine (angle reduced in binary64) and the rotation are off by at most 32 * 2^-24 of |a| + |b|,
  the pair's normalised channels; then one rounding.
* cache: codes, scales and zeros are exact; a value read back is one fused product rounded
  to fp32 and then to its type.
* attention: with M the largest scale * sum |q| (|z| + 15 s) of a key and W the mean of
  |z| + 15 s of a channel's values under the softmax, scores are off by at most
  d = 2^-20 M (fp32 sums of D / 16 tensor products and 2 D / 32 scaled parts, q in 22 bits or
  exact) + 2^-21 (the exponent), weights by 2 d + 2^-21, the float16 weights by 2^-12 for bf16
  and their products with the scales by 2^-12 more (2^-21 in two parts for the other types),
  fp32 sums over n keys by (n / 16 + 48) 2^-24, all relative to W.  Weights and products below
  float16's normal numbers are off by 2^-25 of a unit that is at least 2^-8 of the largest scale
  s: n keys, each 2^-33 s of the largest |z| + 15 s (s at most a fifteenth of that).  Then one
  rounding.
"""
from __future__ import annotations

import numpy as np
import pytest

from oct_b200 import reactor as R
from oracle import serving as O

pytestmark = pytest.mark.gpu

TYPES = {"f32": ("float32", 2.0 ** -24), "bf16": ("bfloat16", 2.0 ** -8), "f16": ("float16", 2.0 ** -11)}


def _torch(x, kind="f32"):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).cuda().to(getattr(torch, TYPES[kind][0]))


def _np(x):
    return x.double().cpu().numpy()


def _int(x):
    import torch
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def _ok(runtime):
    import torch
    torch.cuda.synchronize()
    status = runtime.sync_status()
    assert status.ok, status


def _near(got, want, tol, what=""):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], want[bad][:4], np.broadcast_to(tol, got.shape)[bad][:4])


# ------------------------------------------------------------------ head norm + rotation
def _rotation_case(kind, tokens, heads, kv_heads, dim, rotary, axes, interleaved, normalize, weights, far, seed):
    rng = np.random.default_rng(seed)
    x = _torch(rng.standard_normal((tokens, heads + 2 * kv_heads, dim)) * 3.0, kind)
    pairs = rotary // 2
    axis_pairs = [pairs // axes] * axes
    axis_pairs[-1] += pairs - sum(axis_pairs)
    freq = np.concatenate([10000.0 ** (-np.arange(n) / max(n, 1)) for n in axis_pairs])
    pos = rng.integers(-far, far + 1, (tokens, axes)).astype(np.int32)
    w = [rng.uniform(0.5, 1.5, dim).astype(np.float32) if weights else None for _ in range(2)]
    return x, axis_pairs, freq, pos, w


def _check_rotation(kind, got, x, pos, freq, axis_pairs, interleaved, weight, normalize, eps=1e-6):
    u = TYPES[kind][1]
    x = _np(x)
    weight = None if weight is None else weight.astype(np.float64)
    want = O.qk_norm_rope(x, pos, freq, axis_pairs, interleaved, weight, eps, normalize)
    size = np.abs(O.norm(x, weight, eps) if normalize else x)
    ca, cb = O.pair_channels(2 * len(freq), interleaved)
    both = size.copy()
    both[..., ca] = both[..., cb] = size[..., ca] + size[..., cb]
    tiny = 2.0 ** -25 if kind == "f16" else 0.0
    _near(_np(got), want, u * np.abs(want) * 1.01 + 32 * 2.0 ** -24 * both + tiny)


ROTATIONS = [
    # kind, tokens, heads, kv, dim, rotary, axes, interleaved, normalize, weights, far
    ("bf16", 1, 8, 1, 256, 256, 1, False, True, True, 131071),
    ("f32", 37, 8, 1, 256, 256, 1, False, True, True, 1000000),
    ("f16", 129, 3, 3, 128, 128, 3, True, True, True, 64),
    ("bf16", 300, 24, 24, 128, 128, 3, True, True, True, 64),
    ("f32", 5, 5, 1, 80, 32, 1, False, True, False, 2147483647),
    ("f16", 9, 7, 7, 96, 48, 2, True, True, True, 4096),
    ("bf16", 3, 2, 1, 16, 16, 1, False, True, True, 10),
    ("f32", 2, 1, 1, 512, 512, 4, False, True, True, 99),
    ("f32", 11, 4, 2, 64, 32, 4, True, False, False, 300000),
    ("bf16", 5000, 2, 1, 64, 64, 2, False, True, True, 77),
    ("f16", 20001, 1, 1, 48, 16, 1, True, True, False, 20000),
]


@pytest.mark.parametrize("case", ROTATIONS, ids=lambda c: "-".join(map(str, c)))
def test_rotation_matches_oracle(runtime, case):
    import torch
    kind, tokens, heads, kv, dim, rotary, axes, inter, normalize, weights, far = case
    x, axis_pairs, freq, pos, w = _rotation_case(*case, seed=tokens)
    q, k = x[:, :heads], x[:, heads:heads + kv]  # slices of one projection
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    runtime.qk_norm_rope_device(q, k, qo, ko, _int(pos), torch.from_numpy(freq).cuda(), axis_pairs=axis_pairs,
                                interleaved=inter, normalize=normalize,
                                q_weight=None if w[0] is None else _torch(w[0]),
                                k_weight=None if w[1] is None else _torch(w[1]))
    _ok(runtime)
    _check_rotation(kind, qo, q, pos, freq, axis_pairs, inter, w[0], normalize)
    _check_rotation(kind, ko, k, pos, freq, axis_pairs, inter, w[1], normalize)


def test_rotation_in_place_leaves_the_rest_of_the_projection(runtime):
    import torch
    x, axis_pairs, freq, pos, w = _rotation_case("bf16", 33, 4, 2, 128, 64, 1, False, True, True, 5000, 3)
    before = x.clone()
    q, k = x[:, :4], x[:, 4:6]
    runtime.qk_norm_rope_device(q, k, q, k, _int(pos[:, 0]), torch.from_numpy(freq).cuda(), q_weight=_torch(w[0]),
                                k_weight=_torch(w[1]))
    _ok(runtime)
    assert torch.equal(x[:, 6:], before[:, 6:])
    _check_rotation("bf16", q, before[:, :4], pos, freq, axis_pairs, False, w[0], True)
    _check_rotation("bf16", k, before[:, 4:6], pos, freq, axis_pairs, False, w[1], True)


def test_rotation_of_head_major_rows_and_of_queries_alone(runtime):
    import torch
    x, axis_pairs, freq, pos, w = _rotation_case("f32", 21, 6, 0, 64, 64, 1, False, True, True, 5000, 4)
    q = x.transpose(0, 1).contiguous().transpose(0, 1)  # [heads][tokens][dim] in memory
    out = torch.empty_strided(q.shape, (80, 21 * 80, 1), device="cuda")
    runtime.qk_norm_rope_device(q, None, out, None, _int(pos), torch.from_numpy(freq).cuda(), q_weight=_torch(w[0]))
    _ok(runtime)
    _check_rotation("f32", out, q, pos, freq, axis_pairs, False, w[0], True)


def test_rotation_of_zeros_and_of_one_bad_row(runtime):
    import torch
    x, axis_pairs, freq, pos, w = _rotation_case("f32", 6, 2, 1, 128, 128, 1, False, True, True, 50, 5)
    q, k = x[:, :2], x[:, 2:3]
    q[1] = 0.0
    q[2, 1, 5] = float("nan")
    q[3, 0, 0] = float("inf")
    want_bad = np.zeros((6, 2), bool)
    want_bad[2, 1] = want_bad[3, 0] = True
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    runtime.qk_norm_rope_device(q, k, qo, ko, _int(pos), torch.from_numpy(freq).cuda())
    _ok(runtime)
    got = _np(qo)
    assert (got[1] == 0).all()
    assert np.array_equal(np.isnan(got).any(-1), want_bad)


def test_rotation_refuses_what_it_cannot_address(runtime):
    import torch
    q = torch.zeros((4, 2, 64), device="cuda")
    pos, freq = _int(np.zeros(4)), torch.ones(32, dtype=torch.float64, device="cuda")
    with pytest.raises(TypeError):
        runtime.qk_norm_rope_device(q.double(), None, q.double(), None, pos, freq)
    with pytest.raises(TypeError):
        runtime.qk_norm_rope_device(q, None, q.half(), None, pos, freq)
    with pytest.raises(TypeError):
        runtime.qk_norm_rope_device(q, None, q, None, pos.long(), freq)
    with pytest.raises(ValueError):
        runtime.qk_norm_rope_device(q, None, q[:3], None, pos, freq)
    with pytest.raises(ValueError):
        runtime.qk_norm_rope_device(q, None, q, None, pos[:3], freq)
    with pytest.raises(ValueError):
        runtime.qk_norm_rope_device(q, None, q, None, pos, freq, axis_pairs=(16, 16))
    with pytest.raises(ValueError):
        runtime.qk_norm_rope_device(q.transpose(1, 2), None, q.transpose(1, 2), None, pos, freq)
    with pytest.raises(RuntimeError, match="detail=-7008"):
        runtime.qk_norm_rope_device(q, None, q, None, pos, freq, axis_pairs=(31,))
    with pytest.raises(RuntimeError, match="detail=-7005"):
        flat = torch.zeros(4 * 2 * 64 + 1, device="cuda")
        odd = flat[1:].view(4, 2, 64)
        runtime.qk_norm_rope_device(odd, None, odd, None, pos, freq)


# ------------------------------------------------------------------ the cache
class Host:
    """Sequences, their pages in no order, and a cache full of bytes that mean nothing."""

    def __init__(self, rng, dim, kv_heads, page, new, held, fill=0xFF):
        self.dim, self.kv_heads, self.page, self.new, self.held = dim, kv_heads, page, list(new), list(held)
        width = max(1, -(-max(held) // page))
        order = rng.permutation(len(held) * width + 2)
        self.table = order[: len(held) * width].reshape(len(held), width).astype(np.int32)
        self.cache = O.Cache(len(order), page, kv_heads, dim, fill=fill)
        self.starts = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)

    def fill(self, rng, scale=1.0):
        """Rows for every held position, as the oracle writes them."""
        for b, n in enumerate(self.held):
            for p in range(n):
                for h in range(self.kv_heads):
                    for which in (0, 1):
                        self.cache.write(self.table[b, p // self.page], p % self.page, h, which,
                                         np.float32(rng.standard_normal(self.dim) * scale).astype(np.float64))

    def device(self):
        import torch
        return R.Kv4Cache(torch.from_numpy(self.cache.data.copy()).cuda(), page_size=self.page, kv_heads=self.kv_heads,
                          head_dim=self.dim)

    def batch(self, cu=True, max_tokens=None, max_kv_len=None):
        return R.Kv4Batch(_int(self.table), _int(self.held), _int(self.starts) if cu else None,
                          max_tokens=max(1, max(self.new)) if max_tokens is None else max_tokens,
                          max_kv_len=max_kv_len, page_size=self.page)


def _same_parts(got: np.ndarray, host: Host, want: O.Cache):
    """Codes, scales and zeros of two caches, as numbers (zeros of either sign are the same)."""
    have = O.Cache(want.pages, want.page_size, want.kv_heads, want.dim)
    have.data = got
    for b, n in enumerate(host.held):
        for p in range(n):
            for h in range(host.kv_heads):
                for which in (0, 1):
                    at = (int(host.table[b, p // host.page]), p % host.page, h, which)
                    for x, y in zip(have.parts(*at), want.parts(*at)):
                        assert np.array_equal(x, y, equal_nan=True), (at, x, y)


def _difficult_rows(rng, rows, dim):
    x = rng.standard_normal((rows, dim)) * 10.0 ** rng.integers(-8, 5, (rows, dim // 32)).repeat(32, axis=-1)
    flat = x.reshape(-1, 32)
    kind = rng.integers(0, 10, len(flat))
    flat[kind == 0] = 0.0
    flat[kind == 1] = 1.0 / 3.0
    flat[kind == 2] = rng.integers(-40, 41, (int((kind == 2).sum()), 32)) / 8.0  # ties between codes
    flat[kind == 3] += 1000.0
    flat[kind == 4] *= 1e-7
    flat[kind == 5, 3] = np.inf
    flat[kind == 5, 9] = -1e30
    flat[kind == 6, 17] = np.nan
    return x


CACHES = [
    # kind, dim, kv heads, page, new rows, held
    ("bf16", 128, 2, 32, [1, 1, 1], [1, 16, 33]),
    ("f32", 64, 1, 16, [0, 5, 17, 40], [0, 5, 20, 47]),
    ("f16", 256, 3, 64, [2, 0, 31], [100, 7, 31]),
    ("bf16", 256, 1, 48, [70], [130]),
    ("f32", 128, 5, 256, [1], [1]),
    ("f16", 64, 2, 16, [33, 1], [33, 300]),
]


@pytest.mark.parametrize("case", CACHES, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}-{c[3]}-{sum(c[4])}")
def test_store_then_load(runtime, case):
    import torch
    kind, dim, kv, page, new, held = case
    rng = np.random.default_rng(dim + kv)
    host = Host(rng, dim, kv, page, new, held)
    dev = host.device()
    total = sum(new) + 3  # three rows behind the last sequence
    rows = [_torch(_difficult_rows(rng, total * kv, dim).reshape(total, kv, dim), kind) for _ in range(2)]
    k = torch.cat([rows[0], rows[1]], dim=1)[:, :kv]  # a slice of a wider projection
    v = rows[1].transpose(0, 1).contiguous().transpose(0, 1)  # head-major
    batch = host.batch()
    runtime.kv4_store_device(dev, batch, k, v)
    k_back, v_back = torch.full_like(rows[0], 7.0), torch.full_like(rows[1], 7.0)
    runtime.kv4_load_device(dev, batch, k_back, v_back)
    _ok(runtime)
    for b, n in enumerate(new):
        for i in range(n):
            p = held[b] - n + i
            for h in range(kv):
                for which, src in ((0, k), (1, v)):
                    host.cache.write(host.table[b, p // page], p % page, h, which, _np(src[host.starts[b] + i, h]))
    # every byte that no row owns is untouched; what the rows own has the definition's numbers
    got = dev.data.cpu().numpy()
    _same_parts(got, host, host.cache)
    owned = np.zeros(host.cache.data.shape, bool)
    probe = O.Cache(host.cache.pages, page, kv, dim)
    probe.data = owned.view(np.uint8)
    for b, n in enumerate(new):
        for p in range(held[b] - n, held[b]):
            for h in range(kv):
                for which in (0, 1):
                    for part in probe._at(int(host.table[b, p // page]), h, p % page, which):
                        part[:] = 1
    assert np.array_equal(got[~owned], np.full((~owned).sum(), 0xFF, np.uint8))
    u = TYPES[kind][1]
    for back, src in ((k_back, k), (v_back, v)):
        used = int(host.starts[-1])
        assert (_np(back[used:]) == 7.0).all()
        want = O.values(*O.quantise(_np(src[:used])))
        with np.errstate(over="ignore"):
            typed = np.where(np.isnan(want), 0.0, want)
        have = _np(back[:used])
        assert np.array_equal(np.isnan(have), np.isnan(want))
        _near(np.where(np.isnan(want), 0.0, have), typed, (u + 2.0 ** -23) * np.abs(typed) + (2.0 ** -25 if kind == "f16" else 0.0))


def test_store_without_row_offsets_is_one_row_per_sequence(runtime):
    import torch
    rng = np.random.default_rng(2)
    host = Host(rng, 128, 2, 16, [1, 1, 1, 1], [9, 1, 0, 40])
    host.new[2] = 0  # a sequence that holds nothing cannot take a row: reported, the others written
    dev = host.device()
    k, v = (_torch(rng.standard_normal((4, 2, 128)), "bf16") for _ in range(2))
    runtime.kv4_store_device(dev, host.batch(cu=False, max_tokens=1), k, v)
    torch.cuda.synchronize()
    assert runtime.sync_status().detail == R.DETAIL_KV4_BAD_INDEX
    assert runtime.sync_status().ok  # reported once
    for b in (0, 1, 3):
        p = host.held[b] - 1
        for h in range(2):
            host.cache.write(host.table[b, p // 16], p % 16, h, 0, _np(k[b, h]))
            host.cache.write(host.table[b, p // 16], p % 16, h, 1, _np(v[b, h]))
    assert np.array_equal(np.nan_to_num(dev.data.cpu().numpy()), host.cache.data)


def test_indices_out_of_range_are_skipped_and_reported(runtime):
    """Every index below is checked by the kernels before it is used."""
    import torch
    rng = np.random.default_rng(3)
    host = Host(rng, 64, 1, 16, [2, 2, 2, 2], [20, 20, 20, 20])
    host.fill(rng)
    good = host.table.copy()
    k, v = (_torch(rng.standard_normal((8, 1, 64)), "f32") for _ in range(2))

    def run(table=None, held=None, starts=None, max_kv_len=None):
        host.table, keep = (good if table is None else table), host.table
        dev = host.device()
        batch = R.Kv4Batch(_int(host.table), _int(host.held if held is None else held),
                           _int(host.starts if starts is None else starts), max_tokens=2,
                           max_kv_len=32 if max_kv_len is None else max_kv_len)
        runtime.kv4_store_device(dev, batch, k, v)
        torch.cuda.synchronize()
        status = runtime.sync_status().detail
        back = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
        runtime.kv4_load_device(dev, batch, *back)
        out, lse = torch.full((8, 2, 64), 7.0, device="cuda"), torch.full((8, 2), 7.0, device="cuda")
        q = torch.ones((8, 2, 64), device="cuda")
        ws = torch.empty(runtime.kv4_attention_workspace_bytes(dev, batch, q), dtype=torch.uint8, device="cuda")
        runtime.kv4_attention_device(dev, batch, q, out, lse=lse, workspace=ws)
        torch.cuda.synchronize()
        assert status == runtime.sync_status().detail
        host.table = keep
        return status, _np(back[0])[:, 0, 0] != 7.0, _np(lse)[:, 0] != 7.0

    everyone = np.ones(8, bool)
    status, stored, seen = run()
    assert status == 0 and (stored == everyone).all() and (seen == everyone).all()
    for value in (-1, host.cache.pages, 2 ** 31 - 1, -2 ** 31):
        bad = good.copy()
        bad[1, 1] = value  # the page of its new rows
        status, stored, seen = run(table=bad)
        assert status == R.DETAIL_KV4_BAD_INDEX
        assert (stored == np.array([1, 1, 0, 0, 1, 1, 1, 1], bool)).all()
        assert (seen == everyone).all()  # over the keys of its other page
    for value in (-1, 33, 2 ** 31 - 1, -2 ** 31):
        status, stored, seen = run(held=[20, 20, value, 20])
        want = np.array([1, 1, 1, 1, 0, 0, 1, 1], bool)
        assert status == R.DETAIL_KV4_BAD_INDEX and (stored == want).all() and (seen == want).all()
    for starts, want in (([0, 2, 4, 6, 9], [1, 1, 1, 1, 1, 1, 0, 0]), ([0, 3, 4, 6, 8], [0, 0, 0, 1, 1, 1, 1, 1]),
                         ([-2, 0, 4, 6, 8], [0, 0, 0, 0, 1, 1, 1, 1]), ([0, 2, 1, 3, 5], [1, 1, 1, 1, 1, 0, 0, 0])):
        status, stored, seen = run(starts=starts)
        assert status == R.DETAIL_KV4_BAD_INDEX, starts
        assert (stored == np.array(want, bool)).all() and (seen == np.array(want, bool)).all(), starts


# ------------------------------------------------------------------ attention
def _attend(runtime, host, q, heads, *, window=0, causal=True, scale=None, stream=None, dev=None, batch=None, rows=None):
    import torch
    dev = host.device() if dev is None else dev
    batch = host.batch() if batch is None else batch
    out = torch.full_like(q, 7.0)
    lse = torch.full(q.shape[:2], 7.0, device="cuda", dtype=torch.float32)
    ws = torch.empty(runtime.kv4_attention_workspace_bytes(dev, batch, q, causal=causal, window=window),
                     dtype=torch.uint8, device="cuda")
    runtime.kv4_attention_device(dev, batch, q, out, scale=scale, causal=causal, window=window, lse=lse, workspace=ws,
                                 stream=stream)
    return out, lse, ws


def _check_attention(host, kind, q, out, lse, *, window=0, causal=True, scale=None, sequences=None):
    u = TYPES[kind][1]
    scale = float(np.float32(1.0) / np.sqrt(np.float32(host.dim))) if scale is None else float(np.float32(scale))
    got, got_lse, qn = _np(out), _np(lse), _np(q)
    for b in range(len(host.held)) if sequences is None else sequences:
        sl = slice(int(host.starts[b]), int(host.starts[b + 1]))
        if sl.start == sl.stop:
            continue
        want, want_lse, weight, reach, largest = O.attention(host.cache, host.table[b], host.held[b], qn[sl], scale, causal, window)
        n = host.held[b]
        d = 2.0 ** -20 * reach + 2.0 ** -21
        rel = 2 * d + 2.0 ** -21 + (2.0 ** -11 if kind == "bf16" else 2.0 ** -21) + (n / 16 + 48) * 2.0 ** -24
        nan = np.isnan(want)
        assert np.array_equal(np.isnan(got[sl]), nan), b
        tiny = (2.0 ** -25 if kind == "f16" else 0.0) + n * 2.0 ** -33 * largest ** 2 / 15
        _near(np.where(nan, 0, got[sl]), np.where(nan, 0, want),
              np.where(nan, 0, u * np.abs(want) * 1.01 + rel[..., None] * weight + tiny), f"sequence {b}")
        nan = np.isnan(want_lse)
        empty = want_lse == -np.inf
        assert np.array_equal(got_lse[sl] == -np.inf, empty) and np.array_equal(np.isnan(got_lse[sl]), nan)
        plain = ~(nan | empty)
        _near(got_lse[sl][plain], want_lse[plain], (d + 2.0 ** -22 * np.abs(want_lse) + (n / 16 + 48) * 2.0 ** -24)[plain])
    used = int(host.starts[-1])
    if sequences is None:
        assert (got[used:] == 7.0).all() and (got_lse[used:] == 7.0).all()


ATTENTIONS = [
    # kind, dim, kv heads, query heads per key head, page, queries, held, window, causal
    ("bf16", 128, 2, 4, 16, [1] * 6, [1, 15, 16, 17, 63, 200], 0, True),
    ("f32", 64, 1, 1, 32, [1, 1, 1, 1], [0, 1, 33, 129], 0, True),
    ("f16", 256, 1, 8, 64, [1, 1], [700, 64], 0, True),
    ("f32", 256, 1, 8, 16, [4, 4, 4], [4, 100, 333], 50, True),
    ("bf16", 64, 3, 7, 48, [3, 0, 5, 1], [3, 8, 77, 1], 0, True),
    ("f16", 128, 1, 16, 16, [2, 3], [150, 18], 1, True),
    ("f32", 128, 2, 3, 32, [6, 1], [41, 90], 17, True),
    ("bf16", 256, 2, 1, 16, [9, 2], [5, 40], 0, True),   # more queries than keys: the first see nothing
    ("f16", 64, 1, 32, 16, [2, 1], [65, 64], 0, False),
    ("f32", 128, 1, 20, 256, [3], [50], 0, False),
    ("bf16", 128, 1, 8, 16, [40], [100], 30, True),
]


@pytest.mark.parametrize("case", ATTENTIONS, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}x{c[3]}-q{max(c[5])}-w{c[7]}-{c[8]}")
def test_attention_matches_oracle(runtime, case):
    kind, dim, kv, share, page, new, held, window, causal = case
    rng = np.random.default_rng(dim + share)
    host = Host(rng, dim, kv, page, new, held)  # memory outside the held rows is NaN bits
    host.fill(rng)
    q = _torch(rng.standard_normal((sum(new) + 2, kv * share, dim)), kind)
    out, lse, _ = _attend(runtime, host, q, kv * share, window=window, causal=causal)
    _ok(runtime)
    _check_attention(host, kind, q, out, lse, window=window, causal=causal)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("magnitude", [1e-6, 1e-3, 30.0, 3000.0])
def test_attention_holds_over_magnitudes(runtime, kind, magnitude):
    """Small and large keys, values and queries; the scale keeps the scores moderate."""
    rng = np.random.default_rng(7)
    host = Host(rng, 128, 1, 16, [1, 2], [130, 70])
    host.fill(rng, magnitude)
    q = _torch(rng.standard_normal((3, 4, 128)) * min(magnitude, 100.0), kind)
    scale = 0.3 / np.sqrt(128.0) / magnitude / min(magnitude, 100.0)
    out, lse, _ = _attend(runtime, host, q, 4, scale=scale)
    _ok(runtime)
    _check_attention(host, kind, q, out, lse, scale=scale)


def test_attention_values_that_grow_and_shrink_along_the_keys(runtime):
    """The scale of the weights is renewed as larger values appear; zeros come first."""
    rng = np.random.default_rng(8)
    host = Host(rng, 64, 1, 16, [1, 1], [400, 400])
    host.fill(rng)
    for p in range(400):
        for b, size in ((0, 0.0 if p < 130 else 1e-5 * 1.08 ** (p - 130)), (1, 1e4 * 0.95 ** p)):
            host.cache.write(host.table[b, p // 16], p % 16, 0, 1, np.float32(rng.standard_normal(64) * size).astype(float))
    for kind in TYPES:
        q = _torch(rng.standard_normal((2, 3, 64)), kind)
        out, lse, _ = _attend(runtime, host, q, 3)
        _ok(runtime)
        _check_attention(host, kind, q, out, lse)


def test_attention_scores_that_rise_along_the_keys(runtime):
    rng = np.random.default_rng(9)
    host = Host(rng, 64, 1, 16, [1], [500])
    host.fill(rng)
    direction = rng.standard_normal(64)
    for p in range(500):
        host.cache.write(host.table[0, p // 16], p % 16, 0, 0, np.float32(direction * (p / 40.0)).astype(float))
    q = _torch(np.stack([direction, -direction, 8 * direction])[None], "f32")
    out, lse, _ = _attend(runtime, host, q, 3)
    _ok(runtime)
    _check_attention(host, "f32", q, out, lse)


@pytest.mark.parametrize("kind", list(TYPES))
def test_a_bad_key_or_value_reaches_only_the_rows_that_see_it(runtime, kind):
    rng = np.random.default_rng(10)
    host = Host(rng, 64, 1, 16, [4, 4], [70, 70])
    host.fill(rng)
    bad = np.full(64, 1.0)
    bad[40] = np.nan  # the second group of 32 channels
    host.cache.write(host.table[0, 68 // 16], 68 % 16, 0, 1, bad)  # a value that queries 2 and 3 see
    host.cache.write(host.table[1, 69 // 16], 69 % 16, 0, 0, bad)  # a key that query 3 sees
    q = _torch(rng.standard_normal((8, 2, 64)), kind)
    q[0, 1, 3] = float("nan")
    out, lse, _ = _attend(runtime, host, q, 2)
    _ok(runtime)
    got = np.isnan(_np(out))
    assert got[0, 1].all() and not got[0, 0].any() and not got[1].any()
    assert got[2:4, :, 32:].all() and not got[2:4, :, :32].any()
    assert not got[4:7].any() and got[7].all()
    _check_attention(host, kind, q, out, lse)


def test_attention_of_strided_rows(runtime):
    import torch
    rng = np.random.default_rng(11)
    host = Host(rng, 128, 2, 16, [2, 1], [37, 18])
    host.fill(rng)
    wide = _torch(rng.standard_normal((3, 12, 128)), "bf16")
    q = wide[:, 2:10]
    dev, batch = host.device(), host.batch()
    out = torch.empty_strided((3, 8, 128), (136, 3 * 136, 1), dtype=torch.bfloat16, device="cuda")  # head-major, padded
    runtime.kv4_attention_device(dev, batch, q, out)
    _ok(runtime)
    plain, lse, _ = _attend(runtime, host, q.contiguous(), 8)
    _ok(runtime)
    assert torch.equal(out, plain)
    _check_attention(host, "bf16", q, out, lse)


def _wide(host):
    """The same sequences in a table of many more pages (no pages of the cache): their keys are spread over the GPU."""
    table = np.full((len(host.held), (1 << 18) // host.page), -1, np.int32)
    table[:, : host.table.shape[1]] = host.table
    return R.Kv4Batch(_int(table), _int(host.held), _int(host.starts), max_tokens=max(1, max(host.new)), page_size=host.page)


@pytest.mark.parametrize("kind", list(TYPES))
def test_split_keys_join_to_the_same_result(runtime, kind):
    """A long table makes the host plan many splits; short and empty sequences use few of them."""
    rng = np.random.default_rng(12)
    host = Host(rng, 64, 1, 16, [1, 1, 1, 3], [3000, 0, 5, 260])
    host.fill(rng)
    q = _torch(rng.standard_normal((8, 4, 64)), kind)
    dev, batch = host.device(), _wide(host)
    assert runtime.kv4_attention_workspace_bytes(dev, batch, q) > 0
    out, lse, _ = _attend(runtime, host, q, 4, dev=dev, batch=batch)
    again, lse2, _ = _attend(runtime, host, q, 4, dev=dev, batch=batch)
    _ok(runtime)
    import torch
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    _check_attention(host, kind, q, out, lse)


@pytest.mark.parametrize("case", [c for c in ATTENTIONS if c[7] == 0],
                         ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}x{c[3]}-q{max(c[5])}-{c[8]}")
def test_spread_keys_match_oracle(runtime, case):
    kind, dim, kv, share, page, new, held, _, causal = case
    rng = np.random.default_rng(dim + share)
    host = Host(rng, dim, kv, page, new, held)
    host.fill(rng)
    q = _torch(rng.standard_normal((sum(new) + 2, kv * share, dim)), kind)
    batch = _wide(host)
    assert runtime.kv4_attention_workspace_bytes(host.device(), batch, q, causal=causal) > 0
    out, lse, _ = _attend(runtime, host, q, kv * share, causal=causal, batch=batch)
    _ok(runtime)
    _check_attention(host, kind, q, out, lse, causal=causal)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim, sequences, longest, heads", [
    (64, 1, 400, 2), (64, 120, 400, 3), (64, 1, 2300, 8), (64, 40, 1100, 20), (128, 1, 1500, 8), (128, 30, 700, 9),
    (256, 1, 1000, 5), (256, 20, 520, 8), (256, 70, 300, 12),
])
def test_clusters_of_every_size_join_their_parts(runtime, kind, dim, sequences, longest, heads):
    """One long sequence beside short and empty ones: blocks of a cluster without a part, and none with one.
    (40 sequences of 1100 keys are spread over the GPU in fp32, whose blocks take fewer units.)"""
    rng = np.random.default_rng(dim + sequences + longest)
    held = [longest] + [int(x) for x in rng.integers(0, 20, sequences - 1)]
    host = Host(rng, dim, 1, 16, [1] * sequences, held)
    host.fill(rng)
    q = _torch(rng.standard_normal((sequences, heads, dim)), kind)
    dev, batch = host.device(), host.batch()
    out, lse, _ = _attend(runtime, host, q, heads, dev=dev, batch=batch)
    again, lse2, _ = _attend(runtime, host, q, heads, dev=dev, batch=batch)
    _ok(runtime)
    import torch
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    _check_attention(host, kind, q, out, lse)


def test_captured_step_follows_lengths_and_pages_on_the_device(runtime):
    """Two graphs with a workspace each, replayed on two streams while the lengths grow."""
    import torch
    rng = np.random.default_rng(13)
    host = Host(rng, 64, 1, 16, [1, 1], [1500, 700])
    host.fill(rng)
    dev, batch = host.device(), host.batch()
    qs = [_torch(rng.standard_normal((2, 4, 64)), "bf16") for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, results, keep = [], [], []
    for q, s in zip(qs, streams):
        out, lse, ws = _attend(runtime, host, q, 4, dev=dev, batch=batch)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            runtime.kv4_attention_device(dev, batch, q, out, lse=lse, workspace=ws, stream=s)
        graphs.append(g)
        results.append((out, lse))
        keep.append(ws)
    for held in ([1500, 700], [3, 699], [1490, 0]):
        batch.kv_lens.copy_(_int(held))
        torch.cuda.synchronize()
        for _ in range(3):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        _ok(runtime)
        host.held = held
        for q, (out, lse) in zip(qs, results):
            _check_attention(host, "bf16", q, out, lse)


def test_attention_refuses_a_missing_workspace_and_foreign_types(runtime):
    import torch
    rng = np.random.default_rng(14)
    host = Host(rng, 64, 1, 16, [1], [20000])  # more keys than one cluster of blocks takes
    dev, batch = host.device(), host.batch()
    q = torch.zeros((1, 4, 64), device="cuda")
    out = torch.full_like(q, 7.0)
    with pytest.raises(RuntimeError, match="detail=-7031"):
        runtime.kv4_attention_device(dev, batch, q, out)
    with pytest.raises(TypeError):
        runtime.kv4_attention_device(dev, batch, q, out.half())
    with pytest.raises(ValueError):
        runtime.kv4_attention_device(dev, batch, q[..., :32], out)
    with pytest.raises(RuntimeError, match="detail=-7008"):
        runtime.kv4_attention_device(dev, batch, q, out, causal=False, window=3)
    with pytest.raises(TypeError):
        R.Kv4Batch(_int(host.table).long(), _int([1]), max_kv_len=16)
    with pytest.raises(ValueError):
        R.Kv4Cache(dev.data.view(-1)[:-1].clone(), page_size=16, kv_heads=1, head_dim=64)
    torch.cuda.synchronize()
    assert (out == 7.0).all() and runtime.sync_status().ok


def test_attention_may_write_over_its_queries_and_take_any_scale(runtime):
    import torch
    rng = np.random.default_rng(16)
    host = Host(rng, 128, 2, 16, [1, 3], [900, 70])
    host.fill(rng)
    q = _torch(rng.standard_normal((4, 8, 128)), "bf16")
    dev, batch = host.device(), host.batch()
    ws = torch.empty(runtime.kv4_attention_workspace_bytes(dev, batch, q), dtype=torch.uint8, device="cuda")
    for scale in (0.07, -0.05, 0.0):
        out, lse, _ = _attend(runtime, host, q, 8, scale=scale, dev=dev, batch=batch)
        own = q.clone()
        runtime.kv4_attention_device(dev, batch, own, own, scale=scale, workspace=ws)
        _ok(runtime)
        assert torch.equal(own, out)
        _check_attention(host, "bf16", q, out, lse, scale=scale)


def test_many_short_sequences(runtime):
    """More sequences than thread blocks' threads, most of a few tokens, some of none."""
    rng = np.random.default_rng(17)
    held = [int(x) for x in rng.integers(0, 6, 700)]
    held[3], held[500] = 90, 40
    host = Host(rng, 64, 1, 16, [1] * 700, held)
    host.fill(rng)
    q = _torch(rng.standard_normal((700, 2, 64)), "f16")
    out, lse, _ = _attend(runtime, host, q, 2)
    _ok(runtime)
    _check_attention(host, "f16", q, out, lse)


def test_pages_of_the_largest_size_and_far_positions(runtime):
    import torch
    rng = np.random.default_rng(18)
    host = Host(rng, 64, 1, 65536, [3], [65536 + 40])
    dev, batch = host.device(), host.batch()
    k, v = (_torch(rng.standard_normal((3, 1, 64)), "f32") for _ in range(2))
    runtime.kv4_store_device(dev, batch, k, v)
    for i, p in enumerate(range(host.held[0] - 3, host.held[0])):
        host.cache.write(host.table[0, p // 65536], p % 65536, 0, 0, _np(k[i, 0]))
        host.cache.write(host.table[0, p // 65536], p % 65536, 0, 1, _np(v[i, 0]))
    q = _torch(rng.standard_normal((1, 3, 64)), "f32")
    one = R.Kv4Batch(_int(host.table), _int(host.held), max_kv_len=2 * 65536)
    out, lse, _ = _attend(runtime, host, q, 3, dev=dev, batch=one, window=3)
    _ok(runtime)
    got = dev.data.cpu().numpy()
    assert np.array_equal(got, host.cache.data)
    row = np.array([host.table[0, 1]])
    small = O.Cache(host.cache.pages, 65536, 1, 64)
    small.data = host.cache.data
    kk = np.stack([O.values(*small.parts(int(row[0]), p, 0, 0)) for p in range(37, 40)])
    vv = np.stack([O.values(*small.parts(int(row[0]), p, 0, 1)) for p in range(37, 40)])
    x = _np(q[0]) @ kk.T * float(np.float32(0.125))
    e = np.exp(x - x.max(-1, keepdims=True))
    want = e @ vv / e.sum(-1, keepdims=True)
    _near(_np(out[0]), want, 2.0 ** -15)  # |v| < 4: weights to 2^-18
    _near(_np(lse[0]), x.max(-1) + np.log(e.sum(-1)), 2.0 ** -17)


def test_cache_offsets_beyond_32_bits(runtime):
    """A cache of 6 GB; the sequence's pages lie at its end."""
    import torch
    dim, page, kv = 256, 256, 8
    pages = (6 << 30) // (kv * (page // 16) * R.kv4_tile_bytes(dim))
    data = torch.zeros((pages, kv * (page // 16) * R.kv4_tile_bytes(dim)), dtype=torch.uint8, device="cuda")
    dev = R.Kv4Cache(data, page_size=page, kv_heads=kv, head_dim=dim)
    n = 300
    g = torch.Generator("cuda").manual_seed(1)
    k, v, q = (torch.randn((n, h, dim), device="cuda", generator=g) for h in (kv, kv, kv))
    small = R.Kv4Cache(torch.zeros((2, data.shape[1]), dtype=torch.uint8, device="cuda"), page_size=page, kv_heads=kv,
                       head_dim=dim)
    results = []
    for cache, table in ((dev, [[pages - 1, pages - 2]]), (small, [[1, 0]])):
        batch = R.Kv4Batch(_int(table), _int([n]), _int([0, n]), max_tokens=n, page_size=page)
        runtime.kv4_store_device(cache, batch, k, v)
        back = torch.empty_like(k), torch.empty_like(v)
        runtime.kv4_load_device(cache, batch, *back)
        one = R.Kv4Batch(_int(table), _int([n]), page_size=page)
        out = torch.empty_like(q[:1])
        ws = torch.empty(runtime.kv4_attention_workspace_bytes(cache, one, q[:1]), dtype=torch.uint8, device="cuda")
        runtime.kv4_attention_device(cache, one, q[:1], out, workspace=ws)
        _ok(runtime)
        results.append((*back, out))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    assert not data[: pages - 2].any()
    assert torch.equal(data[pages - 2:], small.data)
    assert (results[0][0] - k).abs().max() <= 0.5  # steps of at most (max - min) / 15 < 10 / 15 and a bit


def test_a_decode_step_captured_on_its_first_call(lib):
    """A new process's first calls are under capture: nothing is loaded, set up or allocated before."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import torch
from oct_b200 import reactor as R
rt = R.Runtime()
g = torch.Generator('cuda').manual_seed(3)
data = torch.zeros((8, 2 * R.kv4_tile_bytes(64)), dtype=torch.uint8, device='cuda')
cache = R.Kv4Cache(data, page_size=32, kv_heads=1, head_dim=64)
lens = torch.zeros(2, dtype=torch.int32, device='cuda')
table = torch.arange(8, dtype=torch.int32, device='cuda').view(2, 4)
batch = R.Kv4Batch(table, lens, page_size=32)
x = torch.zeros((2, 6, 64), dtype=torch.float16, device='cuda')
out = torch.zeros((2, 4, 64), dtype=torch.float16, device='cuda')
pos = torch.zeros((2, 1), dtype=torch.int32, device='cuda')
freq = torch.logspace(0, -4, 32, dtype=torch.float64, device='cuda')
ws = torch.empty(rt.kv4_attention_workspace_bytes(cache, batch, x[:, :4]), dtype=torch.uint8, device='cuda')
s = torch.cuda.Stream()

def step(stream):
    rt.qk_norm_rope_device(x[:, :4], x[:, 4:5], x[:, :4], x[:, 4:5], pos, freq, stream=stream)
    rt.kv4_store_device(cache, batch, x[:, 4:5], x[:, 5:], stream=stream)
    rt.kv4_attention_device(cache, batch, x[:, :4], out, workspace=ws, stream=stream)

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=s):
    step(s)
inputs = [torch.randn(x.shape, device='cuda', generator=g).half() for _ in range(100)]
outs = []
for run in (lambda: graph.replay(), lambda: step(None)):
    data.zero_()
    got = []
    for i, y in enumerate(inputs):
        x.copy_(y); pos.fill_(i); lens.fill_(i + 1)
        torch.cuda.synchronize()
        run()
        torch.cuda.synchronize()
        got.append(out.clone())
    outs.append(torch.stack(got))
    assert rt.sync_status().ok
assert torch.equal(outs[0], outs[1])
assert outs[0].isfinite().all() and outs[0].abs().amax() > 0.1
del graph
rt.close()
print('captured')
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parents[1], capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr


def test_calls_at_once_on_two_streams(runtime):
    """Two sequences' decode steps on streams of their own, each with its workspace and its cache pages."""
    import torch
    rng = np.random.default_rng(19)
    hosts = [Host(rng, 128, 1, 16, [1], [1200]) for _ in range(2)]
    streams, parts = [torch.cuda.Stream() for _ in range(2)], []
    for h in hosts:
        h.fill(rng)
        q = _torch(rng.standard_normal((1, 8, 128)), "bf16")
        dev, batch = h.device(), h.batch()
        ws = torch.empty(runtime.kv4_attention_workspace_bytes(dev, batch, q), dtype=torch.uint8, device="cuda")
        parts.append((dev, batch, q, torch.full_like(q, 7.0), torch.empty((1, 8), device="cuda"), ws))
    torch.cuda.synchronize()
    for _ in range(20):
        for (dev, batch, q, out, lse, ws), s in zip(parts, streams):
            runtime.kv4_attention_device(dev, batch, q, out, lse=lse, workspace=ws, stream=s)
    _ok(runtime)
    for h, (_, _, q, out, lse, _) in zip(hosts, parts):
        _check_attention(h, "bf16", q, out, lse)


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_a_prompt_and_decode_steps_as_they_are_used(runtime, kind):
    """Projection -> norm and rotation -> store -> attention, a prompt and then single tokens, against
    the oracle fed with the rounded tensors of each step."""
    import torch
    rng = np.random.default_rng(15)
    heads, kv, dim, page = 8, 1, 256, 16
    prompts = [19, 1, 0]
    host = Host(rng, dim, kv, page, prompts, [64, 64, 64])
    dev = host.device()
    table, freq = _int(host.table), 10000.0 ** (-np.arange(128) / 128)
    dfreq = torch.from_numpy(freq).cuda()
    weight = rng.uniform(0.5, 1.5, dim).astype(np.float32)
    held = np.zeros(3, int)
    for step, new in enumerate([prompts, [1, 1, 1], [1, 0, 1], [3, 2, 1]]):
        host.new = list(new)
        host.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        held = held + np.array(new)
        host.held = [int(h) for h in held]
        total = sum(new)
        x = _torch(rng.standard_normal((total, heads + 2 * kv, dim)), kind)
        pos = np.concatenate([np.arange(h - n, h) for h, n in zip(held, new)]).astype(np.int32)[:, None]
        q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
        before = x.clone()
        runtime.qk_norm_rope_device(q, k, q, k, _int(pos), dfreq, q_weight=_torch(weight), k_weight=_torch(weight))
        batch = R.Kv4Batch(table, _int(host.held), _int(host.starts), max_tokens=max(new), page_size=page)
        runtime.kv4_store_device(dev, batch, k, v)
        out, lse, _ = _attend(runtime, host, q, heads, dev=dev, batch=batch)
        _ok(runtime)
        _check_rotation(kind, q, before[:, :heads], pos, freq, [128], False, weight, True)
        _check_rotation(kind, k, before[:, heads:heads + kv], pos, freq, [128], False, weight, True)
        for b, n in enumerate(new):
            for i in range(n):
                p = host.held[b] - n + i
                host.cache.write(host.table[b, p // page], p % page, 0, 0, _np(k[host.starts[b] + i, 0]))
                host.cache.write(host.table[b, p // page], p % page, 0, 1, _np(v[host.starts[b] + i, 0]))
        _same_parts(dev.data.cpu().numpy(), host, host.cache)
        _check_attention(host, kind, q, out, lse)
