"""Values at the ends of the formats through the 4-bit cache and the attention over it."""
from __future__ import annotations

import numpy as np
import pytest

from tests.test_serving_gpu import Host, _attend, _check_attention, _np, _ok, _torch, _wide

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("spread", [False, True])  # a cluster's join; whole items and the join kernel
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_float16_results_stay_finite_where_rows_were(runtime, dim, spread):
    """A group from -100 to 65504 reads back as up to 65540, which float16 results are clamped from, as the load's
    are; a row with NaN among its values stays NaN."""
    import torch
    rng = np.random.default_rng(dim)
    held = [1500, 40]
    host = Host(rng, dim, 1, 16, [1, 1], held)
    row = np.full(dim, -100.0)
    row[1::2] = 65504.0
    for b, n in enumerate(held):
        for p in range(n):
            host.cache.write(host.table[b, p // 16], p % 16, 0, 0, np.ones(dim))
            host.cache.write(host.table[b, p // 16], p % 16, 0, 1, row * (1 if b == 0 else -1))
    bad = -row
    bad[3] = np.nan
    host.cache.write(host.table[1, 0], 3, 0, 1, bad)
    q = _torch(rng.standard_normal((2, 4, dim)), "f16")
    out, lse, ws = _attend(runtime, host, q, 4, batch=_wide(host) if spread else None)
    assert (ws.numel() > 0) == spread
    _ok(runtime)
    got = _np(out)
    assert not np.isinf(got).any()
    assert np.isnan(got[1, :, :32]).all() and not np.isnan(got[1, :, 32:]).any() and not np.isnan(got[0]).any()
    assert (got[0, :, 1::2] == 65504.0).all() and (got[1, :, 33::2] == -65504.0).all()
    assert (np.abs(got[0, :, 0::2] + 100.0) <= 100.0 * 2.0 ** -11 + 65536 * 2.0 ** -20).all()
    assert torch.isfinite(lse).all()


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("exponent", [-120, -98, 60, 110])
def test_queries_at_the_ends_of_their_range(runtime, kind, exponent):
    """Tiny and huge queries whose scale brings the scores back to the ordinary; a row of zeros weighs all keys alike."""
    rng = np.random.default_rng(abs(exponent))
    host = Host(rng, 128, 1, 16, [2, 1], [600, 40])
    host.fill(rng)
    x = np.clip(rng.standard_normal((3, 8, 128)), -3.9, 3.9)
    x[0, 5] = 0.0
    q = _torch(x * 2.0 ** exponent, kind)
    scale = float(np.float32(min(0.1 * 2.0 ** -exponent, 2.0 ** 99)))
    out, lse, _ = _attend(runtime, host, q, 8, scale=scale)
    _ok(runtime)
    assert np.isfinite(_np(out)).all()
    _check_attention(host, kind, q, out, lse, scale=scale)
