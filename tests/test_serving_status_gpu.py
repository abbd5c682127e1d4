"""What oct_b200_sync_status reports of calls that skipped a bad index, beside other reports and other streams."""
from __future__ import annotations

import numpy as np
import pytest

from oct_b200 import reactor as R
from tests.test_serving_gpu import _int

pytestmark = pytest.mark.gpu
NONFINITE = -6814


def _bad_store(runtime):
    """A store of one row whose page is none of the cache's."""
    import torch
    cache = R.Kv4Cache(torch.zeros((2, R.kv4_tile_bytes(64)), dtype=torch.uint8, device="cuda"), page_size=16, kv_heads=1,
                       head_dim=64)
    batch = R.Kv4Batch(_int([[7]]), _int([1]), page_size=16)
    k, v = (torch.zeros((1, 1, 64), device="cuda") for _ in range(2))
    return lambda stream=None: runtime.kv4_store_device(cache, batch, k, v, stream=stream)


def test_a_bad_index_does_not_hide_a_non_finite_input(runtime):
    import torch
    store = _bad_store(runtime)
    x = torch.ones((4, 256), device="cuda")
    x[2, 9] = float("nan")
    y, w, inv = torch.empty_like(x), torch.ones(256, device="cuda"), torch.empty(4, device="cuda")
    assert runtime.sync_status().ok
    runtime.rmsnorm_device(x, w, y, inv, 4, 256, 1e-6)
    assert runtime.sync_status().detail == NONFINITE
    store()
    runtime.rmsnorm_device(x, w, y, inv, 4, 256, 1e-6)
    assert {runtime.sync_status().detail, runtime.sync_status().detail} == {
        R.DETAIL_KV4_BAD_INDEX, NONFINITE}
    assert runtime.sync_status().ok


def test_a_bad_index_reported_while_another_stream_is_asked(runtime):
    """The kernel that skips may end at any time of a status call that waits for another stream: its report is
    given by that call or by the next one, once."""
    import torch
    store = _bad_store(runtime)
    busy, asked = torch.cuda.Stream(), torch.cuda.Stream()
    store()
    assert runtime.sync_status().detail == R.DETAIL_KV4_BAD_INDEX
    lost = twice = 0
    for i in range(600):
        torch.cuda.synchronize()
        with torch.cuda.stream(busy):
            torch.cuda._sleep(200 * i)  # 0 to about 60 us
        store(busy)
        first = runtime.sync_status(asked).detail
        torch.cuda.synchronize()
        reports = [first, runtime.sync_status().detail].count(R.DETAIL_KV4_BAD_INDEX)
        lost, twice = lost + (reports == 0), twice + (reports == 2)
    assert (lost, twice) == (0, 0)
