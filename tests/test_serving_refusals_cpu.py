"""Calls of the serving entries that their documentation rules out, refused on the host (no GPU)."""
from __future__ import annotations

import ctypes as C

import pytest

from oct_b200 import reactor as R
from tests.test_abi import _handle
from tests.test_serving_cpu import INVALID, NO_DEVICE, P, _attention, _batch, _cache


@pytest.fixture
def handle(lib):
    h = _handle(lib, R.TESTCFG_FAIL_DEVICE_CREATE)
    yield h
    lib.prometheus_reactor_runtime_destroy(h)


# over the queries: row for row, or not at all (7 tokens of 8 heads of 128)
@pytest.mark.parametrize("change, code", [
    (dict(), NO_DEVICE),
    (dict(out_token_stride=128, out_head_stride=7 * 128), INVALID),  # head-major over token-major
    (dict(q_token_stride=1152, out_token_stride=1024), INVALID),
    (dict(q_head_stride=256, q_token_stride=2048, out_token_stride=2048), INVALID),
    (dict(q_token_stride=128, q_head_stride=896, out_token_stride=128, out_head_stride=896), NO_DEVICE),
    (dict(out=64 * P, out_token_stride=128, out_head_stride=896), NO_DEVICE),
    (dict(tokens=1, out_token_stride=4096), NO_DEVICE),              # the stride of a dimension of one is not used
])
def test_attention_over_its_queries_keeps_their_strides(lib, handle, change, code):
    detail = C.c_int()
    rc = lib.oct_b200_kv4_attention_device(handle, _cache(), _batch(), _attention(**change), None, detail)
    assert (rc, detail.value) == (R.PROM_ERROR, code)


@pytest.mark.parametrize("scale, code", [
    (2.0 ** 99, NO_DEVICE), (-2.0 ** 99, NO_DEVICE), (2.0 ** 100, INVALID), (-2.0 ** 127, INVALID), (3e38, INVALID),
    (float("nan"), INVALID), (0.0, NO_DEVICE), (1e-45, NO_DEVICE),
])
def test_a_scale_whose_factors_would_not_be_finite_is_refused(lib, handle, scale, code):
    """The kernel multiplies a scale by powers of two up to 2^24 and by log2(e) on its way to a score: a row of zero
    queries must not meet an infinite factor."""
    detail, size = C.c_int(), C.c_uint64()
    rc = lib.oct_b200_kv4_attention_device(handle, _cache(), _batch(), _attention(scale=scale), None, detail)
    assert (rc, detail.value) == (R.PROM_ERROR, code)
    rc = lib.oct_b200_kv4_attention_workspace_bytes(_cache(), _batch(), _attention(scale=scale), size, detail)
    assert (rc, detail.value) == ((R.PROM_OK, 0) if code == NO_DEVICE else (R.PROM_ERROR, INVALID))
