"""The token-by-token serving entries without a GPU: struct layouts, refusals, workspace
arithmetic, and the oracle of the 4-bit cache against its own definition."""
from __future__ import annotations

import ctypes as C
import subprocess

import numpy as np
import pytest

from oct_b200 import reactor as R
from oracle import serving as O
from tests.test_abi import HEADER, _handle

STRUCTS = {
    "OctB200QkNormRopeRequest": R.OctB200QkNormRopeRequest,
    "OctB200Kv4Cache": R.OctB200Kv4Cache,
    "OctB200Kv4Batch": R.OctB200Kv4Batch,
    "OctB200Kv4Rows": R.OctB200Kv4Rows,
    "OctB200Kv4AttentionRequest": R.OctB200Kv4AttentionRequest,
}
INVALID, UNALIGNED, SHAPE, NO_DEVICE = -7008, -7005, -7007, -6006
P = 1 << 20  # an aligned address that nothing reads: these calls all end before a launch


def test_struct_layouts_match_the_header(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void){"]
    for name, py in STRUCTS.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f[0]} %zu\\n", offsetof({name}, {f[0]}));' for f in py._fields_]
    lines.append("return 0;}")
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-o", str(tmp_path / "layout"), str(src)], check=True)
    got = dict(line.split() for line in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True,
                                                       text=True).stdout.splitlines())
    for name, py in STRUCTS.items():
        assert int(got[name]) == C.sizeof(py), name
        for f in py._fields_:
            assert int(got[f"{name}.{f[0]}"]) == getattr(py, f[0]).offset, (name, f[0])


@pytest.fixture
def handle(lib):
    h = _handle(lib, R.TESTCFG_FAIL_DEVICE_CREATE)
    yield h
    lib.prometheus_reactor_runtime_destroy(h)


def _rope(**kw):
    r = R.OctB200QkNormRopeRequest()
    base = dict(struct_size=C.sizeof(r), dtype=R.DTYPE_BF16, tokens=3, q_heads=4, k_heads=2, head_dim=128, rotary_dim=96,
                interleaved=0, normalize=1, eps=1e-6, axes=2, axis_pairs=(C.c_uint32 * 4)(16, 32), q=P, k=P, q_out=P,
                k_out=3 * P, q_token_stride=512, q_head_stride=128, k_token_stride=256, k_head_stride=128,
                q_out_token_stride=512, q_out_head_stride=128, k_out_token_stride=256, k_out_head_stride=128,
                positions=P, position_stride=2, frequencies=P)
    for name, value in (base | kw).items():
        setattr(r, name, value)
    return r


@pytest.mark.parametrize("change, code", [
    (dict(), NO_DEVICE), (dict(struct_size=8), INVALID), (dict(dtype=3), INVALID), (dict(axes=0), INVALID),
    (dict(axes=5), INVALID), (dict(axis_pairs=(C.c_uint32 * 4)(16, 33)), INVALID), (dict(eps=0.0), INVALID),
    (dict(eps=float("nan")), INVALID), (dict(head_dim=96, rotary_dim=96), NO_DEVICE), (dict(head_dim=80), INVALID),
    (dict(head_dim=120), SHAPE), (dict(head_dim=528), SHAPE), (dict(q=None), INVALID), (dict(k_out=None), INVALID),
    (dict(k=None, k_out=None, k_heads=0), NO_DEVICE), (dict(positions=None), INVALID), (dict(frequencies=P + 4), UNALIGNED),
    (dict(positions=P + 2), UNALIGNED), (dict(position_stride=1), INVALID), (dict(q=P + 2), UNALIGNED),
    (dict(q_token_stride=516), UNALIGNED), (dict(q_out=2 * P, q_out_token_stride=504), INVALID),
    (dict(q_out=2 * P, q_out_head_stride=64), INVALID), (dict(q_out_token_stride=128, q_out_head_stride=384), INVALID),
    (dict(q_out=2 * P, q_out_token_stride=128, q_out_head_stride=384), NO_DEVICE), (dict(q_weight=P + 4), UNALIGNED),
    (dict(k_out=P), INVALID), (dict(tokens=1 << 31), SHAPE), (dict(tokens=0), NO_DEVICE),
    (dict(rotary_dim=0, axis_pairs=(C.c_uint32 * 4)(0, 0)), SHAPE),
])
def test_qk_norm_rope_refusals(lib, handle, change, code):
    detail = C.c_int()
    rc = lib.oct_b200_qk_norm_rope_device(handle, _rope(**change), None, detail)
    assert (rc, detail.value) == (R.PROM_ERROR, code)


def test_a_stale_handle_is_refused(lib):
    detail = C.c_int()
    assert lib.oct_b200_qk_norm_rope_device(None, _rope(), None, detail) == R.PROM_INVALID_HANDLE
    assert lib.oct_b200_kv4_store_device(None, _cache(), _batch(), _rows(), None, detail) == R.PROM_INVALID_HANDLE
    assert lib.oct_b200_kv4_load_device(None, _cache(), _batch(), _rows(), None, detail) == R.PROM_INVALID_HANDLE
    assert lib.oct_b200_kv4_attention_device(None, _cache(), _batch(), _attention(), None, detail) == R.PROM_INVALID_HANDLE


def _fill(cls, base, kw):
    r = cls()
    for name, value in (base | kw).items():
        setattr(r, name, value)
    return r


def _cache(**kw):
    return _fill(R.OctB200Kv4Cache, dict(struct_size=C.sizeof(R.OctB200Kv4Cache), page_size=32, kv_heads=2,
                                         head_dim=128, pages=9, data=P), kw)


def _batch(**kw):
    return _fill(R.OctB200Kv4Batch, dict(struct_size=C.sizeof(R.OctB200Kv4Batch), batch=3, page_table=P,
                                         page_table_stride=4, page_table_width=4, max_tokens=5, max_kv_len=128,
                                         kv_lens=P, cu_tokens=P), kw)


def _rows(**kw):
    return _fill(R.OctB200Kv4Rows, dict(struct_size=C.sizeof(R.OctB200Kv4Rows), dtype=R.DTYPE_F32, tokens=7, k=P, v=2 * P,
                                        k_token_stride=256, k_head_stride=128, v_token_stride=256,
                                        v_head_stride=128), kw)


def _attention(**kw):
    return _fill(R.OctB200Kv4AttentionRequest, dict(struct_size=C.sizeof(R.OctB200Kv4AttentionRequest),
                                                    dtype=R.DTYPE_F16, q_heads=8, causal=1, scale=0.1, tokens=7, q=P,
                                                    out=P, q_token_stride=1024, q_head_stride=128,
                                                    out_token_stride=1024, out_head_stride=128, workspace=P,
                                                    workspace_bytes=1 << 40), kw)


CACHE_CHANGES = [
    (dict(struct_size=8), INVALID), (dict(data=None), INVALID), (dict(data=P + 8), UNALIGNED), (dict(pages=0), INVALID),
    (dict(page_size=0), SHAPE), (dict(page_size=24), SHAPE), (dict(page_size=1 << 17), SHAPE), (dict(head_dim=96), SHAPE),
    (dict(kv_heads=0), INVALID), (dict(kv_heads=5000), SHAPE), (dict(reserved=1), INVALID),
]
BATCH_CHANGES = [
    (dict(struct_size=8), INVALID), (dict(kv_lens=None), INVALID), (dict(page_table=None), INVALID),
    (dict(max_kv_len=129), INVALID), (dict(page_table_stride=3), INVALID), (dict(cu_tokens=None), INVALID),
    (dict(cu_tokens=None, max_tokens=1), INVALID), (dict(batch=65536, max_kv_len=1), SHAPE), (dict(reserved=1), INVALID),
    (dict(max_tokens=1 << 30), SHAPE), (dict(kv_lens=P + 1), UNALIGNED), (dict(page_table=P + 2), UNALIGNED),
    (dict(batch=0), NO_DEVICE), (dict(max_tokens=0), NO_DEVICE),
]


@pytest.mark.parametrize("change, code", CACHE_CHANGES)
def test_cache_refusals(lib, handle, change, code):
    detail = C.c_int()
    for fn, arg in ((lib.oct_b200_kv4_store_device, _rows()), (lib.oct_b200_kv4_load_device, _rows()),
                    (lib.oct_b200_kv4_attention_device, _attention())):
        assert (fn(handle, _cache(**change), _batch(), arg, None, detail), detail.value) == (R.PROM_ERROR, code)


@pytest.mark.parametrize("change, code", BATCH_CHANGES)
def test_batch_refusals(lib, handle, change, code):
    detail = C.c_int()
    for fn, arg in ((lib.oct_b200_kv4_store_device, _rows()), (lib.oct_b200_kv4_load_device, _rows()),
                    (lib.oct_b200_kv4_attention_device, _attention())):
        assert (fn(handle, _cache(), _batch(**change), arg, None, detail), detail.value) == (R.PROM_ERROR, code)


@pytest.mark.parametrize("change, code", [
    (dict(), NO_DEVICE), (dict(struct_size=8), INVALID), (dict(dtype=7), INVALID), (dict(k=None), INVALID),
    (dict(v=P + 4), UNALIGNED), (dict(k_token_stride=258), UNALIGNED), (dict(tokens=0, k=None, v=None), NO_DEVICE),
    (dict(k_token_stride=1 << 40), INVALID),
])
def test_row_refusals(lib, handle, change, code):
    detail = C.c_int()
    for fn in (lib.oct_b200_kv4_store_device, lib.oct_b200_kv4_load_device):
        assert (fn(handle, _cache(), _batch(), _rows(**change), None, detail), detail.value) == (R.PROM_ERROR, code)


def test_keys_and_values_are_not_read_back_into_one_tensor(lib, handle):
    detail = C.c_int()
    one = _rows(v=P)
    assert lib.oct_b200_kv4_load_device(handle, _cache(), _batch(), one, None, detail) == R.PROM_ERROR
    assert detail.value == INVALID
    assert lib.oct_b200_kv4_store_device(handle, _cache(), _batch(), one, None, detail) == R.PROM_ERROR
    assert detail.value == NO_DEVICE


def test_rows_that_share_elements_may_be_read_and_not_written(lib, handle):
    detail = C.c_int()
    shared = _rows(k_token_stride=0, k_head_stride=0)
    assert lib.oct_b200_kv4_store_device(handle, _cache(), _batch(), shared, None, detail) == R.PROM_ERROR
    assert detail.value == NO_DEVICE
    assert lib.oct_b200_kv4_load_device(handle, _cache(), _batch(), shared, None, detail) == R.PROM_ERROR
    assert detail.value == INVALID


def test_the_stride_of_a_dimension_of_one_is_not_used(lib, handle):
    detail, odd = C.c_int(), (1 << 50) + 1
    one_token = dict(tokens=1, q_token_stride=odd, q_out_token_stride=odd + 1, k_token_stride=odd, k_out_token_stride=odd)
    one_head = dict(q_heads=1, q_head_stride=odd, q_out_head_stride=odd + 2, k_heads=1, k_head_stride=3, k_out_head_stride=0)
    for change in (one_token, one_head):
        assert lib.oct_b200_qk_norm_rope_device(handle, _rope(**change), None, detail) == R.PROM_ERROR
        assert detail.value == NO_DEVICE
    rows = _rows(tokens=1, k_token_stride=odd, v_token_stride=7)
    for fn in (lib.oct_b200_kv4_store_device, lib.oct_b200_kv4_load_device):
        assert (fn(handle, _cache(), _batch(), rows, None, detail), detail.value) == (R.PROM_ERROR, NO_DEVICE)
    rows = _attention(q_heads=1, q_head_stride=odd, out_head_stride=odd)
    got = lib.oct_b200_kv4_attention_device(handle, _cache(kv_heads=1), _batch(), rows, None, detail)
    assert (got, detail.value) == (R.PROM_ERROR, NO_DEVICE)


@pytest.mark.parametrize("change, code", [
    (dict(), NO_DEVICE), (dict(struct_size=8), INVALID), (dict(dtype=4), INVALID), (dict(q_heads=0), INVALID),
    (dict(q_heads=7), INVALID), (dict(scale=float("inf")), INVALID), (dict(window=5, causal=0), INVALID),
    (dict(window=5), NO_DEVICE), (dict(q=None), INVALID), (dict(out=P + 8), UNALIGNED), (dict(lse=P + 2), UNALIGNED),
    (dict(out_token_stride=1016), INVALID), (dict(workspace=None), -7031), (dict(workspace_bytes=16), -7031),
    (dict(workspace=P + 8), UNALIGNED), (dict(q_heads=65536 * 2), SHAPE),
])
def test_attention_refusals(lib, handle, change, code):
    detail = C.c_int()
    rc = lib.oct_b200_kv4_attention_device(handle, _cache(pages=999), _batch(page_table_width=300, page_table_stride=300,
                                                                             max_kv_len=9000),
                                           _attention(**change), None, detail)
    assert (rc, detail.value) == (R.PROM_ERROR, code)


def test_workspace_is_a_function_of_sizes(lib):
    size, detail = C.c_uint64(), C.c_int()

    def ask(batch, request):
        rc = lib.oct_b200_kv4_attention_workspace_bytes(_cache(), batch, request, size, detail)
        return rc, size.value

    assert ask(_batch(max_kv_len=16), _attention()) == (R.PROM_OK, 0)  # too few keys to split
    wide = dict(page_table_width=1 << 12, page_table_stride=1 << 12, max_kv_len=1 << 17)
    rc, long = ask(_batch(**wide), _attention())
    assert rc == R.PROM_OK and 0 < long < 1 << 25  # two parts per thread block, however many the keys
    assert ask(_batch(**(wide | dict(max_kv_len=1 << 16))), _attention()) == (R.PROM_OK, long)
    assert ask(_batch(), _attention()) == (R.PROM_OK, 0)  # a cluster's blocks join in shared memory
    rc, few = ask(_batch(**(wide | dict(max_kv_len=1 << 14))), _attention())
    assert rc == R.PROM_OK and 0 < few <= long
    assert ask(_batch(**wide), _attention(window=512)) == (R.PROM_OK, 0)  # the window bounds an item's keys
    assert ask(_batch(batch=0), _attention()) == (R.PROM_OK, 0)
    assert ask(_batch(), _attention(q_heads=3))[0] == R.PROM_ERROR


def test_tile_bytes(lib):
    for dim in (64, 128, 256):
        assert lib.oct_b200_kv4_tile_bytes(dim) == R.kv4_tile_bytes(dim) == O.tile_bytes(dim) == 20 * dim
    assert lib.oct_b200_kv4_tile_bytes(96) == 0


def test_oracle_quantiser_keeps_its_definition():
    rng = np.random.default_rng(5)
    x = rng.standard_normal((40, 128)) * 10.0 ** rng.integers(-9, 6, (40, 1))
    x[3, 40] = np.inf
    x[4, 70] = np.nan
    x[5] = 0.25
    codes, s, z = O.quantise(x)
    y = O.values(codes, s, z)
    assert codes.max() == 15
    clipped = np.clip(x, -O.F16_MAX, O.F16_MAX)
    nan = np.repeat(np.isnan(z), 32, axis=-1)
    assert nan.sum() == 32 and np.isnan(y[nan]).all()
    assert (np.abs(y - clipped)[~nan] <= np.repeat(s, 32, axis=-1)[~nan] / 2).all()
    for scale, zero in zip(s.ravel(), z.ravel()):
        assert np.isnan(zero) or (np.float16(scale) == scale and np.float16(zero) == zero)


def test_oracle_cache_rows_round_trip():
    rng = np.random.default_rng(6)
    c = O.Cache(3, 32, 2, 64, fill=0xFF)
    x = rng.standard_normal((2, 64))
    c.write(1, 17, 1, 0, x[0])
    c.write(1, 17, 1, 1, x[1])
    for which in (0, 1):
        assert np.array_equal(O.values(*c.parts(1, 17, 1, which)), O.values(*O.quantise(x[which])))
    untouched = np.ones(c.data.shape, bool)
    untouched[1, 1, 1] = False
    assert (c.data[untouched] == 0xFF).all()
