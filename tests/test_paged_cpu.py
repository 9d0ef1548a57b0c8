"""Argument checks of the paged cache's C entry points (made on the host before any launch)
and of the Python layer's CPU tensors."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from dsa_b200 import _capi as capi


@pytest.fixture(scope="module")
def lib():
    from dsa_b200.build import build

    build()
    return capi.lib()


def _cache(**kw):
    base = dict(keys=4096, values=8192, page_stride=4096, row_stride=256, head_stride=128, pages=4,
                page_size=16, kv_heads=2, head_dim=128, dtype=capi.TDSA_BF16)
    base.update(kw)
    return capi.TdsaPagedCache(**base)


def _batch(**kw):
    base = dict(page_table=4096, table_stride=8, query_starts=4096, lengths=4096, batch=2,
                max_pages=8, tokens=2, max_new=1)
    base.update(kw)
    return capi.TdsaPagedBatch(**base)


def _rows(data=4096, token=1024, head=128):
    return capi.TdsaTokenRows(data, token, head)


def _attend(lib, cache, batch, q=None, out=None, heads=8, scale=1.0, window=0, ws=4096,
            ws_bytes=1 << 40):
    return lib.tdsa_paged_attention(C.byref(cache), C.byref(batch), C.byref(q or _rows()), heads,
                                    scale, window, C.byref(out or _rows(data=16384)),
                                    None, ws, ws_bytes,
                                    None)


INVALID, UNSUP = capi.TDSA_ERR_INVALID, capi.TDSA_ERR_UNSUPPORTED
ALIGN, WORK = capi.TDSA_ERR_ALIGN, capi.TDSA_ERR_WORKSPACE


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=capi.TDSA_F32), UNSUP), (dict(head_dim=96), UNSUP), (dict(page_size=24), UNSUP),
    (dict(page_size=8), UNSUP), (dict(page_size=2048), UNSUP), (dict(pages=0), INVALID),
    (dict(kv_heads=0), INVALID), (dict(keys=None), INVALID), (dict(values=8200), ALIGN),
    (dict(row_stride=250), ALIGN), (dict(row_stride=64), INVALID), (dict(head_stride=64), INVALID),
    (dict(page_stride=-8), INVALID)])
def test_cache_checks(lib, kw, code):
    assert _attend(lib, _cache(**kw), _batch()) == code
    assert capi.last_error()


@pytest.mark.parametrize("kw,code", [
    (dict(batch=0), INVALID), (dict(batch=70000), INVALID), (dict(tokens=-1), INVALID),
    (dict(max_new=-1), INVALID), (dict(max_pages=0), INVALID), (dict(page_table=None), INVALID),
    (dict(query_starts=None), INVALID), (dict(lengths=None), INVALID),
    (dict(table_stride=7), INVALID), (dict(max_pages=1 << 27, table_stride=1 << 27), UNSUP)])
def test_batch_checks(lib, kw, code):
    assert _attend(lib, _cache(), _batch(**kw)) == code


def test_attention_checks(lib):
    c, b = _cache(), _batch()
    assert _attend(lib, c, b, heads=3) == INVALID
    assert _attend(lib, c, b, heads=0) == INVALID
    assert _attend(lib, c, b, q=_rows(data=None)) == INVALID
    assert _attend(lib, c, b, q=_rows(data=4098)) == ALIGN
    assert _attend(lib, c, b, out=_rows(token=1025)) == ALIGN
    assert _attend(lib, c, b, out=_rows()) == INVALID  # q itself
    assert _attend(lib, c, b, heads=4096) == UNSUP     # 2048 query heads per key/value head
    assert _attend(lib, c, b, out=_rows(token=-1024)) == INVALID
    assert _attend(lib, c, b, scale=0.0) == INVALID
    assert _attend(lib, c, b, scale=float("nan")) == INVALID
    assert _attend(lib, c, b, window=-1) == INVALID
    assert _attend(lib, c, b, ws=None) == WORK
    assert _attend(lib, c, b, ws=4100) == WORK
    assert _attend(lib, c, b, ws_bytes=16) == WORK
    assert _attend(lib, c, _batch(tokens=0)) == capi.TDSA_OK
    assert lib.tdsa_paged_attention(None, C.byref(b), None, 8, 1.0, 0, None, None, None, 0,
                                    None) == INVALID
    assert lib.tdsa_paged_workspace_bytes(96) == 0


def test_selected_checks(lib):
    def call(idx=4096, nbytes=4, stride=16, k=16):
        return lib.tdsa_selected_attention(
            C.byref(_cache()), C.byref(_batch()), C.byref(_rows()), 8, 1.0, idx, nbytes, stride, k,
            C.byref(_rows(data=16384)), None, 4096, 1 << 40, None)

    assert call(idx=None) == INVALID
    assert call(nbytes=2) == INVALID
    assert call(idx=4098) == ALIGN
    assert call(k=0) == INVALID
    assert call(stride=15) == INVALID


def test_append_checks(lib):
    def call(cache=None, k=None, v=None, q=None, q_out=None, heads=8, freq=4096, rope=64):
        ref = [None if r is None else C.byref(r) for r in (k, v, q, q_out)]
        return lib.tdsa_paged_append(C.byref(cache or _cache()), C.byref(_batch()), *ref, heads,
                                     freq, rope, 0, None, None)

    r = _rows
    assert call(k=r(), v=None) == INVALID
    assert call(k=None, v=r()) == INVALID
    assert call(k=r(), v=r(data=4104)) == ALIGN
    assert call(k=r(), v=r(), q=r()) == INVALID  # no q_out
    assert call(k=r(), v=r(), q=r(), q_out=r(), heads=0) == INVALID
    assert call(k=r(), v=r(), rope=24) == INVALID
    assert call(k=r(), v=r(), rope=144) == INVALID
    assert call(k=r(), v=r(), freq=None) == INVALID
    assert call(cache=_cache(head_dim=64), k=r(), v=r(), rope=80) == INVALID


def test_cpu_tensors_are_refused():
    from dsa_b200.paged import PagedBatch, PagedKV

    pages = torch.zeros(2, 16, 1, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        PagedKV(pages, pages)
    i = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(ValueError):
        PagedBatch(i, torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
