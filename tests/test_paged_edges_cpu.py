"""Checks of the paged cache that are made on the host, where no device is needed."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from dsa_b200 import paged


def _on(index):
    """A cache and a batch as the checks see them, on device ``index``."""
    device = torch.device("cuda", index)
    cache = SimpleNamespace(_index=index, device=device, dtype=torch.bfloat16, head_dim=128,
                            kv_heads=2)
    return cache, SimpleNamespace(_index=index, device=device)


@pytest.mark.parametrize("current,where", [(0, 1), (1, 0), (3, 2)])
def test_a_cache_on_another_device_than_the_current_one_is_refused(monkeypatch, current, where):
    monkeypatch.setattr(paged, "_current_device", lambda: current)
    cache, batch = _on(where)
    q = torch.zeros(1, 8, 128, dtype=torch.bfloat16)
    app = object.__new__(paged.PagedAppender)
    app.cache = cache
    for call in (lambda: paged.paged_attention(q, cache, batch),
                 lambda: paged.selected_attention(q, cache, batch, torch.zeros(1, 4)),
                 lambda: app.append(batch, q[:, :2], q[:, :2])):
        with pytest.raises(ValueError, match="current device"):
            call()


def test_a_batch_on_another_device_than_the_cache_is_refused(monkeypatch):
    monkeypatch.setattr(paged, "_current_device", lambda: 0)
    with pytest.raises(ValueError, match="one device"):
        paged.paged_attention(torch.zeros(1, 8, 128), _on(0)[0], _on(1)[1])


@pytest.mark.parametrize("reset", [True, False])
def test_a_timeout_ends_the_workspaces_of_its_device(monkeypatch, reset):
    # a call that was cut off may leave its arrival counters above zero
    from dsa_b200 import _capi as capi
    from dsa_b200 import device_status

    kept = {(0, 5, 64): "a", (0, 0, 128): "b", (1, 5, 64): "c"}
    monkeypatch.setattr(paged, "_WORKSPACES", dict(kept))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    status = capi.TDSA_STATUS_RANGE
    monkeypatch.setattr(capi, "device_status", lambda r=True: status if r == reset else None)
    assert device_status(reset) == status
    assert paged._WORKSPACES == kept
    status |= capi.TDSA_ERR_TIMEOUT
    assert device_status(reset) == status
    assert paged._WORKSPACES == {(1, 5, 64): "c"}
    paged.release_paged_workspaces()
    assert not paged._WORKSPACES


# ------------------------------------------------------------------ outputs that overlap

def _rows_overlap(q, heads, out, out_heads, tokens, dim):
    """By listing every element."""
    def taken(r, n):
        return {r[0] // 2 + t * r[1] + h * r[2] + d
                for t in range(tokens) for h in range(n) for d in range(dim)}

    return bool(taken(q, heads) & taken(out, out_heads))


def _attend_rc(q, out, heads, tokens, dim):
    """The C entry's answer for rows (address, token stride, head stride): no workspace is given,
    so a call that passes the checks of its rows is refused for that."""
    import ctypes as C

    from dsa_b200 import _capi as capi

    cache = capi.TdsaPagedCache(4096, 8192, 4096, 256, 128, 4, 16, 1, dim, capi.TDSA_BF16)
    batch = capi.TdsaPagedBatch(4096, 8, 4096, 4096, 2, 8, tokens, tokens)
    rc = capi.lib().tdsa_paged_attention(
        C.byref(cache), C.byref(batch), C.byref(capi.TdsaTokenRows(*q)), heads, 1.0, 0,
        C.byref(capi.TdsaTokenRows(*out)), None, None, 0, None)
    if rc == capi.TDSA_ERR_WORKSPACE:
        return False
    assert rc == capi.TDSA_ERR_INVALID and "overlap" in capi.last_error()
    return True


@pytest.fixture(scope="module")
def lib():
    from dsa_b200.build import build

    build()


def test_overlapping_outputs_are_refused(lib):
    # every offset of out from q over the same strides: as the listed elements have it
    for tokens, heads, ts, hs in ((3, 2, 128, 64), (3, 2, 320, 64), (4, 3, 64, 256), (3, 2, 384, 128),
                                  (2, 3, 72, 144), (1, 3, 0, 128), (3, 1, 192, 0)):
        for off in range(-1200, 1200, 8):
            q, out = (65536, ts, hs), (65536 + 2 * off, ts, hs)
            want = off == 0 or _rows_overlap(q, heads, out, heads, tokens, 64)
            assert _attend_rc(q, out, heads, tokens, 64) == want, (tokens, heads, ts, hs, off)


@pytest.mark.parametrize("tokens,heads,ts,hs,fine", [
    (3, 2, 128, 64, True), (3, 2, 64, 192, True), (3, 2, 0, 64, False), (3, 2, 128, 0, False),
    (3, 2, 128, 56, False), (3, 2, 64, 128, False), (2, 3, 120, 64, False), (1, 2, 0, 64, True),
    (3, 1, 64, 0, True), (3, 1, 56, 0, False), (4, 3, 136, 64, False), (4, 3, 64, 256, True)])
def test_outputs_whose_rows_overlap_each_other_are_refused(lib, tokens, heads, ts, hs, fine):
    assert _attend_rc((65536, 1024, 128), (1 << 20, ts, hs), heads, tokens, 64) == (not fine)


def _append_rc(k, v, q, q_out, tokens=3, heads=2, dim=64):
    import ctypes as C

    from dsa_b200 import _capi as capi

    cache = capi.TdsaPagedCache(4096, 8192, 4096, 256, 128, 4, 16, 1, dim, capi.TDSA_BF16)
    batch = capi.TdsaPagedBatch(4096, 8, 4096, 4096, 2, 8, tokens, tokens)
    rc = capi.lib().tdsa_paged_append(
        C.byref(cache), C.byref(batch),
        *(C.byref(capi.TdsaTokenRows(*r)) for r in (k, v, q, q_out)), heads, 4096, 64, 0, None, None)
    return rc == capi.TDSA_ERR_INVALID and "overlap" in capi.last_error()


def test_append_refuses_queries_that_overlap(lib):
    at = 1 << 16
    k, v = (1 << 20, 64, 64), (1 << 21, 64, 64)
    assert _append_rc(k, v, (at, 128, 64), (at + 128, 128, 64))      # a head on
    assert _append_rc(k, v, (at, 128, 64), (at - 16, 128, 64))
    assert _append_rc(k, v, (at, 128, 64), (at, 256, 64))            # in place, other strides
    assert _append_rc(k, v, (at, 128, 64), (at, 128, 192))
    assert _append_rc((at, 256, 64), v, (at + 4096, 256, 64), (at - 64, 256, 64))
    assert _append_rc(k, (at + 128, 256, 64), (at + 4096, 256, 64), (at, 256, 64))
    assert _append_rc(k, v, (at, 128, 64), (at + 4096, 64, 64))      # its own rows
