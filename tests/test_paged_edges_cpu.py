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
