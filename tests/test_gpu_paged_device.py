"""A cache's batches are on its pool's device, whatever device is current when they are made."""

from __future__ import annotations

import pytest
import torch

from klcquant_amd.paged_kv import PagedKVCache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["cuda", "cuda:0"])
def test_the_device_is_the_pools(gpu, name):
    cache = PagedKVCache(name, 1, 2, 64, 4, 16)
    assert cache.device == cache.pool.device == gpu and cache.device.index == 0
    assert cache.stats()["device"] == "cuda:0"
    batch = cache.extend([cache.add()], 3)
    assert all(t.device == gpu for t in (batch.positions, batch.slots, batch.starts, batch.prefix_table))
