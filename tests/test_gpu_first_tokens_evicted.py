"""Windowed layers that see first tokens, over a cache that is cut: against attention's definition over what every head holds."""

from __future__ import annotations

import pytest

from test_gpu_long_conversations import Run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first,page", [(1, 16), (5, 64), (40, 16)])
def test_first_tokens_stay_in_place(gpu, first, page):
    run = Run(gpu, "fp16", page, 80, first_tokens=first)
    a, b = run.add(), run.add()
    run.extend([a, b], [150, 47])
    run.extend([a, b], [9, 1])
    run.evict([a, b], 96, 30, first)
    child, = run.fork(a, 1)
    for _ in range(3):
        run.extend([a, b, child], [1, 20, 2])
    run.evict([a, b, child], 80, 24, first + 3)
    run.extend([child, a, b], [40, 1, 1])
    cut = run.add()
    run.extend([cut], [100])
    with pytest.raises(ValueError, match="beside their windows"):
        run.cache.evict([cut], 90, 30, first - 1)
    assert run.cache.length(cut) == 100
    run.extend([cut, a], [1, 1])
