"""What BatchedAttention refuses of a model before it touches a cache (no GPU)."""

from __future__ import annotations

import pytest

from klcquant_amd.attention import AttentionConfig
from klcquant_amd.paged_kv import BatchedAttention


@pytest.mark.parametrize("heads,kv,dim,text", [(33, 1, 64, "33 query heads"), (64, 1, 64, "64 query heads"), (9, 2, 64, "9 query heads"),
                                               (8, 0, 64, "over 0"), (0, 2, 64, "0 query heads"), (8, 2, 60, "head size"),
                                               (8, 2, 136, "head size"), (8, 2, 0, "head size"), (8192, 512, 64, "8192 query heads")])
def test_models_that_a_step_cannot_take_are_refused(heads, kv, dim, text):
    """Prompts take any group; a prompt whose steps are refused must not fill a cache."""
    with pytest.raises(ValueError, match=text):
        BatchedAttention(AttentionConfig(256, heads, kv, dim))


@pytest.mark.parametrize("heads,kv,dim", [(32, 1, 64), (64, 8, 64), (4096, 128, 8), (5, 5, 128)])
def test_models_at_the_limits(heads, kv, dim):
    assert BatchedAttention(AttentionConfig(256, heads, kv, dim)).config.num_heads == heads
