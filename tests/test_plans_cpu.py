"""Plans of batches for sequences that run past the cache's tokens."""
import pytest
import torch

from yalm_amd.cache import CacheManager, KVRequest, StateRequest
from yalm_amd.generate import plan_batches


def test_plans_of_sequences_that_outgrow_the_cache_s_tokens():
    """Where every line keeps a window, a sequence holds its ring of pages, however long its text runs."""
    assert plan_batches([5, 9], 1000, None, 64 * 4, 8, 2000, ring_pages=2) == [[0, 1]]
    assert plan_batches([5, 9, 3], 1000, None, 64 * 4, 8, 2000, ring_pages=2) == [[0, 1], [2]]
    assert plan_batches([5, 9, 3], 1000, 1, 64 * 4, 8, 2000, ring_pages=4) == [[0], [1], [2]]
    # what fits by its tokens is planned as before
    assert plan_batches([100, 100, 100], 28, None, 256, 8, 512, ring_pages=1) == [[0, 1], [2]]
    with pytest.raises(ValueError, match="cache"):
        plan_batches([5], 1000, None, 64 * 4, 8, 2000, ring_pages=5)
    with pytest.raises(ValueError, match="cache"):
        plan_batches([5], 1000, None, 64 * 4, 8, 2000)


def test_the_pages_that_a_sequence_never_outgrows():
    kv = lambda *windows: {i: KVRequest(1, 4, w) for i, w in enumerate(windows)}  # noqa: E731
    make = lambda reqs, tokens, length, **kw: CacheManager(reqs, tokens, length, torch.float32, "cpu", n_slots=2, **kw)  # noqa: E731
    assert make(kv(100, 200), 1024, 4000).whole_rings() == 5
    assert make(kv(100), 1024, 4000, max_draft=70).whole_rings() == 4
    assert make(kv(0, 100), 1024, 4000).whole_rings() == 0          # one line keeps everything
    assert make(kv(100), 128, 4000).whole_rings() == 0              # the ring itself is cut short
    assert make({0: StateRequest((3,))}, 128, 4000).whole_rings() == 0
