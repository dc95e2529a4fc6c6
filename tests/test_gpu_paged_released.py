"""Windows whose earlier pages the caller has given back: the same bits as with the pages there."""
import numpy as np
import pytest

from tests.paged_cases import Case, close
from tests.test_gpu_paged_paths import dense

pytestmark = pytest.mark.gpu

TYPES = ["f16", "bf16", "f32"]


def needed(c):
    """First key of its own that some row of each sequence sees, and of the prefix."""
    own = [max(0, int(n) - int(r) - c.window + 1) for n, r in zip(c.kv_len, np.diff(c.start))]
    pre = min(max(0, c.prefix + int(n) - int(r) - c.window + 1)
              for n, r in zip(c.kv_len, np.diff(c.start)))
    return own, min(pre, max(0, c.prefix - 1))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("gone", [-1, 1 << 30])
@pytest.mark.parametrize("kw", [
    dict(new=[1, 1, 1], kv=[300, 77, 20]),                       # tokens, whole in a wave
    dict(new=[1, 3], kv=[3000, 2500]),                           # ... cut, and merged
    dict(new=[1, 1], kv=[500, 300], page=4),                     # pages that end inside a tile
    dict(new=[90, 40], kv=[900, 500]),                           # prompts
    dict(new=[300, 200], kv=[900, 500], heads=64, kv_heads=32),  # ... of many row tiles
    dict(new=[1, 2], kv=[9, 30], prefix=700),                    # a prefix among the sequences
    dict(new=[1] * 32, kv=[9] * 32, prefix=3000, heads=64, kv_heads=16),  # ... and apart
    dict(new=[50, 40], kv=[90, 45], prefix=130)])
def test_pages_before_every_window(t, gone, kw):
    kw = dict(page=16, window=100) | kw
    c = Case(**kw, t=t)
    want, tol = dense(c)
    there = c.run()
    close(there, want, tol)
    own, pre = needed(c)
    lost = 0
    for b, first in enumerate(own):
        c.pages[b, :first // c.page] = gone
        lost += first // c.page
    c.prefix_pages[:pre // c.page] = gone
    lost += pre // c.page
    assert lost
    y = c.run()
    c.free()
    assert np.array_equal(y.view(np.int32), there.view(np.int32))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("new,kv", [([1, 1], [300, 400]), ([40, 1], [300, 400])])
def test_a_page_that_the_window_needs_is_still_missed(t, new, kv):
    c = Case(new, kv, t=t, page=16, window=100)
    own, _ = needed(c)
    c.pages[0, own[0] // 16] = -1
    c.pages[1, :own[1] // 16] = -1
    y = c.run()
    c.free()
    assert np.isnan(y[0]).all() and np.isfinite(y[c.start[1]:]).all()
