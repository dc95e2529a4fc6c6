"""The prompts' kernel with more sequences than a wave has lanes."""
import numpy as np
import pytest

from tests.paged_cases import Case, close
from tests.test_gpu_paged_paths import dense

pytestmark = pytest.mark.gpu

TYPES = ["f16", "bf16", "f32"]
# rows of a kv head: 40 and more, of which 32 would take the tokens' kernel
FORMS = [dict(batch=70, new=5, kv=200, heads=16, kv_heads=2),     # eight waves a tile, merged
         dict(batch=130, new=5, kv=60, heads=32, kv_heads=4),     # tiles of 64 rows
         dict(batch=300, new=9, kv=40, heads=16, kv_heads=2),     # tiles of 128 rows
         dict(batch=70, new=6, kv=50, heads=16, kv_heads=2, prefix=100)]


def build(t, batch, new, kv, **kw):
    rows = [0 if i % 11 == 3 else 1 + (i * 5) % new for i in range(batch)]
    rows[batch // 2] = new
    return Case(rows, [n + (i * 7) % kv for i, n in enumerate(rows)], t=t, head=64, page=16, **kw)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("mod", [{}, dict(window=30, bias=True)])
def test_many_prompts(t, form, mod):
    c = build(t, **form, **mod)
    assert c.max_q * c.heads // c.kv_heads > 32 and len(c.kv) > 64
    want, tol = dense(c)
    y = c.run()
    c.free()
    close(y, want, tol)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("form", FORMS)
def test_one_that_breaks_the_promises(t, form):
    c = build(t, **form)
    want, tol = dense(c)
    b = len(c.kv) - 5
    assert c.new[b] > 0
    c.kv_len[b] = -1
    y = c.run()
    c.free()
    lost = np.zeros(c.tokens, bool)
    lost[c.start[b]:c.start[b + 1]] = True
    assert np.isnan(y[lost]).all()
    close(y[~lost], want[~lost], tol[~lost])
