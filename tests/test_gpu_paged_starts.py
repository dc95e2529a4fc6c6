"""Row starts that do not rise: the sequence that ends before it begins gets nothing, and the
others' rows and pages are as ever."""
import pytest

from tests.paged_cases import Case, close
from tests.test_gpu_paged_append import run, same, want
from tests.test_gpu_paged_paths import dense

pytestmark = pytest.mark.gpu

TYPES = ["f16", "bf16", "f32"]


def broken(c, to):
    """The last sequence, which has no rows, ends at row `to`."""
    assert c.start[-1] == c.start[-2] == c.tokens
    c.start[-1] = to
    return c


BATCHES = [([10, 2, 0], [40, 60, 20], 3), ([3, 1, 0], [7, 5, 5], 1), ([1] * 70 + [0], [9] * 71, 0),
           ([2] * 300 + [0], [30] * 301, 17)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("new,kv,to", BATCHES)
def test_append(t, new, kv, to):
    c = broken(Case(new, kv, t=t, head=32, heads=2, kv_heads=1, page=8), to)
    ins, got = run(c, 16)
    same(got, want(c, ins), t)
    c.free()


def check(c, to):
    exp, tol = dense(c)
    y = broken(c, to).run()
    c.free()
    close(y, exp, tol)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("new,kv,to", BATCHES)
def test_tokens(t, new, kv, to):
    check(Case(new, kv, t=t), to)
    # keys cut between waves, whose pieces are merged
    check(Case(new, [n + 400 for n in kv], t=t, page=64), to)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("new,kv,to", [([40, 7, 0], [50, 60, 20], 3), ([40] * 3 + [0], [900] * 4, 0)])
def test_prompts(t, new, kv, to):
    check(Case(new, kv, t=t), to)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("mod", [{}, dict(window=40, bias=True)])
@pytest.mark.parametrize("new,kv,to,prefix,heads,kv_heads", [
    ([10, 2, 0], [40, 60, 20], 3, 300, 4, 2), ([1] * 70 + [0], [9] * 71, 0, 300, 4, 2),
    ([1] * 32 + [0], [9] * 33, 5, 3000, 64, 16), ([1] * 70 + [0], [9] * 71, 5, 3000, 64, 16)])
def test_behind_a_prefix(t, mod, new, kv, to, prefix, heads, kv_heads):
    check(Case(new, kv, t=t, prefix=prefix, heads=heads, kv_heads=kv_heads, **mod), to)
