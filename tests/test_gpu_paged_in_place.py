"""Queries turned in place in a row of projections, through the public calls."""
import numpy as np
import pytest

from onnx_runtime_dart_amd import paged
from tests.paged_cases import Case
from tests.test_gpu_paged_append import tables, want

pytestmark = pytest.mark.gpu


def setup(c, half):
    """The call's arguments with a row of queries, keys and values, and what it is to give."""
    H, G, D, T = c.heads, c.kv_heads, c.head, c.tokens
    x = np.random.default_rng(3).standard_normal((T, H + 2 * G, D)).astype(np.float32)
    cos, sin = tables(c.max_kv, half)
    buf, ld = c.put(x), (H + 2 * G) * D
    at = buf.ptr.value
    args = (c.cache(), c.batch(), at, at + 4 * H * D, at + 4 * (H + G) * D, c.put(cos), c.put(sin))
    kw = dict(heads=H, max_pos=c.max_kv, half_rot=half, ldq=ld, ldk=ld, ldv=ld, ctx=c.ctx)
    return buf, args, kw, want(c, (x[:, :H], x[:, H:H + G], x[:, H + G:], cos, sin))[0]


@pytest.mark.parametrize("half", [32, 5])
def test_in_place_without_an_output_stride(half):
    c = Case([40, 3, 300], [41, 90, 300])
    buf, args, kw, y = setup(c, half)
    paged.append(*args, args[2], **kw)
    c.ctx.synchronize()
    assert np.array_equal(buf.numpy()[:, :c.heads], y)
    c.free()


def test_another_rows_place_is_refused_and_nothing_is_written():
    c = Case([40, 3], [41, 90])
    buf, args, kw, _ = setup(c, 32)
    before = buf.numpy()
    for out, ldqo in ((args[2], kw["ldq"] - 8), (args[2], c.heads * c.head),
                      (args[2] + 4 * kw["ldq"], kw["ldq"]), (args[2] + 16, kw["ldq"])):
        with pytest.raises(ValueError, match="overlaps"):
            paged.append(*args, out, ldqo=ldqo, **kw)
    c.ctx.synchronize()
    assert np.array_equal(buf.numpy(), before)
    c.free()
