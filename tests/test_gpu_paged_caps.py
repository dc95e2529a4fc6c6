"""Caps and scales far from a score's own size."""
import numpy as np
import pytest

from tests.paged_cases import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("new,kv", [([1, 1, 3], [40, 300, 90]), ([70, 5], [70, 140])])
@pytest.mark.parametrize("cap", [1e-42, 1e-30, 1e20, 1e30, 1e35, 3.4e38])
def test_caps(t, new, kv, cap):
    cap = float(np.float32(cap))
    c = Case(new, kv, t=t, cap=cap)
    c.q[0] = 0.0  # products of zero
    y = c.run()
    # past every score a cap changes nothing; below all of them all weights are alike
    d = Case(new, kv, t=t, cap=0.0 if cap > 1 else cap)
    d.q[0] = 0.0
    want, tol = d.want()
    c.free()
    d.free()
    assert np.isfinite(y).all()
    off = float((np.abs(y - want) / tol).max())
    print(f"{off:.3g} of the tolerance", flush=True)
    assert off <= 1.0


@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("scale", [1e-44, 1e-30])
def test_scales_that_leave_all_weights_alike(t, scale):
    Case([1, 40], [40, 90], t=t, scale=float(np.float32(scale))).check()
