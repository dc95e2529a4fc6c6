"""An error that a call has reported is not the next call's."""
import pytest

from onnx_runtime_dart_amd import _lib
from tests.paged_cases import Case, close

pytestmark = pytest.mark.gpu


def test_a_call_after_one_that_ran_out_of_memory():
    c = Case([1, 3], [40, 50])
    call = c.device()
    with pytest.raises(MemoryError):
        _lib.default_context().alloc(1 << 50)
    call()
    want, tol = c.want()
    close(c.read(), want, tol)
    c.free()
