"""``_native.empty``: device arrays to write results into, on the CPU with the
stand-in for the library."""
import numpy as np
import pytest

from macmetalpy_amd import _gate
from test_native_gate import stub  # noqa: F401  (a fixture)

F16, F32, F64, I64 = (np.dtype(t) for t in (np.float16, np.float32, np.float64, np.int64))


@pytest.mark.parametrize("shape,dt", [((), F32), ((3, 4), F16), ((0, 5), F64), ((1 << 40, 1 << 40, 0), I64)])
def test_empty(stub, shape, dt):  # noqa: F811
    a = _gate._native.empty(shape, dt)
    assert a.shape == shape and a.dtype == dt and a.size == np.prod(shape, dtype=object)
    assert a._buffer.nbytes == a.size * dt.itemsize and a._offset == 0 and a._base is None


@pytest.mark.parametrize("shape,dt", [((1 << 32, 1 << 32), F16), ((1 << 31, 1 << 30), F64),
                                      ((1 << 62, 4), F32), ((1 << 20, 1 << 20, 1 << 24), F32),
                                      ((1 << 63, 1), F32), (((1 << 61) + 1,), F64)])
def test_empty_refuses_what_no_memory_holds(stub, shape, dt):  # noqa: F811
    """Sizes past 64 bits are an error, not what is left of them."""
    live = stub.stub_live()
    with pytest.raises(MemoryError):
        _gate._native.empty(shape, dt)
    assert stub.stub_live() == live


@pytest.mark.parametrize("args", [((3,), np.dtype("c8")), ([3], F32), ((3.0,), F32), ((3,),)])
def test_empty_refuses_other_arguments(stub, args):  # noqa: F811
    with pytest.raises(TypeError):
        _gate._native.empty(*args)
