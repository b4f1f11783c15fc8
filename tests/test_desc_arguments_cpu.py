"""What acestep_ops.ops makes of operands that are not plain DTensors over one lasting buffer."""
import gc
import weakref

from acestep_ops import ops
from acestep_ops._lib import F32, Q4_0, Q8_0
from acestep_ops.device import DTensor


class Mem:
    ptr, nbytes = 1 << 20, 4096


def fields(t):
    a = ops._p(t)._obj
    return a.data, a.type, list(a.ne), list(a.nb)


def test_subclasses_and_look_alikes():
    class Named(DTensor):
        pass

    class View:  # what a view needs, and nothing to keep an argument in
        __slots__ = ("buf", "shape", "dtype", "strides", "offset")

        def __init__(self, shape):
            self.buf, self.shape, self.dtype, self.strides, self.offset = Mem(), shape, "f32", (shape[1], 1), 0

    class Blocks(ops.Q4):
        pass

    want = (1 << 20, F32, [8, 3, 1, 1], [4, 32, 96, 96])
    assert fields(DTensor(Mem(), (3, 8), "f32")) == want
    assert fields(Named(Mem(), (3, 8), "f32")) == want
    v = View((3, 8))
    assert fields(v) == want
    v.offset = 32
    assert fields(v) == (want[0] + 32, *want[1:])
    assert fields(Blocks(DTensor(Mem(), (3, 36), "u8")))[1:3] == (Q4_0, [64, 3, 1, 1])
    assert fields(ops.Q8(Named(Mem(), (3, 68), "u8")))[1:3] == (Q8_0, [64, 3, 1, 1])


def test_a_kept_argument_keeps_no_buffer():
    class Buf:
        ptr, nbytes = 1 << 20, 4096

    x = DTensor(Buf(), (4, 8), "f32")
    first = ops._p(x)
    assert ops._p(x) is first
    old = weakref.ref(x.buf)
    x.buf = Buf()
    gc.collect()
    assert old() is None
    x.buf.ptr = 1 << 21
    assert fields(x)[0] == 1 << 21


def test_lists_changed_in_place():
    x = DTensor(Mem(), (4, 8), "f32")
    x.shape = [4, 8]
    assert fields(x)[2] == [8, 4, 1, 1]
    x.shape[0] = 2
    assert fields(x)[2] == [8, 2, 1, 1]


def test_a_view_past_a_smaller_buffer_is_still_refused():
    import pytest

    x = DTensor(Mem(), (4, 256), "f32")
    ops._p(x)
    x.buf = Mem()
    x.buf.nbytes = 4095
    with pytest.raises(ValueError):
        ops._p(x)
