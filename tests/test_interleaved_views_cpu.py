"""CPU: y may be other columns of the buffer that holds x or y0; only views that share bytes are refused."""
import ctypes

from acestep_ops import _lib
from acestep_ops._lib import BF16, I32
from test_serving_ops_cpu import _t

R = ctypes.byref
L = _lib.load()
BASE = 1 << 20


def test_adapters_on_columns_of_one_buffer():
    m, k, n, r, P = 7, 64, 96, 8, 400  # rows of 400 floats

    def col(at, w, rows=m, pitch=P):
        return _t([w, rows], data=BASE + 4 * at, nb=[4, 4 * pitch, 4 * pitch * rows, 4 * pitch * rows])

    def f(y0, x, y, rows=m):
        # a workspace that is not aligned: what no overlap refuses (-6) is refused for it (-5), before any launch
        return L.mi_lora_add(R(y0), R(x), R(_t([k, r, 1], BF16)), R(_t([r, n, 1], BF16)), R(_t([rows], I32)), None, R(y),
                             (16 << 20) + 8, 1 << 30, None, None)

    far = _t([k, m], data=64 << 20)
    assert f(col(0, n), col(200, k), col(100, n)) == -5             # x, y0 and y side by side
    assert f(col(0, n), col(96, k), col(160, n)) == -5              # touching
    assert f(col(100, n), col(300, k), col(0, n)) == -5             # y before y0
    assert f(col(100, n), col(P + 100, k), col(P, n)) == -5         # y one row on, before y0's columns
    assert f(col(304, n), far, col(P, n)) == -5                     # y0 up to the row's end
    assert f(col(0, n), col(200, k), col(104 + 36, n)) == -6        # y's last columns are x's first
    assert f(col(0, n), col(200, k), col(95, n)) == -6              # y's first column is y0's last
    assert f(col(305, n), far, col(P, n)) == -6                     # y0 reaches into the next row of y
    assert f(col(0, n), far, col(P, n)) == -6                       # y0 one row on
    assert f(col(0, n), far, col(100, n, pitch=401)) == -6          # two distances
    assert f(col(100, n), far, col(0, n, rows=0), rows=0) == -3     # no row, but y0 has some
