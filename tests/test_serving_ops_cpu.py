"""CPU: what mi_lora_add and mi_logits_adjust refuse, before any launch."""
import ctypes

from acestep_ops import _lib
from acestep_ops._lib import BF16, F16, F32, I32, MiTensor

R = ctypes.byref
L = _lib.load()
ES = {F32: 4, I32: 4, BF16: 2, F16: 2}


def _t(shape, typ=F32, data=1 << 20, nb=None):
    """Descriptor with a fake (never dereferenced) data pointer."""
    es, ne = ES[typ], list(shape) + [1] * (4 - len(shape))
    d = MiTensor()
    d.data, d.type, d.reserved = data, typ, 0
    nb = nb or [es, es * ne[0], es * ne[0] * ne[1], es * ne[0] * ne[1] * ne[2]]
    for i in range(4):
        d.ne[i], d.nb[i] = ne[i], nb[i]
    return d


def _p(t):
    return None if t is None else R(t)


def test_lora_add():
    m, k, n, r, e = 7, 64, 96, 8, 3
    ok = dict(y0=_t([n, m]), x=_t([k, m], data=2 << 20), a=_t([k, r, e], BF16), b=_t([r, n, e], BF16), ids=_t([m], I32),
              scales=_t([e]), y=_t([n, m], data=3 << 20))
    ws = ctypes.c_size_t(0)
    assert L.mi_lora_add_workspace(R(ok["x"]), R(ok["a"]), R(ok["b"]), ctypes.byref(ws)) == 0 and ws.value >= m * 16 * 4
    assert L.mi_lora_add_workspace(R(ok["x"]), R(ok["a"]), R(ok["b"]), None) == -1

    def f(wp=16 << 20, wn=None, err=None, **kw):
        t = {**ok, **kw}
        return L.mi_lora_add(_p(t["y0"]), _p(t["x"]), _p(t["a"]), _p(t["b"]), _p(t["ids"]), _p(t["scales"]), _p(t["y"]),
                             wp, ws.value if wn is None else wn, err, None)

    for name in ("y0", "x", "a", "b", "ids", "y"):
        assert f(**{name: None}) == -1, name
    assert f(x=_t([k, m], BF16)) == -2 and f(y=_t([n, m], BF16, data=3 << 20)) == -2
    assert f(a=_t([k, r, e]), b=_t([r, n, e])) == -2                   # F32 weights
    assert f(b=_t([r, n, e], F16)) == -2                               # two types
    assert f(ids=_t([m])) == -2 and f(scales=_t([e], BF16)) == -2
    assert f(ids=_t([m + 1], I32)) == -3 and f(scales=_t([e + 1])) == -3
    assert f(b=_t([r + 1, n, e], BF16)) == -3 and f(b=_t([r, n, e + 1], BF16)) == -3
    assert f(a=_t([k + 32, r, e], BF16)) == -3 and f(y0=_t([n + 1, m])) == -3 and f(y=_t([n, m + 1], data=3 << 20)) == -3
    assert f(x=_t([40, m]), a=_t([40, r, e], BF16)) == -3              # k not a multiple of 32
    assert f(x=_t([k, 7, 1, 2], nb=[4, 4 * k, 28 * k, 100 * k])) == -3  # rows at two distances
    assert f(a=_t([k, 257, e], BF16), b=_t([257, n, e], BF16)) == -7
    assert f(a=_t([k, r, e], BF16, nb=[4, 256, 2048, 6144])) == -4
    assert f(wn=ws.value - 1) == -6 and f(wp=None) == -6 and f(wp=(16 << 20) + 8) == -5 and f(err=4098) == -5
    assert f(y=_t([n, m], data=2 << 20)) == -6                          # y over x
    assert f(y=_t([n, m], data=(1 << 20) + 4 * n)) == -6                # y one row into y0
    assert f(y=_t([n, m], nb=[4, 8 * n, 56 * n, 56 * n])) == -6         # y0's start at another distance
    # nothing to do
    assert f(x=_t([k, 0]), y0=_t([n, 0]), y=_t([n, 0]), ids=_t([0], I32)) == 0


def test_logits_adjust():
    m, V, n = 4, 100, 20
    ok = dict(logits=_t([V, m]), history=_t([n, m], I32), lengths=_t([m], I32), penalties=_t([3, m]), bias=_t([V, m]),
              allowed=_t([4, 2], I32), state=_t([m], I32), y=_t([V, m], data=3 << 20))

    def f(err=None, **kw):
        t = {**ok, **kw}
        return L.mi_logits_adjust(*[_p(t[x]) for x in ("logits", "history", "lengths", "penalties", "bias", "allowed",
                                                       "state", "y")], err, None)

    assert f(logits=None) == -1 and f(y=None) == -1
    assert f(history=None) == -1 and f(penalties=None) == -1 and f(allowed=None) == -1  # one of a pair
    assert f(history=None, penalties=None) == -1                                        # lengths of nothing
    assert f(y=_t([V, m], BF16, data=3 << 20)) == -2 and f(logits=_t([V, m], I32), y=_t([V, m], I32, data=3 << 20)) == -2
    assert f(history=_t([n, m])) == -2 and f(penalties=_t([3, m], BF16)) == -2 and f(bias=_t([V, m], BF16)) == -2
    assert f(allowed=_t([4, 2])) == -2 and f(state=_t([m])) == -2 and f(lengths=_t([m])) == -2
    assert f(y=_t([V, m + 1], data=3 << 20)) == -3 and f(history=_t([n, m + 1], I32)) == -3
    assert f(penalties=_t([2, m])) == -3 and f(penalties=_t([3, 1])) == -3
    assert f(bias=_t([V, 2])) == -3 and f(bias=_t([V - 1, m])) == -3
    assert f(allowed=_t([3, 2], I32)) == -3 and f(state=_t([m - 1], I32)) == -3 and f(lengths=_t([m - 1], I32)) == -3
    assert f(state=None) == -3                                   # 2 states for 4 rows, and no row says which
    assert f(logits=_t([V, m, 2]), y=_t([V, m, 2], data=3 << 20)) == -3
    assert f(y=_t([V, m], data=(1 << 20) + 4)) == -6             # shifted over its input
    assert f(err=4098) == -5 and f(logits=_t([V, m], data=(1 << 20) + 2)) == -5
    big = [_t([V, 70000], data=d << 30) for d in (1, 2)]
    assert L.mi_logits_adjust(R(big[0]), None, None, None, None, None, None, R(big[1]), None, None) == -7
    assert L.mi_logits_adjust(R(_t([0, m])), None, None, None, None, None, None, R(_t([0, m])), None, None) == 0


def test_sizes_past_32_bits():
    """Rows, tokens and places that the kernels' 32-bit counters could not hold (views of one row at stride 0)."""
    big = 1 << 31
    x = _t([64, big - 1], nb=[4, 0, 0, 0])
    ws = ctypes.c_size_t(0)
    assert L.mi_lora_add_workspace(R(x), R(_t([64, 8, 1], BF16)), R(_t([8, 32, 1], BF16)), ctypes.byref(ws)) == -7
    one = _t([1 << 30 | 32, 1], BF16)
    assert L.mi_logits_adjust(R(one), None, None, None, None, None, None, R(one), None, None) == -7
    lg, pen = _t([64, 2]), _t([3, 2])
    for n in (1 << 30 | 1, big - 1):
        assert L.mi_logits_adjust(R(lg), R(_t([n, 2], I32)), None, R(pen), None, None, None, R(lg), None, None) == -7
    assert L.mi_logits_adjust(R(_t([8, 65536])), None, None, None, None, None, None, R(_t([8, 65536])), None, None) == -7
