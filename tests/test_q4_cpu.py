"""CPU: the tests' Q4_0 quantizer against what the format says, and the library's
refusals of Q4_0 operands before any launch."""
import ctypes

import numpy as np
import pytest
import q4
from helpers import rng

from acestep_ops import _lib
from acestep_ops._lib import BF16, F16, F32, I32, Q4_0, Q8_0, MiTensor

R = ctypes.byref
L = _lib.load()
ES = {F32: 4, I32: 4, BF16: 2, F16: 2, Q8_0: 34, Q4_0: 18}


def _t(shape, typ=F32, data=4096, nb=None):
    """Descriptor with a fake (never dereferenced) data pointer."""
    es, ne = ES[typ], list(shape) + [1] * (4 - len(shape))
    d = MiTensor()
    d.data, d.type, d.reserved = data, typ, 0
    if nb is None:
        nb = [es, es * ne[0] // (32 if typ in (Q8_0, Q4_0) else 1)]
        nb += [nb[1] * ne[1], nb[1] * ne[1] * ne[2]]
    for i in range(4):
        d.ne[i], d.nb[i] = ne[i], nb[i]
    return d


def test_levels_and_scale():
    b = np.zeros((3, 32), np.float32)
    b[0, :16] = np.arange(16) - 8.0          # -8 is the largest magnitude: d = 1, levels 0..15
    b[1, 3], b[1, 9] = 4.0, -4.0             # equal magnitudes: the first one's sign, d = -0.5
    q = q4.quantize(b)
    assert (q[0, 2:] & 15).tolist() == list(range(16)) and (q[0, 2:] >> 4 == 8).all()
    assert q[1, :2].view(np.float16)[0] == -0.5
    assert np.array_equal(q4.dequantize(q)[0], b[0])
    v = q4.dequantize(q)[1]
    assert v[3] == 4.0 and v[9] == -3.5 and (np.delete(v, [3, 9]) == 0).all()  # level 16 is cut to 15
    assert q[2, :2].view(np.float16)[0] == 0 and (q4.dequantize(q)[2] == 0).all()  # d = 0 / -8 = -0


def test_error_is_half_a_step_but_at_the_cut_end():
    """|v - x| <= |d| / 2 (+ the fp16 rounding of d, 8 |d| 2^-11), a whole step where the cut end takes it."""
    x = rng(3).standard_normal((500, 32)).astype(np.float32)
    v, d = q4.dequantize(q4.quantize(x)), np.abs(x).max(1, keepdims=True).astype(np.float64) / 8
    assert (np.abs(v - x) <= d * (1 + 8 * 2.0 ** -11)).all()
    m = x[np.arange(len(x)), np.abs(x).argmax(1)][:, None]
    inner = x / m > -0.9375  # levels below 15.5 of 15
    assert (np.abs(v - x)[inner] <= np.broadcast_to(d, x.shape)[inner] * (0.5 + 8 * 2.0 ** -11 + 2.0 ** -20)).all()


def test_blocks_that_are_not_finite_stay_so():
    x = rng(4).standard_normal((3, 32)).astype(np.float32)
    x[0, 5], x[1, 7], x[2, 9] = np.nan, np.inf, -np.inf
    v = q4.dequantize(q4.quantize(x))
    assert not np.isfinite(v).any() and np.isnan(v[0]).all()
    assert v[1, 7] == np.inf and v[2, 9] == -np.inf


def test_copies_and_tables_refused():
    src, dst, ids = _t([128, 8, 4]), _t([128, 8, 4], Q4_0), _t([16], I32)
    assert L.mi_cpy(R(src), R(_t([128, 8, 5], Q4_0)), None) == -3
    assert L.mi_cpy(R(dst), R(_t([128, 8, 4])), None) == -2                       # from Q4_0: get_rows' work
    assert L.mi_cpy(R(src), R(_t([128, 8, 4], Q4_0, data=4097)), None) == -5
    assert L.mi_cpy(R(_t([100, 8])), R(_t([100, 8], Q4_0)), None) == -3           # not whole blocks
    assert L.mi_cpy(R(src), R(_t([128, 8, 4], Q4_0, nb=[34, 72, 576, 2304])), None) == -4
    assert L.mi_get_rows(R(_t([100, 50], Q4_0)), R(ids), R(_t([100, 16])), None, None) == -3
    assert L.mi_get_rows(R(_t([128, 50], Q4_0)), R(ids), R(_t([128, 16], F16)), None, None) == -2
    assert L.mi_rms_norm(R(_t([128, 8], Q4_0)), None, 1e-6, R(_t([128, 8])), None) == -2
    assert L.mi_swiglu_split(R(dst), R(dst), R(src), None) == -2


def test_kv_store_refused():
    k, pos0 = _t([128, 8, 3, 2]), _t([2], I32)
    cache = _t([128, 512, 8, 4], Q4_0)
    f = L.mi_kv_store
    assert f(R(k), R(_t([128, 512, 7, 4], Q4_0)), None, None, R(pos0), None, 0, None, None) == -3
    assert f(R(k), R(cache), R(k), R(_t([128, 512, 8, 4], Q8_0)), R(pos0), None, 0, None, None) == -3
    assert f(R(k), R(cache), None, None, R(pos0), None, 7, None, None) == -6
    assert f(R(k), R(_t([128, 512, 8, 4], Q4_0, data=4099)), None, None, R(pos0), None, 0, None, None) == -5


@pytest.mark.parametrize("typ,bsz", [(Q8_0, 34), (Q4_0, 18)])
def test_descriptors_of_block_views(typ, bsz):
    from acestep_ops import ops
    from acestep_ops.device import DTensor

    class Mem:
        ptr, nbytes = 1 << 20, 2 * 3 * 64 * 4 * bsz

    x = DTensor(Mem(), (2, 3, 64, 4 * bsz), "u8")
    w = (ops.Q8 if typ == Q8_0 else ops.Q4)(x[:, :, :40])
    d = ops.desc(w)
    assert d.type == typ and list(d.ne) == [128, 40, 3, 2]
    assert list(d.nb) == [bsz, 4 * bsz, 64 * 4 * bsz, 3 * 64 * 4 * bsz] and w.shape == (2, 3, 40, 128)
    with pytest.raises(ValueError):
        ops.desc((ops.Q4 if typ == Q8_0 else ops.Q8)(x))


def test_attention_refused():
    D, n_q, nh, nkv, n, N = 128, 3, 8, 2, 100, 2
    q, k, v, y = _t([D, n_q, nh, N], BF16), _t([D, n, nkv, N], Q4_0), _t([D, n, nkv, N], Q4_0), _t([D, nh, n_q, N])

    def fa(q=q, k=k, v=v, y=y, mask=None, scale=0.1):
        return L.mi_flash_attn_ext(R(q), R(k), R(v), R(mask) if mask else None, scale, 0.0, 0.0, R(y), None, 0, None)

    assert fa(v=_t([D, n, nkv, N], Q8_0)) == -2                                      # K and V of two types
    assert fa(y=_t([D, nh, n_q, N], F16)) == -2
    assert fa(q=_t([D, n_q, nh, N]), y=_t([D, nh, n_q, N], BF16)) == -2              # BF16 y needs BF16 q
    assert fa(k=_t([D, n, nkv, N], F16), v=_t([D, n, nkv, N], F16), y=_t([D, nh, n_q, N], BF16)) == -2
    assert fa(k=_t([D, n, nkv, N], Q4_0, data=4098)) == -5                           # rows at a 4-byte boundary
    assert fa(k=_t([D, n, nkv, N], Q4_0, nb=[18, 74, 7400, 14800])) == -5
    assert fa(q=_t([96, n_q, nh, N]), k=_t([96, n, nkv, N], Q4_0), v=_t([96, n, nkv, N], Q4_0), y=_t([96, nh, n_q, N])) == -7
    assert fa(k=_t([D, n, 3, N], Q4_0), v=_t([D, n, 3, N], Q4_0)) == -3
    assert fa(scale=float("nan")) == -6
    assert fa(mask=_t([n, n_q - 1, 1, 1], F16)) == -3
    big = _t([D, 1 << 28, nkv, N], Q4_0)
    assert fa(k=big, v=big) == -7
    # long caches with few heads are split: a workspace is needed
    one, long = _t([D, 1, nh, N]), _t([D, 20000, nkv, N], Q4_0)
    nb = ctypes.c_size_t(0)
    assert L.mi_flash_attn_ext_workspace(R(one), R(long), R(long), ctypes.byref(nb)) == 0 and nb.value > 0
    yo = _t([D, nh, 1, N])
    assert L.mi_flash_attn_ext(R(one), R(long), R(long), None, 0.1, 0.0, 0.0, R(yo), None, 0, None) == -6
    assert L.mi_flash_attn_ext(R(one), R(long), R(long), None, 0.1, 0.0, 0.0, R(yo), ctypes.c_void_p(4097),
                               nb.value, None) == -5
