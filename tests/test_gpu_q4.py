"""GPU parity, bit-exact: Q4_0 quantization through mi_cpy, mi_kv_store and
mi_qk_norm_rope_kv_store, and mi_get_rows of Q4_0 tables, against the fp32
operations of the format one by one (q4.py)."""
import numpy as np
import pytest
import q4
from helpers import randn, rng, to_dev, to_np
from oracle import oracle as orc

from acestep_ops import ops
from acestep_ops.device import DTensor, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu


def _up(x, dt):
    """(device tensor, the F32 values it holds)"""
    if dt == "bf16":
        h = orc.f32_to_bf16(x)
        return to_dev(h, bf16=True), orc.bf16_to_f32(h)
    if dt == "f16":
        h = x.astype(np.float16)
        return to_dev(h.view(np.uint16), f16=True), h.astype(np.float32)
    return to_dev(x), x


def _blocks():
    """Blocks where levels fall on a border, magnitudes tie, or scales leave fp16."""
    r = rng(5)
    b = [np.arange(32) - 16.0, np.arange(32) * -0.25, np.zeros(32), np.full(32, -0.0), np.full(32, 3.0),
         np.where(np.arange(32) % 2, 2.0, -2.0), np.where(np.arange(32) % 2, -2.0, 2.0)]
    for at in (0, 15, 16, 31):  # one large value, in each lane's share
        x = r.standard_normal(32) * 0.1
        x[at] = -5.0
        b.append(x)
    for s in (1e-9, 1e-40, 1e-44, 3e5, 3e38, 6e-8):  # subnormal and overflowing scales
        b.append(r.standard_normal(32).clip(-1, 1) * s)
    for bad in (np.nan, np.inf, -np.inf):
        for at in (2, 20):
            x = r.standard_normal(32)
            x[at] = bad
            b.append(x)
    b.append(np.repeat([7.5, -7.5, 8.0, -8.0], 8))  # levels exactly between two
    with np.errstate(over="ignore"):
        return np.stack(b).astype(np.float32)


def _same_blocks(got, want):
    """The same bytes, but for the payload of a NaN scale and the levels beside it (they all read back as NaN)."""
    g, w = got.reshape(-1, 18), want.reshape(-1, 18)
    gd, wd = g[:, :2].copy().view(np.float16)[:, 0], w[:, :2].copy().view(np.float16)[:, 0]
    assert np.array_equal(np.isnan(gd), np.isnan(wd))
    ok = ~np.isnan(wd)
    bad = np.nonzero((g[ok] != w[ok]).any(1))[0]
    assert bad.size == 0, f"{bad.size} blocks differ, the first {np.nonzero(ok)[0][bad[:3]]}: {g[ok][bad[:1]]} {w[ok][bad[:1]]}"


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_cpy_special_blocks(dev, dt):
    d, x = _up(_blocks(), dt)
    dst = ops.Q4(DTensor.zeros((x.shape[0], 18), "u8"))
    ops.cpy(d, dst)
    _same_blocks(to_np(dst.data), q4.quantize(x))


@pytest.mark.parametrize("rows,n", [(1, 32), (5, 96), (700, 128), (33, 2560)])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("odd", [False, True])
def test_cpy_shapes(dev, rows, n, dt, odd):
    """Rows into a wider destination; `odd`: source rows that no 16-byte load reaches (the generic kernel)."""
    print(f"cpy q4_0 {rows}x{n} {dt} odd={odd}", flush=True)
    pad = 1 if odd else 16
    d, x = _up(randn((rows, n + pad), seed=n + rows), dt)
    wide = DTensor.full_byte((rows, n // 32 * 18 + 6), 0x77)
    dst = ops.Q4(wide[:, :n // 32 * 18])
    ops.cpy(d[:, pad:], dst)
    got = to_np(wide)
    _same_blocks(got[:, :n // 32 * 18], q4.quantize(np.ascontiguousarray(x[:, pad:])))
    assert (got[:, n // 32 * 18:] == 0x77).all()


def _kv_case(dt, D, B, T, Nkv, seed, bad=False):
    max_seq, n_sets = T + 37, B + 2
    k, kx = _up(randn((B, T, Nkv, D), seed=seed), dt)
    v, vx = _up(randn((B, T, Nkv, D), seed=seed + 1), dt)
    r = rng(seed)
    pos0 = r.integers(0, max_seq - T + 1, B).astype(np.int32)
    sets = r.permutation(n_sets)[:B].astype(np.int32)
    if bad:
        pos0[0], sets[-1] = max_seq - T + 1, -1
    kc = ops.Q4(DTensor.full_byte((n_sets, Nkv, max_seq, D // 32 * 18), 0xA5))
    vc = ops.Q4(DTensor.full_byte((n_sets, Nkv, max_seq, D // 32 * 18), 0x5A))
    want = [np.full((n_sets, Nkv, max_seq, D // 32 * 18), f, np.uint8) for f in (0xA5, 0x5A)]
    errs = 0
    for b in range(B):
        for t in range(T):
            if not (0 <= pos0[b] + t < max_seq and 0 <= sets[b] < n_sets):
                errs += 2 * Nkv
                continue
            want[0][sets[b], :, pos0[b] + t] = q4.quantize(kx[b, t])
            want[1][sets[b], :, pos0[b] + t] = q4.quantize(vx[b, t])
    return k, v, pos0, sets, kc, vc, want, errs


@pytest.mark.parametrize("D,B,T,Nkv", [(128, 1, 1, 8), (128, 8, 1, 8), (64, 3, 19, 2), (256, 2, 33, 1), (128, 2, 130, 5),
                                       (32, 2, 3, 3), (96, 1, 7, 2)])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_kv_store(dev, D, B, T, Nkv, dt):
    """Every byte of both caches: the rows written, and every other row left as it was."""
    print(f"kv_store q4_0 D={D} B={B} T={T} Nkv={Nkv} {dt}", flush=True)
    k, v, pos0, sets, kc, vc, want, _ = _kv_case(dt, D, B, T, Nkv, seed=D + T)
    ops.kv_store(k, kc, to_dev(pos0), v, vc, to_dev(sets))
    for c, w in zip((kc, vc), want):
        _same_blocks(to_np(c.data), w)


def test_kv_store_bad_slots_are_counted(dev):
    k, v, pos0, sets, kc, vc, want, errs = _kv_case("f32", 128, 3, 4, 2, seed=9, bad=True)
    err = DTensor.zeros((1,), "i32")
    ops.kv_store(k, kc, to_dev(pos0), v, vc, to_dev(sets), err=err)
    assert int(err.item()) == errs > 0
    for c, w in zip((kc, vc), want):
        _same_blocks(to_np(c.data), w)


@pytest.mark.parametrize("n,n_ids", [(32, 1), (64, 77), (96, 333), (128, 4099), (2560, 64)])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_get_rows(dev, n, n_ids, out):
    """Strided ids, padded output rows, ids that name no row (zeros, counted)."""
    print(f"get_rows q4_0 n={n} ids={n_ids} {out}", flush=True)
    n_rows = 500
    tab = q4.quantize(randn((n_rows, n), seed=n + n_ids))
    ids2 = rng(n_ids).integers(0, n_rows, (n_ids, 2)).astype(np.int32)
    bad = np.arange(n_ids) % 97 == 5
    ids2[bad, 0] = np.where(np.arange(bad.sum()) % 2 == 0, -3, n_rows)
    yfull = DTensor.full_byte((n_ids, n + 8), 0x7F, out)
    err = DTensor.zeros((1,), "i32")
    ops.get_rows(ops.Q4(to_dev(tab)), to_dev(ids2)[:, 0], out=yfull[:, :n], err=err)
    got = to_np(yfull)
    ref = np.zeros((n_ids, n), np.float32)
    ref[~bad] = q4.dequantize(tab)[ids2[~bad, 0]].astype(np.float32)  # exact in fp32
    if out == "bf16":
        ref = orc.f32_to_bf16(ref)
    assert np.array_equal(got[:, :n].view(np.uint8), ref.view(np.uint8))
    assert (np.ascontiguousarray(got[:, n:]).view(np.uint8) == 0x7F).all()
    assert int(err.item()) == int(bad.sum())


@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_get_rows_all_levels_and_scales_any_alignment(dev, out):
    """Every level with scales of every kind, into output rows that no 16-byte store reaches."""
    scales = np.array([0x0000, 0x0001, 0x03FF, 0x0400, 0x3C00, 0x7BFF, 0x8001, 0xBC00, 0x7C00, 0x7E00], np.uint16)
    row = np.zeros((len(scales), 18), np.uint8)
    row[:, :2] = scales.view(np.uint8).reshape(-1, 2)
    row[:, 2:] = np.arange(16) | (15 - np.arange(16)) << 4
    ids = np.arange(len(scales), dtype=np.int32)
    y = DTensor.zeros((len(scales), 33), out)[:, 1:]
    ops.get_rows(ops.Q4(to_dev(row)), to_dev(ids), out=y)
    with np.errstate(invalid="ignore"):
        ref = q4.dequantize(row).astype(np.float32)
    got = to_np(y) if out == "f32" else orc.bf16_to_f32(to_np(y))
    ref = ref if out == "f32" else orc.bf16_to_f32(orc.f32_to_bf16(ref))
    assert np.array_equal(got, ref, equal_nan=True)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("D,B,T,nh,nkv", [(128, 8, 1, 32, 8), (64, 2, 5, 4, 2), (256, 1, 7, 4, 1), (128, 2, 65, 16, 5)])
@pytest.mark.parametrize("clamp", [False, True])
def test_qk_norm_rope_kv_store(dev, dt, D, B, T, nh, nkv, clamp):
    """One launch against the three calls it stands for: q_out, both caches and the count of bad slots, bit for bit."""
    print(f"qk_norm_rope_kv_store q4_0 {dt} D={D} B={B} T={T} {nh}/{nkv} clamp={clamp}", flush=True)
    n = B * T
    x = randn((n, (nh + 2 * nkv) * D), seed=D + T)
    x[:, (nh + nkv) * D::97] *= 1e5 if clamp else 1.0
    xd, _ = _up(x, dt)
    q = xd[:, :nh * D].unflatten(1, (nh, D))
    k = xd[:, nh * D:(nh + nkv) * D].unflatten(1, (nkv, D))
    v = xd[:, (nh + nkv) * D:].unflatten(1, (nkv, D))
    qw, kw = to_dev(randn(D, seed=1, scale=0.1, mean=1.0)), to_dev(randn(D, seed=2, scale=0.1, mean=1.0))
    pos = to_dev(rng(3).integers(0, 8192, n).astype(np.int32))
    pos0, sets = np.arange(B, dtype=np.int32), np.arange(B, 0, -1).astype(np.int32)
    sets[0] = B + 9  # the first sequence has no such set
    got = []
    for fused in (False, True):
        kc, vc = (ops.Q4(DTensor.full_byte((B + 1, nkv, T + B, D // 32 * 18), f)) for f in (0xA5, 0x5A))
        err = DTensor.zeros((1,), "i32")
        if fused:
            qo = ops.qk_norm_rope_kv_store(q, qw, k, kw, v, pos, 1e-6, D, 1e6, kc, vc, to_dev(pos0), sets=to_dev(sets),
                                           clamp_v=clamp, err=err)
        else:
            qo, ko = ops.qk_norm_rope(q, qw, pos, 1e-6, D, 1e6, k=k, k_w=kw)
            vs = ops.add_clamp(v, None, -65504.0, 65504.0) if clamp else v
            ops.kv_store(ko.unflatten(0, (B, T)), kc, to_dev(pos0), v=vs.unflatten(0, (B, T)), v_cache=vc, sets=to_dev(sets),
                         err=err)
        got.append([to_np(t) for t in (qo, kc.data, vc.data, err)])
    for a, b in zip(*got):
        assert np.array_equal(a, b)
    assert got[1][3][0] == 2 * nkv * T


def test_store_and_read_back_in_a_graph(dev):
    """A captured store and read-back, replayed with new inputs between eager work."""
    st = Stream()
    k = DTensor.zeros((2, 3, 4, 128))
    pos0 = DTensor.zeros((2,), "i32")
    kc = ops.Q4(DTensor.zeros((2, 4, 16, 72), "u8"))
    rows = ops.Q4(kc.data.view(-1, 72))
    ids, y = to_dev(np.arange(2 * 4 * 16, dtype=np.int32)), DTensor.zeros((128, 128))
    g = Graph()
    with g.capture(st):
        ops.kv_store(k, kc, pos0, stream=st.handle)
        ops.get_rows(rows, ids, out=y, stream=st.handle)
    from acestep_ops.device import D2D, check, hip

    for i in range(3):
        x = randn((2, 3, 4, 128), seed=40 + i)
        src = to_dev(x)
        check(hip().hipMemcpy(k.ptr, src.ptr, x.nbytes, D2D), "hipMemcpy")
        synchronize()
        g.launch()
        st.synchronize()
        want = np.zeros((2, 4, 16, 128), np.float32)
        want[:, :, :3] = q4.dequantize(q4.quantize(x)).transpose(0, 2, 1, 3)
        assert np.array_equal(to_np(y).reshape(want.shape), want)
