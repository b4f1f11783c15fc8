"""GPU: low-rank adapters of many requests (mi_lora_add) against 64 bits, within the bound of the
kernels' arithmetic, u = 2^-24: x and h as three bf16 parts, u each (8 + 8 + 8 bits); F16 weights as two,
the product of both last parts left out, u; sums of up to 5 products a term in fp32,
8 sqrt(5 n) u (the probabilistic bound of Higham and Mary); the scale, y0's addition and y, u each."""
import numpy as np
import pytest
from helpers import randn, rng, to_dev, to_np
from oracle import oracle as orc

from acestep_ops import ops
from acestep_ops.device import DTensor, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _w(x, dt):
    """(device tensor, the values it holds in 64 bits)"""
    if dt == "bf16":
        h = orc.f32_to_bf16(x)
        return to_dev(h, bf16=True), orc.bf16_to_f32(h).astype(np.float64)
    h = x.astype(np.float16)
    return to_dev(h.view(np.uint16), f16=True), h.astype(np.float64)


def _ref(y0, x, a, b, ids, scales):
    """(y, bound) in 64 bits"""
    m, k = x.shape
    r = a.shape[1]
    y = y0.astype(np.float64).copy()
    bound = np.zeros_like(y)
    for i in range(m):
        j = ids[i]
        if not 0 <= j < len(a):
            continue
        xi, s = x[i].astype(np.float64), 1.0 if scales is None else float(scales[j])
        h, ha = a[j] @ xi, np.abs(a[j]) @ np.abs(xi)
        dh = (2 + 8 * np.sqrt(5.0 * k)) * U * ha
        y[i] += s * (b[j] @ h)
        bound[i] = abs(s) * (np.abs(b[j]) @ (dh + (4 + 8 * np.sqrt(5.0 * r)) * U * np.abs(h)))
        bound[i] += 2 * U * (np.abs(y[i]) + np.abs(y0[i])) + 1e-37
    return y, bound


def _check(got, y0, x, a, b, ids, scales):
    ref, bound = _ref(y0, x, a, b, ids, scales)
    err = np.abs(got.astype(np.float64) - ref)
    none = (np.asarray(ids) < 0) | (np.asarray(ids) >= len(a))
    assert np.array_equal(got[none], y0[none]), "rows without an adapter"
    assert np.isfinite(got).all() and (err <= bound).all(), f"off by {err.max():.3g}, {np.max(err / bound):.3g} of the bound"
    live = bound > 0
    print(f"  worst {np.max(err[live] / bound[live]) if live.any() else 0:.3g} of the bound", flush=True)


def _case(m, k, n, r, e, dt, seed, ids=None):
    x, y0 = randn((m, k), seed=seed), randn((m, n), seed=seed + 1)
    a, ah = _w(randn((e, r, k), seed=seed + 2, scale=k ** -0.5), dt)
    b, bh = _w(randn((e, n, r), seed=seed + 3, scale=r ** -0.5), dt)
    ids = rng(seed).integers(-1, e, m).astype(np.int32) if ids is None else np.asarray(ids, np.int32)
    scales = (rng(seed + 4).random(e) + 0.5).astype(np.float32)
    return x, y0, a, ah, b, bh, ids, scales


def _run(x, y0, a, b, ids, scales, out=None, err=None):
    xd, yd = to_dev(x), to_dev(y0)
    ws = DTensor.full_byte((max(ops.lora_add_workspace(xd, a, b), 16),), 0xFF)
    return to_np(ops.lora_add(yd, xd, a, b, to_dev(ids), None if scales is None else to_dev(scales),
                              out=yd if out == "y0" else None, workspace=ws, err=err))


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("m,k,n,r,e", [(1, 32, 1, 1, 1), (1, 2560, 6144, 16, 8), (8, 2560, 6144, 16, 8), (3, 64, 17, 4, 2),
                                       (16, 1024, 100, 8, 16), (17, 96, 260, 12, 5), (48, 4096, 2560, 64, 24),
                                       (64, 320, 515, 20, 64), (33, 2048, 1023, 33, 3), (5, 9728, 300, 128, 4),
                                       (20, 256, 64, 250, 3), (130, 1024, 777, 48, 2), (257, 2048, 1024, 64, 7)])
def test_shapes(dev, m, k, n, r, e, dt):
    print(f"lora m={m} k={k} n={n} r={r} e={e} {dt}", flush=True)
    x, y0, a, ah, b, bh, ids, scales = _case(m, k, n, r, e, dt, seed=m + r)
    _check(_run(x, y0, a, b, ids, scales), y0, x, ah, bh, ids, scales)


@pytest.mark.parametrize("m,run", [(1, 1), (40, 40), (200, 67), (1000, 250), (515, 1)])
@pytest.mark.parametrize("out", [None, "y0"])
def test_runs_of_one_adapter_and_in_place(dev, m, run, out):
    ids = np.repeat(rng(m).integers(-1, 5, (m + run - 1) // run), run)[:m]
    x, y0, a, ah, b, bh, ids, scales = _case(m, 256, 384, 16, 5, "bf16", seed=m, ids=ids)
    _check(_run(x, y0, a, b, ids, None, out=out), y0, x, ah, bh, ids, None)


def test_ids_that_name_nothing(dev):
    ids = [0, -1, 3, 2, -7, 1 << 30, 1, 4]
    x, y0, a, ah, b, bh, ids, scales = _case(8, 64, 40, 8, 3, "bf16", seed=2, ids=ids)
    err = DTensor.zeros((1,), "i32")
    _check(_run(x, y0, a, b, ids, scales, err=err), y0, x, ah, bh, ids, scales)
    assert int(err.item()) == 3
    none = np.full(8, -1, np.int32)
    assert np.array_equal(_run(x, y0, a, b, none, scales), y0)


def test_weights_and_rows_that_are_not_finite_stay_apart(dev):
    """An adapter with NaN and infinite weights, and a row of x with a NaN: every other row is as without them."""
    m, ids = 24, np.arange(24) % 4
    x, y0, a, ah, b, bh, ids, scales = _case(m, 128, 96, 16, 4, "bf16", seed=3, ids=ids)
    clean = _run(x, y0, a, b, ids, scales)
    bits = to_np(a).copy()
    bits[2, 5, 7], bits[2, 0, 0] = 0x7FC0, 0x7F80
    bb = to_np(b).copy()
    bb[2, 50, 3] = 0x7F80
    x2 = x.copy()
    x2[5, 9] = np.nan
    got = _run(x2, y0, to_dev(bits, bf16=True), to_dev(bb, bf16=True), ids, scales)
    bad = (ids == 2) | (np.arange(m) == 5)
    assert np.array_equal(got[~bad], clean[~bad])
    assert not np.isfinite(got[ids == 2]).any() and np.isnan(got[5]).all()


def test_strided_rows_and_views_of_larger_stacks(dev):
    """x, y0 and y rows inside wider buffers at odd offsets, adapters inside larger ones, strided ids."""
    m, k, n, r, e = 21, 96, 50, 12, 3
    xw, y0w = randn((m, k + 3), seed=1), randn((m, n + 5), seed=2)
    aw, awh = _w(randn((e, r + 2, k + 7), seed=3, scale=0.1), "f16")
    bw, bwh = _w(randn((e, n + 1, r + 3), seed=4), "f16")
    idw = rng(5).integers(-1, e, (m, 2)).astype(np.int32)
    yw = DTensor.full_byte((m, n + 9), 0x7F, "f32")
    ops.lora_add(to_dev(y0w)[:, 5:], to_dev(xw)[:, 3:], aw[:, :r, 7:], bw[:, 1:, 3:], to_dev(idw)[:, 1], out=yw[:, 4:4 + n])
    full = to_np(yw)
    _check(np.ascontiguousarray(full[:, 4:4 + n]), y0w[:, 5:], xw[:, 3:], awh[:, :r, 7:], bwh[:, 1:, 3:], idw[:, 1], None)
    rest = np.concatenate([full[:, :4], full[:, 4 + n:]], 1)
    assert (np.ascontiguousarray(rest).view(np.uint8) == 0x7F).all()


def test_same_bits_twice_and_whatever_the_workspace_held(dev):
    x, y0, a, ah, b, bh, ids, scales = _case(40, 2560, 1000, 32, 9, "bf16", seed=6)
    xd, yd, idd, sd = to_dev(x), to_dev(y0), to_dev(ids), to_dev(scales)
    need = ops.lora_add_workspace(xd, a, b)
    got = [to_np(ops.lora_add(yd, xd, a, b, idd, sd, workspace=DTensor.full_byte((need,), f))) for f in (0, 0xFF, 0x3C)]
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])


def test_beside_the_projection_in_a_graph(dev):
    """The Q8_0 product and the adapters after it, captured once, replayed for new x and ids with eager work between."""
    m, k, n, r, e = 8, 256, 192, 16, 4
    wq = orc.quantize_q8_0(randn((n, k), seed=1, scale=0.1), "ref")
    w = ops.q8_0_repack(ops.Q8(to_dev(wq)))
    x, y0, a, ah, b, bh, ids, scales = _case(m, k, n, r, e, "bf16", seed=7)
    xd, yd, idd, sd = DTensor.zeros((m, k)), DTensor.zeros((m, n)), DTensor.zeros((m,), "i32"), to_dev(scales)
    ws1 = DTensor.empty((ops.mul_mat_q8_0_workspace(w, xd),), "u8")
    ws2 = DTensor.empty((ops.lora_add_workspace(xd, a, b),), "u8")
    st, g = Stream(), Graph()
    with g.capture(st):
        ops.mul_mat_q8_0(w, xd, out=yd, workspace=ws1, stream=st.handle)
        ops.lora_add(yd, xd, a, b, idd, sd, out=yd, workspace=ws2, stream=st.handle)
    from acestep_ops.device import D2D, check, hip

    for i in range(3):
        x = randn((m, k), seed=20 + i)
        ids = rng(30 + i).integers(-1, e, m).astype(np.int32)
        for dst, src in ((xd, to_dev(x)), (idd, to_dev(ids))):
            check(hip().hipMemcpy(dst.ptr, src.ptr, src.numel() * src.es, D2D), "hipMemcpy")
        synchronize()
        g.launch()
        st.synchronize()
        eager = to_np(ops.mul_mat_q8_0(w, to_dev(x)))
        _check(to_np(yd), eager, x, ah, bh, ids, scales)
