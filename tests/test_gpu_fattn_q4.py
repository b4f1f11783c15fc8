"""GPU: flash attention over Q4_0 K and V against 64 bits, within the error bound of
the kernels' arithmetic (fa4_bound.py), at head sizes 64, 128 and 256, one to many
query positions, every kind of mask, views, and caches with bytes that are no numbers
behind the last key."""
import numpy as np
import pytest
import q4
from fa4_bound import row
from helpers import randn, rng, to_dev, to_np
from oracle import oracle as orc

from acestep_ops import ops
from acestep_ops.device import DTensor, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu


def _q(x, dt):
    if dt == "bf16":
        h = orc.f32_to_bf16(x)
        return to_dev(h, bf16=True), orc.bf16_to_f32(h)
    if dt == "f16":
        h = x.astype(np.float16)
        return to_dev(h.view(np.uint16), f16=True), h.astype(np.float32)
    return to_dev(x), x


def _cache(n_sets, nkv, n, D, seed, scale=1.0):
    return q4.quantize(randn((n_sets, nkv, n, D), seed=seed, scale=scale))


def _mask_dev(m):
    return to_dev(np.ascontiguousarray(m).astype(np.float16).view(np.uint16), f16=True)


def _values(y):
    return to_np(y).astype(np.float64) if y.dtype == "f32" else orc.bf16_to_f32(to_np(y)).astype(np.float64)


def _check(y, qx, k, v, mask, scale, rows=None):
    """y (N, n_q, Nh, D); qx (N, Nh, n_q, D); k, v (Nk3, Nkv, n, bytes); mask (m3, m2, >= n_q, n) float64 or None."""
    N, Nh, n_q, D = qx.shape
    got = _values(y)
    pick = rows if rows is not None else [(b, h, i) for b in range(N) for h in range(Nh) for i in range(n_q)]
    worst = 0.0
    for b, h, i in pick:
        kb, g = b // (N // k.shape[0]), h // (Nh // k.shape[1])
        m = None if mask is None else mask[b % mask.shape[0], h % mask.shape[1], i]
        ref, bound = row(qx[b, h, i].astype(np.float64), k[kb, g], v[kb, g], m, scale, y.dtype == "f32")
        out = got[b, i, h]
        if np.isnan(ref).all():
            assert np.isnan(out).all(), f"({b}, {h}, {i}): no live key"
            continue
        err = np.abs(out - ref)
        assert np.isfinite(out).all() and (err <= bound).all(), \
            f"({b}, {h}, {i}): off by {err.max():.3g}, {np.nanmax(err / bound):.3g} of the bound"
        worst = max(worst, float((err / bound).max()))
    print(f"  worst {worst:.3g} of the bound", flush=True)


def _lengths_mask(N, n_q, n, past):
    """(N, 1, n_q, n): position i of sequence b sees slots <= past[b] + i."""
    last = np.asarray(past)[:, None] + np.arange(n_q)
    return np.where(np.arange(n)[None, None] <= last[:, :, None], 0.0, -np.inf)[:, None]


def _run(D, N, nh, nkv, n_q, n, dt, out, mask, seed, nk3=None, q_scale=1.0):
    qd, qx = _q(randn((N, n_q, nh, D), seed=seed, scale=q_scale), dt)
    k, v = _cache(nk3 or N, nkv, n, D, seed + 1), _cache(nk3 or N, nkv, n, D, seed + 2)
    scale = float(np.float32(D ** -0.5))
    y = DTensor.full_byte((N, n_q, nh, D), 0xFF, out)
    qv = qd.permute(0, 2, 1, 3)
    kd, vd = ops.Q4(to_dev(k)), ops.Q4(to_dev(v))
    need = ops.flash_attn_workspace(qv, kd, vd)
    ws = DTensor.full_byte((max(need, 16),), 0xFF)
    ops.flash_attn_ext(qv, kd, vd, None if mask is None else _mask_dev(mask), scale, out=y, workspace=ws)
    _check(y, qx.transpose(0, 2, 1, 3), k, v, mask, scale)


TYPES = [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f32")]


@pytest.mark.parametrize("dt,out", TYPES)
@pytest.mark.parametrize("D,nh,nkv", [(128, 4, 1), (128, 2, 2), (64, 6, 2), (256, 3, 1), (64, 16, 1), (128, 20, 1)])
@pytest.mark.parametrize("n", [1, 31, 64, 65, 700])
def test_single_token(dev, dt, out, D, nh, nkv, n):
    print(f"q4 attention one token D={D} {nh}/{nkv} n={n} {dt}->{out}", flush=True)
    N = 2
    mask = _lengths_mask(N, 1, n, [n - 1, n // 3])
    _run(D, N, nh, nkv, 1, n, dt, out, mask, seed=D + n)


@pytest.mark.parametrize("dt,out", TYPES)
@pytest.mark.parametrize("D,nh,nkv,n_q,n", [(128, 4, 2, 3, 200), (64, 2, 1, 17, 130), (256, 4, 1, 5, 97), (128, 8, 2, 40, 333),
                                            (128, 1, 1, 129, 129), (64, 4, 4, 70, 300), (256, 2, 1, 80, 100),
                                            (128, 6, 2, 33, 64), (128, 16, 1, 200, 517), (64, 8, 2, 260, 260),
                                            (256, 4, 2, 130, 190)])
def test_many_positions_causal(dev, dt, out, D, nh, nkv, n_q, n):
    print(f"q4 attention D={D} {nh}/{nkv} n_q={n_q} n={n} {dt}->{out}", flush=True)
    _run(D, 2, nh, nkv, n_q, n, dt, out, _lengths_mask(2, n_q, n, [n - n_q, (n - n_q) // 2]), seed=n_q + n)


@pytest.mark.parametrize("dt,out", TYPES[:2])
@pytest.mark.parametrize("D,n_q,n", [(128, 1, 300), (128, 90, 300), (64, 1, 77), (256, 70, 65)])
def test_no_mask(dev, dt, out, D, n_q, n):
    print(f"q4 attention without a mask D={D} n_q={n_q} n={n} {dt}", flush=True)
    _run(D, 2, 4, 2, n_q, n, dt, out, None, seed=n)


@pytest.mark.parametrize("dt,out", TYPES[:2])
@pytest.mark.parametrize("D,n_q,n", [(128, 1, 200), (128, 2, 200), (128, 100, 200), (64, 33, 90), (256, 65, 130)])
def test_masks_with_values_holes_and_empty_rows(dev, dt, out, D, n_q, n):
    """A mask row per head: finite values, the type's lowest, holes, rows with no key and rows with one."""
    print(f"q4 attention odd masks D={D} n_q={n_q} n={n} {dt}", flush=True)
    N, nh, nkv = 2, 4, 2
    r = rng(n + n_q)
    mask = r.choice([0.0, 0.0, 0.5, -2.0, -65504.0, -np.inf, -np.inf], (N, nh, n_q, n))
    mask[0, 1, n_q // 2] = -np.inf
    mask[1, 2, 0] = -np.inf
    mask[1, 2, 0, n - 1] = 0.25
    mask[0, 3, n_q - 1] = -65504.0
    mask[1, 0, :, 64:128] = -np.inf
    _run(D, N, nh, nkv, n_q, n, dt, out, mask, seed=n)


@pytest.mark.parametrize("n_q", [1, 70])
@pytest.mark.parametrize("dt,out", TYPES[:2])
def test_sequence_with_nothing_to_attend_to(dev, dt, out, n_q):
    mask = _lengths_mask(3, n_q, 256, [256 - n_q, -n_q, 10])
    _run(128, 3, 4, 2, n_q, 256, dt, out, mask, seed=3)


@pytest.mark.parametrize("n_q", [1, 4, 66])
def test_views_broadcast_caches_and_a_longer_mask(dev, n_q):
    """K and V views into larger caches at an offset, one cache for two sequences, a mask with more rows than
    queries, a strided y."""
    D, N, nh, nkv, n = 128, 4, 4, 2, 150
    qd, qx = _q(randn((N, n_q, nh, D), seed=1), "f32")
    k, v = _cache(2, nkv, 400, D, 2), _cache(2, nkv, 400, D, 3)
    kd, vd = ops.Q4(to_dev(k)[:, :, 7:7 + n]), ops.Q4(to_dev(v)[:, :, 7:7 + n])
    mask = rng(4).choice([0.0, -1.0, -np.inf], (2, 2, n_q + 3, n))
    yw = DTensor.full_byte((N, n_q, nh + 1, D + 4), 0x7F, "f32")
    y = yw[:, :, :nh, :D]
    ops.flash_attn_ext(qd.permute(0, 2, 1, 3), kd, vd, _mask_dev(mask), 0.1, out=y)
    _check(y, qx.transpose(0, 2, 1, 3), k[:, :, 7:7 + n], v[:, :, 7:7 + n], mask, 0.1)
    rest = to_np(yw)
    assert (np.ascontiguousarray(rest[:, :, nh:]).view(np.uint8) == 0x7F).all()
    assert (np.ascontiguousarray(rest[..., D:]).view(np.uint8) == 0x7F).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n_q", [1, 5, 80])
def test_bytes_that_are_no_numbers_in_masked_slots(dev, n_q, D):
    """Slots that no query attends to hold NaN and infinite scales: the output is that of clean slots."""
    n, N = 200, 2
    k, v = _cache(N, 2, n, D, 5), _cache(N, 2, n, D, 6)
    past = [130, 70]
    for b in range(N):
        for c, bits in ((k, 0x7E00), (v, 0x7C00), (v, 0xFE00)):
            at = slice(past[b] + n_q + (bits == 0xFE00), None, 2)
            blocks = c[b, :, at].reshape(2, -1, D // 32, 18).copy()
            blocks[..., 0], blocks[..., 1] = bits & 255, bits >> 8
            c[b, :, at] = blocks.reshape(2, -1, D // 32 * 18)
    for dt, out in TYPES[:2]:
        qd, qx = _q(randn((N, n_q, 4, D), seed=7), dt)
        mask = _lengths_mask(N, n_q, n, past)
        y = DTensor.zeros((N, n_q, 4, D), out)
        ops.flash_attn_ext(qd.permute(0, 2, 1, 3), ops.Q4(to_dev(k)), ops.Q4(to_dev(v)), _mask_dev(mask), 0.1, out=y)
        _check(y, qx.transpose(0, 2, 1, 3), k, v, mask, 0.1)


@pytest.mark.parametrize("n_q", [1, 65])
def test_a_live_block_that_is_not_finite_shows(dev, n_q):
    D, n = 128, 100
    k, v = _cache(1, 1, n, D, 5), _cache(1, 1, n, D, 6)
    v[0, 0, 17, 18:20] = np.array([0x7E00], np.uint16).view(np.uint8)
    y = to_np(ops.flash_attn_ext(to_dev(randn((1, 2, n_q, D), seed=1)), ops.Q4(to_dev(k)), ops.Q4(to_dev(v)), None, 0.1))
    assert np.isnan(y[..., 32:64]).all() and np.isfinite(y[..., :32]).all() and np.isfinite(y[..., 64:]).all()


@pytest.mark.parametrize("n_q", [1, 70])
@pytest.mark.parametrize("dt,out", TYPES[:2])
def test_large_and_small_values(dev, dt, out, n_q):
    """V past fp16 (d above 8188), tiny V, queries of 1e5 and 1e-30, and scores of some hundreds."""
    D, n = 128, 140
    mask = _lengths_mask(1, n_q, n, [n - n_q])
    for vs, ks, qs in ((1e5, 1.0, 1.0), (1e-6, 1.0, 1.0), (1.0, 1e-4, 1e5), (1.0, 1e3, 1e-3), (1.0, 1.0, 1e-30), (1.0, 30.0, 3.0)):
        qd, qx = _q(randn((1, n_q, 2, D), seed=8, scale=qs), dt)
        k, v = _cache(1, 1, n, D, 9, ks), _cache(1, 1, n, D, 10, vs)
        y = DTensor.zeros((1, n_q, 2, D), out)
        ops.flash_attn_ext(qd.permute(0, 2, 1, 3), ops.Q4(to_dev(k)), ops.Q4(to_dev(v)), _mask_dev(mask), 0.1, out=y)
        _check(y, qx.transpose(0, 2, 1, 3), k, v, mask, 0.1)


@pytest.mark.parametrize("n_q", [1, 3, 64])
def test_no_keys_and_no_queries(dev, n_q):
    D = 128
    k = ops.Q4(DTensor.zeros((1, 1, 4, 72), "u8")[:, :, :0])
    y = ops.flash_attn_ext(to_dev(randn((1, 2, n_q, D), seed=1)), k, k, None, 0.1)
    assert np.isnan(to_np(y)).all()
    full = ops.Q4(DTensor.zeros((1, 1, 4, 72), "u8"))
    y = ops.flash_attn_ext(DTensor.zeros((1, 2, n_q, D))[:, :, :0], full, full, None, 0.1,
                           out=DTensor.full_byte((1, n_q, 2, D), 0x11, "f32")[:, :0])
    assert y.numel() == 0


def test_a_cache_past_four_gigabytes(dev):
    """One sequence of 60 million slots (K and V 4.3 GB each): a few live keys on both sides of 2^31 and 2^32 bytes."""
    D, n = 128, 60_000_000
    kd, vd = DTensor.zeros((1, 1, n, 72), "u8"), DTensor.zeros((1, 1, n, 72), "u8")
    at = np.array([0, 5, 29826161, 29826162, 59652322, 59652323, 59652324, n - 2, n - 1])
    mask = np.full(n, 0xFC00, np.uint16)
    mask[at] = 0
    k, v = _cache(1, 1, len(at), D, 1), _cache(1, 1, len(at), D, 2)
    from acestep_ops.device import H2D, PinnedBuffer, check, hip
    import ctypes

    stage = PinnedBuffer(72)
    for i, slot in enumerate(at):
        for c, h in ((kd, k), (vd, v)):
            src = np.ascontiguousarray(h[0, 0, i])
            ctypes.memmove(stage.ptr, src.ctypes.data, 72)
            check(hip().hipMemcpy(c.ptr + int(slot) * 72, stage.ptr, 72, H2D), "hipMemcpy")
    for n_q in (1, 2):
        qd, qx = _q(randn((1, n_q, 2, D), seed=3), "f32")
        m = to_dev(np.repeat(mask[None, None, None], n_q, 2), f16=True)
        y = ops.flash_attn_ext(qd.permute(0, 2, 1, 3), ops.Q4(kd), ops.Q4(vd), m, 0.1)
        _check(y, qx.transpose(0, 2, 1, 3), k, v, None, 0.1)


@pytest.mark.parametrize("N,nh,nkv,n,past", [(8, 32, 8, 6656, 6599), (1, 16, 8, 40960, 40959), (64, 8, 4, 512, 500)])
@pytest.mark.parametrize("dt,out", TYPES[:2])
def test_decode_sizes(dev, N, nh, nkv, n, past, dt, out):
    """The serving sizes, on sampled rows; two calls give the same bits."""
    print(f"q4 attention decode {N} x {nh}/{nkv} n={n} {dt}", flush=True)
    D = 128
    qd, qx = _q(randn((N, 1, nh, D), seed=1), dt)
    base = _cache(1, nkv, n, D, 2)
    k = np.concatenate([np.roll(base, 37 * i, axis=2) for i in range(N)])
    v = np.concatenate([np.roll(base, 11 * i + 5, axis=2) for i in range(N)])
    lens = rng(3).integers(past // 9, past + 1, N)
    lens[0] = past
    mask = _lengths_mask(N, 1, n, lens)
    kd, vd, md = ops.Q4(to_dev(k)), ops.Q4(to_dev(v)), _mask_dev(mask)
    got = []
    for _ in range(2):
        y = DTensor.zeros((N, 1, nh, D), out)
        ops.flash_attn_ext(qd.permute(0, 2, 1, 3), kd, vd, md, 0.088, out=y)
        got.append(to_np(y))
    assert np.array_equal(got[0], got[1])
    pick = [(b, h, 0) for b in {0, N // 2, N - 1} for h in range(0, nh, 5)]
    _check(y, qx.transpose(0, 2, 1, 3), k, v, mask, float(np.float32(0.088)), pick)


@pytest.mark.parametrize("N,nh,nkv,S,past", [(2, 32, 8, 512, 0), (1, 16, 8, 257, 130), (1, 4, 1, 1500, 300)])
@pytest.mark.parametrize("dt,out", TYPES[:2])
def test_prompt_sizes(dev, N, nh, nkv, S, past, dt, out):
    print(f"q4 attention prompt {N} x {S} past {past} {nh}/{nkv} {dt}", flush=True)
    D, n = 128, S + past
    qd, qx = _q(randn((N, S, nh, D), seed=1), dt)
    k, v = _cache(N, nkv, n, D, 2), _cache(N, nkv, n, D, 3)
    mask = _lengths_mask(N, S, n, [past] + [past // 2] * (N - 1))
    y = DTensor.zeros((N, S, nh, D), out)
    ops.flash_attn_ext(qd.permute(0, 2, 1, 3), ops.Q4(to_dev(k)), ops.Q4(to_dev(v)), _mask_dev(mask), 0.088, out=y)
    r = rng(5)
    pick = [(int(r.integers(N)), int(r.integers(nh)), int(i)) for i in [0, 1, 63, 64, S - 1, S - 2] + list(r.integers(0, S, 40))]
    _check(y, qx.transpose(0, 2, 1, 3), k, v, mask, float(np.float32(0.088)), pick)


def test_store_then_attend_in_a_graph(dev):
    """The cache's append and the attention that reads it, captured once and replayed for three tokens with eager
    work between."""
    D, N, nh, nkv, slots = 128, 2, 8, 2, 96
    st = Stream()
    k, v = _cache(N, nkv, slots, D, 1), _cache(N, nkv, slots, D, 2)
    kc, vc = ops.Q4(to_dev(k)), ops.Q4(to_dev(v))
    q, kn, vn = DTensor.zeros((N, 1, nh, D)), DTensor.zeros((N, 1, nkv, D)), DTensor.zeros((N, 1, nkv, D))
    pos0, mask = DTensor.zeros((N,), "i32"), DTensor.zeros((N, 1, 1, slots), "f16")
    y = DTensor.zeros((N, 1, nh, D))
    qv = q.permute(0, 2, 1, 3)
    ws = DTensor.empty((max(ops.flash_attn_workspace(qv, kc, vc), 16),), "u8")
    g = Graph()
    with g.capture(st):
        ops.kv_store(kn, kc, pos0, vn, vc, stream=st.handle)
        ops.flash_attn_ext(qv, kc, vc, mask, 0.1, out=y, workspace=ws, stream=st.handle)
    from acestep_ops.device import D2D, check, hip

    def put(dst, a):
        check(hip().hipMemcpy(dst.ptr, a.ptr, a.numel() * a.es, D2D), "hipMemcpy")

    for i in range(3):
        qx, kx, vx = (randn((N, 1, w, D), seed=10 * i + j) for j, w in enumerate((nh, nkv, nkv)))
        past = np.array([60 + i, 20 + i], np.int32)
        m = _lengths_mask(N, 1, slots, past)
        for dst, a in ((q, to_dev(qx)), (kn, to_dev(kx)), (vn, to_dev(vx)), (pos0, to_dev(past)), (mask, _mask_dev(m))):
            put(dst, a)
        synchronize()
        g.launch()
        st.synchronize()
        for b in range(N):
            k[b, :, past[b]], v[b, :, past[b]] = q4.quantize(kx[b, 0]), q4.quantize(vx[b, 0])
        _check(y, qx.transpose(0, 2, 1, 3), k, v, m, float(np.float32(0.1)))
