"""GPU parity, bit-exact: mi_logits_adjust against its fp32 operations one by one in numpy."""
import numpy as np
import pytest
from helpers import randn, rng, to_dev, to_np
from oracle import oracle as orc

from acestep_ops import ops
from acestep_ops.device import DTensor, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu


def _ref(l, hist, lens, pen, bias, allowed, state):
    """fp32, one rounding per operation."""
    m, V = l.shape
    y = l.astype(np.float32).copy()
    with np.errstate(all="ignore"):
        for r in range(m):
            if hist is not None:
                n = hist.shape[1] if lens is None else min(max(int(lens[r]), 0), hist.shape[1])
                t = hist[r, :n]
                c = np.bincount(t[(t >= 0) & (t < V)], minlength=V).astype(np.float32)
                rep, freq, pres = pen[r]
                x = np.where(y[r] > 0, y[r] / rep, y[r] * rep).astype(np.float32)
                x = ((x - (c * freq).astype(np.float32)).astype(np.float32) - pres).astype(np.float32)
                y[r] = np.where(c > 0, x, y[r])
            if bias is not None:
                y[r] = y[r] + bias[r if len(bias) > 1 else 0]
            if allowed is not None:
                s = (0 if len(allowed) == 1 else r) if state is None else int(state[r])
                if 0 <= s < len(allowed):
                    v = np.arange(V)
                    y[r, allowed[s].view(np.uint32)[v >> 5] >> (v & 31).astype(np.uint32) & 1 == 0] = -np.inf
    return y


def _up(x, dt):
    if dt == "bf16":
        h = orc.f32_to_bf16(x)
        return to_dev(h, bf16=True), orc.bf16_to_f32(h)
    if dt == "f16":
        h = x.astype(np.float16)
        return to_dev(h.view(np.uint16), f16=True), h.astype(np.float32)
    return to_dev(x), x


def _same(y, ref, dt):
    got = to_np(y)
    with np.errstate(over="ignore"):
        want = ref if dt == "f32" else orc.f32_to_bf16(ref) if dt == "bf16" else ref.astype(np.float16).view(np.uint16)
    if dt == "f32":
        assert np.array_equal(got, want, equal_nan=True)
    else:
        assert np.array_equal(got, want)


def _case(m, V, L, S, seed):
    r = rng(seed)
    hist = (V * r.random((m, L)) ** 3).astype(np.int32).clip(0, V - 1)
    lens = r.integers(0, L + 1, m).astype(np.int32)
    lens[0] = L
    pen = np.stack([1 + r.random(m) * 0.5, r.random(m) * 0.3, r.random(m)], 1).astype(np.float32)
    bias = (r.standard_normal((m, V)) * (r.random((m, V)) < 0.05)).astype(np.float32)
    allowed = r.integers(-2 ** 31, 2 ** 31, (S, (V + 31) // 32)).astype(np.int32)
    state = r.integers(-1, S, m).astype(np.int32)
    return hist, lens, pen, bias, allowed, state


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,V,L,S", [(1, 1, 1, 1), (3, 31, 5, 2), (2, 33, 40, 3), (5, 8192, 700, 4), (4, 8193, 300, 9),
                                     (3, 16391, 4000, 2), (8, 151669, 1200, 5), (2, 217204, 9000, 3)])
def test_all_together(dev, m, V, L, S, dt):
    print(f"logits m={m} V={V} L={L} S={S} {dt}", flush=True)
    hist, lens, pen, bias, allowed, state = _case(m, V, L, S, seed=V + L)
    x, xh = _up(randn((m, V), seed=V, scale=3.0), dt)
    y = ops.logits_adjust(x, to_dev(hist), to_dev(lens), to_dev(pen), to_dev(bias), to_dev(allowed), to_dev(state))
    _same(y, _ref(xh, hist, lens, pen, bias, allowed, state), dt)


@pytest.mark.parametrize("use", ["history", "bias", "grammar", "nothing"])
def test_each_alone_and_in_place(dev, use):
    m, V = 6, 9001
    hist, lens, pen, bias, allowed, state = _case(m, V, 333, 4, seed=1)
    x = randn((m, V), seed=2, scale=3.0)
    kw, ref = {}, [None] * 6
    if use == "history":  # no lengths: all of it
        kw, ref = {"history": to_dev(hist), "penalties": to_dev(pen)}, [hist, None, pen, None, None, None]
    elif use == "bias":   # one row for all
        kw, ref = {"bias": to_dev(bias[0])}, [None, None, None, bias[:1], None, None]
    elif use == "grammar":
        kw, ref = {"allowed": to_dev(allowed[:1])}, [None, None, None, None, allowed[:1], None]
    d = to_dev(x)
    y = ops.logits_adjust(d, out=d, **kw)
    _same(y, _ref(x, *ref), "f32")


def test_a_state_per_row_without_state(dev):
    m, V = 3, 500
    allowed = _case(m, V, 1, m, seed=3)[4]
    x = randn((m, V), seed=4)
    _same(ops.logits_adjust(to_dev(x), allowed=to_dev(allowed)), _ref(x, None, None, None, None, allowed, None), "f32")


def test_values_that_are_not_finite_and_empty_masks(dev):
    """-inf, inf and NaN logits under penalties, a state that allows nothing, lengths of zero and past the end."""
    m, V = 5, 70
    hist, lens, pen, bias, allowed, state = _case(m, V, 50, 3, seed=5)
    x = randn((m, V), seed=6)
    x[0, ::3], x[1, ::4], x[2, ::5], x[3, 7] = -np.inf, np.inf, np.nan, 0.0
    hist[:, :20] = np.arange(20)
    lens[:] = [50, 20, 50, 0, 1 << 30]
    allowed[1] = 0
    state[:] = [0, 1, 2, -1, 2]
    y = ops.logits_adjust(to_dev(x), to_dev(hist), to_dev(lens), to_dev(pen), None, to_dev(allowed), to_dev(state))
    ref = _ref(x, hist, lens, pen, None, allowed, state)
    assert (ref[1] == -np.inf).all()
    _same(y, ref, "f32")
    lens[:] = -5
    y = ops.logits_adjust(to_dev(x), to_dev(hist), to_dev(lens), to_dev(pen))
    _same(y, x, "f32")


def test_a_long_history_of_one_token(dev):
    """Counts are whole numbers however often a token comes: 100000 times one, the rest once."""
    V, L = 20000, 100007
    hist = np.full((1, L), 12345, np.int32)
    hist[0, 100000:] = np.arange(7) * 2777
    pen = np.array([[1.25, 0.001, 0.5]], np.float32)
    x = randn((1, V), seed=7)
    _same(ops.logits_adjust(to_dev(x), to_dev(hist), penalties=to_dev(pen)), _ref(x, hist, None, pen, None, None, None), "f32")


def test_bad_tokens_and_states_are_counted(dev):
    m, V = 4, 20000
    hist, lens, pen, bias, allowed, state = _case(m, V, 60, 2, seed=8)
    hist[:, 5], hist[1, 9], hist[2, 11] = -1, V, 1 << 30
    lens[:] = 60
    state[:] = [0, 2, -9, 1 << 20]
    x = randn((m, V), seed=9)
    err = DTensor.zeros((1,), "i32")
    y = ops.logits_adjust(to_dev(x), to_dev(hist), to_dev(lens), to_dev(pen), None, to_dev(allowed), to_dev(state), err=err)
    assert int(err.item()) == m + 2 + 2
    _same(y, _ref(x, hist, lens, pen, None, allowed, state), "f32")


def test_views_inside_wider_buffers(dev):
    m, V, L = 5, 3001, 77
    hist, lens, pen, bias, allowed, state = _case(m, V, L, 3, seed=10)
    for dt in ("f32", "bf16"):
        xw, xh = _up(randn((m, V + 7), seed=11), dt)
        hw = np.full((m, L + 4), -1, np.int32)
        hw[:, 2:2 + L] = hist
        aw = np.zeros((3, allowed.shape[1] + 2), np.int32)
        aw[:, 1:-1] = allowed
        yw = DTensor.full_byte((m, V + 9), 0x7F, dt)
        ops.logits_adjust(xw[:, 3:3 + V], to_dev(hw)[:, 2:2 + L], to_dev(np.stack([lens, lens], 1))[:, 1],
                          to_dev(np.concatenate([pen, pen], 1))[:, 1:4], None, to_dev(aw)[:, 1:-1], to_dev(state),
                          out=yw[:, 5:5 + V])
        pen2 = np.concatenate([pen, pen], 1)[:, 1:4]
        full = to_np(yw)
        ref = _ref(xh[:, 3:3 + V], hist, lens, pen2, None, allowed, state)
        want = ref if dt == "f32" else orc.f32_to_bf16(ref)
        assert np.array_equal(full[:, 5:5 + V], want)
        rest = np.concatenate([full[:, :5], full[:, 5 + V:]], 1)
        assert (np.ascontiguousarray(rest).view(np.uint8) == 0x7F).all()


def test_captured_and_replayed(dev):
    m, V, L = 3, 12000, 64
    hist, lens, pen, bias, allowed, state = _case(m, V, L, 3, seed=12)
    x, y = DTensor.zeros((m, V)), DTensor.zeros((m, V))
    ld, hd, pd, ad, sd = DTensor.zeros((m,), "i32"), to_dev(hist), to_dev(pen), to_dev(allowed), to_dev(state)
    st, g = Stream(), Graph()
    with g.capture(st):
        ops.logits_adjust(x, hd, ld, pd, None, ad, sd, out=y, stream=st.handle)
    from acestep_ops.device import D2D, check, hip

    for i in range(3):
        xh, lh = randn((m, V), seed=20 + i), np.array([i, 10 * i, L], np.int32)
        for dst, src in ((x, to_dev(xh)), (ld, to_dev(lh))):
            check(hip().hipMemcpy(dst.ptr, src.ptr, src.numel() * src.es, D2D), "hipMemcpy")
        synchronize()
        g.launch()
        st.synchronize()
        _same(y, _ref(xh, hist, lh, pen, None, allowed, state), "f32")
