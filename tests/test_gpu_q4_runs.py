"""GPU parity, bit-exact: the Q4_0 append where a sequence's tokens fill whole waves of rows (a multiple of 32 rows of
32 values, 16 of 64, 8 of 128, 4 of 256): every byte of both caches, and the count of rows that have no slot or set."""
import numpy as np
import pytest
import q4
from helpers import rng, to_dev, to_np
from test_gpu_q4 import _kv_case, _same_blocks, _up

from acestep_ops import ops
from acestep_ops.device import DTensor

pytestmark = pytest.mark.gpu
RUNS = [(32, 2, 32, 3), (64, 3, 16, 2), (64, 2, 48, 5), (128, 2, 8, 8), (128, 3, 40, 2), (128, 1, 2048, 2), (256, 2, 4, 3), (256, 3, 36, 1)]


@pytest.mark.parametrize("D,B,T,Nkv", RUNS)
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_kv_store(dev, D, B, T, Nkv, dt):
    print(f"kv_store q4_0, whole waves, D={D} B={B} T={T} Nkv={Nkv} {dt}", flush=True)
    k, v, pos0, sets, kc, vc, want, _ = _kv_case(dt, D, B, T, Nkv, seed=D + T)
    err = DTensor.zeros((1,), "i32")
    ops.kv_store(k, kc, to_dev(pos0), v, vc, to_dev(sets), err=err)
    for c, w in zip((kc, vc), want):
        _same_blocks(to_np(c.data), w)
    assert err.item() == 0
    only = ops.Q4(DTensor.full_byte(kc.data.shape, 0xA5))  # K alone
    ops.kv_store(k, only, to_dev(pos0), sets=to_dev(sets))
    _same_blocks(to_np(only.data), want[0])


@pytest.mark.parametrize("D,B,T,Nkv", [(32, 4, 32, 2), (64, 4, 32, 2), (128, 4, 24, 2), (256, 4, 12, 1)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_bad_slots_and_sets(dev, D, B, T, Nkv, dt):
    """A wave's rows that straddle the last slot, or slot 0 from below; a set that is not there, one past the last."""
    print(f"kv_store q4_0, whole waves, bad slots D={D} T={T} {dt}", flush=True)
    max_seq, n_sets = T + 20, B + 1
    x = rng(D + T).standard_normal((2, B, T, Nkv, D)).astype(np.float32)
    (k, kx), (v, vx) = (_up(t, dt) for t in x)
    pos0 = np.array([max_seq - T + 3, -5, 7, 1], np.int32)
    sets = np.array([2, 0, -1, n_sets], np.int32)
    want = [np.full((n_sets, Nkv, max_seq, D // 32 * 18), f, np.uint8) for f in (0xA5, 0x5A)]
    errs = 0
    for b in range(B):
        for t in range(T):
            if 0 <= pos0[b] + t < max_seq and 0 <= sets[b] < n_sets:
                for w, s in zip(want, (kx, vx)):
                    w[sets[b], :, pos0[b] + t] = q4.quantize(s[b, t])
            else:
                errs += 2 * Nkv
    kc, vc = (ops.Q4(DTensor.full_byte(w.shape, f)) for w, f in zip(want, (0xA5, 0x5A)))
    err = DTensor.zeros((1,), "i32")
    ops.kv_store(k, kc, to_dev(pos0), v, vc, to_dev(sets), err=err)
    assert err.item() == errs == 2 * Nkv * (3 + 5 + 2 * T)
    for c, w in zip((kc, vc), want):
        _same_blocks(to_np(c.data), w)
    _, _, p0, st, c0, c1, w0, _ = _kv_case(dt, D, 2, T, Nkv, seed=1)  # strided source rows and heads
    src = np.zeros((2, T, Nkv + 1, D + 16), np.float32)
    src[:, :, 1:, 16:] = x[0, :2]
    sd, sx = _up(src, dt)
    ops.kv_store(sd[:, :, 1:, 16:], c0, to_dev(p0), sets=to_dev(st))
    ref = np.full(w0[0].shape, 0xA5, np.uint8)
    for b in range(2):
        ref[st[b], :, p0[b]:p0[b] + T] = q4.quantize(np.ascontiguousarray(sx[b, :, 1:, 16:])).transpose(1, 0, 2)
    _same_blocks(to_np(c0.data), ref)
