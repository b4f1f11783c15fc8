"""GPU: a NaN that one key brings into attention over Q4_0 K and V shows in y however many workgroups the keys
are split over: also where that key is the only one its split attends to, or its weight underflows to zero."""
import numpy as np
import pytest
import q4
from helpers import randn, to_dev, to_np
from oracle import oracle as orc
from test_gpu_fattn_q4 import _cache, _mask_dev, _q

from acestep_ops import ops
from acestep_ops.device import DTensor

pytestmark = pytest.mark.gpu


def _splits(qv, kd, vd, mask_bytes=0):
    """How many parts the workspace has room for: (D + 4) floats a row and part."""
    N, nh, n_q, D = qv.shape
    return (ops.flash_attn_workspace(qv, kd, vd) - mask_bytes) // (N * nh * n_q * (D + 4) * 4)


def _nan_block(c, key, blk):
    c[:, :, key, blk * 18:blk * 18 + 2] = np.array([0x7E00], np.uint16).view(np.uint8)


def _run(D, N, nh, nkv, n_q, dt, out, k, v, mask):
    qd, _ = _q(randn((N, n_q, nh, D), seed=1), dt)
    qv, kd, vd = qd.permute(0, 2, 1, 3), ops.Q4(to_dev(k)), ops.Q4(to_dev(v))
    need = ops.flash_attn_workspace(qv, kd, vd)
    ws = DTensor.full_byte((max(need, 16),), 0x55)
    y = DTensor.zeros((N, n_q, nh, D), out)
    ops.flash_attn_ext(qv, kd, vd, _mask_dev(mask), 0.1, out=y, workspace=ws)
    return qv, kd, vd, to_np(y) if out == "f32" else orc.bf16_to_f32(to_np(y))


@pytest.mark.parametrize("dt,out", [("f32", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("D,n,least", [(64, 2100, 2), (64, 8001, 9), (64, 70001, 33), (128, 700, 2), (128, 3301, 9), (128, 60013, 17),
                                       (256, 1000, 2), (256, 30011, 9)])
@pytest.mark.parametrize("n_q", [1, 2])
def test_the_only_live_key_of_a_split(dev, D, n, least, n_q, dt, out):
    print(f"q4 attention, a NaN alone in its split, D={D} n={n} n_q={n_q} {dt}->{out}", flush=True)
    N, nh, nkv = 2, 4, 2
    k0, v0 = _cache(N, nkv, n, D, 2), _cache(N, nkv, n, D, 3)
    for at in (n - 1, n // 2, 321):
        mask = np.full((1, 1, n_q, n), -np.inf)
        mask[..., :32] = 0.0
        mask[..., at] = 0.0
        k, v = k0.copy(), v0.copy()
        _nan_block(k, at, 1)
        qv, kd, vd, y = _run(D, N, nh, nkv, n_q, dt, out, k, v0, mask)
        assert _splits(qv, kd, vd) >= least, "the keys are split"
        assert np.isnan(y).all(), f"K of key {at}"
        mask[..., at] = -60000.0  # weight zero: 0 * NaN
        _nan_block(v, at, 1)
        _, _, _, y = _run(D, N, nh, nkv, n_q, dt, out, k0, v, mask)
        assert np.isnan(y[..., 32:64]).all(), f"V of key {at}"
        assert np.isfinite(y[..., :32]).all() and np.isfinite(y[..., 64:]).all()


@pytest.mark.parametrize("dt,out", [("f32", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("D,nh,n_q", [(64, 16, 512), (128, 16, 512), (256, 16, 512)])
def test_the_only_live_key_of_a_split_many_rows(dev, D, nh, n_q, dt, out):
    """Positions from 256 on attend to the key with a NaN, the others (of other workgroups) do not."""
    print(f"q4 attention, a NaN alone in its split, many rows D={D} {dt}->{out}", flush=True)
    n, nkv = 5120, 8
    k, v = _cache(1, nkv, n, D, 2), _cache(1, nkv, n, D, 3)
    mask = np.full((1, 1, n_q, n), -np.inf)
    mask[..., :64] = 0.0
    mask[..., 256:, n - 1] = 0.0
    _nan_block(k, n - 1, 1)
    qv, kd, vd, y = _run(D, 1, nh, nkv, n_q, dt, out, k, v, mask)
    summary = nh * ((n_q + 15) // 16) * (n // 64)
    assert _splits(qv, kd, vd, summary) >= 2, "the keys are split"
    assert np.isnan(y[:, 256:]).all()
    assert np.isfinite(y[:, :256]).all()


@pytest.mark.parametrize("dt,out", [("f32", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("D,N,nh,nkv,n_q,n", [(64, 1, 4, 2, 1, 100), (128, 2, 8, 2, 1, 700), (256, 1, 2, 1, 5, 90), (64, 8, 32, 8, 130, 200),
                                              (128, 8, 32, 8, 130, 200), (256, 8, 16, 4, 130, 100)])
def test_an_infinity_in_a_live_key(dev, D, N, nh, nkv, n_q, n, dt, out):
    """Its block reads back as no finite value, so every row that attends to it is NaN, whatever its sign and q's."""
    print(f"q4 attention, an infinite K element D={D} n_q={n_q} {dt}->{out}", flush=True)
    x = randn((N, nkv, n, D), seed=2)
    x[:, :, 17, 5], x[:, ::2, n - 3, D - 1] = np.inf, -np.inf
    k, v = q4.quantize(x), _cache(N, nkv, n, D, 3)
    mask = np.zeros((1, 1, n_q, n))
    _, _, _, y = _run(D, N, nh, nkv, n_q, dt, out, k, v, mask)
    assert np.isnan(y).all()
    mask[..., 17] = mask[..., n - 3] = -np.inf
    _, _, _, y = _run(D, N, nh, nkv, n_q, dt, out, k, v, mask)
    assert np.isfinite(y).all()
