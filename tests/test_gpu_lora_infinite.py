"""GPU: adapters (mi_lora_add) with infinities and magnitudes next to fp32's largest in x, A x and the weights:
signed infinities and NaN where the formula has them, finite values within test_gpu_lora's bound, and every row
and column that meets none of them bit-identical to a call without them."""
import numpy as np
import pytest
from helpers import randn, rng, to_dev
from test_gpu_lora import _ref, _run, _w

pytestmark = pytest.mark.gpu
MAX = np.finfo(np.float32).max

# rows, keys, columns, rank, adapters: every kernel of the first product and both kinds of tiles of the second
SHAPES = [(5, 64, 40, 1, 5), (24, 128, 96, 16, 6), (20, 96, 50, 24, 7), (40, 256, 130, 64, 8), (9, 64, 70, 200, 9), (33, 320, 17, 100, 6),
          (1505, 64, 1002, 16, 7), (1505, 64, 1001, 64, 6), (1505, 32, 1003, 129, 6), (1505, 64, 1000, 1, 6)]


def _make(m, k, n, r, e, seed):
    x, y0 = randn((m, k), seed=seed), randn((m, n), seed=seed + 1)
    a, b = randn((e, r, k), seed=seed + 2, scale=0.25 / k), randn((e, n, r), seed=seed + 3, scale=0.5 / r)
    ids = (np.arange(m) % e).astype(np.int32)
    return x, y0, a, b, ids, (rng(seed + 4).random(e) + 0.5).astype(np.float32)


def _same(got, y0, x, ah, bh, ids, scales):
    with np.errstate(all="ignore"):
        ref, bound = _ref(y0, x, ah, bh, ids, scales)
    assert np.array_equal(np.isnan(got), np.isnan(ref)), "NaN"
    inf = np.isinf(ref)
    assert np.array_equal(got[inf], ref[inf].astype(np.float32)), "infinities"
    ok = np.isfinite(ref)
    err = np.abs(got[ok].astype(np.float64) - ref[ok])
    assert np.isfinite(got[ok]).all() and (err <= bound[ok]).all(), f"{np.max(err / bound[ok]):.3g} of the bound"


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("m,k,n,r,e", SHAPES)
def test_infinities(dev, m, k, n, r, e, dt):
    print(f"lora with infinities m={m} k={k} n={n} r={r} e={e} {dt}", flush=True)
    x, y0, a, b, ids, scales = _make(m, k, n, r, e, seed=m + r)
    ad, ah = _w(a, dt)
    bd, bh = _w(b, dt)
    clean = _run(x, y0, ad, bd, ids, scales)
    x[0, 3], x[m - 1, k - 1] = np.inf, -np.inf
    x[2 % m, 5], x[2 % m, k - 2] = MAX, np.float32(-3.3962e38)
    x[4 % m, 7], x[4 % m, 8] = np.inf, np.inf
    a[3, r - 1, 7], b[1, n - 1, 0], b[1, 3, r - 1] = np.inf, -np.inf, np.inf
    ad, ah = _w(a, dt)
    bd, bh = _w(b, dt)
    got = _run(x, y0, ad, bd, ids, scales)
    _same(got, y0, x, ah, bh, ids, scales)
    rows = ~np.isin(np.arange(m), [0, 2 % m, 4 % m, m - 1]) & (ids != 3)
    cols = ~np.isin(np.arange(n), [3, n - 1])
    assert np.array_equal(got[rows & (ids != 1)], clean[rows & (ids != 1)]), "rows that meet none"
    assert np.array_equal(got[rows][:, cols], clean[rows][:, cols]), "columns that meet none"
    assert np.array_equal(got, _run(x, y0, ad, bd, ids, scales, out="y0"), equal_nan=True)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("m,k,n,r,e", SHAPES)
def test_a_x_next_to_the_largest_and_past_it(dev, m, k, n, r, e, dt):
    """A x is one element of x, or the sum of two: 3.4e38 in the rows of even number, infinite in the others."""
    print(f"lora, A x next to fp32's largest m={m} r={r} {dt}", flush=True)
    x, y0, a, b, ids, scales = _make(m, k, n, r, e, seed=m + r)
    a[:, 0] = 0.0
    a[:, 0, :2] = 1.0
    x[:, 0] = np.where(np.arange(m) % 4 < 2, MAX, np.float32(-3.3962e38))
    x[:, 1] = np.where(np.arange(m) % 2, x[:, 0], 0.0)
    a[:, 1:, :2] *= 1e-30
    b[:, :, 0] = np.where(rng(m).random((e, n)) < 0.5, -1.0, 1.0) * 2.0 ** -12
    ad, ah = _w(a, dt)
    bd, bh = _w(b, dt)
    got = _run(x, y0, ad, bd, ids, None)
    even = np.arange(m) % 2 == 0
    _same(got[even], y0[even], x[even], ah, bh, ids[even], None)
    odd = ~even
    sign = np.sign(x[odd, 0])[:, None] * np.sign(bh[ids[odd], :, 0])
    assert np.array_equal(got[odd], np.where(sign > 0, np.inf, -np.inf).astype(np.float32))


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("m,k,n,r,e", [(24, 128, 96, 16, 6), (1505, 64, 1001, 64, 6)])
def test_infinities_in_y0(dev, m, k, n, r, e, dt):
    """In rows with an adapter and without: they stay, and no other element changes; in place as well."""
    print(f"lora with infinities in y0 m={m} r={r} {dt}", flush=True)
    x, y0, a, b, ids, scales = _make(m, k, n, r, e, seed=m + r)
    ids[5::7] = -1
    (ad, ah), (bd, bh) = _w(a, dt), _w(b, dt)
    clean = _run(x, y0, ad, bd, ids, scales)
    y0[5, 3], y0[6, n - 1], y0[7, 0], y0[12, 8] = np.inf, -np.inf, np.nan, np.nan
    got = _run(x, y0, ad, bd, ids, scales)
    odd = ~np.isfinite(y0)
    assert np.array_equal(got[odd], y0[odd], equal_nan=True) and np.array_equal(got[~odd], clean[~odd])
    assert np.array_equal(got, _run(x, y0, ad, bd, ids, scales, out="y0"), equal_nan=True)
