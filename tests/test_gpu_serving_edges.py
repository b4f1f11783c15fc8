"""GPU: the serving operators' operands at the edges of what they take: views at odd offsets for both attention
kernels, high ranks with many rows, two streams at once; each against the oracle of its own tests."""
import numpy as np
import pytest
from helpers import randn, rng, to_dev, to_np
from test_gpu_fattn_q4 import _cache, _check as check_attention, _lengths_mask, _mask_dev, _q
from test_gpu_logits import _case as logits_case, _ref as logits_ref
from test_gpu_lora import _case as lora_case, _check as check_lora, _run as run_lora

from acestep_ops import ops
from acestep_ops.device import DTensor, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu


def _wide(x, dt, lead):
    """x inside rows that start `lead` elements into wider ones: (view, values)"""
    w = np.concatenate([np.ones(x.shape[:-1] + (lead,), np.float32), x, np.ones(x.shape[:-1] + (3,), np.float32)], -1)
    d, v = _q(w, dt)
    return d[..., lead:lead + x.shape[-1]], v[..., lead:lead + x.shape[-1]]


@pytest.mark.parametrize("dt,out", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("D,N,nh,nkv,n_q", [(64, 2, 4, 2, 1), (128, 2, 4, 2, 7), (64, 8, 32, 8, 130), (128, 8, 32, 8, 130),
                                            (256, 8, 16, 4, 130)])
def test_attention_operands_at_odd_offsets(dev, D, N, nh, nkv, n_q, dt, out):
    """q, y and mask rows at odd elements, caches from an odd slot of larger ones, a mask row per head, replayed."""
    print(f"q4 attention, odd offsets, D={D} n_q={n_q} {dt}->{out}", flush=True)
    n, lead = 205, 9
    qd, qx = _wide(randn((N, n_q, nh, D), seed=D), dt, 3)
    k, v = _cache(N, nkv, 300, D, 2), _cache(N, nkv, 300, D, 3)
    kd, vd = ops.Q4(to_dev(k)[:, :, 5:5 + n]), ops.Q4(to_dev(v)[:, :, 5:5 + n])
    assert D != 64 or (kd.data.ptr - kd.data.buf.ptr) % 8 == 4  # rows of 36 bytes: 4-byte aligned
    mask = np.where(rng(4).random((N, nh, n_q, n)) < 0.4, -np.inf, rng(5).standard_normal((N, nh, n_q, n)).astype(np.float16))
    mask[0, 1, 0] = -np.inf
    mw = np.zeros((N, nh, n_q, n + lead + 2))
    mw[..., lead:lead + n] = mask
    yw = DTensor.full_byte((N, n_q, nh, D + 5), 0x7F, out)
    y = yw[..., 1:1 + D]
    args = (qd.permute(0, 2, 1, 3), kd, vd, _mask_dev(mw)[..., lead:lead + n], 0.1)
    st, g = Stream(), Graph()
    ws = DTensor.full_byte((max(ops.flash_attn_workspace(*args[:3]), 16),), 0xFF)
    ops.flash_attn_ext(*args, out=y, workspace=ws, stream=st.handle)
    st.synchronize()
    eager = to_np(yw)
    pick = [(0, 1, 0), (0, 0, 0), (N - 1, nh - 1, n_q - 1)]
    pick += [(i % N, (7 * i) % nh, (11 * i) % n_q) for i in range(40)]
    pos = DTensor.from_numpy(np.ascontiguousarray(eager[..., 1:1 + D]), out) if out == "bf16" else DTensor.from_numpy(
        np.ascontiguousarray(eager[..., 1:1 + D]))
    check_attention(pos, qx.transpose(0, 2, 1, 3), k[:, :, 5:5 + n], v[:, :, 5:5 + n], mask, 0.1, pick)
    edge = np.ascontiguousarray(np.concatenate([eager[..., :1], eager[..., 1 + D:]], -1))
    assert (edge.view(np.uint8) == 0x7F).all(), "around y"
    with g.capture(st):
        ops.flash_attn_ext(*args, out=y, workspace=ws, stream=st.handle)
    for rep in range(2):
        yw.fill_byte(0x7F)
        ws.fill_byte(0xFF)
        synchronize()
        g.launch()
        st.synchronize()
        assert np.array_equal(to_np(yw).view(np.uint8), eager.view(np.uint8)), f"replay {rep}"


@pytest.mark.parametrize("m,k,n,r,e,dt", [(100, 64, 515, 256, 3, "bf16"), (70, 96, 258, 100, 9, "f16"), (65, 64, 4, 129, 2, "bf16"),
                                          (200, 320, 1030, 33, 40, "f16"), (66, 32, 3, 7, 5, "f16"), (64, 64, 130, 200, 70, "bf16"),
                                          (1000, 32, 257, 1, 1, "f16")])
def test_adapters_of_many_rows_and_ranks(dev, m, k, n, r, e, dt):
    print(f"lora m={m} k={k} n={n} r={r} e={e} {dt}", flush=True)
    x, y0, a, ah, b, bh, ids, scales = lora_case(m, k, n, r, e, dt, seed=m + r)
    got = run_lora(x, y0, a, b, ids, scales)
    check_lora(got, y0, x, ah, bh, ids, scales)
    assert np.array_equal(got, run_lora(x, y0, a, b, ids, scales, out="y0"))


@pytest.mark.parametrize("run", [1, 37, 400])
@pytest.mark.parametrize("m,k,n,r,e,dt", [(1500, 32, 1030, 33, 40, "f16"), (1500, 64, 1027, 256, 3, "bf16"), (1600, 32, 1001, 100, 9, "bf16"),
                                          (1501, 96, 1000, 16, 5, "f16"), (3100, 64, 515, 64, 7, "bf16"), (1505, 32, 1002, 129, 2, "f16")])
def test_adapters_of_wide_tiles(dev, m, k, n, r, e, dt, run):
    """Enough rows and columns for the kernel with 4 columns a lane, runs of one adapter, columns that are no whole 4."""
    print(f"lora wide m={m} k={k} n={n} r={r} e={e} {dt} run={run}", flush=True)
    ids = np.repeat(rng(m).integers(-1, e, (m + run - 1) // run), run)[:m]
    x, y0, a, ah, b, bh, ids, scales = lora_case(m, k, n, r, e, dt, seed=m + r, ids=ids)
    got = run_lora(x, y0, a, b, ids, scales)
    check_lora(got, y0, x, ah, bh, ids, scales)
    assert np.array_equal(got, run_lora(x, y0, a, b, ids, scales, out="y0"))


def test_adapters_in_place_on_columns_of_a_wider_buffer(dev):
    """Two products' columns of one buffer take their own adapters in place; x with outer dimensions."""
    print("lora, columns of a wider buffer", flush=True)
    for m in (12, 90, 16000):
        x, y0, a, ah, b, bh, ids, scales = lora_case(m, 64, 96, 16, 4, "bf16", seed=m)
        wide = np.concatenate([randn((m, 33), seed=1), y0, randn((m, 40), seed=2)], 1)
        wd = to_dev(wide)
        xd = to_dev(x.reshape(2, m // 2, 64))
        y = wd[:, 33:129].unflatten(0, (2, m // 2))
        ops.lora_add(y, xd, a, b, to_dev(ids), to_dev(scales), out=y)
        got = to_np(wd)
        check_lora(np.ascontiguousarray(got[:, 33:129]), y0, x, ah, bh, ids, scales)
        assert np.array_equal(got[:, :33], wide[:, :33]) and np.array_equal(got[:, 129:], wide[:, 129:])


def test_two_streams_at_once(dev):
    """Attention, adapters and logits on two streams with workspaces of their own give what one stream gives."""
    print("serving operators on two streams", flush=True)
    st = [Stream(), Stream()]
    jobs = []
    for i, (N, nh, nkv, n_q, n) in enumerate(((4, 8, 2, 1, 900), (8, 32, 8, 130, 300))):
        qd, _ = _q(randn((N, n_q, nh, 128), seed=i), "f32")
        k, v = _cache(N, nkv, n, 128, 10 + i), _cache(N, nkv, n, 128, 20 + i)
        kd, vd = ops.Q4(to_dev(k)), ops.Q4(to_dev(v))
        mask = _mask_dev(_lengths_mask(N, n_q, n, np.arange(N) * 10))
        x, y0, a, _, b, _, ids, scales = lora_case(16 * N, 256, 300, 16, 5, "bf16", seed=30 + i)
        hist, lens, pen, bias, allowed, state = (to_dev(t) for t in logits_case(N, 5000, 300, 3, seed=40 + i))
        xd, yd, idd, sd, lg = to_dev(x), to_dev(y0), to_dev(ids), to_dev(scales), to_dev(randn((N, 5000), seed=50 + i))
        outs = [DTensor.empty((N, n_q, nh, 128), "f32"), DTensor.empty(y0.shape, "f32"), DTensor.empty((N, 5000), "f32")]
        qv = qd.permute(0, 2, 1, 3)
        ws = [DTensor.empty((max(ops.flash_attn_workspace(qv, kd, vd), 16),), "u8"), DTensor.empty((ops.lora_add_workspace(xd, a, b),), "u8")]

        def job(s, qv=qv, kd=kd, vd=vd, mask=mask, outs=outs, ws=ws, xd=xd, yd=yd, a=a, b=b, idd=idd, sd=sd, lg=lg, hist=hist,
                lens=lens, pen=pen, bias=bias, allowed=allowed, state=state):
            ops.flash_attn_ext(qv, kd, vd, mask, 0.09, out=outs[0], workspace=ws[0], stream=s)
            ops.lora_add(yd, xd, a, b, idd, sd, out=outs[1], workspace=ws[1], stream=s)
            ops.logits_adjust(lg, hist, lens, pen, bias, allowed, state, out=outs[2], stream=s)

        jobs.append((job, outs))
    synchronize()
    want = []
    for job, outs in jobs:
        job(st[0].handle)
        st[0].synchronize()
        want.append([to_np(o) for o in outs])
    for rep in range(4):
        for _, outs in jobs:
            for o in outs:
                o.fill_byte(0xFF)
        synchronize()
        for _ in range(3):
            for s, (job, _) in zip(st, jobs):
                job(s.handle)
        for s in st:
            s.synchronize()
        for (_, outs), w in zip(jobs, want):
            for o, ref in zip(outs, w):
                assert np.array_equal(to_np(o), ref, equal_nan=True), f"round {rep}"


def test_logits_of_one_row_state_and_one_token_histories(dev):
    print("logits, histories of one token, a bias per row and for all", flush=True)
    m, V = 4, 4097
    x = randn((m, V), seed=1)
    hist = np.array([[V - 1], [0], [4096 - 1], [2048]], np.int32)
    pen = np.array([[2, 0, 0], [1, 0.5, 0], [1, 0, 0.25], [0.5, 1, 1]], np.float32)
    allowed = rng(2).integers(-2 ** 31, 2 ** 31, (1, (V + 31) // 32)).astype(np.int32)
    for bias in (randn((1, V), seed=3), randn((m, V), seed=4)):
        y = ops.logits_adjust(to_dev(x), to_dev(hist), None, to_dev(pen), to_dev(bias), to_dev(allowed))
        assert np.array_equal(to_np(y), logits_ref(x, hist, None, pen, bias, allowed, None))
