"""GPU: the kernel that takes many query rows over Q4_0 K and V (enough of them that it is chosen: a masked
call then needs workspace for the mask's summary whatever else), rows sampled, against 64 bits."""
import numpy as np
import pytest
from helpers import randn, rng, to_dev
from test_gpu_fattn_q4 import TYPES, _cache, _check, _lengths_mask, _mask_dev, _q

from acestep_ops import ops
from acestep_ops.device import DTensor, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu
HEADS = {64: (32, 8), 128: (32, 8), 256: (16, 4)}
N, NQ = 8, 130


class Call:
    def __init__(self, D, n, dt, out, mask, seed, n_q=NQ, n_seqs=N, nk3=None, heads=None):
        self.nh, self.nkv = heads or HEADS[D]
        self.D, self.n, self.n_q, self.N, self.mask = D, n, n_q, n_seqs, mask
        self.qd, self.qx = _q(randn((n_seqs, n_q, self.nh, D), seed=seed), dt)
        self.k, self.v = _cache(nk3 or n_seqs, self.nkv, n, D, seed + 1), _cache(nk3 or n_seqs, self.nkv, n, D, seed + 2)
        self.scale = float(np.float32(D ** -0.5))
        self.y = DTensor.full_byte((n_seqs, n_q, self.nh, D), 0xFF, out)
        self.md = None if mask is None else _mask_dev(mask)
        self.upload()

    def upload(self):
        self.kd, self.vd = ops.Q4(to_dev(self.k)), ops.Q4(to_dev(self.v))
        qv = self.qd.permute(0, 2, 1, 3)
        need = ops.flash_attn_workspace(qv, self.kd, self.vd)
        assert need >= self.N * self.nh * ((self.n_q + 15) // 16) * ((self.n + 63) // 64), "the kernel for many rows"
        self.ws = DTensor.full_byte((max(need, 16),), 0xFF)

    def run(self, stream=None):
        ops.flash_attn_ext(self.qd.permute(0, 2, 1, 3), self.kd, self.vd, self.md, self.scale, out=self.y, workspace=self.ws,
                           stream=stream)

    def check(self, count=60, rows=()):
        r = rng(self.n + self.D)
        pick = [(0, 0, 0), (self.N - 1, self.nh - 1, self.n_q - 1), *rows]
        pick += [(int(r.integers(self.N)), int(r.integers(self.nh)), int(r.integers(self.n_q))) for _ in range(count)]
        _check(self.y, self.qx.transpose(0, 2, 1, 3), self.k, self.v, self.mask, self.scale, pick)


@pytest.mark.parametrize("dt,out", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 31, 64, 65, 700])
def test_masks_with_values_holes_and_empty_rows(dev, dt, out, D, n):
    print(f"q4 attention many rows D={D} n={n} {dt}->{out}", flush=True)
    r = rng(n)
    mask = np.where(r.random((N, 1, NQ, n)) < 0.3, -np.inf, r.standard_normal((N, 1, NQ, n)).astype(np.float16))
    mask[1] = np.where(np.arange(n) <= np.arange(NQ)[:, None] * n // NQ, 0.0, -np.inf)  # no values: a tile may be clean
    mask[2, 0, 3:40] = -np.inf
    mask[3] = -np.inf
    mask[4] = -65504.0
    c = Call(D, n, dt, out, mask, seed=D + n)
    c.run()
    c.check(rows=[(b, h, i) for b, h, i in ((1, 3, 0), (1, 0, NQ - 1), (2, 5, 3), (2, 1, 40), (3, 0, 0), (4, 2, 77))])


@pytest.mark.parametrize("dt,out", TYPES[:2])
@pytest.mark.parametrize("D,n", [(64, 300), (128, 257), (128, 1025), (256, 130)])
def test_no_mask_and_a_mask_per_head(dev, dt, out, D, n):
    print(f"q4 attention many rows, no mask / per head, D={D} n={n} {dt}->{out}", flush=True)
    c = Call(D, n, dt, out, None, seed=D + n)
    c.run()
    c.check()
    nh = HEADS[D][0]
    c.mask = np.where(rng(3).random((1, nh, NQ, n)) < 0.5, -np.inf, 0.0).astype(np.float64)
    c.mask[0, 1] = -np.inf
    c.md = _mask_dev(c.mask)
    c.run()
    c.check(rows=[(0, 1, 0), (5, 1, 9), (5, 0, 9)])


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_bytes_that_are_no_numbers_behind_the_mask(dev, D, out):
    """Slots past the last position of a sequence hold NaN and infinite blocks, or the largest d."""
    print(f"q4 attention many rows, bad bytes behind the mask D={D} {out}", flush=True)
    n, past = 333, np.array([0, 5, 100, 202, 203, 60, 63, 64])
    c = Call(D, n, "bf16", out, _lengths_mask(N, NQ, n, past), seed=D)
    k0, v0 = c.k.copy(), c.v.copy()
    for b in range(N):
        for t, bits in ((c.k, 0x7E00), (c.v, 0xFC00), (c.v, 0x7C00)):
            sl = slice(past[b] + NQ, n, 2 if bits == 0x7C00 else 1)
            w = t[b, :, sl].reshape(*t[b, :, sl].shape[:-1], D // 32, 18)
            w[..., :2] = np.array([bits], np.uint16).view(np.uint8)
            t[b, :, sl] = w.reshape(t[b, :, sl].shape)
    c.upload()
    c.run()
    c.k, c.v = k0, v0  # what is behind the mask does not count
    c.check(rows=[(b, 0, NQ - 1) for b in range(N)])


@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_large_scales_in_some_tiles(dev, out):
    print(f"q4 attention many rows, d near fp16's largest, {out}", flush=True)
    c = Call(128, 400, "bf16", out, None, seed=9)
    for t, f in ((c.v, 30000.0), (c.k, 0.0)):
        w = t.reshape(*t.shape[:-1], -1, 18)
        w[:, :, 100:140, 1, :2] = np.array([f], np.float16).view(np.uint8)
    c.upload()
    c.run()
    c.check()


@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_more_keys_than_a_workgroup_lists(dev, out):
    """Every workgroup slot taken and more tiles than one workgroup keeps a bit for: still split."""
    print(f"q4 attention many rows, 270000 keys, {out}", flush=True)
    n, n_q = 270000, 5
    mask = np.zeros((1, 1, n_q, n))
    mask[0, 0, 1, 1000:] = -np.inf
    mask[0, 0, 2, :269999] = -np.inf
    mask[0, 0, 3] = -np.inf
    c = Call(64, n, "bf16", out, mask, seed=1, n_q=n_q, n_seqs=512, nk3=1, heads=(16, 1))
    c.run()
    c.check(count=6, rows=[(7, 3, i) for i in range(5)])


def test_two_graphs_share_a_workspace_in_turn(dev):
    print("q4 attention many rows, two graphs", flush=True)
    st = Stream()
    calls = [Call(128, n, "bf16", out, _lengths_mask(N, NQ, n, np.arange(N) * 3), seed=n) for n, out in ((160, "f32"), (900, "bf16"))]
    ws = max((c.ws for c in calls), key=lambda w: w.numel())
    graphs = []
    for c in calls:
        c.ws = ws
        c.run(st.handle)
        st.synchronize()
        c.want = c.y.numpy()
        g = Graph()
        with g.capture(st):
            c.run(st.handle)
        graphs.append(g)
    for rep in range(3):
        for c in calls:
            c.y.fill_byte(0xFF)
        ws.fill_byte(0xFF)
        ops.add(to_dev(randn((8, 8), seed=1)), to_dev(randn((8, 8), seed=2)))
        synchronize()
        for g in graphs:
            g.launch()
        st.synchronize()
        for c in calls:
            assert np.array_equal(c.y.numpy(), c.want), f"replay {rep}"
    for c in calls:
        c.check(count=20)
