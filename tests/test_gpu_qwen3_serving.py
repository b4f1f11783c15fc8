"""GPU: decode and prompt steps of requests that share a layer (acestep_ops.qwen3.Qwen3Layer and
Qwen3Head): Q4_0 caches, each row's own low-rank adapter on all four products, and the requests'
penalties, biases and grammars on the logits. Every stage is checked against the oracle applied to the
device's own inputs of that stage, at that operator's own bar; a captured step replays to the same bits."""
import numpy as np
import pytest
import q4
from helpers import assert_f32_close, assert_mul_mat_q8_0, randn, rng, to_dev, to_np
from oracle import oracle as orc
from test_gpu_fattn_q4 import _check as check_attention
from test_gpu_logits import _case as logits_case
from test_gpu_logits import _ref as logits_ref
from test_gpu_lora import _check as check_adapters
from test_gpu_lora import _w as adapter_weights

from acestep_ops import ops
from acestep_ops.device import DTensor, Graph, Stream, synchronize
from acestep_ops.qwen3 import Qwen3Head, Qwen3Layer, causal_mask, decode_mask

pytestmark = pytest.mark.gpu
EPS, THETA = 1e-6, 1e6
# H, Nh, Nkv, D, I, slots, sets, first set
SIZES = {"small": (256, 4, 2, 128, 512, 300, 6, 1), "0.6b": (1024, 16, 8, 128, 3584, 2048, 9, 1)}


class Case:
    def __init__(self, size, clamp=False, stream=None, rank=8, n_adapters=4, only=("qkv", "o", "gu", "down")):
        self.H, self.Nh, self.Nkv, self.D, self.I, self.max_seq, n_sets, self.s0 = SIZES[size]
        H, Nh, Nkv, D, I = self.H, self.Nh, self.Nkv, self.D, self.I
        shapes = {"qkv": ((Nh + 2 * Nkv) * D, H), "o": (H, Nh * D), "gu": (2 * I, H), "down": (H, I)}
        self.w = {n: orc.quantize_q8_0(randn(s, seed=i, scale=0.05)) for i, (n, s) in enumerate(shapes.items())}
        self.norms = [(1 + 0.1 * randn((n,), seed=10 + i)).astype(np.float32) for i, n in enumerate((H, H, D, D))]
        self.lora, dev = {}, {}
        for i, n in enumerate(only):
            a, ah = adapter_weights(randn((n_adapters, rank, shapes[n][1]), seed=20 + i, scale=0.05), "bf16")
            b, bh = adapter_weights(randn((n_adapters, shapes[n][0], rank), seed=30 + i, scale=0.1), "bf16")
            self.lora[n], dev[n] = (ah, bh), (a, b)
        self.scales = np.linspace(0.5, 2.0, n_adapters).astype(np.float32)
        self.layer = Qwen3Layer(*(ops.Q8(to_dev(self.w[n])) for n in ("qkv", "o", "gu", "down")),
                                *(to_dev(n) for n in self.norms), H, Nh, Nkv, D, I, self.max_seq, n_sets, "q4_0", EPS,
                                THETA, clamp_fp16=clamp, stream=stream, adapters=dev, adapter_scales=to_dev(self.scales))
        self.cache0 = [q4.quantize(randn((n_sets, Nkv, self.max_seq, D), seed=40 + i, scale=0.5)) for i in (0, 1)]
        self.layer.k_cache, self.layer.v_cache = (ops.Q4(to_dev(c)) for c in self.cache0)

    def _product(self, name, x, got, ids):
        """The product of x (a buffer's name) and its adapters, both as the operators alone give them."""
        base = to_np(ops.mul_mat_q8_0(self.layer.w[name], self.layer._bufs[x]))
        xh = to_np(self.layer._bufs[x])
        assert_mul_mat_q8_0(base, self.w[name], xh)
        if name in self.lora:
            check_adapters(got, base, xh, *self.lora[name], ids, self.scales)
        else:
            assert np.array_equal(got, base)

    def check(self, y, hidden, pos, row_sets, ids, mask, S):
        """hidden, y (rows, H); pos, row_sets, ids per row; mask (N, 1, S, read) float."""
        Nh, Nkv, D = self.Nh, self.Nkv, self.D
        rows, N, read = len(hidden), len(hidden) // S, mask.shape[-1]
        L = self.layer
        b = {k: to_np(v) for k, v in L._bufs.items() if not k.startswith("ws")}
        assert_f32_close(b["n1"], orc.rms_norm_mul(hidden, self.norms[0], EPS), row_floor=True)
        self._product("qkv", "n1", b["qkv"], ids)
        q = b["qkv"][:, :Nh * D].reshape(rows, Nh, D)
        v = b["qkv"][:, (Nh + Nkv) * D:].reshape(rows, Nkv, D)
        dq = L._bufs["qkv"]
        _, ko = ops.qk_norm_rope(dq[:, :Nh * D].unflatten(1, (Nh, D)), to_dev(self.norms[2]), to_dev(pos), EPS, D,
                                 THETA, k=dq[:, Nh * D:(Nh + Nkv) * D].unflatten(1, (Nkv, D)), k_w=to_dev(self.norms[3]))
        assert_f32_close(b["qo"], orc.qk_norm_rope(q, self.norms[2], pos, EPS, D, THETA), row_floor=True)
        if L.clamp_fp16:
            v = orc.clamp(v, -65504.0, 65504.0)
        cache = [to_np(c.data) for c in (L.k_cache, L.v_cache)]
        want = [c.copy() for c in self.cache0]
        for c, x in zip(want, (to_np(ko), v)):
            c[row_sets, :, pos] = q4.quantize(x)
        assert np.array_equal(cache[0], want[0]) and np.array_equal(cache[1], want[1]), "caches"
        kr, vr = (c[self.s0:self.s0 + N, :, :read] for c in cache)
        qx = b["qo"].reshape(N, S, Nh, D).transpose(0, 2, 1, 3)
        pick = None if rows * Nh <= 256 else [(i % N, i % Nh, i % S) for i in range(0, rows * Nh, 7)]
        attn = DTensor.from_numpy(b["attn"].reshape(N, S, Nh, D))
        check_attention(attn, qx, kr, vr, mask, float(np.float32(D ** -0.5)), pick)
        L._bufs["a2"] = DTensor.from_numpy(b["attn"].reshape(rows, Nh * D))
        self._product("o", "a2", b["ao"], ids)
        h1 = orc.add_clamp(hidden, b["ao"]) if L.clamp_fp16 else orc.add(hidden, b["ao"])
        assert np.array_equal(b["h1"], h1)
        assert_f32_close(b["n2"], orc.rms_norm_mul(h1, self.norms[1], EPS), row_floor=True)
        self._product("gu", "n2", b["gu"], ids)
        assert np.array_equal(b["ff"], to_np(ops.swiglu(L._bufs["gu"])))
        assert_f32_close(b["ff"], orc.swiglu(b["gu"]), row_floor=True)
        self._product("down", "ff", b["dn"], ids)
        assert np.array_equal(y, orc.add_clamp(h1, b["dn"]) if L.clamp_fp16 else orc.add(h1, b["dn"]))


@pytest.mark.parametrize("size,N,clamp", [("small", 4, False), ("small", 1, True), ("0.6b", 8, False)])
def test_decode_step_and_head(dev, size, N, clamp):
    print(f"serving decode {size} N={N} clamp={clamp}", flush=True)
    c = Case(size, clamp)
    r = rng(5)
    pos = np.concatenate([[c.max_seq - 1], r.integers(0, c.max_seq, N - 1)]).astype(np.int32)
    sets = np.arange(c.s0, c.s0 + N, dtype=np.int32)
    ids = np.array([2, -1, 0, 2, 1, 3, 3, -1], np.int32)[:N]
    hidden = randn((N, c.H), seed=6)
    y = c.layer.forward(to_dev(hidden), to_dev(pos), to_dev(sets), c.s0, c.max_seq, decode_mask(pos, c.max_seq),
                        adapter_ids=to_dev(ids))
    mask = np.where(np.arange(c.max_seq) <= pos[:, None], 0.0, -np.inf).reshape(N, 1, 1, -1)
    c.check(to_np(y), hidden, pos, sets, ids, mask, 1)

    V = 1003
    wv, nw = orc.quantize_q8_0(randn((V, c.H), seed=7, scale=0.05)), randn((c.H,), seed=8)
    head = Qwen3Head(ops.Q8(to_dev(wv)), to_dev(nw), V, EPS)
    bare = to_np(head.forward(y))
    assert_mul_mat_q8_0(bare, wv, orc.rms_norm_mul(to_np(y), nw, EPS))
    hist, lens, pen, bias, allowed, state = logits_case(N, V, 200, 3, seed=9)
    got = head.forward(y, history=to_dev(hist), lengths=to_dev(lens), penalties=to_dev(pen), bias=to_dev(bias),
                       allowed=to_dev(allowed), state=to_dev(state))
    assert np.array_equal(to_np(got), logits_ref(bare, hist, lens, pen, bias, allowed, state))


@pytest.mark.parametrize("size,N,S", [("small", 2, 5), ("small", 1, 150), ("0.6b", 3, 40)])
def test_prompt_step(dev, size, N, S):
    print(f"serving prompt {size} N={N} S={S}", flush=True)
    c = Case(size)
    kv_pos = np.array([c.max_seq - S, 0, 17][:N])
    ids = np.array([1, -1, 3], np.int32)[:N]
    hidden = randn((N, S, c.H), seed=11)
    y = to_np(c.layer.prefill(to_dev(hidden), kv_pos, c.s0, adapter_ids=ids)).reshape(N * S, c.H)
    mask = to_np(causal_mask(kv_pos, S, int(kv_pos.max()) + S)).view(np.float16).astype(np.float64)
    pos = (kv_pos[:, None] + np.arange(S)).reshape(-1).astype(np.int32)
    c.check(y, hidden.reshape(N * S, c.H), pos, np.repeat(np.arange(c.s0, c.s0 + N), S), np.repeat(ids, S), mask, S)


@pytest.mark.parametrize("only", [("qkv", "o", "gu", "down"), ("qkv",), ("o", "down"), ("gu",)])
def test_rows_without_an_adapter_are_the_layer_without_adapters(dev, only):
    print(f"serving, adapters on {only}, no row has one", flush=True)
    N, pos = 4, np.array([3, 299, 0, 120], np.int32)
    hidden, sets = to_dev(randn((N, 256), seed=6)), to_dev(np.arange(1, 5, dtype=np.int32))
    mask = decode_mask(pos, 300)
    c, plain = Case("small", only=only), Case("small", only=())
    want = to_np(plain.layer.forward(hidden, to_dev(pos), sets, 1, 300, mask))
    assert np.array_equal(to_np(c.layer.forward(hidden, to_dev(pos), sets, 1, 300, mask)), want)
    none = to_dev(np.full(N, -1, np.int32))
    assert np.array_equal(to_np(c.layer.forward(hidden, to_dev(pos), sets, 1, 300, mask, adapter_ids=none)), want)
    mixed = to_dev(np.array([-1, 2, -1, 0], np.int32))
    got = to_np(c.layer.forward(hidden, to_dev(pos), sets, 1, 300, mask, adapter_ids=mixed))
    assert np.array_equal(got[[0, 2]], want[[0, 2]]) and (got[[1, 3]] != want[[1, 3]]).any(1).all()


def test_decode_steps_captured_and_replayed(dev):
    """Two steps of all operators in one graph; replays with eager work between them give the eager bits."""
    print("serving, captured", flush=True)
    st, N = Stream(), 4
    c = Case("small", stream=st.handle)
    V = 1003
    head = Qwen3Head(ops.Q8(to_dev(orc.quantize_q8_0(randn((V, c.H), seed=7, scale=0.05)))), to_dev(randn((c.H,), seed=8)),
                     V, EPS, stream=st.handle)
    hidden, sets, ids = to_dev(randn((N, c.H), seed=6)), to_dev(np.arange(1, 5, dtype=np.int32)), to_dev(
        np.array([2, -1, 0, 2], np.int32))
    steps = [np.array([3, 298, 0, 120], np.int32) + i for i in (0, 1)]
    pos, masks = [to_dev(p) for p in steps], [decode_mask(p, 300) for p in steps]
    hist, lens, pen, bias, allowed, state = (to_dev(t) for t in logits_case(N, V, 200, 3, seed=9))
    h, logits = DTensor.empty((N, c.H), "f32"), DTensor.empty((N, V), "f32")

    def run():
        x = hidden
        for p, m in zip(pos, masks):
            x = c.layer.forward(x, p, sets, c.s0, 300, m, out=h, adapter_ids=ids)
        head.forward(x, out=logits, history=hist, lengths=lens, penalties=pen, bias=bias, allowed=allowed, state=state)

    synchronize()
    run()
    st.synchronize()
    want = [to_np(t) for t in (h, logits, c.layer.k_cache.data, c.layer.v_cache.data)]
    g = Graph()
    with g.capture(st):
        run()
    for rep in range(3):
        for t in (h, logits):
            t.fill_byte(0xFF)
        for t, b in zip((c.layer.k_cache.data, c.layer.v_cache.data), c.cache0):  # the slots of both steps as before
            ops.cpy(to_dev(b.view(np.float32)), DTensor(t.buf, t.shape[:-1] + (t.shape[-1] // 4,), "f32"))
        ops.add(hidden, hidden)
        synchronize()
        g.launch()
        st.synchronize()
        for t, w in zip((h, logits, c.layer.k_cache.data, c.layer.v_cache.data), want):
            assert np.array_equal(to_np(t), w, equal_nan=t is logits), f"replay {rep}"


@pytest.mark.parametrize("kv_type", ["q4_0", "q8_0"])
def test_a_graph_per_read_length(dev, kv_type):
    """Steps captured at growing read lengths, each needing more workspace than the one before, all replayed."""
    print(f"serving, a graph per read length, {kv_type}", flush=True)
    st, N, H = Stream(), 2, 256
    w = {n: orc.quantize_q8_0(randn(s, seed=i, scale=0.05))
         for i, (n, s) in enumerate({"qkv": (1024, H), "o": (H, 512), "gu": (1024, H), "down": (H, 512)}.items())}
    layer = Qwen3Layer(*(ops.Q8(to_dev(w[n])) for n in ("qkv", "o", "gu", "down")), *(to_dev(randn((n,), seed=n)) for n in (H, H, 128, 128)),
                       H, 4, 2, 128, 512, 4096, N, kv_type, EPS, THETA, stream=st.handle)
    hidden, sets, out = to_dev(randn((N, H), seed=6)), to_dev(np.arange(N, dtype=np.int32)), DTensor.empty((N, H), "f32")
    steps = []
    for read in (256, 1024, 4096):
        pos = np.array([read - 1, read // 2], np.int32)
        args = (hidden, to_dev(pos), sets, 0, read, decode_mask(pos, read))
        layer.forward(*args, out=out)
        st.synchronize()
        want, g = to_np(out), Graph()
        with g.capture(st):
            layer.forward(*args, out=out)
        steps.append((g, want, args))
    filler = [DTensor.full_byte((1 << 20,), 0xFF) for _ in range(8)]  # over memory that was given back, were it
    for rep in range(2):
        for g, want, _ in steps:
            out.fill_byte(0xFF)
            synchronize()
            g.launch()
            st.synchronize()
            assert np.array_equal(to_np(out), want), f"replay {rep}"
    assert all((to_np(f) == 0xFF).all() for f in filler)
