"""Serving operators of the LM, each one pass: a Q4_0 KV cache, adapters, logits.

  append     keys and values of new tokens quantized into Q4_0 caches (mi_kv_store), the written
             rows read back as numbers (mi_get_rows)
  attention  flash attention over Q4_0 K and V: single tokens and prompts (mi_flash_attn_ext)
  lora       low-rank adapters of many requests beside a shared projection (mi_lora_add)
  logits     repetition, frequency and presence penalties, biases and grammar masks (mi_logits_adjust)

With own = False each pass is computed by elementary torch operations in 32 bits; with
own = True by the library. exact() gives the same outputs in 64 bits.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

# H, query heads, KV heads, head size of the served LMs
QWEN3 = {"0.6B": (1024, 16, 8, 128), "1.7B": (2048, 16, 8, 128), "4B": (2560, 32, 8, 128)}
VOCAB = 151669
_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# --- the cases --------------------------------------------------------------------
def listed():
    return [
        # one decode step's K and V of a batch of four songs with CFG
        {"name": "append_decode_b8", "op": "append", "seqs": 8, "tokens": 1, "slots": 1024, "heads": 8, "d": 128,
         "type": "f32", "read": "f32"},
        # a prompt batch's K and V, read back whole
        {"name": "append_prompt_8x2048", "op": "append", "seqs": 8, "tokens": 2048, "slots": 2304, "heads": 8, "d": 128,
         "type": "bf16", "read": "bf16"},
        # one token of one sequence on the smallest LM: latency
        {"name": "attn_0.6b_b1", "op": "attention", "seqs": 1, "nq": 1, "past": 699, "heads": 16, "kv_heads": 8, "d": 128,
         "type": "bf16", "idle": 0},
        # a batch of four songs with CFG, long contexts, F32 activations as the LM layer has them
        {"name": "attn_4b_b8", "op": "attention", "seqs": 8, "nq": 1, "past": 6599, "heads": 32, "kv_heads": 8, "d": 128,
         "type": "f32", "idle": 0},
        # few sequences at a context far past the usual, one place of the batch idle
        {"name": "attn_4b_b3_long", "op": "attention", "seqs": 3, "nq": 1, "past": 60012, "heads": 32, "kv_heads": 8,
         "d": 128, "type": "bf16", "idle": 1},
        # an odd-sized continuation of a cached prompt
        {"name": "attn_1.7b_257", "op": "attention", "seqs": 1, "nq": 257, "past": 130, "heads": 16, "kv_heads": 8,
         "d": 128, "type": "f32", "idle": 0},
        # the largest prompt batch
        {"name": "attn_4b_8x2048", "op": "attention", "seqs": 8, "nq": 2048, "past": 0, "heads": 32, "kv_heads": 8,
         "d": 128, "type": "bf16", "idle": 0},
        # decode: eight requests, each its own adapter, on the QKV projection
        {"name": "lora_qkv_b8", "op": "lora", "rows": 8, "k": 2560, "n": 6144, "rank": 16, "adapters": 8, "run": 1,
         "type": "bf16"},
        # decode: a large batch over many adapters of high rank, on the O projection
        {"name": "lora_o_b48", "op": "lora", "rows": 48, "k": 4096, "n": 2560, "rank": 64, "adapters": 24, "run": 1,
         "type": "f16"},
        # prompts of three requests one after another, on the gate/up projection
        {"name": "lora_gate_up_4005", "op": "lora", "rows": 4005, "k": 2560, "n": 19456, "rank": 32, "adapters": 3,
         "run": 1335, "type": "bf16"},
        # a batch of eight requests, one of them without a grammar
        {"name": "logits_b8", "op": "logits", "rows": 8, "vocab": VOCAB, "history": 1200, "states": 5, "type": "f32"},
        # the largest batch with long histories
        {"name": "logits_b64", "op": "logits", "rows": 64, "vocab": VOCAB, "history": 8000, "states": 40, "type": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "attention", "lora", "lora", "logits"])
    if op == "append":
        seqs, tokens = rng.randint(1, 8), rng.choice([1, 1, _log(rng, 2, 2048)])
        return {"op": op, "seqs": seqs, "tokens": tokens, "slots": tokens + rng.randint(0, 300),
                "heads": rng.choice([1, 2, 4, 5, 8]), "d": rng.choice([64, 128, 128, 256]),
                "type": rng.choice(["f32", "bf16", "f16"]), "read": rng.choice(["f32", "bf16"])}
    if op == "attention":
        d = rng.choice([64, 128, 128, 128, 256])
        kv_heads = rng.choice([1, 2, 4, 8, 8])
        heads = kv_heads * rng.choice([1, 2, 2, 4, 4, 6, 8] if kv_heads > 1 else [1, 4, 8, 16])
        seqs = rng.randint(1, 8)
        kind = rng.choice(["token", "token", "few", "prompt", "prompt"])
        if kind == "prompt":
            nq, past = _log(rng, 16, 2000), rng.choice([0, 0, rng.randint(1, 400)])
            seqs = min(seqs, max(1, 6000 // nq))
            heads = min(heads, 32) // kv_heads * kv_heads
        else:
            nq = 1 if kind == "token" else rng.randint(2, 7)
            past = _log(rng, 1, 60000) - 1
            seqs = min(seqs, max(1, 150000 // (past + 1)))
        idle = 1 if seqs > 1 and rng.random() < 0.25 else 0
        return {"op": op, "seqs": seqs, "nq": nq, "past": past, "heads": heads, "kv_heads": kv_heads, "d": d,
                "type": rng.choice(["f32", "bf16"]), "idle": idle}
    if op == "lora":
        H, Nh, Nkv, D = QWEN3[rng.choice(list(QWEN3))]
        k, n = rng.choice([(H, (Nh + 2 * Nkv) * D), (Nh * D, H), (2560, 19456), (9728, 2560)])
        if rng.random() < 0.5:
            rows, run = rng.randint(1, 64), 1
            adapters = rng.randint(1, 32)
        else:
            rows = _log(rng, 65, 3900)
            run = max(1, rows // rng.randint(1, 9))
            adapters = rng.randint(1, 8)
        return {"op": op, "rows": rows, "k": k, "n": n, "rank": rng.choice([1, 4, 8, 12, 16, 16, 20, 32, 64]),
                "adapters": adapters, "run": run, "type": rng.choice(["bf16", "f16"])}
    return {"op": op, "rows": _log(rng, 1, 60), "vocab": _log(rng, 700, 150000), "history": _log(rng, 1, 8000),
            "states": rng.randint(0, 12), "type": rng.choice(["f32", "f32", "bf16"])}


# --- inputs, made from the seed alone -------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 29)


def _randn(g, *shape, std=1.0, mean=0.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(dtype)


def _randint(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int32)


def _q4_pack(x):
    """(..., D) F32 -> Q4_0 bytes (..., D / 32 * 18): per block d = (its first value of the largest
    magnitude) / -8, q = min(15, floor(x / d + 8.5)); fp16 d, then 16 bytes of q_j | q_(j+16) << 4."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    a = b.abs()
    first = torch.where(a == a.amax(-1, keepdim=True), torch.arange(32, device=x.device), 32).amin(-1, keepdim=True)
    d = torch.gather(b, -1, first.clamp(max=31)) / -8.0
    inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
    q = torch.clamp(torch.floor(b * inv + 8.5), 0, 15).to(torch.uint8)
    out = torch.empty(*b.shape[:-1], 18, dtype=torch.uint8, device=x.device)
    out[..., :2] = d.half().view(torch.uint8)
    out[..., 2:] = q[..., :16] | (q[..., 16:] << 4)
    return out.reshape(*x.shape[:-1], -1)


def _q4_values(c):
    """Q4_0 bytes (..., D / 32 * 18) -> the F32 values (..., D) they stand for."""
    b = c.reshape(*c.shape[:-1], -1, 18)
    d = b[..., :2].contiguous().view(torch.float16).float()
    q = torch.cat([b[..., 2:] & 15, b[..., 2:] >> 4], -1).float() - 8.0
    return (q * d).reshape(*c.shape[:-1], -1)


def _append_inputs(case, seed):
    g = _gen(seed)
    B, T, M, H, D = case["seqs"], case["tokens"], case["slots"], case["heads"], case["d"]
    t = _TORCH[case["type"]]
    s = {"k": _randn(g, B, T, H, D, dtype=t), "v": _randn(g, B, T, H, D, dtype=t),
         "k_cache": _q4_pack(_randn(g, B, H, M, D)), "v_cache": _q4_pack(_randn(g, B, H, M, D)),
         "pos0": _randint(g, 0, M - T + 1, B), "sets": torch.randperm(B, generator=g, device="cuda").to(torch.int32)}
    # the written rows of the caches seen as tables of B * H * M rows, in (sequence, head, token) order
    slot = s["pos0"][:, None] + torch.arange(T, device="cuda", dtype=torch.int32)
    row = (s["sets"][:, None] * H + torch.arange(H, device="cuda", dtype=torch.int32)) * M
    s["rows"] = (row[:, :, None] + slot[:, None, :]).reshape(-1).to(torch.int32)
    for name in ("k_read", "v_read"):
        s[name] = torch.empty(B * H * T, D, dtype=_TORCH[case["read"]], device="cuda")
    return s


def _attention_inputs(case, seed):
    g = _gen(seed)
    N, S, Nh, Nkv, D = case["seqs"], case["nq"], case["heads"], case["kv_heads"], case["d"]
    kv = case["past"] + S
    read = (kv + 255) // 256 * 256 if S == 1 else kv  # single tokens read the cache bucketed by 256 slots
    t = _TORCH[case["type"]]
    chan = torch.exp(0.3 * torch.randn(D, generator=g, device="cuda"))  # K's channels differ in size
    s = {"q": _randn(g, N, S, Nh, D, dtype=t), "k": _q4_pack(_randn(g, N, Nkv, read, D) * chan),
         "v": _q4_pack(_randn(g, N, Nkv, read, D)), "scale": float(np.float32(1.0 / math.sqrt(D)))}
    past = _randint(g, case["past"] // 8, case["past"] + 1, N)
    past[0] = case["past"]
    if case["idle"]:
        past[N - 1] = -S  # nothing to attend to
    s["past"] = past
    last = past[:, None] + torch.arange(S, device="cuda")
    dead = torch.arange(read, device="cuda")[None, None, :] > last[:, :, None]
    if case["idle"]:
        dead[N - 1] = True
    s["mask"] = torch.zeros(N, 1, S, read, dtype=torch.float16, device="cuda").masked_fill_(dead[:, None], float("-inf"))
    s["y"] = torch.empty(N, S, Nh, D, dtype=t, device="cuda")
    return s


def _lora_inputs(case, seed):
    g = _gen(seed)
    m, k, n, r, e = case["rows"], case["k"], case["n"], case["rank"], case["adapters"]
    t = _TORCH[case["type"]]
    ids = _randint(g, 0, e, (m + case["run"] - 1) // case["run"])
    if m > 4:
        ids[-1] = -1  # a request without an adapter
    return {"x": _randn(g, m, k), "y0": _randn(g, m, n), "a": _randn(g, e, r, k, std=k ** -0.5, dtype=t),
            "b": _randn(g, e, n, r, std=r ** -0.5, dtype=t), "ids": ids.repeat_interleave(case["run"])[:m].contiguous(),
            "scales": torch.rand(e, generator=g, device="cuda") + 0.5, "y": torch.empty(m, n, device="cuda")}


def _logits_inputs(case, seed):
    g = _gen(seed)
    m, V, L, S = case["rows"], case["vocab"], case["history"], case["states"]
    t = _TORCH[case["type"]]
    u = torch.rand(m, L, generator=g, device="cuda")
    s = {"logits": _randn(g, m, V, std=3.0, dtype=t),
         # tokens come back: a few often, most once
         "history": (V * u * u * u).to(torch.int32).clamp(max=V - 1),
         "lengths": _randint(g, 0, L + 1, m),
         "penalties": torch.stack([1.0 + 0.5 * torch.rand(m, generator=g, device="cuda"),
                                   0.3 * torch.rand(m, generator=g, device="cuda"),
                                   0.5 * torch.rand(m, generator=g, device="cuda")], 1),
         "bias": _randn(g, 1, V) * (torch.rand(1, V, generator=g, device="cuda") < 0.01),
         "y": torch.empty(m, V, dtype=t, device="cuda")}
    if S:
        words = (V + 31) // 32
        bits = torch.randint(-2 ** 31, 2 ** 31, (S, words), generator=g, device="cuda")
        bits[0] &= torch.randint(-2 ** 31, 2 ** 31, (words,), generator=g, device="cuda")
        s["allowed"] = bits.to(torch.int32)
        s["state"] = _randint(g, 0, S, m)
        if m > 1:
            s["state"][m // 2] = -1  # a request without a grammar
    return s


def prepare(case, seed):
    make = {"append": _append_inputs, "attention": _attention_inputs, "lora": _lora_inputs, "logits": _logits_inputs}
    s = make[case["op"]](case, seed)
    s["op"] = case["op"]
    return s


# --- the plain forms --------------------------------------------------------------------
def _plain_append(s):
    got = []
    for name in ("k", "v"):
        x, cache = s[name], s[name + "_cache"]
        rows = cache.reshape(-1, cache.shape[-1])
        rows[s["rows"].long()] = _q4_pack(x.float().transpose(1, 2)).reshape(-1, cache.shape[-1])
        got.append(_q4_values(rows[s["rows"].long()]).to(s[name + "_read"].dtype))
    return got


def _plain_attention(s):
    N, S, Nh, D = s["q"].shape
    Nkv, n = s["k"].shape[1], s["k"].shape[2]
    rep = Nh // Nkv
    q = s["q"].float().permute(0, 2, 1, 3).reshape(N * Nkv, rep * S, D)
    k, v = (_q4_values(s[c]).reshape(N * Nkv, n, D) for c in ("k", "v"))
    p = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(s["scale"]).view(N, Nkv, rep, S, n)
    p += s["mask"].float()[:, :, None]
    p -= p.amax(-1, keepdim=True)
    p = p.exp_().view(N * Nkv, rep * S, n)
    y = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return y.view(N, Nh, S, D).transpose(1, 2).to(s["q"].dtype)


def _plain_lora(s):
    e, r, k = s["a"].shape
    h = torch.matmul(s["x"], s["a"].float().reshape(e * r, k).t().contiguous()).view(-1, e, r)
    use = (s["ids"][:, None] == torch.arange(e, device="cuda")) * s["scales"]
    b = s["b"].float().permute(0, 2, 1).reshape(e * r, -1)
    return s["y0"] + torch.matmul((h * use[:, :, None]).view(-1, e * r), b)


def _plain_logits(s):
    l = s["logits"].float()
    m, V = l.shape
    L = s["history"].shape[1]
    live = (torch.arange(L, device="cuda") < s["lengths"][:, None]).float()
    n = torch.zeros_like(l).scatter_add_(1, s["history"].long(), live)
    rep, freq, pres = (s["penalties"][:, j:j + 1] for j in range(3))
    l = torch.where(n > 0, torch.where(l > 0, l / rep, l * rep) - n * freq - pres, l) + s["bias"]
    if "allowed" in s:
        w = s["allowed"][s["state"].long().clamp(min=0)]
        bit = (w[:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        stop = (bit.reshape(m, -1)[:, :V] == 0) & (s["state"][:, None] >= 0)
        l = l.masked_fill(stop, float("-inf"))
    return l.to(s["logits"].dtype)


# --- the library's calls -------------------------------------------------------------------
_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hbd-acestep.cpp_amd")


class _Mem:
    """A torch tensor's memory, kept alive by the views over it."""

    def __init__(self, t):
        self.t, self.ptr, self.nbytes = t, t.data_ptr(), t.numel() * t.element_size()


def _kept(s):
    """The library's views of a state's tensors and its workspaces, which a program makes once."""
    kept = s.get("kept")
    if kept is None:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        from acestep_ops import ops
        from acestep_ops.device import DTensor

        names = {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16", torch.int32: "i32", torch.uint8: "u8"}
        kept = {k: DTensor(_Mem(t), t.shape, names[t.dtype]) for k, t in s.items() if torch.is_tensor(t)}
        kept["ops"] = ops
        if s["op"] == "append":
            for c in ("k_cache", "v_cache"):
                rows = kept[c].view(-1, kept[c].shape[-1])
                kept[c], kept[c + "_rows"] = ops.Q4(kept[c]), ops.Q4(rows)
        elif s["op"] == "attention":
            kept["q"] = kept["q"].permute(0, 2, 1, 3)
            kept["k"], kept["v"] = ops.Q4(kept["k"]), ops.Q4(kept["v"])
            need = ops.flash_attn_workspace(kept["q"], kept["k"], kept["v"])
            kept["ws"] = _workspace(DTensor, need)
        elif s["op"] == "lora":
            kept["ws"] = _workspace(DTensor, ops.lora_add_workspace(kept["x"], kept["a"], kept["b"]))
        s["kept"] = kept
    return kept


def _workspace(DTensor, need):
    return DTensor(_Mem(torch.empty(max(need, 256), dtype=torch.uint8, device="cuda")), (max(need, 256),), "u8")


def _own(s):
    t = _kept(s)
    ops = t["ops"]
    if s["op"] == "append":
        ops.kv_store(t["k"], t["k_cache"], t["pos0"], t["v"], t["v_cache"], t["sets"])
        ops.get_rows(t["k_cache_rows"], t["rows"], out=t["k_read"])
        ops.get_rows(t["v_cache_rows"], t["rows"], out=t["v_read"])
        return [s["k_read"], s["v_read"]]
    if s["op"] == "attention":
        ops.flash_attn_ext(t["q"], t["k"], t["v"], t["mask"], s["scale"], out=t["y"], workspace=t["ws"])
    elif s["op"] == "lora":
        ops.lora_add(t["y0"], t["x"], t["a"], t["b"], t["ids"], t["scales"], out=t["y"], workspace=t["ws"])
    else:
        ops.logits_adjust(t["logits"], history=t["history"], lengths=t["lengths"], penalties=t["penalties"],
                          bias=t["bias"], allowed=t.get("allowed"), state=t.get("state"), out=t["y"])
    return s["y"]


def run(s):
    if own:
        return _own(s)
    plain = {"append": _plain_append, "attention": _plain_attention, "lora": _plain_lora, "logits": _plain_logits}
    return plain[s["op"]](s)


# --- what a pass cannot do without ------------------------------------------------------------
def work(case):
    b = {"f32": 4, "bf16": 2, "f16": 2}
    if case["op"] == "append":
        rows = 2 * case["seqs"] * case["tokens"] * case["heads"]
        held = case["d"] // 32 * 18
        return {"bytes": rows * (case["d"] * (b[case["type"]] + b[case["read"]]) + 2 * held + 4), "flops": 4 * rows * case["d"]}
    if case["op"] == "attention":
        S, past, D = case["nq"], case["past"], case["d"]
        lens = [past] + [(past // 8 + past) / 2.0] * (case["seqs"] - 1 - case["idle"])  # drawn evenly between the two
        keys = sum(p + S for p in lens)
        pairs = sum(S * p + S * (S + 1) / 2 for p in lens)
        io = 2 * case["seqs"] * S * case["heads"] * D * b[case["type"]]
        return {"bytes": keys * case["kv_heads"] * 2 * D // 32 * 18 + io + pairs * 2, "flops": 4.0 * pairs * case["heads"] * D}
    if case["op"] == "lora":
        m, k, n, r = case["rows"], case["k"], case["n"], case["rank"]
        used = min(case["adapters"], -(-m // case["run"]))
        return {"bytes": m * (k + 2 * n) * 4 + used * r * (k + n) * 2, "flops": 2.0 * m * r * (k + n)}
    m, V = case["rows"], case["vocab"]
    grammar = V / 8 * min(m, case["states"])
    return {"bytes": 2.0 * m * V * b[case["type"]] + 4 * V + grammar + 2 * m * case["history"], "flops": 6.0 * m * V}


# --- the same in 64 bits -------------------------------------------------------------------
def _exact_rows(x):
    """The values a Q4_0 row of x stands for. What the format defines in 32 bits (1 / d, the product, the
    sum with 8.5) and in 16 bits (d as stored) is rounded there."""
    x = x.float().cpu().numpy().reshape(-1, 32)
    top = x[np.arange(len(x)), np.abs(x).argmax(1)]
    d = (top / np.float32(-8)).astype(np.float32)
    with np.errstate(divide="ignore"):
        inv = np.where(d != 0, np.float32(1) / d, np.float32(0)).astype(np.float32)
    level = np.minimum(15, np.floor((x * inv[:, None]).astype(np.float32) + np.float32(8.5)))
    return (level - 8.0) * d.astype(np.float16).astype(np.float64)[:, None]


def _exact_cache(c):
    """Q4_0 bytes (rows, D / 32 * 18) as numbers in 64 bits."""
    b = c.contiguous().view(-1, 18)
    d = b[:, :2].contiguous().view(torch.float16).double()
    low, high = (b[:, 2:] % 16).double(), torch.div(b[:, 2:], 16, rounding_mode="floor").double()
    return ((torch.cat([low, high], 1) - 8.0) * d).view(c.shape[0], -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        got = []
        for name in ("k", "v"):
            x = s[name].permute(0, 2, 1, 3).contiguous()
            got.append(torch.from_numpy(_exact_rows(x).reshape(-1, case["d"])))
        return got
    if case["op"] == "attention":
        N, S, Nh, D = s["q"].shape
        rep = Nh // case["kv_heads"]
        y = torch.empty(N, S, Nh, D, dtype=torch.float64, device="cuda")
        for i in range(N):
            bias = s["mask"][i, 0].double()
            for h in range(Nh):
                k, v = _exact_cache(s["k"][i, h // rep]), _exact_cache(s["v"][i, h // rep])
                w = s["q"][i, :, h].double() @ k.t() * s["scale"] + bias
                w = torch.exp(w - w.max(1, keepdim=True).values)
                y[i, :, h] = (w @ v) / w.sum(1, keepdim=True)
        return y
    if case["op"] == "lora":
        y = s["y0"].double()
        for j in range(case["adapters"]):
            at = torch.nonzero(s["ids"] == j)[:, 0]
            down = s["x"][at].double() @ s["a"][j].double().t()
            y[at] += float(s["scales"][j]) * (down @ s["b"][j].double().t())
        return y
    y = s["logits"].double()
    for i in range(case["rows"]):
        seen = s["history"][i, :int(s["lengths"][i])].long()
        token, count = torch.unique(seen, return_counts=True)
        rep, freq, pres = (float(v) for v in s["penalties"][i])
        l = y[i, token]
        y[i, token] = torch.where(l > 0, l / rep, l * rep) - freq * count - pres
        y[i] += s["bias"][0].double()
        if case["states"] and int(s["state"][i]) >= 0:
            word = s["allowed"][int(s["state"][i])].long()
            at = torch.arange(case["vocab"], device="cuda")
            y[i, (word[at // 32] >> (at % 32)) % 2 == 0] = float("-inf")
    return y
