"""The operators of a batched serving step, as they are measured: sizes, inputs, a plain form, a 64-bit
form and the work each cannot do without.

cache_write  per-head RMS norms and the NeoX rotation of a step's queries and keys, values normed
             without a weight, and keys and values quantised into one-byte ring caches, in one pass
cache_read   a range of positions of one sequence's quantised cache, read back as fp32
attention    a step's rows over quantised caches: each row over its own sequence's positions, and all
             rows over one shared prefix whose scores are formed once for the batch
sample       one token per row of logits: nucleus, min-p and top-k cuts, temperature, and a draw from
             a given uniform

Layer shapes are the decoder's two (16 query heads over 8 kv heads of 256 with a window of 1024, and
16 over 2 of 512 without one) and generic ones; the vocabulary is the model's 262,144 or odd.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

TINY = 2.0 ** -100          # the smallest scale a cache vector is stored with
CODE_MAX = {"int8": 127.0, "e4m3": 448.0}
CODE_TYPE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
SLIDING = dict(q_heads=16, kv_heads=8, head_dim=256, window=1024, pairs=128, theta=10000.0)
FULL = dict(q_heads=16, kv_heads=2, head_dim=512, window=0, pairs=64, theta=1000000.0)


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "turbo-winfare_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import gtmoe.kvcache
    import gtmoe.sampling
    return gtmoe


def listed():
    return [
        # one generated token of one sequence in a sliding-window layer
        dict(name="write_one_token", op="cache_write", n=1, fmt="int8", far=700, seqs=1, capacity=1024, **SLIDING),
        # a decode step of 32 sequences far into their contexts, full-attention layer (V is K's projection)
        dict(name="write_batch32_far", op="cache_write", n=32, fmt="e4m3", far=131072, seqs=32, capacity=2048, **FULL),
        # 512 consecutive prompt tokens of one sequence
        dict(name="write_prompt512", op="cache_write", n=512, fmt="int8", far=8192, seqs=1, capacity=1536, **SLIDING),
        # a sliding layer's window of one sequence, wrapped round its ring
        dict(name="read_window", op="cache_read", fmt="e4m3", first=700, count=1000, capacity=1024, kv_heads=8, head_dim=256),
        # a long sequence of a full-attention layer, all of it
        dict(name="read_long", op="cache_read", fmt="int8", first=0, count=131071, capacity=131072, kv_heads=2, head_dim=512),
        # the latency of a single stream: one row over a sliding window
        dict(name="attn_one_row", op="attention", n=1, fmt="int8", prefix=0, own_min=1024, own_max=1024, chunk=False, **SLIDING),
        # 32 sequences with long contexts of their own and no common part, ragged
        dict(name="attn_batch32_own", op="attention", n=32, fmt="e4m3", prefix=0, own_min=77, own_max=8192, chunk=False, **FULL),
        # 32 sequences behind one long common prompt, each with its own turn so far
        dict(name="attn_batch32_prefix", op="attention", n=32, fmt="int8", prefix=16384, own_min=1, own_max=1024, chunk=False, **FULL),
        # 61 sequences behind a common prompt in a sliding layer: some windows still reach into it, some not
        dict(name="attn_batch61_window", op="attention", n=61, fmt="int8", prefix=2048, own_min=1, own_max=1500, chunk=False, **SLIDING),
        # the last 512 tokens of a 32,768-token prompt: rows of one sequence, causal
        dict(name="attn_prompt512", op="attention", n=512, fmt="int8", prefix=32768, own_min=0, own_max=0, chunk=True, **FULL),
        # one sampled token of one sequence, the model's vocabulary
        dict(name="sample_one", op="sample", n=1, vocab=262144, rules="nucleus"),
        # a step of 64 sequences, each with its own settings
        dict(name="sample_batch64", op="sample", n=64, vocab=262144, rules="mixed"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _shape(rng):
    kind = rng.choice(("sliding", "full", "other"))
    if kind == "sliding":
        return dict(SLIDING)
    if kind == "full":
        return dict(FULL)
    hd = rng.choice((128, 256, 512))
    kv = rng.randint(1, 8)
    return dict(q_heads=kv * rng.randint(1, 8), kv_heads=kv, head_dim=hd, window=rng.choice((0, 0, 333, 1024)),
                pairs=rng.randint(0, hd // 2), theta=rng.choice((10000.0, 1000000.0)))


def draw(rng):
    op = rng.choice(("cache_write", "cache_read", "attention", "attention", "sample"))
    fmt = rng.choice(("int8", "e4m3"))
    if op == "cache_write":
        s = _shape(rng)
        n = _log(rng, 1, 512)
        seqs = rng.choice((1, n))
        return dict(op=op, n=n, fmt=fmt, far=_log(rng, 1000, 131072), seqs=seqs, capacity=rng.randint(600, 2000), **s)
    if op == "cache_read":
        cap = _log(rng, 2, 131072)
        return dict(op=op, fmt=fmt, first=rng.randint(0, 5000), count=_log(rng, 1, cap), capacity=cap,
                    kv_heads=rng.randint(1, 2), head_dim=rng.choice((128, 256, 512)))
    if op == "attention":
        s = _shape(rng)
        if rng.random() < 0.25:   # consecutive rows of one sequence
            n = _log(rng, 2, 512)
            return dict(op=op, n=n, fmt=fmt, prefix=n + _log(rng, 1, 16384), own_min=0, own_max=0, chunk=True, **s)
        n = _log(rng, 1, 64)
        hi = _log(rng, 2, 2048)
        return dict(op=op, n=n, fmt=fmt, prefix=rng.choice((0, _log(rng, 1, 16384))), own_min=rng.randint(1, hi), own_max=hi,
                    chunk=False, **s)
    return dict(op=op, n=_log(rng, 1, 64), vocab=_log(rng, 1000, 262144), rules=rng.choice(("nucleus", "top_k", "min_p", "mixed", "all")))


# ---- inputs -----------------------------------------------------------------------------------------

def _spread(i, n, lo, hi):
    """The i-th of n lengths spread over [lo, hi], not in order."""
    return hi if n == 1 else lo + (hi - lo) * ((i * 7919) % n) // (n - 1)


def _quantised(x, fmt):
    """Codes and scales of vectors along the last axis, as a cache holds them."""
    s = (x.abs().amax(-1).double() / CODE_MAX[fmt]).clamp_min(TINY).float()
    u = x / s[..., None]
    return (u.round().clamp(-127, 127) if fmt == "int8" else u.clamp(-448, 448)).to(CODE_TYPE[fmt]), s


def _cache(g, seqs, capacity, kv_heads, head_dim, fmt):
    """A cache as earlier steps left it: normed keys and values."""
    out = {"fmt": fmt}
    for name in ("k", "v"):
        codes = torch.empty(seqs, capacity, kv_heads, head_dim, dtype=CODE_TYPE[fmt], device="cuda")
        scales = torch.empty(seqs, capacity, kv_heads, device="cuda")
        step = max(1, (1 << 26) // (seqs * kv_heads * head_dim))
        for a in range(0, capacity, step):
            b = min(capacity, a + step)
            codes[:, a:b], scales[:, a:b] = _quantised(torch.randn(seqs, b - a, kv_heads, head_dim, generator=g, device="cuda"), fmt)
        out[name], out[name + "_scale"] = codes, scales.transpose(1, 2).contiguous()   # scales [seqs][kv_heads][capacity]
    return out


def _spans(case):
    """Each attention row's position, and its [first, end) in the shared prefix and in its own cache."""
    n, P = case["n"], case["prefix"]
    pos = [P - n + i if case["chunk"] else P + _spread(i, n, case["own_min"], case["own_max"]) - 1 for i in range(n)]
    first = [max(0, p + 1 - case["window"]) if case["window"] else 0 for p in pos]
    shared = [(min(f, P), min(P, p + 1)) for f, p in zip(first, pos)]
    mine = [(max(f, P), max(P, p + 1)) for f, p in zip(first, pos)]
    return pos, shared, mine


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7 + 3)
    s = {"case": case}
    op = case["op"]
    if op == "cache_write":
        n, hd, H, KV = case["n"], case["head_dim"], case["q_heads"], case["kv_heads"]
        s["q"] = torch.randn(n, H * hd, generator=g, device="cuda") * 1.7
        s["k"] = torch.randn(n, KV * hd, generator=g, device="cuda") * 0.6
        s["v"] = s["k"] if case["window"] == 0 else torch.randn(n, KV * hd, generator=g, device="cuda")
        s["q_w"] = (1 + 0.1 * torch.randn(hd, generator=g, device="cuda")).to(torch.bfloat16)
        s["k_w"] = (1 + 0.1 * torch.randn(hd, generator=g, device="cuda")).to(torch.bfloat16)
        s["q_out"] = torch.empty_like(s["q"])
        s["cache"] = _cache(g, case["seqs"], case["capacity"], KV, hd, case["fmt"])
        r = random.Random(seed)
        if case["seqs"] == 1:
            p0 = r.randint(0, max(0, case["far"] - n))
            pos, seq = [p0 + i for i in range(n)], [0] * n
        else:
            pos, seq = [r.randint(0, case["far"] - 1) for _ in range(n)], r.sample(range(case["seqs"]), n)
        s["positions"], s["seqs"] = np.array(pos, dtype=np.uint32), np.array(seq, dtype=np.uint32)
        s["pos_dev"], s["seq_dev"] = (torch.tensor(v, device="cuda") for v in (pos, seq))
    elif op == "cache_read":
        s["cache"] = _cache(g, 2, case["capacity"], case["kv_heads"], case["head_dim"], case["fmt"])
        s["k_out"] = torch.empty(case["count"], case["kv_heads"] * case["head_dim"], device="cuda")
        s["v_out"] = torch.empty_like(s["k_out"])
    elif op == "attention":
        n, hd, H, KV = case["n"], case["head_dim"], case["q_heads"], case["kv_heads"]
        pos, shared, mine = _spans(case)
        s["q"] = torch.randn(n, H * hd, generator=g, device="cuda") * (3.0 / math.sqrt(hd))
        s["ctx"] = torch.empty_like(s["q"])
        if case["prefix"]:
            lo = min(a for a, _ in shared)
            s["prefix"] = _cache(g, 1, max(1, case["prefix"] - lo), KV, hd, case["fmt"])
        if not case["chunk"]:
            s["cache"] = _cache(g, n, max(b - a for a, b in mine), KV, hd, case["fmt"])
        else:
            s["cache"] = s["prefix"]
        s["positions"] = np.array(pos, dtype=np.uint32)
        s["seqs"] = np.array([0] * n if case["chunk"] else list(range(n))[::-1], dtype=np.uint32)
        s["seq_dev"] = torch.tensor(s["seqs"].astype(np.int64), device="cuda")
        s["shared"], s["mine"] = (torch.tensor(v, device="cuda") for v in (shared, mine))
    else:
        n, V = case["n"], case["vocab"]
        z = torch.randn(n, V, generator=g, device="cuda") * 2.5
        peaks = torch.randint(0, V, (n, 40), generator=g, device="cuda")   # the words a context makes likely
        z.scatter_add_(1, peaks, 12 * torch.rand(n, 40, generator=g, device="cuda"))
        s["logits"] = 30 * torch.tanh(z / 30)
        s["uniforms"] = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
        r = random.Random(seed)
        rows = []
        for i in range(n):
            rule = case["rules"] if case["rules"] != "mixed" else ("greedy", "nucleus", "top_k", "min_p", "all", "plain")[i % 6]
            t = 0.0 if rule == "greedy" else round(r.uniform(0.6, 1.3), 3)
            top_p = r.choice((0.8, 0.9, 0.95)) if rule in ("nucleus", "all") else 1.0
            min_p = r.choice((0.02, 0.05, 0.1)) if rule in ("min_p", "all") else 0.0
            rows.append((t, top_p, min_p, r.choice((20, 50, 200)) if rule in ("top_k", "all") else 0))
        s["rows"] = rows
        s["t"], s["top_p"], s["min_p"] = (torch.tensor([float(np.float32(row[j])) for row in rows], dtype=torch.float64, device="cuda") for j in range(3))
        s["top_k"] = torch.tensor([row[3] if row[3] else V for row in rows], device="cuda")
    return s


# ---- the framework's calls ----------------------------------------------------------------------------

def _handle(s):
    """What a user's program builds once: the cache objects over its tensors, the attention's and the sampler's workspace."""
    if "handle" not in s:
        gtmoe, case, h = _package(), s["case"], {}
        for name in ("cache", "prefix"):
            if name in s:
                c = s[name]
                h[name] = gtmoe.kvcache.KvCache.over(c["k"], c["v"], c["k_scale"], c["v_scale"])
        if case["op"] == "attention":
            h["attention"] = gtmoe.kvcache.KvAttention(case["q_heads"], case["kv_heads"], case["head_dim"], case["n"])
        if case["op"] == "sample":
            h["sampler"] = gtmoe.sampling.RowSampler(case["vocab"], case["n"])
            h["rows"] = gtmoe.sampling.sampling_rows([gtmoe.sampling.RowParams(*row) for row in s["rows"]])
        s["handle"] = h
    return s["handle"]


def _run_own(s):
    case, h = s["case"], _handle(s)
    op = case["op"]
    if op == "cache_write":
        h["cache"].write(s["q"], s["k"], s["v"], s["q_out"], s["positions"], s["seqs"], q_w=s["q_w"], k_w=s["k_w"], eps=1e-6,
                         rotated_pairs=case["pairs"], theta=case["theta"])
        return [s["q_out"]] + [s["cache"][name] for name in ("k", "v", "k_scale", "v_scale")]
    if op == "cache_read":
        h["cache"].read(1, case["first"], case["count"], s["k_out"], s["v_out"])
        return [s["k_out"], s["v_out"]]
    if op == "attention":
        h["attention"](s["q"], h["cache"], s["seqs"], s["positions"], s["ctx"], window=case["window"], prefix=h.get("prefix"),
                       prefix_len=case["prefix"])
        return [s["ctx"]]
    r = h["sampler"](s["logits"], h["rows"], s["uniforms"])
    return [r.tokens, r.kept, r.logprobs]


# ---- the plain form -----------------------------------------------------------------------------------

def _normed(x, w, eps=1e-6):
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    return y if w is None else y * w.double()


def _rotated(y, pos, pairs, theta):
    """y [n][heads][head_dim], in 64 bits: far positions' angles need them."""
    hd = y.shape[-1]
    freq = theta ** (-2.0 * torch.arange(pairs, dtype=torch.float64, device=y.device) / hd)
    a = (pos.double()[:, None] * freq)[:, None, :]
    c, s = torch.cos(a), torch.sin(a)
    y0, y1 = y[..., :pairs], y[..., hd // 2:hd // 2 + pairs]
    return torch.cat((y0 * c - y1 * s, y[..., pairs:hd // 2], y0 * s + y1 * c, y[..., hd // 2 + pairs:]), -1)


def _store(cache, name, y, slots, seqs):
    """Quantises y [n][kv_heads][head_dim] (64 bits: values next to a rounding border) into its ring rows."""
    fmt = cache["fmt"]
    scale = (y.abs().amax(-1) / CODE_MAX[fmt]).clamp_min(TINY).float()
    u = y / scale.double()[..., None]
    if fmt == "int8":
        codes = torch.round(u).clamp(-127, 127).to(torch.int8)
    else:   # three fraction bits; steps of 2^-9 below 2^-6
        step = torch.exp2(torch.floor(torch.log2(u.abs().clamp_min(2.0 ** -6))) - 3)
        codes = (torch.round(u / step) * step).clamp(-448, 448).float().to(torch.float8_e4m3fn)
    cache[name].view(torch.int8)[seqs, slots] = codes.view(torch.int8)
    cache[name + "_scale"][seqs, :, slots] = scale


def _values(codes, scales, rows):
    """Ring rows of one sequence as fp32 [len(rows)][kv_heads][head_dim]."""
    return codes.view(torch.int8)[rows].view(codes.dtype).float() * scales[:, rows].t()[..., None]


def _span_mask(spans, t):
    return (t >= spans[:, :1]) & (t < spans[:, 1:])


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "cache_write":
        n, hd = case["n"], case["head_dim"]
        q, k, v = (s[x].double().view(n, -1, hd) for x in ("q", "k", "v"))
        s["q_out"].copy_(_rotated(_normed(q, s["q_w"]), s["pos_dev"], case["pairs"], case["theta"]).view(n, -1))
        slots = s["pos_dev"] % case["capacity"]
        _store(s["cache"], "k", _rotated(_normed(k, s["k_w"]), s["pos_dev"], case["pairs"], case["theta"]), slots, s["seq_dev"])
        _store(s["cache"], "v", _normed(v, None), slots, s["seq_dev"])
        return [s["q_out"]] + [s["cache"][name] for name in ("k", "v", "k_scale", "v_scale")]
    if op == "cache_read":
        c = s["cache"]
        rows = (torch.arange(case["count"], device="cuda") + case["first"]) % case["capacity"]
        return [_values(c[x][1], c[x + "_scale"][1], rows).view(case["count"], -1) for x in ("k", "v")]
    if op == "attention":
        n, hd, KV, P = case["n"], case["head_dim"], case["kv_heads"], case["prefix"]
        q = s["q"].view(n, KV, -1, hd)
        scores, values = [], []
        if P:
            c = s["prefix"]
            t = torch.arange(P - c["k"].shape[1], P, device="cuda")
            k, v = (_values(c[x][0], c[x + "_scale"][0], t % c["k"].shape[1]) for x in ("k", "v"))
            z = torch.einsum("nhgd,thd->nhgt", q, k)
            scores.append(z.masked_fill(~_span_mask(s["shared"], t)[:, None, None], -math.inf))
            values.append(("nhgt,thd->nhgd", v, len(t)))
        if not case["chunk"]:
            c = s["cache"]
            t = s["mine"][:, :1] + torch.arange(c["k"].shape[1], device="cuda")   # each row's own positions
            slots = t % c["k"].shape[1]
            seq = s["seq_dev"][:, None]
            k, v = (c[x].view(torch.int8)[seq, slots].view(c[x].dtype).float() * c[x + "_scale"].transpose(1, 2)[seq, slots][..., None]
                    for x in ("k", "v"))
            z = torch.einsum("nhgd,nthd->nhgt", q, k)
            scores.append(z.masked_fill(~_span_mask(s["mine"], t)[:, None, None], -math.inf))
            values.append(("nhgt,nthd->nhgd", v, t.shape[1]))
        z = torch.cat(scores, -1)
        p = torch.exp(z - z.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        out = sum(torch.einsum(rule, part, v) for (rule, v, _), part in zip(values, p.split([m for _, _, m in values], -1)))
        return [out.reshape(n, -1)]
    z = s["logits"].double()
    n, V = z.shape
    order = torch.sort(s["logits"], descending=True, stable=True).indices   # ties to the lower id
    w = torch.exp(z - z.amax(-1, keepdim=True))   # sums over the vocabulary, next to a cut or a draw: 64 bits
    total = w.sum(-1, keepdim=True)
    sorted_w = w.gather(1, order)
    before = torch.cumsum(sorted_w, -1) - sorted_w
    rank = torch.arange(V, device="cuda")
    keep = (rank < s["top_k"][:, None]) & (sorted_w >= s["min_p"][:, None])
    keep &= (before < s["top_p"][:, None] * total) | (s["top_p"][:, None] >= 1)
    keep &= (s["t"][:, None] > 0)
    keep[:, 0] = True
    kept = keep.sum(-1)
    mask = torch.zeros_like(keep).scatter_(1, order, keep)
    t = torch.where(s["t"] > 0, s["t"], 1.0)[:, None]
    mass = torch.cumsum(torch.where(mask, torch.exp((z - z.amax(-1, keepdim=True)) / t), 0.0), -1)
    tokens = torch.searchsorted(mass, s["uniforms"][:, None] * mass[:, -1:], right=True)
    logprobs = torch.log(w.gather(1, tokens) / total)
    return [tokens[:, 0].int(), kept.int(), logprobs[:, 0].float()]


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


# ---- the definition in 64 bits ------------------------------------------------------------------------

def _exact_write(s, case):
    n, hd = case["n"], case["head_dim"]
    out = []
    for name, w in (("q", s["q_w"]), ("k", s["k_w"]), ("v", None)):
        x = s[name].cpu().double().numpy().reshape(n, -1, hd)
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6)
        if w is not None:
            y = y * w.float().cpu().double().numpy()
            r = y.copy()
            for i in range(case["pairs"]):
                a = s["positions"].astype(np.float64)[:, None] * case["theta"] ** (-2.0 * i / hd)
                r[..., i] = y[..., i] * np.cos(a) - y[..., hd // 2 + i] * np.sin(a)
                r[..., hd // 2 + i] = y[..., i] * np.sin(a) + y[..., hd // 2 + i] * np.cos(a)
            y = r
        out.append(y)
    scales = []
    for name, y in (("k", out[1]), ("v", out[2])):
        c = s["cache"][name + "_scale"].double().cpu().numpy().copy()
        c[s["seqs"].astype(np.int64), :, (s["positions"] % case["capacity"]).astype(np.int64)] = \
            np.maximum(np.abs(y).max(-1) / CODE_MAX[case["fmt"]], TINY)
        scales.append(c)
    # a code has no 64-bit value of its own
    return [out[0].reshape(n, -1), None, None, scales[0], scales[1]]


def _exact_attention(s, case):
    """Row by row over its own list of positions."""
    n, hd, KV, P = case["n"], case["head_dim"], case["kv_heads"], case["prefix"]
    _, shared, mine = _spans(case)

    def values(c, name, seq, a, b):
        at = torch.arange(a, b, device="cuda") % c[name].shape[1]
        return c[name][seq].view(torch.int8)[at].view(c[name].dtype).double() * c[name + "_scale"][seq][:, at].double().t()[..., None]

    lo = min(a for a, _ in shared)
    pk, pv = (values(s["prefix"], x, 0, lo, P) for x in ("k", "v")) if P else (None, None)
    out = torch.empty(n, KV, case["q_heads"] // KV, hd, dtype=torch.float64, device="cuda")
    for i in range(n):
        k, v = [], []
        if shared[i][1] > shared[i][0]:
            k.append(pk[shared[i][0] - lo:shared[i][1] - lo])
            v.append(pv[shared[i][0] - lo:shared[i][1] - lo])
        if mine[i][1] > mine[i][0]:
            k.append(values(s["cache"], "k", int(s["seqs"][i]), *mine[i]))
            v.append(values(s["cache"], "v", int(s["seqs"][i]), *mine[i]))
        k, v = torch.cat(k).transpose(0, 1), torch.cat(v).transpose(0, 1)
        p = torch.softmax(s["q"][i].double().view(KV, -1, hd) @ k.transpose(1, 2), -1)
        out[i] = p @ v
    return [out.view(n, -1)]


def _exact_sample(s, case):
    z = s["logits"].double().cpu().numpy()
    u = s["uniforms"].cpu().numpy()
    tokens, counts, logs = [], [], []
    for i, (t, top_p, min_p, top_k) in enumerate(s["rows"]):
        t, top_p, min_p = (float(np.float32(x)) for x in (t, top_p, min_p))
        order = np.argsort(-z[i], kind="stable")
        w = np.exp(z[i] - z[i].max())
        total = math.fsum(w)
        m = len(order)
        if t <= 0:
            m = 1
        else:
            if top_p < 1:
                m = min(m, int(np.searchsorted(np.cumsum(w[order]), top_p * total, side="left")) + 1)
            m = min(m, int((w >= min_p).sum()), top_k or m)
            m = max(1, m)
        ids = np.sort(order[:m])
        mass = np.cumsum(np.exp((z[i][ids] - z[i].max()) / (t if t > 0 else 1.0)))
        token = int(ids[min(m - 1, int(np.searchsorted(mass, u[i] * mass[-1], side="right")))])
        tokens.append(token)
        counts.append(m)
        logs.append(z[i][token] - z[i].max() - math.log(total))
    return [np.array(tokens, dtype=np.int32), np.array(counts, dtype=np.int32), np.array(logs)]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "cache_write":
        return _exact_write(s, case)
    if case["op"] == "cache_read":
        c = s["cache"]
        at = np.arange(case["first"], case["first"] + case["count"]) % case["capacity"]
        return [(c[x][1].float().cpu().double().numpy()[at] * c[x + "_scale"][1].double().cpu().numpy().T[at][..., None]).reshape(len(at), -1)
                for x in ("k", "v")]
    return _exact_attention(s, case) if case["op"] == "attention" else _exact_sample(s, case)


# ---- what a pass cannot do without --------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "cache_write":
        n, hd, H, KV = case["n"], case["head_dim"], case["q_heads"], case["kv_heads"]
        inputs = H + KV * (1 if case["window"] == 0 else 2)   # V may be K's projection: read once
        return {"bytes": n * hd * (4 * inputs + 4 * H + 2 * KV) + n * KV * 8 + 4 * hd, "flops": n * hd * (9 * H + 14 * KV)}
    if op == "cache_read":
        vectors = 2 * case["count"] * case["kv_heads"]
        return {"bytes": vectors * (5 * case["head_dim"] + 4), "flops": vectors * case["head_dim"]}
    if op == "attention":
        hd, KV, H, n = case["head_dim"], case["kv_heads"], case["q_heads"], case["n"]
        _, shared, mine = _spans(case)
        ranges = [r for r in shared if r[1] > r[0]]
        positions = (max(b for _, b in ranges) - min(a for a, _ in ranges) if ranges else 0) + sum(b - a for a, b in mine)
        attended = sum(b - a for a, b in shared) + sum(b - a for a, b in mine)
        return {"bytes": positions * KV * 2 * (hd + 4) + 8 * n * H * hd, "flops": 4 * attended * H * hd}
    return {"bytes": case["n"] * (4 * case["vocab"] + 20), "flops": 4 * case["n"] * case["vocab"]}
