"""One-byte ring KV caches on the device (include/gtmoe_attention.h): writing, reading back and
attending, against plain 64-bit numpy forms.

Bars. Codes and scales: equal (both sides form them in 64 bits, where a value is within ~1e-15 of a
rounding border with a chance of ~1e-13). Queries: half an fp32 step, 2^-24 relative, plus the
64-bit forms' 1e-12. Reads: one fp32 product of an exact code, half a step. Attention, fp32 sums
against 64 bits: a score of head_dim products is summed in at most 64 dependent steps of one fp32
rounding (2^-23 of S = sum |q k|, truncated), so it is off by at most ds = 64 * 2^-23 * S; exp turns
that into a relative error of the weights, so an output is off by at most 2 (ds + 2^-20) times the
largest |v| attended, 2^-20 covering the weights' and outputs' own sums. Roundings average out over
a whole output, whose 2-norm is held to 2e-5 (eight times 2^-24 of S ~ 40).
"""
from __future__ import annotations

import os
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "turbo-winfare_b200")]

pytestmark = pytest.mark.gpu

MOST = {"int8": 127.0, "e4m3": 448.0}


# ---- plain forms --------------------------------------------------------------------------------

def e4m3_table():
    v = np.zeros(256)
    for b in range(256):
        e, m = (b >> 3) & 15, b & 7
        v[b] = (m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)) * (-1 if b & 128 else 1)
    return v


E4M3 = e4m3_table()


def code_values(codes, fmt):
    """Raw bytes to the values they stand for."""
    return codes.view(np.int8).astype(np.float64) if fmt == "int8" else E4M3[codes.view(np.uint8)]


def to_code(u, fmt):
    """The nearest code's value; ties to the even code."""
    if fmt == "int8":
        return np.clip(np.rint(u), -127, 127)
    pos = E4M3[:127]   # 0 .. 448
    a = np.minimum(np.abs(u), 448.0)
    hi = np.clip(np.searchsorted(pos, a), 1, 126)
    lo = hi - 1
    up = (a - pos[lo] > pos[hi] - a) | ((a - pos[lo] == pos[hi] - a) & (hi % 2 == 0))
    return np.copysign(np.where(up, pos[hi], pos[lo]), u)


def norm_rotate(x, w, eps, pos, pairs, theta):
    """x [n][heads][hd]; pos [n], or None for values."""
    hd = x.shape[-1]
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(eps)))
    if w is not None:
        y = y * w
    if pos is not None and pairs:
        a = pos.astype(np.float64)[:, None] * theta ** (-2.0 * np.arange(pairs) / hd)
        c, s = np.cos(a)[:, None], np.sin(a)[:, None]
        y0, y1 = y[..., :pairs].copy(), y[..., hd // 2:hd // 2 + pairs].copy()
        y[..., :pairs], y[..., hd // 2:hd // 2 + pairs] = y0 * c - y1 * s, y0 * s + y1 * c
    return y


def quantise(y, fmt):
    s = np.maximum(np.abs(y).max(-1) / MOST[fmt], 2.0 ** -100).astype(np.float32)
    return to_code(y / s.astype(np.float64)[..., None], fmt), s


def raw(t):
    import torch
    return t.view(torch.uint8).cpu().numpy()


def values(cache, which):
    """A cache's values [num_seqs][capacity][kv_heads][hd] in 64 bits."""
    codes = code_values(raw(getattr(cache, which)), cache.fmt)
    return codes * getattr(cache, which + "_scale").cpu().numpy().astype(np.float64).transpose(0, 2, 1)[..., None]


def fill(cache, seed, spread=1.0):
    """Quantised normal vectors in every ring row."""
    import torch
    g = torch.Generator().manual_seed(seed)
    shape = tuple(cache.k.shape)
    for name in ("k", "v"):
        x = torch.randn(shape, generator=g).numpy().astype(np.float64)
        if spread != 1.0:
            x *= spread ** torch.randn(shape[:3] + (1,), generator=g).numpy()
        codes, s = quantise(x, cache.fmt)
        if cache.fmt == "int8":
            b = codes.astype(np.int8).view(np.uint8)
        else:
            b = torch.from_numpy(codes).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()
        getattr(cache, name).view(torch.uint8).copy_(torch.from_numpy(b.copy()))
        getattr(cache, name + "_scale").copy_(torch.from_numpy(s.transpose(0, 2, 1).copy()))


def attend(q, cache, seqs, pos, window, prefix, pseq, plen):
    """Row by row in 64 bits: (ctx, largest allowed error of each row)."""
    n = q.shape[0]
    KV, hd = cache.kv_heads, cache.head_dim
    q = q.reshape(n, KV, -1, hd)
    own = {w: values(cache, w) for w in "kv"}
    pre = {w: values(prefix, w)[pseq] for w in "kv"} if plen else None
    ctx, tol = np.zeros(q.shape), np.zeros(n)
    for i in range(n):
        first = max(0, pos[i] + 1 - window) if window else 0
        t = np.arange(first, pos[i] + 1)
        kv = []
        for w in "kv":
            parts = []
            if plen and (t < plen).any():
                parts.append(pre[w][t[t < plen] % prefix.capacity])
            if (t >= plen).any():
                parts.append(own[w][seqs[i]][t[t >= plen] % cache.capacity])
            kv.append(np.concatenate(parts))
        k, v = kv
        s = np.einsum("hgd,thd->hgt", q[i], k)
        p = np.exp(s - s.max(-1, keepdims=True))
        ctx[i] = np.einsum("hgt,thd->hgd", p / p.sum(-1, keepdims=True), v)
        S = np.einsum("hgd,thd->hgt", np.abs(q[i]), np.abs(k)).max()
        tol[i] = 2 * (64 * 2.0 ** -23 * S + 2.0 ** -20) * np.abs(v).max()
    return ctx.reshape(n, -1), tol


def run_attention(cache, q, seqs, pos, window=0, prefix=None, pseq=0, plen=0, stream=None, op=None):
    import torch
    from gtmoe.kvcache import KvAttention
    H = q.shape[1] // cache.head_dim
    op = op or KvAttention(H, cache.kv_heads, cache.head_dim, max(1, q.shape[0]))
    ctx = torch.full((q.shape[0], q.shape[1]), 777.0, device="cuda")
    op(q, cache, seqs, pos, ctx, window=window, prefix=prefix, prefix_seq=pseq, prefix_len=plen, stream=stream)
    return ctx


def check_attention(cache, q, seqs, pos, window=0, prefix=None, pseq=0, plen=0):
    got = run_attention(cache, q, seqs, pos, window, prefix, pseq, plen).cpu().numpy().astype(np.float64)
    want, tol = attend(q.cpu().numpy().astype(np.float64), cache, seqs, pos, window, prefix, pseq, plen)
    off = np.abs(got - want).max(1)
    assert (off <= tol).all(), (off / tol).max()
    rel = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert rel <= 2e-5, rel


def queries(n, H, hd, seed=5):
    import torch
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, H * hd, generator=g) * (3.0 / hd ** 0.5)).cuda()


# ---- writing ------------------------------------------------------------------------------------

WRITES = [  # n, q_heads, kv_heads, hd, pairs, theta, positions, seqs, capacity, v is k
    (1, 16, 8, 256, 128, 1e4, [0], [0], 4, False),
    (1, 16, 2, 512, 64, 1e6, [131071], [2], 100, True),
    (7, 3, 3, 128, 64, 1e4, [5, 6, 7, 8, 9, 10, 11], [1] * 7, 9, False),
    (33, 21, 7, 512, 0, 1e4, list(range(0, 330, 10)), [i % 3 for i in range(33)], 400, False),
    (64, 8, 1, 256, 7, 1e6, list(range(1000000, 1000064)), [0] * 64, 64, False),
    (512, 4, 2, 128, 33, 5e5, list(range(3000, 3512)), [0] * 512, 600, True),
]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("case", WRITES)
def test_write(case, fmt):
    import torch
    from gtmoe.kvcache import KvCache
    n, H, KV, hd, pairs, theta, pos, seqs, cap, shared = case
    g = torch.Generator().manual_seed(n)
    q, k, v = (torch.randn(n, heads * hd, generator=g) * m for heads, m in ((H, 2.0), (KV, 0.3), (KV, 30.0)))
    v = k if shared else v
    q_w, k_w = ((1 + 0.2 * torch.randn(hd, generator=g)).to(torch.bfloat16) for _ in range(2))
    cache = KvCache(3, cap, KV, hd, fmt)
    fill(cache, 1)
    before = {x: raw(getattr(cache, x)).copy() for x in ("k", "v", "k_scale", "v_scale")}
    out = torch.zeros(n, H * hd, device="cuda")
    kd = k.cuda()
    cache.write(q.cuda(), kd, kd if shared else v.cuda(), out, pos, seqs, q_w=q_w.cuda(), k_w=k_w.cuda(), eps=1e-6,
                rotated_pairs=pairs, theta=theta)
    p = np.array(pos)
    want = norm_rotate(q.double().numpy().reshape(n, H, hd), q_w.double().numpy(), 1e-6, p, pairs, theta).reshape(n, -1)
    got = out.cpu().double().numpy()
    assert (np.abs(got - want) <= 2.0 ** -24 * np.abs(want) + 1e-12).all()
    slots = p % cap
    for name, x, w, ps in (("k", k, k_w.double().numpy(), p), ("v", v, None, None)):
        y = norm_rotate(x.double().numpy().reshape(n, KV, hd), w, 1e-6, ps, pairs, theta)
        codes, s = quantise(y, fmt)
        r, rs = raw(getattr(cache, name)), getattr(cache, name + "_scale").cpu().numpy()
        assert np.array_equal(rs[seqs, :, slots], s)
        assert np.array_equal(code_values(r[seqs, slots], fmt), codes)
        # every other ring row stays as it was
        r[seqs, slots] = before[name][seqs, slots]
        assert np.array_equal(r, before[name])
        rs[seqs, :, slots] = before[name + "_scale"].view(np.float32).reshape(rs.shape)[seqs, :, slots]
        assert np.array_equal(rs, before[name + "_scale"].view(np.float32).reshape(rs.shape))


def test_write_strided_unaligned_and_in_place():
    import torch
    from gtmoe.kvcache import KvCache
    n, H, KV, hd = 5, 4, 2, 128
    g = torch.Generator().manual_seed(2)
    flat = torch.randn(n * 1100 + 3, generator=g).cuda()
    rows = flat[1:1 + n * 1100].view(n, 1100)          # one packed projection, 4-byte aligned
    q, k, v = rows[:, :512], rows[:, 512:768], rows[:, 768:1024]
    pos, seqs = [9, 8, 7, 6, 5], [0, 0, 1, 1, 0]
    a, b = KvCache(2, 16, KV, hd), KvCache(2, 16, KV, hd)
    oa = torch.zeros(n, H * hd, device="cuda")
    a.write(q, k, v, oa, pos, seqs, rotated_pairs=64)
    ob = q.contiguous()
    b.write(ob, k.contiguous(), v.contiguous(), ob, pos, seqs, rotated_pairs=64)
    assert torch.equal(oa, ob)
    for x in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(a, x), getattr(b, x))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_write_zeros_ties_and_nonfinite(fmt):
    import torch
    from gtmoe.kvcache import KvCache
    hd, cap = 128, 8
    c = KvCache(1, cap, 1, hd, fmt)
    x = torch.zeros(4, hd)
    x[1, 3] = float("nan")
    x[2, 100] = float("-inf")
    x[3] = torch.arange(hd) - 64.0   # every half step and both ends
    v = x.clone()
    out = torch.zeros(4, hd, device="cuda")
    c.write(torch.ones(4, hd).cuda(), x.cuda(), v.cuda(), out, [0, 1, 2, 3], [0] * 4, eps=1.0)
    k, kv = c.read(0, 0, 4)
    for got in (k.cpu().numpy(), kv.cpu().numpy()):
        assert (got[0] == 0).all() and np.isnan(got[1]).all() and np.isnan(got[2]).all()
        y = norm_rotate(x[3].double().numpy()[None, None], None, 1.0, None, 0, 1e4)[0, 0]
        codes, s = quantise(y, fmt)
        assert np.array_equal(got[3], (codes * s).astype(np.float32))
    assert c.k_scale[0, 0, 0].item() == 2.0 ** -100 and not raw(c.k)[0, 1:3].any()


# ---- reading ------------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("hd,KV,cap,first,count", [(128, 1, 1, 0, 1), (256, 3, 37, 30, 37), (512, 2, 1000, 4294967000, 296),
                                                   (128, 5, 64, 63, 2)])
def test_read(fmt, hd, KV, cap, first, count):
    import torch
    from gtmoe.kvcache import KvCache
    c = KvCache(2, cap, KV, hd, fmt)
    fill(c, 3)
    k, v = c.read(1, first, count)
    at = np.arange(first, first + count) % cap
    for got, name in ((k, "k"), (v, "v")):
        want = values(c, name)[1][at].reshape(count, -1)
        assert np.array_equal(got.cpu().numpy(), want.astype(np.float32))   # one product, rounded once
    only = torch.full_like(v, 5.0)
    assert c.read(1, first, count, None, only)[0] is None and torch.equal(only, v)
    only = torch.full_like(k, 5.0)
    c.read(1, first, count, only, None)
    assert torch.equal(only, k)


# ---- attention ----------------------------------------------------------------------------------

ATTENDS = [  # n, q_heads, kv_heads, hd, window, prefix, prefix capacity, own lengths
    (1, 16, 8, 256, 0, 0, 0, [1]),
    (1, 16, 2, 512, 0, 0, 0, [1000]),
    (3, 4, 4, 128, 0, 0, 0, [1, 2, 129]),
    (5, 21, 7, 256, 50, 0, 0, [1, 49, 50, 51, 333]),
    (2, 24, 3, 512, 0, 1, 1, [1, 70]),
    (9, 16, 2, 512, 0, 700, 700, [1, 2, 3, 63, 64, 65, 127, 128, 400]),
    (40, 16, 8, 256, 100, 300, 200, list(range(1, 121, 3))),
    (33, 8, 1, 128, 0, 1025, 2000, [5] * 33),
    (70, 6, 3, 256, 0, 130, 130, [(i * 37) % 90 + 1 for i in range(70)]),
    (64, 16, 2, 512, 64, 4000, 64, [1 + i for i in range(64)]),
    (20, 5, 1, 512, 0, 257, 257, [3] * 20),
]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("case", ATTENDS)
def test_attention(case, fmt):
    from gtmoe.kvcache import KvCache
    n, H, KV, hd, window, P, pcap, lens = case
    cap = max(min(m, window) if window else m for m in lens) + 3
    cache = KvCache(n, cap, KV, hd, fmt)
    fill(cache, 11)
    prefix = None
    if P:
        prefix = KvCache(2, pcap, KV, hd, fmt)
        fill(prefix, 12)
    seqs = [(i * 7 + 3) % n if n % 7 else i for i in range(n)]
    check_attention(cache, queries(n, H, hd), seqs, [P + m - 1 for m in lens], window, prefix, 1, P)


# Prefixes long enough, over the rows together, to be computed once for all (98,304 positions x kv heads)
SHARED = [  # as above
    (3, 8, 8, 128, 0, 5000, 5000, [1, 2, 3]),
    (2, 8, 8, 128, 0, 7000, 7000, [1, 2]),
    (40, 16, 8, 256, 0, 400, 400, list(range(1, 121, 3))),
    (64, 16, 2, 512, 0, 1000, 1000, [1 + (i * 5) % 70 for i in range(64)]),
    (33, 8, 1, 128, 0, 3100, 4000, [5] * 33),                           # ring larger than the prefix
    (37, 14, 2, 256, 0, 1400, 1400, [1] * 37),                          # groups of 7 across units of 64
    (64, 8, 4, 256, 700, 4000, 900, [1 + i for i in range(64)]),        # a wrapped ring, spans that move
    (64, 4, 4, 128, 700, 4096, 768, [1 + i for i in range(64)]),        # a ring of whole tiles
    (200, 16, 8, 128, 300, 2000, 2000, [1 + 3 * i for i in range(200)]),  # half of the rows past the prefix
    (512, 3, 3, 512, 0, 65, 65, [2] * 512),
    (100, 8, 8, 128, 0, 129, 129, [1] * 100),
]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("case", SHARED)
def test_attention_over_a_prefix_computed_once(case, fmt):
    test_attention(case, fmt)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("n,H,KV,hd,start,window", [(300, 16, 2, 512, 200, 0), (400, 8, 2, 256, 1000, 333), (2, 16, 8, 256, 0, 0), (130, 16, 2, 512, 77, 0), (200, 6, 2, 128, 1000, 333),
                                                    (300, 8, 4, 256, 3, 17), (512, 2, 1, 128, 0, 0)])
def test_attention_causal_rows_of_one_sequence(fmt, n, H, KV, hd, start, window):
    from gtmoe.kvcache import KvCache
    cap = start + n if not window else min(start + n, window + n + 5)
    cache = KvCache(2, cap, KV, hd, fmt)
    fill(cache, 21)
    check_attention(cache, queries(n, H, hd), [1] * n, list(range(start, start + n)), window, cache, 1, start + n)


def test_attention_rows_inside_a_prefix_and_beyond():
    from gtmoe.kvcache import KvCache
    cache, prefix = KvCache(4, 40, 2, 256), KvCache(1, 90, 2, 256)
    fill(cache, 31)
    fill(prefix, 32)
    check_attention(cache, queries(4, 16, 256), [0, 1, 2, 3], [0, 44, 89, 129], 0, prefix, 0, 90)


@pytest.mark.parametrize("fmt,hd,H,KV,rise", [("int8", 128, 8, 1, 1.0), ("int8", 128, 8, 1, 2.0), ("e4m3", 256, 8, 1, 2.0), ("int8", 512, 8, 1, 2.0)])
def test_attention_over_a_prefix_of_many_tiles(fmt, hd, H, KV, rise):
    """More tiles for a CTA than are summed in one go; with `rise` the later keys' scores pass all before them."""
    from gtmoe.kvcache import KvCache
    n, P = 512, 8000
    cache, prefix = KvCache(n, 2, KV, hd, fmt), KvCache(1, P, KV, hd, fmt)
    fill(cache, 21)
    fill(prefix, 22)
    prefix.k_scale[..., P // 2:] *= rise
    q, some = queries(n, H, hd), list(range(0, n, 37))
    got = run_attention(cache, q, list(range(n)), [P] * n, 0, prefix, 0, P).cpu().numpy().astype(np.float64)[some]
    want, tol = attend(q.cpu().numpy().astype(np.float64)[some], cache, some, [P] * len(some), 0, prefix, 0, P)
    assert (np.abs(got - want).max(1) <= tol).all()
    assert np.linalg.norm(got - want) <= 2e-5 * rise * np.linalg.norm(want)   # as above, of S ~ 40 rise


@pytest.mark.parametrize("spread", [1e3, 1e-3])
def test_attention_uneven_scales(spread):
    # vectors whose scales differ by many powers of ten: the weighted sum keeps the large ones' precision
    from gtmoe.kvcache import KvCache
    cache = KvCache(2, 200, 2, 128)
    fill(cache, 41)
    f = np.float32(spread) ** np.random.default_rng(1).uniform(-2, 2, tuple(cache.v_scale.shape)).astype(np.float32)
    import torch
    cache.v_scale.mul_(torch.from_numpy(f).cuda())
    check_attention(cache, queries(2, 8, 128), [1, 0], [199, 100])
    for n in (30, 400):   # row by row, and once for all
        check_attention(cache, queries(n, 8, 128), [0] * n, [150] * n, 0, cache, 1, 151)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("many", [1, 40, 400])
def test_masked_rows_of_a_cache_do_not_matter(fmt, many):
    import torch
    from gtmoe.kvcache import KvCache
    P, cap = 100, 64
    cache, prefix = KvCache(2, cap, 4, 256, fmt), KvCache(1, 128, 4, 256, fmt)
    fill(cache, 51)
    fill(prefix, 52)
    pos = [P + 20] * many
    q = queries(many, 16, 256)
    seqs = [1] * many
    clean = run_attention(cache, q, seqs, pos, 90, prefix, 0, P)
    # everything outside [pos + 1 - window, pos]: NaN and infinite scales, codes of all ones
    first = P + 20 + 1 - 90
    for c, lo, hi, s in ((prefix, first, P, 0), (cache, P, P + 21, 1)):
        live = np.zeros(c.capacity, bool)
        live[np.arange(lo, hi) % c.capacity] = True
        dead = torch.from_numpy(~live).cuda()
        for x in ("k", "v"):
            getattr(c, x).view(torch.uint8)[s][dead] = 0x7F
            sc = getattr(c, x + "_scale")[s]
            sc[:, dead] = float("nan") if x == "k" else float("inf")
    assert torch.equal(run_attention(cache, q, seqs, pos, 90, prefix, 0, P), clean)


@pytest.mark.parametrize("repeat", [1, 45])
@pytest.mark.parametrize("which", ["k", "v"])
def test_nan_vectors_reach_the_rows_that_attend_them_only(repeat, which):
    import torch
    from gtmoe.kvcache import KvCache
    cache = KvCache(1, 64, 8, 128)
    fill(cache, 61)
    n = 11 * repeat
    q = queries(n, 16, 128)
    pos = sorted(list(range(20, 31)) * repeat)
    clean = run_attention(cache, q, [0] * n, pos, 0, cache, 0, 64).view(n, 16, 128)
    getattr(cache, which + "_scale")[0, 1, 25] = float("nan")   # kv head 1 (query heads 2 and 3), position 25
    got = run_attention(cache, q, [0] * n, pos, 0, cache, 0, 64).view(n, 16, 128)
    others = [h for h in range(16) if h not in (2, 3)]
    assert torch.equal(got[:, others], clean[:, others]) and torch.equal(got[:5 * repeat], clean[:5 * repeat])
    assert torch.isnan(got[5 * repeat:, 2:4]).all()


def test_rows_behind_the_last_stay_and_repeats_are_equal():
    import torch
    from gtmoe.kvcache import KvAttention, KvCache
    cache = KvCache(4, 300, 2, 512)
    fill(cache, 71)
    op = KvAttention(16, 2, 512, 8)
    ctx = torch.full((8, 16 * 512), 3.5, device="cuda")
    q = queries(8, 16, 512)
    op(q[:3], cache, [2, 2, 0], [299, 299, 10], ctx[:3], prefix=cache, prefix_seq=1, prefix_len=5)
    assert (ctx[3:] == 3.5).all()
    again = torch.empty_like(ctx[:3])
    op(q[:3], cache, [2, 2, 0], [299, 299, 10], again, prefix=cache, prefix_seq=1, prefix_len=5)
    assert torch.equal(again, ctx[:3])


@pytest.mark.parametrize("n", [6, 300])
def test_streams_and_graphs(n):
    import torch
    from gtmoe.kvcache import KvAttention, KvCache
    cache = KvCache(2, 400, 2, 256)
    fill(cache, 81)
    H = 8
    q, kv = queries(n, H, 256, 1), queries(n, 4, 256, 2)
    k, v = kv[:, :512].contiguous(), kv[:, 512:].contiguous()
    pos, seqs = list(range(40, 40 + n)), [1] * n
    op = KvAttention(H, 2, 256, n)
    qo, ctx = torch.empty_like(q), torch.empty_like(q)

    def step(stream=None):
        cache.write(q, k, v, qo, pos, seqs, rotated_pairs=128, stream=stream)
        op(qo, cache, seqs, pos, ctx, prefix=cache, prefix_seq=1, prefix_len=40 + n, stream=stream)

    step()
    want = ctx.clone()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    ctx.zero_()
    s.wait_stream(torch.cuda.current_stream())
    step(s)
    s.synchronize()
    assert torch.equal(ctx, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    q2 = q.flip(0).contiguous()
    q.copy_(q2)
    g.replay()
    torch.cuda.synchronize()
    got = ctx.clone()
    step()
    assert torch.equal(got, ctx) and not torch.equal(got, want)


def test_a_cache_beyond_4_gib():
    import torch
    from gtmoe.kvcache import KvCache
    cap, seqs = 131072, 34   # 131072 * 1024 bytes a sequence: the last starts at 4.4e9
    c = KvCache(seqs, cap, 2, 512)
    n = 64
    g = torch.Generator().manual_seed(9)
    k, q = torch.randn(n, 1024, generator=g).cuda(), torch.randn(n, 8 * 512, generator=g).cuda()
    qo = torch.empty_like(q)
    pos = list(range(cap - 32, cap + 32))
    c.write(q, k, k, qo, pos, [seqs - 1] * n, rotated_pairs=64, theta=1e6)
    got, _ = c.read(seqs - 1, cap - 32, n)
    small = KvCache(1, 64, 2, 512)
    small.write(q, k, k, qo, pos, [0] * n, rotated_pairs=64, theta=1e6)
    want, _ = small.read(0, cap - 32, n)
    assert torch.equal(got, want) and (c.k[:seqs - 1] == 0).all()
    a = run_attention(c, qo[:2] * 0.1, [seqs - 1] * 2, pos[-2:], 60)
    b = run_attention(small, qo[:2] * 0.1, [0] * 2, pos[-2:], 60)
    assert torch.equal(a, b)


def test_a_step_of_write_read_and_attend_together():
    """Three sequences behind one prompt, written token by token, against fp32 attention in numpy on
    the values that the cache holds."""
    import torch
    from gtmoe.kvcache import KvAttention, KvCache
    H, KV, hd, P, n = 16, 8, 256, 37, 3
    prefix, cache = KvCache(1, P, KV, hd), KvCache(n, 20, KV, hd)
    op = KvAttention(H, KV, hd, P)
    g = torch.Generator().manual_seed(4)

    def rows(m):
        return [(torch.randn(m, heads * hd, generator=g)).cuda() for heads in (H, KV, KV)]

    q, k, v = rows(P)
    qo, ctx = torch.empty_like(q), torch.empty_like(q)
    prefix.write(q, k, v, qo, range(P), [0] * P, rotated_pairs=128)
    qo *= 0.2
    op(qo, prefix, [0] * P, range(P), ctx, prefix=prefix, prefix_len=P)
    want, tol = attend(qo.cpu().double().numpy(), prefix, [0] * P, list(range(P)), 0, prefix, 0, P)
    assert (np.abs(ctx.cpu().numpy() - want).max(1) <= tol).all()
    for step in range(10):
        q, k, v = rows(n)
        qo, ctx = torch.empty_like(q), torch.empty_like(q)
        pos = [P + step] * n
        cache.write(q, k, v, qo, pos, [2, 0, 1], rotated_pairs=128)
        qo *= 0.2
        op(qo, cache, [2, 0, 1], pos, ctx, window=30, prefix=prefix, prefix_len=P)
    want, tol = attend(qo.cpu().double().numpy(), cache, [2, 0, 1], pos, 30, prefix, 0, P)
    assert (np.abs(ctx.cpu().numpy() - want).max(1) <= tol).all()
    kr, _ = cache.read(2, P, 10)
    assert np.array_equal(kr.cpu().numpy(), values(cache, "k")[2][np.arange(P, P + 10) % 20].reshape(10, -1).astype(np.float32))


def test_host_tensors_are_refused():
    """Before any launch: a kernel is never given a host pointer."""
    import torch
    import gtmoe
    from gtmoe.kvcache import KvAttention, KvCache
    from gtmoe.sampling import RowParams, RowSampler
    c, q = KvCache(1, 4, 1, 128, device="cpu"), torch.zeros(1, 128)
    for call in (lambda: c.write(q, q, q, q, [0], [0]), lambda: c.read(0, 0, 1),
                 lambda: KvAttention(1, 1, 128, 1, device="cpu")(q, c, [0], [0], torch.zeros(1, 128)),
                 lambda: RowSampler(4, 1, device="cpu")(torch.zeros(1, 4), [RowParams()])):
        with pytest.raises(gtmoe.GtmError, match="not on a GPU"):
            call()


def test_two_calls_at_once_on_two_streams():
    """Each with its own workspace, over one cache and prefix: the results of the calls one by one."""
    import torch
    from gtmoe.kvcache import KvAttention, KvCache
    torch.manual_seed(9)
    n, H, KV, hd, P = 24, 8, 2, 256, 4096
    pre, own = KvCache(1, P, KV, hd), KvCache(n, 64, KV, hd)
    for c in (pre, own):
        for t in (c.k, c.v):
            t.copy_(torch.randint(-127, 128, t.shape, device="cuda", dtype=torch.int8))
        for t in (c.k_scale, c.v_scale):
            t.copy_(torch.rand_like(t) * 0.01 + 0.001)
    q = [torch.randn(n, H * hd, device="cuda") * 0.1 for _ in range(2)]
    pos = [P + i for i in range(n)]
    ops = [KvAttention(H, KV, hd, n) for _ in range(2)]
    want = [torch.empty_like(x) for x in q]
    for x, w in zip(q, want):
        ops[0](x, own, list(range(n)), pos, w, prefix=pre, prefix_len=P)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [torch.zeros_like(x) for x in q]
    torch.cuda.synchronize()
    for _ in range(8):
        for i in range(2):
            ops[i](q[i], own, list(range(n)), pos, got[i], prefix=pre, prefix_len=P, stream=streams[i])
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.parametrize("prefix", [False, True])
def test_a_query_of_nan_spoils_its_own_row_only(prefix):
    import torch
    from gtmoe.kvcache import KvAttention, KvCache
    torch.manual_seed(11)
    n, H, KV, hd, P = 20, 8, 2, 256, 4096
    pre, own = KvCache(1, P, KV, hd), KvCache(n, 300, KV, hd)
    for c in (pre, own):
        for t in (c.k, c.v):
            t.copy_(torch.randint(-127, 128, t.shape, device="cuda", dtype=torch.int8))
        for t in (c.k_scale, c.v_scale):
            t.fill_(0.004)
    q = torch.randn(n, H * hd, device="cuda") * 0.1
    kw = dict(prefix=pre, prefix_len=P) if prefix else {}
    pos = [(P if prefix else 0) + 10 * i for i in range(n)]
    op, want, got = KvAttention(H, KV, hd, n), torch.empty_like(q), torch.empty_like(q)
    op(q, own, list(range(n)), pos, want, **kw)
    q[7, 2 * hd + 5] = float("nan")
    op(q, own, list(range(n)), pos, got, **kw)
    want, got = (t.view(n, H, hd) for t in (want, got))
    assert got[7, 2].isnan().all()
    got[7, 2] = want[7, 2]
    # the stabilisers of the heads beside it may move by other steps: a few roundings of fp32 sums
    assert float((got - want).abs().max()) <= 1e-5 * float(want.abs().max())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("hd", [128, 256, 512])
def test_a_shared_prefix_whose_scores_rise_with_every_tile(hd, fmt):
    """Each tile of 128 keys scores 9 more (base 2) than the one before, so that the sums so far are rescaled at
    every tile of a CTA's run, while the products of the next wait: equal bits in every repeat, and the formula's
    values. A key has one value only, so a row's scores are q[0] * k[0], S the largest of them."""
    import torch
    from gtmoe.kvcache import KvAttention, KvCache
    n, H, P = 512, 8, 3000
    cache, prefix = KvCache(n, 2, 1, hd, fmt), KvCache(1, P, 1, hd, fmt)
    fill(cache, 91)
    fill(prefix, 92)
    for c in (cache, prefix):
        c.k.view(torch.uint8).zero_()
        c.k.view(torch.uint8)[..., 0] = 1 if fmt == "int8" else 0x38   # 1.0
    step = 9 * np.log(2.0)
    t = torch.arange(P, device="cuda")
    prefix.k_scale[0, 0] = ((t // 128) * step + (t % 128) * (step / 256) + 1e-3).float()
    cache.k_scale.fill_(float(P // 128 * step))
    q = queries(n, H, hd)
    q.view(n, H, hd)[..., 0] = torch.linspace(1.0, 1.05, n * H, device="cuda").view(n, H)
    some, pos = list(range(0, n, 37)), [P] * n
    want, tol = attend(q.cpu().numpy().astype(np.float64)[some], cache, some, [P] * len(some), 0, prefix, 0, P)
    op, first = KvAttention(H, 1, hd, n), None
    for _ in range(30):
        got = run_attention(cache, q, list(range(n)), pos, 0, prefix, 0, P, op=op)
        first = got if first is None else first
        assert torch.equal(got, first)
    off = np.abs(first.cpu().numpy().astype(np.float64)[some] - want).max(1)
    assert (off <= tol).all(), (off / tol).max()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("hd,shared", [(128, False), (512, False), (128, True), (512, True)])
def test_a_long_tail_of_small_weights_counts(hd, shared, fmt):
    """One key 18.4 ahead of thousands of others, whose weights of 10^-8 each (2^-26.5 of the largest) together make
    the second half of the output's dims: the first key's value is 0 there. Relative to that tail a result is off
    by 2 (ds + 2^-20), as above, with S = 18.4: 2.9e-4; and by the rounding of the weights, which are all alike: a weight
    p is held in two fp16 limbs, hi + lo, so within half of fp16's smallest step, 2^-25, where the largest is
    at least 2^15.9 / 2^8 (over a shared prefix: the stabiliser stays while weights grow by up to 2^8) or 2^15.9. The
    tail's are e^-18.4 of that: 1.2e-2 of them, or 4.8e-5."""
    import torch
    from gtmoe.kvcache import KvCache
    n, H, KV, T = (512, 8, 1, 8192) if shared else (64, 8, 8, 4096)
    c = KvCache(1, T, KV, hd, fmt)
    one, top = (1, 127) if fmt == "int8" else (0x38, 0x7E)   # 1.0, and the largest code
    k, v = c.k.view(torch.uint8), c.v.view(torch.uint8)
    k[:, 0, :, 0] = one
    v[:, 0, :, :hd // 2] = top
    v[:, 1:, :, hd // 2:] = top
    c.k_scale.fill_(18.4)
    c.v_scale.fill_(0.01)
    q = torch.zeros(n, H, hd, device="cuda")
    q[..., 0] = 1.0
    q, pos, some = q.view(n, -1), [T - 1 - i % 7 for i in range(n)], [0, 1, n - 1]
    kw = dict(prefix=c, pseq=0, plen=T) if shared else {}
    got = run_attention(c, q, [0] * n, pos, **kw).cpu().numpy().astype(np.float64)[some]
    want, _ = attend(q.cpu().numpy().astype(np.float64)[some], c, [0] * 3, [pos[i] for i in some], 0, c, 0, T if shared else 0)
    got, want = (x.reshape(3, H, hd)[..., hd // 2:] for x in (got, want))
    off = float(np.abs(got / want - 1).max())
    held = 2.0 ** -25 / (2.0 ** (7.9 if shared else 15.9) * np.exp(-18.4))
    assert (want > 0).all() and off <= 2 * (64 * 2.0 ** -23 * 18.4 + 2.0 ** -20) + held, off


@pytest.mark.parametrize("many", [1, 40, 400])
def test_values_of_zero_beside_others(many):
    """Vectors of zeros have the least scale, 2^-100: their weights still count in the softmax's sum."""
    from gtmoe.kvcache import KvCache
    cache, prefix = KvCache(1, 40, 2, 128), KvCache(1, 2000, 2, 128)
    fill(cache, 95)
    fill(prefix, 96)
    prefix.v.zero_()
    prefix.v_scale.fill_(2.0 ** -100)
    check_attention(cache, queries(many, 8, 128), [0] * many, [2000 + i % 40 for i in range(many)], 0, prefix, 0, 2000)


@pytest.mark.parametrize("fmt,hd,H,KV", [("int8", 256, 16, 8), ("e4m3", 512, 16, 2), ("int8", 128, 8, 2)])
def test_a_wait_over_the_prefix_runs_out_then_workspace_recovers(fmt, hd, H, KV):
    """gtm_attention_kv_test_wait: a wait of 2 ms that nothing ends. The call returns, check() reports it once, the rows
    that attend the prefix are NaN, those past it are right, and the same workspace then gives what it gave before."""
    import time

    import gtmoe
    import torch
    from gtmoe.kvcache import KvAttention, KvCache
    n, P, window = 64, 6000, 5000
    cache, prefix = KvCache(n, window, KV, hd, fmt), KvCache(1, P, KV, hd, fmt)
    for c in (cache, prefix):
        c.k.view(torch.uint8).random_(0, 120)
        c.v.view(torch.uint8).random_(0, 120)
        c.k_scale.uniform_(1e-4, 2e-4)
        c.v_scale.uniform_(1e-4, 2e-4)
    op, q, seqs = KvAttention(H, KV, hd, n), queries(n, H, hd), list(range(n))
    pos = [P + (10 + i if i % 4 else window + i) for i in range(n)]   # every fourth window is past the prefix
    kw = dict(window=window, prefix=prefix, plen=P, op=op)
    want = run_attention(cache, q, seqs, pos, **kw)
    op.check()
    assert torch.isfinite(want).all()
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    gtmoe.check(gtmoe.lib().gtm_attention_kv_test_wait())
    got = run_attention(cache, q, seqs, pos, **kw)
    with pytest.raises(gtmoe.GtmError, match="timed out") as e:
        op.check()
    assert e.value.status == gtmoe.ERR_TIMEOUT and time.perf_counter() - t0 < 1.0
    op.check()   # the failing check cleared the error word
    assert torch.isnan(got[[i for i in range(n) if i % 4]]).all() and torch.equal(got[::4], want[::4])
    assert torch.equal(run_attention(cache, q, seqs, pos, **kw), want)
    op.check()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("hd,many", [(128, 1), (128, 64), (512, 64)])
@pytest.mark.parametrize("q_top", [2.0 ** 99, 1.0, 2.0 ** -10])
def test_scores_at_their_bound(hd, many, q_top, fmt):
    """sum |q_d k_d| up to 2^20, with value scales of all sizes: a head whose best key's part of the result is e^30 times
    the next one's (nine in ten of them here) gives that key's value, to 2^-20 (the weight's two limbs and the last
    division); all are finite."""
    import torch
    from gtmoe.kvcache import KvCache
    P, KV, H = 1600, 1, 8
    prefix, cache = KvCache(1, P, KV, hd, fmt), KvCache(1, 1, KV, hd, fmt)
    fill(prefix, 97)
    fill(cache, 98)
    prefix.v_scale.mul_(torch.exp2(torch.linspace(-40, 20, P))[torch.randperm(P, generator=torch.Generator().manual_seed(1))].cuda())
    q = queries(many, H, hd)
    q *= q_top * 0.999 / q.abs().max()
    qs = q.cpu().numpy().astype(np.float64).reshape(-1, hd)
    keys = np.concatenate([values(c, "k")[0] for c in (prefix, cache)])[:, 0]
    scale = 2.0 ** 19.99 / (np.abs(qs) @ np.abs(keys).T).max()
    for c in (prefix, cache):
        c.k_scale.mul_(scale)
    got = run_attention(cache, q, [0] * many, [P] * many, 0, prefix, 0, P).cpu().numpy().astype(np.float64).reshape(-1, hd)
    keys, vals = (np.concatenate([values(c, w)[0] for c in (prefix, cache)])[:, 0] for w in "kv")
    parts = qs @ keys.T + np.log(np.concatenate([c.v_scale[0, 0].cpu().numpy() for c in (prefix, cache)]).astype(np.float64))
    best, two = (qs @ keys.T).argmax(1), np.sort(parts, 1)[:, -2:]
    clear = (two[:, 1] - two[:, 0] >= 30) & (parts.argmax(1) == best)
    assert clear.mean() >= 0.9 and np.isfinite(got).all()
    want = vals[best][clear]
    assert (np.abs(got[clear] - want).max(1) <= 2.0 ** -20 * np.abs(want).max(1)).all()


@pytest.mark.parametrize("n,H,KV,hd", [(1, 16, 8, 256), (300, 21, 3, 128), (512, 16, 2, 512)])
def test_write_in_place_over_many_heads(n, H, KV, hd):
    """q_out is q, a warp taking several heads of a row in turn: the bits of the call with an output of its own."""
    import torch
    from gtmoe.kvcache import KvCache
    g = torch.Generator(device="cuda").manual_seed(n)
    q, k = (torch.randn(n, heads * hd, generator=g, device="cuda") for heads in (H, KV))
    a, b = KvCache(1, n, KV, hd), KvCache(1, n, KV, hd)
    own = torch.empty_like(q)
    a.write(q, k, k, own, range(n), [0] * n, rotated_pairs=hd // 2)
    b.write(q, k, k, q, range(n), [0] * n, rotated_pairs=hd // 2)
    assert torch.equal(q, own)
    for x in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(a, x), getattr(b, x))


@pytest.mark.parametrize("n,P,own", [(1, 0, 40), (1, 0, 3000), (40, 3000, 50), (3, 20, 300)])
def test_attention_in_place(n, P, own):
    """ctx is q: one run a row, several, and a shared prefix, each with the bits of the call with two buffers."""
    from gtmoe.kvcache import KvAttention, KvCache
    cache, prefix = KvCache(n, own, 2, 256), KvCache(1, max(1, P), 2, 256)
    fill(cache, 99)
    fill(prefix, 100)
    q, pos = queries(n, 16, 256), [P + own - 1 - i % own for i in range(n)]
    want = run_attention(cache, q, range(n), pos, 0, prefix, 0, P)
    KvAttention(16, 2, 256, n)(q, cache, range(n), pos, q, prefix=prefix, prefix_len=P)
    import torch
    assert torch.equal(q, want)


def test_read_on_another_stream_leaves_what_is_queued_alone():
    """Outputs allocated for another stream must not be memory that the current stream has given up and still reads."""
    import torch
    from gtmoe.kvcache import KvCache
    c = KvCache(1, 4096, 2, 128)
    fill(c, 101)
    want, _ = c.read(0, 0, 4096)
    s = torch.cuda.Stream()
    kept = torch.empty(4096, 256, device="cuda")
    torch.cuda.synchronize()
    for _ in range(3):
        given_up = [torch.full((4096, 256), 5.0, device="cuda") for _ in range(4)]
        torch.cuda._sleep(20_000_000)   # ~10 ms of the current stream
        for t in given_up:
            kept.copy_(t)
        ptrs = {t.data_ptr() for t in given_up}
        del given_up, t
        k, v = c.read(0, 0, 4096, stream=s)
        assert not ptrs & {k.data_ptr(), v.data_ptr()}
        s.synchronize()
        assert torch.equal(k, want)
        torch.cuda.synchronize()
        assert (kept == 5.0).all()
        del k, v


def test_two_threads_attend_at_once():
    """Each on its own stream with its own workspace, the first calls over a shared prefix among them."""
    import threading

    import torch
    from gtmoe.kvcache import KvAttention, KvCache
    n, P = 32, 4096
    cache, prefix = KvCache(n, 8, 2, 256), KvCache(1, P, 2, 256)
    fill(cache, 102)
    fill(prefix, 103)
    torch.cuda.synchronize()
    out, errors = {}, []

    def work(i):
        try:
            q, s = queries(n, 16, 256, i % 2), torch.cuda.Stream()
            op, ctx = KvAttention(16, 2, 256, n), torch.empty(n, 16 * 256, device="cuda")
            torch.cuda.synchronize()
            for _ in range(20):
                op(q, cache, range(n), [P + j % 8 for j in range(n)], ctx, prefix=prefix, prefix_len=P, stream=s)
            s.synchronize()
            out[i] = ctx
        except Exception as e:   # told to the test's own thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    assert torch.equal(out[0], out[2]) and torch.equal(out[1], out[3]) and not torch.equal(out[0], out[1])


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("hd,many", [(128, 2), (512, 2), (128, 64), (512, 64)])
@pytest.mark.parametrize("outlier", [2.0 ** 13, 2.0 ** 20])
def test_an_outlier_in_a_query_leaves_its_other_dims_their_bits(hd, many, outlier, fmt):
    """One dim of each query is thousands of times the others, and no key has a value there: the scores are the other
    dims', S too, and as exact as without it, beside the limbs' end, 2^-39 of the largest |q| times the keys' sum of
    |k_d|: a quarter of ds for an outlier of 2^20, which the bar's 64 steps cover, as a sum has at most 32."""
    import torch
    from gtmoe.kvcache import KvCache
    P, H = 1600, 8
    prefix, cache = KvCache(1, P, 1, hd, fmt), KvCache(1, 1, 1, hd, fmt)
    fill(prefix, 104)
    fill(cache, 105)
    for c in (prefix, cache):
        c.k.view(torch.uint8)[..., 7] = 0
    q = queries(many, H, hd)
    q.view(many, H, hd)[..., 7] = outlier * 3.0 / hd ** 0.5
    check_attention(cache, q, [0] * many, [P] * many, 0, prefix, 0, P)
