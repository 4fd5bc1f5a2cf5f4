"""Host-side checks of the one-byte KV cache and row-sampling entries: arguments they reject before
touching the GPU, and the workspace plan. The device tests are in tests/test_kvcache_gpu.py and
tests/test_sample_rows_gpu.py."""
from __future__ import annotations

import ctypes as C
import os
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "turbo-winfare_b200")]

import gtmoe  # noqa: E402

P = 256   # never dereferenced: every case fails its host-side checks


def cache(**kw):
    d = dict(k_dev=P, v_dev=P, k_scale_dev=P, v_scale_dev=P, format=0, num_seqs=2, capacity=16, kv_heads=2, head_dim=256,
             reserved=0)
    d.update(kw)
    return C.byref(gtmoe.KvCacheDesc(*d.values()))


def u32(*v):
    return (C.c_uint32 * len(v))(*v)


def write(c=None, q_heads=16, n=1, q=P, k=P, v=P, qs=4096, ks=512, vs=512, qw=None, kw=None, eps=1e-6, pairs=0, theta=1e4,
          pos=(3,), seqs=(0,), out=P):
    return gtmoe.lib().gtm_qkv_cache_rows(c if c is not None else cache(), q_heads, n, q, k, v, qs, ks, vs, qw, kw, eps, pairs,
                                          theta, u32(*pos), u32(*seqs), out, None)


def attend(c=None, prefix=None, pseq=0, plen=0, q_heads=16, n=1, window=0, q=P, seqs=(0,), pos=(3,), ctx=P, ws=P, wsb=1 << 30):
    return gtmoe.lib().gtm_attention_kv_rows(c if c is not None else cache(), prefix, pseq, plen, q_heads, n, window, q, u32(*seqs),
                                             u32(*pos), ctx, ws, wsb, None)


BAD_CACHES = [(dict(k_dev=None), gtmoe.ERR_INVALID), (dict(v_scale_dev=None), gtmoe.ERR_INVALID),
              (dict(format=2), gtmoe.ERR_UNSUPPORTED), (dict(head_dim=192), gtmoe.ERR_UNSUPPORTED),
              (dict(num_seqs=0), gtmoe.ERR_INVALID), (dict(capacity=0), gtmoe.ERR_INVALID), (dict(kv_heads=0), gtmoe.ERR_INVALID),
              (dict(reserved=1), gtmoe.ERR_INVALID), (dict(v_dev=264), gtmoe.ERR_MISALIGNED),
              (dict(k_scale_dev=258), gtmoe.ERR_MISALIGNED)]


@pytest.mark.parametrize("kw,rc", BAD_CACHES)
def test_bad_caches(kw, rc):
    c = cache(**kw)
    assert write(c) == rc
    assert gtmoe.lib().gtm_kv_read(c, 0, 0, 1, P, P, None) == rc
    assert attend(c) == rc
    assert attend(prefix=c, plen=2) == rc and "prefix" in gtmoe.last_error()


def test_null_cache():
    L = gtmoe.lib()
    assert L.gtm_qkv_cache_rows(None, 16, 1, P, P, P, 1, 1, 1, None, None, 0.0, 0, 1e4, u32(0), u32(0), P, None) == gtmoe.ERR_INVALID
    assert L.gtm_kv_read(None, 0, 0, 1, P, P, None) == gtmoe.ERR_INVALID
    assert attend(prefix=None, plen=1) == gtmoe.ERR_INVALID


@pytest.mark.parametrize("kw,rc", [
    (dict(n=513), gtmoe.ERR_INVALID), (dict(q=None), gtmoe.ERR_INVALID), (dict(v=None), gtmoe.ERR_INVALID),
    (dict(out=None), gtmoe.ERR_INVALID), (dict(q_heads=0), gtmoe.ERR_UNSUPPORTED), (dict(pairs=129), gtmoe.ERR_INVALID),
    (dict(theta=0.0), gtmoe.ERR_INVALID), (dict(theta=float("inf")), gtmoe.ERR_INVALID), (dict(eps=-1.0), gtmoe.ERR_INVALID),
    (dict(eps=float("nan")), gtmoe.ERR_INVALID), (dict(out=264), gtmoe.ERR_MISALIGNED), (dict(q=258), gtmoe.ERR_MISALIGNED),
    (dict(qw=257), gtmoe.ERR_MISALIGNED), (dict(seqs=(2,)), gtmoe.ERR_INVALID),
    (dict(n=2, pos=(3, 19), seqs=(1, 1)), gtmoe.ERR_INVALID),          # ring row 3 twice (capacity 16)
    (dict(n=2, pos=(3, 3), seqs=(0, 0)), gtmoe.ERR_INVALID),
    (dict(n=2, pos=(3, 4), seqs=(0, 0), qs=4095), gtmoe.ERR_INVALID), (dict(n=2, pos=(3, 4), seqs=(0, 0), vs=8), gtmoe.ERR_INVALID),
    (dict(n=2, pos=(3, 4), seqs=(0, 0), qs=5000, out=P), gtmoe.ERR_INVALID),   # in place over strided rows
])
def test_write_refusals(kw, rc):
    assert write(**kw) == rc and "gtm_qkv_cache_rows" in gtmoe.last_error()


def test_ring_rows_of_a_full_step_are_told_apart():
    # 512 rows that differ only in the last one; the refusal needs no GPU
    n = 512
    c = cache(num_seqs=1, capacity=4096)
    assert write(c, n=n, pos=tuple(range(n - 1)) + (4096,), seqs=(0,) * n, q=P, out=4096) == gtmoe.ERR_INVALID
    assert "ring row" in gtmoe.last_error()


def test_read_refusals():
    L = gtmoe.lib()
    assert L.gtm_kv_read(cache(), 2, 0, 1, P, P, None) == gtmoe.ERR_INVALID
    assert L.gtm_kv_read(cache(), 0, 0, 17, P, P, None) == gtmoe.ERR_INVALID
    assert L.gtm_kv_read(cache(), 0, 0xFFFFFFFF, 2, P, P, None) == gtmoe.ERR_INVALID
    assert L.gtm_kv_read(cache(), 0, 0, 1, None, None, None) == gtmoe.ERR_INVALID
    assert L.gtm_kv_read(cache(), 0, 0, 1, 264, P, None) == gtmoe.ERR_MISALIGNED
    assert L.gtm_kv_read(cache(), 0, 5, 0, None, None, None) == gtmoe.OK


@pytest.mark.parametrize("kw,rc", [
    (dict(n=513), gtmoe.ERR_INVALID), (dict(q=None), gtmoe.ERR_INVALID), (dict(ctx=None), gtmoe.ERR_INVALID),
    (dict(q=264), gtmoe.ERR_MISALIGNED), (dict(ctx=264), gtmoe.ERR_MISALIGNED), (dict(ws=264), gtmoe.ERR_MISALIGNED),
    (dict(ws=None), gtmoe.ERR_WORKSPACE), (dict(wsb=64), gtmoe.ERR_WORKSPACE),
    (dict(q_heads=0), gtmoe.ERR_UNSUPPORTED), (dict(q_heads=15), gtmoe.ERR_UNSUPPORTED), (dict(q_heads=18), gtmoe.ERR_UNSUPPORTED),
    (dict(seqs=(2,)), gtmoe.ERR_INVALID), (dict(pos=(16,)), gtmoe.ERR_INVALID),            # 17 positions, ring of 16
    (dict(pos=(0xFFFFFFFF,), window=4), gtmoe.ERR_INVALID),
    (dict(pos=(40,), plen=24, prefix=cache()), gtmoe.ERR_INVALID),                         # 17 own positions
    (dict(pos=(20,), plen=17, prefix=cache()), gtmoe.ERR_INVALID),                         # the prefix's ring holds 16
    (dict(plen=2, prefix=cache(format=1)), gtmoe.ERR_INVALID), (dict(plen=2, prefix=cache(kv_heads=4)), gtmoe.ERR_INVALID),
    (dict(plen=2, prefix=cache(head_dim=128)), gtmoe.ERR_INVALID), (dict(plen=2, prefix=cache(), pseq=2), gtmoe.ERR_INVALID),
])
def test_attention_refusals(kw, rc):
    assert attend(**kw) == rc and "gtm_attention_kv_rows" in gtmoe.last_error()


def test_empty_calls_do_nothing():
    assert write(n=0, q=None, k=None, v=None, out=None) == gtmoe.OK
    assert attend(n=0, q=None, ctx=None, ws=None, wsb=0) == gtmoe.OK
    assert gtmoe.lib().gtm_sample_rows(None, 0, 10, 10, None, None, None, None, None, None) == gtmoe.OK


def test_workspace_plan():
    f = gtmoe.lib().gtm_attention_kv_workspace_bytes
    assert f(16, 3, 256, 4) == 0 and f(16, 8, 192, 4) == 0 and f(32, 2, 256, 4) == 0 and f(16, 8, 256, 0) == 0
    assert f(16, 8, 256, 513) == 0
    sizes = [f(16, 2, 512, n) for n in (1, 2, 32, 512)]
    assert sizes == sorted(sizes) and sizes[0] > 0


def sample(n=1, vocab=1000, stride=1000, rows=((1.0, 1.0, 0.0, 0),), logits=P, u=P, token=P, kept=P, logprob=P):
    r = (gtmoe.SamplingRow * len(rows))(*[gtmoe.SamplingRow(*x) for x in rows])
    return gtmoe.lib().gtm_sample_rows(logits, n, vocab, stride, r, u, token, kept, logprob, None)


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("row", [(-1.0, 1.0, 0.0, 0), (NAN, 1.0, 0.0, 0), (INF, 1.0, 0.0, 0), (1.0, 0.0, 0.0, 0), (1.0, 1.01, 0.0, 0),
                                 (1.0, NAN, 0.0, 0), (1.0, 1.0, -0.1, 0), (1.0, 1.0, 1.1, 0), (1.0, 1.0, NAN, 0), (1.0, 1.0, 0.0, -1)])
def test_sampling_rows_refused(row):
    good = (1.0, 1.0, 0.0, 0)
    assert sample(n=2, rows=(good, row)) == gtmoe.ERR_INVALID and "row 1" in gtmoe.last_error()


def test_sampling_arguments_refused():
    assert sample(logits=None) == gtmoe.ERR_INVALID and sample(token=None) == gtmoe.ERR_INVALID
    assert sample(u=None) == gtmoe.ERR_INVALID
    assert sample(vocab=0) == gtmoe.ERR_INVALID and sample(vocab=(1 << 22) + 1) == gtmoe.ERR_INVALID
    assert sample(n=2, stride=999, rows=((1.0, 1.0, 0.0, 0),) * 2) == gtmoe.ERR_INVALID
    assert sample(n=513, rows=((0.0, 1.0, 0.0, 0),) * 513) == gtmoe.ERR_INVALID
    assert sample(logits=258) == gtmoe.ERR_MISALIGNED and sample(u=260) == gtmoe.ERR_MISALIGNED


def test_python_wrappers_check_shapes_and_types():
    import torch
    from gtmoe.kvcache import KvCache, _u32
    from gtmoe.sampling import RowParams, RowSampler
    c = KvCache(2, 16, 2, 128, device="cpu")
    assert c.k.dtype == torch.int8 and KvCache(1, 4, 1, 128, "e4m3", device="cpu").k.dtype == torch.float8_e4m3fn
    with pytest.raises(gtmoe.GtmError):
        KvCache(2, 16, 2, 128, "int4", device="cpu")
    with pytest.raises(gtmoe.GtmError):
        KvCache.over(c.k, c.v, c.k_scale, c.v_scale.transpose(1, 2))
    q, k = torch.zeros(3, 512), torch.zeros(3, 256)
    for bad in (dict(q=q.double()), dict(k=k[:, :128]), dict(v=k[:2]), dict(q_out=torch.zeros(3, 256)), dict(positions=[0, 1]),
                dict(positions=[0, 1, -1]), dict(positions=[0.5, 1, 2]), dict(q_w=torch.zeros(64, dtype=torch.bfloat16))):
        args = dict(q=q, k=k, v=k, q_out=torch.zeros(3, 512), positions=[0, 1, 2], seqs=[0, 0, 0], q_w=None)
        args.update(bad)
        with pytest.raises(gtmoe.GtmError):
            c.write(args.pop("q"), args.pop("k"), args.pop("v"), args.pop("q_out"), args.pop("positions"), args.pop("seqs"), **args)
    a = np.arange(3, dtype=np.uint32)
    p, owner = _u32(a, 3)
    assert p == a.ctypes.data and owner is a
    s = RowSampler(10, 2, device="cpu")
    with pytest.raises(gtmoe.GtmError):
        s(torch.zeros(3, 10), [RowParams()] * 3)
    with pytest.raises(gtmoe.GtmError):
        s(torch.zeros(2, 10), [RowParams()])
    with pytest.raises(gtmoe.GtmError):
        s(torch.zeros(2, 11), [RowParams()] * 2)
    with pytest.raises(gtmoe.GtmError):
        s(torch.zeros(2, 10), [RowParams(1.0)] * 2, torch.zeros(2))


def test_python_wrappers_refuse_what_a_uint32_would_wrap():
    import torch
    from gtmoe.kvcache import KvAttention, KvCache
    from gtmoe.sampling import RowParams, sampling_rows
    c, q = KvCache(2, 16, 2, 128, device="cpu"), torch.zeros(1, 512)
    for args in ((-1, 0, 1), (0, -1, 1), (0, 0, -1), (0, 1 << 32, 1)):
        with pytest.raises(gtmoe.GtmError, match="2\\^32"):
            c.read(*args, k_out=torch.zeros(1, 256))
    with pytest.raises(gtmoe.GtmError, match="rotated_pairs"):
        c.write(q, q[:, :256], q[:, :256], q, [0], [0], rotated_pairs=-1)
    att = KvAttention(4, 2, 128, 1, device="cpu")
    for kw in (dict(window=-1), dict(prefix_len=-1, prefix=c), dict(prefix_seq=1 << 32, prefix=c)):
        with pytest.raises(gtmoe.GtmError, match="2\\^32"):
            att(q, c, [0], [0], torch.zeros(1, 512), **kw)
    for top_k in (-1, 1 << 32):
        with pytest.raises(gtmoe.GtmError, match="top_k"):
            sampling_rows([RowParams(1.0, 1.0, 0.0, top_k)])


def test_check_needs_a_workspace():
    assert gtmoe.lib().gtm_attention_kv_check(None, None) == gtmoe.ERR_INVALID and "workspace" in gtmoe.last_error()


A = 1 << 20   # addresses apart from one another; never dereferenced


@pytest.mark.parametrize("kw,bad", [
    (dict(out=A + 16), True), (dict(q=A + 4, out=A + 4 * 4096), True),     # q, shifted by a little; q's last float
    (dict(k=2 * A, out=2 * A - 4 * 4096 + 16), True), (dict(k=2 * A, out=2 * A - 4 * 4096), False),   # k's first floats, and just before them
    (dict(v=3 * A, out=3 * A + 4 * 508), True), (dict(v=3 * A, out=3 * A + 4 * 512), False),           # v's last ones, and just behind
    (dict(n=2, pos=(3, 4), seqs=(0, 0), qs=100000, out=A + 4 * 4096), False),         # between two strided rows
    (dict(n=2, pos=(3, 4), seqs=(0, 0), qs=12284, out=A + 4 * 4096), True),            # not quite
    (dict(out=A), False),                                                               # in place
    (dict(out=A, k=A + 4 * 4000), True),
])
def test_write_refuses_an_output_over_its_inputs(kw, bad):
    args = dict(q=A, k=4 * A, v=5 * A, out=8 * A)
    args.update(kw)
    import torch
    if not bad and torch.cuda.is_available():
        pytest.skip("made-up addresses: only on a machine without a GPU")
    rc = write(**args)
    assert (rc == gtmoe.ERR_INVALID and "overlap" in gtmoe.last_error()) == bad


def test_attention_refuses_overlaps():
    n = dict(n=2, seqs=(0, 0), pos=(3, 3))
    size, ws = 2 * 16 * 256 * 4, gtmoe.lib().gtm_attention_kv_workspace_bytes(16, 2, 256, 2)
    for kw in (dict(q=A, ctx=A + 16), dict(q=A, ctx=A - size + 16), dict(q=A, ctx=2 * A, ws=A + size - 16),
               dict(q=A, ctx=A + 64 * A, ws=A + 64 * A - ws + 16)):
        assert attend(**{**n, **{"ws": 512 * A}, **kw}) == gtmoe.ERR_INVALID and "overlap" in gtmoe.last_error(), kw


def test_norm_weights_are_bf16_or_its_bits():
    import torch
    from gtmoe.kvcache import _bf16
    cpu = torch.device("cpu")
    for dt in (torch.bfloat16, torch.int16, torch.uint16):
        t = torch.zeros(4, dtype=dt)
        assert _bf16(t, "q_w", cpu, 4) == t.data_ptr()
    assert _bf16(None, "q_w", cpu, 4) is None
    for t in (torch.zeros(4, dtype=torch.float16), torch.zeros(4), torch.zeros(4, dtype=torch.int8), torch.zeros(8, dtype=torch.bfloat16)[::2]):
        with pytest.raises(gtmoe.GtmError, match="q_w must be 4 contiguous bf16"):
            _bf16(t, "q_w", cpu, 4)
