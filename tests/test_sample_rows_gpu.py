"""gtm_sample_rows against its definition in 64-bit numpy: tokens and kept counts equal (weights
differ by less than 2^-40 of the largest, so a draw or cut lands between the two with a chance of
~1e-6 a row; equal logits, whose sums are exact on both sides, land on it by design), log
probabilities to half an fp32 step plus 1e-9."""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "turbo-winfare_b200")]

pytestmark = pytest.mark.gpu


def one_row(z, t, top_p, min_p, top_k, u):
    z = np.where(np.isnan(z), -np.inf, z.astype(np.float64))
    t, top_p, min_p = (float(np.float32(x)) for x in (t, top_p, min_p))
    mx = z.max()
    if np.isinf(mx):
        return -1, 0, math.nan
    order = np.argsort(-z, kind="stable")
    order = order[: int((z > -np.inf).sum())]
    w = np.exp(z - mx)
    total = math.fsum(w)
    m = len(order)
    if t <= 0:
        m = 1
    else:
        if top_p < 1:
            m = min(m, int(np.searchsorted(np.cumsum(w[order]), top_p * total, side="left")) + 1)
        if min_p > 0:
            m = min(m, int((w >= min_p).sum()))
        if top_k > 0:
            m = min(m, top_k)
        m = max(1, m)
    ids = np.sort(order[:m])
    u = 0.0 if not u >= 0 else min(u, 1.0)
    mass = np.cumsum(np.exp((z[ids] - mx) / (t if t > 0 else 1.0)))
    i = min(int(np.searchsorted(mass, u * mass[-1], side="right")), int(np.flatnonzero(mass == mass[-1])[0]))
    return int(ids[i]), m, z[ids[i]] - mx - math.log(total)


def check(z, rules, u, logits=None, stream=None):
    import torch
    from gtmoe.sampling import RowParams, RowSampler
    n, V = z.shape
    s = RowSampler(V, n)
    x = torch.from_numpy(z).cuda() if logits is None else logits
    r = s(x, [RowParams(*q) for q in rules], torch.tensor(u, dtype=torch.float64, device="cuda"), stream=stream)
    torch.cuda.synchronize()
    tokens, kept, logp = (v.cpu().numpy() for v in r)
    for i in range(n):
        want = one_row(z[i], *rules[i], u[i])
        assert (int(tokens[i]), int(kept[i])) == want[:2], (i, rules[i], u[i], want, tokens[i], kept[i])
        if want[0] >= 0:
            assert abs(logp[i] - want[2]) <= 2.0 ** -24 * abs(want[2]) + 1e-9
        else:
            assert math.isnan(logp[i])


RULES = [(0.0, 1.0, 0.0, 0), (1.0, 1.0, 0.0, 0), (0.7, 0.9, 0.0, 0), (1.3, 0.999, 0.0, 0), (1.0, 1e-6, 0.0, 0), (1.0, 1.0, 0.05, 0),
         (1.0, 1.0, 1.0, 0), (0.8, 1.0, 0.0, 1), (0.8, 1.0, 0.0, 50), (2.0, 1.0, 0.0, 5000), (1.0, 0.95, 0.01, 40), (1e-3, 1.0, 0.0, 0),
         (1.0, 0.5, 0.001, 300), (0.0, 0.3, 0.5, 7), (50.0, 1.0, 0.0, 0), (1.0, 1.0, 0.0, 1 << 30)]


def rows_of(n, V, seed, scale=2.5):
    r = np.random.default_rng(seed)
    z = r.standard_normal((n, V)) * scale
    z[np.arange(n)[:, None], r.integers(0, V, (n, 20))] += 8 * r.random((n, 20))
    return (30 * np.tanh(z / 30)).astype(np.float32), list(r.random(n))


@pytest.mark.parametrize("V", [1, 2, 31, 1000, 1024, 8191, 32003, 262144, 400001])
def test_rules(V):
    z, u = rows_of(len(RULES), V, V)
    check(z, RULES, u)


def test_a_step_of_512_rows():
    z, u = rows_of(512, 997, 3)
    check(z, [RULES[i % len(RULES)] for i in range(512)], u)


@pytest.mark.parametrize("n,V", [(8, 700001), (9, 5000), (9, 70003), (20, 262144), (33, 70000), (40, 262147), (34, 600001), (129, 66001), (40, 262144), (130, 131072),
                                 (130, 20000)])
def test_numbers_of_rows(n, V):
    """On either side of every change of the CTAs per row."""
    z, u = rows_of(n, V, n + V)
    check(z, [RULES[(5 * i + 2) % len(RULES)] for i in range(n)], u)


@pytest.mark.parametrize("scale", [1e-5, 1.0, 1e4, 1e30])
def test_ranges_of_logits(scale):
    r = np.random.default_rng(7)
    z = (r.standard_normal((len(RULES), 5000)) * scale).astype(np.float32)
    check(z, RULES, list(r.random(len(RULES))))


def test_equal_logits_take_the_lowest_ids():
    V = 4096
    z = np.full((8, V), -1.25, np.float32)
    rules = [(0.0, 1.0, 0.0, 0), (1.0, 0.5, 0.0, 0), (1.0, 1.0, 0.0, 7), (1.0, 0.25, 0.0, 100), (1.0, 1.0, 0.0, 0), (1.0, 1.0, 1.0, 0),
             (1.0, 2.0 ** -12, 0.0, 0), (1.0, 1.0, 0.0, 4096)]
    check(z, rules, [0.3, 0.5, 0.999, 0.0, 0.25, 0.75, 0.9, 1 - 2.0 ** -53])


def test_ties_at_the_border_across_the_row():
    V = 70000
    r = np.random.default_rng(11)
    z = r.integers(0, 9, (6, V)).astype(np.float32) * 0.5   # few values, thousands of ties each
    z[:, 5] = 0.0
    z[:, 69999] = -0.0
    check(z, [(1.0, 1.0, 0.0, 3), (1.0, 1.0, 0.0, 12345), (1.0, 0.3, 0.0, 0), (1.0, 0.9, 0.0, 30000), (1.0, 0.9, 0.3, 0), (1.0, 0.99, 0.0, 0)],
          list(r.random(6)))


def test_masked_and_infinite_logits():
    V = 3001
    r = np.random.default_rng(13)
    z = r.standard_normal((8, V)).astype(np.float32)
    z[0] = -np.inf
    z[1] = np.nan
    z[2, 17] = np.inf
    z[3, :] = -np.inf
    z[3, 1234] = -3.0
    z[4, ::2] = -np.inf
    z[5, 1::3] = np.nan
    z[6, :] = np.finfo(np.float32).min
    z[7, 7:] = np.finfo(np.float32).min
    check(z, [(1.0, 0.9, 0.0, 0)] * 3 + [(1.0, 0.5, 0.1, 9)] + [(1.0, 0.9, 0.0, 0), (0.9, 1.0, 0.0, 0), (1.0, 1.0, 0.0, 5), (1.0, 0.99, 0.0, 0)],
          list(r.random(8)))
    check(z, [(0.0, 1.0, 0.0, 0)] * 8, [0.5] * 8)


def test_uniforms_at_and_beyond_the_ends():
    z, _ = rows_of(7, 2000, 17)
    check(z, [(1.0, 0.9, 0.0, 0)] * 7, [0.0, 1 - 2.0 ** -53, 1.0, 7.0, -0.5, math.nan, math.inf])


def test_strided_unaligned_rows_on_another_stream():
    import torch
    z, u = rows_of(5, 1237, 19)
    flat = torch.zeros(5 * 1501 + 1, device="cuda")
    x = flat[1:].view(5, 1501)[:, :1237]
    x.copy_(torch.from_numpy(z))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    check(z, RULES[1:6], u, logits=x, stream=s)


def test_rows_do_not_depend_on_their_batch():
    import torch
    from gtmoe.sampling import RowParams, RowSampler
    z, u = rows_of(16, 50000, 23)
    x, ud = torch.from_numpy(z).cuda(), torch.tensor(u, dtype=torch.float64, device="cuda")
    s = RowSampler(50000, 16)
    params = [RowParams(*q) for q in RULES]
    whole = [v.clone() for v in s(x, params, ud)]
    for i in range(16):
        part = s(x[i:i + 1], params[i:i + 1], ud[i:i + 1])
        assert all(torch.equal(a[i:i + 1], b) for a, b in zip(whole, part))
    tail = RowSampler(50000, 20)
    tail.tokens.fill_(77)
    tail(x, params, ud)
    assert (tail.tokens[16:] == 77).all()


def test_greedy_needs_no_uniforms_and_graphs_replay():
    import torch
    from gtmoe.sampling import RowParams, RowSampler, sampling_rows
    z, u = rows_of(4, 9000, 29)
    x = torch.from_numpy(z).cuda()
    s = RowSampler(9000, 4)
    assert s(x, [RowParams()] * 4).tokens.cpu().tolist() == z.argmax(1).tolist()
    rows = sampling_rows([RowParams(*q) for q in RULES[1:5]])
    ud = torch.tensor(u, dtype=torch.float64, device="cuda")
    s(x, rows, ud)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s(x, rows, ud)
    z2, u2 = rows_of(4, 9000, 31)
    x.copy_(torch.from_numpy(z2))
    ud.copy_(torch.tensor(u2, dtype=torch.float64))
    g.replay()
    torch.cuda.synchronize()
    assert s.tokens.cpu().tolist() == [one_row(z2[i], *RULES[1 + i], u2[i])[0] for i in range(4)]


@pytest.mark.parametrize("top", [0.0, 25.0, 2000.0, -2000.0])
def test_weights_around_half_a_unit(top):
    """41 ln 2 = 28.419 below the largest a weight is half of 2^-40: up to there it is one unit, beyond it 0. At u = 0 the
    token is the lowest id with a weight. Logits of 2,000 (in steps of 2^-13) take the other form of the weight."""
    import torch
    from gtmoe.sampling import RowParams, RowSampler
    V = 300
    z = np.full((4, V), top, np.float32)
    z[:, :V - 1] -= np.linspace(28.4215, 29.3, V - 1).astype(np.float32)   # no weight: (-43,000, -42,000) / 1,024 in base 2
    z[1, 7] = np.float32(top - 28.4175)
    z[2, V - 3:V - 1] = np.float32(top - 28.4175), np.float32(top - 28.0)
    z[3, :V - 1] -= 2.0
    s = RowSampler(V, 4)
    r = s(torch.from_numpy(z).cuda(), [RowParams(1.0)] * 4, torch.zeros(4, dtype=torch.float64, device="cuda"))
    assert r.tokens.cpu().tolist() == [V - 1, 7, V - 3, V - 1] and r.kept.cpu().tolist() == [V] * 4
