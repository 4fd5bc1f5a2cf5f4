"""gtmoe.batch.BatchDecoder with one-byte caches, a shared prefix and sampled tokens: the operators of
a serving step run together, on random-init layers of the decoder's shapes.

Bars. The last hidden state of a sequence behind a shared prefix against the same sequence run whole:
both hold the same keys and values up to codes that differ where the two runs' fp32 activations (which
differ in their last bits: other batch sizes, other orders of sums) fall on either side of a rounding
border, one step of 1/127 of a vector's largest value for a few codes in a thousand; 1% of the norm.
Against fp32 caches: a code is off by at most half a step, 1/254 of the largest value, i.e. at most
4 / 254 = 1.6% of a normed vector's rms on values and, through scores of a few units, as much again;
layer norms pass it on, two layers: 10%.
"""
from __future__ import annotations

import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "turbo-winfare_b200")]

pytestmark = pytest.mark.gpu

VOCAB, SEQS, NEW = 2000, 5, 6
PREFIX = [(17 * i + 3) % VOCAB for i in range(43)]
TAILS = [[5, 9, 11], [700], [801, 802, 803, 804], [5, 9, 12], [33, 44]]


@pytest.fixture(scope="module")
def model():
    import gtmoe
    from gtmoe import batch
    return gtmoe.SynthModel(2, seed=3), batch.synth_decoder(num_layers=2, vocab=VOCAB, seed=5, window=24, full_every=2)


def decoder(model, fmt):
    from gtmoe.batch import BatchDecoder, LocalMoe
    moe, (attn, embed, norm) = model
    return BatchDecoder(attn, LocalMoe(moe.layers, SEQS), embed, norm, 80, SEQS, kv_format=fmt)


def run(bd, prompts):
    """Greedy tokens, and each sequence's hidden state after its last prompt token."""
    import torch
    seen = {}

    def keep(step):
        torch.cuda.synchronize()
        for i, p in enumerate(prompts):
            if step == len(p) - 1:
                seen[i] = bd.hidden[i].clone()
    tokens = bd.greedy(prompts, NEW, stops=(), on_step=keep)
    return tokens, [seen[i] for i in range(len(prompts))]


def off(a, b):
    return max(float((x - y).norm() / y.norm()) for x, y in zip(a, b))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_a_shared_prefix_stands_for_each_sequence_holding_it(model, fmt):
    whole_tokens, whole = run(decoder(model, fmt), [PREFIX + t for t in TAILS])
    bd = decoder(model, fmt)
    bd.set_prefix(PREFIX)
    tokens, states = run(bd, TAILS)
    assert off(states, whole) <= 0.01, off(states, whole)
    assert [len(t) for t in tokens] == [NEW] * len(TAILS) == [len(t) for t in whole_tokens]
    again, _ = run(bd, TAILS)   # the prefix stays, and is not written over
    assert again == tokens
    bd.set_prefix([])
    assert bd.prefix_len == 0
    assert off(run(bd, [PREFIX + t for t in TAILS])[1], whole) <= 0.01


def test_one_byte_caches_against_fp32_ones(model):
    prompts = [PREFIX[:30] + t for t in TAILS]
    a, b = run(decoder(model, "int8"), prompts)[1], run(decoder(model, None), prompts)[1]
    assert 0 < off(a, b) <= 0.1, off(a, b)


def test_sampled_tokens(model):
    import torch
    from gtmoe.sampling import RowParams
    bd = decoder(model, "int8")
    bd.set_prefix(PREFIX)
    greedy = bd.greedy(TAILS, NEW, stops=())
    assert bd.sample(TAILS, NEW, RowParams(), stops=()) == greedy
    params = [RowParams(1.0, 0.9), RowParams(0.8, 1.0, 0.05), RowParams(1.0, 1.0, 0.0, 5), RowParams(), RowParams(1.2, 0.95, 0.01, 50)]
    runs = []
    for _ in range(2):
        g = torch.Generator(device="cuda").manual_seed(7)
        runs.append(bd.sample(TAILS, NEW, params, generator=g, stops=()))
    assert runs[0] == runs[1] and runs[0][3] == greedy[3]
    # the tied random embedding makes the last token's logit the softcap's 30: only heat leaves it
    g = torch.Generator(device="cuda").manual_seed(7)
    hot = bd.sample(TAILS, NEW, RowParams(20.0), generator=g, stops=())
    assert hot != greedy and len({t for seq in hot for t in seq}) > NEW
    assert all(0 <= t < VOCAB for seq in hot for t in seq)
    plain = decoder(model, None)   # sampling needs no one-byte cache
    assert len(plain.sample(TAILS, 2, RowParams(1.0, 0.9), stops=())[0]) == 2


def test_refusals(model):
    from gtmoe.sampling import RowParams
    with pytest.raises(ValueError, match="kv_format"):
        decoder(model, None).set_prefix([1])
    bd = decoder(model, "int8")
    with pytest.raises(ValueError, match="position"):
        bd.set_prefix([1] * 80)
    bd.set_prefix([1] * 70)
    with pytest.raises(ValueError, match="max_pos"):
        bd.greedy([[1, 2, 3]], 8)
    with pytest.raises(ValueError, match="settings"):
        bd.sample([[1]], 2, [RowParams(), RowParams()])


def test_a_wait_that_ran_out_in_attention_ends_the_generation(model):
    import gtmoe
    import torch
    bd = decoder(model, "int8")
    bd.set_prefix(PREFIX)
    for call in (lambda: bd.greedy(TAILS, 2, stops=()), lambda: bd.set_prefix(PREFIX)):
        next(iter(bd.kv_ops.values())).workspace[:4].view(torch.int32).fill_(2)   # as a kernel leaves it
        with pytest.raises(gtmoe.GtmError, match="timed out"):
            call()
    bd.set_prefix(PREFIX)
    assert len(bd.greedy(TAILS, 2, stops=())[0]) == 2
