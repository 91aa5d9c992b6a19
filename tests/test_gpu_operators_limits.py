"""GPU: the device operators (mg_kv8_attention, mg_token_logprobs*) where their
precision or their inputs are at an end, against the plain 64-bit forms."""
import math

import numpy as np
import pytest

import grokking_abmod_amd as G
import operators_lib as L
from test_gpu_operators import attend, filled, score

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("width,heads,kv_heads,capacity,count,lengths", [
    (128, 8, 2, 128, 1, [1, 7, 20, 33]), (64, 2, 2, 2048, 1, [40, 1500, 3]), (256, 2, 1, 64, 3, [33, 5]),
    (32, 8, 1, 64, 2, [30, 21]), (50, 4, 4, 64, 1, [11, 29]),  # single tokens, a few
    (32, 2, 1, 256, 200, [200, 204]), (64, 2, 2, 128, 100, [100, 103]), (64, 1, 1, 1024, 200, [1024, 230]),
    (128, 2, 1, 128, 70, [70, 80]), (256, 1, 1, 192, 140, [140, 150]), (80, 1, 1, 128, 100, [100, 101])])  # prompts
def test_probabilities_of_16_bit_calls_keep_15_bits(kind, width, heads, kv_heads, capacity, count, lengths):
    """Beside the output's own rounding, a half step of the type, a call in 16 bits
    is off by no more than two BF16 pieces of each probability leave: the first one
    cut after 8 bits, the rest, under 2^-7 of it, rounded by 2^-8 of itself; once in
    the sum over the values, once in that of the probabilities.  Flat weights over
    few keys, so that little else adds to it."""
    rng = np.random.default_rng(width + count)
    cache = L.Cache(len(lengths), kv_heads, width, capacity, rng)
    filled(cache, lengths, rng)
    q = L.stored(rng.normal(size=(len(lengths), count, heads, width)), kind)
    scale = 0.2 / math.sqrt(width)
    with L.Device() as dev:
        got = attend(dev, cache.on(dev), q, kind, lengths, None, scale)
    k, v = cache.decoded()
    want, size, mass, far = L.attention(L.values(q, kind), k, v, lengths, [count] * len(lengths), scale)
    # As attention_tolerance, whose terms for scores, sums and the output stand.
    step = 2.0**-24
    exponent = 2 * (width + 2) * step * mass + 6 * step * (1.5 * far + 1)
    sums = (max(lengths) / 8 + 64) * step
    least = {"f16": 2.0**-25, "bf16": 2.0**-133}[kind]
    limit = (2 * exponent + 2 * sums + 2 * 2.0**-15) * size * 1.01 + L.HALF_STEP[kind] * np.abs(want) * 1.01 + least
    assert (np.abs(got - want) <= limit).all(), np.max(np.abs(got - want) / limit)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("count,lengths", [(1, [5, 16, 70, 128]), (40, [40, 41, 90, 128]), (130, [130, 131, 300, 320])])
@pytest.mark.parametrize("scale", [1e-11, 1e-30, 1e-42])
def test_scales_that_leave_the_scores_nothing(kind, count, lengths, scale):
    """Zero keys, whose blocks have the smallest scale, under a scale with which
    their product is no f32 any more: every key that a row sees weighs the same."""
    rng = np.random.default_rng(count)
    width, capacity = 64, 320
    cache = L.Cache(len(lengths), 1, width, capacity, rng)
    filled(cache, lengths, rng, spread=1)
    for s, n in enumerate(lengths):
        cache.k[s, :, :n] = 0
        cache.ks[s, :, :(n + 15) // 16] = 10
    q = L.stored(rng.normal(size=(len(lengths), count, 1, width)), kind)
    with L.Device() as dev:
        got = attend(dev, cache.on(dev), q, kind, lengths, None, scale)
    _, v = cache.decoded()
    for s, n in enumerate(lengths):
        for i in range(count):
            seen = v[s, 0, :n - count + i + 1]
            want, size = seen.mean(0), np.abs(seen).mean(0)
            limit = 2 * (max(lengths) / 8 + 64) * 2.0**-24 * size + L.HALF_STEP[kind] * np.abs(want) * 1.01
            assert (np.abs(got[s, i, 0] - want) <= limit + 2.0**-25).all(), (s, i)


def gradient(dev, z, kind, tokens, stats, entropy, d_logprob, d_entropy, temperature=1.0):
    rows, vocab = z.shape
    out = dev.alloc(z.nbytes)
    G.token_logprobs_backward_noalloc(L.CODES[kind], dev.put(z), rows, vocab, vocab,
                                      None if tokens is None else dev.put(np.asarray(tokens, np.uint32)), temperature, stats,
                                      entropy, None if d_logprob is None else dev.put(d_logprob),
                                      None if d_entropy is None else dev.put(d_entropy), out, vocab)
    return L.values(dev.get(out, z.shape, L.STORED[kind]), kind)


def test_tokens_do_not_matter_to_the_entropys_gradient():
    """Without a gradient of the log probabilities, a token outside the vocabulary
    is like any other."""
    rng = np.random.default_rng(1)
    z, e = (rng.normal(size=s).astype(np.float32) for s in ((4, 300), 4))
    with L.Device() as dev:
        *_, (_, h, st) = score(dev, z, "f32", [1, 2, 3, 4], 1.0, 0)
        plain = gradient(dev, z, "f32", [1, 2, 3, 4], st, h, None, e)
        assert np.isfinite(plain).all() and np.abs(plain).max() > 0
        for tokens in ([300, 1 << 31, G.IGNORE_TARGET - 1, 7], None):
            assert np.array_equal(gradient(dev, z, "f32", tokens, st, h, None, e), plain)
        # With one, its row alone is NaN.
        got = gradient(dev, z, "f32", [300, 2, 3, 4], st, h, e, None)
        assert np.isnan(got[0]).all() and np.isfinite(got[1:]).all()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [40, 5000])
def test_ignored_rows_take_no_gradient_whatever_they_hold(kind, vocab):
    """Rows behind a sequence, as a padded batch has them: their logits may be
    anything, NaN and infinities among it, and so may their d_logprob."""
    rng = np.random.default_rng(vocab)
    z = (rng.normal(size=(6, vocab)) * 3).astype(np.float32)
    z[1] = np.nan
    z[2, 3] = np.inf
    z[3, 4], z[3, 5] = -np.inf, np.nan
    z[4] = -np.inf
    z = L.stored(z, kind)
    tokens = np.full(6, G.IGNORE_TARGET, np.uint32)
    tokens[5] = 7
    g = np.array([1, 2, np.nan, np.inf, 3, 1], np.float32)
    e = np.array([0, 0, -0.0, 0, 0, 0.5], np.float32)
    with L.Device() as dev:
        lp, h, *_, (_, hp, st) = score(dev, z, kind, tokens, 1.0, 0)
        assert (lp[:5] == 0).all() and np.isnan(h[1:4]).all()
        for d_entropy in (None, e):
            got = gradient(dev, z, kind, tokens, st, hp, g, d_entropy)
            assert (got[:5] == 0).all() and np.isfinite(got[5]).all() and np.abs(got[5]).max() > 0
        # The entropy of such a row is NaN, and asked for, its gradient is.
        assert np.isnan(gradient(dev, z, kind, tokens, st, hp, None, np.ones(6, np.float32))[1:4]).all()
