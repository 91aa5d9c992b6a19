"""GPU: models with an 8-bit KV cache (mg_set_cache) against the oracle's decode
with its cache rounded the same way."""
import os
import subprocess

import numpy as np
import pytest

import grokking_abmod_amd as G
import oracle_lib as O
from conftest import assert_close

pytestmark = pytest.mark.gpu


def clear_case(kw, prompt, count):
    """Weights and a prompt whose keys and values all lie away from ties: FP32
    sums of up to a few hundred terms move a value by some 1e-6 of itself, 16 times
    that in steps of its rounding, a tenth of the margin asked for."""
    c = O.config(**kw)
    for seed in range(4000):
        params = O.initialize_normal(c, seed, 0.5) if seed % 2 else O.initialize(c, seed)
        tokens = np.random.default_rng(seed).integers(0, c.vocab_size, prompt).astype(np.uint32)
        out, logits, margin = O.generate_kv8(c, params, tokens, count, 0.0, 7)
        top = np.sort(logits)[::-1]
        if margin > 2e-4 and np.isfinite(logits).all() and top[0] - top[1] > 1e-2:
            return params, tokens, out, logits
    raise AssertionError("no clear case")


CASES = [
    # config, prompt, tokens: the decode kernels of a width, prompts from one token on
    (dict(vocab_size=64, context=64, width=128, heads=4, layers=2, connectivity=1), 9, 6),
    (dict(vocab_size=64, context=64, width=64, heads=2, layers=2), 17, 6),
    (dict(vocab_size=50, context=48, width=48, heads=3, layers=3), 5, 8),
    (dict(vocab_size=40, context=40, width=32, heads=4, layers=1), 1, 20),
    (dict(vocab_size=40, context=100, width=80, heads=1, layers=1), 33, 4),
    (dict(vocab_size=64, context=80, width=128, heads=1, layers=1, xsa=0, qk_norm=0), 16, 5),
]


@pytest.mark.parametrize("kw,prompt,count", CASES)
def test_decode_from_an_8_bit_cache_matches_the_oracle(kw, prompt, count):
    params, tokens, want, logits = clear_case(kw, prompt, count)
    with G.MeshGpt(0, G.GptConfig(**kw), 7) as model:
        model.set_parameters(params)
        model.set_cache(G.MG_CACHE_E4M3)
        model.prefill(tokens[None], 0.0, 7, reserve=prompt + count)
        if count > 1:
            model.decode(count - 1)
        got = model.read_tokens(1)[0]
        assert np.array_equal(got, want)
        assert_close(model.last_logits(1)[0], logits)
        # The same from one call, on a cache that held another batch.
        assert np.array_equal(model.generate_tokens(tokens[None], count, 0.0, 7)[0], want)


def test_batches_steps_and_graphs_agree():
    """Sequences of a batch alone, in one batch and in slices of it, stepped and
    through graphs of eight steps: the same tokens and logits."""
    kw = dict(vocab_size=64, context=256, width=128, heads=4, layers=2, connectivity=1)
    rng = np.random.default_rng(3)
    prompts = rng.integers(0, 64, (70, 37)).astype(np.uint32)
    with G.MeshGpt(0, G.GptConfig(**kw), 7) as model:
        model.set_cache(G.MG_CACHE_E4M3)
        model.prefill(prompts, 0.8, 11, reserve=37 + 31)
        model.decode(30)
        tokens, logits = model.read_tokens(70), model.last_logits(70)
        model.prefill(prompts, 0.8, 11, reserve=37 + 31)
        for n in (1, 3, 8, 18):
            model.decode(n)
        assert np.array_equal(model.read_tokens(70), tokens)
        assert np.array_equal(model.last_logits(70), logits)
        for b in (0, 69):
            model.prefill(prompts[b:b + 1], 0.8, 11 + b, reserve=37 + 31)
            model.decode(30)
            assert_close(model.last_logits(1)[0], logits[b])
            assert np.array_equal(model.read_tokens(1)[0], tokens[b])


def test_past_the_context_windows_are_recomputed():
    """Beyond the context nothing comes from a cache: the tokens are the FP32 ones
    from the first window on, given the same tokens before."""
    kw = dict(vocab_size=32, context=24, width=32, heads=2, layers=2)
    tokens = np.random.default_rng(1).integers(0, 32, 24).astype(np.uint32)
    with G.MeshGpt(0, G.GptConfig(**kw), 7) as model:
        want = model.generate_tokens(tokens[None], 6, 0.0, 7)
        model.set_cache(G.MG_CACHE_E4M3)
        assert np.array_equal(model.generate_tokens(tokens[None], 6, 0.0, 7), want)


def test_going_back_to_fp32_gives_the_fp32_results():
    kw = dict(vocab_size=64, context=128, width=128, heads=4, layers=2, connectivity=1)
    prompts = np.random.default_rng(2).integers(0, 64, (3, 20)).astype(np.uint32)
    with G.MeshGpt(0, G.GptConfig(**kw), 7) as model:
        want = model.generate_tokens(prompts, 40, 0.7, 5)
        model.set_cache(G.MG_CACHE_E4M3)
        model.set_cache(G.MG_CACHE_E4M3)  # no change, no effect
        rounded = model.generate_tokens(prompts, 40, 0.7, 5)
        assert rounded.shape == want.shape and np.array_equal(rounded[:, :21], want[:, :21])
        model.set_cache(G.MG_CACHE_F32)
        assert np.array_equal(model.generate_tokens(prompts, 40, 0.7, 5), want)


def test_what_an_8_bit_cache_refuses():
    kw = dict(vocab_size=64, context=128, width=128, heads=4, layers=2, connectivity=1)
    prompts = np.random.default_rng(2).integers(0, 64, (3, 20)).astype(np.uint32)
    with G.MeshGpt(0, G.GptConfig(**kw), 7) as model:
        with pytest.raises(G.MeshGptError, match="unknown cache type") as info:
            model.set_cache(2)
        assert info.value.status == G.MG_INVALID_ARGUMENT
        model.set_cache(G.MG_CACHE_E4M3)
        with pytest.raises(G.MeshGptError, match="prefilled batch"):
            model.decode(1)
        model.prefill(prompts, 0.0, 7, reserve=40)
        for call in (model.rewind, lambda: model.decode_traced(2)):
            with pytest.raises(G.MeshGptError) as info:
                call()
            assert info.value.status == G.MG_UNSUPPORTED
        assert (model.decode_profiled(3) > 0).all()
        model.set_cache(G.MG_CACHE_F32)
        with pytest.raises(G.MeshGptError, match="prefilled batch"):
            model.decode(1)
    with G.MeshGpt(0, G.GptConfig(vocab_size=8, context=16, width=512, heads=1, layers=1), 7) as model:
        with pytest.raises(G.MeshGptError, match="head widths") as info:
            model.set_cache(G.MG_CACHE_E4M3)
        assert info.value.status == G.MG_UNSUPPORTED


def test_scores_of_a_decoded_batch():
    """The last step's logits of an 8-bit decode, scored on the device: the drawn
    tokens' log probabilities against those of the logits in 64 bits."""
    kw = dict(vocab_size=64, context=64, width=64, heads=2, layers=2)
    prompts = np.random.default_rng(4).integers(0, 64, (5, 12)).astype(np.uint32)
    with G.MeshGpt(0, G.GptConfig(**kw), 7) as model:
        model.set_cache(G.MG_CACHE_E4M3)
        model.prefill(prompts, 0.9, 3, reserve=30)
        model.decode(9)
        logits, drawn = model.last_logits(5), model.read_tokens(5)[:, -1]
    lp, entropy, ids, best = G.token_logprobs(logits, drawn, temperature=0.9, top=3)
    z = logits.astype(np.float64) / np.float32(0.9)
    p = np.exp(z - z.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    assert_close(lp, np.log(p[np.arange(5), drawn]), 1e-5)
    assert_close(entropy, -(p * np.log(p)).sum(1), 1e-5)
    assert np.array_equal(ids[:, 0], logits.argmax(1))
    assert_close(best[:, 0], np.log(p.max(1)), 1e-5)


def test_the_command_line_takes_the_cache():
    run = lambda *a: subprocess.run([G.CLI_PATH, "generate", "--config", "tiny", "--random-prompt", "20", "--tokens", "12",  # noqa: E731
                                     "--temperature", "0", *a], capture_output=True, text=True, timeout=100)
    plain, rounded = run("--cache", "f32"), run("--cache", "e4m3")
    assert plain.returncode == 0 and rounded.returncode == 0, rounded.stderr
    assert len(rounded.stdout) == len(plain.stdout) and rounded.stdout[:20] == plain.stdout[:20]
    assert os.path.exists(G.CLI_PATH)
