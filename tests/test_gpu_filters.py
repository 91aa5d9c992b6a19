"""GPU: a model that samples through filters (mg_set_sampling): its tokens are the
plain form's (tests/steps_lib.py) of its own logits and of the reference's random
numbers, on every path that a generation takes."""
import subprocess

import numpy as np
import pytest

import grokking_abmod_amd as G
import steps_lib as S

pytestmark = pytest.mark.gpu

M = (1 << 64) - 1


class Random:
    """Random::unit (src/mesh.rs:256-265)."""

    def __init__(self, seed):
        self.state = seed & M

    def unit(self):
        self.state = (self.state + 0x9E3779B97F4A7C15) & M
        z = self.state
        z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & M
        z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & M
        return ((z ^ (z >> 31)) >> 40) / 2.0**24


def drawn(logits, temperature, top_k, top_p, min_p, rng):
    f32 = lambda v: float(np.float32(v))  # noqa: E731
    return S.draw(logits, f32(temperature), top_k, f32(top_p), f32(min_p), rng.unit())[0]


MODELS = [dict(vocab_size=64, context=64, width=128, heads=4, layers=2, attention_mesh_depth=7, ffn_mesh_depth=7, connectivity=1),
          dict(vocab_size=300, context=40, width=48, heads=3, layers=2, xsa=0),
          dict(vocab_size=5000, context=24, width=32, heads=4, layers=1)]
FILTERS = [dict(top_k=5), dict(top_p=0.8), dict(min_p=0.1), dict(top_k=20, top_p=0.9, min_p=0.01)]


@pytest.mark.parametrize("kw", MODELS)
@pytest.mark.parametrize("filters", FILTERS)
@pytest.mark.parametrize("cache", [G.MG_CACHE_F32, G.MG_CACHE_E4M3])
def test_decoded_tokens_are_drawn_from_the_models_logits(kw, filters, cache):
    config, batch, temperature, seed = G.GptConfig(**kw), 3, 0.9, 11
    prompts = G.random_prompts(config.vocab_size, batch, 7, 3)
    rngs = [Random(seed + b) for b in range(batch)]
    full = {**dict(top_k=0, top_p=1.0, min_p=0.0), **filters}
    with G.MeshGpt(0, config, 5, batch) as model:
        model.set_parameters(G.normal_parameters(config, 5))
        model.set_cache(cache)
        model.set_sampling(**filters)
        model.prefill(prompts, temperature, seed, reserve=7 + 13)
        for step in range(12):
            logits, tokens = model.last_logits(batch), model.read_tokens(batch)
            want = [drawn(logits[b], temperature, rng=rngs[b], **full) for b in range(batch)]
            assert tokens[:, -1].tolist() == want, step
            if step < 11:
                model.decode(1)
        # A generation, and decode steps several at a time, give the same.
        assert np.array_equal(model.generate_tokens(prompts, 12, temperature, seed), tokens)
        model.prefill(prompts, temperature, seed, reserve=7 + 13)
        model.decode(11)
        assert np.array_equal(model.read_tokens(batch), tokens)


@pytest.mark.parametrize("kw", MODELS[:2])
def test_tokens_past_the_context(kw):
    """There every token comes from a whole window: mg_logits' logits of it."""
    config, temperature, seed = G.GptConfig(**kw), 1.1, 4
    prompt = G.random_prompts(config.vocab_size, 1, 5, 9)
    with G.MeshGpt(0, config, 6) as model:
        model.set_parameters(G.normal_parameters(config, 6))
        model.set_sampling(top_k=6, top_p=0.9)
        count = config.context + 10
        tokens = model.generate_tokens(prompt, count, temperature, seed)[0]
        rng = Random(seed)
        for n in range(5, 5 + count):
            window = tokens[max(0, n - config.context):n]
            token = drawn(model.logits(window, len(window), True)[0], temperature, 6, 0.9, 0.0, rng)
            assert tokens[n] == token, n


def test_without_filters_the_tokens_are_what_they_were():
    config = G.named_config("tiny")
    prompts = G.random_prompts(config.vocab_size, 2, 9, 1)
    with G.MeshGpt(0, config, 5, 2) as model:
        model.set_parameters(G.normal_parameters(config, 5))
        plain = model.generate_tokens(prompts, 30, 0.8, 3)
        greedy = model.generate_tokens(prompts, 30, 0.0, 3)
        model.set_sampling(top_k=3)
        through = model.generate_tokens(prompts, 30, 0.8, 3)
        assert not np.array_equal(plain, through)
        assert np.array_equal(model.generate_tokens(prompts, 30, 0.0, 3), greedy)  # greedy ones stay
        model.set_sampling(top_k=1)
        assert np.array_equal(model.generate_tokens(prompts, 30, 0.8, 3), greedy)
        model.set_sampling()
        assert np.array_equal(model.generate_tokens(prompts, 30, 0.8, 3), plain)
        # A change between decode steps holds from the next token on.
        model.prefill(prompts, 0.8, 3, reserve=9 + 30)
        model.decode(9)
        model.set_sampling(top_k=1)
        model.decode(5)
        tokens = model.read_tokens(2)
        assert np.array_equal(tokens[:, :19], plain[:, :19])
        assert tokens[0, -1] == np.argmax(model.last_logits(2)[0])


def test_settings_that_cannot_be():
    with G.MeshGpt(0, G.named_config("tiny"), 5) as model:
        for kw, match in ((dict(top_p=0.0), "top_p"), (dict(top_p=1.5), "top_p"), (dict(top_p=float("nan")), "top_p"),
                          (dict(min_p=-0.1), "min_p"), (dict(min_p=1.1), "min_p"), (dict(min_p=float("nan")), "min_p")):
            with pytest.raises(G.MeshGptError, match=match) as info:
                model.set_sampling(**kw)
            assert info.value.status == G.MG_INVALID_ARGUMENT
        model.set_sampling(top_k=4)
        model.prefill(G.random_prompts(64, 1, 4, 1), 0.5, 1, reserve=20)
        with pytest.raises(G.MeshGptError) as info:
            model.decode_traced(2)
        assert info.value.status == G.MG_UNSUPPORTED
        # Logits that are not finite are reported, as without filters.
        model.set_parameters(np.full(G.parameter_count(G.named_config("tiny")), 1e30, dtype=np.float32))
        with pytest.raises(G.MeshGptError) as info:
            model.generate_tokens(G.random_prompts(64, 1, 4, 1), 3, 0.5, 1)
        assert info.value.status == G.MG_NONFINITE


def test_the_command_line_samples_through_the_filters_it_is_given():
    config = G.named_config("tiny")
    prompt = G.random_prompts(config.vocab_size, 1, 20, 3)
    with G.MeshGpt(0, config, 3) as model:
        model.set_parameters(G.normal_parameters(config, 3))
        model.set_sampling(top_k=9, top_p=0.85, min_p=0.02)
        tokens = model.generate_tokens(prompt, 40, 0.9, 3)[0]
    run = subprocess.run([G.CLI_PATH, "generate", "--config", "tiny", "--init", "normal", "--random-prompt", "20", "--tokens", "40",
                          "--temperature", "0.9", "--seed", "3", "--top-k", "9", "--top-p", "0.85", "--min-p", "0.02"],
                         capture_output=True, timeout=100)
    assert run.returncode == 0, run.stderr
    assert run.stdout.decode() == "".join(chr(0x20 + t) for t in tokens) + "\n"
    bad = subprocess.run([G.CLI_PATH, "generate", "--config", "tiny", "--top-p", "2"], capture_output=True, timeout=100)
    assert bad.returncode != 0 and b"top_p must be in (0, 1]" in bad.stderr
