"""GPU: the 8-bit cache of a model (mg_set_cache) where a prompt is one token, and
as the command line asks for it."""
import subprocess

import numpy as np
import pytest

import grokking_abmod_amd as G
from conftest import assert_close
from test_gpu_cache8 import clear_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [dict(vocab_size=40, context=40, width=32, heads=4, layers=3),
                                dict(vocab_size=64, context=64, width=128, heads=4, layers=2, connectivity=1),
                                dict(vocab_size=50, context=48, width=48, heads=3, layers=2, xsa=0)])
@pytest.mark.parametrize("count", [1, 2, 9])
def test_a_prompt_of_one_token_attends_in_fp32(kw, count):
    """The prompt's token is quantised after its own attention, as longer ones are,
    and later layers' keys and values follow from that."""
    params, tokens, want, logits = clear_case(kw, 1, count)
    with G.MeshGpt(0, G.GptConfig(**kw), 7) as model:
        model.set_parameters(params)
        model.set_cache(G.MG_CACHE_E4M3)
        model.prefill(tokens[None], 0.0, 7, reserve=1 + count)
        if count > 1:
            model.decode(count - 1)
        assert np.array_equal(model.read_tokens(1)[0], want)
        # FP32 against the oracle's 64 bits: the roundings are the same, and a
        # prompt that attended to rounded values is off by some 1e-4.
        assert_close(model.last_logits(1)[0], logits, 1e-5)


def test_the_command_line_decodes_from_the_cache_it_is_asked_for():
    """The text of --cache e4m3 is that of the tokens of a model with such a cache,
    for a seed where the FP32 cache's are others."""
    config = G.named_config("tiny")
    for seed in range(1, 200):
        prompt = G.random_prompts(config.vocab_size, 1, 20, seed)
        with G.MeshGpt(0, config, seed) as model:
            model.set_parameters(G.normal_parameters(config, seed))
            plain = model.generate_tokens(prompt, 40, 0.0, seed)[0]
            model.set_cache(G.MG_CACHE_E4M3)
            rounded = model.generate_tokens(prompt, 40, 0.0, seed)[0]
        if not np.array_equal(plain, rounded):
            break
    else:
        raise AssertionError("no seed whose tokens the rounding changes")
    for cache, tokens in (("e4m3", rounded), ("f32", plain)):
        run = subprocess.run([G.CLI_PATH, "generate", "--config", "tiny", "--init", "normal", "--random-prompt", "20", "--tokens",
                              "40", "--temperature", "0", "--seed", str(seed), "--cache", cache], capture_output=True,
                             timeout=100)
        assert run.returncode == 0, run.stderr
        first = 0x20 if config.vocab_size == 64 else 0
        assert run.stdout.decode() == "".join(chr(first + t) for t in tokens) + "\n"
