"""CPU: the oracle's decode from an 8-bit cache, where it has to be the FP32 one's."""
import ctypes

import numpy as np
import pytest

import oracle_lib as O


def unrounded(c, params, prompt, count):
    """The tokens and the last step's logits of the same decode from 64 bits."""
    out, logits = np.zeros(prompt.size + count, dtype=np.uint32), np.zeros(c.vocab_size, dtype=np.float32)
    assert O.lib().og_generate_cached(ctypes.byref(c), O.ptr(O.f32(params), O._f32p), O.ptr(prompt, O._u32p), prompt.size,
                                      count, 0.0, 7, O.ptr(out, O._u32p), O.ptr(logits, O._f32p)) == 0
    return out, logits


@pytest.mark.parametrize("prompt", [1, 2, 15, 16, 17])
@pytest.mark.parametrize("kw", [dict(layers=1), dict(layers=2), dict(layers=3, xsa=0), dict(layers=2, heads=1, qk_norm=0)])
def test_prompts_of_every_length_attend_before_they_are_rounded(kw, prompt):
    """The first token's logits come from the prompt alone, so they are those of
    the cache that is not rounded; the second one's are not."""
    c = O.config(**kw)
    changed = 0
    for seed in range(4):
        params = O.initialize_normal(c, seed, 0.5)
        tokens = np.random.default_rng(seed).integers(0, c.vocab_size, prompt).astype(np.uint32)
        for count in (1, 2):
            plain, want = unrounded(c, params, tokens, count)
            rounded, got, _ = O.generate_kv8(c, params, tokens, count, 0.0, 7)
            if count == 1:
                assert np.array_equal(got, want) and np.array_equal(rounded, plain)
            else:
                changed += not np.array_equal(got, want)
    assert changed
