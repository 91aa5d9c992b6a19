"""GPU: the 8-bit cache of a model (mg_set_cache) where a prompt is one token."""
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
