"""GPU: what setting a model's filters leaves of the batch that it has."""
import pytest

import grokking_abmod_amd as G

pytestmark = pytest.mark.gpu


def test_a_batch_goes_on_after_its_filters_are_taken_away():
    config = G.named_config("mid")
    prompts = G.random_prompts(config.vocab_size, 2, 9, 1)
    with G.MeshGpt(0, config, 5, 2) as model:
        model.set_parameters(G.normal_parameters(config, 5))
        model.prefill(prompts, 0.8, 3, reserve=9 + 20)
        model.set_sampling(top_k=3)
        model.decode(4)
        model.set_sampling()
        stamps = model.decode_traced(3)
        assert stamps.shape[:2] == (3 * 2 + 2 * config.heads, 3)
        assert model.read_tokens(2).shape == (2, 9 + 1 + 4 + 3)
