"""CPU: what the Python binding keeps of a model's batch beside the library."""
import pytest

import grokking_abmod_amd as G


class Succeeds:
    """A library of which every call succeeds and does nothing."""

    def __getattr__(self, name):
        return lambda *args: 0


@pytest.fixture
def model(monkeypatch):
    monkeypatch.setattr(G, "lib", Succeeds)
    m = G.MeshGpt(0, G.named_config("tiny"), 5, 3)
    m._batch = 3
    return m


def test_another_cache_drops_the_batch(model):
    model.set_cache(G.MG_CACHE_E4M3)
    assert model._batch == 0


def test_filters_leave_the_batch(model):
    model.set_sampling(top_k=4)
    assert model._batch == 3
