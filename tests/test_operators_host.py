"""CPU: what the device operators (mg_kv8_*, mg_token_logprobs*) refuse before
they touch a device, their sizes, and the plain forms the GPU tests compare with."""
import math
import os

import numpy as np
import pytest

import grokking_abmod_amd as G
import operators_lib as L

S = (64, 64, 64)


def cache(batch=2, kv_heads=2, head_width=64, capacity=128, k=256, v=256, ks=256, vs=256):
    return G.Kv8(batch, kv_heads, head_width, capacity, k, v, ks, vs)


def refused(match, f, *args, **kw):
    with pytest.raises(G.MeshGptError, match=match) as info:
        f(*args, **kw)
    assert info.value.status == G.MG_INVALID_ARGUMENT


@pytest.mark.parametrize("kw,match", [
    (dict(head_width=0), "head width must be in 1..256"), (dict(head_width=257), "head width must be in 1..256"),
    (dict(capacity=0), "multiple of 64"), (dict(capacity=100), "multiple of 64"), (dict(capacity=1 << 25), "multiple of 64"),
    (dict(kv_heads=0), "heads must be in 1..4096"), (dict(kv_heads=5000), "heads must be in 1..4096"),
    (dict(batch=(1 << 24) + 1), "out of range"), (dict(batch=1 << 24, kv_heads=4096), "below 2\\^31"),
    (dict(k=0), "must not be null"), (dict(vs=0), "must not be null"), (dict(k=264), "aligned to 16"),
    (dict(v=257), "aligned to 16"), (dict(ks=257), "aligned to 4"), (dict(vs=258), "aligned to 4")])
def test_caches_that_cannot_be(kw, match):
    c = cache(**kw)
    refused(match, G.kv8_append, c, G.MG_F32, 1, 256, S, 256, S, 256)
    refused(match, G.kv8_read, c, G.MG_F32, 0, 1, 256, S, 256, S)
    refused(match, G.kv8_attention, c, G.MG_F32, 5000 if "kv_heads" in kw else 2, 1, 256, S, 256, S, 256, None, 1.0)
    if not {"k", "v", "ks", "vs"} & set(kw):
        refused(match, G.kv8_sizes, c)


def test_append_refusals():
    c = cache()
    refused("element type", G.kv8_append, c, 3, 1, 256, S, 256, S, 256)
    refused("element type", G.kv8_append, c, -1, 1, 256, S, 256, S, 256)
    refused("capacity", G.kv8_append, c, G.MG_F32, 129, 256, S, 256, S, 256)
    refused("null", G.kv8_append, c, G.MG_F32, 1, None, S, 256, S, 256)
    refused("null", G.kv8_append, c, G.MG_F32, 1, 256, S, None, S, 256)
    refused("null", G.kv8_append, c, G.MG_F32, 1, 256, S, 256, S, None)
    refused("aligned to their type", G.kv8_append, c, G.MG_F32, 1, 258, S, 256, S, 256)
    refused("aligned to their type", G.kv8_append, c, G.MG_BF16, 1, 256, S, 257, S, 256)
    big = cache(batch=1 << 23, kv_heads=255, capacity=1 << 24)
    refused("too large", G.kv8_append, big, G.MG_F32, 1 << 20, 256, S, 256, S, 256)


def test_read_refusals():
    c = cache()
    refused("element type", G.kv8_read, c, 7, 0, 1, 256, S, 256, S)
    refused("inside the cache's capacity", G.kv8_read, c, G.MG_F32, 129, 0, 256, S, 256, S)
    refused("inside the cache's capacity", G.kv8_read, c, G.MG_F32, 100, 29, 256, S, 256, S)
    refused("inside the cache's capacity", G.kv8_read, c, G.MG_F32, (1 << 64) - 1, 2, 256, S, 256, S)
    refused("null", G.kv8_read, c, G.MG_F32, 0, 1, None, S, 256, S)
    refused("aligned to their type", G.kv8_read, c, G.MG_F16, 0, 1, 256, S, 259, S)


def test_attention_refusals():
    c = cache()
    call = lambda **kw: G.kv8_attention(**{**dict(cache=c, type=G.MG_F32, heads=4, count=1, q=256, q_strides=S, out=256,  # noqa: E731
                                                  out_strides=S, lengths=256, counts=None, scale=0.125), **kw})
    refused("element type", call, type=3)
    refused("multiple of the cache's heads", call, heads=3)
    refused("multiple of the cache's heads", call, heads=0)
    refused("capacity", call, count=129)
    refused("null", call, q=None)
    refused("null", call, out=None)
    refused("null", call, lengths=None)
    for scale in (0.0, -1.0, math.inf, math.nan, 3e38):
        refused("scale must be finite and positive", call, scale=scale)
    refused("aligned to their type", call, q=257)
    refused("aligned to its type", call, out=258)
    long = cache(capacity=4096)
    room = G.kv8_attention_workspace(long, 4, 1)
    assert room > 0
    refused("workspace is too small", call, cache=long)
    refused("workspace is too small", call, cache=long, workspace=256, workspace_bytes=15)
    refused("aligned to 16", call, cache=long, workspace=264, workspace_bytes=room)
    refused("too large", call, cache=cache(kv_heads=1, capacity=1 << 20), heads=65536, count=1 << 20)
    refused("capacity", G.kv8_attention_workspace, c, 4, 129)
    refused("multiple of the cache's heads", G.kv8_attention_workspace, c, 3, 1)


def test_log_probability_refusals():
    call = lambda **kw: G.token_logprobs_noalloc(**{**dict(type=G.MG_F32, logits=256, rows=2, vocab=100, stride=100,  # noqa: E731
                                                           tokens=256, temperature=1.0, logprob=256), **kw})
    refused("element type", call, type=9)
    refused("1..2\\^24", call, vocab=0)
    refused("1..2\\^24", call, vocab=(1 << 24) + 1, stride=1 << 25)
    refused("stride must be at least", call, stride=99)
    for temperature in (0.0, -1.0, math.nan, math.inf, 1e-45, 4e-39):
        refused("temperature must be finite and positive", call, temperature=temperature)
    refused("at most 32", call, top=33, top_tokens=256)
    refused("too large", call, rows=1 << 24, vocab=2000, stride=2000, workspace=256, workspace_bytes=1 << 60)
    refused("too large", call, rows=(1 << 26) + 4)
    refused("more alternatives than tokens", call, vocab=5, top=6, top_tokens=256)
    refused("null", call, logits=None)
    refused("null", call, tokens=None)
    refused("null", call, top=3)
    refused("aligned to their type", call, logits=257)
    refused("below 2\\^31", call, rows=1 << 31)
    refused("workspace is too small", call, vocab=50000, stride=50000)
    refused("aligned to 8", call, vocab=50000, stride=50000, workspace=260, workspace_bytes=1 << 30)
    refused("at most 32", G.token_logprobs_workspace, 2, 100, 33)
    back = lambda **kw: G.token_logprobs_backward_noalloc(**{**dict(type=G.MG_F32, logits=256, rows=2, vocab=100, stride=100,  # noqa: E731
                                                                    tokens=256, temperature=1.0, stats=256, entropy=256,
                                                                    d_logprob=256, d_entropy=256, d_logits=256, d_stride=100), **kw})
    refused("strides must be at least", back, d_stride=99)
    refused("null", back, stats=None)
    refused("null", back, d_logits=None)
    refused("null", back, tokens=None)
    refused("needs the entropy", back, entropy=None)
    refused("temperature", back, temperature=0.0)
    refused("aligned to its type", back, d_logits=258)
    refused("at most 32", G.token_logprobs, np.zeros((1, 50)), [0], top=33)
    refused("equal rows", G.token_logprobs, np.zeros((2, 50)), [0])
    refused("outside the vocabulary", G.token_logprobs, np.zeros((1, 50)), [50])


def test_sizes():
    assert G.kv8_sizes(cache(3, 2, 50, 192, 0, 0, 0, 0)) == (3 * 2 * 192 * 64, 3 * 2 * 12)
    assert G.kv8_sizes(cache(0)) == (0, 0)
    assert G.kv8_attention_workspace(cache(0), 4, 1) == 0 and G.kv8_attention_workspace(cache(), 4, 0) == 0
    assert G.token_logprobs_workspace(0, 50000, 5) == 0 and G.token_logprobs_workspace(7, 1024, 32) == 0
    assert G.token_logprobs_workspace(1, 50000, 5) > 0


def test_calls_of_nothing_need_no_device():
    G.kv8_append(cache(0), G.MG_F32, 1, None, S, None, S, None)
    G.kv8_append(cache(), G.MG_F32, 0, None, S, None, S, None)
    G.kv8_read(cache(), G.MG_F32, 5, 0, None, S, None, S)
    G.kv8_attention(cache(), G.MG_F32, 2, 0, None, S, None, S, None, None, 1.0)
    G.token_logprobs_noalloc(G.MG_F32, None, 0, 10, 10, None, 1.0, None)
    lp, h, ids, best = G.token_logprobs(np.zeros((0, 10)), [], top=2)
    assert lp.shape == h.shape == (0,) and ids.shape == best.shape == (0, 2)


@pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="there is a GPU")
def test_calls_without_a_device_are_errors():
    for call in (lambda: G.kv8_append(cache(), G.MG_F32, 1, 256, S, 256, S, 256),
                 lambda: G.token_logprobs(np.zeros((1, 50)), [0])):
        with pytest.raises(G.MeshGptError) as info:
            call()
        assert info.value.status == G.MG_DEVICE_ERROR


def test_the_plain_forms():
    """E4M3 rounding against the table, scales against their definition."""
    finite = np.sort(L.E4M3[~np.isnan(L.E4M3)])
    x = np.random.default_rng(0).normal(size=4000) * 2.0 ** np.random.default_rng(1).integers(-12, 8, 4000)
    x = np.clip(x, -448, 448)
    near = np.abs(x[:, None] - finite).min(1)
    assert np.array_equal(np.abs(L.e4m3(x) - x), near)
    for top, e in ((448.0, 0), (449.0, 1), (224.0, -1), (0.0, -117), (1e-45, -117), (3.4e38, 120)):
        assert L.scale_exponent(np.array([top, 0.0, np.nan, np.inf])) == e


def test_the_command_line_checks_the_cache():
    import subprocess
    r = subprocess.run([G.CLI_PATH, "generate", "--config", "tiny", "--cache", "int4"], capture_output=True, text=True)
    assert r.returncode != 0 and "unknown cache: int4; use f32 or e4m3" in r.stdout + r.stderr
    r = subprocess.run([G.CLI_PATH, "--help"], capture_output=True, text=True)
    assert "--cache NAME" in r.stdout + r.stderr
