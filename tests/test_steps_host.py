"""CPU: what the operators around a step's matrix products (mg_sample_filtered_noalloc,
mg_rope_*, mg_rms_norm*) refuse before they touch a device, the frequencies, and
the plain forms the GPU tests compare with."""
import math

import numpy as np
import pytest

import grokking_abmod_amd as G
import operators_lib as L
import steps_lib as S

THREE = (64, 64, 64)


def refused(match, f, **kw):
    with pytest.raises(G.MeshGptError, match=match) as info:
        f(**kw)
    assert info.value.status == G.MG_INVALID_ARGUMENT


def test_sampling_refusals():
    call = lambda **kw: G.sample_filtered_noalloc(**{**dict(type=G.MG_F32, logits=256, rows=2, vocab=10, stride=10,  # noqa: E731
                                                            temperatures=None, top_k=None, top_p=None, min_p=None,
                                                            uniforms=256, tokens=256), **kw})
    for code in (-1, 3):
        refused("element type", call, type=code)
    refused("1..2\\^20 tokens", call, vocab=0)
    refused("1..2\\^20 tokens", call, vocab=(1 << 20) + 1, stride=1 << 21)
    refused("row stride", call, stride=9)
    refused("rows must stay below", call, rows=1 << 22)
    for name in ("logits", "uniforms", "tokens"):
        refused("must not be null", call, **{name: None})
    refused("aligned to their type", call, logits=258)
    refused("aligned to their type", call, logits=257, type=G.MG_BF16)
    call(rows=0, logits=None, uniforms=None, tokens=None)


def test_rope_refusals():
    how = dict(head_width=64, rotary=64, layout=0, magnitude=1.0, frequencies=256)
    call = lambda how=how, **kw: G.rope(**{**dict(rope=G.Rope(*how.values()), type=G.MG_F32, batch=2, count=3, heads=4,  # noqa: E731
                                                  q=256, q_strides=THREE, q_out=256, q_out_strides=THREE, kv_heads=2, k=256,
                                                  k_strides=THREE, k_out=256, k_out_strides=THREE), **kw})
    refused("element type", call, type=7)
    refused("layout code", call, how={**how, "layout": 2})
    refused("head width must be in 1..1024", call, how={**how, "head_width": 0, "rotary": 0})
    refused("head width must be in 1..1024", call, how={**how, "head_width": 1025})
    for rotary in (63, 66, 1 << 31):
        refused("even number up to the head width", call, how={**how, "rotary": rotary})
    for m in (math.inf, math.nan):
        refused("magnitude must be finite", call, how={**how, "magnitude": m})
    refused("frequencies must not be null", call, how={**how, "frequencies": None})
    refused("frequencies must be aligned", call, how={**how, "frequencies": 260})
    refused("heads must be at most 65536", call, heads=65537)
    refused("heads must be at most 65536", call, kv_heads=1 << 40)
    refused("too large for one launch", call, batch=1 << 12, count=1 << 12)
    refused("too large for one launch", call, batch=1 << 60, count=1 << 60)
    for name in ("q", "q_out", "k", "k_out"):
        refused("must not be null", call, **{name: None})
        refused("aligned to their type", call, **{name: 258})
    for name in ("q_strides", "q_out_strides", "k_strides", "k_out_strides"):
        refused("strides must not be null", call, **{name: None})
    with pytest.raises(G.MeshGptError, match="rope must not be null"):
        G.rope(None, G.MG_F32, 1, 1, 1, 256, THREE, 256, THREE, 0, None, None, None, None)
    # Nothing to do is no error, and what has no heads is not looked at.
    call(batch=0)
    call(count=0)
    call(heads=0, kv_heads=0, q=None, q_out=None, q_strides=None, q_out_strides=None, k=None, k_out=None, k_strides=None,
         k_out_strides=None)


@pytest.mark.parametrize("rotary", [0, 2, 24, 50, 128])
@pytest.mark.parametrize("kw", [dict(), dict(base=500000.0), dict(scaling=1, factor=4.0), dict(scaling=2, factor=8.0),
                                dict(scaling=3, factor=16.0, context=2048.0, low=1.0, high=32.0)])
def test_frequencies_are_the_formulas(rotary, kw):
    got = G.rope_frequencies(rotary, **kw)
    want = S.frequencies(rotary, **kw)
    assert got.shape == (rotary // 2,)
    assert np.allclose(got, want, rtol=1e-14, atol=0)
    if kw.get("scaling") == 2 and rotary > 2:  # the last is divided by the factor, the first left
        plain = S.frequencies(rotary)
        assert got[0] == plain[0] and math.isclose(got[-1], plain[-1] / 8.0, rel_tol=1e-12)
    if kw.get("scaling") == 3 and rotary == 128:
        plain = S.frequencies(rotary)
        assert got[0] == plain[0] and math.isclose(got[-1], plain[-1] / 16.0, rel_tol=1e-14)
        assert np.any((got < plain * 0.999) & (got > plain / 15.9))


def test_frequency_refusals():
    f = G.rope_frequencies
    refused("even number", f, rotary=3)
    refused("even number", f, rotary=1026)
    for base in (1.0, 0.0, math.nan, math.inf):
        refused("base must be finite", f, rotary=8, base=base)
    for code in (-1, 4):
        refused("scaling code", f, rotary=8, scaling=code)
    for factor in (0.5, math.nan, math.inf):
        refused("factor must be", f, rotary=8, scaling=1, factor=factor)
    refused("context must be", f, rotary=8, scaling=3, factor=2.0, context=0.0)
    refused("turns must rise", f, rotary=8, scaling=3, factor=2.0, context=64.0, low=4.0, high=4.0)
    refused("turns must rise", f, rotary=8, scaling=3, factor=2.0, context=64.0, low=math.nan)
    assert G.lib().mg_rope_frequencies(8, 10000.0, 0, 0.0, 0.0, 0.0, 0.0, None) == G.MG_INVALID_ARGUMENT


def norm_call(f=G.rms_norm, **kw):
    args = dict(type=G.MG_F32, rows=2, width=64, x=256, x_stride=64, residual=256, residual_stride=64, sum=256, sum_stride=64,
                weight=256, epsilon=1e-5)
    args |= dict(out=256, out_stride=64) if f is G.rms_norm else dict(codes=256, codes_stride=64, scales=256, scales_stride=2)
    f(**{**args, **kw})


@pytest.mark.parametrize("f", [G.rms_norm, G.rms_norm_e4m3])
def test_norm_refusals(f):
    call = lambda **kw: norm_call(f, **kw)  # noqa: E731
    refused("element type", call, type=3)
    refused("width must be in 1..16384", call, width=0)
    refused("width must be in 1..16384", call, width=16385)
    refused("rows must stay below", call, rows=1 << 22)
    for name in ("x_stride", "residual_stride", "sum_stride"):
        refused("row strides", call, **{name: 63})
    for e in (0.0, -1.0, math.nan, math.inf):
        refused("epsilon must be finite and positive", call, epsilon=e)
    refused("rows must not be null", call, x=None)
    for name in ("x", "residual", "sum", "weight"):
        refused("aligned to their type", call, **{name: 258})
        refused("aligned to their type", call, **{name: 257}, type=G.MG_F16)
    if f is G.rms_norm:
        refused("row strides", call, out_stride=63)
        refused("output must not be null", call, out=None)
        refused("output must be aligned", call, out=258)
        call(rows=0, x=None, out=None)
    else:
        refused("strides of codes and scales", call, codes_stride=63)
        refused("strides of codes and scales", call, scales_stride=1)
        refused("strides of codes and scales", call, width=65, x_stride=65, residual_stride=65, sum_stride=65, codes_stride=65)
        refused("must not be null", call, codes=None)
        refused("must not be null", call, scales=None)
        call(rows=0, x=None, codes=None, scales=None)


def test_norm_gradient_refusals():
    need = G.rms_norm_backward_workspace(5000, 64)
    assert need % (64 * 4) == 0 and need > 0
    assert G.rms_norm_backward_workspace(0, 64) == G.rms_norm_backward_workspace(5, 64) == 0
    base = dict(type=G.MG_F32, rows=5000, width=64, sum=256, sum_stride=64, weight=256, rstd=256, d_out=256, d_out_stride=64,
                d_sum=256, d_sum_stride=64, d_x=256, d_x_stride=64, d_weight=256, workspace=256, workspace_bytes=need)
    call = lambda **kw: G.rms_norm_backward(**{**base, **kw})  # noqa: E731
    refused("element type", call, type=-1)
    refused("width must be", call, width=0)
    refused("width must be", G.rms_norm_backward_workspace, rows=1, width=16385)
    refused("rows must stay below", call, rows=1 << 22)
    refused("rows must stay below", call, rows=1 << 40, d_weight=None)
    for name in ("sum_stride", "d_out_stride", "d_sum_stride", "d_x_stride"):
        refused("row strides", call, **{name: 63})
    for name in ("sum", "rstd", "d_out", "d_x"):
        refused("must not be null", call, **{name: None})
    for name in ("sum", "weight", "d_out", "d_sum", "d_x"):
        refused("aligned to their type", call, **{name: 258})
    refused("workspace is too small", call, workspace_bytes=need - 1)
    refused("workspace is too small", call, workspace=None)
    refused("aligned to 4", call, workspace=258)
    call(rows=0, d_weight=None, sum=None, rstd=None, d_out=None, d_x=None)


# ---- the plain forms ------------------------------------------------------------

def test_the_plain_draw():
    z = [0.0, 2.0, 1.0, 2.0]
    w = np.exp(np.array([2.0, 2.0, 1.0, 0.0]) - 2)  # tokens 1, 3, 2, 0
    for u, token in ((0.0, 1), (0.99 * w[0] / w.sum(), 1), (1.01 * w[0] / w.sum(), 3), (0.999, 0)):
        assert S.draw(z, 1.0, 0, 1.0, 0.0, u)[0] == token
    assert S.draw(z, 1.0, 1, 1.0, 0.0, 0.99) == (1, 0.0)
    assert S.draw(z, 1.0, 2, 1.0, 0.0, 0.5)[0] == 3  # what is reached exactly is passed
    assert S.draw(z, 1.0, 0, 0.5, 0.0, 0.99)[0] == 3
    assert S.draw(z, 1.0, 2, 0.5, 0.0, 0.99)[0] == 1  # top_p of what top_k left
    assert S.draw(z, 1.0, 0, 0.0, 0.0, 0.99)[0] == 1
    assert S.draw(z, 1.0, 0, 1.0, 0.2, 0.999)[0] == 2
    assert S.draw(z, 1.0, 0, 1.0, 5.0, 0.999)[0] == 3
    assert S.draw(z, 0.0, 3, 1.0, 0.0, 7.0) == (1, 0.0)
    for bad in ([math.nan, 0.0], [math.inf, 0.0], [-math.inf] * 2):
        assert S.draw(bad, 1.0, 0, 1.0, 0.0, 0.5)[0] == S.NO_TOKEN


def test_the_plain_turn_keeps_lengths_and_turns_back():
    rng = np.random.default_rng(3)
    x = rng.normal(size=(2, 5, 3, 10))
    f = S.frequencies(8)
    at = rng.integers(0, 10**6, (2, 5))
    for interleaved in (False, True):
        y = S.turned(x, at, f, interleaved, 1.5)
        assert np.allclose(np.sum(y[..., :8] ** 2, 3), 2.25 * np.sum(x[..., :8] ** 2, 3))
        assert np.array_equal(y[..., 8:], x[..., 8:])
        assert np.allclose(S.turned(y, at, f, interleaved, 1 / 1.5, backward=True), x)


def test_the_plain_norm_gradient_is_that_of_differences():
    rng = np.random.default_rng(4)
    x, r = L.stored(rng.normal(size=(3, 9)), "f32"), None
    w, d_out, d_sum = (rng.normal(size=s) for s in ((9,), (3, 9), (3, 9)))
    value = lambda h, w: np.sum(d_out * (h / np.sqrt(np.mean(h**2, 1, keepdims=True) + 1e-5) * w)) + np.sum(d_sum * h)  # noqa: E731
    _, h, rstd, _ = S.norm(x, r, None, 1e-5, "f32")
    dx, dw = S.norm_gradient(h, w, rstd, d_out, d_sum)
    for i in range(3):
        for j in range(9):
            e = np.zeros_like(h)
            e[i, j] = 1e-5
            assert math.isclose((value(h + e, w) - value(h - e, w)) / 2e-5, dx[i, j], rel_tol=1e-5, abs_tol=1e-6)
    for j in range(9):
        e = np.zeros(9)
        e[j] = 1e-5
        assert math.isclose((value(h, w + e) - value(h, w - e)) / 2e-5, dw[j], rel_tol=1e-5, abs_tol=1e-6)
