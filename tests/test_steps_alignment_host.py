"""CPU: pointers to 32-bit values that are not aligned to them are refused by the operators
around a step's matrix products (a scalar load would read from another address)."""
import pytest

import grokking_abmod_amd as G

THREE = (64, 64, 64)


def draws(**kw):
    G.sample_filtered_noalloc(**{**dict(type=G.MG_BF16, logits=258, rows=2, vocab=10, stride=10, temperatures=256, top_k=256,
                                        top_p=256, min_p=256, uniforms=256, tokens=256, logprob=256), **kw})


def turns(f, **kw):
    q, k = ("q", "k") if f is G.rope else ("d_q_out", "d_k_out")
    q_out, k_out = ("q_out", "k_out") if f is G.rope else ("d_q", "d_k")
    at = {name: 256 for name in (q, k, q_out, k_out)} | {name + "_strides": THREE for name in (q, k, q_out, k_out)}
    f(**{**dict(rope=G.Rope(64, 64, 0, 1.0, 256), type=G.MG_F32, batch=2, count=3, heads=4, kv_heads=2, lengths=256, counts=256,
                positions=256), **at, **kw})


def norms(f, **kw):
    args = dict(type=G.MG_F32, rows=2, width=64, x=256, x_stride=64, residual=None, residual_stride=0, sum=None, sum_stride=0,
                weight=None, epsilon=1e-5, rstd=256)
    args |= dict(out=256, out_stride=64) if f is G.rms_norm else dict(codes=257, codes_stride=64, scales=257, scales_stride=2)
    f(**{**args, **kw})


def norm_gradients(**kw):
    G.rms_norm_backward(**{**dict(type=G.MG_F32, rows=2, width=64, sum=256, sum_stride=64, weight=None, rstd=256, d_out=256,
                                  d_out_stride=64, d_sum=None, d_sum_stride=0, d_x=256, d_x_stride=64, d_weight=256), **kw})


CALLS = [(draws, name) for name in ("temperatures", "top_k", "top_p", "min_p", "uniforms", "tokens", "logprob")]
CALLS += [(lambda f=f, **kw: turns(f, **kw), name) for f in (G.rope, G.rope_backward) for name in ("lengths", "counts", "positions")]
CALLS += [(lambda f=f, **kw: norms(f, **kw), "rstd") for f in (G.rms_norm, G.rms_norm_e4m3)]
CALLS += [(norm_gradients, name) for name in ("rstd", "d_weight")]


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("call,name", CALLS)
def test_words_off_their_alignment_are_refused(call, name, off):
    with pytest.raises(G.MeshGptError, match="aligned to 4 bytes") as info:
        call(**{name: 256 + off})
    assert info.value.status == G.MG_INVALID_ARGUMENT
