"""GPU: calls of the operators around a step's matrix products at the borders of what
include/meshgpt.h allows, against plain 64-bit forms (tests/steps_lib.py)."""
import math

import numpy as np
import pytest

import grokking_abmod_amd as G
import operators_lib as L
from test_gpu_steps import KINDS, SETTINGS, check_drawn, sampled, setting

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [1, 5, 200, 700, 9000, 40003, 90003])
@pytest.mark.parametrize("kind", KINDS)
def test_greedy_rows_look_at_no_filter_and_no_number(kind, vocab):
    """At temperature 0 settings that are no numbers do not matter, nor do their values."""
    rng = np.random.default_rng(vocab)
    choices = [0.0, 0.5, 7.0, -1.0, math.nan, math.inf]
    p, m = (a.ravel() for a in np.meshgrid(choices, choices))
    rows = len(p)
    z = L.stored(rng.normal(size=(rows, vocab)), kind)
    with L.Device() as dev:
        for kw in (dict(top_p=p, min_p=m), dict(top_p=p), dict(min_p=m), dict(top_p=p, min_p=m, top_k=np.full(rows, 3))):
            tokens, logprob, _ = sampled(dev, z, kind, temperature=np.zeros(rows), u=rng.choice([math.nan, 2.0, 0.5], rows), **kw)
            assert np.array_equal(tokens, np.argmax(L.values(z, kind), 1))
            assert not logprob.any()


@pytest.mark.parametrize("vocab", [65, 256, 257, 4096, 8192, 16384, 16385, 32768])
@pytest.mark.parametrize("kind", KINDS)
def test_rows_at_which_the_way_to_draw_changes(kind, vocab):
    """The longest and shortest rows of each way, also with a top_k of more than the threads that
    have a logit (a group of 16 bytes each: 65 or 33 of 257)."""
    rng = np.random.default_rng(vocab)
    rows = 10
    with L.Device() as dev:
        for i, kw in enumerate(SETTINGS + [dict(top_k=[60, 100, 128, 129, 200]),
                                           dict(top_k=[40, 90, 128], top_p=[0.9, 1.0], min_p=[0.0, 0.01])]):
            z = rng.normal(size=(rows, vocab)) * rng.choice([0.01, 1.0, 2.0, 8.0], (rows, 1))
            z[1::4, rng.random(vocab) < 0.7] = -np.inf
            z[:, vocab // 2] = 0.25
            u = rng.random(rows, dtype=np.float32)
            u[0], u[-1] = 0.0, 1 - 2.0**-24
            kw = {k: setting(rng, rows, v) for k, v in kw.items()}
            check_drawn(sampled(dev, L.stored(z, kind), kind, u=u, stride=vocab + i % 3, **kw))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,vocab", [(513, 256), (513, 257), (513, 32768), (513, 32769)])
def test_many_rows_at_which_the_way_to_draw_changes(kind, rows, vocab):
    rng = np.random.default_rng(vocab)
    z = rng.normal(size=(rows, vocab)) * 2
    u = rng.random(rows, dtype=np.float32)
    kw = dict(top_k=rng.choice([0, 5, 90, 200, 1000], rows), top_p=rng.choice([0.3, 0.95, 1.0], rows),
              min_p=rng.choice([0.0, 0.01], rows), temperature=rng.choice([0.0, 0.7, 1.0, 3.0], rows))
    with L.Device() as dev:
        check_drawn(sampled(dev, L.stored(z, kind), kind, u=u, **kw))


def next_to_ties(rng, width):
    """A row x and a weight with which values of the norm lie within 2^-24 of the middle of two
    codes, on the side of the odd one: (x, w, y in 64 bits)."""
    x = np.float32(rng.normal(size=width) + np.copysign(0.5, rng.normal(size=width)))
    rstd = 1 / np.sqrt(np.mean(x.astype(np.longdouble) ** 2) + np.longdouble(np.float32(1e-5)))
    # Each block of 32 begins with its largest, 400 codes' units of 2^-6; the others are codes of
    # 8 to 15 units of 2^-2 .. 2^3 and a half.
    code, power = rng.integers(8, 16, width), rng.integers(-2, 4, width)
    tie = (code + 0.5) * 2.0**power
    wanted = np.where(np.arange(width) % 32 == 0, 400.0, tie) * 2.0**-6 / (x * rstd)
    w = wanted.astype(np.float32)
    for i in np.flatnonzero(np.arange(width) % 32):
        for step in range(-3, 4):  # the floats next to it
            near = np.float32(w[i] + step * np.spacing(w[i]))
            t = x[i].astype(np.longdouble) * near * rstd * 64
            off = t / tie[i] - 1
            if 2.0**-40 < abs(off) < 2.0**-26 and (off > 0) == (code[i] % 2 == 0):
                w[i] = near
                break
    y = x.astype(np.longdouble) * w.astype(np.longdouble) * rstd
    return x, w, y


def test_codes_next_to_the_middle_of_two_are_the_nearest():
    """They are rounded once: 2^-52 of a value, FP64's, is all that they may be off by."""
    rng = np.random.default_rng(40)
    apart = 0
    with L.Device() as dev:
        for width in (64, 1000, 5000):
            x, w, y = next_to_ties(rng, width)
            codes, scales = dev.alloc(width), dev.alloc((width + 31) // 32)
            G.rms_norm_e4m3(G.MG_F32, 1, width, dev.put(x), width, None, 0, None, 0, dev.put(w), 1e-5, codes, width, scales,
                            (width + 31) // 32)
            e = dev.get(scales, (width + 31) // 32, np.uint8).astype(np.int64) - 127
            t = (y * 2.0 ** -np.repeat(e, 32)[:width]).astype(np.float64)
            nearest = L.e4m3(t)
            assert np.array_equal(L.E4M3[dev.get(codes, width, np.uint8)], nearest)
            apart += np.sum(L.e4m3(t.astype(np.float32).astype(np.float64)) != nearest)
    assert apart > 100  # by way of FP32 so many would be others


@pytest.mark.parametrize("kind,width,rows", [("bf16", 8, (1 << 22) - 1), ("bf16", 1000, 2000000), ("f32", 516, 1500000),
                                             ("f32", 4100, 700000), ("bf16", 16384, 400000)])
def test_the_weights_gradient_of_many_rows(kind, width, rows):
    """Rows of one value v, which are the gradient of the output too, and one rstd: the weight's
    gradient is rows v^2 rstd.  FP32 sums of all rows of a workgroup would be off by 2^-18 or more."""
    size = 4 if kind == "f32" else 2
    v = float(L.values(np.frombuffer(b"\x3f" * size, dtype=L.STORED[kind]), kind)[0])
    rstd = np.float32(1.2345678)
    with L.Device() as dev:
        at = dev.filled(rows * width * size, 0x3F)
        room = G.rms_norm_backward_workspace(rows, width)
        dw = dev.alloc(4 * width)
        G.rms_norm_backward(L.CODES[kind], rows, width, at, width, None, dev.put(np.full(rows, rstd)), at, width, None, 0, at,
                            width, dw, dev.alloc(room), room)
        got = dev.get(dw, width, np.float32).astype(np.float64)
    want = rows * v * v * float(rstd)
    # Runs of up to 64 rows in FP32; hat, a part and the sum are rounded to it once each.
    assert np.all(np.abs(got - want) <= (64 + 4) * 2.0**-24 * want)
