"""GPU: the operators around a step's matrix products (mg_sample_filtered_noalloc,
mg_rope_*, mg_rms_norm*) against plain 64-bit forms (tests/steps_lib.py)."""
import math

import numpy as np
import pytest

import grokking_abmod_amd as G
import operators_lib as L
import steps_lib as S

pytestmark = pytest.mark.gpu

KINDS = ["f32", "f16", "bf16"]
LEAST = {"f32": 2.0**-149, "f16": 2.0**-25, "bf16": 2.0**-133}  # half the smallest step, or the smallest


# ---- sampling --------------------------------------------------------------------

def setting(rng, rows, value):
    """None, one value for all rows, or a draw for each from a list of choices."""
    if value is None:
        return None
    return rng.choice(value, rows) if isinstance(value, list) else np.full(rows, value)


def sampled(dev, z, kind, temperature=None, top_k=None, top_p=None, min_p=None, u=None, stride=None, stream=None):
    """Tokens and log probabilities of rows z (stored form), and the settings as the
    plain form takes them.  Logits lie `stride` apart, NaN between and around them."""
    rows, vocab = z.shape
    stride = vocab if stride is None else stride
    room = L.stored(np.full((rows + 2) * stride + 16, np.nan), kind)
    for r in range(rows):
        room[stride + r * stride:stride + r * stride + vocab] = z[r]
    f32 = lambda a: None if a is None else np.asarray(a, dtype=np.float32)  # noqa: E731
    temperature, top_p, min_p, u = f32(temperature), f32(top_p), f32(min_p), f32(u)
    top_k = None if top_k is None else np.asarray(top_k, dtype=np.int32)
    put = lambda a: None if a is None else dev.put(a)  # noqa: E731
    at = dev.put(room) + stride * room.itemsize
    out = dev.filled(4 * (rows + 2), 0x5A)
    lp = dev.filled(4 * (rows + 2), 0x5A)
    G.sample_filtered_noalloc(L.CODES[kind], at, rows, vocab, stride, put(temperature), put(top_k), put(top_p), put(min_p),
                              put(u), out + 4, lp + 4, stream)
    tokens, logprob = dev.get(out, rows + 2, np.uint32), dev.get(lp, rows + 2, np.uint32)
    for a in (tokens, logprob):
        assert a[0] == a[-1] == 0x5A5A5A5A
    of = lambda a, r, off: off if a is None else float(a[r])  # noqa: E731
    plain = [S.draw(L.values(z[r], kind), of(temperature, r, 1.0), int(of(top_k, r, 0)), of(top_p, r, 1.0), of(min_p, r, 0.0),
                    float(u[r])) for r in range(rows)]
    return tokens[1:-1], logprob[1:-1].view(np.float32), plain


def check_drawn(got):
    tokens, logprob, plain = got
    for r, (token, lp) in enumerate(plain):
        assert tokens[r] == token, (r, tokens[r], token)
        if math.isnan(lp):
            assert math.isnan(logprob[r])
        else:  # FP64 to the last step; sums are exact to 2^-34 of a weight
            assert abs(logprob[r] - lp) <= 1.01 * 2.0**-24 * abs(lp) + 2.0**-32, (r, logprob[r], lp)


SETTINGS = [dict(), dict(top_k=1), dict(top_k=[1, 2, 5, 50, 400]), dict(top_k=[600, 1000, 3000, 7000]), dict(top_p=0.9),
            dict(top_p=[0.0, 1e-6, 0.5, 0.999, 1.0, 3.0]), dict(min_p=[0.0, 1e-9, 0.03, 0.5, 1.0, 7.0]),
            dict(top_k=[0, 3, 40, 2000], top_p=[0.3, 0.95, 1.0], min_p=[0.0, 0.02, 0.3]),
            dict(top_k=[0, 3000], top_p=[0.97, 1.0], min_p=[1e-6, 1e-3]), dict(top_p=[0.5, 0.9], min_p=[1e-4, 0.05]),
            dict(top_k=[-1, 1 << 30, 20], temperature=[0.0, 0.01, 0.7, 1.0, 5.0, 300.0])]


@pytest.mark.parametrize("vocab", [1, 2, 3, 17, 64, 255, 1000, 1024, 1025, 1031, 2048, 2049, 4097, 20011, 131073])
@pytest.mark.parametrize("kind", KINDS)
def test_tokens_are_those_of_the_formulas(kind, vocab):
    rng = np.random.default_rng(vocab)
    with L.Device() as dev:
        for i, kw in enumerate(SETTINGS):
            rows = 12 if vocab < 5000 else 6
            z = rng.normal(size=(rows, vocab)) * rng.choice([0.01, 1.0, 2.0, 8.0], (rows, 1))
            if vocab > 2:
                z[1::4, rng.random(vocab) < 0.7] = -np.inf
                z[:, vocab // 2] = 0.25
            u = rng.random(rows, dtype=np.float32)
            u[0], u[-1] = 0.0, 1 - 2.0**-24
            kw = {k: setting(rng, rows, v) for k, v in kw.items()}
            check_drawn(sampled(dev, L.stored(z, kind), kind, u=u, stride=vocab + i % 3, **kw))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("vocab", [32768, 32769, 81919, 81920, 131064, 131071, 131072])
def test_long_rows_of_16_bits(kind, vocab):
    rng = np.random.default_rng(vocab)
    rows = 6
    z = rng.normal(size=(rows, vocab)) * np.array([[0.01], [1.0], [2.0], [8.0], [1.0], [2.0]])
    z[1, rng.random(vocab) < 0.7] = -np.inf
    z[4, rng.random(vocab) < 0.9] = -65504.0  # a mask's value
    z[5, rng.random(vocab) < 0.3] = -0.0
    u = rng.random(rows, dtype=np.float32)
    with L.Device() as dev:
        for i, kw in enumerate(SETTINGS):
            kw = {k: setting(rng, rows, v) for k, v in kw.items()}
            check_drawn(sampled(dev, L.stored(z, kind), kind, u=u, stride=vocab + i % 3, **kw))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("most", [3.0, 0.0, -0.5, -1000.0, -np.inf])
@pytest.mark.parametrize("vocab", [100003, 131071])
def test_one_value_in_most_of_a_long_row(kind, most, vocab):
    """Seven of eight tokens; in the second row the eighth is each one whose place in
    its group of eight is that of the group in eight groups."""
    rng = np.random.default_rng(12)
    z = np.full((4, vocab), most)
    token = np.arange(vocab)
    for r, others in enumerate((token % 8 == 0, token % 8 == token // 8 % 8, rng.random(vocab) < 0.125, token == 77)):
        z[r, others] = rng.normal(size=others.sum())
    u = np.array([0.1, 0.6, 0.99, 0.5], dtype=np.float32)
    with L.Device() as dev:
        for kw in (dict(), dict(top_p=np.full(4, 0.9)), dict(top_k=np.full(4, 60000), top_p=np.full(4, 0.7)),
                   dict(top_k=np.full(4, 20)), dict(top_p=np.full(4, 0.95), min_p=np.full(4, 0.05))):
            check_drawn(sampled(dev, L.stored(z, kind), kind, u=u, **kw))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(512, 4099), (513, 270), (513, 4099), (513, 8192), (513, 8193), (520, 16400)])
def test_many_rows(kind, rows, vocab):
    rng = np.random.default_rng(vocab)
    z = rng.normal(size=(rows, vocab)) * 2
    u = rng.random(rows, dtype=np.float32)
    kw = dict(top_k=rng.choice([0, 5, 90, 200, 1000], rows), top_p=rng.choice([0.3, 0.95, 1.0], rows),
              min_p=rng.choice([0.0, 0.01], rows), temperature=rng.choice([0.0, 0.7, 1.0, 3.0], rows))
    with L.Device() as dev:
        check_drawn(sampled(dev, L.stored(z, kind), kind, u=u, **kw))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_the_largest_vocabulary(kind):
    rng = np.random.default_rng(13)
    rows, vocab = 4, 1 << 20
    z = rng.normal(size=(rows, vocab))
    z[1], z[2, ::2] = 0.5, -0.25
    z[2, 1::2] = -0.125
    u = np.array([0.3, 0.7, 0.9, 1 - 2.0**-24], dtype=np.float32)
    with L.Device() as dev:
        for kw in (dict(), dict(top_p=np.full(rows, 0.8)), dict(top_k=np.full(rows, 50)), dict(top_k=np.full(rows, 400000)),
                   dict(top_p=np.full(rows, 0.9), min_p=np.full(rows, 0.3))):
            check_drawn(sampled(dev, L.stored(z, kind), kind, u=u, **kw))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("vocab", [900, 3001, 30011, 40003, 90003])
def test_equal_logits_go_by_their_tokens(kind, vocab):
    rows = 9
    rng = np.random.default_rng(5)
    z = np.full((rows, vocab), 1.5)
    z[3:6, ::7] = 1.75
    z[6:, rng.random(vocab) < 0.4] = -np.inf
    z[6:, 11] = 0.0
    z[7, ::3] = -0.0
    z[7, 1::3] = 0.0
    u = np.array([0.0, 0.5, 1 - 2.0**-24] * 3, dtype=np.float32)
    with L.Device() as dev:
        for kw in (dict(), dict(top_k=np.full(rows, min(vocab - 1, 2500))), dict(top_p=np.full(rows, 0.75)),
                   dict(min_p=np.full(rows, 1.0)), dict(top_k=np.full(rows, 2600), top_p=np.full(rows, 0.5)),
                   dict(top_p=np.full(rows, 0.75), min_p=np.full(rows, 0.9)),
                   dict(top_k=np.full(rows, vocab - 3), min_p=np.full(rows, 1e-3))):
            check_drawn(sampled(dev, L.stored(z, kind), kind, u=u, **kw))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("spread", [1e-6, 1e-3, 0.02])
@pytest.mark.parametrize("vocab", [3900, 25001, 40003, 90003])
def test_many_tokens_in_one_bin(kind, spread, vocab):
    rng = np.random.default_rng(6)
    rows = 8
    z = 3.0 + spread * rng.random((rows, vocab))
    z[4:, :100] = -40.0 + rng.random((4, 100))
    u = rng.random(rows, dtype=np.float32)
    u[:3] = 0.0, 1 - 2.0**-24, 0.5
    with L.Device() as dev:
        for kw in (dict(), dict(top_k=rng.integers(vocab // 10, vocab - 200, rows)), dict(top_p=rng.random(rows)),
                   dict(top_k=rng.integers(vocab // 10, vocab - 200, rows), top_p=rng.random(rows), min_p=np.full(rows, math.exp(-spread / 2))),
                   dict(temperature=np.full(rows, 1e3), top_p=rng.random(rows))):
            check_drawn(sampled(dev, L.stored(z, kind), kind, u=u, **kw))


@pytest.mark.parametrize("vocab,kind", [(5, "f32"), (200, "f32"), (700, "f32"), (9000, "f32"), (9000, "bf16"), (40003, "f32"),
                                        (40003, "f16"), (40003, "bf16")])
def test_rows_and_settings_that_cannot_be(vocab, kind):
    rng = np.random.default_rng(7)
    rows = 16
    z = rng.normal(size=(rows, vocab))
    z[1] = -np.inf
    z[2, vocab - 1] = np.nan
    z[3, 0] = np.inf
    z[4, 1:] = -np.inf
    z[5, :-1] = -np.inf
    t, p, m, u = np.ones(rows), np.full(rows, 0.9), np.full(rows, 0.01), np.full(rows, 0.7)
    t[6], t[7], t[8] = -1.0, np.nan, np.inf
    p[9], m[10] = np.nan, np.nan
    u[11], u[12], u[13] = 1.0, -1e-9, np.nan
    t[14], u[14] = 0.0, np.nan  # greedy: the random number does not matter
    t[15], z[15, 2] = 0.0, np.nan
    k = np.full(rows, 4)
    with L.Device() as dev:
        for kw in (dict(top_k=k, top_p=p, min_p=m), dict(top_p=p, min_p=m)):
            got = sampled(dev, L.stored(z, kind), kind, temperature=t, u=u, **kw)
            check_drawn(got)
            assert [r for r in range(rows) if got[0][r] == S.NO_TOKEN] == [1, 2, 3, 6, 7, 8, 9, 10, 11, 12, 13, 15]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("vocab", [3, 100, 1000, 5003, 20003, 40003, 90003])
def test_rows_with_a_value_that_cannot_be(kind, vocab):
    """NaN of either sign and +inf, in whole groups and behind them, with every way to draw."""
    rng = np.random.default_rng(14)
    places = [0, 1, vocab // 2, vocab - 2, vocab - 1]
    z = rng.normal(size=(3 * len(places), vocab))
    for i, at in enumerate(places):
        z[3 * i, at], z[3 * i + 1, at], z[3 * i + 2, at] = np.nan, np.copysign(np.nan, -1.0), np.inf
    rows = len(z)
    with L.Device() as dev:
        for kw in (dict(), dict(top_k=np.full(rows, 2)), dict(top_p=np.full(rows, 0.5)), dict(min_p=np.full(rows, 0.5)),
                   dict(temperature=np.zeros(rows))):
            tokens, logprob, _ = sampled(dev, L.stored(z, kind), kind, u=np.full(rows, 0.5), **kw)
            assert np.all(tokens == S.NO_TOKEN) and np.all(np.isnan(logprob))


def test_logits_and_temperatures_of_every_size():
    rng = np.random.default_rng(8)
    with L.Device() as dev:
        for vocab in (100, 5000):
            for size, t in ((1e-38, 1e-38), (3e38, 1e38), (3e38, 1.0), (1e30, 2e29), (1e-3, 1e-30), (1.0, 3e38), (1.0, 1e-45)):
                z = np.clip(rng.normal(size=(6, vocab)) / 3, -1, 1) * size
                z[0, 3] = size
                z[0, 5] = -size
                for kw in (dict(), dict(top_k=np.full(6, 7)), dict(top_p=np.full(6, 0.8)), dict(min_p=np.full(6, 0.2))):
                    u = rng.random(6, dtype=np.float32)
                    check_drawn(sampled(dev, L.stored(z, "f32"), "f32", temperature=np.full(6, t), u=u, **kw))


def test_a_row_gives_the_same_wherever_it_stands():
    rng = np.random.default_rng(9)
    vocab = 60001
    row = L.stored(rng.normal(size=vocab), "bf16")
    with L.Device() as dev:
        seen = set()
        for rows, stride in ((1, vocab), (5, vocab + 1), (300, vocab + 3)):
            u = np.full(rows, 0.4321)
            tokens, logprob, plain = sampled(dev, np.tile(row, (rows, 1)), "bf16", top_p=np.full(rows, 0.95), u=u, stride=stride)
            seen |= set(zip(tokens.tolist(), logprob.tolist()))
        assert len(seen) == 1


def test_draws_over_all_numbers_have_the_probabilities():
    """Of n evenly spread numbers a token gets its share of n, but for one at each end."""
    rng = np.random.default_rng(10)
    n, vocab = 4096, 40
    z = rng.normal(size=vocab)
    u = (np.arange(n) + 0.5) / n
    with L.Device() as dev:
        tokens, _, _ = sampled(dev, L.stored(np.tile(z, (n, 1)), "f32"), "f32", top_k=np.full(n, 30), u=u)
    w = np.exp(np.float32(z).astype(np.float64))
    w[np.argsort(-z)[30:]] = 0
    assert np.all(np.abs(np.bincount(tokens, minlength=vocab) - n * w / w.sum()) <= 1.001)


# ---- rotary positions --------------------------------------------------------------

def strided(x, order, pad):
    """x [s][t][h][d] in memory order `order` (of "sthd", d last) with `pad` elements
    behind each head: (flat array, strides); the rest is 0x5A bytes."""
    shape = dict(zip("sthd", x.shape))
    at, strides = shape["d"] + pad, {}
    for axis in reversed(order[:-1]):
        strides[axis] = at
        at *= shape[axis]
    flat = np.frombuffer(b"\x5a" * (at * x.itemsize + 16 * x.itemsize), dtype=x.dtype).copy()
    view = np.lib.stride_tricks.as_strided(flat, x.shape, [strides[a] * x.itemsize for a in "sth"] + [x.itemsize])
    view[:] = x
    return flat, [strides[a] for a in "sth"]


def viewed(flat, shape, strides):
    return np.lib.stride_tricks.as_strided(flat, shape, [s * flat.itemsize for s in strides] + [flat.itemsize])


def turn_tolerance(x, kind, rotary, interleaved, magnitude):
    """Of both products of a pair: the sine and cosine (series to 2^-26, their
    argument and sums 4 * 2^-24, the magnitude's product 2^-24), the products and
    the sum (2 * 2^-24); the output's half step."""
    pair = np.abs(np.array(x))
    first, second = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else (slice(0, rotary // 2), slice(rotary // 2, rotary))
    both = pair[..., first] + pair[..., second]
    pair[..., first] = pair[..., second] = both
    return pair * abs(magnitude) * 8 * 2.0**-24


ROPES = [
    # kind, batch, count, heads, kv_heads, width, rotary, interleaved, order, pad, lengths, counts
    ("f32", 2, 3, 2, 1, 64, 64, False, "sthd", 0, [3, 100], None),
    ("f32", 1, 1, 1, 1, 2, 2, True, "sthd", 0, [1], None),
    ("f32", 2, 5, 3, 3, 50, 24, False, "shtd", 1, [5, 9], [5, 0]),
    ("f16", 3, 7, 4, 2, 80, 50, False, "sthd", 3, [7, 100000, 8], [7, 3, 8]),
    ("f16", 3, 7, 4, 2, 80, 50, True, "tshd", 0, [7, 100000, 2], [7, 3, 3]),
    ("bf16", 2, 33, 8, 2, 128, 128, False, "sthd", 0, [33, 1 << 30], [20, 33]),
    ("bf16", 2, 17, 5, 0, 96, 96, True, "sthd", 7, None, [17, 4]),
    ("bf16", 2, 17, 0, 3, 256, 130, False, "sthd", 0, None, None),
    ("f32", 1, 9, 2, 2, 1024, 1024, False, "sthd", 0, [1 << 20], None),
    ("f16", 1, 9, 2, 1, 1023, 1022, True, "sthd", 0, [50], None),
    ("f32", 2, 3, 2, 1, 1024, 2, False, "sthd", 0, [50, 3], None),
    ("f32", 1, 3, 2, 1, 1023, 2, False, "sthd", 1, [50], None),
    ("f32", 1, 3, 1, 1, 1023, 10, False, "sthd", 0, [50], None),
    ("f32", 2, 4, 2, 1, 20, 0, False, "sthd", 0, [4, 4], [-1, 4]),
    ("bf16", 1, 1, 1, 1, 1, 0, True, "sthd", 0, [1], None),
    ("f32", 40, 70, 3, 2, 36, 36, True, "sthd", 0, [70 + 1000 * i for i in range(40)], None),
]


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("place", ["apart", "in place"])
@pytest.mark.parametrize("kind,batch,count,heads,kv_heads,width,rotary,interleaved,order,pad,lengths,counts", ROPES)
def test_turns_are_those_of_the_formulas(kind, batch, count, heads, kv_heads, width, rotary, interleaved, order, pad, lengths,
                                         counts, place, backward):
    rng = np.random.default_rng(width + rotary + count)
    f, magnitude = S.frequencies(rotary), 1.25
    given = rng.integers(-5, 1 << 31, (batch, count)).astype(np.int32) if width == 96 else None
    with L.Device() as dev:
        ints = lambda a: None if a is None else dev.put(np.asarray(a, dtype=np.int32))  # noqa: E731
        how = G.Rope(width, rotary, int(interleaved), magnitude, dev.put(f))
        sides, args = [], []
        for n in (heads, kv_heads):
            if n == 0:
                sides.append(None)
                args += [0, None, None, None, None]
                continue
            x = L.stored(rng.normal(size=(batch, count, n, width)) * 4, kind)
            flat, strides = strided(x, order, pad)
            at = dev.put(flat)
            out, out_flat, out_strides = at, flat, strides
            if place == "apart":
                out_flat, out_strides = strided(np.zeros_like(x), "hstd", 5)
                out = dev.put(out_flat)
            sides.append((x, out, out_flat, out_strides))
            args += [n, at, strides, out, out_strides]
        (G.rope_backward if backward else G.rope)(how, L.CODES[kind], batch, count, *args, ints(lengths), ints(counts), ints(given))
        at, there = S.positions(batch, count, lengths, counts, given)
        for side in sides:
            if side is None:
                continue
            x, out, flat, strides = side
            got = dev.get(out, flat.shape, flat.dtype)
            want = flat.copy()
            y = L.values(viewed(got, x.shape, strides), kind)
            v = L.values(x, kind)
            plain = S.turned(v, at, f, interleaved, magnitude, backward)
            tol = (turn_tolerance(v, kind, rotary, interleaved, magnitude) + L.HALF_STEP[kind] * np.abs(plain)) * 1.01 + LEAST[kind]
            assert np.all(np.abs(y - plain)[there] <= tol[there])
            viewed(want, x.shape, strides)[there] = viewed(got, x.shape, strides)[there]
            viewed(want, x.shape, strides)[there, :, rotary:] = x[there][:, :, rotary:]
            assert np.array_equal(got.view(np.uint8), want.view(np.uint8))  # nothing else is touched


def test_what_stays_is_left_bit_for_bit_and_nan_stays_in_its_pair():
    rng = np.random.default_rng(3)
    x = L.stored(rng.normal(size=(1, 2, 2, 48)), "bf16")
    x[0, 0, 0, 40:] = [0x7FC1, 0xFF80, 0x7F80, 0x8000, 0x0001, 0x7FFF, 0xFFFF, 0x8001]
    x[0, 1, 1, 3] = 0x7FC0
    with L.Device() as dev:
        how = G.Rope(48, 36, G.MG_ROPE_HALF, 1.0, dev.put(S.frequencies(36)))
        out = dev.filled(x.nbytes, 0)
        strides = [2 * 2 * 48, 2 * 48, 48]
        G.rope(how, G.MG_BF16, 1, 2, 2, dev.put(x), strides, out, strides, 0, None, None, None, None)
        got = dev.get(out, x.shape, np.uint16)
    assert np.array_equal(got[..., 36:], x[..., 36:])
    nan = np.isnan(L.values(got, "bf16"))[..., :36]
    assert nan[0, 1, 1, [3, 21]].all() and nan.sum() == 2


def test_a_turn_at_far_positions_keeps_its_precision():
    """Positions up to 2^31 - 1: FP64 angles are off by 2^-22 turns there at most."""
    at = np.array([[1, 4095, 1 << 20, (1 << 24) + 1, (1 << 30) + 7, (1 << 31) - 1]], dtype=np.int32)
    f = S.frequencies(64, base=500000.0, scaling=3, factor=8.0, context=8192.0)
    x = np.zeros((1, 6, 1, 64), dtype=np.float32)
    x[..., :32] = 1.0
    with L.Device() as dev:
        how = G.Rope(64, 64, G.MG_ROPE_HALF, 1.0, dev.put(f))
        p, strides = dev.put(x), [6 * 64, 64, 64]
        G.rope(how, G.MG_F32, 1, 6, 1, p, strides, p, strides, 0, None, None, None, None, None, None, dev.put(at))
        got = dev.get(p, x.shape, np.float32)
    want = S.turned(x, at, f, False, 1.0)
    # position * frequency / 2 pi in FP64: three roundings of a value of up to 2^28.4 turns.
    far = at[0][:, None, None] * np.concatenate([f, f])[None, None] * 3 * 2.0**-53
    assert np.all(np.abs(got - want)[0] <= far + 8 * 2.0**-24)


def test_the_gradient_of_a_turn_is_its_transpose():
    rng = np.random.default_rng(4)
    shape = (2, 11, 3, 40)
    x, d = (L.stored(rng.normal(size=shape), "f32") for _ in range(2))
    strides = [11 * 3 * 40, 3 * 40, 40]
    with L.Device() as dev:
        for layout in (0, 1):
            how = G.Rope(40, 30, layout, 0.8, dev.put(S.frequencies(30)))
            y, g = dev.filled(x.nbytes, 0), dev.filled(x.nbytes, 0)
            lengths = dev.put(np.array([11, 500], dtype=np.int32))
            G.rope(how, G.MG_F32, 2, 11, 3, dev.put(x), strides, y, strides, 0, None, None, None, None, lengths)
            G.rope_backward(how, G.MG_F32, 2, 11, 3, dev.put(d), strides, g, strides, 0, None, None, None, None, lengths)
            y, g = (dev.get(p, shape, np.float32).astype(np.float64) for p in (y, g))
            # <d, R x> = <R' d, x>, each to the tolerance of its 1320 pairs' outputs.
            assert abs(np.sum(d * y) - np.sum(g * x)) <= 2 * 10 * 2.0**-24 * np.sum(np.abs(d) * np.abs(x).max()) * 2


# ---- the norm ------------------------------------------------------------------------

def rows_of(dev, a, stride, lead=0):
    """Rows on the device, `stride` elements apart, the rest 0x5A bytes: (pointer, fetch)."""
    rows, width = a.shape
    flat = np.frombuffer(b"\x5a" * (a.itemsize * (lead + rows * stride + 16)), dtype=a.dtype).copy()
    view = np.lib.stride_tricks.as_strided(flat[lead:], (rows, stride), (stride * a.itemsize, a.itemsize))
    view[:, :width] = a
    p = dev.put(flat)

    def fetch():
        got = dev.get(p, flat.shape, flat.dtype)
        back = np.lib.stride_tricks.as_strided(got[lead:], (rows, stride), (stride * a.itemsize, a.itemsize))
        held = back[:, :width].copy()
        back[:, :width] = view[:, :width]
        assert np.array_equal(got.view(np.uint8), flat.view(np.uint8))  # nothing else is touched
        return held
    return p + lead * a.itemsize, fetch


def norm_inputs(rng, rows, width, kind):
    spread = np.exp(0.5 * rng.normal(size=width))
    x = L.stored(rng.normal(size=(rows, width)) * spread, kind)
    r = L.stored(3 * rng.normal(size=(rows, width)), kind)
    w = L.stored(1 + 0.2 * rng.normal(size=width), kind)
    return x, r, w


def norm_tolerance(y, kind):
    """rstd rounded, two scalings and the weight's product, in FP32; the output's half step."""
    return (4 * 2.0**-24 + L.HALF_STEP[kind]) * np.abs(y) * 1.01 + LEAST[kind]


NORMS = [(3, 1), (5, 2), (2, 7), (4, 8), (3, 31), (9, 32), (2, 33), (5, 100), (33, 256), (32, 512), (3, 1000), (2, 2048), (3, 2049),
         (2, 4096), (3, 4097), (1, 5120), (2, 8192), (2, 8200), (2, 16383), (1, 16384), (1030, 40), (700, 3001)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,width", NORMS)
def test_norms_are_those_of_the_formulas(kind, rows, width):
    rng = np.random.default_rng(rows + width)
    x, r, w = norm_inputs(rng, rows, width, kind)
    with L.Device() as dev:
        for residual, weight, keep, lead, extra in ((None, None, False, 0, 0), (r, w, True, 1, 3), (r, None, False, 0, 8),
                                                    (None, w, True, 3, 0)):
            put = lambda a: rows_of(dev, a, width + extra, lead)  # noqa: E731
            blank = np.full_like(x, 0)
            (px, fx), (ps, fs), (po, fo) = put(x), put(blank), put(blank)
            pr = put(residual)[0] if residual is not None else None
            pw = rows_of(dev, weight[None], width, lead)[0] if weight is not None else None
            stat = dev.filled(4 * rows + 8, 0x5A)
            n = width + extra
            G.rms_norm(L.CODES[kind], rows, width, px, n, pr, n, ps if keep else None, n, pw, 1e-5, po, n, stat)
            kept, h, rstd, y = S.norm(x, residual, weight, 1e-5, kind)
            got = L.values(fo(), kind)
            assert np.all(np.abs(got - y) <= norm_tolerance(y, kind))
            assert np.array_equal(fs(), kept if keep else blank)
            assert np.array_equal(fx(), x)
            s = dev.get(stat, rows + 2, np.float32)
            assert np.all(np.abs(s[:rows] - rstd) <= 1.01 * 2.0**-24 * rstd) and s[rows:].view(np.uint32).tolist() == [0x5A5A5A5A] * 2


@pytest.mark.parametrize("kind", KINDS)
def test_norms_over_their_inputs(kind):
    rng = np.random.default_rng(12)
    for rows, width in ((5, 100), (3, 5001), (2, 16000)):
        x, r, w = norm_inputs(rng, rows, width, kind)
        kept, h, rstd, y = S.norm(x, r, w, 1e-6, kind)
        with L.Device() as dev:
            pw = dev.put(w)
            # The residual takes the sum and the rows the output, or the other way about.
            for swap in (False, True):
                px, pr = dev.put(x), dev.put(r)
                out, total = (pr, px) if swap else (px, pr)
                G.rms_norm(L.CODES[kind], rows, width, px, width, pr, width, total, width, pw, 1e-6, out, width, None)
                assert np.array_equal(dev.get(total, x.shape, x.dtype), kept)
                got = L.values(dev.get(out, x.shape, x.dtype), kind)
                assert np.all(np.abs(got - y) <= norm_tolerance(y, kind))


def test_norms_of_every_magnitude():
    rng = np.random.default_rng(13)
    width = 300
    x = rng.normal(size=(9, width))
    size = np.array([0.0, 1e-45, 1e-30, 1e-3, 1.0, 1e10, 1e25, 1e37, 1e38])[:, None]
    x = np.float32(np.clip(x, -3, 3) * size)
    w = np.float32(rng.normal(size=width))
    with L.Device() as dev:
        for epsilon in (1e-5, 1e-30):
            po, stat = dev.alloc(x.nbytes), dev.alloc(4 * 9)
            G.rms_norm(G.MG_F32, 9, width, dev.put(x), width, None, width, None, width, dev.put(w), epsilon, po, width, stat)
            _, h, rstd, y = S.norm(x, None, w, epsilon, "f32")
            got = dev.get(po, x.shape, np.float32)
            # Under 2^-126 a rounding is half of 2^-149: that of h rstd, which the weight multiplies, and that of the product.
            assert np.all(np.abs(got - y) <= norm_tolerance(y, "f32") + 2.0**-150 * np.abs(w.astype(np.float64)))


@pytest.mark.parametrize("codes", [False, True])
def test_nan_and_infinities_stay_in_their_rows(codes):
    rng = np.random.default_rng(14)
    x = np.float32(rng.normal(size=(4, 100)))
    x[1, 7], x[2, 40], x[2, 41] = np.nan, np.inf, -np.inf
    with L.Device() as dev:
        out, scales = dev.filled(4 * x.size, 0), dev.filled(16, 0)
        args = [G.MG_F32, 4, 100, dev.put(x), 100, None, 0, None, 0, None, 1e-5, out, 100]
        if codes:
            G.rms_norm_e4m3(*args, scales, 4)
            got = L.E4M3[dev.get(out, x.shape, np.uint8)]
        else:
            G.rms_norm(*args)
            got = dev.get(out, x.shape, np.float32)
    assert np.isnan(got[1]).all() and not np.isnan(got[[0, 3]]).any()
    assert np.isnan(got[2, 40:42]).all() and not np.delete(got[2], [40, 41]).any()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,width", [(3, 1), (4, 31), (5, 32), (3, 33), (2, 100), (7, 512), (2, 2049), (3, 4104), (2, 9000), (1, 16200)])
def test_8_bit_norms_are_the_nearest_codes(kind, rows, width):
    rng = np.random.default_rng(rows + width)
    x, r, w = norm_inputs(rng, rows, width, kind)
    if width >= 100:
        x[0, 32:64] = r[0, 32:64] = 0  # a block of zeros
    blocks = (width + 31) // 32
    with L.Device() as dev:
        for residual, weight, lead, extra in ((r, w, 0, 0), (None, None, 1, 5)):
            n = width + extra
            (px, _), (ps, fs) = rows_of(dev, x, n, lead), rows_of(dev, np.zeros_like(x), n, lead)
            pr = rows_of(dev, residual, n, lead)[0] if residual is not None else None
            pc, fc = rows_of(dev, np.zeros((rows, width), dtype=np.uint8), n, lead)
            pb, fb = rows_of(dev, np.zeros((rows, blocks), dtype=np.uint8), blocks + extra, lead)
            stat = dev.alloc(4 * rows)
            G.rms_norm_e4m3(L.CODES[kind], rows, width, px, n, pr, n, ps, n, None if weight is None else dev.put(weight), 1e-5,
                            pc, n, pb, blocks + extra, stat)
            kept, h, rstd, y = S.norm(x, residual, weight, 1e-5, kind)
            values, scales = S.to_codes(y)
            assert np.array_equal(fs(), kept)
            assert np.array_equal(fb(), scales)
            assert np.all(np.abs(dev.get(stat, rows, np.float32) - rstd) <= 1.01 * 2.0**-24 * rstd)
            got, e = L.E4M3[fc()], scales.astype(np.float64) - 127
            # FP64, then FP32, then the code: next to a tie (2^-24 of it) either neighbour.
            t = y / 2.0 ** np.repeat(e, 32, 1)[:, :width]
            step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(t), 2.0**-6))) - 3)
            assert np.all(np.abs(got - t) <= step * 0.5 + np.abs(t) * 2.0**-24)
            assert np.mean(got != values) <= 1e-3


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,width", NORMS + [(4000, 64), (2500, 130), (1500, 5000)])
def test_norm_gradients_are_those_of_the_formulas(kind, rows, width):
    rng = np.random.default_rng(rows * width)
    x, d_out, w = norm_inputs(rng, rows, width, kind)
    d_sum = L.stored(rng.normal(size=x.shape), kind)
    h, g, ds, wv = (L.values(a, kind) for a in (x, d_out, d_sum, w))
    rstd = np.float32(1 / np.sqrt(np.mean(h**2, 1) + 1e-5))
    room = G.rms_norm_backward_workspace(rows, width)
    with L.Device() as dev:
        pr, pw = dev.put(rstd), dev.put(w)
        for weight, with_sum, place, lead, extra in ((True, True, None, 0, 0), (False, False, None, 1, 3), (True, False, "sum", 0, 0),
                                                     (True, True, "d_out", 0, 1), (False, True, "d_sum", 3, 0)):
            n = width + extra
            at = {name: rows_of(dev, a, n, lead) for name, a in (("sum", x), ("d_out", d_out), ("d_sum", d_sum))}
            pd, fd = at[place] if place else rows_of(dev, np.zeros_like(x), n, lead)
            dw = dev.filled(4 * width + 8, 0x5A)
            G.rms_norm_backward(L.CODES[kind], rows, width, at["sum"][0], n, pw if weight else None, pr, at["d_out"][0], n,
                                at["d_sum"][0] if with_sum else None, n, pd, n, dw, dev.alloc(room), room)
            hat = h * rstd.astype(np.float64)[:, None]
            dx, want = S.norm_gradient(h, wv if weight else None, rstd.astype(np.float64), g, ds if with_sum else None)
            gw = np.abs(g) * (np.abs(wv) if weight else 1)
            mass = np.mean(gw * np.abs(hat), 1, keepdims=True)
            # hat: 2 roundings, the weight's product 1.  The mean: those and 8 sums; then its product with hat, the
            # difference, rstd's product, the residual's addition and the output's half step.
            tol = rstd[:, None] * (gw * 4 + np.abs(hat) * mass * 16) * 2.0**-24 + np.abs(dx) * 2 * 2.0**-24
            tol = (tol + L.HALF_STEP[kind] * np.abs(dx)) * 1.01 + LEAST[kind]
            assert np.all(np.abs(L.values(fd(), kind) - dx) <= tol)
            # Each part sums at most rows / 512 + 4 rows in FP32, parts of four waves four more.
            got = dev.get(dw, width + 2, np.float32)
            assert np.all(np.abs(got[:width] - want) <= (rows / 512 + 12) * 2.0**-24 * np.sum(np.abs(g * hat), 0) * 1.01 + 1e-40)
            assert got[width:].view(np.uint32).tolist() == [0x5A5A5A5A] * 2


def test_the_weights_gradient_is_the_same_in_every_call_and_0_without_rows():
    rng = np.random.default_rng(15)
    rows, width = 3000, 1500
    x, d_out, w = norm_inputs(rng, rows, width, "bf16")
    room = G.rms_norm_backward_workspace(rows, width)
    with L.Device() as dev:
        px, pd, pw, pr = dev.put(x), dev.put(d_out), dev.put(w), dev.put(np.ones(rows, dtype=np.float32))
        out, dw, space = dev.alloc(x.nbytes), dev.alloc(4 * width), dev.alloc(room)
        seen = set()
        for _ in range(3):
            G.rms_norm_backward(G.MG_BF16, rows, width, px, width, pw, pr, pd, width, None, 0, out, width, dw, space, room)
            seen.add(dev.get(dw, width, np.uint32).tobytes())
        assert len(seen) == 1
        # Without the weight's gradient there is no workspace, and the rows' is the same.
        first = dev.get(out, x.shape, np.uint16)
        G.rms_norm_backward(G.MG_BF16, rows, width, px, width, pw, pr, pd, width, None, 0, out, width)
        assert np.array_equal(dev.get(out, x.shape, np.uint16), first)
        G.rms_norm_backward(G.MG_BF16, 0, width, None, width, None, None, None, width, None, 0, None, width, dw)
        assert not dev.get(dw, width, np.uint32).any()


# ---- together --------------------------------------------------------------------------

def decode_step(dev, kind, rng, batch=3, heads=4, kv_heads=2, d=32, vocab=1500, capacity=64):
    """A decode step of a transformer's parts around its products, on a stream: the
    norm, then (from given products) turned queries and keys, the 8-bit cache, its
    attention, the norm of the residual, and a token from given logits.  Returns
    (enqueue(stream), check())."""
    code = L.CODES[kind]
    width = heads * d
    x, r, w = norm_inputs(rng, batch, width, kind)
    qkv = L.stored(rng.normal(size=(batch, 1, heads + 2 * kv_heads, d)), kind)
    logits = L.stored(rng.normal(size=(batch, vocab)) * 2, kind)
    lengths = np.array([1, 17, 40], dtype=np.int32)[:batch]
    f = S.frequencies(d)
    cache = L.Cache(batch, kv_heads, d, capacity, rng)
    cache.k[:], cache.v[:] = (rng.integers(0x20, 0x40, a.shape, dtype=np.uint8) for a in (cache.k, cache.v))
    cache.ks[:], cache.vs[:] = 127, 127
    before = [a.copy() for a in cache.arrays()]
    handle = cache.on(dev)
    p = {name: dev.put(a) for name, a in dict(x=x, r=r, w=w, qkv=qkv, logits=logits, lengths=lengths, f=f,
                                              u=rng.random(batch, dtype=np.float32), k=np.full(batch, 50, dtype=np.int32),
                                              p=np.full(batch, 0.9, dtype=np.float32)).items()}
    fresh = dev.put(qkv)
    out, total, attn, tokens = dev.alloc(x.nbytes), dev.alloc(x.nbytes), dev.alloc(x.nbytes), dev.alloc(4 * batch)
    room = G.kv8_attention_workspace(handle, heads, 1)
    space = dev.alloc(room)
    n = (heads + 2 * kv_heads) * d
    strides, size = [n, n, d], qkv.itemsize
    how = G.Rope(d, d, G.MG_ROPE_HALF, 1.0, p["f"])

    def enqueue(stream):
        G.rms_norm(code, batch, width, p["x"], width, p["r"], width, total, width, p["w"], 1e-5, out, width, None, stream)
        q, k, v = p["qkv"], p["qkv"] + heads * d * size, p["qkv"] + (heads + kv_heads) * d * size
        G.rope(how, code, batch, 1, heads, q, strides, q, strides, kv_heads, k, strides, k, strides, p["lengths"], None, None,
               stream)
        G.kv8_append(handle, code, 1, k, strides, v, strides, p["lengths"], None, stream)
        G.kv8_attention(handle, code, heads, 1, q, strides, attn, [width, width, d], p["lengths"], None, d**-0.5,
                        space if room else None, room, stream)
        G.rms_norm(code, batch, width, attn, width, total, width, total, width, p["w"], 1e-5, out, width, None, stream)
        G.sample_filtered_noalloc(code, p["logits"], batch, vocab, vocab, None, p["k"], p["p"], None, p["u"], tokens, None, stream)

    def renew():
        dev.put(qkv, p["qkv"])
        for a, at in zip(before, cache.at):
            dev.put(a, at)
        dev.put(np.full(batch, 0xFFFF, dtype=np.uint32), tokens)

    def check():
        kept, h, rstd, y = S.norm(x, r, w, 1e-5, kind)
        at, _ = S.positions(batch, 1, lengths, None, None)
        got = dev.get(p["qkv"], qkv.shape, qkv.dtype)
        turned = S.turned(L.values(qkv[:, :, :heads + kv_heads], kind), at, f, False, 1.0)
        tol = (turn_tolerance(L.values(qkv[:, :, :heads + kv_heads], kind), kind, d, False, 1.0)
               + L.HALF_STEP[kind] * np.abs(turned)) * 1.01 + LEAST[kind]
        assert np.all(np.abs(L.values(got[:, :, :heads + kv_heads], kind) - turned) <= tol)
        assert np.array_equal(got[:, :, heads + kv_heads:], qkv[:, :, heads + kv_heads:])
        # What is cached and attended are the turned rows as they were stored.
        now = cache.fetch(dev)
        keys, new = L.values(got[:, :, heads:heads + kv_heads], kind), L.values(got[:, :, heads + kv_heads:], kind)
        for which, (held, _) in enumerate(L.appended(cache, before, keys, new, lengths, np.ones(batch, dtype=np.int32))):
            codes = now[0] if which == 0 else now[1].transpose(0, 1, 2, 4, 3).reshape(now[0].shape)
            for (s, hh, place), want in held.items():
                assert np.array_equal(L.E4M3[codes[s, hh, place]], want, equal_nan=True)
        k8, v8 = cache.decoded(now)
        q = L.values(got[:, :, :heads], kind)
        o, mass, far_mass, far = L.attention(q, k8, v8, lengths, np.ones(batch, dtype=np.int32), d**-0.5)
        tol = L.attention_tolerance(kind, o, mass, far_mass, far, d, capacity)
        a = dev.get(attn, x.shape, x.dtype)
        assert np.all(np.abs(L.values(a, kind).reshape(o.shape) - o) <= tol)
        kept2, _, _, y2 = S.norm(a, kept, w, 1e-5, kind)
        assert np.array_equal(dev.get(total, x.shape, x.dtype), kept2)
        assert np.all(np.abs(L.values(dev.get(out, x.shape, x.dtype), kind) - y2) <= norm_tolerance(y2, kind))
        u = dev.get(p["u"], batch, np.float32)
        want = [S.draw(L.values(logits[s], kind), 1.0, 50, float(np.float32(0.9)), 0.0, float(u[s]))[0] for s in range(batch)]
        assert dev.get(tokens, batch, np.uint32).tolist() == want

    return enqueue, renew, check


@pytest.mark.parametrize("kind", KINDS)
def test_a_decode_step(kind):
    with L.Device() as dev:
        enqueue, _, check = decode_step(dev, kind, np.random.default_rng(20))
        enqueue(None)
        check()


@pytest.mark.parametrize("kind", KINDS)
def test_a_decode_step_as_a_graph(kind):
    with L.Device() as dev:
        enqueue, renew, check = decode_step(dev, kind, np.random.default_rng(21))
        other, renew_other, check_other = decode_step(dev, kind, np.random.default_rng(22))
        stream = dev.stream()
        graph = dev.graph(stream, lambda: enqueue(stream))
        for _ in range(3):
            renew()
            renew_other()
            dev.replay(graph, stream)
            check()
            other(None)  # eager work between the replays
            check_other()


def test_steps_on_two_streams_at_once():
    with L.Device() as dev:
        a, b = (decode_step(dev, "bf16", np.random.default_rng(s)) for s in (23, 24))
        s, t = dev.stream(), dev.stream()
        for _ in range(3):
            for step in (a, b):
                step[1]()
            a[0](s)
            b[0](t)
            a[2]()
            b[2]()


def test_a_training_steps_gradient_is_that_of_differences():
    """loss = sum c log p(tokens) of logits = norm(x + r) turned: the gradient of x
    through mg_token_logprobs_backward_noalloc, mg_rope_backward and
    mg_rms_norm_backward, captured, against differences of the 64-bit forms."""
    rng = np.random.default_rng(25)
    rows, width = 6, 40
    x, r, w = norm_inputs(rng, rows, width, "f32")
    tokens, c = rng.integers(0, width, rows).astype(np.uint32), np.float32(rng.normal(size=rows))
    f, at = S.frequencies(20), np.arange(rows)[None]
    with L.Device() as dev:
        size, stream = x.nbytes, dev.stream()
        px, pr, pw, pt, pc = (dev.put(a) for a in (x, r, w, tokens, c))
        h, y, z, dz, dx = (dev.alloc(size) for _ in range(5))
        rstd, stats, lp, dw = (dev.alloc(8 * max(rows, width)) for _ in range(4))
        how = G.Rope(width, 20, G.MG_ROPE_INTERLEAVED, 1.0, dev.put(f))
        strides, room = [rows * width, width, width], G.rms_norm_backward_workspace(rows, width)
        space = dev.alloc(room)

        def enqueue(s):
            G.rms_norm(G.MG_F32, rows, width, px, width, pr, width, h, width, pw, 1e-5, y, width, rstd, s)
            G.rope(how, G.MG_F32, 1, rows, 1, y, strides, z, strides, 0, None, None, None, None, None, None, None, s)
            G.token_logprobs_noalloc(G.MG_F32, z, rows, width, width, pt, 1.0, lp, None, stats, stream=s)
            G.token_logprobs_backward_noalloc(G.MG_F32, z, rows, width, width, pt, 1.0, stats, None, pc, None, dz, width, s)
            G.rope_backward(how, G.MG_F32, 1, rows, 1, dz, strides, dz, strides, 0, None, None, None, None, None, None, None, s)
            G.rms_norm_backward(G.MG_F32, rows, width, h, width, pw, rstd, dz, width, None, 0, dx, width, dw, space, room, s)

        graph = dev.graph(stream, lambda: enqueue(stream))
        results = []
        for replayed in (False, True, True):
            for p in (dx, dw):
                dev.put(np.zeros(width, dtype=np.float32), p)
            dev.replay(graph, stream) if replayed else enqueue(None)
            results.append((dev.get(dx, x.shape, np.float32), dev.get(dw, width, np.float32)))
    for got in results[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(got, results[0]))

    def loss(x, w):
        h = x + r.astype(np.float64)
        y = h / np.sqrt(np.mean(h**2, 1, keepdims=True) + np.float32(1e-5)) * w
        z = S.turned(y[None, :, None], at, f, True, 1.0)[0, :, 0]
        m = z.max(1, keepdims=True)
        logp = z - m - np.log(np.exp(z - m).sum(1, keepdims=True))
        return float(np.sum(c * logp[np.arange(rows), tokens]))

    x64, w64, e = x.astype(np.float64), w.astype(np.float64), 1e-5
    dx, dw = results[0]
    # Differences of a smooth function at 1e-5: off by under 1e-7; FP32 forms by a few 1e-6 of values of order 1.
    for i, j in [(int(a), int(b)) for a, b in zip(rng.integers(0, rows, 40), rng.integers(0, width, 40))]:
        d = np.zeros_like(x64)
        d[i, j] = e
        assert abs((loss(x64 + d, w64) - loss(x64 - d, w64)) / (2 * e) - dx[i, j]) <= 2e-5
    for j in range(width):
        d = np.zeros(width)
        d[j] = e
        assert abs((loss(x64, w64 + d) - loss(x64, w64 - d)) / (2 * e) - dw[j]) <= 2e-5
