"""GPU: the operators on device buffers (mg_kv8_*, mg_token_logprobs*) against
plain 64-bit forms (tests/operators_lib.py)."""
import math

import numpy as np
import pytest

import grokking_abmod_amd as G
import operators_lib as L

pytestmark = pytest.mark.gpu


def strides_of(shape, order="sthd"):
    """Element strides (sequence, token, head) of a tensor held in `order`."""
    sizes = dict(zip("sthd", shape))
    at, out = 1, {}
    for axis in reversed(order):
        out[axis] = at
        at *= sizes[axis]
    return [out[a] for a in "sth"]


def laid_out(x, order):
    """x [s][t][h][d] in memory order `order`."""
    return np.ascontiguousarray(np.transpose(x, ["sthd".index(a) for a in order]))


def same_code_values(codes, want):
    got = L.E4M3[codes]
    return np.array_equal(got, want, equal_nan=True)


def check_append(cache, before, after, k, v, lengths, counts):
    """Every byte of the cache after an append: what it writes, and what it leaves."""
    batch, heads, cap = cache.batch, cache.heads, cache.capacity
    for which, (held, exponents) in enumerate(L.appended(cache, before, k, v, lengths, counts)):
        rows = lambda a: a[which] if which == 0 else a[1].transpose(0, 1, 2, 4, 3).reshape(cache.k.shape)  # noqa: E731
        was, now = rows(before), rows(after)
        left = np.ones((batch, heads, cap), dtype=bool)
        for (s, h, place), want in held.items():
            assert same_code_values(now[s, h, place], want), (which, s, h, place)
            left[s, h, place] = False
        assert np.array_equal(now[left], was[left]), which
        scales = before[2 + which].copy()
        for (s, h, block), e in exponents.items():
            scales[s, h, block] = e + 127
        assert np.array_equal(after[2 + which], scales), which


APPENDS = [
    # kind, width, heads, count, lengths, counts, order
    ("f32", 64, 2, 1, [1, 17, 128], None, "sthd"),
    ("f32", 32, 1, 40, [40, 61, 64], [40, 0, 13], "sthd"),
    ("bf16", 128, 2, 33, [33, 100, 128], [33, 1, 32], "sthd"),
    ("f16", 256, 1, 20, [20, 37, 64], None, "shtd"),
    ("bf16", 50, 3, 17, [17, 49, 64], [17, 16, 15], "tshd"),
    ("f32", 1, 2, 5, [5, 16, 33], [5, 4, 1], "sthd"),
    ("f16", 80, 1, 64, [64, 128, 127], [64, 64, 63], "sthd"),
    ("bf16", 200, 1, 18, [18, 35, 64], None, "sthd"),
]


@pytest.mark.parametrize("kind,width,heads,count,lengths,counts,order", APPENDS)
def test_append_writes_the_nearest_codes_and_nothing_else(kind, width, heads, count, lengths, counts, order):
    rng = np.random.default_rng(width + count)
    cache = L.Cache(len(lengths), heads, width, 128, rng)
    # Blocks that are begun hold what an append can have left: ordinary scales.
    cache.ks[:], cache.vs[:] = (rng.integers(120, 128, cache.ks.shape, dtype=np.uint8) for _ in range(2))
    shape = (len(lengths), count, heads, width)
    k, v = (L.stored(rng.normal(size=shape) * 2.0 ** rng.integers(-12, 12, (len(lengths), count, 1, 1)), kind)
            for _ in range(2))
    new = [count] * len(lengths) if counts is None else counts
    with L.Device() as dev:
        handle = cache.on(dev)
        G.kv8_append(handle, L.CODES[kind], count, dev.put(laid_out(k, order)), strides_of(shape, order),
                     dev.put(laid_out(v, order)), strides_of(shape, order), dev.put(np.array(lengths, np.int32)),
                     None if counts is None else dev.put(np.array(counts, np.int32)))
        after = cache.fetch(dev)
    check_append(cache, cache.arrays(), after, L.values(k, kind), L.values(v, kind), lengths, new)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_keys_and_values_have_their_own_strides(kind):
    """Values one element off their alignment, rows of an odd length, keys in
    another order and with one head's rows for both (stride 0)."""
    rng = np.random.default_rng(21)
    cache = L.Cache(2, 2, 64, 128, rng)
    lengths, count = np.array([37, 30], np.int32), 30
    shape = (2, count, 2, 64)
    k = np.broadcast_to(L.stored(rng.normal(size=(2, count, 1, 64)), kind), shape)
    v = L.stored(rng.normal(size=shape), kind)
    odd = np.zeros((2, count, 2, 67), v.dtype)
    odd[..., 1:65] = v
    cache.ks[:], cache.vs[:] = 120, 121
    size = odd.dtype.itemsize
    with L.Device() as dev:
        handle = cache.on(dev)
        kp, vp = dev.put(np.ascontiguousarray(k[:, :, 0])), dev.put(odd)
        at = dev.put(lengths)
        G.kv8_append(handle, L.CODES[kind], count, kp, (count * 64, 64, 0), vp + size, (count * 134, 134, 67), at)
        after = cache.fetch(dev)
        check_append(cache, cache.arrays(), after, L.values(k, kind), L.values(v, kind), lengths, [count] * 2)
        outs = [dev.put(L.stored(np.full((2, 20, 2, 67), -77.0), kind)) for _ in range(2)]
        G.kv8_read(handle, L.CODES[kind], 9, 20, outs[0], (20 * 134, 134, 67), outs[1] + size, (20 * 134, 134, 67))
        back = [L.values(dev.get(p, (2, 20, 2, 67), L.STORED[kind]), kind) for p in outs]
    for got, want, off in zip(back, cache.decoded(after), (0, 1)):
        want = L.values(L.stored(want[:, :, 9:29].transpose(0, 2, 1, 3), kind), kind)
        assert np.array_equal(got[..., off:off + 64], want, equal_nan=True)
        rest = np.delete(got, np.s_[off:off + 64], axis=3)
        assert (rest == -77.0).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("width,pitch,off", [(50, 54, 2), (51, 54, 2), (51, 64, 0), (33, 48, 8), (1, 2, 0), (130, 135, 1)])
def test_rows_of_16_bits_at_every_alignment(kind, width, pitch, off):
    """Rows on 16 bytes, on 4 and on 2, of even and odd lengths."""
    rng = np.random.default_rng(26)
    cache = L.Cache(2, 2, width, 128, rng)
    lengths, count = np.array([37, 30], np.int32), 30
    x = [L.stored(rng.normal(size=(2, count, 2, width)), kind) for _ in range(2)]
    wide = [np.zeros((2, count, 2, pitch), x[0].dtype) for _ in range(2)]
    cache.ks[:], cache.vs[:] = 120, 121
    where, st = np.s_[..., off:off + width], (count * 2 * pitch, 2 * pitch, pitch)
    with L.Device() as dev:
        handle = cache.on(dev)
        for w, y in zip(wide, x):
            w[where] = y
        kp, vp = (dev.put(np.append(w, np.zeros(off, w.dtype))) + 2 * off for w in wide)
        G.kv8_append(handle, L.CODES[kind], count, kp, st, vp, st, dev.put(lengths))
        after = cache.fetch(dev)
        check_append(cache, cache.arrays(), after, *(L.values(y, kind) for y in x), lengths, [count] * 2)
        outs = [dev.put(L.stored(np.full((2, count, 2, pitch), -77.0), kind)) for _ in range(2)]
        G.kv8_read(handle, L.CODES[kind], 0, count, outs[0] + 2 * off, st, outs[1] + 2 * off, st)
        back = [L.values(dev.get(p, (2, count, 2, pitch), L.STORED[kind]), kind) for p in outs]
    for got, want in zip(back, cache.decoded(after)):
        want = L.values(L.stored(want[:, :, :count].transpose(0, 2, 1, 3), kind), kind)
        assert np.array_equal(got[where], want, equal_nan=True)
        assert (np.delete(got, np.s_[off:off + width], axis=3) == -77.0).all()


@pytest.mark.parametrize("width", [32, 64])
def test_append_keeps_every_magnitude(width):
    """Zeros, subnormals, the largest values, infinities and NaN."""
    rng = np.random.default_rng(5)
    cache = L.Cache(8, 1, width, 64, rng)
    x = rng.normal(size=(8, 16, 1, width)).astype(np.float32)
    big = np.float32(3.4028235e38)
    x[0] = 0.0
    x[1] *= np.float32(1e-38)
    x[2] = np.where(np.abs(x[2]) > 1, np.sign(x[2]) * big, x[2])
    x[3, 4, 0, 7], x[3, 5, 0, 8], x[3, 9, 0, 1] = np.nan, np.inf, -np.inf
    x[4] = np.nan
    x[5] *= np.float32(1e-45)
    x[6] = np.float32(448.0) * np.sign(x[6])
    x[7] = np.nextafter(np.float32(448.0), np.float32(1e9))
    lengths = np.full(8, 16, np.int32)
    with L.Device() as dev:
        handle = cache.on(dev)
        p = dev.put(x)
        G.kv8_append(handle, G.MG_F32, 16, p, strides_of(x.shape), p, strides_of(x.shape), dev.put(lengths))
        after = cache.fetch(dev)
    check_append(cache, cache.arrays(), after, x.astype(np.float64), x.astype(np.float64), lengths, lengths)


@pytest.mark.parametrize("kind,width", [("f32", 64), ("bf16", 32)])
def test_tokens_one_by_one_raise_their_blocks_scale(kind, width):
    rng = np.random.default_rng(11)
    cache = L.Cache(2, 2, width, 64, rng)
    with L.Device() as dev:
        handle = cache.on(dev)
        length = np.array([0, 7], np.int32)
        cache.ks[1, :, 0] = cache.vs[1, :, 0] = 118
        handle = cache.on(dev)
        at = dev.put(length)
        before = [a.copy() for a in cache.arrays()]
        for step in range(24):
            length = length + 1
            k, v = (L.stored(rng.normal(size=(2, 1, 2, width)) * 2.0 ** (step % 11 - 4), kind) for _ in range(2))
            dev.put(length, at)
            G.kv8_append(handle, L.CODES[kind], 1, dev.put(k), strides_of(k.shape), dev.put(v), strides_of(v.shape), at)
            after = cache.fetch(dev)
            check_append(cache, before, after, L.values(k, kind), L.values(v, kind), length, [1, 1])
            before = after


def test_append_leaves_impossible_sequences():
    rng = np.random.default_rng(3)
    lengths, counts = np.array([-1, 129, 5, 20, 20, 64], np.int32), np.array([1, 1, 6, -1, 9, 8], np.int32)
    cache = L.Cache(6, 1, 64, 128, rng)
    x = rng.normal(size=(6, 8, 1, 64)).astype(np.float32)
    with L.Device() as dev:
        handle = cache.on(dev)
        p = dev.put(x)
        G.kv8_append(handle, G.MG_F32, 8, p, strides_of(x.shape), p, strides_of(x.shape), dev.put(lengths),
                     dev.put(counts))
        after = cache.fetch(dev)
    x = x.astype(np.float64)
    check_append(cache, cache.arrays(), after, x, x, [0, 0, 0, 0, 0, 64], [0, 0, 0, 0, 0, 8])


@pytest.mark.parametrize("kind,width,first,count,lengths,order", [
    ("f32", 64, 0, 128, None, "sthd"), ("f32", 32, 3, 1, None, "sthd"), ("f16", 128, 17, 100, [16, 18, 128], "shtd"),
    ("bf16", 256, 60, 9, [61, 0, 64], "sthd"), ("f32", 50, 15, 33, [20, 47, 48], "tshd"), ("bf16", 1, 0, 65, None, "sthd"),
    ("f16", 80, 64, 64, None, "sthd")])
def test_read_gives_the_values_of_the_codes(kind, width, first, count, lengths, order):
    rng = np.random.default_rng(width)
    cache = L.Cache(3, 2, width, 128, rng)
    cache.ks[:], cache.vs[:] = (rng.integers(100, 140, cache.ks.shape, dtype=np.uint8) for _ in range(2))
    shape = (3, count, 2, width)
    mark = L.stored(np.full(shape, -77.0), kind)
    with L.Device() as dev:
        handle = cache.on(dev)
        outs = [dev.put(laid_out(mark, order)) for _ in range(2)]
        G.kv8_read(handle, L.CODES[kind], first, count, outs[0], strides_of(shape, order), outs[1],
                   strides_of(shape, order), None if lengths is None else dev.put(np.array(lengths, np.int32)))
        back = [dev.get(p, [shape["sthd".index(a)] for a in order], L.STORED[kind]) for p in outs]
        assert all(np.array_equal(a, b) for a, b in zip(cache.fetch(dev), cache.arrays()))
    for got, want in zip(back, cache.decoded()):
        got = np.transpose(got, [order.index(a) for a in "sthd"])
        want = L.values(L.stored(want[:, :, first:first + count].transpose(0, 2, 1, 3), kind), kind)
        inside = np.ones((3, count), dtype=bool)
        if lengths is not None:
            inside = np.arange(first, first + count)[None] < np.array(lengths)[:, None]
        want = np.where(inside[:, :, None, None], want, -77.0)
        assert np.array_equal(L.values(got, kind), want, equal_nan=True)


@pytest.mark.parametrize("kind,batch,width,count", [("f32", 4, 100, 11000), ("f16", 8, 128, 9000)])
def test_read_of_more_than_the_caches_hold(kind, batch, width, count):
    rng = np.random.default_rng(27)
    heads, capacity, first = 8, (count + 127) // 64 * 64, 37
    cache = L.Cache(batch, heads, width, capacity, rng)
    cache.ks[:], cache.vs[:] = (rng.integers(120, 128, cache.ks.shape, dtype=np.uint8) for _ in range(2))
    shape = (batch, count, heads, width)
    size = int(np.prod(shape)) * np.dtype(L.STORED[kind]).itemsize
    assert 2 * size > 256 << 20
    with L.Device() as dev:
        handle, outs, st = cache.on(dev), [dev.alloc(size) for _ in range(2)], strides_of(shape)
        G.kv8_read(handle, L.CODES[kind], first, count, outs[0], st, outs[1], st)
        table = L.E4M3.astype(np.float32)
        for which, codes in enumerate((cache.k, cache.v.transpose(0, 1, 2, 4, 3).reshape(cache.k.shape))):
            got = dev.get(outs[which], shape, L.STORED[kind])
            scale = np.ldexp(np.float32(1), np.repeat((cache.ks, cache.vs)[which], 16, 2).astype(np.int32) - 127)
            for s in range(batch):  # exact: 4 bits times a power of two
                want = table[codes[s, :, first:first + count, :width]] * scale[s, :, first:first + count, None]
                assert np.array_equal(got[s], want.transpose(1, 0, 2).astype(got.dtype), equal_nan=True)


def filled(cache, lengths, rng, spread=4):
    """Codes and scales of ordinary tokens inside the sequences; behind them stays
    whatever was there, NaN codes and scales of every kind among it."""
    for s, n in enumerate(lengths):
        k, v = (rng.integers(0, 254, (cache.heads, n, cache.pad), dtype=np.uint8) for _ in range(2))
        k[k == 127] = 126
        v[v == 127] = 126
        k[:, :, cache.width:] = 0
        cache.k[s, :, :n] = k
        flat = cache.v[s].transpose(0, 1, 3, 2).reshape(cache.heads, cache.capacity, cache.pad).copy()
        flat[:, :n] = v
        cache.v[s] = flat.reshape(cache.heads, cache.capacity // 64, 64, cache.pad).transpose(0, 1, 3, 2)
        blocks = (n + 15) // 16
        cache.ks[s, :, :blocks] = rng.integers(117 - spread, 118, (cache.heads, blocks), dtype=np.uint8)
        cache.vs[s, :, :blocks] = rng.integers(119 - spread, 119 + spread, (cache.heads, blocks), dtype=np.uint8)


def attend(dev, handle, q, kind, lengths, counts, scale, order="sthd", stream=None, mark=-77.0):
    shape = q.shape
    out = dev.put(laid_out(L.stored(np.full(shape, mark), kind), order))
    room = G.kv8_attention_workspace(handle, shape[2], shape[1])
    G.kv8_attention(handle, L.CODES[kind], shape[2], shape[1], dev.put(laid_out(q, order)), strides_of(shape, order), out,
                    strides_of(shape, order), dev.put(np.array(lengths, np.int32)),
                    None if counts is None else dev.put(np.array(counts, np.int32)), scale,
                    dev.alloc(room) if room else None, room, stream)
    got = dev.get(out, [shape["sthd".index(a)] for a in order], L.STORED[kind])
    return L.values(np.transpose(got, [order.index(a) for a in "sthd"]), kind)


def check_attention(got, q, kind, cache, lengths, counts, scale, mark=-77.0):
    k, v = cache.decoded()
    with np.errstate(invalid="ignore"):
        want, size, mass, far = L.attention(L.values(q, kind), k, v, lengths, counts, scale)
    limit = L.attention_tolerance(kind, want, size, mass, far, cache.width, max(lengths))
    for s, n in enumerate(counts):
        assert (got[s, n:] == mark).all(), s  # rows behind the sequence's own
        g, w, t = got[s, :n], want[s, :n], limit[s, :n]
        assert np.array_equal(np.isnan(g), np.isnan(w)), s
        bad = np.abs(g - w) > t
        assert not bad.any(), (s, bad.sum(), np.nanmax(np.abs(g - w) / t))


ATTENTIONS = [
    # kind, width, heads, kv_heads, capacity, count, lengths, counts, order
    ("f32", 64, 2, 2, 192, 1, [1, 2, 15, 16, 17, 63, 64, 65, 192], None, "sthd"),
    ("f32", 32, 4, 2, 576, 1, [1, 64, 257, 576], None, "sthd"),
    ("bf16", 128, 8, 2, 1024, 1, [1, 129, 1000, 1024], None, "sthd"),
    ("f16", 256, 2, 1, 320, 1, [1, 250, 320], None, "shtd"),
    ("bf16", 50, 3, 3, 128, 1, [1, 49, 128], None, "sthd"),
    ("f32", 1, 2, 1, 64, 1, [1, 64], None, "sthd"),
    ("f16", 64, 16, 1, 128, 1, [3, 128], None, "sthd"),
    ("bf16", 64, 24, 1, 128, 1, [3, 128], None, "sthd"),  # more rows than one tile
    ("f32", 64, 2, 2, 128, 3, [3, 70, 128], [3, 1, 0], "sthd"),
    ("f32", 64, 2, 2, 192, 65, [65, 129, 192, 100], [65, 64, 17, 1], "sthd"),
    ("bf16", 128, 4, 2, 320, 150, [150, 320, 200], [150, 149, 33], "shtd"),
    ("f16", 80, 2, 2, 256, 130, [130, 256], None, "tshd"),
    ("bf16", 256, 2, 1, 192, 70, [70, 192, 180], [70, 69, 68], "sthd"),
    ("f32", 256, 1, 1, 128, 40, [40, 128], None, "sthd"),
    ("f32", 128, 2, 1, 256, 100, [100, 256], [100, 77], "sthd"),
    ("bf16", 32, 2, 2, 640, 300, [300, 640], None, "sthd"),
    ("f16", 31, 1, 1, 64, 20, [20, 64, 50], [20, 19, 1], "sthd"),
    ("bf16", 64, 1, 1, 2048, 1, [2048], None, "sthd"),  # one pair, keys in shares
    ("f32", 64, 4, 1, 2048, 30, [2048, 70], None, "sthd"),  # several tiles of 16 rows, keys in shares
    ("bf16", 128, 4, 1, 1088, 30, [1088, 300], [30, 11], "sthd"),
    ("f16", 32, 1, 1, 1024, 64, [1024, 64], [64, 63], "sthd"),
    ("f32", 64, 1, 1, 1024, 30, [1024, 33], [30, 30], "sthd"),
    ("bf16", 64, 4, 1, 2048, 200, [2048, 300, 200], [200, 150, 200], "sthd"),  # tiles of 128 rows, keys in shares
    ("f32", 256, 1, 1, 1024, 140, [1024, 200, 0], [140, 129, 0], "sthd"),
    ("f16", 128, 1, 1, 1024, 400, [1000, 500], None, "shtd"),
]


@pytest.mark.parametrize("kind,width,heads,kv_heads,capacity,count,lengths,counts,order", ATTENTIONS)
def test_attention_matches_64_bits(kind, width, heads, kv_heads, capacity, count, lengths, counts, order):
    rng = np.random.default_rng(width * 7 + count)
    cache = L.Cache(len(lengths), kv_heads, width, capacity, rng)
    filled(cache, lengths, rng)
    q = L.stored(rng.normal(size=(len(lengths), count, heads, width)), kind)
    scale = 1.0 / math.sqrt(width)
    with L.Device() as dev:
        got = attend(dev, cache.on(dev), q, kind, lengths, counts, scale, order)
    check_attention(got, q, kind, cache, lengths, [count] * len(lengths) if counts is None else counts, scale)


@pytest.mark.parametrize("kind,count", [("f32", 1), ("f32", 50), ("bf16", 50)])
def test_what_a_row_does_not_see_has_no_effect(kind, count):
    """NaN keys, values and scales at the last token: only its own row sees them;
    NaN and infinite queries: only their own rows."""
    rng = np.random.default_rng(8)
    n, width = 90, 64
    cache = L.Cache(3, 1, width, 128, rng)
    filled(cache, [n] * 3, rng)
    cache.k[0, 0, n - 1, 3] = 127
    cache.v[1, 0, (n - 1) // 64, 5, (n - 1) % 64] = 255
    q = rng.normal(size=(3, count, 1, width)).astype(np.float32)
    q[2, 0, 0, 9] = np.inf
    q = L.stored(q, kind)
    with L.Device() as dev:
        got = attend(dev, cache.on(dev), q, kind, [n] * 3, None, 0.125)
    assert np.isnan(got[0, -1]).all() and np.isnan(got[1, -1, 0, 5]) and np.isnan(got[1, -1]).sum() == 1
    assert np.isnan(got[2, 0]).all()
    keep = np.ones((3, count), dtype=bool)
    keep[0, -1] = keep[1, -1] = keep[2, 0] = False
    cache.k[0, 0, n - 1, 3] = cache.v[1, 0, (n - 1) // 64, 5, (n - 1) % 64] = 0
    plain = q.copy()
    plain[2, 0] = 0
    k, v = cache.decoded()
    want, size, mass, far = L.attention(L.values(plain, kind), k, v, [n] * 3, [count] * 3, 0.125)
    limit = L.attention_tolerance(kind, want, size, mass, far, width, n)
    assert (np.abs(got - want) <= limit)[keep].all()


def test_attention_of_impossible_sequences_is_nan():
    rng = np.random.default_rng(2)
    for count, capacity in ((1, 128), (3, 128), (40, 128), (100, 128), (1, 2048), (3, 2048), (200, 1024)):
        lengths, counts = [-1, capacity + 1, count - 1, count + 60], [1, 1, count, count]
        cache = L.Cache(4, 1, 64, capacity, rng)
        lengths[3] = min(lengths[3], capacity)
        filled(cache, [0, 0, 0, lengths[3]], rng)
        q = rng.normal(size=(4, count, 2, 64)).astype(np.float32)
        with L.Device() as dev:
            got = attend(dev, cache.on(dev), q, "f32", lengths, counts, 0.125)
        assert np.isnan(got[:3]).all() and np.isfinite(got[3]).all(), count


@pytest.mark.parametrize("kind,count", [("f32", 1), ("bf16", 40), ("f16", 40)])
def test_attention_rows_off_their_alignment(kind, count):
    rng = np.random.default_rng(31)
    lengths, width = [70, 128], 64
    cache = L.Cache(2, 1, width, 128, rng)
    filled(cache, lengths, rng)
    q = L.stored(rng.normal(size=(2, count, 2, width)), kind)
    wide = np.zeros((2, count, 2, 67), q.dtype)
    wide[..., 1:65] = q
    size, strides = q.dtype.itemsize, (count * 134, 134, 67)
    with L.Device() as dev:
        handle = cache.on(dev)
        p = dev.put(wide)
        room = G.kv8_attention_workspace(handle, 2, count)
        G.kv8_attention(handle, L.CODES[kind], 2, count, p + size, strides, p + size, strides,  # in place
                        dev.put(np.array(lengths, np.int32)), None, 0.125, dev.alloc(room) if room else None, room)
        got = L.values(dev.get(p, wide.shape, wide.dtype), kind)
    assert (got[..., 0] == 0).all() and (got[..., 65:] == 0).all()
    check_attention(got[..., 1:65], q, kind, cache, lengths, [count] * 2, 0.125)


@pytest.mark.parametrize("kind,count,capacity", [("f32", 1, 128), ("bf16", 1, 2048), ("f16", 70, 128), ("f32", 140, 2048)])
def test_attention_over_its_queries(kind, count, capacity):
    """The output in the queries' place is that of one beside them."""
    rng = np.random.default_rng(23)
    lengths = [capacity, max(count, capacity - 77)]
    cache = L.Cache(2, 2, 64, capacity, rng)
    filled(cache, lengths, rng)
    q = L.stored(rng.normal(size=(2, count, 4, 64)), kind)
    with L.Device() as dev:
        handle, st = cache.on(dev), strides_of(q.shape)
        beside = attend(dev, handle, q, kind, lengths, None, 0.125)
        room, at = G.kv8_attention_workspace(handle, 4, count), dev.put(q)
        G.kv8_attention(handle, L.CODES[kind], 4, count, at, st, at, st, dev.put(np.array(lengths, np.int32)), None, 0.125,
                        dev.alloc(room) if room else None, room)
        assert np.array_equal(L.values(dev.get(at, q.shape, L.STORED[kind]), kind), beside)


def test_queries_that_heads_and_tokens_share():
    """Strides of 0 for heads and tokens: one query a sequence."""
    rng = np.random.default_rng(24)
    cache = L.Cache(2, 2, 64, 192, rng)
    filled(cache, [192, 100], rng)
    q = rng.normal(size=(2, 1, 1, 64)).astype(np.float32)
    with L.Device() as dev:
        handle, n = cache.on(dev), dev.put(np.array([192, 100], np.int32))
        whole = np.ascontiguousarray(np.broadcast_to(q, (2, 20, 4, 64)))
        want = attend(dev, handle, whole, "f32", [192, 100], None, 0.125)
        out = dev.alloc(whole.nbytes)
        G.kv8_attention(handle, G.MG_F32, 4, 20, dev.put(q), (64, 0, 0), out, strides_of(whole.shape), n, None, 0.125)
        assert np.array_equal(dev.get(out, whole.shape, np.float32), want)


def test_values_of_very_different_scales():
    """Blocks 2^200 apart: a block's scale meets its own probabilities."""
    rng = np.random.default_rng(4)
    for kind in ("f32", "bf16"):
        cache = L.Cache(2, 1, 64, 128, rng)
        filled(cache, [128, 100], rng)
        cache.vs[:, 0] = np.array([20, 220, 20, 60, 90, 127, 150, 20], np.uint8)
        cache.k[:, :, 16:32] = 0  # weights of the large block: those of score 0
        q = L.stored(rng.normal(size=(2, 30, 1, 64)), kind)
        with L.Device() as dev:
            got = attend(dev, cache.on(dev), q, kind, [128, 100], None, 0.125)
        check_attention(got, q, kind, cache, [128, 100], [30, 30], 0.125)


# ---- log probabilities ---------------------------------------------------------------

@pytest.mark.parametrize("kind,count", [("f32", 1), ("bf16", 40)])
def test_a_cache_of_more_than_4_gib(kind, count):
    """Two sequences of 2^24 tokens of width 256, all of them zeros but the last."""
    capacity, width = 1 << 24, 256
    rng = np.random.default_rng(21)
    new = [L.stored(rng.normal(size=(2, count, 1, width)), kind) for _ in range(2)]
    q = L.stored(rng.normal(size=(2, count, 1, width)) * 6, kind)
    at = [capacity, capacity - 70]
    with L.Device() as dev:
        codes, scales = 2 * capacity * width, 2 * capacity // 16
        handle = G.Kv8(2, 1, width, capacity, dev.filled(codes, 0), dev.filled(codes, 0), dev.filled(scales, 60),
                       dev.filled(scales, 60))
        st = strides_of(new[0].shape)
        G.kv8_append(handle, L.CODES[kind], count, dev.put(new[0]), st, dev.put(new[1]), st,
                     dev.put(np.array(at, np.int32)), None, None)
        tail = [dev.put(np.full((2, 128, 1, width), 9, np.float32)) for _ in range(2)]
        st = strides_of((2, 128, 1, width))
        G.kv8_read(handle, G.MG_F32, capacity - 128, 128, tail[0], st, tail[1], st, None, None)
        k, v = (dev.get(p, (2, 128, width), np.float32).astype(np.float64) for p in tail)
        got = attend(dev, handle, q, kind, at, None, 1 / 16)
    qd = L.values(q, kind)[:, :, 0]
    for s in range(2):
        end = at[s] - (capacity - 128)
        assert not k[s, :end - count].any() and not v[s, :end - count].any() and not v[s, end:].any()
        for i in range(2):
            want = L.values(new[i], kind)[s, :, 0]
            # A block's scale is at most 2^-8 of its largest magnitude, rounded up
            # to a power of two; a code is off by 2^-4 of it or 2^-10 scales.
            assert (np.abs((k, v)[i][s, end - count:end] - want) <= np.abs(want) / 16 + np.abs(want).max() * 2.0**-17).all()
        for i in range(count):
            last = end - count + i + 1
            x = k[s, :last] @ qd[s, i] / 16
            e = np.exp(x)
            total = at[s] - count + i + 1 - last + e.sum()
            want, size = e @ v[s, :last] / total, e @ np.abs(v[s, :last]) / total
            # 256 shares of up to 256 tiles a wave, a rounding of the sums in each,
            # three in a share's joining: 1024 half steps and some.  A score has 256
            # terms, and its error counts in the numerator and in the sum.  BF16
            # calls round each probability by 2^-9 and the output by 2^-8.
            score = (np.abs(k[s, :last]) @ np.abs(qd[s, i])).max() / 16
            limit = size * (1200 + 600 * score) * 2.0**-24 + (0 if kind == "f32" else (size + np.abs(want)) / 256)
            assert (np.abs(got[s, i, 0] - want) <= limit + 2.0**-126).all()


def test_calls_on_two_streams_at_once():
    """Each with a workspace of its own gives what it gives alone."""
    rng = np.random.default_rng(22)
    cases = []
    with L.Device() as dev:
        for i, (batch, count, rows) in enumerate(((2, 1, 3), (1, 70, 5))):
            cache = L.Cache(batch, 2, 64, 4096, rng)
            lengths = [4096 - 100 * s - i for s in range(batch)]
            filled(cache, lengths, rng)
            q = L.stored(rng.normal(size=(batch, count, 4, 64)), "bf16")
            z = rng.normal(size=(rows, 40000)).astype(np.float32)
            handle, stream, st = cache.on(dev), dev.stream(), strides_of(q.shape)
            room, more = G.kv8_attention_workspace(handle, 4, count), G.token_logprobs_workspace(rows, 40000, 5)
            assert room and more
            p = dict(q=dev.put(q), n=dev.put(np.array(lengths, np.int32)), out=dev.alloc(q.nbytes), space=dev.alloc(room),
                     z=dev.put(z), t=dev.put(np.arange(rows, dtype=np.uint32)), lp=dev.alloc(4 * rows),
                     h=dev.alloc(4 * rows), ids=dev.alloc(20 * rows), best=dev.alloc(20 * rows), more=dev.alloc(more))

            def run(p=p, handle=handle, stream=stream, st=st, count=count, rows=rows, room=room, more=more):
                G.kv8_attention(handle, G.MG_BF16, 4, count, p["q"], st, p["out"], st, p["n"], None, 0.125, p["space"],
                                room, stream)
                G.token_logprobs_noalloc(G.MG_F32, p["z"], rows, 40000, 40000, p["t"], 1.0, p["lp"], p["h"], None, 5,
                                         p["ids"], p["best"], p["more"], more, stream)

            def results(p=p, q=q, rows=rows):
                return [dev.get(p["out"], q.shape, np.uint16)] + [dev.get(p[n], w * rows, np.uint32)
                                                                 for n, w in (("lp", 1), ("h", 1), ("ids", 5), ("best", 5))]
            run()
            cases.append((run, results, results()))
        for _ in range(20):
            for run, _, _ in cases:
                run()
        for _, results, alone in cases:
            for a, b in zip(results(), alone):
                assert np.array_equal(a, b)


def score(dev, z, kind, tokens, temperature, top, stride=None, stream=None):
    rows, vocab = z.shape
    stride = vocab if stride is None else stride
    wide = np.zeros((rows, stride), dtype=z.dtype)
    wide[:, :vocab] = z
    out = [dev.put(np.full(n * rows, -7.0, np.float32)) for n in (1, 1, 2)]
    ids, best = dev.put(np.full(rows * top, 9, np.uint32)), dev.put(np.full(rows * top, -7.0, np.float32))
    room = G.token_logprobs_workspace(rows, vocab, top)
    zp = dev.put(wide)
    G.token_logprobs_noalloc(L.CODES[kind], zp, rows, vocab, stride, dev.put(np.asarray(tokens, np.uint32)), temperature,
                             *out, top, ids if top else None, best if top else None, dev.alloc(room) if room else None,
                             room, stream)
    lp, h, stats = (dev.get(p, s, np.float32) for p, s in zip(out, (rows, rows, (rows, 2))))
    return lp, h, stats, dev.get(ids, (rows, top), np.uint32), dev.get(best, (rows, top), np.float32), zp, out


def check_scores(z64, tokens, temperature, top, lp, h, ids, best):
    want = L.logprobs(z64, tokens, temperature, top)
    vocab = z64.shape[1]
    assert np.array_equal(ids, want[2])
    with np.errstate(invalid="ignore"):
        spread = (z64.max(1) - z64.min(1, initial=np.inf, where=z64 > -np.inf)) / temperature
    spread = np.where(np.isfinite(spread), spread, 0)
    # The sum of `vocab` exponentials: the largest share of a thread and the join
    # are 128 + 32 additions, each exponential's argument is off by 2 roundings of
    # up to `spread` log2 units (those far down weigh nothing: 24 of them at most).
    step = 2.0**-24
    of_sum = (160 + 3 * np.minimum(spread * 1.5, 24) + 8) * step
    # The entropy's second sum has terms e^d |d|, together at most e^-1 a token or
    # S times the entropy and the log of S.
    log_s = math.log(vocab + 1)
    for got, w, limit in ((lp, want[0], of_sum + 4 * step * np.abs(np.where(np.isfinite(want[0]), want[0], 0))),
                          (h, want[1], of_sum * (1 + 2 * log_s) + 8 * step * (1 + log_s))):
        same = np.isfinite(w)
        assert np.array_equal(got[~same], w[~same].astype(np.float32), equal_nan=True)
        assert (np.abs(got[same] - w[same]) <= limit[same]).all(), np.max(np.abs(got[same] - w[same]) / limit[same])
    if top:
        same = np.isfinite(want[3])
        assert np.array_equal(best[~same], want[3][~same].astype(np.float32), equal_nan=True)
        limit = of_sum[:, None] + 4 * step * np.abs(np.where(same, want[3], 0))
        assert (np.abs(best[same] - want[3][same]) <= limit[same]).all()


SCORES = [
    # kind, rows, vocab, stride, temperature, top
    ("f32", 5, 1, 1, 1.0, 1), ("f32", 3, 2, 3, 0.5, 2), ("f32", 70, 256, 256, 0.8, 5), ("bf16", 9, 99, 101, 1.0, 32),
    ("f16", 4, 1000, 1000, 1.5, 20), ("f32", 4, 1025, 1025, 1.0, 32), ("bf16", 3, 5003, 5003, 1.0, 20),
    ("f16", 2, 50257, 50264, 0.7, 5), ("f32", 1, 131072, 131072, 1.0, 32), ("bf16", 3, 131071, 131073, 2.0, 1),
    ("f32", 2, 1000003, 1000003, 1.0, 32), ("bf16", 1, 1 << 24, 1 << 24, 1.0, 32), ("f16", 12, 200000, 200000, 1.0, 20),
    ("f32", 600, 4099, 4099, 1.0, 3), ("bf16", 1030, 2051, 2051, 1.0, 0), ("f32", 2, 64, 64, 1.0, 0)]


@pytest.mark.parametrize("kind,rows,vocab,stride,temperature,top", SCORES)
def test_log_probabilities_match_64_bits(kind, rows, vocab, stride, temperature, top):
    rng = np.random.default_rng(vocab)
    z = L.stored(rng.normal(size=(rows, vocab)) * 3, kind)
    tokens = rng.integers(0, vocab, rows).astype(np.uint32)
    if rows > 3:
        tokens[1], tokens[2] = G.IGNORE_TARGET, vocab
    with L.Device() as dev:
        lp, h, stats, ids, best, *_ = score(dev, z, kind, tokens, temperature, top, stride)
    z64 = L.values(z, kind)
    check_scores(z64, tokens, temperature, top, lp, h, ids, best)
    assert np.array_equal(stats[:, 0], z64.max(1).astype(np.float32))


def test_temperatures_from_the_smallest_to_the_largest():
    rng = np.random.default_rng(12)
    z = rng.normal(size=(6, 1500)).astype(np.float32)
    tokens = z.argmax(1).astype(np.uint32)
    for temperature in (1e-38, 1e-3, 1e3, 1e38):
        t = float(np.float32(temperature))
        with L.Device() as dev:
            lp, h, _, ids, best, *_ = score(dev, z, "f32", tokens, t, 3)
        with np.errstate(over="ignore"):
            check_scores(z.astype(np.float64), tokens, 1 / float(np.float32(1) / np.float32(t)), 3, lp, h, ids, best)


@pytest.mark.parametrize("vocab", [70, 1000, 6000, 40000])
def test_log_probabilities_of_masked_and_odd_rows(vocab):
    rng = np.random.default_rng(vocab)
    low = np.float32(-3.4028235e38)
    z = (rng.normal(size=(14, vocab)) * 2).astype(np.float32)
    z[0] = -np.inf
    z[1] = low
    z[2] = 0.0
    z[3, 5:] = -np.inf
    z[4, 5:] = low
    z[5] = np.where(np.arange(vocab) % 2, -0.0, 0.0)
    z[6, vocab // 2] = np.nan
    z[7, vocab - 1] = np.inf
    z[8] = np.arange(vocab) / vocab
    z[9] = -np.arange(vocab) / vocab
    z[10] = np.round(z[10])  # ties
    z[11, :-3] = -np.inf
    z[12] = 3e38
    z[13, 0] = 100.0
    tokens = np.full(14, 2, np.uint32)
    tokens[11] = vocab - 1
    for top in (0, 7, 32):
        with L.Device() as dev:
            lp, h, stats, ids, best, *_ = score(dev, z, "f32", tokens, 1.0, top)
        check_scores(z.astype(np.float64), tokens, 1.0, top, lp, h, ids, best)
        assert stats[0, 0] == -np.inf and np.isnan(stats[6]).all()


GRADIENTS = [("f32", 5, 1, 1, 1.0), ("f32", 70, 99, 99, 0.8), ("bf16", 9, 1001, 1003, 1.0), ("f16", 4, 1024, 1024, 1.5),
             ("f32", 3, 1025, 1027, 1.0), ("bf16", 3, 40001, 40001, 1.0), ("f16", 2, 33000, 33008, 0.7),
             # about the ends of a wave's share, rows off their lines by any amount
             ("f32", 40, 736, 737, 1.0), ("f32", 40, 737, 737, 1.0), ("f32", 40, 1473, 1475, 1.0),
             ("bf16", 70, 1472, 1473, 1.0), ("bf16", 70, 1473, 1473, 1.0), ("f16", 70, 2945, 2951, 1.0)]


@pytest.mark.parametrize("kind,rows,vocab,stride,temperature", GRADIENTS)
@pytest.mark.parametrize("which", ["both", "logprob", "entropy", "in place", "apart"])
def test_the_gradient_matches_64_bits(kind, rows, vocab, stride, temperature, which):
    rng = np.random.default_rng(vocab + rows)
    z = rng.normal(size=(rows, vocab)) * 3
    if rows > 2 and vocab > 10:
        z[0, ::3] = -np.inf
        z[1] = -np.inf
    z = L.stored(z, kind)
    tokens = rng.integers(0, vocab, rows).astype(np.uint32)
    tokens[-1] = G.IGNORE_TARGET
    g, e = rng.normal(size=rows).astype(np.float32), rng.normal(size=rows).astype(np.float32)
    z64 = L.values(z, kind)
    with L.Device() as dev:
        lp, h, stats, _, _, zp, (_, hp, sp) = score(dev, z, kind, tokens, temperature, 0, stride)
        # Apart: the gradient has a stride and an alignment of its own.
        wide, off = (stride + 3, 1) if which == "apart" else (stride, 0)
        out = zp if which == "in place" else dev.put(L.stored(np.full(rows * wide + off, -77.0), kind))
        G.token_logprobs_backward_noalloc(L.CODES[kind], zp, rows, vocab, stride, dev.put(tokens), temperature, sp,
                                          hp if which != "logprob" else None, dev.put(g) if which != "entropy" else None,
                                          dev.put(e) if which != "logprob" else None, out + off * z.itemsize, wide)
        got = L.values(dev.get(out, rows * wide + off, L.STORED[kind]), kind)
    assert which == "in place" or (got[:off] == -77.0).all()
    got = got[off:].reshape(rows, wide)
    if which != "in place":
        assert (got[:, vocab:] == -77.0).all()
    gg, ee = g * (which != "entropy"), e * (which != "logprob")
    with np.errstate(invalid="ignore"):
        want = L.logprob_gradient(z64, tokens, temperature, gg, ee)
        logp = np.where(np.isfinite(z64), (z64 - z64.max(1, keepdims=True)) / temperature, 0)
    logp = np.nan_to_num(logp)
    size = np.exp(logp) * (np.abs(gg)[:, None] + np.abs(ee)[:, None] * (np.abs(logp) + 2 * math.log(vocab + 1)))
    # p is off by the roundings of its exponent (|log p| up to 24 before it weighs
    # nothing) and of the sum; the terms by a few roundings each.
    relative = (8 * 40 + 200) * 2.0**-24
    least = {"f32": 2.0**-126, "f16": 2.0**-25, "bf16": 2.0**-126}[kind]
    limit = (relative * size + 4 * 2.0**-24 * np.abs(gg)[:, None]) / temperature + L.HALF_STEP[kind] * np.abs(want) * 1.01 + least
    assert (np.abs(got[:, :vocab] - want) <= limit).all(), np.max(np.abs(got[:, :vocab] - want) / limit)


def test_the_gradient_of_more_than_the_caches_hold():
    """The same rows again and again, beside those of a small call."""
    rng = np.random.default_rng(28)
    rows, vocab, times = 8, 50257, 340
    assert rows * times * vocab * 2 > 256 << 20
    z = L.stored(rng.normal(size=(rows, vocab)) * 3, "bf16")
    t = rng.integers(0, vocab, rows).astype(np.uint32)
    g, e = (rng.normal(size=rows).astype(np.float32) for _ in range(2))
    with L.Device() as dev:
        *_, zp, (_, hp, sp) = score(dev, z, "bf16", t, 1.0, 0)
        out = dev.alloc(z.nbytes)
        G.token_logprobs_backward_noalloc(G.MG_BF16, zp, rows, vocab, vocab, dev.put(t), 1.0, sp, hp, dev.put(g), dev.put(e),
                                          out, vocab)
        want, h, stats = dev.get(out, z.shape, np.uint16), dev.get(hp, rows, np.float32), dev.get(sp, (rows, 2), np.float32)
        many = dev.put(np.tile(z, (times, 1)))
        G.token_logprobs_backward_noalloc(G.MG_BF16, many, rows * times, vocab, vocab, dev.put(np.tile(t, times)), 1.0,
                                          dev.put(np.tile(stats, (times, 1))), dev.put(np.tile(h, times)),
                                          dev.put(np.tile(g, times)), dev.put(np.tile(e, times)), many, vocab)
        got = dev.get(many, (times, rows, vocab), np.uint16)
    assert (got == want).all()


def test_the_gradient_is_that_of_the_forward_pass():
    """Differences of the forward kernel's own log probability and entropy."""
    rng = np.random.default_rng(1)
    vocab, step = 12, 2.0**-6
    z = rng.normal(size=(1, vocab)).astype(np.float32)
    z = np.round(z * 256) / 256  # z +- step is exact
    rows = np.repeat(z, 2 * vocab + 1, 0).astype(np.float32)
    for v in range(vocab):
        rows[2 * v, v] += step
        rows[2 * v + 1, v] -= step
    tokens = np.full(2 * vocab + 1, 4, np.uint32)
    one = np.ones(2 * vocab + 1, np.float32)
    with L.Device() as dev:
        for which in (0, 1):
            lp, h, _, _, _, zp, (_, hp, sp) = score(dev, rows, "f32", tokens, 1.0, 0)
            out = dev.alloc(rows.nbytes)
            G.token_logprobs_backward_noalloc(G.MG_F32, zp, len(rows), vocab, vocab, dev.put(tokens), 1.0, sp, hp,
                                              dev.put(one) if which == 0 else None, dev.put(one) if which else None, out,
                                              vocab)
            got = dev.get(out, rows.shape, np.float32)[-1]
            f = (lp if which == 0 else h).astype(np.float64)
            slope = (f[0:-1:2] - f[1:-1:2]) / (2 * step)
            # A third derivative of at most 4 times step^2 / 6, and two values of
            # size 4 off by 40 roundings over 2 step.
            limit = 4 * step**2 / 6 + 2 * 4 * 40 * 2.0**-24 / (2 * step)
            assert np.abs(got - slope).max() <= limit


def test_a_scored_step_and_its_gradient_as_a_graph():
    """Rows in several chunks, replayed with new logits in the same buffers, with
    eager calls of other data between the replays."""
    rng = np.random.default_rng(25)
    rows, vocab = 6, 30000
    t = rng.integers(0, vocab, rows).astype(np.uint32)
    g, gh = (rng.normal(size=rows).astype(np.float32) for _ in range(2))
    with L.Device() as dev:
        stream = dev.stream()
        room = G.token_logprobs_workspace(rows, vocab, 4)
        assert room
        zp, dz, tp, gp, ghp = dev.alloc(4 * rows * vocab), dev.alloc(4 * rows * vocab), dev.put(t), dev.put(g), dev.put(gh)
        lp, h, st, ids, best, space = (dev.alloc(n) for n in (4 * rows, 4 * rows, 8 * rows, 16 * rows, 16 * rows, room))

        def enqueue(on=stream, z=zp, more=space):
            G.token_logprobs_noalloc(G.MG_F32, z, rows, vocab, vocab, tp, 0.9, lp, h, st, 4, ids, best, more, room, on)
            G.token_logprobs_backward_noalloc(G.MG_F32, z, rows, vocab, vocab, tp, 0.9, st, h, gp, ghp, dz, vocab, on)

        def results():
            return [dev.get(p, n, np.uint32) for p, n in ((lp, rows), (h, rows), (st, 2 * rows), (ids, 4 * rows),
                                                         (best, 4 * rows), (dz, rows * vocab))]
        step = dev.graph(stream, enqueue)
        other, spare = dev.put(rng.normal(size=(rows, vocab)).astype(np.float32)), dev.alloc(room)
        for i in range(4):
            z = (rng.normal(size=(rows, vocab)) * (1 + i)).astype(np.float32)
            dev.put(z, zp)
            dev.replay(step, stream)
            replayed = results()
            enqueue(None, other, spare)
            enqueue(None)
            for a, b in zip(replayed, results()):
                assert np.array_equal(a, b), i


def test_host_arrays_give_the_same():
    rng = np.random.default_rng(6)
    z = (rng.normal(size=(37, 300)) * 2).astype(np.float32)
    tokens = rng.integers(0, 300, 37).astype(np.uint32)
    tokens[3] = G.IGNORE_TARGET
    lp, h, ids, best = G.token_logprobs(z, tokens, temperature=0.9, top=4)
    check_scores(z.astype(np.float64), tokens, 0.9, 4, lp, h, ids, best)
    with pytest.raises(G.MeshGptError, match="outside the vocabulary"):
        G.token_logprobs(z, np.full(37, 300, np.uint32))


# ---- together ---------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_a_serving_step_as_a_graph(kind):
    """A prompt, then steps of one token: append, attend, score the output's
    projection; captured once on a stream of its own and replayed with new inputs,
    each replay against the plain forms on the cache it left."""
    rng = np.random.default_rng(9)
    batch, heads, kv_heads, width, capacity, vocab, prompt = 3, 4, 2, 64, 2048, 300, 21
    cache = L.Cache(batch, kv_heads, width, capacity, rng)
    lengths = np.array([21, 5, 14], np.int32)
    scale = 0.125
    with L.Device() as dev:
        handle = cache.on(dev)
        stream = dev.stream()
        k, v = (L.stored(rng.normal(size=(batch, prompt, kv_heads, width)), kind) for _ in range(2))
        at, counts = dev.put(lengths), dev.put(lengths)
        G.kv8_append(handle, L.CODES[kind], prompt, dev.put(k), strides_of(k.shape), dev.put(v), strides_of(v.shape), at,
                     counts, stream)
        assert dev.hip.hipStreamSynchronize(stream) == 0
        q1, k1 = (batch, 1, heads, width), (batch, 1, kv_heads, width)
        size = np.dtype(L.STORED[kind]).itemsize
        qp, op, kp, vp = (dev.alloc(size * math.prod(s)) for s in (q1, q1, k1, k1))
        room = G.kv8_attention_workspace(handle, heads, 1)
        assert room > 0
        space = dev.alloc(room)
        zp, tp = dev.alloc(4 * batch * vocab), dev.put(np.zeros(batch, np.uint32))
        lp, hp, ip, bp = dev.alloc(4 * batch), dev.alloc(4 * batch), dev.alloc(4 * batch * 3), dev.alloc(4 * batch * 3)

        def enqueue():
            G.kv8_append(handle, L.CODES[kind], 1, kp, strides_of(k1), vp, strides_of(k1), at, None, stream)
            G.kv8_attention(handle, L.CODES[kind], heads, 1, qp, strides_of(q1), op, strides_of(q1), at, None, scale,
                            space, room, stream)
            G.token_logprobs_noalloc(G.MG_F32, zp, batch, vocab, vocab, tp, 1.0, lp, hp, None, 3, ip, bp, stream=stream)

        step = dev.graph(stream, enqueue)
        before = cache.fetch(dev)
        for _ in range(5):
            lengths = lengths + 1
            q, k, v = (L.stored(rng.normal(size=s), kind) for s in (q1, k1, k1))
            z, t = (rng.normal(size=(batch, vocab))).astype(np.float32), rng.integers(0, vocab, batch).astype(np.uint32)
            for a, p in ((q, qp), (k, kp), (v, vp), (lengths, at), (z, zp), (t, tp)):
                dev.put(a, p)
            dev.replay(step, stream)
            after = cache.fetch(dev)
            check_append(cache, before, after, L.values(k, kind), L.values(v, kind), lengths, [1] * batch)
            got = L.values(dev.get(op, q1, L.STORED[kind]), kind)
            now = L.Cache.__new__(L.Cache)
            now.__dict__.update(cache.__dict__)
            now.k, now.v, now.ks, now.vs = after
            check_attention(got, q, kind, now, lengths, [1] * batch, scale)
            check_scores(z.astype(np.float64), t, 1.0, 3, dev.get(lp, batch, np.float32), dev.get(hp, batch, np.float32),
                         dev.get(ip, (batch, 3), np.uint32), dev.get(bp, (batch, 3), np.float32))
            before = after
