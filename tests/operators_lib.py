"""Plain 64-bit forms of the device operators (include/meshgpt.h: mg_kv8_*,
mg_token_logprobs*) on numpy arrays, and device buffers to call them with."""
import ctypes
import math

import numpy as np

import grokking_abmod_amd as G

BLOCK, TILE = 16, 64


class Device:
    """Device memory, streams and graphs for the caller's side of the operators."""

    def __init__(self):
        vp, sz, i = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int
        self.hip = hip = ctypes.CDLL("libamdhip64.so")
        for name, args in dict(hipMalloc=[ctypes.POINTER(vp), sz], hipFree=[vp], hipMemcpy=[vp, vp, sz, i], hipMemset=[vp, i, sz],
                               hipDeviceSynchronize=[], hipGetDevice=[ctypes.POINTER(i)],
                               hipStreamCreate=[ctypes.POINTER(vp)], hipStreamDestroy=[vp], hipStreamSynchronize=[vp],
                               hipStreamBeginCapture=[vp, i], hipStreamEndCapture=[vp, ctypes.POINTER(vp)],
                               hipGraphInstantiate=[ctypes.POINTER(vp), vp, vp, vp, sz], hipGraphLaunch=[vp, vp],
                               hipGraphExecDestroy=[vp], hipGraphDestroy=[vp]).items():
            getattr(hip, name).argtypes = args
        self.blocks = []
        self.streams, self.graphs, self.execs = [], [], []

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.hip.hipDeviceSynchronize()
        for e in self.execs:
            self.hip.hipGraphExecDestroy(e)
        for g in self.graphs:
            self.hip.hipGraphDestroy(g)
        for s in self.streams:
            self.hip.hipStreamDestroy(s)
        for p in self.blocks:
            self.hip.hipFree(p)

    def alloc(self, nbytes):
        p = ctypes.c_void_p()
        assert self.hip.hipMalloc(ctypes.byref(p), max(int(nbytes), 16)) == 0
        self.blocks.append(p.value)
        return p.value

    def filled(self, nbytes, byte):
        p = self.alloc(nbytes)
        assert self.hip.hipMemset(p, byte, nbytes) == 0
        return p

    def put(self, array, p=None):
        array = np.ascontiguousarray(array)
        p = self.alloc(array.nbytes) if p is None else p
        if array.nbytes:
            assert self.hip.hipMemcpy(p, array.ctypes.data, array.nbytes, 1) == 0
        return p

    def get(self, p, shape, dtype):
        out = np.empty(shape, dtype=dtype)
        assert self.hip.hipDeviceSynchronize() == 0
        if out.nbytes:
            assert self.hip.hipMemcpy(out.ctypes.data, p, out.nbytes, 2) == 0
        return out

    def stream(self):
        s = ctypes.c_void_p()
        assert self.hip.hipStreamCreate(ctypes.byref(s)) == 0
        self.streams.append(s)
        return s

    def graph(self, stream, enqueue):
        """What enqueue() puts on the stream, as an executable graph."""
        g, e = ctypes.c_void_p(), ctypes.c_void_p()
        assert self.hip.hipStreamBeginCapture(stream, 0) == 0
        enqueue()
        assert self.hip.hipStreamEndCapture(stream, ctypes.byref(g)) == 0
        self.graphs.append(g)
        assert self.hip.hipGraphInstantiate(ctypes.byref(e), g, None, None, 0) == 0
        self.execs.append(e)
        return e

    def replay(self, e, stream):
        assert self.hip.hipGraphLaunch(e, stream) == 0
        assert self.hip.hipStreamSynchronize(stream) == 0


# ---- element types -------------------------------------------------------------

CODES = {"f32": G.MG_F32, "f16": G.MG_F16, "bf16": G.MG_BF16}
HALF_STEP = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}
STORED = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}


def stored(x, kind):
    """Values rounded to the type, in the form it has in memory."""
    x = np.asarray(x, dtype=np.float32)
    if kind != "bf16":
        with np.errstate(over="ignore"):
            return x.astype(STORED[kind])
    u = x.view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def values(a, kind):
    if kind != "bf16":
        return a.astype(np.float64)
    return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


# ---- the 8-bit cache -------------------------------------------------------------

E4M3 = np.array([(-1.0 if c & 128 else 1.0) * (math.nan if c & 127 == 127 else (c & 7) * 2.0**-9 if c & 120 == 0
                                               else (8 + (c & 7)) * 2.0**((c >> 3 & 15) - 10)) for c in range(256)])


def e4m3(x):
    """The nearest E4M3 values of x, |x| <= 448, ties to the even one; NaN stays."""
    step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(x), 2.0**-6))) - 3)
    return np.round(x / step) * step


def padded(width):
    return next(p for p in (32, 64, 128, 256) if width <= p)


def scale_exponent(x):
    """Of a block's values: the smallest e in -117..120 with max |x| <= 448 * 2^e."""
    finite = np.abs(x[np.isfinite(x)])
    top = finite.max() if finite.size else 0.0
    e = -117
    while e < 120 and top > 448 * 2.0**e:
        e += 1
    return e


class Cache:
    """A cache's bytes on the host, as read and written by the plain forms."""

    def __init__(self, batch, heads, width, capacity, rng):
        p = padded(width)
        self.batch, self.heads, self.width, self.capacity, self.pad = batch, heads, width, capacity, p
        # Whatever was there: codes and scales of any kind, NaN among them.
        self.k = rng.integers(0, 256, (batch, heads, capacity, p), dtype=np.uint8)
        self.v = rng.integers(0, 256, (batch, heads, capacity // TILE, p, TILE), dtype=np.uint8)
        self.ks = rng.integers(0, 256, (batch, heads, capacity // BLOCK), dtype=np.uint8)
        self.vs = rng.integers(0, 256, (batch, heads, capacity // BLOCK), dtype=np.uint8)

    def arrays(self):
        return self.k, self.v, self.ks, self.vs

    def on(self, dev):
        self.at = [dev.put(a) for a in self.arrays()]
        return G.Kv8(self.batch, self.heads, self.width, self.capacity, *self.at)

    def fetch(self, dev):
        return [dev.get(p, a.shape, np.uint8) for p, a in zip(self.at, self.arrays())]

    def decoded(self, arrays=None):
        """(keys, values) [batch, heads, capacity, width] of the bytes."""
        k, v, ks, vs = self.arrays() if arrays is None else arrays
        out = []
        for codes, scale in ((k, ks), (v.transpose(0, 1, 2, 4, 3).reshape(k.shape), vs)):
            s = 2.0 ** (np.repeat(scale, BLOCK, 2).astype(np.float64) - 127)
            with np.errstate(invalid="ignore"):
                out.append((E4M3[codes] * s[..., None])[..., :self.width])
        return out


def appended(cache, arrays, k, v, lengths, counts):
    """(code values, exponents) that the blocks of `arrays` hold after the new
    tokens k, v [batch][count][heads][width] (float64): for keys and for values, a
    dict of (sequence, head, position) -> code values [pad] and one of
    (sequence, head, block) -> exponent, for what an append may change."""
    result = []
    for new, codes, scales in ((k, arrays[0], arrays[2]),
                               (v, arrays[1].transpose(0, 1, 2, 4, 3).reshape(cache.k.shape), arrays[3])):
        held, exponents = {}, {}
        for s in range(cache.batch):
            length, count = int(lengths[s]), int(counts[s])
            start = length - count
            for h in range(cache.heads):
                for block in range(start // BLOCK, (length + BLOCK - 1) // BLOCK if count else 0):
                    lo, hi = max(start, BLOCK * block), min(length, BLOCK * (block + 1))
                    if lo >= hi:
                        continue
                    x = new[s, lo - start:hi - start, h]
                    e = scale_exponent(x)
                    if lo > BLOCK * block:
                        was = int(scales[s, h, block]) - 127
                        e = max(e, was)
                        for place in range(BLOCK * block, lo):
                            held[s, h, place] = e4m3(E4M3[codes[s, h, place]] * 2.0 ** (was - e))
                    exponents[s, h, block] = e
                    limit = 240.0 if e == 120 else 448.0
                    for i in range(hi - lo):
                        y = np.zeros(cache.pad)
                        t = x[i] / 2.0**e
                        y[:cache.width] = np.where(np.isfinite(t), e4m3(np.clip(t, -limit, limit)), np.nan)
                        held[s, h, lo + i] = y
        result.append((held, exponents))
    return result


# ---- attention -------------------------------------------------------------------

def attention(q, k, v, lengths, counts, scale):
    """(output, sum of p |v|, largest sum |q k| scale, largest |score|) in 64 bits: q
    [batch][count][heads][width], k and v [batch][kv_heads][capacity][width]."""
    out, size, mass, far = (np.zeros(q.shape) for _ in range(4))
    group = q.shape[2] // k.shape[1]
    for s in range(q.shape[0]):
        length, count = int(lengths[s]), int(counts[s])
        for i in range(count):
            n = length - count + i + 1
            for h in range(q.shape[2]):
                kk, vv = k[s, h // group, :n], v[s, h // group, :n]
                with np.errstate(invalid="ignore", over="ignore"):
                    score = kk @ q[s, i, h] * scale
                    p = np.exp(score - score.max())
                    p /= p.sum()
                    # A weight of 0 times NaN is NaN: the row sees it.
                    out[s, i, h] = p @ vv
                    size[s, i, h] = p @ np.abs(vv)
                    mass[s, i, h] = (np.abs(kk) @ np.abs(q[s, i, h]) * scale).max()
                    far[s, i, h] = np.abs(score).max()
    return out, size, mass, far


def attention_tolerance(kind, out, size, mass, far, width, keys):
    """|error| of an attention output by its roundings.  Scores: a product of
    `width` terms in FP32, then two roundings of a value of up to 1.5 |score| in
    log2 units and as much for the maximum; exp2 1 ulp; the same twice, for the sum
    over `keys` and the output; probabilities cut to their pieces; the output's
    half step."""
    step = 2.0**-24
    exponent = 2 * (width + 2) * step * mass + 6 * step * (1.5 * far + 1)
    sums = (keys / 8 + 64) * step
    piece = {"f32": 2.0**-23, "f16": 2.0**-15, "bf16": 2.0**-8}[kind]
    least = {"f32": 2.0**-149, "f16": 2.0**-25, "bf16": 2.0**-133}[kind]
    return (2 * exponent + 2 * sums + piece) * size * 1.01 + HALF_STEP[kind] * np.abs(out) * 1.01 + least


# ---- log probabilities -------------------------------------------------------------

def logprobs(z, tokens, temperature, top):
    """(logprob, entropy, top tokens, top logprobs) of rows z in 64 bits."""
    rows, vocab = z.shape
    lp, h = np.zeros(rows), np.zeros(rows)
    ids, best = np.zeros((rows, top), dtype=np.uint32), np.zeros((rows, top))
    for r in range(rows):
        if np.isnan(z[r]).any() or (z[r] == np.inf).any():
            lp[r], h[r], ids[r], best[r] = math.nan, math.nan, np.arange(top), math.nan
        elif (z[r] == -np.inf).all():
            lp[r], h[r], ids[r], best[r] = -math.inf, 0.0, np.arange(top), -math.inf
        else:
            d = (z[r] - z[r].max()) / temperature
            e = np.exp(d)
            logp = d - np.log(e.sum())
            lp[r] = logp[tokens[r]] if tokens[r] < vocab else math.nan
            h[r] = -np.sum(np.where(e > 0, e / e.sum() * np.where(e > 0, logp, 0), 0))
            order = np.lexsort((np.arange(vocab), -z[r]))[:top]
            ids[r], best[r] = order, logp[order]
        if tokens[r] == G.IGNORE_TARGET:
            lp[r] = 0.0
    return lp, h, ids, best


def logprob_gradient(z, tokens, temperature, d_logprob, d_entropy):
    """The gradient of the logits in 64 bits."""
    out = np.zeros(z.shape)
    for r in range(z.shape[0]):
        if (z[r] == -np.inf).all():
            continue
        d = (z[r] - z[r].max()) / temperature
        e = np.exp(d)
        p = e / e.sum()
        logp = np.where(p > 0, d - np.log(e.sum()), 0)
        entropy = -np.sum(p * logp)
        g = 0.0 if tokens[r] == G.IGNORE_TARGET else d_logprob[r]
        out[r] = -p * (g + d_entropy[r] * (logp + entropy))
        if tokens[r] != G.IGNORE_TARGET:
            out[r, tokens[r]] += g
    return out / temperature
