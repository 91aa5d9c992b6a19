"""Plain 64-bit forms of the operators around a step's matrix products
(include/meshgpt.h: mg_sample_filtered_noalloc, mg_rope_*, mg_rms_norm*) on numpy
arrays."""
import math

import numpy as np

import operators_lib as L

NO_TOKEN = 0xFFFFFFFF


def draw(z, temperature, top_k, top_p, min_p, u):
    """(token, log probability) of one row; sums in numpy's longest type."""
    z = np.asarray(z, dtype=np.float64)
    if (np.isnan(z).any() or (z == np.inf).any() or (z == -np.inf).all() or not 0 <= temperature < math.inf
            or math.isnan(top_p) or math.isnan(min_p) or (temperature > 0 and not 0 <= u < 1)):
        return NO_TOKEN, math.nan
    order = np.argsort(-z, kind="stable")
    if temperature == 0:
        return int(order[0]), 0.0
    with np.errstate(over="ignore", under="ignore"):
        w = np.exp(((z[order] - z[order[0]]) / np.float64(temperature)).astype(np.longdouble))
    if 0 < top_k < len(w):
        w = w[:top_k]
    if top_p < 1:
        running = np.cumsum(w)
        w = w[:int(np.sum(running < np.longdouble(top_p) * running[-1])) + 1]
    if min_p > 0:
        w = w[:max(1, int(np.sum(w >= np.longdouble(min(min_p, 1.0)))))]
    w = w[w > 0]
    running = np.cumsum(w)
    at = min(int(np.sum(running <= np.longdouble(u) * running[-1])), len(w) - 1)
    return int(order[at]), float(np.log(w[at] / running[-1]))


def frequencies(rotary, base=10000.0, scaling=0, factor=1.0, context=0.0, low=1.0, high=32.0):
    """Radians a position, of each pair."""
    if scaling == 2 and rotary > 2:
        base = base * factor ** (rotary / (rotary - 2))
    f = base ** (-np.arange(0, rotary, 2, dtype=np.float64) / max(rotary, 1))
    if scaling == 1:
        return f / factor
    if scaling == 3:
        kept = np.clip((context * f / (2 * np.pi) - low) / (high - low), 0, 1)
        return f * kept + f / factor * (1 - kept)
    return f


def positions(batch, count, lengths, counts, given):
    """(position, whether it is there) of each token, [batch][count]."""
    at = np.zeros((batch, count), dtype=np.int64)
    there = np.zeros((batch, count), dtype=bool)
    for s in range(batch):
        n = count if counts is None else int(counts[s])
        length = n if lengths is None else int(lengths[s])
        if n < 0 or n > count or length < n:
            continue
        there[s, :n] = True
        at[s, :n] = given[s, :n] if given is not None else length - n + np.arange(n)
    return at, there


def turned(x, at, f, interleaved, magnitude, backward=False):
    """x [batch][count][heads][width] with its first 2 len(f) channels turned."""
    r = 2 * len(f)
    angle = at[:, :, None].astype(np.longdouble) * f.astype(np.longdouble)
    # numpy's longest pi has 64 bits: angles up to 2^31 keep 30 behind the point.
    angle = np.remainder(angle, 2 * np.longdouble("3.14159265358979323846264")).astype(np.float64)
    c, s = (magnitude * np.cos(angle))[:, :, None], (magnitude * np.sin(angle))[:, :, None]
    if backward:
        s = -s
    y = np.array(x, dtype=np.float64)
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = np.array(y[..., first]), np.array(y[..., second])
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    return y


def norm(x, residual, weight, epsilon, kind):
    """(kept sum as stored, its values, rstd, output) of rows in their stored form."""
    kept = x
    if residual is not None:
        with np.errstate(over="ignore", invalid="ignore"):
            kept = L.stored(L.values(x, kind).astype(np.float32) + L.values(residual, kind).astype(np.float32), kind)
    h = L.values(kept, kind)
    with np.errstate(invalid="ignore", over="ignore"):
        rstd = 1 / np.sqrt(np.mean(h.astype(np.longdouble) ** 2, 1) + np.longdouble(np.float32(epsilon)))
        y = h * rstd[:, None] * (1 if weight is None else L.values(weight, kind)[None])
    return kept, h, rstd.astype(np.float64), y.astype(np.float64)


def to_codes(y):
    """(values of the codes, scale bytes) of rows of y, 32 channels a scale."""
    rows, width = y.shape
    codes, scales = np.zeros(y.shape), np.zeros((rows, (width + 31) // 32), dtype=np.uint8)
    for r in range(rows):
        for b in range(scales.shape[1]):
            part = y[r, 32 * b:32 * b + 32]
            e = L.scale_exponent(part)
            with np.errstate(invalid="ignore"):
                t = part / 2.0**e
                codes[r, 32 * b:32 * b + 32] = np.where(np.abs(t) < 464, L.e4m3(t), np.nan)
            scales[r, b] = e + 127
    return codes, scales


def norm_gradient(h, weight, rstd, d_out, d_sum):
    """(d_x, d_weight) in 64 bits, of values."""
    hat = h * rstd[:, None]
    g = d_out * (1 if weight is None else weight[None])
    d = rstd[:, None] * (g - hat * np.mean(g * hat, 1, keepdims=True))
    return d + (0 if d_sum is None else d_sum), np.sum(d_out * hat, 0)
