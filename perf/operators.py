"""Operators of serving and scoring, as a program with its tensors on the GPU calls them.

The 8-bit KV cache (append, read back, attention over it) and the log
probabilities of tokens (with entropy and top alternatives, and their
gradient).  Every case runs in a plain form made of elementary torch
operations in 32 bits, or, with `own`, through the entry points of
include/meshgpt.h; `exact` has the results of the definitions in 64 bits.

The cache: keys [batch][kv_heads][capacity][P] and values
[batch][kv_heads][capacity / 64][P][64] in E4M3 codes, where P is the head
width padded to 32, 64, 128 or 256; a scale 2^(byte - 127) for each 16 tokens
and head, [batch][kv_heads][capacity / 16], of keys and of values.
"""
import math

import numpy as np
import torch

own = False

IGNORE = 0xFFFFFFFF
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # The alternatives of a sampled step: the benchmark's vocabulary and batch, where latency counts.
        dict(name="logprobs step", op="logprobs", type="f32", rows=32, vocab=256, top=5, temperature=0.8),
        # A scored batch of prompts at a word-piece vocabulary that is no multiple of anything.
        dict(name="logprobs large", op="logprobs", type="bf16", rows=1000, vocab=128001, top=20, temperature=1.0),
        # The symbolic model's training batch: 256 equations of four tokens.
        dict(name="backward symbolic", op="backward", type="f32", rows=1024, vocab=99, temperature=1.0),
        # The loss's gradient over a training batch of text.
        dict(name="backward text", op="backward", type="bf16", rows=4096, vocab=50257, temperature=1.0),
        # One decode step of the mid model: a token of each sequence joins its cache.
        dict(name="append step", op="append", type="f32", batch=32, kv_heads=8, width=64, capacity=1024, count=1,
             shortest=64, longest=576, ragged=False, fused=False),
        # Prompts of a batch written at once, out of a fused projection, each with its own length.
        dict(name="append prompts", op="append", type="bf16", batch=8, kv_heads=8, width=128, capacity=8192, count=4000,
             shortest=4000, longest=8000, ragged=True, fused=True),
        # A prefix read back to be moved or looked at: small, in the framework's own type.
        dict(name="read prefix", op="read", type="f32", batch=4, kv_heads=8, width=64, capacity=1024, first=37, count=475),
        # A whole cache read back for a consumer in 16 bits.
        dict(name="read cache", op="read", type="f16", batch=16, kv_heads=8, width=128, capacity=8192, first=0, count=8000),
        # Decode of the mid model: batch 32, 8 heads of 64, in the framework's own type.
        dict(name="attention step", op="attention", type="f32", batch=32, heads=8, kv_heads=8, width=64, capacity=1024,
             count=1, shortest=64, longest=576, ragged=False),
        # Decode of long sequences with shared heads.
        dict(name="attention long step", op="attention", type="bf16", batch=64, heads=32, kv_heads=8, width=128,
             capacity=16384, count=1, shortest=2000, longest=16000, ragged=False),
        # Prompts of uneven length in the framework's own type, after a cached prefix.
        dict(name="attention prompts", op="attention", type="f32", batch=3, heads=8, kv_heads=8, width=64, capacity=2048,
             count=1001, shortest=1001, longest=1501, ragged=True),
        # Long prompts with shared heads.
        dict(name="attention long prompts", op="attention", type="bf16", batch=4, heads=32, kv_heads=8, width=128,
             capacity=4096, count=4096, shortest=4096, longest=4096, ragged=False),
    ]


def _span(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["logprobs", "backward", "append", "read", "attention", "attention"])
    kind = rng.choice(["f32", "f16", "bf16"])
    if op in ("logprobs", "backward"):
        vocab = _span(rng, 17, 131072)
        rows = _span(rng, 1, max(1, min(8192, 128_000_000 // vocab)))
        case = dict(op=op, type=kind, rows=rows, vocab=vocab, temperature=rng.choice([1.0, 1.0, 0.7, 1.5]))
        if op == "logprobs":
            case["top"] = min(vocab, rng.choice([0, 1, 5, 20, 32]))
        return case
    width = rng.choice([32, 64, 64, 128, 128, 256, 80, 96, 50])
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    if op in ("append", "read"):
        count = _span(rng, 1, 8000)
        batch = _span(rng, 1, max(1, min(128, 64_000_000 // (count * kv_heads * width))))
        prefix = _span(rng, 1, 1000)
        capacity = (prefix + count + 32 + 63) // 64 * 64
        if op == "read":
            return dict(op=op, type=kind, batch=batch, kv_heads=kv_heads, width=width, capacity=capacity, first=prefix,
                        count=count)
        return dict(op=op, type=kind, batch=batch, kv_heads=kv_heads, width=width, capacity=capacity, count=count,
                    shortest=count, longest=count + prefix, ragged=rng.random() < 0.5, fused=rng.random() < 0.5)
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    if rng.random() < 0.5:  # single tokens, or a few
        count = rng.choice([1, 1, 1, 2, 5])
        longest = _span(rng, 5, 16000)
        batch = _span(rng, 1, max(1, min(64, 32_000_000 // (longest * kv_heads * width))))
    else:
        count = _span(rng, 16, 4000)
        longest = count + _span(rng, 1, 1000)
        batch = max(1, min(8, _span(rng, 1, max(1, 500_000_000 // (count * longest * heads)))))
    return dict(op=op, type=kind, batch=batch, heads=heads, kv_heads=kv_heads, width=width,
                capacity=(longest + 32 + 63) // 64 * 64, count=count, shortest=max(count, longest // 4), longest=longest,
                ragged=rng.random() < 0.5)


def _padded(width):
    return 32 if width <= 32 else 64 if width <= 64 else 128 if width <= 128 else 256


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


# ---- the cache in elementary operations -------------------------------------

def _times_power(x, e):
    """x 2^e, exact: what lies under 2^-126 rounds to no code but zero."""
    return x * ((e.clamp(-126, 127) + 127) << 23).view(torch.float32)


def _scale_byte(amax):
    """The byte of the smallest power of two whose 448-fold reaches amax."""
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, e - 9 + (m > 0.875).to(e.dtype), torch.full_like(e, -1000))
    return (e + 127).clamp(10, 247)


def _encode(x):
    return x.to(torch.float8_e4m3fn).view(torch.uint8)


def _decode(codes):
    return codes.view(torch.float8_e4m3fn).float()


def _quantised(x):
    """The codes [batch, heads, tokens, P] and scale bytes of float32 values of that shape."""
    b, h, t, p = x.shape
    blocks = x.view(b, h, t // 16, 16, p)
    byte = _scale_byte(blocks.abs().amax((3, 4)))
    codes = _encode(_times_power(blocks, (127 - byte)[..., None, None]))
    return codes.view(b, h, t, p), byte.to(torch.uint8)


def _filled_cache(case, g):
    """A cache as earlier calls have left it: every position quantised, also
    behind the sequences, where older tokens stand."""
    b, h, c, p, d = case["batch"], case["kv_heads"], case["capacity"], _padded(case["width"]), case["width"]
    cache = {"k": torch.empty(b, h, c, p, dtype=torch.uint8, device="cuda"),
             "v": torch.empty(b, h, c // 64, p, 64, dtype=torch.uint8, device="cuda"),
             "k_scale": torch.empty(b, h, c // 16, dtype=torch.uint8, device="cuda"),
             "v_scale": torch.empty(b, h, c // 16, dtype=torch.uint8, device="cuda")}
    spread = torch.exp(0.5 * torch.randn(2, h, 1, d, generator=g, device="cuda"))  # channels differ in size
    for i in range(b):
        for name, s in (("k", spread[0]), ("v", spread[1])):
            x = torch.zeros(1, h, c, p, device="cuda")
            x[..., :d] = torch.randn(1, h, c, d, generator=g, device="cuda") * s
            codes, byte = _quantised(x)
            cache[name + "_scale"][i] = byte[0]
            cache[name][i] = codes[0] if name == "k" else codes[0].view(h, c // 64, 64, p).transpose(2, 3)
    return cache


def _lengths(case, g):
    """Tokens of each sequence, the new ones among them, and how many are new."""
    b = case["batch"]
    n = torch.randint(case["shortest"], case["longest"] + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    n[0] = case["longest"]
    new = torch.full((b,), case["count"], dtype=torch.int32, device="cuda")
    if case["ragged"]:
        new = torch.randint(case["count"] // 4, case["count"] + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        new[0] = case["count"]
    return n, new


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": case}
    kind = TYPES[case["type"]]
    if case["op"] in ("logprobs", "backward"):
        rows, vocab = case["rows"], case["vocab"]
        z = torch.empty(rows, vocab, dtype=kind, device="cuda")
        for i in range(0, rows, 512):
            n = min(512, rows - i)
            part = torch.randn(n, vocab, generator=g, device="cuda") * (1 + 3 * torch.rand(n, 1, generator=g, device="cuda"))
            z[i:i + n] = part.to(kind)
        if rows >= 4:  # one row in four allows every eighth token alone
            z[1::4, (torch.arange(vocab, device="cuda") % 8) != 3] = -math.inf
        tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int64)
        if rows >= 4:
            tokens[1::4] = 3 + 8 * (tokens[1::4] % ((vocab - 4) // 8 + 1))
        s["logits"] = z
        s["targets"] = tokens.to(torch.int32)
        if case["op"] == "backward":
            if rows > 8:
                s["targets"][5::9] = -1  # rows without supervision: all bits set
            d = (z.double() - z.double().amax(1, keepdim=True)) / case["temperature"]
            e = d.exp()
            total = e.sum(1)
            s["stats"] = torch.stack([z.float().amax(1), total.log().float()], 1).contiguous()
            s["entropy"] = (total.log() - torch.where(e > 0, e * d, 0.0).sum(1) / total).float()
            s["d_logprob"] = torch.randn(rows, generator=g, device="cuda")
            s["d_entropy"] = 0.1 * torch.randn(rows, generator=g, device="cuda")
        return s
    s["cache"] = _filled_cache(case, g)
    b, d = case["batch"], case["width"]
    if case["op"] == "read":
        return s
    s["lengths"], s["counts"] = _lengths(case, g)
    if case["op"] == "append":
        n, h = case["count"], case["kv_heads"]
        if case["fused"]:
            both = torch.randn(b, n, 2, h, d, generator=g, device="cuda").to(kind)
            s["new_k"], s["new_v"] = both[:, :, 0], both[:, :, 1]
        else:
            s["new_k"] = torch.randn(b, n, h, d, generator=g, device="cuda").to(kind)
            s["new_v"] = torch.randn(b, n, h, d, generator=g, device="cuda").to(kind)
    else:
        s["q"] = torch.randn(b, case["count"], case["heads"], d, generator=g, device="cuda").to(kind)
        s["out"] = torch.zeros_like(s["q"])  # rows behind a sequence's own stay as they are
    return s


# ---- one pass ----------------------------------------------------------------

def run(state):
    if own:
        return _own(state)
    return {"logprobs": _plain_logprobs, "backward": _plain_backward, "append": _plain_append, "read": _plain_read,
            "attention": _plain_attention}[state["case"]["op"]](state)


def _plain_logprobs(s):
    case, z = s["case"], s["logits"].float()
    top = z.amax(1, keepdim=True)
    d = (z - top) / case["temperature"]
    e = d.exp()
    total = e.sum(1)
    log_total = total.log()
    at = d.gather(1, s["targets"].long()[:, None])[:, 0]
    out = {"logprob": at - log_total, "entropy": log_total - torch.where(e > 0, e * d, 0.0).sum(1) / total,
           "stats": torch.stack([top[:, 0], log_total], 1)}
    if case["top"]:
        bits = (z + 0.0).view(torch.int32)
        key = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).long() * (1 << 31)  # ordered as the values are
        key = key + ((1 << 31) - 1 - torch.arange(case["vocab"], device=z.device))  # of equal ones the first
        ids = ((1 << 31) - 1) - (key.topk(case["top"], dim=1).values & ((1 << 31) - 1))
        out["top_tokens"] = ids.to(torch.int32)
        out["top_logprobs"] = d.gather(1, ids) - log_total[:, None]
    return out


def _plain_backward(s):
    case, z = s["case"], s["logits"].float()
    logp = (z - s["stats"][:, :1]) / case["temperature"] - s["stats"][:, 1:]
    p = logp.exp()
    wanted = s["targets"] != -1
    g = torch.where(wanted, s["d_logprob"], 0.0)[:, None]
    grad = -p * (g + s["d_entropy"][:, None] * (torch.where(p > 0, logp, 0.0) + s["entropy"][:, None]))
    at = torch.where(wanted, s["targets"], 0).long()[:, None]
    grad = grad.scatter_add(1, at, g)
    return {"d_logits": (grad / case["temperature"]).to(s["logits"].dtype)}


def _plain_append(s):
    case, cache = s["case"], s["cache"]
    b, h, n, d = case["batch"], case["kv_heads"], case["count"], case["width"]
    blocks = (n + 30) // 16
    start = (s["lengths"] - s["counts"]).long()
    base = torch.minimum(start - start % 16, torch.full_like(start, case["capacity"] - 16 * blocks))
    slot = torch.arange(blocks * 16, device="cuda")
    place = base[:, None] + slot[None]  # a window of whole blocks with every position that is written
    token = place - start[:, None]
    fresh = (token >= 0) & (token < s["counts"].long()[:, None])
    older = (token < 0) & (token >= -(start % 16)[:, None]) & (s["counts"] > 0)[:, None]
    rows = torch.arange(b, device="cuda")[:, None]
    block = (base // 16)[:, None] + torch.arange(blocks, device="cuda")[None]
    written = fresh.view(b, blocks, 16).any(2)
    begun = older.view(b, blocks, 16).any(2)
    for name in ("k", "v"):
        x = s["new_" + name].float()[rows, token.clamp(0, n - 1)] * fresh[:, :, None, None]  # [b, slots, h, d]
        scales = cache[name + "_scale"]
        old = scales[rows, :, block].int()  # [b, blocks, h]
        byte = _scale_byte(x.view(b, blocks, 16, h, d).abs().amax((2, 4)))
        byte = torch.where(begun[..., None], torch.maximum(byte, old), byte)
        codes = _encode(_times_power(x.view(b, blocks, 16, h, d), (127 - byte)[:, :, None, :, None])).view(b, -1, h, d)
        at = (rows, slice(None), place) if name == "k" else (rows, slice(None), place // 64, slice(None), place % 64)
        was = cache[name][at]  # [b, slots, h, P]
        again = _encode(_times_power(_decode(was).view(b, blocks, 16, h, -1), (old - byte)[:, :, None, :, None])).view_as(was)
        now = torch.where(older[:, :, None, None], again, was)
        now[..., :d] = torch.where(fresh[:, :, None, None], codes, now[..., :d])
        now[..., d:] = torch.where(fresh[:, :, None, None], torch.zeros_like(now[..., d:]), now[..., d:])
        cache[name][at] = now
        scales[rows, :, block] = torch.where(written[..., None], byte, old).to(torch.uint8)
    return _held(cache)


def _held(cache):
    """What the cache holds: the codes' values and the scales' bytes."""
    return {"k": cache["k"].view(torch.float8_e4m3fn), "v": cache["v"].view(torch.float8_e4m3fn),
            "k_scale": cache["k_scale"], "v_scale": cache["v_scale"]}


def _values(cache, name, longest, d):
    """The float32 values [b, h, longest, d] of the cache's first positions."""
    if name == "k":
        codes = cache["k"][:, :, :longest, :d]
    else:
        codes = cache["v"][:, :, :(longest + 63) // 64, :d].transpose(3, 4).flatten(2, 3)[:, :, :longest]
    byte = cache[name + "_scale"][:, :, :(longest + 15) // 16].int().repeat_interleave(16, 2)[:, :, :longest]
    return _times_power(_decode(codes), (byte - 127)[..., None])


def _plain_read(s):
    case = s["case"]
    first, last = case["first"], case["first"] + case["count"]
    return {n: _values(s["cache"], n, last, case["width"])[:, :, first:].transpose(1, 2).to(TYPES[case["type"]])
            .contiguous() for n in ("k", "v")}


def _plain_attention(s):
    case, cache = s["case"], s["cache"]
    b, n, h, hk, d, longest = (case[x] for x in ("batch", "count", "heads", "kv_heads", "width", "longest"))
    k, v = _values(cache, "k", longest, d), _values(cache, "v", longest, d)
    q = s["q"].float().view(b, n, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, h // hk * n, d)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()).view(b, hk, h // hk, n, longest) * (1 / math.sqrt(d))
    key = torch.arange(longest, device="cuda")
    place = (s["lengths"] - s["counts"])[:, None] + torch.arange(n, device="cuda", dtype=torch.int32)[None]
    seen = key[None, None] <= place[:, :, None]  # [b, n, longest]
    score = torch.where(seen[:, None, None], score, -math.inf)
    e = (score - score.amax(4, keepdim=True)).exp()
    total = e.sum(4, keepdim=True)
    out = torch.matmul(e.view(b, hk, -1, longest), v).view(b, hk, h // hk, n, d) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(b, n, h, d)
    real = torch.arange(n, device="cuda")[None] < s["counts"][:, None]
    return {"out": torch.where(real[:, :, None, None], out, 0.0).to(s["q"].dtype)}


def _own(s):
    import grokking_abmod_amd as G

    case, op = s["case"], s["case"]["op"]
    kind, stream = {"f32": G.MG_F32, "f16": G.MG_F16, "bf16": G.MG_BF16}[case["type"]], torch.cuda.current_stream().cuda_stream
    if op == "logprobs":
        z, rows, top = s["logits"], case["rows"], case["top"]
        floats = torch.empty(4 * rows, device="cuda")
        logprob, entropy, stats = floats[:rows], floats[rows:2 * rows], floats[2 * rows:].view(rows, 2)
        out = {"logprob": logprob, "entropy": entropy, "stats": stats}
        ids = alternatives = None
        if top:
            ids = out["top_tokens"] = torch.empty(rows, top, dtype=torch.int32, device="cuda")
            alternatives = out["top_logprobs"] = torch.empty(rows, top, device="cuda")
        room = G.token_logprobs_workspace(rows, case["vocab"], top)
        space = torch.empty(room, dtype=torch.uint8, device="cuda") if room else None
        G.token_logprobs_noalloc(kind, z.data_ptr(), rows, case["vocab"], z.stride(0), s["targets"].data_ptr(),
                                 case["temperature"], logprob.data_ptr(), entropy.data_ptr(), stats.data_ptr(), top,
                                 ids.data_ptr() if top else None, alternatives.data_ptr() if top else None,
                                 space.data_ptr() if room else None, room, stream)
        return out
    if op == "backward":
        z = s["logits"]
        grad = torch.empty_like(z)
        G.token_logprobs_backward_noalloc(kind, z.data_ptr(), case["rows"], case["vocab"], z.stride(0),
                                          s["targets"].data_ptr(), case["temperature"], s["stats"].data_ptr(),
                                          s["entropy"].data_ptr(), s["d_logprob"].data_ptr(), s["d_entropy"].data_ptr(),
                                          grad.data_ptr(), grad.stride(0), stream)
        return {"d_logits": grad}
    c = s["cache"]
    cache = G.Kv8(case["batch"], case["kv_heads"], case["width"], case["capacity"], c["k"].data_ptr(), c["v"].data_ptr(),
                  c["k_scale"].data_ptr(), c["v_scale"].data_ptr())
    if op == "append":
        k, v = s["new_k"], s["new_v"]
        G.kv8_append(cache, kind, case["count"], k.data_ptr(), k.stride()[:3], v.data_ptr(), v.stride()[:3],
                     s["lengths"].data_ptr(), s["counts"].data_ptr(), stream)
        return _held(c)
    if op == "read":
        k = torch.empty(case["batch"], case["count"], case["kv_heads"], case["width"], dtype=TYPES[case["type"]], device="cuda")
        v = torch.empty_like(k)
        G.kv8_read(cache, kind, case["first"], case["count"], k.data_ptr(), k.stride()[:3], v.data_ptr(), v.stride()[:3],
                   None, stream)
        return {"k": k, "v": v}
    q, out = s["q"], s["out"]
    room = G.kv8_attention_workspace(cache, case["heads"], case["count"])
    space = torch.empty(room, dtype=torch.uint8, device="cuda") if room else None
    G.kv8_attention(cache, kind, case["heads"], case["count"], q.data_ptr(), q.stride()[:3], out.data_ptr(),
                    out.stride()[:3], s["lengths"].data_ptr(), s["counts"].data_ptr(), 1 / math.sqrt(case["width"]),
                    space.data_ptr() if room else None, room, stream)
    return {"out": out}


# ---- what a pass cannot do without ---------------------------------------------

def work(case):
    size = SIZE[case["type"]]
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (20 + 8 * case["top"]), "flops": 6 * n}
    if case["op"] == "backward":
        n = case["rows"] * case["vocab"]
        return {"bytes": 2 * n * size + 24 * case["rows"], "flops": 8 * n}
    b, hk, d = case["batch"], case["kv_heads"], case["width"]
    if case["op"] in ("append", "read"):
        tokens = b * case["count"]
        if case["op"] == "append" and case["ragged"]:
            tokens *= 0.625  # a quarter to all of the count, the same everywhere between
        n = 2 * tokens * hk * d
        return {"bytes": n * (size + 1 + 1 / (16 * d)), "flops": 4 * n}
    n, h = case["count"], case["heads"]
    lengths = b * (case["shortest"] + case["longest"]) / 2
    mean = n * (0.625 if case["ragged"] else 1.0)
    seen = b * mean * (lengths / b - (mean - 1) / 2)
    return {"bytes": lengths * hk * (2 * d + 1 / 8) + 2 * b * mean * h * d * size, "flops": 4 * d * h * seen}


# ---- the definitions in 64 bits ------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"logprobs": _exact_logprobs, "backward": _exact_backward, "append": _exact_append, "read": _exact_read,
            "attention": _exact_attention}[case["op"]](case, s)


def _exact_logprobs(case, s):
    out = {"logprob": [], "entropy": [], "stats": [], "top_tokens": None, "top_logprobs": []}
    for i in range(0, case["rows"], 256):
        z = s["logits"][i:i + 256].double()
        logp = torch.log_softmax(z / case["temperature"], 1)
        p = logp.exp()
        top = z.amax(1)
        out["logprob"].append(logp.gather(1, s["targets"][i:i + 256].long()[:, None])[:, 0])
        out["entropy"].append(-torch.where(p > 0, p * logp, 0.0).sum(1))
        out["stats"].append(torch.stack([top, torch.logsumexp(z / case["temperature"], 1) - top / case["temperature"]], 1))
        if case["top"]:
            out["top_logprobs"].append(logp.sort(1, descending=True).values[:, :case["top"]])
    return {k: torch.cat(v) if v else None for k, v in out.items() if k[:3] != "top" or case["top"]}


def _exact_backward(case, s):
    grads = []
    for i in range(0, case["rows"], 256):
        z = s["logits"][i:i + 256].double().requires_grad_(False)
        logp = torch.log_softmax(z / case["temperature"], 1)
        p = logp.exp()
        logp = torch.where(p > 0, logp, 0.0)
        entropy = -(p * logp).sum(1, keepdim=True)
        t = s["targets"][i:i + 256].long()
        hot = (torch.arange(case["vocab"], device="cuda")[None] == t[:, None]).double()
        g = torch.where(t >= 0, s["d_logprob"][i:i + 256].double(), 0.0)[:, None]
        h = s["d_entropy"][i:i + 256].double()[:, None]
        grads.append((g * (hot - p) - h * p * (logp + entropy)) / case["temperature"])
    return {"d_logits": torch.cat(grads)}


_E4M3 = np.array([(-1.0 if c & 128 else 1.0) * (math.nan if c & 127 == 127 else (c & 7) * 2.0 ** -9 if c & 120 == 0
                                               else (8 + (c & 7)) * 2.0 ** ((c >> 3 & 15) - 10)) for c in range(256)])


def _table():
    return torch.tensor(_E4M3, device="cuda")


def _rounded(x):
    """x to the nearest E4M3 value, ties to the even one."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_append(case, s):
    cache, table = s["cache"], _table()
    out = {"k": table[cache["k"].long()], "v": table[cache["v"].long()], "k_scale": None, "v_scale": None}
    d = case["width"]
    for b in range(case["batch"]):
        length, new = int(s["lengths"][b]), int(s["counts"][b])
        at = length - new
        while at < length:  # one block of 16 tokens after the other
            block = at // 16
            until = min(length, 16 * (block + 1))
            first = at - (length - new)
            for name in ("k", "v"):
                x = s["new_" + name][b, first:first + until - at].double()  # [tokens, h, d]
                top = x.abs().amax((0, 2))
                e = torch.where(top > 0, torch.ceil(torch.log2(top / 448)), -1000.0).clamp(-117, 120)
                e = torch.where(448 * torch.exp2(e - 1) >= top, e - 1, e).clamp(-117, 120)
                values = out[name][b] if name == "k" else out[name][b, :, block // 4]
                if at % 16:
                    was = cache[name + "_scale"][b, :, block].double() - 127
                    e = torch.maximum(e, was)
                    shift = torch.exp2(was - e)
                    if name == "k":
                        values[:, 16 * block:at] = _rounded(values[:, 16 * block:at] * shift[:, None, None])
                    else:
                        part = slice(16 * block % 64, 16 * block % 64 + at % 16)
                        values[:, :, part] = _rounded(values[:, :, part] * shift[:, None, None])
                codes = _rounded(x / torch.exp2(e)[None, :, None]).permute(1, 0, 2)  # [h, tokens, d]
                if name == "k":
                    values[:, at:until, :d] = codes
                    values[:, at:until, d:] = 0
                else:
                    values[:, :d, at % 64:at % 64 + until - at] = codes.transpose(1, 2)
                    values[:, d:, at % 64:at % 64 + until - at] = 0
            at = until
    return out


def _exact_values(case, s, name):
    c, table = s["cache"], _table()
    codes = c["k"] if name == "k" else c["v"].transpose(3, 4).reshape(case["batch"], case["kv_heads"], case["capacity"], -1)
    scale = torch.exp2(c[name + "_scale"].double() - 127)
    return lambda b, h: (table[codes[b, h].long()].view(-1, 16, codes.shape[3]) * scale[b, h, :, None, None]).flatten(0, 1)


def _exact_read(case, s):
    out = {}
    for name in ("k", "v"):
        of = _exact_values(case, s, name)
        rows = slice(case["first"], case["first"] + case["count"])
        out[name] = torch.stack([torch.stack([of(b, h)[rows, :case["width"]] for h in range(case["kv_heads"])], 1)
                                 for b in range(case["batch"])])
    return out


def _exact_attention(case, s):
    keys, values = _exact_values(case, s, "k"), _exact_values(case, s, "v")
    d, group = case["width"], case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        length, new = int(s["lengths"][b]), int(s["counts"][b])
        place = torch.arange(length - new, length, device="cuda")
        hidden = torch.arange(length, device="cuda")[None] > place[:, None]
        for h in range(case["kv_heads"]):
            k, v = keys(b, h)[:length, :d], values(b, h)[:length, :d]
            for j in range(h * group, (h + 1) * group):
                score = (s["q"][b, :new, j].double() @ k.t()) / math.sqrt(d)
                out[b, :new, j] = torch.softmax(score.masked_fill(hidden, -math.inf), 1) @ v
    return {"out": out}
