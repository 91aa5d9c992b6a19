"""Operators around a decode or training step's matrix products, as a program with its tensors on the GPU calls them.

Sampling with temperature, top-k, top-p and min-p from given random numbers;
rotary positions (both pair layouts, part of the head, scaled frequencies) with
their gradient; the root-mean-square norm with the residual's addition, with an
output in 8 bits, and its gradient.  Every case runs in a plain form made of
elementary torch operations, or, with `own`, through the entry points of
include/meshgpt.h; `exact` has the results of the definitions in 64 bits.

Sampling: tokens are ranked by their logits, the largest first, of equal ones
the lowest token first.  A row's candidates are its first top_k tokens; of these
the shortest run from the first whose probabilities reach top_p of the run's
whole; of these the ones with at least min_p times the largest probability.
The token drawn is the first in rank at which the candidates' running sum
exceeds the random number times their sum.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPSILON = 1e-5


def listed():
    return [
        # The sampled step of the mid model's decode: the benchmark's vocabulary and batch, where latency counts.
        dict(name="sample step", op="sample", type="f32", rows=32, vocab=256, settings="both"),
        # A serving batch at a byte-pair vocabulary whose rows come from requests with settings of their own.
        dict(name="sample requests", op="sample", type="f32", rows=64, vocab=50257, settings="mixed"),
        # Rollouts at a word-piece vocabulary that is no multiple of anything, by the nucleus alone.
        dict(name="sample nucleus", op="sample", type="bf16", rows=1000, vocab=128001, settings="nucleus"),
        # One decode step of the mid model: 32 sequences, 8 heads of 64, in the framework's own type.
        dict(name="rope step", op="rope", type="f32", batch=32, count=1, heads=8, kv_heads=8, width=64, rotary=64,
             layout="half", scaling="none", longest=576, ragged=False, fused=False),
        # Prompts of uneven length after a prefix, neighbours as pairs, part of an odd head, shared heads.
        dict(name="rope part", op="rope", type="f16", batch=3, count=1001, heads=12, kv_heads=4, width=80, rotary=50,
             layout="interleaved", scaling="linear", longest=1501, ragged=True, fused=False),
        # Pieces of long prompts far into their context, as views of the fused projection's output.
        dict(name="rope long", op="rope", type="bf16", batch=4, count=8192, heads=32, kv_heads=8, width=128, rotary=128,
             layout="half", scaling="bands", longest=1000000, ragged=False, fused=True),
        # The gradient of a training batch of text.
        dict(name="rope gradient", op="rope_backward", type="bf16", batch=8, count=2048, heads=16, kv_heads=16, width=64,
             rotary=64, layout="half", scaling="none", longest=2048, ragged=False, fused=False),
        # The norm of one decode step of the mid model, without a residual and parameter-free, as its own is.
        dict(name="norm step", op="norm", type="f32", rows=32, width=512, residual=False, weight=False),
        # The norm before a block of long prompts: residual added and kept.
        dict(name="norm long", op="norm", type="bf16", rows=16384, width=4096, residual=True, weight=True),
        # The input of an 8-bit product over a batch of prompts.
        dict(name="norm to 8 bits", op="norm8", type="f16", rows=4001, width=5120, residual=True, weight=True),
        # The symbolic model's training batch: 256 equations of four tokens.
        dict(name="norm gradient symbolic", op="norm_backward", type="f32", rows=1024, width=128, residual=True, weight=True),
        # A training batch of text.
        dict(name="norm gradient text", op="norm_backward", type="bf16", rows=8192, width=4096, residual=True, weight=True),
    ]


def _span(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["sample", "sample", "rope", "rope_backward", "norm", "norm8", "norm_backward"])
    kind = rng.choice(["f32", "f16", "bf16"])
    if op == "sample":
        vocab = _span(rng, 17, 131072)
        rows = _span(rng, 1, max(1, min(4096, 64_000_000 // vocab)))
        return dict(op=op, type=kind, rows=rows, vocab=vocab,
                    settings=rng.choice(["mixed", "both", "nucleus", "top_k", "min_p", "temperature"]))
    if op in ("rope", "rope_backward"):
        width = rng.choice([32, 64, 64, 128, 128, 256, 80, 96, 50])
        kv_heads = rng.choice([1, 2, 4, 8, 12])
        heads = kv_heads * rng.choice([1, 1, 2, 4])
        count = _span(rng, 1, 8192)
        batch = _span(rng, 1, max(1, min(128, 160_000_000 // (count * (heads + kv_heads) * width))))
        return dict(op=op, type=kind, batch=batch, count=count, heads=heads, kv_heads=kv_heads, width=width,
                    rotary=rng.choice([width, width, width // 4 * 2]), layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "bands"]), longest=count + _span(rng, 1, 100000),
                    ragged=rng.random() < 0.5, fused=rng.random() < 0.5)
    width = _span(rng, 32, 16384)
    rows = _span(rng, 1, max(1, min(32768, 32_000_000 // width)))
    return dict(op=op, type=kind, rows=rows, width=width, residual=rng.random() < 0.7, weight=rng.random() < 0.7)


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _frequencies(case):
    """Radians a position, of each pair: 10000^(-2i / rotary), for longer contexts
    divided by a factor, or only where fewer than `high` turns fit into the
    original context (wholly under `low`, in proportion between them)."""
    f = 10000.0 ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64, device="cuda") / case["rotary"])
    if case["scaling"] == "linear":
        return f / 4.0
    if case["scaling"] == "bands":
        turns = 8192.0 * f / (2 * math.pi)
        share = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        return f * share + f / 128.0 * (1 - share)
    return f


def prepare(case, seed):
    g = _generator(seed)
    kind = TYPES[case["type"]]
    s = {"case": case}
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        z = torch.empty(rows, vocab, dtype=kind, device="cuda")
        for i in range(0, rows, 512):
            n = min(512, rows - i)
            part = torch.randn(n, vocab, generator=g, device="cuda") * (1 + 3 * torch.rand(n, 1, generator=g, device="cuda"))
            z[i:i + n] = part.to(kind)
        if rows >= 4 and vocab >= 32:  # one row in four allows every eighth token alone, as a grammar would
            z[1::4, (torch.arange(vocab, device="cuda") % 8) != 3] = -math.inf
        s["logits"] = z
        s["uniforms"] = torch.rand(rows, generator=g, device="cuda")
        some = lambda low, high: low + (high - low) * torch.rand(rows, generator=g, device="cuda")  # noqa: E731
        with_ = case["settings"]
        s["temperatures"] = some(0.6, 1.3)
        s["top_k"] = s["top_p"] = s["min_p"] = None
        if with_ in ("both", "mixed", "top_k"):
            s["top_k"] = torch.randint(20, 101, (rows,), generator=g, device="cuda", dtype=torch.int32)
        if with_ in ("both", "mixed", "nucleus"):
            s["top_p"] = some(0.8, 0.99)
        if with_ in ("min_p", "mixed"):
            s["min_p"] = some(0.01, 0.1)
        if with_ == "mixed":  # a request has each of the three or not, and one in eight is greedy
            s["top_k"] = torch.where(some(0, 1) < 0.5, s["top_k"], 0)
            s["top_p"] = torch.where(some(0, 1) < 0.5, s["top_p"], 1.0)
            s["min_p"] = torch.where(some(0, 1) < 0.5, s["min_p"], 0.0)
            s["temperatures"] = torch.where(some(0, 1) < 0.125, 0.0, s["temperatures"])
        return s
    if case["op"] in ("rope", "rope_backward"):
        b, n, h, hk, d = (case[x] for x in ("batch", "count", "heads", "kv_heads", "width"))
        if case["fused"]:
            x = torch.randn(b, n, h + 2 * hk, d, generator=g, device="cuda").to(kind)
            s["q"], s["k"] = x[:, :, :h], x[:, :, h:h + hk]
        else:
            s["q"] = torch.randn(b, n, h, d, generator=g, device="cuda").to(kind)
            s["k"] = torch.randn(b, n, hk, d, generator=g, device="cuda").to(kind)
        s["q_out"] = torch.zeros(b, n, h, d, dtype=kind, device="cuda")  # rows behind a sequence's own stay as they are
        s["k_out"] = torch.zeros(b, n, hk, d, dtype=kind, device="cuda")
        s["lengths"] = torch.randint(n, case["longest"] + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        s["lengths"][0] = case["longest"]
        s["counts"] = torch.full((b,), n, dtype=torch.int32, device="cuda")
        if case["ragged"]:
            s["counts"] = torch.randint(n // 4, n + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
            s["counts"][0] = n
        s["frequencies"] = _frequencies(case)
        s["magnitude"] = 1.0 if case["scaling"] == "none" else 0.1 * math.log(4.0) + 1.0
        return s
    rows, width = case["rows"], case["width"]
    of = lambda: torch.randn(rows, width, generator=g, device="cuda").to(kind)  # noqa: E731
    spread = torch.exp(0.5 * torch.randn(width, generator=g, device="cuda"))  # channels differ in size
    s["x"] = (of().float() * spread).to(kind)
    s["weight"] = (1 + 0.2 * torch.randn(width, generator=g, device="cuda")).to(kind) if case["weight"] else None
    if case["op"] == "norm_backward":  # x is the sum that the forward call kept
        s["rstd"] = torch.rsqrt(s["x"].double().square().mean(1) + EPSILON).float()
        s["d_out"] = of()
        s["d_sum"] = of() if case["residual"] else None
    else:
        s["residual"] = (3 * of().float()).to(kind) if case["residual"] else None
    return s


# ---- one pass ----------------------------------------------------------------

def run(state):
    if own:
        return _own(state)
    return {"sample": _plain_sample, "rope": _plain_rope, "rope_backward": _plain_rope, "norm": _plain_norm,
            "norm8": _plain_norm8, "norm_backward": _plain_norm_backward}[state["case"]["op"]](state)


def _plain_sample(s):
    z, order = s["logits"].float().sort(dim=1, descending=True, stable=True)
    rank = torch.arange(z.shape[1], device="cuda")[None]
    t = s["temperatures"].double()[:, None]
    greedy = t == 0
    w = ((z.double() - z[:, :1].double()) / torch.where(greedy, 1.0, t)).exp()
    w = torch.where(greedy & (rank > 0), 0.0, w)
    if s["top_k"] is not None:
        k = s["top_k"][:, None]
        w = torch.where((rank < k) | (k <= 0), w, 0.0)
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        before = w.cumsum(1) - w
        w = torch.where((before < p * w.sum(1, keepdim=True)) | (p >= 1) | (rank == 0), w, 0.0)
    if s["min_p"] is not None:
        w = torch.where((w >= s["min_p"].double()[:, None]) | (rank == 0), w, 0.0)
    total = w.sum(1, keepdim=True)
    reached = w.cumsum(1) <= s["uniforms"].double()[:, None] * total
    at = torch.minimum(reached.sum(1), (w > 0).sum(1) - 1)[:, None]
    return {"tokens": order.gather(1, at)[:, 0].to(torch.int32), "logprob": (w.gather(1, at) / total).log()[:, 0].float()}


def _plain_rope(s):
    case = s["case"]
    n, r, half = case["count"], case["rotary"], case["rotary"] // 2
    place = (s["lengths"] - s["counts"])[:, None] + torch.arange(n, device="cuda", dtype=torch.int32)[None]
    angle = place[:, :, None].double() * s["frequencies"]  # [b, n, half]
    c, sn = (angle.cos() * s["magnitude"]).float()[:, :, None], (angle.sin() * s["magnitude"]).float()[:, :, None]
    if case["op"] == "rope_backward":
        sn = -sn
    real = (torch.arange(n, device="cuda")[None] < s["counts"][:, None])[:, :, None, None]
    out = {}
    for name in ("q", "k"):
        x = s[name].float()
        if case["layout"] == "half":
            a, b = x[..., :half], x[..., half:r]
            y = torch.cat([a * c - b * sn, b * c + a * sn, x[..., r:]], 3)
        else:
            a, b = x[..., :r:2], x[..., 1:r:2]
            y = torch.cat([torch.stack([a * c - b * sn, b * c + a * sn], 4).flatten(3), x[..., r:]], 3)
        out[name] = torch.where(real, y, 0.0).to(s[name].dtype)
    return out


def _plain_sum(s):
    """The rows that are normalised, as they are kept."""
    if s["residual"] is None:
        return s["x"]
    return (s["x"].float() + s["residual"].float()).to(s["x"].dtype)


def _plain_norm(s):
    kept = _plain_sum(s)
    h = kept.float()
    rstd = torch.rsqrt(h.square().mean(1, keepdim=True) + EPSILON)
    y = h * rstd
    if s["weight"] is not None:
        y = y * s["weight"].float()
    out = {"out": y.to(s["x"].dtype), "rstd": rstd[:, 0]}
    if s["residual"] is not None:
        out["sum"] = kept
    return out


def _plain_norm8(s):
    kept = _plain_sum(s)
    h = kept.double()  # a block's largest value can lie next to a power of two
    y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPSILON)
    if s["weight"] is not None:
        y = y * s["weight"].double()
    rows, width = y.shape
    blocks = torch.nn.functional.pad(y, (0, -width % 32)).view(rows, -1, 32)
    top = blocks.abs().amax(2)
    m, e = torch.frexp(top)
    e = torch.where(top > 0, e - 9 + (m > 0.875).to(e.dtype), -1000).clamp(-117, 120)  # 448 is 0.875 * 2^9
    scaled = torch.ldexp(blocks, -e[:, :, None]).float()
    codes = scaled.to(torch.float8_e4m3fn).view(torch.uint8).view(rows, -1)[:, :width].contiguous()
    out = {"codes": codes.view(torch.float8_e4m3fn), "scales": (e + 127).to(torch.uint8)}
    if s["residual"] is not None:
        out["sum"] = kept
    return out


def _plain_norm_backward(s):
    rstd = s["rstd"][:, None]
    g, hat = s["d_out"].float(), s["x"].float() * rstd
    out = {}
    if s["weight"] is not None:
        out["d_weight"] = (g * hat).sum(0)
        g = g * s["weight"].float()
    d = rstd * (g - hat * (g * hat).mean(1, keepdim=True))
    if s["d_sum"] is not None:
        d = d + s["d_sum"].float()
    out["d_x"] = d.to(s["x"].dtype)
    return out


def _own(s):
    import grokking_abmod_amd as G

    case, op = s["case"], s["case"]["op"]
    kind, stream = {"f32": G.MG_F32, "f16": G.MG_F16, "bf16": G.MG_BF16}[case["type"]], torch.cuda.current_stream().cuda_stream
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    if op == "sample":
        z, rows = s["logits"], case["rows"]
        tokens = torch.empty(rows, dtype=torch.int32, device="cuda")
        logprob = torch.empty(rows, device="cuda")
        G.sample_filtered_noalloc(kind, z.data_ptr(), rows, case["vocab"], z.stride(0), at(s["temperatures"]),
                                  at(s["top_k"]), at(s["top_p"]), at(s["min_p"]), at(s["uniforms"]), tokens.data_ptr(),
                                  logprob.data_ptr(), stream)
        return {"tokens": tokens, "logprob": logprob}
    if op in ("rope", "rope_backward"):
        rope = G.Rope(case["width"], case["rotary"], G.MG_ROPE_HALF if case["layout"] == "half" else G.MG_ROPE_INTERLEAVED,
                      s["magnitude"], s["frequencies"].data_ptr())
        q, k, q_out, k_out = s["q"], s["k"], s["q_out"], s["k_out"]
        (G.rope if op == "rope" else G.rope_backward)(
            rope, kind, case["batch"], case["count"], case["heads"], q.data_ptr(), q.stride()[:3], q_out.data_ptr(),
            q_out.stride()[:3], case["kv_heads"], k.data_ptr(), k.stride()[:3], k_out.data_ptr(), k_out.stride()[:3],
            s["lengths"].data_ptr(), s["counts"].data_ptr(), None, stream)
        return {"q": q_out, "k": k_out}
    x, weight, rows, width = s["x"], s["weight"], case["rows"], case["width"]
    if op == "norm_backward":
        out = {}
        d_sum = s["d_sum"]
        if weight is not None:
            out["d_weight"] = torch.empty(width, device="cuda")
        out["d_x"] = torch.empty_like(x)
        room = G.rms_norm_backward_workspace(rows, width)
        space = torch.empty(room, dtype=torch.uint8, device="cuda") if room and weight is not None else None
        G.rms_norm_backward(kind, rows, width, x.data_ptr(), x.stride(0), at(weight), s["rstd"].data_ptr(),
                            s["d_out"].data_ptr(), s["d_out"].stride(0), at(d_sum), width, out["d_x"].data_ptr(), width,
                            at(out.get("d_weight")), at(space), room, stream)
        return out
    residual = s["residual"]
    out, kept = {}, None
    if op == "norm":
        out["out"], out["rstd"] = torch.empty_like(x), torch.empty(rows, device="cuda")
    else:
        codes = torch.empty(rows, width, dtype=torch.uint8, device="cuda")
        out["codes"] = codes.view(torch.float8_e4m3fn)
        out["scales"] = torch.empty(rows, (width + 31) // 32, dtype=torch.uint8, device="cuda")
    if residual is not None:
        kept = out["sum"] = torch.empty_like(x)
    if op == "norm":
        G.rms_norm(kind, rows, width, x.data_ptr(), x.stride(0), at(residual), width, at(kept), width, at(weight), EPSILON,
                   out["out"].data_ptr(), width, out["rstd"].data_ptr(), stream)
    else:
        G.rms_norm_e4m3(kind, rows, width, x.data_ptr(), x.stride(0), at(residual), width, at(kept), width, at(weight),
                        EPSILON, codes.data_ptr(), width, out["scales"].data_ptr(), out["scales"].stride(0), None, stream)
    return out


# ---- what a pass cannot do without ---------------------------------------------

def work(case):
    size = SIZE[case["type"]]
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + 28 * case["rows"], "flops": 4 * n}
    if case["op"] in ("rope", "rope_backward"):
        tokens = case["batch"] * case["count"] * (0.625 if case["ragged"] else 1.0)  # a quarter to all of the count
        n = tokens * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * n * case["width"] * size, "flops": 3 * n * case["rotary"]}
    n = case["rows"] * case["width"]
    extra = 4 * case["rows"] + (case["width"] * (size + 4) if case["weight"] else 0)
    if case["op"] == "norm_backward":
        return {"bytes": n * size * (4 if case["residual"] else 3) + extra, "flops": 9 * n}
    moved = size * (3 if case["residual"] else 1) + (size if case["op"] == "norm" else 1 + 1 / 32)
    return {"bytes": n * moved + extra, "flops": 5 * n}


# ---- the definitions in 64 bits ------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"sample": _exact_sample, "rope": _exact_rope, "rope_backward": _exact_rope, "norm": _exact_norm,
            "norm8": _exact_norm8, "norm_backward": _exact_norm_backward}[case["op"]](case, s)


def _exact_sample(case, s):
    """Row by row: the probabilities of the ranked tokens, cut one filter after the other."""
    tokens, logprob = [], []
    for r in range(case["rows"]):
        z = s["logits"][r].double()
        order = torch.argsort(-z, stable=True)
        t = float(s["temperatures"][r])
        if t == 0:
            tokens.append(order[:1])
            logprob.append(torch.zeros(1, dtype=torch.float64, device="cuda"))
            continue
        ranked = z[order] / t
        if s["top_k"] is not None and int(s["top_k"][r]) > 0:
            ranked = ranked[:int(s["top_k"][r])]
        p = torch.softmax(ranked, 0)
        if s["top_p"] is not None and float(s["top_p"][r]) < 1:
            wanted = float(s["top_p"][r])
            p = p[:int(torch.searchsorted(p.cumsum(0), torch.tensor([wanted], dtype=torch.float64, device="cuda"))[0]) + 1]
        if s["min_p"] is not None:
            p = p[:max(1, int((p >= float(s["min_p"][r]) * p[0]).sum()))]
        p = p[p > 0]
        share = p.cumsum(0) / p.sum()
        at = int(torch.searchsorted(share, s["uniforms"][r].double()[None], right=True)[0].clamp(max=p.numel() - 1))
        tokens.append(order[at:at + 1])
        logprob.append((p[at] / p.sum()).log()[None])
    return {"tokens": torch.cat(tokens).to(torch.int32), "logprob": torch.cat(logprob)}


def _exact_rope(case, s):
    """Each pair as a complex number, times the unit number of its angle."""
    r, sign = case["rotary"], -1.0 if case["op"] == "rope_backward" else 1.0
    out = {}
    for name in ("q", "k"):
        y = torch.zeros(s[name].shape, dtype=torch.float64, device="cuda")
        for b in range(case["batch"]):
            new = int(s["counts"][b])
            place = int(s["lengths"][b]) - new + torch.arange(new, dtype=torch.float64, device="cuda")
            x = s[name][b, :new].double()
            turn = torch.polar(torch.full((), s["magnitude"], dtype=torch.float64, device="cuda").expand(new, r // 2).contiguous(),
                               sign * torch.outer(place, s["frequencies"]))[:, None]
            part = x[..., :r]
            pairs = part.unflatten(2, (2, r // 2)).transpose(2, 3) if case["layout"] == "half" else part.unflatten(2, (r // 2, 2))
            turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            y[b, :new, :, :r] = turned.transpose(2, 3).flatten(2) if case["layout"] == "half" else turned.flatten(2)
            y[b, :new, :, r:] = x[..., r:]
        out[name] = y
    return out


def _exact_kept(s):
    """What a call keeps is part of its definition: the sum, rounded to the rows' type."""
    if s["residual"] is None:
        return s["x"].double()
    return (s["x"].double() + s["residual"].double()).to(s["x"].dtype).double()


def _exact_norm(case, s):
    h = _exact_kept(s)
    rstd = 1 / torch.sqrt((h * h).sum(1) / case["width"] + EPSILON)
    out = {"out": torch.einsum("ij,i->ij", h, rstd) * (1.0 if s["weight"] is None else s["weight"].double()), "rstd": rstd}
    if s["residual"] is not None:
        out["sum"] = s["x"].double() + s["residual"].double()
    return out


def _exact_norm8(case, s):
    h = _exact_kept(s)
    y = h / torch.sqrt((h * h).sum(1, keepdim=True) / case["width"] + EPSILON)
    if s["weight"] is not None:
        y = y * s["weight"].double()
    codes, scales = torch.empty_like(y), []
    for i in range(0, case["width"], 32):
        block = y[:, i:i + 32]
        top = block.abs().amax(1)
        e = torch.where(top > 0, torch.ceil(torch.log2(top / 448)), -1000.0)
        e = torch.where(448 * torch.exp2(e) < top, e + 1, torch.where(448 * torch.exp2(e - 1) >= top, e - 1, e)).clamp(-117, 120)
        v = block / torch.exp2(e)[:, None]
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
        codes[:, i:i + 32] = torch.round(v / step) * step
        scales.append(e + 127)
    out = {"codes": codes, "scales": torch.stack(scales, 1).to(torch.uint8)}
    if s["residual"] is not None:
        out["sum"] = s["x"].double() + s["residual"].double()
    return out


def _exact_norm_backward(case, s):
    """Of sum(d_out * (x rstd w)), where rstd depends on x: rstd^3 / width is what d(rstd) / dx carries."""
    x, g, rstd = s["x"].double(), s["d_out"].double(), s["rstd"].double()[:, None]
    out = {}
    if s["weight"] is not None:
        out["d_weight"] = (g * x * rstd).sum(0)
        g = g * s["weight"].double()
    d = g * rstd - x * (rstd ** 3 / case["width"]) * (g * x).sum(1, keepdim=True)
    out["d_x"] = d if s["d_sum"] is None else d + s["d_sum"].double()
    return out
