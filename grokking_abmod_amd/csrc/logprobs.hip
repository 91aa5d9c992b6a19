// Log probabilities of given tokens under rows of logits z at a temperature T,
// with the entropy and the best alternatives, and their gradient.
//
//   d_v = (z_v - max z) / T,  S = sum_v exp(d_v),  log p_v = d_v - ln S
//   entropy H = ln S - sum_v exp(d_v) d_v / S
//   dz_v = [g (1[v = token] - p_v) - h p_v (log p_v + H)] / T
//
// The forward pass reads a row once: each thread keeps its running maximum, the
// sum and the sum of exp(d) d against it, in FP32, and they join at the end.
// The alternatives come out of the same pass.  The k-th largest of the threads'
// maxima bounds the k-th largest logit from below, so only the threads whose
// maximum reaches it hold any of the best k; those look at their logits again
// (from the cache) and a few more than k of them are sorted by counting.
// Reading the logits is what bounds it.  Rows are cut into chunks of at most
// 64 logits a thread, so that the logits over the bound always fit the list,
// and shorter ones where there are few rows; a second launch joins a row's chunks.
// Rows of up to 1024 logits stay in a wave's registers.  1000 BF16 rows of
// 128001 logits with 20 alternatives take 72 us (3.6 TB/s; 61 where the same logits
// come again and some of them lie in the Infinity Cache) and 6 us for the join, 20000 of
// 1000 with 32 take 33 us, and 22 with none.
//
// The gradient reads and writes each logit once, which bounds it, closely followed by
// its instructions (4096 BF16 rows of 50257: 6.2 TB/s, vector units busy for 0.9).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>

#include "dpp.hpp"
#include "operators.hpp"
#include "types.hpp"

namespace meshgpt::kern {
namespace {

constexpr int kBlock = 256;
constexpr int kSmall = kSmallVocab;    // logits of a row that one wave holds
constexpr int kThreadMost = 64;        // logits of a thread's share of a chunk, at most
constexpr int kList = 2048;            // candidates of a chunk: kTopMax threads' shares
constexpr int kHeld = 128;             // candidates of such a row
constexpr uint32_t kIgnore = 0xffffffffu;
constexpr float kLog2e = 1.4426950408889634f;

// A thread's share of a chunk is its groups and at most one logit before and
// behind them.
constexpr int kChunkMost = kBlock * (kThreadMost - 16);
static_assert(kTopMax * kThreadMost <= kList, "the logits over the bound fit the list");
constexpr int kChunksMost = (1 << 24) / kChunkMost + 1;

// Orders as the floats do, -0 with 0; NaN is not asked for.
__device__ __forceinline__ uint32_t order(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unorder(uint32_t k) {
    return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// Larger logits first, of equal ones the lower token.
__device__ __forceinline__ uint64_t candidate(uint32_t k, uint32_t token) { return (uint64_t(k) << 32) | uint32_t(~token); }

// Maximum, sum and sum of exp(d) d of some logits.  `m` starts at -inf; sums
// are against max(m, -FLT_MAX), so that -inf logits add 0 to both.
struct Sums {
    float m = -INFINITY, s = 0.0f, a = 0.0f;
    // The sums against a maximum of at least `top`.
    __device__ __forceinline__ void raise(float top, float c) {
        const float to = fmaxf(m, top), step = fmaxf((fmaxf(m, -FLT_MAX) - fmaxf(to, -FLT_MAX)) * c, -1e20f);
        const float f = __builtin_amdgcn_exp2f(step);
        a = f * fmaf(step, s, a);
        s *= f;
        m = to;
    }
    __device__ __forceinline__ void join(float m2, float s2, float a2, float c) {
        Sums o;
        o.m = m2;
        o.s = s2;
        o.a = a2;
        raise(m2, c);
        o.raise(m, c);
        s += o.s;
        a += o.a;
    }
};

// d in log2 units against base; exp(d) d of -inf is 0.
__device__ __forceinline__ void add(float x, float base, float c, float &s, float &a) {
    const float d = __builtin_elementwise_maximum((x - base) * c, -1000.0f), e = __builtin_amdgcn_exp2f(d);
    s += e;
    a = fmaf(e, d, a);
}

__device__ __forceinline__ void wave_join(Sums &t, float c) {
    t.raise(wave_largest(t.m), c);
    t.s = wave_sum(t.s);
    t.a = wave_sum(t.a);
}

// A row's results from its sums (a in log2 units); one thread.
template <class T>
__device__ __forceinline__ void write_row(const LogprobArgs &a, size_t row, const Sums &t, float &log_sum) {
    const auto *z = static_cast<const typename T::Raw *>(a.logits) + row * a.stride;
    const bool empty = t.s == 0.0f;  // no token is allowed: log probabilities are -inf
    log_sum = empty ? -INFINITY : logf(t.s);
    if (a.logprob) {
        const uint32_t token = a.tokens[row];
        float v = 0.0f;
        if (token != kIgnore) {
            if (token >= a.vocab)
                v = __builtin_nanf("");
            else
                v = empty ? -INFINITY : (T::to_float(z[token]) - t.m) * a.inv_temperature - log_sum;
        }
        a.logprob[row] = v;
    }
    if (a.entropy) a.entropy[row] = empty ? 0.0f : log_sum - t.a / (t.s * kLog2e);
    if (a.stats) {
        a.stats[2 * row] = t.s == t.s ? t.m : __builtin_nanf("");
        a.stats[2 * row + 1] = log_sum;
    }
}

// Alternative i of a row.  A row with a NaN or +inf has no probabilities (s is
// NaN): its alternatives are its first tokens, at NaN.
__device__ __forceinline__ void write_top(const LogprobArgs &a, size_t row, int i, uint64_t best, const Sums &t,
                                          float log_sum) {
    const bool none = !(t.s == t.s);
    const uint32_t token = none ? uint32_t(i) : ~uint32_t(best);
    a.top_tokens[row * a.top + i] = token;
    if (a.top_logprobs)
        a.top_logprobs[row * a.top + i] =
            none ? __builtin_nanf("")
                 : t.s == 0.0f ? -INFINITY : (unorder(uint32_t(best >> 32)) - t.m) * a.inv_temperature - log_sum;
}

// Rows of up to 64 N logits, a wave a row.
template <class T, int N>
__global__ void __launch_bounds__(kBlock) logprob_small_kernel(LogprobArgs a) {
    const size_t row = size_t(blockIdx.x) * (kBlock / 64) + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= a.rows) return;
    const auto *z = static_cast<const typename T::Raw *>(a.logits) + row * a.stride;
    const float c = a.inv_temperature * kLog2e;
    float x[N];
    Sums t;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t v = lane + 64 * i;
        x[i] = v < a.vocab ? T::to_float(z[v]) : -INFINITY;
        t.m = fmaxf(t.m, x[i]);
    }
    const float base = fmaxf(t.m, -FLT_MAX);
#pragma unroll
    for (int i = 0; i < N; ++i) add(x[i], base, c, t.s, t.a);
    wave_join(t, c);
    float log_sum = 0.0f;
    if (lane == 0) write_row<T>(a, row, t, log_sum);
    if (!a.top) return;
    log_sum = __shfl(log_sum, 0, 64);
    if (!(t.s == t.s)) {  // a NaN
        if (lane < a.top) write_top(a, row, lane, 0, t, log_sum);
        return;
    }
    uint32_t k[N];
#pragma unroll
    for (int i = 0; i < N; ++i) k[i] = lane + 64 * i < int(a.vocab) ? order(x[i]) : 0;
    // As in a chunk, the top-th largest of the lanes' maxima bounds the top-th
    // largest logit; where too many reach it (equal ones), that one itself.  20000
    // BF16 rows of 1000 with 1, 2, 5 and 32 alternatives take 29, 29, 30 and 33 us;
    // taking the largest of what is left once for each took 26, 29, 39 and 147.
    uint32_t best = k[0];
#pragma unroll
    for (int i = 1; i < N; ++i) best = max(best, k[i]);
    uint32_t least = 0;
    for (uint32_t bit = 1u << 31; bit; bit >>= 1) {
        const int n = __popcll(__ballot(best >= (least | bit)));
        if (n >= a.top) least |= bit;
        if (n == a.top) break;  // it parts them as well as the top-th does
    }
    __shared__ uint64_t list[kBlock / 64][kHeld];
    uint64_t *const mine = list[threadIdx.x >> 6];
    const uint64_t below = (uint64_t(1) << lane) - 1;
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint64_t all = __ballot(k[i] >= least);
        const int at = n + __popcll(all & below);
        if (k[i] >= least && at < kHeld) mine[at] = candidate(k[i], lane + 64 * i);
        n += __popcll(all);
    }
    if (n > kHeld) {
        least = 0;
        for (uint32_t bit = 1u << 31; bit; bit >>= 1) {
            n = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) n += __popcll(__ballot(k[i] >= (least | bit)));
            if (n >= a.top) least |= bit;
        }
        // The larger ones, and of equal ones the first.
        int larger = 0, equal = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) equal += __popcll(__ballot(k[i] > least));
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint64_t above = __ballot(k[i] > least), same = __ballot(k[i] == least);
            const int at = k[i] > least ? larger + __popcll(above & below) : equal + __popcll(same & below);
            if (k[i] >= least && at < a.top) mine[at] = candidate(k[i], lane + 64 * i);
            larger += __popcll(above);
            equal += __popcll(same);
        }
        n = a.top;
    }
    __builtin_amdgcn_wave_barrier();
    for (int j = lane; j < n; j += 64) {
        const uint64_t v = mine[j];
        int before = 0;
        for (int o = 0; o < n; ++o) before += mine[o] > v;
        if (before < a.top) write_top(a, row, before, v, t, log_sum);
    }
}

// One chunk of a row.
template <class T>
__global__ void __launch_bounds__(kBlock) logprob_kernel(LogprobArgs a) {
    using Raw = typename T::Raw;
    constexpr int G = T::kGroup;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t row = blockIdx.x / uint32_t(a.chunks);
    const int chunk = int(blockIdx.x - uint32_t(row) * uint32_t(a.chunks));
    const auto *z = static_cast<const Raw *>(a.logits) + row * a.stride;
    const float c = a.inv_temperature * kLog2e;
    const uint32_t lo = uint32_t(chunk) * uint32_t(a.chunk);
    const uint32_t hi = uint32_t(min(size_t(lo) + size_t(a.chunk), a.vocab));
    // [lo, body) and [tail, hi) lie outside whole 16-byte groups.
    const uint32_t off = uint32_t(reinterpret_cast<uintptr_t>(z + lo) % 16 / sizeof(Raw));
    const uint32_t body = min(hi, lo + (G - off) % G), groups = (hi - body) / G, tail = body + groups * G;
    const uint4 *const zg = reinterpret_cast<const uint4 *>(z + body);

    Sums t;
    auto one = [&](float x) {
        if (x > t.m) t.raise(x, c);
        add(x, fmaxf(t.m, -FLT_MAX), c, t.s, t.a);
    };
    if (uint32_t(tid) < body - lo) one(T::to_float(z[lo + tid]));
    if (uint32_t(tid) < hi - tail) one(T::to_float(z[tail + tid]));
    // All groups of a 16-bit chunk are under way at once, half of an F32 one's, and
    // their maximum comes first, so that sums are raised once.
    for (uint32_t i = tid; i < groups; i += 6 * kBlock) {
        uint4 w[6];
#pragma unroll
        for (int u = 0; u < 6; ++u) w[u] = zg[min(i + u * kBlock, groups - 1)];
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < 6; ++u) {
            float x[G];
            T::unpack(w[u], x);
            if (i + u * kBlock >= groups) continue;
#pragma unroll
            for (int j = 0; j < G; ++j) top = fmaxf(top, x[j]);
        }
        if (top > t.m) t.raise(top, c);
        const float base = fmaxf(t.m, -FLT_MAX);
#pragma unroll
        for (int u = 0; u < 6; ++u) {
            if (i + u * kBlock >= groups) continue;
            float x[G];
            T::unpack(w[u], x);
            float s = 0.0f, q = 0.0f;
#pragma unroll
            for (int j = 0; j < G; ++j) add(x[j], base, c, s, q);
            t.s += s;
            t.a += q;
        }
    }

    __shared__ float joined[kBlock / 64][3];
    __shared__ uint32_t tops[kBlock];
    __shared__ uint32_t bound, found, over, picked;
    __shared__ uint8_t picks[kBlock];
    __shared__ uint64_t list[kList];
    const bool any = uint32_t(tid) < body - lo || uint32_t(tid) < hi - tail || uint32_t(tid) < groups;
    const uint32_t mine = any ? order(t.m) : 0;
    if (a.top) tops[tid] = mine;
    wave_join(t, c);
    if (lane == 0) {
        joined[wave][0] = t.m;
        joined[wave][1] = t.s;
        joined[wave][2] = t.a;
    }
    if (tid == 0) found = over = picked = 0;
    __syncthreads();
    t.m = joined[0][0];
    t.s = joined[0][1];
    t.a = joined[0][2];
#pragma unroll
    for (int w = 1; w < kBlock / 64; ++w) t.join(joined[w][0], joined[w][1], joined[w][2], c);
    float log_sum = 0.0f;
    if (a.chunks > 1) {
        if (tid == 0) {
            float *p = a.part_stats + (row * a.chunks + chunk) * 3;
            p[0] = t.m;
            p[1] = t.s;
            p[2] = t.a;
        }
    } else {
        if (tid == 0) write_row<T>(a, row, t, log_sum);
        log_sum = t.s == 0.0f ? -INFINITY : logf(t.s);
    }
    if (!a.top) return;
    uint64_t *const part = a.part_top + (row * a.chunks + chunk) * a.top;
    const int top = a.top, have = int(min(uint32_t(top), hi - lo));  // the chunk may hold fewer
    if (!(t.s == t.s)) {  // a NaN: any tokens do, they are not used
        if (tid < top) {
            if (a.chunks > 1)
                part[tid] = 0;
            else
                write_top(a, row, tid, 0, t, log_sum);
        }
        return;
    }
    // The have-th largest of the threads' maxima, bit by bit, where so many
    // threads hold any; with fewer (a short chunk) every logit is looked at.
    if (wave == 0) {
        uint32_t k[kBlock / 64], at = 0;
#pragma unroll
        for (int w = 0; w < kBlock / 64; ++w) k[w] = tops[lane + 64 * w];
        for (uint32_t bit = 1u << 31; bit; bit >>= 1) {
            int n = 0;
#pragma unroll
            for (int w = 0; w < kBlock / 64; ++w) n += __popcll(__ballot(k[w] >= (at | bit)));
            if (n >= have) at |= bit;
            if (n == have) break;  // it parts them as well as the have-th does
        }
        if (lane == 0) bound = at;
    }
    __syncthreads();
    const uint32_t least = bound;
    auto offer = [&](float x, uint32_t v, uint32_t from) {
        const uint32_t k = order(x);
        if (k < from) return;
        const uint32_t at = atomicAdd(&found, 1u);
        if (at < uint32_t(kList))
            list[at] = candidate(k, v);
        else
            over = 1;
    };
    // The shares of the threads that hold any, spread over all threads.
    const uint32_t steps = (groups + kBlock - 1) / kBlock + 1;
    auto look = [&](uint32_t from) {
        if (any && mine >= from) picks[atomicAdd(&picked, 1u)] = uint8_t(tid);
        __syncthreads();
        for (uint32_t i = tid; i < picked * steps; i += kBlock) {
            const uint32_t who = picks[i / steps], step = i % steps, j = who + step * kBlock;
            if (step + 1 == steps) {  // what lies outside the groups
                if (who < body - lo) offer(T::to_float(z[lo + who]), lo + who, from);
                if (who < hi - tail) offer(T::to_float(z[tail + who]), tail + who, from);
            } else if (j < groups) {
                float x[G];
                T::unpack(zg[j], x);
#pragma unroll
                for (int e = 0; e < G; ++e) offer(x[e], body + j * G + e, from);
            }
        }
        __syncthreads();
    };
    look(least);
    if (over) {
        // Many logits equal the bound (most of a masked row, say): the ones
        // over it, which fit, then equal ones in the order of their tokens
        // until there are enough.
        __syncthreads();
        if (tid == 0) found = picked = 0;
        __syncthreads();
        look(least + 1);
        for (uint32_t from = lo; from < hi; from += kBlock) {
            if (found >= uint32_t(have)) break;
            __syncthreads();
            const uint32_t v = from + tid;
            if (v < hi && order(T::to_float(z[v])) == least) {
                const uint32_t at = atomicAdd(&found, 1u);
                list[min(at, uint32_t(kList - 1))] = candidate(least, v);
            }
            __syncthreads();
        }
    }
    // A candidate's place is the number of those before it.
    const int n = min(int(found), kList);
    for (int j = tid; j < n; j += kBlock) {
        const uint64_t v = list[j];
        int before = 0;
        for (int o = 0; o < n; ++o) before += list[o] > v;
        if (before < top) {
            if (a.chunks > 1)
                part[before] = v;
            else
                write_top(a, row, before, v, t, log_sum);
        }
    }
    if (a.chunks > 1 && tid >= have && tid < top) part[tid] = 0;
}

// Joins a row's chunks: a workgroup, whose waves each have all the sums.  Of the
// chunks' n-th best candidates, with n * chunks >= top, the (top / n)-th largest
// bounds the top-th best of the row from below; the few candidates that reach it
// take their places by counting.
template <class T>
__global__ void __launch_bounds__(kBlock) logprob_join_kernel(LogprobArgs a) {
    const size_t row = blockIdx.x;
    const int tid = threadIdx.x, threads = blockDim.x, n = a.chunks * a.top;
    const float c = a.inv_temperature * kLog2e;
    const uint64_t *const lists = a.part_top + row * a.chunks * a.top;
    uint64_t next = tid < n ? lists[tid] : 0;
    Sums t;
    for (int k = tid & 63; k < a.chunks; k += 64) {
        const float *p = a.part_stats + (row * a.chunks + k) * 3;
        t.join(p[0], p[1], p[2], c);
    }
    wave_join(t, c);
    float log_sum = 0.0f;
    if (tid == 0) write_row<T>(a, row, t, log_sum);
    if (!a.top) return;
    log_sum = t.s == 0.0f ? -INFINITY : logf(t.s);
    if (!(t.s == t.s)) {  // a NaN
        if (tid < a.top) write_top(a, row, tid, 0, t, log_sum);
        return;
    }
    __shared__ uint64_t nth[kChunksMost], list[kTopMax * kTopMax], bound;
    __shared__ uint32_t found;
    const int each = (a.top + a.chunks - 1) / a.chunks, most = (a.top + each - 1) / each;
    for (int k = tid; k < a.chunks; k += threads) nth[k] = lists[size_t(k) * a.top + each - 1];
    if (tid == 0) bound = found = 0;
    __syncthreads();
    for (int k = tid; k < a.chunks; k += threads) {
        const uint64_t v = nth[k];
        int before = 0;
        for (int o = 0; o < a.chunks; ++o) before += nth[o] > v;
        if (v && before == most - 1) bound = v;  // 0: fewer chunks have as many
    }
    __syncthreads();
    // At most `most` chunks have more than each - 1 candidates from the bound on.
    const uint64_t least = bound;
    for (int i = tid; i < n; i += threads) {
        if (i != tid) next = lists[i];
        if (next && next >= least) list[atomicAdd(&found, 1u)] = next;
    }
    __syncthreads();
    for (int j = tid; j < int(found); j += threads) {
        const uint64_t v = list[j];
        int before = 0;
        for (int o = 0; o < int(found); ++o) before += list[o] > v;
        if (before < a.top) write_top(a, row, before, v, t, log_sum);
    }
}

constexpr int kGradGroups = 3;  // 16-byte groups of a lane
template <class T>
constexpr size_t kLine = 128 / sizeof(typename T::Raw);
// Logits of a share at most, beside what moves a row's shares to whole lines.
template <class T>
constexpr size_t kGradMost = 64 * kGradGroups * T::kGroup - kLine<T>;
static_assert(kGradMost<F32> == kGradRun && kGradMost<BF16> >= kGradRun, "as the launch's size is checked");

template <class T>
__device__ __forceinline__ float grad_of(float x, uint32_t v, const LogprobBackwardArgs &a, uint32_t token, float m,
                                         float log_sum, float g, float h, float entropy) {
    // log p in natural units; a row without any allowed token has m = -inf.
    const float lp = (x - m) * a.inv_temperature - log_sum, p = __builtin_amdgcn_exp2f(lp * kLog2e);
    const float of_p = h == 0.0f ? g : fmaf(h, (p > 0.0f ? lp : 0.0f) + entropy, g);
    float d = -p * of_p;
    if (v == token) d += g;
    return d * a.inv_temperature;
}

// A wave's share of a row: `size` logits, all under way at once.  Shares end at
// 128-byte lines.  Short shares keep what is read and written at a time close
// together in memory: 4096 BF16 rows of 50257 take 192 us with 32768 logits a
// workgroup, 146 with 2048 a wave, 140 with 1536, 147 with 1024; past the caches
// 133 (6.2 TB/s).
template <class T, bool STREAM>
__global__ void __launch_bounds__(kBlock) logprob_backward_kernel(LogprobBackwardArgs a, uint32_t shares, uint32_t size) {
    using Raw = typename T::Raw;
    constexpr int G = T::kGroup;
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t unit = blockIdx.x * (kBlock / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const size_t row = unit / shares;
    if (row >= a.rows) return;
    const uint32_t share = unit - uint32_t(row) * shares;
    const auto *z = static_cast<const Raw *>(a.logits) + row * a.stride;
    auto *out = static_cast<Raw *>(a.d_logits) + row * a.d_stride;
    const uint32_t token = a.tokens ? a.tokens[row] : kIgnore;
    const float m = a.stats[2 * row], log_sum = a.stats[2 * row + 1];
    const bool scored = a.d_logprob && token != kIgnore;
    float g = scored ? a.d_logprob[row] : 0.0f;
    if (scored && token >= a.vocab) g = __builtin_nanf("");
    const float h = a.d_entropy ? a.d_entropy[row] : 0.0f, entropy = a.d_entropy ? a.entropy[row] : 0.0f;
    // No token is allowed, so that nothing depends on the logits, or nothing is asked
    // of the row, whose logits may then be anything (0 times its NaN would be NaN).
    const bool none = m == -INFINITY || (!scored && h == 0.0f);
    auto grad = [&](float x, uint32_t v) {
        return none ? 0.0f : grad_of<T>(x, v, a, token, m, log_sum, g, h, entropy);
    };
    const uint32_t shift = uint32_t(reinterpret_cast<uintptr_t>(z) % 128 / sizeof(Raw));
    const uint32_t lo = share ? share * size - shift : 0;
    const uint32_t hi = share + 1 == shares ? uint32_t(a.vocab) : (share + 1) * size - shift;
    const uint32_t off = uint32_t(reinterpret_cast<uintptr_t>(z + lo) % 16);
    if (off != uint32_t(reinterpret_cast<uintptr_t>(out + lo) % 16)) {  // no common 16-byte groups
        for (uint32_t v = lo + lane; v < hi; v += 64) out[v] = T::from_float(grad(T::to_float(z[v]), v));
        return;
    }
    const uint32_t body = min(hi, lo + (G - off / uint32_t(sizeof(Raw))) % G), groups = (hi - body) / G,
                   tail = body + groups * G;
    if (lane < body - lo) out[lo + lane] = T::from_float(grad(T::to_float(z[lo + lane]), lo + lane));
    if (lane < hi - tail) out[tail + lane] = T::from_float(grad(T::to_float(z[tail + lane]), tail + lane));
    if (groups == 0) return;
    const uint4 *const zg = reinterpret_cast<const uint4 *>(z + body);
    uint4 *const og = reinterpret_cast<uint4 *>(out + body);
    uint4 w[kGradGroups];
#pragma unroll
    for (int u = 0; u < kGradGroups; ++u) w[u] = get<STREAM>(zg + min(lane + 64 * u, groups - 1));
#pragma unroll
    for (int u = 0; u < kGradGroups; ++u) {
        const uint32_t i = lane + 64 * u;
        if (i >= groups) continue;
        float x[G];
        T::unpack(w[u], x);
#pragma unroll
        for (int j = 0; j < G; ++j) x[j] = grad(x[j], body + i * G + j);
        put<STREAM>(og + i, __builtin_bit_cast(u32x4, T::pack(x)));
    }
}

template <class T>
void forward_of(const LogprobArgs &a, hipStream_t stream) {
    if (a.vocab <= size_t(kSmall)) {
        const dim3 grid(uint32_t((a.rows + kBlock / 64 - 1) / (kBlock / 64)));
        if (a.vocab <= 256)
            hipLaunchKernelGGL((logprob_small_kernel<T, 4>), grid, dim3(kBlock), 0, stream, a);
        else
            hipLaunchKernelGGL((logprob_small_kernel<T, kSmall / 64>), grid, dim3(kBlock), 0, stream, a);
        return;
    }
    hipLaunchKernelGGL((logprob_kernel<T>), dim3(uint32_t(a.rows * size_t(a.chunks))), dim3(kBlock), 0, stream, a);
    if (a.chunks > 1)
        hipLaunchKernelGGL((logprob_join_kernel<T>), dim3(uint32_t(a.rows)), dim3(a.top ? kBlock : 64), 0, stream, a);
}

template <class T>
void backward_of(const LogprobBackwardArgs &a, hipStream_t stream) {
    // Equal shares, of whole lines; the first is shorter by what its row lies off a
    // line, the last may be longer by as much.
    const size_t parts = (a.vocab + kGradMost<T> - 1) / kGradMost<T>, even = (a.vocab + parts - 1) / parts;
    const size_t size = (even + kLine<T> - 1) / kLine<T> * kLine<T>, shares = (a.vocab + size - 1) / size;
    const size_t units = a.rows * shares;
    const dim3 grid(uint32_t((units + kBlock / 64 - 1) / (kBlock / 64)));
    if (double(a.rows) * double(a.vocab) * sizeof(typename T::Raw) > kCached)
        hipLaunchKernelGGL((logprob_backward_kernel<T, true>), grid, dim3(kBlock), 0, stream, a, uint32_t(shares),
                           uint32_t(size));
    else
        hipLaunchKernelGGL((logprob_backward_kernel<T, false>), grid, dim3(kBlock), 0, stream, a, uint32_t(shares),
                           uint32_t(size));
}

}  // namespace

void logprob_chunks(size_t rows, size_t vocab, int &chunks, int &chunk) {
    chunks = 1;
    chunk = int(vocab);
    if (vocab <= size_t(kSmall)) return;
    // About 1024 workgroups, each of 2048 logits or more, and even.
    size_t want = std::min<size_t>((1024 + rows - 1) / std::max<size_t>(rows, 1), (vocab + 2047) / 2048);
    want = std::max<size_t>(want, (vocab + kChunkMost - 1) / kChunkMost);
    const size_t size = std::min<size_t>(((vocab + want - 1) / want + 63) / 64 * 64, size_t(kChunkMost));
    chunk = int(size);
    chunks = int((vocab + size - 1) / size);
}

void token_logprobs(const LogprobArgs &a, Type type, hipStream_t stream) {
    switch (type) {
    case Type::F32: return forward_of<F32>(a, stream);
    case Type::F16: return forward_of<F16>(a, stream);
    default: return forward_of<BF16>(a, stream);
    }
}

void token_logprobs_backward(const LogprobBackwardArgs &a, Type type, hipStream_t stream) {
    switch (type) {
    case Type::F32: return backward_of<F32>(a, stream);
    case Type::F16: return backward_of<F16>(a, stream);
    default: return backward_of<BF16>(a, stream);
    }
}

}  // namespace meshgpt::kern
