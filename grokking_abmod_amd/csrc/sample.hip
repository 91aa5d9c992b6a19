// Sampling with temperature, top-k, top-p and min-p from given random numbers.
//
// Tokens are ranked by their logits z, the largest first, of equal ones the
// lowest token first.  With w_j = exp((z_j - max z) / T), the first top_k in
// rank are left; of these the shortest run from the first whose weights reach
// top_p of theirs; of these the ones with w >= min_p; and u picks the first
// token in rank at which the sum of what is left exceeds u times the whole.
// Everything is a prefix of the ranking, so no row is sorted: a border is found
// by the weights of bins, and inside one bin by sorting that bin.
//
// A row has a workgroup.  Where the candidates are few (top_k bounds them by
// the k-th largest of the threads' maxima, min_p by itself), they are gathered
// and sorted.  Else the row goes into kBins bins of (max z - z) / T, 64 for each
// power of e, and the bins that hold a border or the drawn token are gathered.
// A bin with too many tokens is divided by the bits of its logits until it has
// few enough or all are equal.
//
// Sums decide which of many close borders is met: at 100000 equally likely
// tokens one is 1e-5 of the whole.  So weights are summed in 64 bits: a bin's as
// a count and a fixed-point sum of 1 - w / (w at its begin), in one LDS word, exact
// to 2^-34 of a weight and the same in any order; gathered ones in FP64.
#include <cfloat>

#include "dpp.hpp"
#include "operators.hpp"
#include "types.hpp"

namespace meshgpt::kern {
namespace {

constexpr int kBins = 2048;
constexpr double kPerUnit = 64.0;  // bins of a factor e
constexpr int kMost = 2048;        // tokens that are sorted at a time, in long rows
constexpr int kShort = 1024;       // rows of so many logits are sorted whole
constexpr uint32_t kNoToken = 0xffffffffu;

// Logits as integers in the same order; -0 is 0.
__device__ __forceinline__ uint32_t order(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t k) {
    return __builtin_bit_cast(float, k ^ (uint32_t(int32_t(~k) >> 31) | 0x80000000u));
}
// Ranked by the logit, then the lowest token.
__device__ __forceinline__ uint64_t candidate(float x, uint32_t token) {
    return uint64_t(order(x)) << 32 | uint32_t(~token);
}

// f(logit, token) for every logit of a row, 16 bytes a load, four loads under way.
template <class T, int THREADS, class F>
__device__ __forceinline__ void each(const typename T::Raw *z, uint32_t vocab, F &&f) {
    constexpr int G = T::kGroup, U = 4;
    const uint32_t groups = vocab / G;
    uint32_t j = threadIdx.x;
    for (; j + (U - 1) * THREADS < groups; j += U * THREADS) {
        uint4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = get_any(z + size_t(j + u * THREADS) * G);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float x[G];
            T::unpack(w[u], x);
#pragma unroll
            for (int e = 0; e < G; ++e) f(x[e], (j + u * THREADS) * G + e);
        }
    }
    for (; j < groups; j += THREADS) {
        float x[G];
        T::unpack(get_any(z + size_t(j) * G), x);
#pragma unroll
        for (int e = 0; e < G; ++e) f(x[e], j * G + e);
    }
    const uint32_t last = groups * G + threadIdx.x;
    if (last < vocab) f(T::to_float(z[last]), last);
}

template <class V>
__device__ __forceinline__ V wave_scan(V v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const V o = __shfl_up(v, d, 64);
        if (lane >= d) v += o;
    }
    return v;
}

struct Settings {
    double temperature, top_p, min_p, uniform;
    uint32_t top_k;  // 0: all
    bool with_p, with_min;
};

// Where a prefix of the ranking ends: inside a bin, after `in` of its tokens,
// with the sum of all weights up to there.
struct Border {
    int bin;
    uint32_t in;
    double weight;
};

enum class Ask { Count, Reach, Draw };

template <class T, int THREADS, int MOST, bool LONG>
struct Row {
    using Element = T;
    static constexpr int kThreads = THREADS, kWaves = THREADS / 64, kMostRanked = MOST;
    struct Shared {
        uint64_t list[MOST];
        union {
            double sums[MOST];  // running sums of the sorted list
            uint64_t bins[LONG ? kBins : 1];
            uint32_t counts[LONG ? kBins : 1];
        };
        double before[LONG ? kBins + 1 : 1];    // weights of the bins before each
        uint32_t tokens[LONG ? kBins + 1 : 1];  // and their tokens
        double wave_d[kWaves + 1];
        uint32_t wave_u[kWaves + 1];
        float wave_f[kWaves];
        uint32_t n, lo, hi, found;
        double weight;
    };

    const typename T::Raw *z;
    uint32_t vocab;
    Shared &s;
    int tid, lane, wave;
    float top;
    double inv, scale;  // 1 / T, bins of a unit of a logit
    int dev_bits, shift;

    __device__ Row(const typename T::Raw *z_, uint32_t vocab_, Shared &s_) : z(z_), vocab(vocab_), s(s_) {
        tid = threadIdx.x;
        lane = tid & 63;
        wave = tid >> 6;
    }

    __device__ double weight_of(float x) const { return exp((double(x) - double(top)) * inv); }
    // Bins from the largest logit.
    __device__ double place(float x) const { return (double(top) - double(x)) * scale; }

    // The sum over the workgroup of each thread's value, and (scan) of the threads before.
    template <class V>
    __device__ V block_scan(V v, V *room, V &total) {
        const V in = wave_scan(v, lane);
        if (lane == 63) room[wave] = in;
        __syncthreads();
        V base = 0, sum = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const V o = room[w];
            if (w < wave) base += o;
            sum += o;
        }
        total = sum;
        __syncthreads();
        return base + in - v;
    }
    __device__ uint32_t block_count(uint32_t v) {
        uint32_t total;
        block_scan<uint32_t>(v, s.wave_u, total);
        return total;
    }

    // Appends what `in` takes; more than MOST are only counted.
    template <class In>
    __device__ uint32_t gather(In &&in) {
        if (tid == 0) s.n = 0;
        __syncthreads();
        each<T, THREADS>(z, vocab, [&](float x, uint32_t token) {
            if (in(x)) {
                const uint32_t at = atomicAdd(&s.n, 1u);
                if (at < uint32_t(MOST)) s.list[at] = candidate(x, token);
            }
        });
        __syncthreads();
        const uint32_t n = s.n;
        __syncthreads();
        return n;
    }

    // Sorts the first n of the list, the first in rank first, and makes their running sums.
    __device__ void rank(uint32_t n) {
        uint32_t size = 2;
        while (size < n) size *= 2;
        for (uint32_t i = n + tid; i < size; i += THREADS) s.list[i] = 0;
        __syncthreads();
        for (uint32_t k = 2; k <= size; k *= 2)
            for (uint32_t j = k / 2; j > 0; j /= 2) {
                for (uint32_t i = tid; i < size / 2; i += THREADS) {
                    const uint32_t a = 2 * i - (i & (j - 1)), b = a + j;
                    const uint64_t x = s.list[a], y = s.list[b];
                    if ((x < y) == ((a & k) == 0)) {
                        s.list[a] = y;
                        s.list[b] = x;
                    }
                }
                __syncthreads();
            }
        constexpr int E = (MOST + THREADS - 1) / THREADS;
        double w[E], sum = 0.0, total;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint32_t i = tid * E + e;
            w[e] = i < n ? weight_of(unordered(uint32_t(s.list[i] >> 32))) : 0.0;
            sum += w[e];
        }
        double run = block_scan<double>(sum, s.wave_d, total);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint32_t i = tid * E + e;
            run += w[e];
            if (i < n) s.sums[i] = run;
        }
        __syncthreads();
    }

    // How many of the n ranked ones' running sums lie under t, or (up) do not exceed it.
    __device__ uint32_t below(uint32_t n, double t, bool up) {
        uint32_t c = 0;
        for (uint32_t i = tid; i < n; i += THREADS) c += up ? s.sums[i] <= t : s.sums[i] < t;
        return block_count(c);
    }

    // Bins of the row, or (within) the keys lo..hi of bin `of`, 2^step keys each.
    __device__ void fill_bins(bool within, int of, uint32_t lo, uint32_t hi, int step) {
        for (int i = tid; i < kBins; i += THREADS) s.bins[i] = 0;
        __syncthreads();
        // e^-r - 1 for r from 0 to 1/64, in units of 2^-dev_bits: the sixth term is under 2^-45.
        // (r = 0, and so the sum of weights that equal the largest, is exact.)
        const double unit = double(uint64_t(1) << dev_bits), c1 = -unit * 0x1p-6, c2 = unit * (0x1p-12 / 2),
                     c3 = -unit * (0x1p-18 / 6), c4 = unit * (0x1p-24 / 24), c5 = -unit * (0x1p-30 / 120);
        const uint64_t one = uint64_t(1) << shift;
        each<T, THREADS>(z, vocab, [&](float x, uint32_t) {
            const double y = place(x);
            int bin;
            double r;
            if (within) {
                const uint32_t k = order(x);
                if (k < lo || k > hi) return;
                bin = int((hi - k) >> step);
                r = y - double(of);
            } else {
                if (!(y < double(kBins - 1))) return;
                const double at = floor(y);
                bin = int(at);
                r = y - at;
            }
            const double d = r * fma(r, fma(r, fma(r, fma(r, c5, c4), c3), c2), c1);
            atomicAdd(reinterpret_cast<unsigned long long *>(&s.bins[bin]),
                      static_cast<unsigned long long>(one + uint64_t(int64_t(int32_t(rint(d))))));
        });
        __syncthreads();
    }

    static constexpr int kEach = (kBins + THREADS - 1) / THREADS;  // bins of a thread

    // A thread's bins with the weights and tokens before them; `of` as above, or -1.
    struct Mine {
        double weight[kEach], before, total;
        uint32_t tokens[kEach], taken, all;
    };
    __device__ Mine scan_bins(int of) {
        Mine m;
        double w = 0.0;
        uint32_t c = 0;
        const double unit = 1.0 / double(uint64_t(1) << dev_bits);
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int b = tid * kEach + e;
            const uint64_t h = s.bins[b];
            const int64_t dev = int64_t(h << (64 - shift)) >> (64 - shift);
            m.tokens[e] = uint32_t((h - uint64_t(dev)) >> shift);
            m.weight[e] = exp(-double(of < 0 ? b : of) / kPerUnit) * (double(m.tokens[e]) + double(dev) * unit);
            w += m.weight[e];
            c += m.tokens[e];
        }
        m.before = block_scan<double>(w, s.wave_d, m.total);
        m.taken = block_scan<uint32_t>(c, s.wave_u, m.all);
        return m;
    }
    __device__ void keep_bins() {
        Mine m = scan_bins(-1);
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            s.before[tid * kEach + e] = m.before;
            s.tokens[tid * kEach + e] = m.taken;
            m.before += m.weight[e];
            m.taken += m.tokens[e];
        }
        if (tid == 0) {
            s.before[kBins] = m.total;
            s.tokens[kBins] = m.all;
        }
        __syncthreads();
    }
    // The first bin that `is` takes, kBins where there is none.
    template <class Is>
    __device__ int first_bin(Is &&is) {
        if (tid == 0) s.found = kBins;
        __syncthreads();
        for (int b = tid; b < kBins; b += THREADS)
            if (is(b)) {
                atomicMin(&s.found, uint32_t(b));
                break;
            }
        __syncthreads();
        const int b = int(s.found);
        __syncthreads();
        return b;
    }

    // The n-th token, from 0, whose logit is that of key k.
    __device__ uint32_t nth_of(uint32_t k, uint32_t n) {
        const uint32_t share = (vocab + THREADS - 1) / THREADS * 64, from = min(vocab, wave * share),
                       to = min(vocab, from + share);
        uint32_t c = 0;
        for (uint32_t i = from + lane; i < to; i += 64) c += order(T::to_float(z[i])) == k;
        uint32_t total, before = block_scan<uint32_t>(c, s.wave_u, total);
        const uint32_t first = __shfl(before, 0, 64);
        uint32_t here = __shfl(before + c, 63, 64) - first;
        if (n >= first && n < first + here) {  // this wave has it
            uint32_t left = n - first;
            for (uint32_t i = from; i < to; i += 64) {
                const bool is = i + lane < to && order(T::to_float(z[i + lane])) == k;
                const uint64_t mask = __ballot(is);
                const uint32_t c64 = uint32_t(__popcll(mask));
                if (left < c64) {
                    if (is && uint32_t(__popcll(mask & ((uint64_t(1) << lane) - 1))) == left) s.found = i + lane;
                    break;
                }
                left -= c64;
            }
        }
        __syncthreads();
        const uint32_t token = s.found;
        __syncthreads();
        return token;
    }

    struct Answer {
        uint32_t in;    // tokens of the bin up to the border
        double weight;  // of all up to there (Draw: of the token)
        uint32_t token;
    };
    // In n ranked tokens, after `taken` of the bin and weights of `base`.
    __device__ Answer answer(uint32_t n, Ask ask, double t, uint32_t q, double base, uint32_t taken) {
        if (ask == Ask::Draw) {
            const uint32_t at = min(below(n, t - base, true), min(n, q - taken) - 1);
            const uint64_t v = s.list[at];
            return {0, weight_of(unordered(uint32_t(v >> 32))), ~uint32_t(v)};
        }
        const uint32_t c = ask == Ask::Count ? min(n, q - taken) : min(n, below(n, t - base, false) + 1);
        return {taken + c, base + s.sums[c - 1], 0};
    }

    // Inside a bin that holds tokens: its first q tokens (Count); the tokens up to
    // where the sum of all weights reaches t (Reach); the first of its first q
    // tokens at which that sum exceeds t, or the last of them (Draw).
    __device__ Answer resolve(int bin, Ask ask, double t, uint32_t q) {
        const double from = double(bin), until = double(bin + 1);
        double base = s.before[bin];
        uint32_t taken = 0;
        const uint32_t n = gather([&](float x) {
            const double y = place(x);
            return y >= from && y < until;
        });
        if (n <= uint32_t(MOST)) {
            rank(n);
            return answer(n, ask, t, q, base, 0);
        }
        if (tid == 0) {
            s.lo = 0xffffffffu;
            s.hi = 0;
        }
        __syncthreads();
        uint32_t lo = 0xffffffffu, hi = 0, count = n;
        each<T, THREADS>(z, vocab, [&](float x, uint32_t) {
            const double y = place(x);
            if (y >= from && y < until) {
                lo = min(lo, order(x));
                hi = max(hi, order(x));
            }
        });
        atomicMin(&s.lo, lo);
        atomicMax(&s.hi, hi);
        __syncthreads();
        lo = s.lo;
        hi = s.hi;
        __syncthreads();
        while (lo != hi) {
            const int step = max(0, 32 - __clz(int(hi - lo)) - 11);  // (hi - lo) >> step < kBins
            fill_bins(true, bin, lo, hi, step);
            const Mine m = scan_bins(bin);
            if (tid == 0) {
                s.found = kBins;
                s.n = 0;
            }
            __syncthreads();
            double w = base + m.before;
            uint32_t c = taken + m.taken;
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                w += m.weight[e];
                c += m.tokens[e];
                if (!m.tokens[e]) continue;
                atomicMax(&s.n, uint32_t(tid * kEach + e));
                if (ask == Ask::Count ? c >= q : ask == Ask::Reach ? w >= t : w > t || c >= q)
                    atomicMin(&s.found, uint32_t(tid * kEach + e));
            }
            __syncthreads();
            const uint32_t sub = s.found < uint32_t(kBins) ? s.found : s.n;
            __syncthreads();
            w = base + m.before;
            c = taken + m.taken;
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                if (sub == uint32_t(tid * kEach + e)) {
                    s.weight = w;
                    s.lo = c;
                    s.hi = m.tokens[e];
                }
                w += m.weight[e];
                c += m.tokens[e];
            }
            __syncthreads();
            base = s.weight;
            taken = s.lo;
            count = s.hi;
            __syncthreads();
            hi -= sub << step;
            const uint32_t span = (uint32_t(1) << step) - 1;
            if (hi - lo > span) lo = hi - span;
            if (count <= uint32_t(MOST)) {
                gather([&](float x) { return order(x) >= lo && order(x) <= hi; });
                rank(count);
                return answer(count, ask, t, q, base, taken);
            }
        }
        // Equal logits, in the order of their tokens.
        const double w = weight_of(unordered(lo)), steps = (t - base) / w;
        if (ask == Ask::Draw) {
            const uint32_t last = min(count, q - taken) - 1;
            const uint32_t at = steps >= double(last) ? last : steps > 0.0 ? uint32_t(steps) : 0;
            return {0, w, nth_of(lo, at)};
        }
        const uint32_t c = ask == Ask::Count       ? min(count, q - taken)
                           : steps >= double(count) ? count
                           : steps > 1.0            ? uint32_t(ceil(steps))
                                                    : 1;
        return {taken + c, base + double(c) * w, 0};
    }
};

struct Drawn {
    uint32_t token;
    double weight, of;
};

// Draws from the n first in rank, of which the whole is `whole` to top_p, or (negative) their own.
template <class R>
__device__ Drawn draw_ranked(R &r, uint32_t n, const Settings &set, double whole) {
    r.rank(n);
    if (set.top_k) n = min(n, set.top_k);
    if (set.with_p) n = min(n, r.below(n, set.top_p * (whole < 0.0 ? r.s.sums[n - 1] : whole), false) + 1);
    if (set.with_min) {
        uint32_t c = 0;
        for (uint32_t i = r.tid; i < n; i += blockDim.x)
            c += r.weight_of(unordered(uint32_t(r.s.list[i] >> 32))) >= set.min_p;
        n = max(1u, r.block_count(c));
    }
    const double all = r.s.sums[n - 1];
    const uint64_t v = r.s.list[min(r.below(n, set.uniform * all, true), n - 1)];
    return {~uint32_t(v), r.weight_of(unordered(uint32_t(v >> 32))), all};
}

// The bin of the k-th largest of the threads' maxima bounds the k-th largest logit
// from below; bins past the last with a weight hold nothing that can be drawn.
template <class R>
__device__ int bound_bin(R &r, float mine, uint32_t k) {
    for (int i = r.tid; i < kBins; i += int(blockDim.x)) r.s.counts[i] = 0;
    __syncthreads();
    const double y = r.place(mine);
    if (y < double(kBins - 1)) atomicAdd(&r.s.counts[int(y)], 1u);
    __syncthreads();
    constexpr int E = R::kEach;
    uint32_t c[E], sum = 0, total;
#pragma unroll
    for (int e = 0; e < E; ++e) sum += c[e] = r.s.counts[r.tid * E + e];
    uint32_t before = r.template block_scan<uint32_t>(sum, r.s.wave_u, total);
    if (r.tid == 0) r.s.found = kBins - 2;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (before < k && before + c[e] >= k) r.s.found = uint32_t(r.tid * E + e);
        before += c[e];
    }
    __syncthreads();
    const int b = int(r.s.found);
    __syncthreads();
    return b;
}

// A logit that is at or below every logit with place < `until`.
template <class R>
__device__ float least_of(const R &r, double until) {
    const double down = until / r.scale, x = double(r.top) - down - (fabs(double(r.top)) + down) * 0x1p-20;
    return x > -double(FLT_MAX) ? float(x) : -FLT_MAX;
}

// The whole row by its bins.
template <class R>
__device__ Drawn draw_long(R &r, const Settings &set) {
    auto &s = r.s;
    r.shift = 63 - max(1, 32 - __clz(int(r.vocab)));
    r.dev_bits = min(36, 2 * r.shift - 58);  // a bin's sum, vocab terms under 0.0156, stays in its field
    r.fill_bins(false, 0, 0, 0, 0);
    r.keep_bins();
    const auto few = [&](int b) { return s.tokens[b + 1] <= uint32_t(R::kMostRanked); };
    const auto ranked = [&](int b, double whole) {
        const double until = double(b + 1);
        const uint32_t n = r.gather([&](float x) { return r.place(x) < until; });
        return draw_ranked(r, n, set, whole);
    };
    Border end{kBins, 0, s.before[kBins]};
    double whole = -1.0;
    if (set.top_k && set.top_k < s.tokens[kBins]) {
        const int b = r.first_bin([&](int i) { return s.tokens[i + 1] >= set.top_k; });
        if (few(b)) return ranked(b, -1.0);
        const auto at = r.resolve(b, Ask::Count, 0.0, set.top_k - s.tokens[b]);
        end = {b, at.in, at.weight};
    }
    if (set.with_p) {
        whole = end.weight;
        const double t = set.top_p * whole;
        const int b = r.first_bin([&](int i) { return s.before[i + 1] >= t; });
        if (b < kBins && b <= end.bin) {
            if (few(b)) return ranked(b, whole);
            const auto at = r.resolve(b, Ask::Reach, t, 0);
            if (b < end.bin || at.in < end.in) end = {b, at.in, at.weight};
        }
    }
    if (set.with_min) {
        const double y = -log(set.min_p) * kPerUnit;
        const int b = y < double(kBins - 1) ? max(0, int(y)) : kBins;
        if (b < kBins && b <= end.bin) {
            if (few(b)) return ranked(b, whole);
            const double from = double(b), until = double(b + 1);
            double w = 0.0, in;
            uint32_t c = 0;
            each<typename R::Element, R::kThreads>(r.z, r.vocab, [&](float x, uint32_t) {
                const double at = r.place(x);
                if (at >= from && at < until) {
                    const double v = r.weight_of(x);
                    if (v >= set.min_p) {
                        w += v;
                        ++c;
                    }
                }
            });
            r.template block_scan<double>(w, s.wave_d, in);
            c = r.block_count(c);
            if (b < end.bin || c < end.in) end = {b, c, s.before[b] + in};
        }
    }
    const double t = set.uniform * end.weight;
    int b = r.first_bin([&](int i) { return s.before[i + 1] > t && s.tokens[i + 1] > s.tokens[i]; });
    if (b >= end.bin && (end.in == 0 || b >= kBins)) {  // rounding: the last that is left
        if (end.bin < kBins && end.in)
            b = end.bin;
        else
            b = kBins - 1 - r.first_bin([&](int i) {
                const int j = kBins - 1 - i;
                return j < end.bin && s.tokens[j + 1] > s.tokens[j];
            });
    }
    b = min(b, end.bin);
    const auto at = r.resolve(b, Ask::Draw, t, b == end.bin ? end.in : s.tokens[b + 1] - s.tokens[b]);
    return {at.token, at.weight, end.weight};
}

template <class T, int THREADS, int MOST, bool LONG>
__global__ void __launch_bounds__(THREADS) sample_kernel(SampleArgs a) {
    using R = Row<T, THREADS, MOST, LONG>;
    __shared__ typename R::Shared shared;
    const size_t row = blockIdx.x;
    R r(static_cast<const typename T::Raw *>(a.logits) + row * a.stride, uint32_t(a.vocab), shared);
    Settings set;
    set.temperature = a.temperatures ? double(a.temperatures[row]) : 1.0;
    set.top_p = a.top_p ? double(a.top_p[row]) : 1.0;
    set.min_p = a.min_p ? double(a.min_p[row]) : 0.0;
    set.uniform = double(a.uniforms[row]);
    const int k = a.top_k ? a.top_k[row] : 0;
    set.top_k = k > 0 && uint32_t(k) < r.vocab ? uint32_t(k) : 0;
    set.with_p = set.top_p < 1.0;
    set.with_min = set.min_p > 0.0;
    const bool greedy = set.temperature == 0.0;
    const bool valid = set.temperature >= 0.0 && set.temperature <= double(FLT_MAX) && set.top_p == set.top_p &&
                       set.min_p == set.min_p && (greedy || (set.uniform >= 0.0 && set.uniform < 1.0));
    set.min_p = fmin(set.min_p, 1.0);  // the largest is always left

    float mine = -INFINITY;
    bool bad = false;
    each<T, THREADS>(r.z, r.vocab, [&](float x, uint32_t) {
        mine = fmaxf(mine, x);
        bad |= !(x < INFINITY);
    });
    const float wave_top = wave_largest(mine);
    const bool wave_bad = __ballot(bad) != 0;
    if (r.lane == 0) {
        shared.wave_f[r.wave] = wave_top;
        shared.wave_u[r.wave] = wave_bad;
    }
    __syncthreads();
    r.top = -INFINITY;
    uint32_t any_bad = 0;
#pragma unroll
    for (int w = 0; w < R::kWaves; ++w) {
        r.top = fmaxf(r.top, shared.wave_f[w]);
        any_bad |= shared.wave_u[w];
    }
    __syncthreads();
    if (any_bad || r.top == -INFINITY || !valid) {
        if (r.tid == 0) {
            a.tokens[row] = kNoToken;
            if (a.logprob) a.logprob[row] = NAN;
        }
        return;
    }
    if (greedy) {
        if (r.tid == 0) shared.found = kNoToken;
        __syncthreads();
        uint32_t least = kNoToken;
        each<T, THREADS>(r.z, r.vocab, [&](float x, uint32_t token) {
            if (x == r.top) least = min(least, token);
        });
        if (least != kNoToken) atomicMin(&shared.found, least);
        __syncthreads();
        if (r.tid == 0) {
            a.tokens[row] = shared.found;
            if (a.logprob) a.logprob[row] = 0.0f;
        }
        return;
    }
    r.inv = 1.0 / set.temperature;
    r.scale = kPerUnit * r.inv;

    float least = 0.0f;
    bool few = true;
    if constexpr (LONG) {
        if (set.top_k && set.top_k <= uint32_t(THREADS / 2))
            least = least_of(r, double(bound_bin(r, mine, set.top_k) + 1));
        else if (set.with_min && !set.with_p)
            least = least_of(r, -log(set.min_p) * kPerUnit);
        else
            few = false;
    } else {
        least = -FLT_MAX;
    }
    Drawn d;
    uint32_t n = 0;
    if (few) {
        n = r.gather([&](float x) { return x >= least; });
        few = n <= uint32_t(MOST);
    }
    if constexpr (LONG)
        d = few ? draw_ranked(r, n, set, -1.0) : draw_long(r, set);
    else
        d = draw_ranked(r, n, set, -1.0);
    if (r.tid == 0) {
        a.tokens[row] = d.token;
        if (a.logprob) a.logprob[row] = float(log(d.weight / d.of));
    }
}

template <class T>
void launch(const SampleArgs &a, hipStream_t stream) {
    if (a.vocab <= size_t(kShort))
        sample_kernel<T, 256, kShort, false><<<dim3(unsigned(a.rows)), 256, 0, stream>>>(a);
    else
        sample_kernel<T, 1024, kMost, true><<<dim3(unsigned(a.rows)), 1024, 0, stream>>>(a);
}

}  // namespace

void sample_filtered(const SampleArgs &a, Type type, hipStream_t stream) {
    switch (type) {
        case Type::F32: return launch<F32>(a, stream);
        case Type::F16: return launch<F16>(a, stream);
        case Type::BF16: return launch<BF16>(a, stream);
    }
}

}  // namespace meshgpt::kern
