// Sampling with temperature, top-k, top-p and min-p from given random numbers.
//
// Tokens are ranked by their logits z, the largest first, of equal ones the
// lowest token first.  With w_j = exp((z_j - max z) / T), the first top_k in
// rank are left; of these the shortest run from the first whose weights reach
// top_p of theirs; of these the ones with w >= min_p; and u picks the first
// token in rank at which the sum of what is left exceeds u times the whole.
// Everything is a prefix of the ranking, so no row is sorted: a border is found
// by the weights of bins, and inside one bin by ranking that bin.
//
// Sums decide which of many close borders is met: at 100000 equally likely
// tokens one is 1e-5 of the whole.  So weights are summed in 64 bits, in an
// order that is the same in every call.
//
// A row has a workgroup, in one of three ways (`launch` has the sizes):
//   up to 256 logits: every token counts the tokens and weights before it;
//   many 16-bit logits: a count for each of their 65536 values (sample_codes_kernel);
//   else: bins of (max z - z) / T (sample_bins_kernel), and where top_k or min_p leave few
//   tokens before any weight is summed, these tokens alone.
#include <algorithm>
#include <cfloat>

#include "dpp.hpp"
#include "operators.hpp"
#include "sampler.hpp"
#include "types.hpp"

namespace meshgpt::kern {
namespace {

constexpr double kReach = 31.9;    // powers of e that are looked at
constexpr uint32_t kNoToken = 0xffffffffu;

// Logits as integers in the same order; -0 is 0.
__device__ __forceinline__ uint32_t order(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t k) {
    return __builtin_bit_cast(float, k ^ (uint32_t(int32_t(~k) >> 31) | 0x80000000u));
}

// A value that all lanes have, in scalar registers.
__device__ __forceinline__ double uniform(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readfirstlane(uint32_t(b)), hi = __builtin_amdgcn_readfirstlane(uint32_t(b >> 32));
    return __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}

// f(logit) for every logit of a row, 16 bytes a load, four loads under way.
template <class T, int THREADS, class F>
__device__ __forceinline__ void each(const typename T::Raw *z, uint32_t vocab, F &&f) {
    constexpr int G = T::kGroup, U = 4;
    const uint32_t groups = vocab / G;
    for (uint32_t j = threadIdx.x; j < groups; j += U * THREADS) {
        uint4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u)  // behind the end: its first group again
            w[u] = get_any(z + size_t(j + u * THREADS < groups ? j + u * THREADS : j) * G);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float x[G];
            T::unpack(w[u], x);
#pragma unroll
            for (int e = 0; e < G; ++e) f(x[e]);
        }
    }
    const uint32_t last = groups * G + threadIdx.x;
    if (last < vocab) f(T::to_float(z[last]));
}

// The same for what takes long with each logit: the next group is under way meanwhile.
template <class T, int THREADS, class F>
__device__ __forceinline__ void each_slowly(const typename T::Raw *z, uint32_t vocab, F &&f) {
    constexpr int G = T::kGroup;
    const uint32_t groups = vocab / G;
    uint32_t j = threadIdx.x;
    uint4 now{}, next{};
    if (j < groups) now = get_any(z + size_t(j) * G);
    if (j + THREADS < groups) next = get_any(z + size_t(j + THREADS) * G);
#pragma unroll 1
    for (; j < groups; j += THREADS) {
        uint4 later{};
        if (j + 2 * THREADS < groups) later = get_any(z + size_t(j + 2 * THREADS) * G);
        float x[G];
        T::unpack(now, x);
#pragma unroll
        for (int e = 0; e < G; ++e) f(x[e]);
        now = next;
        next = later;
    }
    const uint32_t last = groups * G + threadIdx.x;
    if (last < vocab) f(T::to_float(z[last]));
}

// f(logit, token) for the few logits of a row from lo to hi.
template <class T, int THREADS, class F>
__device__ __forceinline__ void each_in(const typename T::Raw *z, uint32_t vocab, float lo, float hi, F &&f) {
    constexpr int G = T::kGroup, U = 4;
    const uint32_t groups = vocab / G;
#pragma unroll 1
    for (uint32_t j = threadIdx.x; j < groups; j += U * THREADS) {
        uint4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = get_any(z + size_t(min(j + u * THREADS, groups - 1)) * G);
        uint32_t those = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float x[G];
            T::unpack(w[u], x);
            uint32_t here = 0;
#pragma unroll
            for (int e = 0; e < G; ++e) here |= uint32_t(x[e] >= lo && x[e] <= hi) << e;
            if (j + u * THREADS < groups) those |= here << (u * G);
        }
        while (those) {
            const uint32_t b = __builtin_ctz(those), token = (j + b / G * THREADS) * G + b % G;
            those &= those - 1;
            f(T::to_float(z[token]), token);
        }
    }
    const uint32_t last = groups * G + threadIdx.x;
    if (last < vocab) {
        const float x = T::to_float(z[last]);
        if (x >= lo && x <= hi) f(x, last);
    }
}

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// v of the lane that the DPP pattern CTRL names, 0 where there is none.
template <int CTRL, int ROW_MASK = 0xf>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
    return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, ROW_MASK, 0xf, false));
}
template <int CTRL, int ROW_MASK = 0xf>
__device__ __forceinline__ double moved(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, uint64_t(moved<CTRL, ROW_MASK>(uint32_t(b >> 32))) << 32 | moved<CTRL, ROW_MASK>(uint32_t(b)));
}
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ double lane_value(double v, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, uint64_t(lane_value(uint32_t(b >> 32), lane)) << 32 | lane_value(uint32_t(b), lane));
}
// Running sums over the lanes of a row of 16, and over a wave's.
template <class V>
__device__ __forceinline__ V row_scan(V v) {
    v += moved<0x111>(v);  // row_shr:1
    v += moved<0x112>(v);
    v += moved<0x114>(v);
    v += moved<0x118>(v);
    return v;
}
template <class V>
__device__ __forceinline__ V wave_scan(V v) {
    v = row_scan(v);
    v += moved<0x142, 0xa>(v);  // row_bcast:15
    v += moved<0x143, 0xc>(v);  // row_bcast:31
    return v;
}
template <class V>
__device__ __forceinline__ V wave_total(V v) {
    return lane_value(wave_scan(v), 63);
}

// The sum of the values of the threads before, and of all of them.
template <int THREADS, class V>
__device__ __forceinline__ V block_scan(V v, V *room, V &total) {
    constexpr int WAVES = THREADS / 64;
    static_assert(WAVES <= 16, "a row of lanes has the waves' sums");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const V in = wave_scan(v);
    __syncthreads();
    if (lane == 63) room[wave] = in;
    __syncthreads();
    const V own = lane < WAVES ? room[lane] : V(0), sums = row_scan(own);
    total = lane_value(sums, WAVES - 1);
    return lane_value(sums - own, wave) + (in - v);
}
template <int THREADS, class V>
__device__ __forceinline__ V block_total(V v, V *room) {
    V total;
    block_scan<THREADS>(v, room, total);
    return total;
}

struct Settings {
    double temperature, top_p, min_p, uniform;
    uint32_t top_k;  // 0: all
    bool with_p, with_min, greedy, valid;
};
__device__ __forceinline__ Settings settings_of(const SampleArgs &a, size_t row) {
    Settings s;
    s.temperature = uniform(a.temperatures ? double(a.temperatures[row]) : 1.0);
    s.top_p = uniform(a.top_p ? double(a.top_p[row]) : 1.0);
    s.min_p = uniform(fmin(a.min_p ? double(a.min_p[row]) : 0.0, 1.0));  // the largest is always left
    s.uniform = uniform(double(a.uniforms[row]));
    const int k = a.top_k ? a.top_k[row] : 0;
    s.top_k = k > 0 && size_t(k) < a.vocab ? uint32_t(k) : 0;
    s.with_p = s.top_p < 1.0;
    s.with_min = s.min_p > 0.0;
    s.greedy = s.temperature == 0.0;
    const bool settings = s.top_p == s.top_p && !(a.min_p && a.min_p[row] != a.min_p[row]) && s.uniform >= 0.0 && s.uniform < 1.0;
    s.valid = s.greedy || (s.temperature > 0.0 && s.temperature <= double(FLT_MAX) && settings);
    return s;
}

__device__ __forceinline__ void write(const SampleArgs &a, size_t row, uint32_t token, float logprob) {
    a.tokens[row] = token;
    if (a.logprob) a.logprob[row] = logprob;
}

// How many of n equal weights w reach t, at least 1, and which of them the first to exceed it is.
__device__ __forceinline__ uint32_t equal_reach(double t, double w, uint32_t n) {
    const double steps = t / w;
    return steps >= double(n) ? n : steps > 1.0 ? uint32_t(ceil(steps)) : 1;
}
__device__ __forceinline__ uint32_t equal_draw(double t, double w, uint32_t n) {
    const double steps = t / w;
    return steps >= double(n - 1) ? n - 1 : steps > 0.0 ? uint32_t(steps) : 0;
}

// ---- weights by bins of 1 / UNIT of a power of e ------------------------------------------

template <int UNIT>
struct Powers {
    double wholes[32], parts[UNIT];  // e^-i, e^(-i / UNIT)
};

template <int UNIT>
struct Weights {
    const Powers<UNIT> &powers;  // in LDS
    double top, scale;           // the largest logit, bins of a unit of a logit

    // Makes the powers, as products of e^(-2^b / 128) (to 7 * 2^-53); a barrier has to follow.
    static __device__ __forceinline__ void prepare(Powers<UNIT> &p) {
        static_assert(UNIT == 32 || UNIT == 128, "units of the table");
        constexpr int STEP = UNIT == 128 ? 0 : 2, BITS = UNIT == 128 ? 7 : 5;
        const uint32_t i = threadIdx.x;
        if (i >= UNIT + 32) return;
        const double of[12] = {0x1.fc03fd56aa225p-1, 0x1.f80feabfeefa5p-1, 0x1.f03f56a88b5d8p-1, 0x1.e0fabfbc702a4p-1,
                               0x1.c3d6a24ed8222p-1, 0x1.8ebef9eac820bp-1, 0x1.368b2fc6f960ap-1, 0x1.78b56362cef38p-2,
                               0x1.152aaa3bf81ccp-3, 0x1.2c155b8213cf4p-6, 0x1.5fc21041027adp-12, 0x1.e355bbaee85cbp-24};
        double w = 1.0;
#pragma unroll
        for (int b = 0; b < BITS; ++b) {  // constants, both of them: loads of one or the other would be a chain
            const double part = of[b + STEP], whole = of[min(7 + b, 11)], factor = i < UNIT ? part : whole;
            w *= i >> b & 1 ? factor : 1.0;
        }
        (i < UNIT ? p.parts[i] : p.wholes[i - UNIT]) = w;
    }
    // Bins from the largest logit.
    __device__ __forceinline__ double place(float x) const { return (top - double(x)) * scale; }
    // The weight where a bin begins.
    __device__ __forceinline__ double begin_of(int bin) const { return powers.wholes[bin / UNIT] * powers.parts[bin % UNIT]; }
    // The series of e^(-r / UNIT) - 1 for r from 0 to 1, in units of `unit`, over r: what it
    // leaves out is under 2^-39.  r = 0 is exact, and with it the sum of weights that equal
    // the largest.
    template <class Units>
    static __device__ __forceinline__ double series(double r, Units &&units) {
        constexpr double U = 1.0 / UNIT;
        double v = UNIT == 128 ? units(U * U * U * U / 24)
                               : fma(r, units(-U * U * U * U * U / 120), units(U * U * U * U / 24));
        v = fma(r, v, units(-U * U * U / 6));
        v = fma(r, v, units(U * U / 2));
        return fma(r, v, units(-U));
    }
    __device__ __forceinline__ double of(float x) const {
        const double y = place(x), at = floor(y);
        if (!(y < kReach * UNIT)) return 0.0;
        const double begin = begin_of(int(at));
        const double r = y - at;
        return fma(begin, r * series(r, [](double v) { return v; }), begin);
    }
};

// ---- short rows -------------------------------------------------------------------

// Four threads count the tokens before a token, a quarter of the row each, four to an
// LDS read; then a thread has a place in the ranking, with the running sum of the weights
// up to there.  Its scans and barriers bound it: 32 rows of 256 F32 8.0 us; 1405 rows of 17
// with a call 11 (28 with 1024 threads a row).
template <class T, int TOKENS>
__global__ void __launch_bounds__(4 * TOKENS) sample_short_kernel(SampleArgs a) {
    using Raw = typename T::Raw;
    constexpr int WAVES = TOKENS / 64, THREADS = 4 * TOKENS, UNIT = 32;
    __shared__ uint4 keys[TOKENS / 4];
    __shared__ double weights[TOKENS], sums[TOKENS], room_d[THREADS / 64];
    __shared__ uint32_t tokens[TOKENS], room_u[THREADS / 64], bads[WAVES];
    __shared__ float tops[WAVES];
    __shared__ Powers<UNIT> powers;
    const size_t row = blockIdx.x;
    const uint32_t tid = threadIdx.x, vocab = uint32_t(a.vocab);
    const Raw *const z = static_cast<const Raw *>(a.logits) + row * a.stride;
    const Settings set = settings_of(a, row);
    const uint32_t token = tid / 4, quarter = tid % 4;
    const float x = token < vocab ? T::to_float(z[token]) : -INFINITY;
    if (tid < TOKENS) {
        const float y = tid < vocab ? T::to_float(z[tid]) : -INFINITY;
        reinterpret_cast<uint32_t *>(keys)[tid] = order(y);
        weights[tid] = 0.0;
        const float wave_top = wave_largest(y);
        const bool wave_bad = __ballot(!(y < INFINITY)) != 0;
        if (tid % 64 == 0) {
            tops[tid / 64] = wave_top;
            bads[tid / 64] = wave_bad;
        }
    }
    Weights<UNIT>::prepare(powers);
    const double scale = set.greedy ? 1.0 : uniform(UNIT / set.temperature);
    __syncthreads();
    float top = -INFINITY;
    uint32_t bad = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        top = fmaxf(top, tops[w]);
        bad |= bads[w];
    }
    if (bad || top == -INFINITY || !set.valid) {
        if (tid == 0) write(a, row, kNoToken, NAN);
        return;
    }
    // Of equal keys those of lower tokens are before.  Each quarter begins at other banks.
    const uint32_t key = order(x);
    uint32_t before = 0;
#pragma unroll 4
    for (uint32_t j = 0; j < TOKENS / 16; ++j) {
        const uint32_t at = quarter * (TOKENS / 16) + (j + 4 * quarter) % (TOKENS / 16);
        const uint4 k = keys[at];
        const int lower = int(token) - int(4 * at);  // so many of the four are lower tokens
        before += (k.x > key - (lower > 0)) + (k.y > key - (lower > 1)) + (k.z > key - (lower > 2)) + (k.w > key - (lower > 3));
    }
    before += moved<0xB1>(before);  // quad_perm [1,0,3,2]
    before += moved<0x4E>(before);  // quad_perm [2,3,0,1]
    if (set.greedy) {
        if (before == 0 && quarter == 0) write(a, row, token, 0.0f);
        return;
    }
    if (quarter == 0 && token < vocab) {
        weights[before] = Weights<UNIT>{powers, double(top), scale}.of(x);
        tokens[before] = token;
    }
    __syncthreads();
    // From here on a thread has a place in the ranking.
    const double w = tid < TOKENS ? weights[tid] : 0.0;
    double whole;
    const double sum = block_scan<THREADS>(w, room_d, whole) + w;
    if (tid < TOKENS) sums[tid] = sum;
    __syncthreads();
    const auto count = [&](bool is) { return block_total<THREADS>(uint32_t(is), room_u); };
    uint32_t left = count(w > 0.0);
    if (set.top_k) left = min(left, set.top_k);
    if (set.with_p) {
        const double t = set.top_p * sums[left - 1];
        left = min(left, count(tid < left && sum < t) + 1);
    }
    if (set.with_min) left = max(1u, count(tid < left && w >= set.min_p));
    whole = sums[left - 1];
    const uint32_t at = min(left - 1, count(tid < left && sum <= set.uniform * whole));
    if (tid == at) write(a, row, tokens[tid], float(log(w / whole)));
}

// ---- the general way -----------------------------------------------------------------

// The row's largest logit; then either few candidates (top_k bounds them by the
// k-th largest of the threads' maxima, min_p by itself), which are gathered and
// ranked, or bins of (max z - z) / T, UNIT for each power of e. A bin keeps its
// tokens' count and the fixed-point sum of w / (w where it begins) - 1 in one LDS
// word, each term rounded to 2^-34 of a weight or better up to 2^17 tokens (2^-28 at
// 2^20), so that it is the same in any order.  Where a border falls
// into a bin, its tokens are gathered and ranked; if they are more than MOST, the
// bin is divided by the bits of their logits until they are few enough or equal.
//
// With few rows a row's chain of passes, scans and barriers bounds it: 64 rows of 50257 F32
// with settings of all kinds 37 us, of which filling the bins takes about 10; 256 rows of
// 128000 BF16 with top_k, which need two passes and no bins, 26.
enum Ask { kCount, kReachP, kLeast, kDraw, kAsks };

template <class T, int THREADS, int UNIT, int MOST>
struct Bins {
    static constexpr int BINS = 32 * UNIT;
    static constexpr int kEach = BINS / THREADS;
    static_assert(BINS > kReach * UNIT && BINS % THREADS == 0 && MOST % THREADS == 0, "every place has a bin");
    static constexpr int kCounted = THREADS / 4;  // up to so many are ranked by counting

    struct Bin {
        int at;
        uint32_t taken, count;  // tokens before it and in it
        double base, weight;    // weights before it and in it
    };
    struct Shared {
        uint64_t bins[BINS], fine[THREADS], list[MOST];
        double sums[MOST];
        double before[THREADS];   // weights before a thread's bins
        uint32_t taken[THREADS];  // and tokens
        double room_d[THREADS / 64], base;
        Bin found_by[THREADS / 64];
        uint32_t room_u[THREADS / 64], n, lo, hi, found;
        float room_f[THREADS / 64];
        Powers<UNIT> powers;
    };

    const typename T::Raw *z;
    uint32_t vocab;
    Shared &s;
    int tid;
    float top;
    double scale, until_min;  // bins of a unit of a logit, and to min_p
    int dev_bits, shift;

    __device__ __forceinline__ Bins(const typename T::Raw *z_, uint32_t vocab_, Shared &s_)
        : z(z_), vocab(vocab_), s(s_), tid(threadIdx.x) {}

    __device__ __forceinline__ Weights<UNIT> weights() const { return {s.powers, double(top), scale}; }
    __device__ __forceinline__ double place(float x) const { return weights().place(x); }
    __device__ __forceinline__ double weight_of(float x) const { return weights().of(x); }
    __device__ __forceinline__ double begin_of(int bin) const { return weights().begin_of(bin); }
    // A logit at or below every logit with place < `until`, and one at or above those with place >= `from`.
    __device__ __forceinline__ float least(double until) const {
        const double down = until / scale, x = double(top) - down - (fabs(double(top)) + down) * 0x1p-20;
        return x > -double(FLT_MAX) ? float(x) : -FLT_MAX;
    }
    __device__ __forceinline__ float most(double from) const {
        const double down = from / scale, x = double(top) - down + (fabs(double(top)) + down) * 0x1p-20;
        return x < double(FLT_MAX) ? float(x) : FLT_MAX;
    }

    __device__ __forceinline__ void append(float x, uint32_t token) {
        const uint32_t at = atomicAdd(&s.n, 1u);
        if (at < uint32_t(MOST)) s.list[at] = uint64_t(order(x)) << 32 | uint32_t(~token);
    }

    // Ranks the first n of the list and makes their running sums.
    __device__ __forceinline__ void rank(uint32_t n) {
        if (n <= uint32_t(kCounted)) {  // four threads a token count those before it
            const uint32_t i = tid / 4;
            const uint64_t v = i < n ? s.list[i] : 0;
            uint32_t before = 0;
            if (i < n) {
#pragma unroll 4
                for (uint32_t j = tid % 4; j < n; j += 4) before += s.list[j] > v;
            }
            before += __shfl_xor(before, 1, 64);
            before += __shfl_xor(before, 2, 64);
            __syncthreads();
            if (i < n && tid % 4 == 0) s.list[before] = v;
            __syncthreads();
        } else {
            uint32_t size = 2 * kCounted;
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
                    // Pairs up to 64 apart are a wave's own: its LDS operations are in order.
                    if (j > 64 || (j == 1 && k >= 128))
                        __syncthreads();
                    else
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                }
            __syncthreads();
        }
        constexpr int E = MOST / THREADS;
        double w[E], sum = 0.0, total;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint32_t i = tid * E + e;
            w[e] = i < n ? weight_of(unordered(uint32_t(s.list[i] >> 32))) : 0.0;
            sum += w[e];
        }
        double run = block_scan<THREADS>(sum, s.room_d, total);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint32_t i = tid * E + e;
            run += w[e];
            if (i < n) s.sums[i] = run;
        }
        __syncthreads();
    }

    // How many of the n ranked ones' running sums lie under t, or (up) do not exceed it.
    __device__ __forceinline__ uint32_t below(uint32_t n, double t, bool up) {
        uint32_t c = 0;
        for (uint32_t i = tid; i < n; i += THREADS) c += up ? s.sums[i] <= t : s.sums[i] < t;
        return block_total<THREADS>(c, s.room_u);
    }

    __device__ __forceinline__ void finish(const SampleArgs &a, size_t row, uint64_t v, double whole) {
        if (tid == 0) write(a, row, ~uint32_t(v), float(log(weight_of(unordered(uint32_t(v >> 32))) / whole)));
    }

    // Draws from the n candidates of the list.
    __device__ __forceinline__ void draw_few(const SampleArgs &a, size_t row, const Settings &set, uint32_t n) {
        rank(n);
        if (set.top_k) n = min(n, set.top_k);
        if (set.with_p) n = min(n, below(n, set.top_p * s.sums[n - 1], false) + 1);
        if (set.with_min) {
            uint32_t c = 0;
            for (uint32_t i = tid; i < n; i += THREADS)
                c += weight_of(unordered(uint32_t(s.list[i] >> 32))) >= set.min_p;
            n = max(1u, block_total<THREADS>(c, s.room_u));
        }
        const double whole = s.sums[n - 1];
        finish(a, row, s.list[min(below(n, set.uniform * whole, true), n - 1)], whole);
    }

    // The bin of the k-th largest of the threads' maxima bounds the k-th largest logit
    // from below; what lies past the last bin cannot be drawn.
    __device__ __forceinline__ int bound_bin(float mine, uint32_t k) {
        uint32_t *const counts = reinterpret_cast<uint32_t *>(s.bins);
        for (int i = tid; i < BINS; i += THREADS) counts[i] = 0;
        if (tid == 0) s.found = BINS - 1;
        __syncthreads();
        const double y = place(mine);
        if (y < double(kReach * UNIT)) atomicAdd(&counts[int(y)], 1u);
        __syncthreads();
        uint32_t c[kEach], sum = 0, total;
#pragma unroll
        for (int e = 0; e < kEach; ++e) sum += c[e] = counts[tid * kEach + e];
        uint32_t before = block_scan<THREADS>(sum, s.room_u, total);
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            if (before < k && before + c[e] >= k) s.found = uint32_t(tid * kEach + e);
            before += c[e];
        }
        __syncthreads();
        return int(s.found);
    }

    // 1 for a token, and w / (w where the bin begins) - 1, r bins from there, in units of
    // 2^-dev_bits, rounded by the addition of 1.5 * 2^52.
    __device__ __forceinline__ uint64_t term(double r) const {
        const double d = Weights<UNIT>::series(r, [&](double v) {
            return __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, v) + (uint64_t(dev_bits) << 52));
        });
        const double rounded = fma(r, d, 0x1.8p52);
        return __builtin_bit_cast(uint64_t, rounded) + ((uint64_t(1) << shift) - __builtin_bit_cast(uint64_t, 0x1.8p52));
    }
    __device__ __forceinline__ void split(uint64_t h, double begin, uint32_t &tokens, double &weight) const {
        const int64_t dev = int64_t(h << (64 - shift)) >> (64 - shift);
        tokens = uint32_t((h - uint64_t(dev)) >> shift);
        weight = begin * fma(double(dev), __builtin_bit_cast(double, uint64_t(1023 - dev_bits) << 52), double(tokens));
    }
    __device__ __forceinline__ void fill(uint32_t &all_c, double &all_w) {
        // A bin's sum of `vocab` terms under 1 / UNIT stays in its field.
        shift = 63 - (32 - __clz(int(vocab)));
        dev_bits = min(37, 2 * shift - 64 + (31 - __builtin_clz(UNIT)));
        for (int i = tid; i < BINS; i += THREADS) s.bins[i] = 0;
        __syncthreads();
        const float from = least(kReach * UNIT);
        each_slowly<T, THREADS>(z, vocab, [&](float x) {
            if (x < from) return;
            const double y = place(x), at = floor(y);
            if (y < kReach * UNIT)
                atomicAdd(reinterpret_cast<unsigned long long *>(&s.bins[int(at)]),
                          static_cast<unsigned long long>(term(y - at)));
        });
        __syncthreads();
        double w = 0.0;
        uint32_t c = 0;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            uint32_t tokens;
            double weight;
            split(s.bins[tid * kEach + e], begin_of(tid * kEach + e), tokens, weight);
            w += weight;
            c += tokens;
        }
        s.before[tid] = block_scan<THREADS>(w, s.room_d, all_w);
        s.taken[tid] = block_scan<THREADS>(c, s.room_u, all_c);
        __syncthreads();
    }

    // The first bin that `is` takes; there has to be one.
    template <class Is>
    __device__ __forceinline__ Bin find(Is &&is) {
        Bin b{tid * kEach, s.taken[tid], 0, s.before[tid], 0.0};
        bool mine = false;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            if (!mine) {
                split(s.bins[b.at], begin_of(b.at), b.count, b.weight);
                mine = is(b);
            }
            if (!mine) b = {b.at + 1, b.taken + b.count, 0, b.base + b.weight, 0.0};
        }
        const uint64_t those = __ballot(mine);
        if (those == 0) {
            if (tid % 64 == 0) s.found_by[tid / 64].at = BINS;
        } else if (int(tid % 64) == __builtin_ctzll(those)) {
            s.found_by[tid / 64] = b;
        }
        __syncthreads();
        int w = 0;
        while (w + 1 < THREADS / 64 && s.found_by[w].at == BINS) ++w;
        b = s.found_by[w];
        b.base = uniform(b.base);
        b.weight = uniform(b.weight);
        __syncthreads();
        return b;
    }

    // The n-th token, from 0, whose logit has key k.
    __device__ __forceinline__ uint32_t nth_of(uint32_t k, uint32_t n) {
        const int lane = tid & 63;
        const uint32_t share = (vocab + THREADS - 1) / THREADS * 64, from = min(vocab, (tid >> 6) * share),
                       to = min(vocab, from + share);
        uint32_t c = 0, total;
        for (uint32_t i = from + lane; i < to; i += 64) c += order(T::to_float(z[i])) == k;
        const uint32_t before = block_scan<THREADS>(c, s.room_u, total);
        const uint32_t first = lane_value(before, 0), here = lane_value(before + c, 63) - first;
        if (n >= first && n - first < here) {  // this wave has it
            uint32_t left = n - first;
            for (uint32_t i = from; i < to; i += 64) {
                const bool is = i + lane < to && order(T::to_float(z[i + lane])) == k;
                const uint64_t mask = __ballot(is);
                const uint32_t step = uint32_t(__popcll(mask));
                if (left < step) {
                    if (is && uint32_t(__popcll(mask & ((uint64_t(1) << lane) - 1))) == left) s.found = i + lane;
                    break;
                }
                left -= step;
            }
        }
        __syncthreads();
        return s.found;
    }

    // From the bins: one border after the other, then the token.
    __device__ __forceinline__ void draw_bins(const SampleArgs &a, size_t row, const Settings &set) {
        // What is left: the first `left` tokens, with the weight `whole`.
        uint32_t left;
        double whole;
        fill(left, whole);
        whole = uniform(whole);
#pragma unroll 1
        for (int ask = kCount; ask < kAsks; ++ask) {
            // What depends on them alone is made where it is used, not kept in registers over the loop.
            asm volatile("" : "+v"(tid), "+s"(z));
            // The weight that is asked for, in all that is left or (kCount) its first tokens.
            double t = 0.0;
            if (ask == kCount) {
                if (!set.top_k || set.top_k >= left) continue;
                left = set.top_k;
            } else if (ask == kReachP) {
                if (!set.with_p) continue;
                t = uniform(set.top_p * whole);
            } else if (ask == kLeast) {
                if (!set.with_min) continue;
                // The bin of min_p, and its tokens from min_p on.
                if (!(until_min < kReach * UNIT)) continue;
                const int at = int(until_min);
                const float from = least(double(at + 1)), to = most(double(at));
                double w = 0.0;
                uint32_t c = 0;
                each_in<T, THREADS>(z, vocab, from, to, [&](float x, uint32_t) {
                    const double o = place(x);
                    if (o >= double(at) && o < double(at + 1)) {
                        const double v = weight_of(x);
                        if (v >= set.min_p) {
                            w += v;
                            ++c;
                        }
                    }
                });
                w = block_total<THREADS>(w, s.room_d);
                c = block_total<THREADS>(c, s.room_u);
                const Bin b = find([&](const Bin &o) { return o.at == at; });
                if (b.taken + c < left) {
                    left = b.taken + c;
                    whole = uniform(b.base + w);
                }
                continue;
            } else {
                t = uniform(set.uniform * whole);
            }
            const Bin b = find([&](const Bin &o) {
                return o.count && (o.taken + o.count >= left || (ask == kReachP ? o.base + o.weight >= t
                                                                                : ask == kDraw && o.base + o.weight > t));
            });
            const uint32_t q = left - b.taken;  // tokens of the bin that are left, or more
            // Inside the bin.
            const double from = double(b.at), until = double(b.at + 1);
            const float x_from = least(until), x_to = most(from);
            double base = b.base;
            uint32_t taken = 0, n = b.count;
            uint32_t lo = 0, hi = 0;
            bool ranked = n <= uint32_t(MOST);
            if (ranked) {
                if (tid == 0) s.n = 0;
                __syncthreads();
                each_in<T, THREADS>(z, vocab, x_from, x_to, [&](float x, uint32_t token) {
                    const double y = place(x);
                    if (y >= from && y < until) append(x, token);
                });
                __syncthreads();
                n = min(s.n, uint32_t(MOST));
            } else {
                lo = 0xffffffffu;
                each_in<T, THREADS>(z, vocab, x_from, x_to, [&](float x, uint32_t) {
                    const double y = place(x);
                    if (y >= from && y < until) {
                        lo = min(lo, order(x));
                        hi = max(hi, order(x));
                    }
                });
                if (tid == 0) {
                    s.lo = 0xffffffffu;
                    s.hi = 0;
                }
                __syncthreads();
                atomicMin(&s.lo, lo);
                atomicMax(&s.hi, hi);
                __syncthreads();
                lo = s.lo;
                hi = s.hi;
                __syncthreads();
            }
            const double begin = begin_of(b.at);
            while (!ranked && lo != hi) {
                constexpr int kBits = 31 - __builtin_clz(THREADS);
                const int step = max(0, 32 - __clz(int(hi - lo)) - kBits);  // (hi - lo) >> step < THREADS
                s.fine[tid] = 0;
                __syncthreads();
                each_in<T, THREADS>(z, vocab, unordered(lo), unordered(hi), [&](float x, uint32_t) {
                    atomicAdd(reinterpret_cast<unsigned long long *>(&s.fine[(hi - order(x)) >> step]),
                              static_cast<unsigned long long>(term(place(x) - from)));
                });
                if (tid == 0) {
                    s.found = THREADS;
                    s.n = 0;
                }
                __syncthreads();
                uint32_t c, all_c;
                double w, all_w;
                split(s.fine[tid], begin, c, w);
                const double before_w = base + block_scan<THREADS>(w, s.room_d, all_w);
                const uint32_t before_c = taken + block_scan<THREADS>(c, s.room_u, all_c);
                if (c) {
                    atomicMax(&s.n, uint32_t(tid));
                    if (before_c + c >= q || (ask == kReachP ? before_w + w >= t : ask == kDraw && before_w + w > t))
                        atomicMin(&s.found, uint32_t(tid));
                }
                __syncthreads();
                const uint32_t sub = s.found < uint32_t(THREADS) ? s.found : s.n;
                __syncthreads();
                if (sub == uint32_t(tid)) {
                    s.base = before_w;
                    s.lo = before_c;
                    s.hi = c;
                }
                __syncthreads();
                base = uniform(s.base);
                taken = s.lo;
                n = s.hi;
                hi -= sub << step;
                const uint32_t span = (uint32_t(1) << step) - 1;
                if (hi - lo > span) lo = hi - span;
                ranked = n <= uint32_t(MOST);
                if (ranked) {
                    if (tid == 0) s.n = 0;
                    __syncthreads();
                    each_in<T, THREADS>(z, vocab, unordered(lo), unordered(hi),
                                        [&](float x, uint32_t token) { append(x, token); });
                }
                __syncthreads();
            }
            if (ranked) {
                rank(n);
                if (ask == kDraw) {
                    finish(a, row, s.list[min(below(n, t - base, true), min(n, q - taken) - 1)], whole);
                    return;
                }
                const uint32_t c = ask == kCount ? min(n, q - taken) : min(min(n, q - taken), below(n, t - base, false) + 1);
                left = b.taken + taken + c;
                whole = uniform(base + s.sums[c - 1]);
                __syncthreads();
            } else {  // equal logits, in the order of their tokens
                const double w = weight_of(unordered(lo));
                n = min(n, q - taken);
                if (ask == kDraw) {
                    const uint32_t token = nth_of(lo, equal_draw(t - base, w, n));
                    if (tid == 0) write(a, row, token, float(log(w / whole)));
                    return;
                }
                const uint32_t c = ask == kCount ? n : equal_reach(t - base, w, n);
                left = b.taken + taken + c;
                whole = uniform(base + double(c) * w);
            }
        }
    }
};

// Rows of which few tokens are left before any weight is summed.
__device__ __forceinline__ bool left_few(const Settings &set, int threads) {
    return (set.top_k && set.top_k <= uint32_t(threads / 2)) || (set.with_min && !set.with_p);
}

template <class T, int THREADS, int UNIT, int MOST>
__device__ __forceinline__ void sample_by_bins(const SampleArgs &a, size_t row, const Settings &set,
                                               typename Bins<T, THREADS, UNIT, MOST>::Shared &s) {
    using B = Bins<T, THREADS, UNIT, MOST>;
    B b(static_cast<const typename T::Raw *>(a.logits) + row * a.stride, uint32_t(a.vocab), s);
    b.until_min = uniform(set.with_min ? -log(set.min_p) * UNIT : 0.0);
    Weights<UNIT>::prepare(s.powers);
    float mine = -INFINITY;
    bool bad = false;
    each<T, THREADS>(b.z, b.vocab, [&](float x) {
        mine = fmaxf(mine, x);
        bad |= !(x < INFINITY);
    });
    const float wave_top = wave_largest(mine);
    const bool wave_bad = __ballot(bad) != 0;
    if (b.tid % 64 == 0) {
        s.room_f[b.tid / 64] = wave_top;
        s.room_u[b.tid / 64] = wave_bad;
    }
    if (b.tid == 0) {
        s.n = 0;
        s.found = kNoToken;
    }
    __syncthreads();
    b.top = -INFINITY;
    uint32_t any_bad = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        b.top = fmaxf(b.top, s.room_f[w]);
        any_bad |= s.room_u[w];
    }
    b.top = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(uint32_t, b.top)));
    if (any_bad || b.top == -INFINITY || !set.valid) {
        if (b.tid == 0) write(a, row, kNoToken, NAN);
        return;
    }
    if (set.greedy) {
        uint32_t first = kNoToken;
        each_in<T, THREADS>(b.z, b.vocab, b.top, b.top, [&](float, uint32_t token) { first = min(first, token); });
        if (first != kNoToken) atomicMin(&s.found, first);
        __syncthreads();
        if (b.tid == 0) write(a, row, s.found, 0.0f);
        return;
    }
    b.scale = uniform(UNIT / set.temperature);
    if (left_few(set, THREADS)) {
        const bool by_k = set.top_k && set.top_k <= uint32_t(THREADS / 2);
        const float from = by_k ? b.least(double(b.bound_bin(mine, set.top_k) + 1)) : b.least(b.until_min);
        each_in<T, THREADS>(b.z, b.vocab, from, FLT_MAX, [&](float x, uint32_t token) { b.append(x, token); });
        __syncthreads();
        const uint32_t n = s.n;
        if (n <= uint32_t(MOST)) return b.draw_few(a, row, set, n);
        __syncthreads();
    }
    b.draw_bins(a, row, set);
}

template <class T, int THREADS, int UNIT, int MOST>
__global__ void __launch_bounds__(THREADS) sample_bins_kernel(SampleArgs a) {
    __shared__ typename Bins<T, THREADS, UNIT, MOST>::Shared s;
    const size_t row = blockIdx.x;
    sample_by_bins<T, THREADS, UNIT, MOST>(a, row, settings_of(a, row), s);
}

// ---- rows of 16 bits ------------------------------------------------------------------

// Logits of 16 bits have 65536 values: one pass counts each, two to an LDS word, with
// the row kept in registers, and all the rest follows from the counts, the weights of
// the values and (the n-th of equal logits) a look through the registers.
//
// In rank order the values are q = 0..65535: the positive ones downwards, q = 0x7fff
// minus the code, then the negative ones, q = the code.  They are summed in segments
// of 64.  One code is counted apart, without its LDS word, which all lanes would meet
// in: -inf, or what a sample of the row is full of (a mask's value).  No other code can
// overflow its 16 bits unless it has more than half of the row; then it is looked for
// and counted apart in a second pass.
//
// The counts fill a CU's LDS, so rows follow each other on it: 1000 rows of 128001 BF16
// with top_p 163 us, 1.6 TB/s, four rows a CU of 41 us each: some 20 until the row is
// there and counted as it comes, by LDS atomics (171 in all when counted afterwards), 8 to
// sum and weigh the segments, 11 to find the borders and the token.  1024 rows of 128000
// by bins, whose fill is FP64 work for each logit, take 261.
constexpr int kCodeThreads = 1024;
constexpr int kCodeGroups = 16;  // of 8 logits a thread
constexpr uint32_t kCodeMost = 131071;
static_assert(kCodeMost < kCodeThreads * kCodeGroups * 8, "a row fits the registers");

template <class T>
struct Codes {
    static constexpr int kUnit = 128, THREADS = kCodeThreads, WAVES = THREADS / 64, GROUPS = kCodeGroups;
    // The shortest rows counted.  F16 has eight times the values at a logit's size, so more
    // segments to weigh: counted and by bins, 1000 rows of 64000 take 167 and 142 us, of 96000
    // 190 and 198 (BF16: of 50000 113 and 134 for 1024).
    static constexpr uint32_t kLeast = std::is_same<T, F16>::value ? 81920 : 32769;
    static constexpr uint32_t kInf = std::is_same<T, F16>::value ? 0x7c00 : 0x7f80, kNegative = 0x8000 | kInf;

    struct Part {
        uint32_t segment, taken;
        double base;
    };
    struct Shared {
        uint32_t counts[32768 + THREADS];  // of a code and its negative; then of the code counted apart, a word a thread
        uint32_t in_segment[THREADS];
        double weights[THREADS];
        Powers<kUnit> powers;
        double room_d[WAVES];
        uint32_t room_u[WAVES];
        uint32_t bits[16];
        Part parts[WAVES];
    };

    Shared &s;
    uint32_t tid, lane, wave;
    uint32_t hot, hot_count;  // counted apart
    Weights<kUnit> weights;

    static __device__ __forceinline__ uint32_t code_at(uint32_t q) { return q < 0x8000 ? 0x7fff - q : q; }
    static __device__ __forceinline__ uint32_t segment_of(uint32_t code) { return (code < 0x8000 ? 0x7fff - code : code) / 64; }
    static __device__ __forceinline__ float value(uint32_t code) { return T::to_float(__builtin_bit_cast(typename T::Raw, uint16_t(code))); }
    __device__ __forceinline__ uint32_t count_of(uint32_t code) const {
        if (code == hot) return hot_count;
        return s.counts[code & 0x7fff] >> (code / 0x8000 * 16) & 0xffff;
    }

    // The first segment that `is` takes ((weights, tokens) before and in it), or segment THREADS.
    template <class Is>
    __device__ __forceinline__ Part first(double base, uint32_t taken, Is &&is) {
        const bool mine = is();
        const uint64_t those = __ballot(mine);
        if (those == 0) {
            if (lane == 0) s.parts[wave].segment = THREADS;
        } else if (int(lane) == __builtin_ctzll(those)) {
            s.parts[wave] = {tid, taken, base};
        }
        __syncthreads();
        int w = 0;
        while (w + 1 < WAVES && s.parts[w].segment == uint32_t(THREADS)) ++w;
        Part p = s.parts[w];
        p.segment = __builtin_amdgcn_readfirstlane(p.segment);
        p.taken = __builtin_amdgcn_readfirstlane(p.taken);
        p.base = uniform(p.base);
        __syncthreads();
        return p;
    }

    // The values of a segment, one a lane, with what is before each.
    struct Value {
        uint32_t code, count, taken;
        double weight, base;
    };
    __device__ __forceinline__ Value value_of(uint32_t segment) const {
        Value v{};
        v.code = code_at(segment * 64 + lane);
        v.count = count_of(v.code);
        if (v.code == kNegative) v.count = 0;
        v.weight = v.count ? weights.of(value(v.code)) : 0.0;
        if (v.weight == 0.0) v.count = 0;
        return v;
    }
    __device__ __forceinline__ Value value_in(const Part &p) const {
        Value v = value_of(p.segment);
        const double w = double(v.count) * v.weight;
        v.base = p.base + wave_scan(w) - w;
        v.taken = p.taken + wave_scan(v.count) - v.count;
        return v;
    }
    // Lane l's.
    static __device__ __forceinline__ Value lane_of(Value v, int l) {
        v.code = __builtin_amdgcn_readlane(v.code, l);
        v.count = __builtin_amdgcn_readlane(v.count, l);
        v.taken = __builtin_amdgcn_readlane(v.taken, l);
        v.weight = lane_value(v.weight, l);
        v.base = lane_value(v.base, l);
        return v;
    }
};

// One of the groups, which are in registers (a choice by masks: one by an index would put them into memory).
__device__ __forceinline__ u32x4 group_of(const u32x4 (&w)[kCodeGroups], int at) {
    u32x4 g = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < kCodeGroups; ++j) g |= w[j] & (at == j ? 0xffffffffu : 0u);
    return g;
}

// The code that most of a sample of the row has, if it has a quarter of a wave's.
template <class C>
__device__ __forceinline__ uint32_t sampled_code(C &c, u32x4 g) {
    const uint32_t word = c.lane & 4 ? (c.lane & 2 ? g[3] : g[2]) : (c.lane & 2 ? g[1] : g[0]);
    const uint32_t code = word >> (c.lane % 2 * 16) & 0xffff;
    uint64_t rest = __ballot((code & 0x7fff) != 0x7fff);  // not what fills the last wave
    uint32_t most = 15, at = 0;
#pragma unroll 1
    for (int i = 0; i < 4 && rest; ++i) {
        const uint32_t one = __builtin_amdgcn_readlane(code, __builtin_ctzll(rest));
        const uint64_t same = __ballot(code == one);
        rest &= ~same;
        if (uint32_t(__popcll(same)) > most) {
            most = uint32_t(__popcll(same));
            at = one;
        }
    }
    if (c.lane == 0) c.s.room_u[c.wave] = most << 16 | at;
    __syncthreads();
    uint32_t best = 0;
#pragma unroll
    for (int v = 0; v < C::WAVES; ++v) best = max(best, c.s.room_u[v]);
    __syncthreads();
    return best >> 16 > 15 ? best & 0xffff : C::kNegative;
}

template <class T>
__global__ void __launch_bounds__(kCodeThreads) sample_codes_kernel(SampleArgs a) {
    using C = Codes<T>;
    using Raw = typename T::Raw;
    using Few = typename Bins<T, kCodeThreads, 128, 2048>::Shared;
    __shared__ union {
        typename C::Shared codes;
        Few bins;
    } room;
    const size_t row = blockIdx.x;
    const Settings set = settings_of(a, row);
    // These want only the largest logit and the few next to it.
    if (set.greedy || left_few(set, kCodeThreads)) return sample_by_bins<T, kCodeThreads, 128, 2048>(a, row, set, room.bins);
    typename C::Shared &s = room.codes;
    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = tid / 64, vocab = uint32_t(a.vocab);
    const Raw *const z = static_cast<const Raw *>(a.logits) + row * a.stride;
    // A wave has `each` times 64 groups in a row, and a lane every 64th of them.
    const uint32_t groups = vocab / 8, tail = vocab % 8, each = (groups + C::THREADS - 1) / C::THREADS;
    const auto group = [&](int g) { return (wave * each + uint32_t(g)) * 64 + lane; };
    // All of them are loaded, those past `each` from one place: a load under a condition would
    // make the wait for the first one a wait for all.
    u32x4 w[kCodeGroups];
#pragma unroll
    for (int j = 0; j < kCodeGroups; ++j)
        w[j] = *reinterpret_cast<const u32x4_any *>(z + size_t(uint32_t(j) < each ? min(group(j), groups - 1) : groups - 1) * 8);
    const uint32_t last = tid < tail ? uint32_t(__builtin_bit_cast(uint16_t, z[groups * 8 + tid])) : 0;
    Weights<C::kUnit>::prepare(s.powers);
    C c{s, tid, lane, wave, 0, 0, {s.powers, 0.0, uniform(C::kUnit / set.temperature)}};
    // Behind the row's groups there is NaN, which no token that is drawn is.
    const auto filled = [&](int g) { return group(g) < groups ? w[g] : w[g] | 0x7fff7fffu; };
    c.hot = sampled_code(c, filled(0));  // the others are counted as they come
    uint32_t mine;  // tokens of a thread's segment, without those of -inf
#pragma unroll 1
    for (bool again = false;; again = true) {
#pragma unroll
        for (int i = 0; i < 8; ++i) reinterpret_cast<uint4 *>(s.counts)[i * C::THREADS + tid] = uint4{0, 0, 0, 0};
        s.counts[32768 + tid] = 0;
        __syncthreads();
        // What is counted apart goes to the thread's own word (in the code's word all lanes
        // of a wave would wait for each other: 156 us for 112000 of 128001 logits, else 10).
        const uint32_t own = 32768 + tid;
        const auto count = [&](uint32_t code) {
            atomicAdd(&s.counts[code == c.hot ? own : code & 0x7fff], code & 0x8000 ? 65536u : 1u);
        };
#pragma unroll
        for (int j = 0; j < kCodeGroups; ++j) {
            if (uint32_t(j) < each) {
                asm volatile("" : "+v"(w[j]));  // what is made of it is not kept from one pass for the other
                w[j] = filled(j);
            }
            if (uint32_t(j) < each && group(j) < groups) {
#pragma unroll
                for (int e = 0; e < 8; ++e) count(w[j][e / 2] >> (e % 2 * 16) & 0xffff);
            }
            __builtin_amdgcn_sched_barrier(0);  // one group's registers at a time
        }
        if (tid < tail) count(last);
        __syncthreads();
        c.hot_count = block_total<C::THREADS>(__builtin_amdgcn_sad_u16(s.counts[32768 + tid], 0, 0), s.room_u);
        // A thread's segment: one half of 64 words in a row, begun at another one in each lane.
        const uint32_t from = tid < 512 ? 32768 - 64 * (tid + 1) : 64 * (tid - 512), half = tid < 512 ? 0 : 16;
        uint32_t n = 0;
#pragma unroll 8
        for (uint32_t i = 0; i < 64; ++i) n += s.counts[from + (i + tid) % 64] >> half & 0xffff;
        const uint32_t all = block_total<C::THREADS>(n, s.room_u);
        if (tid == C::segment_of(C::kNegative) && c.hot != C::kNegative) n -= c.count_of(C::kNegative);
        if (tid == C::segment_of(c.hot) && c.hot != C::kNegative) n += c.hot_count;
        mine = n;
        if (again || all + c.hot_count == vocab) break;
        // Some code has overflowed: it has most of the row, and each of its bits most of theirs.
        uint32_t ones[16];
        if (tid < 16) s.bits[tid] = 0;
        __syncthreads();
#pragma unroll
        for (int b = 0; b < 16; ++b) ones[b] = 0;
#pragma unroll 1
        for (uint32_t i = tid; i < (vocab + 63) / 64 * 64; i += C::THREADS) {
            const uint32_t code = i < vocab ? __builtin_bit_cast(uint16_t, z[i]) : 0;
#pragma unroll
            for (int b = 0; b < 16; ++b) ones[b] += uint32_t(__popcll(__ballot(code >> b & 1)));
        }
#pragma unroll
        for (int b = 0; b < 16; ++b)
            if (lane == 0) atomicAdd(&s.bits[b], ones[b]);
        __syncthreads();
        c.hot = uint32_t(__ballot(lane < 16 && 2 * s.bits[lane % 16] > vocab));
        __syncthreads();
    }

    // What is not a number or +inf comes first in the order, and last, with -inf.
    const bool odd = mine && (tid <= C::segment_of(C::kInf) || tid >= C::segment_of(C::kNegative));
    s.in_segment[tid] = mine;
    s.weights[tid] = 0.0;
    const typename C::Part begin = c.first(0.0, 0, [&] { return mine != 0; });
    const bool bad = block_total<C::THREADS>(uint32_t(odd), s.room_u) != 0;
    if (bad || begin.segment == uint32_t(C::THREADS) || !set.valid) {
        if (tid == 0) write(a, row, kNoToken, NAN);
        return;
    }
    uint32_t code = C::code_at(begin.segment * 64 + lane);
    code = __builtin_amdgcn_readlane(code, __builtin_ctzll(__ballot(c.count_of(code) != 0)));
    c.weights.top = uniform(double(C::value(code)));
    // The segments' weights, a wave a segment; and what is over min_p.
    double over = 0.0;
    uint32_t over_count = 0;
    uint64_t full = __ballot(s.in_segment[wave + C::WAVES * lane] != 0);
    while (full) {  // two at a time: each is a chain
        uint32_t segment[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            segment[i] = full ? wave + C::WAVES * uint32_t(__builtin_ctzll(full)) : segment[0];
            full &= full - 1;
        }
        const typename C::Value v[2] = {c.value_of(segment[0]), c.value_of(segment[1])};
        double weight[2];
        uint32_t count[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const double sum = double(v[i].count) * v[i].weight;
            if (set.with_min && v[i].weight >= set.min_p && (i == 0 || segment[1] != segment[0])) {
                over += sum;
                over_count += v[i].count;
            }
            weight[i] = wave_total(sum);
            count[i] = wave_total(v[i].count);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (lane == 0) {
                s.weights[segment[i]] = weight[i];
                s.in_segment[segment[i]] = count[i];
            }
    }
    __syncthreads();
    // What is left: the first `left` tokens, with the weight `whole`.
    const double weight = s.weights[tid];
    const uint32_t count = s.in_segment[tid];
    double whole;
    uint32_t left;
    const double base = block_scan<C::THREADS>(weight, s.room_d, whole);
    const uint32_t taken = block_scan<C::THREADS>(count, s.room_u, left);
    whole = uniform(whole);
    // The value at which the tokens reach `left`, or (p) the weights t, or exceed it.
    const auto find = [&](double t, bool p, bool over_t) {
        const typename C::Part part = c.first(base, taken, [&] {
            return count && (taken + count >= left || (p && base + weight >= t) || (over_t && base + weight > t));
        });
        const typename C::Value v = c.value_in(part);
        const double until = v.base + double(v.count) * v.weight;
        const uint64_t any = __ballot(v.count != 0);
        const uint64_t those = __ballot(v.count && (v.taken + v.count >= left || (p && until >= t) || (over_t && until > t)));
        return C::lane_of(v, those ? __builtin_ctzll(those) : 63 - __builtin_clzll(any));
    };
    if (set.top_k && set.top_k < left) {
        left = set.top_k;
        const typename C::Value v = find(0.0, false, false);
        whole = v.base + double(left - v.taken) * v.weight;
    }
    if (set.with_p) {
        const double t = set.top_p * whole;
        const typename C::Value v = find(t, true, false);
        const uint32_t n = equal_reach(t - v.base, v.weight, min(v.count, left - v.taken));
        left = v.taken + n;
        whole = v.base + double(n) * v.weight;
    }
    if (set.with_min) {
        over = block_total<C::THREADS>(over, s.room_d);
        over_count = block_total<C::THREADS>(over_count, s.room_u);
        if (over_count < left) {
            left = over_count;
            whole = over;
        }
    }
    const double t = set.uniform * whole;
    const typename C::Value v = find(t, false, true);
    uint32_t at = equal_draw(t - v.base, v.weight, min(v.count, left - v.taken));
    code = v.code;
    const double share = uniform(v.weight / whole);  // of the token that is drawn

    // The at-th token of that code, from 0; the two zeros are equal.
    const bool zero = (code & 0x7fff) == 0;
    if (code == 0x8000) at += c.count_of(0);
    const uint32_t bits = zero ? 0x7fff7fffu : 0xffffffffu, wanted = (code & bits) * 0x10001u;
    const auto others = [&](u32x4 g) {  // of its 8 logits, in two halves: a difference has a bit
        u16x2 n = {0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            n += __builtin_elementwise_min(__builtin_bit_cast(u16x2, (g[e] & bits) ^ wanted), u16x2{1, 1});
        return n;
    };
    const auto matches = [&](u32x4 g) {
        const u16x2 n = others(g);
        return uint32_t(8 - n[0] - n[1]);
    };
    const auto in_group = [&](int g) { return uint32_t(g) < each ? matches(w[g]) : 0; };
    u16x2 apart = {0, 0};
#pragma unroll
    for (int g = 0; g < kCodeGroups; ++g)
        if (uint32_t(g) < each) apart += others(w[g]);
    uint32_t n = 8 * each - apart[0] - apart[1];
    // The wave that has it, or the tail behind the waves; there the group; there the lane.
    n = wave_total(n);
    if (lane == 0) s.room_u[wave] = n;
    __syncthreads();
    uint32_t own = lane < C::WAVES ? s.room_u[lane] : 0, sum = row_scan(own);
    uint64_t those = __ballot(lane < C::WAVES && sum > at);
    const bool in_tail = those == 0;
    if ((in_tail ? 0 : uint32_t(__builtin_ctzll(those))) != wave) return;
    uint32_t before = in_tail ? lane_value(sum, C::WAVES - 1) : lane_value(sum - own, int(wave)), skip;
    int g = 0;
    if (in_tail) {
        own = tid < tail && (last & bits) == (wanted & 0xffff);
    } else {
        uint32_t pairs[kCodeGroups / 2];  // two groups' sums, of up to 512 each, a word
#pragma unroll
        for (int i = 0; i < kCodeGroups / 2; ++i) pairs[i] = wave_scan(in_group(2 * i) | in_group(2 * i + 1) << 16);
#pragma unroll
        for (int i = 0; i < kCodeGroups; ++i) {
            const uint32_t here = lane_value(pairs[i / 2], 63) >> (i % 2 * 16) & 0xffff;
            if (before + here > at || g != i) continue;
            before += here;
            ++g;
        }
        own = matches(group_of(w, g));
    }
    sum = before + wave_scan(own);
    those = __ballot(sum > at);
    if (those == 0 || lane != uint32_t(__builtin_ctzll(those))) return;
    skip = at - (sum - own);
    uint32_t token = groups * 8 + tid;
    if (!in_tail) {
        const u32x4 v = group_of(w, g);
        token = group(g) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool is = ((v[e / 2] >> (e % 2 * 16) ^ wanted) & bits & 0xffff) == 0;
            if (is && skip == 0) token += e;
            if (is) --skip;
        }
    }
    write(a, row, token, float(log(share)));
}

// What bounds short rows is the barriers and scans that a row takes, which wait less with
// fewer waves; with bins of 1 / 32 each of 256 threads has four.  Measured, BF16 and top_p, in
// us, with 256 threads and 512: 1024 rows of 300 19 and 43, of 4000 28 and 48, of 8000 38 and
// 53, of 16000 54 and 58; 256 rows of 4000 16 and 19, of 8000 28 and 20.  With 512 and 1024:
// 1024 rows of 30000 75 and 95, 256 of them 30 and 26.  Counting by value has a fixed part:
// 256 rows of 16000 23 where 512 threads take 22, of 50000 29 where 1024 threads and bins
// take 36, of 128000 42 and 78.
template <class T>
void launch(const SampleArgs &a, hipStream_t stream) {
    const dim3 rows(static_cast<unsigned>(a.rows));
    const bool many = a.rows > 512;  // workgroups share the CUs
    if (a.vocab <= 64)
        sample_short_kernel<T, 64><<<rows, 256, 0, stream>>>(a);
    else if (a.vocab <= 256)
        sample_short_kernel<T, 256><<<rows, 1024, 0, stream>>>(a);
    else if (a.vocab <= (many ? 8192 : 4096))
        sample_bins_kernel<T, 256, 32, 1024><<<rows, 256, 0, stream>>>(a);
    else if (a.vocab <= (many ? 32768 : 16384))
        sample_bins_kernel<T, 512, 128, 1024><<<rows, 512, 0, stream>>>(a);
    else if (sizeof(typename T::Raw) == 4 || a.vocab < Codes<T>::kLeast || a.vocab > kCodeMost)
        sample_bins_kernel<T, 1024, 128, 2048><<<rows, 1024, 0, stream>>>(a);
    else if constexpr (sizeof(typename T::Raw) == 2)
        sample_codes_kernel<T><<<rows, kCodeThreads, 0, stream>>>(a);
}

// ---- a model's step ---------------------------------------------------------------------

// A step's scratch: temperatures, top_k, top_p, min_p, random numbers and tokens of `rows` rows.
__global__ void sample_rows_kernel(uint32_t *scratch, size_t rows, float temperature, int top_k, float top_p, float min_p,
                                   uint64_t *rng) {
    const size_t r = size_t(blockIdx.x) * blockDim.x + threadIdx.x;
    if (r >= rows) return;
    uint64_t state = rng[r];
    scratch[r] = __builtin_bit_cast(uint32_t, temperature);
    scratch[rows + r] = uint32_t(top_k);
    scratch[2 * rows + r] = __builtin_bit_cast(uint32_t, top_p);
    scratch[3 * rows + r] = __builtin_bit_cast(uint32_t, min_p);
    scratch[4 * rows + r] = __builtin_bit_cast(uint32_t, rng_unit(state));
    rng[r] = state;
}

// Appends a row's token, a wave a row; one with a logit that is not finite is flagged.
__global__ void __launch_bounds__(64)
sample_append_kernel(SampleArgs a, uint32_t *tokens, int token_stride, int *len, int *flags) {
    const size_t r = blockIdx.x;
    const float *const z = static_cast<const float *>(a.logits) + r * a.stride;
    bool odd = false;
    for (size_t i = threadIdx.x; i < a.vocab; i += 64) odd |= !(fabsf(z[i]) < INFINITY);
    odd = __ballot(odd) != 0;
    if (threadIdx.x) return;
    const uint32_t token = a.tokens[r];
    if (odd) atomicOr(flags, 1);
    const int n = len[r];
    tokens[r * size_t(token_stride) + n] = token < a.vocab ? token : 0;
    len[r] = n + 1;
}

}  // namespace

void sample_step(const float *logits, size_t vocab, size_t batch, float temperature, uint32_t top_k, float top_p,
                 float min_p, uint64_t *rng, void *scratch, uint32_t *tokens, int token_stride, int *len, int *flags,
                 hipStream_t stream) {
    float *const f = static_cast<float *>(scratch);
    SampleArgs a{};
    a.logits = logits;
    a.rows = batch;
    a.vocab = a.stride = vocab;
    a.temperatures = f;
    a.top_k = reinterpret_cast<int *>(f + batch);
    a.top_p = f + 2 * batch;
    a.min_p = f + 3 * batch;
    a.uniforms = f + 4 * batch;
    a.tokens = reinterpret_cast<uint32_t *>(f + 5 * batch);
    const int k = int(std::min<uint32_t>(top_k, 1u << 30));
    sample_rows_kernel<<<dim3(unsigned((batch + 255) / 256)), 256, 0, stream>>>(static_cast<uint32_t *>(scratch), batch,
                                                                                 temperature, k, top_p, min_p, rng);
    launch<F32>(a, stream);
    sample_append_kernel<<<dim3(unsigned(batch)), 64, 0, stream>>>(a, tokens, token_stride, len, flags);
}

void sample_filtered(const SampleArgs &a, Type type, hipStream_t stream) {
    switch (type) {
        case Type::F32: return launch<F32>(a, stream);
        case Type::F16: return launch<F16>(a, stream);
        case Type::BF16: return launch<BF16>(a, stream);
    }
}

}  // namespace meshgpt::kern
