// The root-mean-square norm with the residual's addition, with an output in the
// rows' type or in 8 bits, and its gradient.
//
//   h = x + residual, rounded to the type and kept;
//   rstd = 1 / sqrt(mean(h^2) + epsilon);  y = h rstd w.
// In 8 bits a scale 2^(b - 127) belongs to 32 channels: the smallest power of two
// with which the largest of them is at most 448.
//   g = dy w;  dh = rstd (g - hat mean(g hat)) + dsum;  dw = sum of dy hat over rows, hat = h rstd.
//
// All but the gradient of the widest rows read a row once: it stays in registers, 16 bytes
// a load, in part of a wave for short rows (heads) and in up to 16 for long ones.  The norm's
// sum of a row is FP64, which no FP32 value overflows; so is what decides a scale, where
// values next to a power of two are met in any large batch.  The gradient's products, and
// their sums over 16 bytes of a row, are FP32; a row's sum of those is FP64.  The weight's
// gradient is summed over a team's rows, 64 of them in FP32 and such sums in FP64, then over
// the teams in a fixed order.
//
// Memory bounds all of them at length: with a residual that is kept, 16384 x 4096 BF16 93 us
// (5.8 TB/s), 4001 x 5120 F16 to codes 32 (4.5); 32 x 512 F32 3.1 us, a launch and a chain
// of one load and one join.
#include "dpp.hpp"
#include "operators.hpp"
#include "types.hpp"

namespace meshgpt::kern {
namespace {

// Group g of a row: loaded, and then zero behind the row's end.  A group that the end cuts
// is read by a load that ends there (a row of less than a group by its elements), and
// trimmed once it is used, so that loads stay under way together.
template <class T>
__device__ __forceinline__ uint4 load_group(const typename T::Raw *row, int g, int width) {
    constexpr int G = T::kGroup;
    if (width < G) return g == 0 ? get_part<T>(row, width) : uint4{0, 0, 0, 0};
    return get_any(row + uint32_t(min(g * G, width - G)));
}
template <class T>
__device__ __forceinline__ uint4 trim_group(uint4 w, int g, int width) {
    constexpr int G = T::kGroup;
    const int over = g * G - (width - G);
    if (width >= G && __ballot(over > 0)) w = moved_down<T>(w, min(max(over, 0), G));
    return w;
}
template <class T>
__device__ __forceinline__ void store_group(typename T::Raw *row, int g, int width, uint4 w) {
    const int have = width - g * T::kGroup;
    if (have >= T::kGroup) return put_any(reinterpret_cast<char *>(row) + uint32_t(g) * 16u, w);
    put_part<T>(row + g * T::kGroup, have, w);
}

// How a row is held: in the registers of LANES lanes of a wave (16, 32 or 64), or of a
// workgroup of whole waves: up to 8 (kBlockRow) or 16 (kWideRow), with half the registers.
constexpr int kBlockRow = 0, kWideRow = -1;
template <int LANES_>
struct Team {
    static constexpr int LANES = LANES_ > 0 ? LANES_ : 0;
    int lane, lanes, of;  // this thread in its team, the team's threads, the team in its workgroup
    __device__ __forceinline__ Team()
        : lane(LANES ? threadIdx.x % (LANES ? LANES : 1) : threadIdx.x), lanes(LANES ? LANES : blockDim.x),
          of(LANES ? threadIdx.x / (LANES ? LANES : 1) : 0) {
        if (LANES == 64) of = __builtin_amdgcn_readfirstlane(of);
    }
    // The sum of its values, in all of its threads.
    __device__ __forceinline__ double sum(double v, double *room) const {
#pragma unroll
        for (int d = (LANES ? LANES : 64) / 2; d > 0; d /= 2) v += __shfl_xor(v, d, 64);
        if constexpr (LANES == 0) {
            __syncthreads();  // of the row before
            if (threadIdx.x % 64 == 0) room[threadIdx.x / 64] = v;
            __syncthreads();
            v = 0.0;
            for (int w = 0; w < lanes / 64; ++w) v += room[w];
        }
        return v;
    }
};
constexpr int kBlock = 256;  // threads of a workgroup with several rows
constexpr int kWavesMost = 16;
template <int LANES>
constexpr int kThreads = LANES > 0 ? kBlock : LANES == kBlockRow ? 512 : 1024;  // at most

// v in FP32 for a conversion to fewer bits: 20 bits behind the first, of which what
// follows sets the last, so that a value next to the middle of two codes does not become it.
__device__ __forceinline__ float for_rounding(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return float(__builtin_bit_cast(double, uint64_t(uint32_t(b >> 32) | min(uint32_t(b), 1u)) << 32));
}

// Four E4M3 codes.
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}

// The codes c of a group u w rstd, with the scale 2^n of the 32 channels that it is in.
// V holds the products: FP32 those of F16 values, exactly; others leave its bits or its
// range.  4001 x 5120 take 29.5 us so, in BF16 with FP64's 30.8.
template <class V, int G>
__device__ __forceinline__ void encode_group(const float (&u)[G], const float (&w)[G], double rstd, uint32_t (&c)[G / 4], int &n) {
    V y[G], top = 0;
#pragma unroll
    for (int e = 0; e < G; ++e) {
        y[e] = V(u[e]) * V(w[e]);
        top = sizeof(V) == 4 ? V(fmaxf(float(top), fabsf(float(y[e])))) : V(fmax(double(top), fabs(double(y[e]))));
    }
#pragma unroll
    for (int d = 1; d < 32 / G; d *= 2) {
        const V other = __shfl_xor(top, d, 64);
        top = sizeof(V) == 4 ? V(fmaxf(float(top), float(other))) : V(fmax(double(top), double(other)));
    }
    // The largest is m 2^k, 1 <= m < 2; 448 = 1.75 * 2^8.
    const uint64_t bits = __builtin_bit_cast(uint64_t, double(top) * rstd);
    n = int(bits >> 52) - 1023 - 8 + ((bits & 0xfffffffffffffull) > 0xc000000000000ull);
    n = min(max(n, -117), 120);
    const double by = rstd * __builtin_bit_cast(double, uint64_t(1023 - n) << 52);
#pragma unroll
    for (int e = 0; e < G; e += 4)
        c[e / 4] = encode4(for_rounding(double(y[e]) * by), for_rounding(double(y[e + 1]) * by),
                           for_rounding(double(y[e + 2]) * by), for_rounding(double(y[e + 3]) * by));
}

template <class T, int LANES, int GROUPS, bool CODES>
__global__ void __launch_bounds__(kThreads<LANES>) norm_kernel(NormArgs a) {
    using Raw = typename T::Raw;
    constexpr int G = T::kGroup;
    __shared__ double room[kWavesMost];
    const Team<LANES> team;
    const int lane = team.lane, lanes = team.lanes, width = a.width;
    const size_t row = LANES > 0 ? size_t(blockIdx.x) * (kBlock / (LANES > 0 ? LANES : 1)) + team.of : blockIdx.x;
    if (row >= a.rows) return;  // whole teams, whose sums are their own
    const Raw *const x = static_cast<const Raw *>(a.x) + row * a.xs;
    const Raw *const weight = static_cast<const Raw *>(a.weight);
    uint4 h[GROUPS];
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) h[i] = load_group<T>(x, lane + i * lanes, width);
    if (a.residual) {
        const Raw *const r = static_cast<const Raw *>(a.residual) + row * a.rs;
        uint4 add[GROUPS];
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) add[i] = load_group<T>(r, lane + i * lanes, width);
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            float u[G], v[G];
            T::unpack(trim_group<T>(h[i], lane + i * lanes, width), u);
            T::unpack(trim_group<T>(add[i], lane + i * lanes, width), v);
#pragma unroll
            for (int e = 0; e < G; ++e) u[e] += v[e];
            h[i] = T::pack(u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) h[i] = trim_group<T>(h[i], lane + i * lanes, width);
    }
    double square = 0.0;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
        float u[G];
        T::unpack(h[i], u);
#pragma unroll
        for (int e = 0; e < G; ++e) square = fma(double(u[e]), double(u[e]), square);
    }
    if (a.sum) {
        Raw *const s = static_cast<Raw *>(a.sum) + row * a.ss;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) store_group<T>(s, lane + i * lanes, width, h[i]);
    }
    const double rstd = 1.0 / sqrt(team.sum(square, room) / double(width) + double(a.epsilon));
    if (a.rstd && lane == 0) a.rstd[row] = float(rstd);
    if constexpr (CODES) {
        constexpr int SHARE = 32 / G;  // lanes of a scale
        uint8_t *const codes = a.codes + row * a.os, *const scales = a.scales + row * a.scs;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            const int g = lane + i * lanes, at = g * G;
            float u[G], w[G];
            T::unpack(h[i], u);
            if (weight) {
                T::unpack(trim_group<T>(load_group<T>(weight, g, width), g, width), w);
            } else {
#pragma unroll
                for (int e = 0; e < G; ++e) w[e] = 1.0f;
            }
            uint32_t c[G / 4];
            int n;
            encode_group<std::conditional_t<std::is_same<T, F16>::value, float, double>>(u, w, rstd, c, n);
            if (at + G <= width) {
#pragma unroll
                for (int e = 0; e < G; e += 4) *reinterpret_cast<u32_any *>(codes + at + e) = c[e / 4];
            } else {
#pragma unroll
                for (int e = 0; e < G; ++e)
                    if (at + e < width) codes[at + e] = uint8_t(c[e / 4] >> (8 * (e % 4)));
            }
            if (lane % SHARE == 0 && at < width) scales[at / 32] = uint8_t(n + 127);
        }
    } else {
        // Rows of more than 1e30 have a rstd that FP32 holds with fewer bits: both factors are moved.
        const float pre = rstd < 0x1p-100 ? 0x1p-64f : 1.0f, by = float(rstd / double(pre));
        Raw *const out = static_cast<Raw *>(a.out) + row * a.os;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            const int g = lane + i * lanes;
            float u[G];
            T::unpack(h[i], u);
#pragma unroll
            for (int e = 0; e < G; ++e) u[e] = u[e] * pre * by;
            if (weight) {
                float w[G];
                T::unpack(trim_group<T>(load_group<T>(weight, g, width), g, width), w);
#pragma unroll
                for (int e = 0; e < G; ++e) u[e] *= w[e];
            }
            store_group<T>(out, g, width, T::pack(u));
        }
    }
}

// A row's part of a gradient in a team's registers, trimmed.
template <class T, int GROUPS>
struct Gradient {
    static constexpr int G = T::kGroup;
    uint4 h[GROUPS], d[GROUPS], s[GROUPS];
    float rstd;

    __device__ __forceinline__ void load(const NormBackwardArgs &a, size_t row, int lane, int lanes) {
        using Raw = typename T::Raw;
        const Raw *const x = static_cast<const Raw *>(a.x) + row * a.xs, *const dy = static_cast<const Raw *>(a.d_out) + row * a.dos,
                        *const ds = static_cast<const Raw *>(a.d_sum) + row * a.dss;
        rstd = a.rstd[row];
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            h[i] = load_group<T>(x, lane + i * lanes, a.width);
            d[i] = load_group<T>(dy, lane + i * lanes, a.width);
            if (a.d_sum) s[i] = load_group<T>(ds, lane + i * lanes, a.width);
        }
    }
    __device__ __forceinline__ void trim(const NormBackwardArgs &a, int lane, int lanes) {
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            h[i] = trim_group<T>(h[i], lane + i * lanes, a.width);
            d[i] = trim_group<T>(d[i], lane + i * lanes, a.width);
            if (a.d_sum) s[i] = trim_group<T>(s[i], lane + i * lanes, a.width);
        }
    }
    // A rstd of rows over 1e30 is moved into FP32's range: hat = h * pre * by.
    __device__ __forceinline__ float pre() const { return rstd < 0x1p-100f ? 0x1p-64f : 1.0f; }
    // This lane's sum of g hat; each(i, e, dy, hat) on the way.
    template <class F>
    __device__ __forceinline__ double dot(bool weight, const uint4 (&w)[GROUPS], F &&each) const {
        const float before = pre(), by = rstd / before;
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            float u[G], v[G], k[G], part = 0.0f;
            T::unpack(h[i], u);
            T::unpack(d[i], v);
            if (weight) T::unpack(w[i], k);
#pragma unroll
            for (int e = 0; e < G; ++e) {
                const float hat = u[e] * before * by;
                each(i, e, v[e], hat);
                part = fmaf(weight ? v[e] * k[e] : v[e], hat, part);
            }
            sum += double(part);
        }
        return sum;
    }
    __device__ __forceinline__ void store(const NormBackwardArgs &a, size_t row, int lane, int lanes, float mean,
                                          const uint4 (&w)[GROUPS]) const {
        const float before = pre(), by = rstd / before;
        typename T::Raw *const dx = static_cast<typename T::Raw *>(a.d_x) + row * a.dxs;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            float u[G], v[G], k[G];
            T::unpack(h[i], u);
            T::unpack(d[i], v);
            if (a.weight) T::unpack(w[i], k);
#pragma unroll
            for (int e = 0; e < G; ++e) u[e] = rstd * fmaf(-(u[e] * before * by), mean, a.weight ? v[e] * k[e] : v[e]);
            if (a.d_sum) {
                T::unpack(s[i], v);
#pragma unroll
                for (int e = 0; e < G; ++e) u[e] += v[e];
            }
            store_group<T>(dx, lane + i * lanes, a.width, T::pack(u));
        }
    }
};
template <class T, int GROUPS>
__device__ __forceinline__ void load_weight(const NormBackwardArgs &a, int lane, int lanes, uint4 (&w)[GROUPS]) {
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
        const int g = lane + i * lanes;
        if (a.weight) w[i] = trim_group<T>(load_group<T>(static_cast<const typename T::Raw *>(a.weight), g, a.width), g, a.width);
    }
}

// Rows of the weight's gradient that are summed in FP32; such sums are added up in FP64.
constexpr int kRun = 64;

// Both gradients in one pass.  A team has every teams-th row, and its lanes the same
// channels of each: the sums of the weight's gradient and the weight stay in registers,
// and the next row's loads are under way while a row's mean is joined.  The sums of kRun
// rows go to LDS, a place a thread and channel.
// 8192 x 4096 BF16 with a residual: 51 us (5.3 TB/s); a wave a row, without loads ahead, 114.
template <class T, int LANES, int GROUPS>
__global__ void __launch_bounds__(kThreads<LANES>) norm_backward_kernel(NormBackwardArgs a, uint32_t teams) {
    constexpr int G = T::kGroup;
    __shared__ double room[kWavesMost];
    constexpr int TEAMS = LANES > 0 ? kBlock / (LANES > 0 ? LANES : 1) : 1;
    __shared__ double runs[GROUPS * G * kThreads<LANES>];
    const Team<LANES> team;
    const int lane = team.lane, lanes = team.lanes, width = a.width;
    const double share = 1.0 / double(width);
    uint4 w[GROUPS];
    load_weight<T>(a, lane, lanes, w);
    float dw[GROUPS][G];
#pragma unroll
    for (int i = 0; i < GROUPS; ++i)
#pragma unroll
        for (int e = 0; e < G; ++e) dw[i][e] = 0.0f;
    // Channel i, e of this thread.  Teams of a wave are next to each other, so that its lanes meet no bank twice.
    const auto place = [&](int i, int e) { return (i * G + e) * kThreads<LANES> + int(threadIdx.x); };
    bool any = false;
    const auto add_run = [&] {
#pragma unroll
        for (int i = 0; i < GROUPS; ++i)
#pragma unroll
            for (int e = 0; e < G; ++e) {
                runs[place(i, e)] = (any ? runs[place(i, e)] : 0.0) + double(dw[i][e]);
                dw[i][e] = 0.0f;
            }
        any = true;
    };
    size_t row = size_t(blockIdx.x) * TEAMS + team.of;
    Gradient<T, GROUPS> now, next;
    if (row < a.rows) now.load(a, row, lane, lanes);
    for (int run = 0; row < a.rows; row += teams) {
        if (row + teams < a.rows) next.load(a, row + teams, lane, lanes);
        now.trim(a, lane, lanes);
        const double dot = now.dot(a.weight, w, [&](int i, int e, float dy, float hat) { dw[i][e] = fmaf(dy, hat, dw[i][e]); });
        now.store(a, row, lane, lanes, float(team.sum(dot, room) * share), w);
        now = next;
        if (++run == kRun) {
            add_run();
            run = 0;
        }
    }
    float *const part = a.part + size_t(blockIdx.x) * width;
    if constexpr (LANES > 0) {  // the teams' sums, one after the other
        add_run();
        __syncthreads();
        for (int c = threadIdx.x; c < LANES * GROUPS * G; c += kBlock) {
            const double *const own = runs + c / LANES * kBlock + c % LANES;
            double sum = own[0];
#pragma unroll
            for (int t = 1; t < TEAMS; ++t) sum += own[t * LANES];
            const int at = (c % LANES + c / (LANES * G) * LANES) * G + c / LANES % G;
            if (at < width) part[at] = float(sum);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < GROUPS; ++i)
#pragma unroll
        for (int e = 0; e < G; ++e) {
            const int at = (lane + i * lanes) * G + e;
            if (at < width) part[at] = any ? float(runs[place(i, e)] + double(dw[i][e])) : dw[i][e];
        }
}

// The weight's gradient alone, of SLAB groups of channels: a workgroup sums over every
// parts-th of its rows, U at a time a thread, in a fixed order.
template <class T, int SLAB, int U>
__device__ __forceinline__ void sum_columns(const NormBackwardArgs &a, int slab, size_t part, size_t parts, float *out, float *room) {
    using Raw = typename T::Raw;
    constexpr int G = T::kGroup;
    const int c = threadIdx.x % SLAB, of = threadIdx.x / SLAB, rows = blockDim.x / SLAB, g = slab * SLAB + c, width = a.width;
    float sum[G];
#pragma unroll
    for (int e = 0; e < G; ++e) sum[e] = 0.0f;
    if (g * G < width) {
        const size_t step = parts * rows;
        for (size_t first = part * rows + of; first < a.rows; first += U * step) {
            uint4 h[U], d[U];
            float rstd[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const size_t row = first + u * step, in = row < a.rows ? row : first;
                h[u] = load_group<T>(static_cast<const Raw *>(a.x) + in * a.xs, g, width);
                d[u] = load_group<T>(static_cast<const Raw *>(a.d_out) + in * a.dos, g, width);
                rstd[u] = a.rstd[in];
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (first + u * step >= a.rows) continue;
                const float pre = rstd[u] < 0x1p-100f ? 0x1p-64f : 1.0f, by = rstd[u] / pre;
                float x[G], dy[G];
                T::unpack(trim_group<T>(h[u], g, width), x);
                T::unpack(trim_group<T>(d[u], g, width), dy);
#pragma unroll
                for (int e = 0; e < G; ++e) sum[e] = fmaf(dy[e], x[e] * pre * by, sum[e]);
            }
        }
    }
#pragma unroll
    for (int e = 0; e < G; ++e) room[of * SLAB * G + c * G + e] = sum[e];
    __syncthreads();
    for (int i = threadIdx.x; i < SLAB * G; i += blockDim.x) {
        const int at = slab * SLAB * G + i;
        if (at >= width) break;
        double all = 0.0;
#pragma unroll 8
        for (int r = 0; r < rows; ++r) all += double(room[r * SLAB * G + i]);
        out[at] = float(all);
    }
}
constexpr int kSlab = 64, kNarrow = 2;  // groups of channels of a workgroup: of many rows, of few
template <class T>
__global__ void __launch_bounds__(kBlock) norm_columns_kernel(NormBackwardArgs a, uint32_t slabs, uint32_t parts) {
    __shared__ float room[kBlock * T::kGroup];
    const uint32_t part = blockIdx.x / slabs;
    sum_columns<T, kSlab, 4>(a, int(blockIdx.x - part * slabs), part, parts, a.part + size_t(part) * a.width, room);
}

// The rows' gradient alone, a row a team, in the first workgroups; in the others (few
// rows) the weight's, which needs no row's mean.
template <class T, int LANES, int GROUPS>
__global__ void __launch_bounds__(kThreads<LANES>) norm_rows_kernel(NormBackwardArgs a, uint32_t row_blocks) {
    constexpr int TEAMS = LANES > 0 ? kBlock / (LANES > 0 ? LANES : 1) : 1;
    __shared__ union {
        double sums[kWavesMost];
        float columns[LANES == kWideRow ? 1 : kThreads<LANES> * T::kGroup];
    } room;
    if (blockIdx.x >= row_blocks) {
        if constexpr (LANES != kWideRow) sum_columns<T, kNarrow, 8>(a, int(blockIdx.x - row_blocks), 0, 1, a.d_weight, room.columns);
        return;
    }
    const Team<LANES> team;
    const int lane = team.lane, lanes = team.lanes;
    const size_t row = size_t(blockIdx.x) * TEAMS + team.of;
    if (row >= a.rows) return;  // whole teams, whose sums are their own
    Gradient<T, GROUPS> now;
    uint4 w[GROUPS];
    now.load(a, row, lane, lanes);
    load_weight<T>(a, lane, lanes, w);
    now.trim(a, lane, lanes);
    const double dot = now.dot(a.weight, w, [](int, int, float, float) {});
    now.store(a, row, lane, lanes, float(team.sum(dot, room.sums) / double(a.width)), w);
}

// Sums 32 channels over the parts, 32 threads each.
__global__ void __launch_bounds__(1024) norm_join_kernel(const float *part, uint32_t parts, int width, float *out) {
    __shared__ double room[32][33];
    const int channel = threadIdx.x % 32, share = threadIdx.x / 32, at = int(blockIdx.x) * 32 + channel;
    double sum = 0.0;
    if (at < width) {
#pragma unroll 8
        for (uint32_t p = share; p < parts; p += 32) sum += double(part[size_t(p) * width + at]);
    }
    room[share][channel] = sum;
    __syncthreads();
    if (share) return;
    if (at >= width) return;
#pragma unroll 8
    for (int w = 1; w < 32; ++w) sum += room[w][channel];
    out[at] = float(sum);
}

// How a row is cut: the lanes of a team (or kBlockRow, kWideRow), 16-byte groups of a
// lane, threads of the workgroup.
struct Cut {
    int lanes, groups, threads;
    int teams() const { return lanes > 0 ? kBlock / lanes : 1; }
};
Cut cut_of(size_t width, int group) {
    const size_t n = (width + group - 1) / group;
    for (int lanes : {16, 32, 64})
        if (n <= size_t(lanes)) return {lanes, 1, kBlock};
    if (n <= 128) return {64, 2, kBlock};
    const auto of = [&](int lanes, int groups) { return Cut{lanes, groups, 64 * int((n + 64 * groups - 1) / (64 * groups))}; };
    return n <= 1024 ? of(kBlockRow, 2) : n <= 2048 ? of(kWideRow, 2) : of(kWideRow, 4);
}

// f(LANES, GROUPS) for a row's width.
template <class T, class F>
void for_cut(const Cut &c, F &&f) {
    using std::integral_constant;
    using One = integral_constant<int, 1>;
    using Two = integral_constant<int, 2>;
    switch (c.lanes) {
        case 16: return f(integral_constant<int, 16>(), One());
        case 32: return f(integral_constant<int, 32>(), One());
        case 64: return c.groups == 1 ? f(integral_constant<int, 64>(), One()) : f(integral_constant<int, 64>(), Two());
        case kBlockRow: return f(integral_constant<int, kBlockRow>(), Two());
    }
    if (c.groups == 2) return f(integral_constant<int, kWideRow>(), Two());
    if constexpr (T::kGroup == 4) f(integral_constant<int, kWideRow>(), integral_constant<int, 4>());  // 16-bit rows end before
}

template <class T>
void norm_of(const NormArgs &a, hipStream_t stream) {
    const Cut c = cut_of(size_t(a.width), T::kGroup);
    const dim3 grid(unsigned((a.rows + c.teams() - 1) / c.teams()));
    for_cut<T>(c, [&](auto lanes, auto groups) {
        if (a.codes)
            norm_kernel<T, lanes.value, groups.value, true><<<grid, c.threads, 0, stream>>>(a);
        else
            norm_kernel<T, lanes.value, groups.value, false><<<grid, c.threads, 0, stream>>>(a);
    });
}

uint32_t parts_of(size_t rows, const Cut &c) {
    return uint32_t(std::min<size_t>((rows + c.teams() - 1) / c.teams(), 512));
}
// Of wide rows, for workgroups of norm_columns_kernel: eight a CU, and more where a thread
// would have more than kRun rows.
uint32_t wide_parts_of(size_t rows, size_t width, int group) {
    const size_t slabs = (width + group * kSlab - 1) / (group * kSlab), run = size_t(kBlock / kSlab) * kRun;
    return uint32_t(std::max(std::min(rows, std::min<size_t>(512, std::max<size_t>(1, 2048 / slabs))), (rows + run - 1) / run));
}
// Calls of few rows and elements take one launch, in which some workgroups read the rows
// again for the weight's gradient: 1024 x 128 F32 took launches of 4.0 and 2.5 us, and takes
// one of 6.1, and no workspace.
bool few(size_t rows, size_t width) { return rows <= 1024 && rows * width <= size_t(1) << 18; }

template <class T>
void backward_of(const NormBackwardArgs &a, hipStream_t stream) {
    const Cut c = cut_of(size_t(a.width), T::kGroup);
    const uint32_t row_blocks = uint32_t((a.rows + c.teams() - 1) / c.teams());
    const bool small = few(a.rows, size_t(a.width)) && c.lanes != kWideRow;
    uint32_t parts = parts_of(a.rows, c);
    for_cut<T>(c, [&](auto lanes, auto groups) {
        const auto rows = [&](uint32_t first, uint32_t others) {
            if (first + others) norm_rows_kernel<T, lanes.value, groups.value><<<dim3(first + others), c.threads, 0, stream>>>(a, first);
        };
        if (!a.d_weight) return rows(row_blocks, 0);
        const int width = a.width, group = T::kGroup;
        if (small) {
            const uint32_t slabs = uint32_t((width + group * kNarrow - 1) / (group * kNarrow));
            // What the rows' gradient replaces has to be read before.
            const bool apart = a.d_x == a.x || a.d_x == a.d_out;
            rows(apart ? 0 : row_blocks, slabs);
            if (apart) rows(row_blocks, 0);
            return;
        }
        if constexpr (lanes.value == kWideRow) {
            // Registers do not hold the sums beside a row: 4000 x 15001 BF16 took 268 us so, and
            // takes 173 with the rows read twice.  LDS would hold them, and has not been measured.
            const uint32_t slabs = uint32_t((width + group * kSlab - 1) / (group * kSlab));
            parts = wide_parts_of(a.rows, size_t(width), group);
            if (parts) norm_columns_kernel<T><<<dim3(slabs * parts), kBlock, 0, stream>>>(a, slabs, parts);
        } else if (parts) {
            norm_backward_kernel<T, lanes.value, groups.value><<<dim3(parts), c.threads, 0, stream>>>(a, parts * uint32_t(c.teams()));
        }
        norm_join_kernel<<<dim3(unsigned((width + 31) / 32)), 1024, 0, stream>>>(a.part, parts, width, a.d_weight);
        if constexpr (lanes.value == kWideRow) rows(row_blocks, 0);
    });
}

}  // namespace

size_t norm_parts(size_t rows, size_t width) {
    size_t parts = 0;
    for (int group : {4, 8}) {
        const Cut c = cut_of(width, group);
        if (c.lanes == kWideRow)
            parts = std::max<size_t>(parts, wide_parts_of(rows, width, group));
        else if (!few(rows, width))
            parts = std::max<size_t>(parts, parts_of(rows, c));
    }
    return parts;
}

void rms_norm(const NormArgs &a, Type type, hipStream_t stream) {
    switch (type) {
        case Type::F32: return norm_of<F32>(a, stream);
        case Type::F16: return norm_of<F16>(a, stream);
        case Type::BF16: return norm_of<BF16>(a, stream);
    }
}

void rms_norm_backward(const NormBackwardArgs &a, Type type, hipStream_t stream) {
    switch (type) {
        case Type::F32: return backward_of<F32>(a, stream);
        case Type::F16: return backward_of<F16>(a, stream);
        case Type::BF16: return backward_of<BF16>(a, stream);
    }
}

}  // namespace meshgpt::kern
