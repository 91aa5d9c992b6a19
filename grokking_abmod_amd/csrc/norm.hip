// The root-mean-square norm with the residual's addition, with an output in the
// rows' type or in 8 bits, and its gradient.
//
//   h = x + residual, rounded to the type and kept;
//   rstd = 1 / sqrt(mean(h^2) + epsilon);  y = h rstd w.
// In 8 bits a scale 2^(b - 127) belongs to 32 channels: the smallest power of two
// with which the largest of them is at most 448.
//   g = dy w;  dh = rstd (g - hat mean(g hat)) + dsum;  dw = sum of dy hat over rows, hat = h rstd.
//
// All of them read a row once: it stays in registers, 16 bytes a load, in one
// wave for short rows and in 4 or 16 for longer ones.  Sums of a row are FP64,
// which no FP32 value overflows; so is what decides a scale, where values next to
// a power of two are met in any large batch.  The weight's gradient is summed in
// registers over a team's rows, then over the teams in a fixed order.
#include "dpp.hpp"
#include "operators.hpp"
#include "types.hpp"

namespace meshgpt::kern {
namespace {

// Group g of a row, zero behind its end.
template <class T>
__device__ __forceinline__ uint4 load_group(const typename T::Raw *row, int g, int width) {
    constexpr int G = T::kGroup;
    const int at = g * G;
    if (at + G <= width) return get_any(row + at);
    float x[G];
#pragma unroll
    for (int e = 0; e < G; ++e) x[e] = at + e < width ? T::to_float(row[at + e]) : 0.0f;
    return T::pack(x);
}
template <class T>
__device__ __forceinline__ void store_group(typename T::Raw *row, int g, int width, uint4 w) {
    constexpr int G = T::kGroup;
    const int at = g * G;
    if (at + G <= width) return put_any(row + at, w);
    float x[G];
    T::unpack(w, x);
#pragma unroll
    for (int e = 0; e < G; ++e)
        if (at + e < width) row[at + e] = T::from_float(x[e]);
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int d = 32; d > 0; d /= 2) v += __shfl_xor(v, d, 64);
    return v;
}

// The sum of a team's values, in all of its lanes.
template <int WAVES>
__device__ __forceinline__ double team_sum(double v, double *room) {
    v = wave_sum64(v);
    if constexpr (WAVES > 1) {
        const int wave = threadIdx.x / 64;
        __syncthreads();  // of the row before
        if (threadIdx.x % 64 == 0) room[wave] = v;
        __syncthreads();
        v = 0.0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v += room[w];
    }
    return v;
}

template <int WAVES>
constexpr int kTeams = WAVES == 1 ? 4 : 1;  // of a workgroup
template <int WAVES>
constexpr int kThreads = 64 * WAVES * kTeams<WAVES>;

typedef uint32_t u32_any __attribute__((aligned(1)));

// Four E4M3 codes.
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}

template <class T, int WAVES, int GROUPS, bool CODES>
__global__ void __launch_bounds__(kThreads<WAVES>) norm_kernel(NormArgs a) {
    using Raw = typename T::Raw;
    constexpr int G = T::kGroup, LANES = 64 * WAVES;
    __shared__ double room[WAVES];
    const int lane = threadIdx.x % LANES, width = a.width;
    const size_t row = size_t(blockIdx.x) * kTeams<WAVES> + threadIdx.x / LANES;
    if (row >= a.rows) return;  // of one wave a row, or all of the workgroup
    const Raw *const x = static_cast<const Raw *>(a.x) + row * a.xs;
    const Raw *const weight = static_cast<const Raw *>(a.weight);
    uint4 h[GROUPS];
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) h[i] = load_group<T>(x, lane + i * LANES, width);
    if (a.residual) {
        const Raw *const r = static_cast<const Raw *>(a.residual) + row * a.rs;
        uint4 add[GROUPS];
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) add[i] = load_group<T>(r, lane + i * LANES, width);
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            float u[G], v[G];
            T::unpack(h[i], u);
            T::unpack(add[i], v);
#pragma unroll
            for (int e = 0; e < G; ++e) u[e] += v[e];
            h[i] = T::pack(u);
        }
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
        for (int i = 0; i < GROUPS; ++i) store_group<T>(s, lane + i * LANES, width, h[i]);
    }
    const double rstd = 1.0 / sqrt(team_sum<WAVES>(square, room) / double(width) + double(a.epsilon));
    if (a.rstd && lane == 0) a.rstd[row] = float(rstd);
    if constexpr (CODES) {
        constexpr int SHARE = 32 / G;  // lanes of a scale
        uint8_t *const codes = a.codes + row * a.os, *const scales = a.scales + row * a.scs;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            const int g = lane + i * LANES, at = g * G;
            float u[G], w[G];
            T::unpack(h[i], u);
            if (weight) {
                T::unpack(load_group<T>(weight, g, width), w);
            } else {
#pragma unroll
                for (int e = 0; e < G; ++e) w[e] = 1.0f;
            }
            double y[G], top = 0.0;
#pragma unroll
            for (int e = 0; e < G; ++e) {
                y[e] = double(u[e]) * double(w[e]);
                top = fmax(top, fabs(y[e]));
            }
#pragma unroll
            for (int d = 1; d < SHARE; d *= 2) top = fmax(top, __shfl_xor(top, d, 64));
            top *= rstd;
            // top = m 2^n, 1 <= m < 2; 448 = 1.75 * 2^8.
            const uint64_t bits = __builtin_bit_cast(uint64_t, top);
            int n = int(bits >> 52) - 1023 - 8 + ((bits & 0xfffffffffffffull) > 0xc000000000000ull);
            n = min(max(n, -117), 120);
            const double by = rstd * __builtin_bit_cast(double, uint64_t(1023 - n) << 52);
            uint32_t c[G / 4];
#pragma unroll
            for (int e = 0; e < G; e += 4)
                c[e / 4] = encode4(float(y[e] * by), float(y[e + 1] * by), float(y[e + 2] * by), float(y[e + 3] * by));
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
            const int g = lane + i * LANES;
            float u[G];
            T::unpack(h[i], u);
#pragma unroll
            for (int e = 0; e < G; ++e) u[e] = u[e] * pre * by;
            if (weight) {
                float w[G];
                T::unpack(load_group<T>(weight, g, width), w);
#pragma unroll
                for (int e = 0; e < G; ++e) u[e] *= w[e];
            }
            store_group<T>(out, g, width, T::pack(u));
        }
    }
}

template <class T, int WAVES, int GROUPS>
__global__ void __launch_bounds__(kThreads<WAVES>) norm_backward_kernel(NormBackwardArgs a, uint32_t teams) {
    using Raw = typename T::Raw;
    constexpr int G = T::kGroup, LANES = 64 * WAVES;
    __shared__ double room[WAVES];
    __shared__ float joined[WAVES == 1 ? LANES * GROUPS * G : 1];
    const int lane = threadIdx.x % LANES, width = a.width;
    const int team = threadIdx.x / LANES;
    const Raw *const weight = static_cast<const Raw *>(a.weight);
    float dw[GROUPS][G];
#pragma unroll
    for (int i = 0; i < GROUPS; ++i)
#pragma unroll
        for (int e = 0; e < G; ++e) dw[i][e] = 0.0f;
    for (size_t row = size_t(blockIdx.x) * kTeams<WAVES> + team; row < a.rows; row += teams) {
        const Raw *const x = static_cast<const Raw *>(a.x) + row * a.xs, *const dy = static_cast<const Raw *>(a.d_out) + row * a.dos;
        uint4 h[GROUPS], d[GROUPS];
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            h[i] = load_group<T>(x, lane + i * LANES, width);
            d[i] = load_group<T>(dy, lane + i * LANES, width);
        }
        const float rstd = a.rstd[row];
        const float pre = rstd < 0x1p-100f ? 0x1p-64f : 1.0f, by = rstd / pre;
        double dot = 0.0;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            float u[G], v[G], w[G];
            T::unpack(h[i], u);
            T::unpack(d[i], v);
            if (weight) T::unpack(load_group<T>(weight, lane + i * LANES, width), w);
            float part = 0.0f;
#pragma unroll
            for (int e = 0; e < G; ++e) {
                const float hat = u[e] * pre * by;
                dw[i][e] = fmaf(v[e], hat, dw[i][e]);
                part = fmaf(weight ? v[e] * w[e] : v[e], hat, part);
            }
            dot += double(part);
        }
        const float mean = float(team_sum<WAVES>(dot, room) / double(width));
        Raw *const dx = static_cast<Raw *>(a.d_x) + row * a.dxs;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            const int g = lane + i * LANES;
            float u[G], v[G], w[G];
            T::unpack(h[i], u);
            T::unpack(d[i], v);
            if (weight) T::unpack(load_group<T>(weight, g, width), w);
#pragma unroll
            for (int e = 0; e < G; ++e) u[e] = rstd * fmaf(-(u[e] * pre * by), mean, weight ? v[e] * w[e] : v[e]);
            if (a.d_sum) {
                T::unpack(load_group<T>(static_cast<const Raw *>(a.d_sum) + row * a.dss, g, width), v);
#pragma unroll
                for (int e = 0; e < G; ++e) u[e] += v[e];
            }
            store_group<T>(dx, g, width, T::pack(u));
        }
    }
    if (!a.part) return;
    float *const part = a.part + size_t(blockIdx.x) * width;
    if constexpr (WAVES == 1) {  // the waves one after the other, in one order
        for (int t = 0; t < kTeams<WAVES>; ++t) {
            if (team == t) {
#pragma unroll
                for (int i = 0; i < GROUPS; ++i)
#pragma unroll
                    for (int e = 0; e < G; ++e) {
                        float &at = joined[(i * G + e) * LANES + lane];
                        if (t) dw[i][e] += at;
                        at = dw[i][e];
                    }
            }
            __syncthreads();
        }
        if (team != kTeams<WAVES> - 1) return;
    }
#pragma unroll
    for (int i = 0; i < GROUPS; ++i)
#pragma unroll
        for (int e = 0; e < G; ++e) {
            const int at = (lane + i * LANES) * G + e;
            if (at < width) part[at] = dw[i][e];
        }
}

// Sums 64 channels over the parts.
constexpr int kJoin = 1024;
__global__ void __launch_bounds__(kJoin) norm_join_kernel(const float *part, uint32_t parts, int width, float *out) {
    __shared__ double room[kJoin / 64][64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, at = int(blockIdx.x) * 64 + lane;
    double sum = 0.0;
    if (at < width)
        for (uint32_t p = wave; p < parts; p += kJoin / 64) sum += double(part[size_t(p) * width + at]);
    room[wave][lane] = sum;
    __syncthreads();
    if (wave || at >= width) return;
    for (int w = 1; w < kJoin / 64; ++w) sum += room[w][lane];
    out[at] = float(sum);
}

// Waves and 16-byte groups of a lane that a row takes.
struct Cut {
    int waves, groups;
};
Cut cut_of(size_t width, int group) {
    const size_t groups = (width + group - 1) / group;
    for (int waves : {1, 4, 16})
        for (int n : {1, 2, 4, 8})
            if (groups <= size_t(64 * waves * n)) return {waves, n};
    return {0, 0};
}

template <class T, int WAVES, int GROUPS>
void launch_norm(const NormArgs &a, hipStream_t stream) {
    const dim3 grid(unsigned((a.rows + kTeams<WAVES> - 1) / kTeams<WAVES>));
    if (a.codes)
        norm_kernel<T, WAVES, GROUPS, true><<<grid, kThreads<WAVES>, 0, stream>>>(a);
    else
        norm_kernel<T, WAVES, GROUPS, false><<<grid, kThreads<WAVES>, 0, stream>>>(a);
}

uint32_t parts_of(size_t rows, int waves) {
    const size_t teams = waves == 1 ? 4 : 1;
    return uint32_t(std::min<size_t>((rows + teams - 1) / teams, 512));
}

template <class T, int WAVES, int GROUPS>
void launch_backward(const NormBackwardArgs &a, hipStream_t stream) {
    const uint32_t parts = parts_of(a.rows, WAVES);
    if (parts)
        norm_backward_kernel<T, WAVES, GROUPS><<<dim3(parts), kThreads<WAVES>, 0, stream>>>(a, parts * kTeams<WAVES>);
    if (a.d_weight)
        norm_join_kernel<<<dim3(unsigned((a.width + 63) / 64)), kJoin, 0, stream>>>(a.part, parts, a.width, a.d_weight);
}

// f(WAVES, GROUPS) for a row's width.
template <class T, class F>
void for_cut(size_t width, F &&f) {
    const Cut c = cut_of(width, T::kGroup);
    const auto groups = [&](auto waves) {
        switch (c.groups) {
            case 1: return f(waves, std::integral_constant<int, 1>());
            case 2: return f(waves, std::integral_constant<int, 2>());
            case 4: return f(waves, std::integral_constant<int, 4>());
            default: return f(waves, std::integral_constant<int, 8>());
        }
    };
    switch (c.waves) {
        case 1: return groups(std::integral_constant<int, 1>());
        case 4: return groups(std::integral_constant<int, 4>());
        default: return groups(std::integral_constant<int, 16>());
    }
}

template <class T>
void norm_of(const NormArgs &a, hipStream_t stream) {
    for_cut<T>(size_t(a.width), [&](auto w, auto g) { launch_norm<T, w.value, g.value>(a, stream); });
}
template <class T>
void backward_of(const NormBackwardArgs &a, hipStream_t stream) {
    for_cut<T>(size_t(a.width), [&](auto w, auto g) { launch_backward<T, w.value, g.value>(a, stream); });
}

}  // namespace

size_t norm_parts(size_t rows, size_t width) {
    return std::max(parts_of(rows, cut_of(width, 4).waves), parts_of(rows, cut_of(width, 8).waves));
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
