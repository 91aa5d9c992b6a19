// The 8-bit KV cache: quantising keys and values as they are written, and
// reading them back.
//
// Sixteen tokens of a head share a scale 2^e, the smallest with
// max|x| <= 448 * 2^e (448 is E4M3's largest value), held as the byte e + 127.
// A power of two loses nothing to a scale of more bits, because the codes are
// floating point: x / 2^e is exact, and one rounding to E4M3's 4 significant
// bits is the only error (half a step, 2^-4 of the value, and 2^-10 * 2^e where
// the code is subnormal).  It also makes a block's rescaling exact where later
// tokens need a larger scale: the older codes move down by whole exponents and
// round again only where they become subnormal.
//
// Both directions move bytes: one wave takes 16 tokens of a head, of its keys
// or of its values.  Keys are stored as they come; a lane takes 16 channels of
// a token.  Values are stored transposed, 64 tokens of a channel in a row, the
// order in which the attention's matrix product reads them; a lane takes a
// channel of the 16 tokens.
#include <hip/hip_runtime.h>

#include <cfloat>

#include "operators.hpp"
#include "types.hpp"

namespace meshgpt::kern {
namespace {

// Scales from 2^-117 (a code is at least 2^-9, so every value is a normal f32)
// to 2^120, where codes end at 240: 256 * 2^120 is no f32.
constexpr int kLowScale = 10, kHighScale = 247;

__device__ __forceinline__ int scale_byte(float largest) {
    const uint32_t b = __builtin_bit_cast(uint32_t, largest);
    const int e = int(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(e, kLowScale), kHighScale);
}

__device__ __forceinline__ float power(int byte) { return __builtin_bit_cast(float, uint32_t(byte) << 23); }

// x / 2^(byte - 127) in E4M3's range; what is not finite becomes NaN.
__device__ __forceinline__ float in_range(float x, float inverse, float limit) {
    const float y = fminf(fmaxf(x * inverse, -limit), limit);
    return fabsf(x) <= FLT_MAX ? y : __builtin_nanf("");
}

__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    return uint32_t(w);
}

__device__ __forceinline__ void decode4(uint32_t w, float (&x)[4]) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), true);
    x[0] = lo[0];
    x[1] = lo[1];
    x[2] = hi[0];
    x[3] = hi[1];
}

// Codes times 2^-drop.
__device__ __forceinline__ uint32_t lowered4(uint32_t w, int drop) {
    float x[4];
    decode4(w, x);
    const float f = power(127 - min(drop, 126));
    return encode4(x[0] * f, x[1] * f, x[2] * f, x[3] * f);
}

__device__ __forceinline__ float wave_largest(float v) {
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) v = fmaxf(v, __shfl_xor(v, k, 64));
    return v;
}

// N consecutive elements from p, those at or past `have` as 0.
template <class T, int N>
__device__ __forceinline__ void load_run(const typename T::Raw *p, int have, bool aligned, float (&x)[N]) {
    if (aligned && have >= N) {
#pragma unroll
        for (int i = 0; i < N / T::kGroup; ++i) {
            float g[T::kGroup];
            T::unpack(reinterpret_cast<const uint4 *>(p)[i], g);
#pragma unroll
            for (int j = 0; j < T::kGroup; ++j) x[i * T::kGroup + j] = g[j];
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = i < have ? T::to_float(p[i]) : 0.0f;
}

template <class T, int N>
__device__ __forceinline__ void store_run(typename T::Raw *p, int have, bool aligned, const float (&x)[N]) {
    if (aligned && have >= N) {
#pragma unroll
        for (int i = 0; i < N / T::kGroup; ++i) {
            float g[T::kGroup];
#pragma unroll
            for (int j = 0; j < T::kGroup; ++j) g[j] = x[i * T::kGroup + j];
            reinterpret_cast<uint4 *>(p)[i] = T::pack(g);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (i < have) p[i] = T::from_float(x[i]);
}

template <int N>
__device__ __forceinline__ float finite_largest(const float (&x)[N], float top) {
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, fabsf(x[i]) <= FLT_MAX ? fabsf(x[i]) : 0.0f);
    return top;
}

// How a lane takes part: keys, `kRun` channels of one token, `kPasses` times 64
// channels on; values, `kSlots` tokens of one channel.
template <int PAD>
struct Share {
    static constexpr int kPasses = PAD >= 64 ? PAD / 64 : 1;
    static constexpr int kRun = PAD >= 64 ? 16 : PAD / 4;
    static constexpr int kSlots = PAD >= 64 ? 16 : 8;
};

// Positions [lo, hi) of the block's 16 are new; with lo past the block's first,
// the ones before it are older and keep their values.
template <class T, int PAD>
__device__ __forceinline__ void append_keys(const Kv8AppendArgs &a, int seq, int head, size_t pair, int block, int lo,
                                            int hi, int first) {
    using S = Share<PAD>;
    const int lane = threadIdx.x & 63, place = 16 * block + (lane >> 2);
    const bool fresh = place >= lo && place < hi, begun = lo > 16 * block;
    const auto *row = static_cast<const typename T::Raw *>(a.k) + seq * a.ks.s[0] + int64_t(place - first) * a.ks.s[1] +
                      head * a.ks.s[2];
    uint8_t *const scale = a.cache.ks + pair * (a.cache.capacity / 16) + block;
    const int was = begun ? *scale : 0;
    float x[S::kPasses][S::kRun], top = 0.0f;
#pragma unroll
    for (int p = 0; p < S::kPasses; ++p) {
        const int d = S::kRun * (lane & 3) + 64 * p;
        load_run<T>(row + d, fresh ? a.cache.width - d : 0, a.aligned, x[p]);
        top = finite_largest(x[p], top);
    }
    const int byte = min(max(scale_byte(wave_largest(top)), was), kHighScale);
    const float inverse = power(254 - byte), limit = byte == kHighScale ? 240.0f : 448.0f;
    const bool lower = begun && byte > was && place < lo;
    if (lane == 0) *scale = uint8_t(byte);
    if (!fresh && !lower) return;
    uint8_t *const out = a.cache.k + (pair * a.cache.capacity + place) * PAD;
#pragma unroll
    for (int p = 0; p < S::kPasses; ++p) {
        uint32_t *const w = reinterpret_cast<uint32_t *>(out + S::kRun * (lane & 3) + 64 * p);
        uint32_t c[S::kRun / 4];
        if (fresh) {
#pragma unroll
            for (int i = 0; i < S::kRun / 4; ++i) {
                float y[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = in_range(x[p][4 * i + j], inverse, limit);
                c[i] = encode4(y[0], y[1], y[2], y[3]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < S::kRun / 4; ++i) c[i] = lowered4(w[i], byte - was);
        }
        if constexpr (S::kRun == 16)
            *reinterpret_cast<uint4 *>(w) = uint4{c[0], c[1], c[2], c[3]};
        else
            *reinterpret_cast<uint2 *>(w) = uint2{c[0], c[1]};
    }
}

template <class T, int PAD>
__device__ __forceinline__ void append_values(const Kv8AppendArgs &a, int seq, int head, size_t pair, int block, int lo,
                                              int hi, int first) {
    using S = Share<PAD>;
    const int lane = threadIdx.x & 63, slot0 = PAD >= 64 ? 0 : 8 * (lane >> 5), place0 = 16 * block + slot0;
    const bool begun = lo > 16 * block;
    const auto *base = static_cast<const typename T::Raw *>(a.v) + seq * a.vs.s[0] + head * a.vs.s[2];
    uint8_t *const scale = a.cache.vs + pair * (a.cache.capacity / 16) + block;
    const int was = begun ? *scale : 0;
    float x[S::kPasses][S::kSlots], top = 0.0f;
#pragma unroll
    for (int p = 0; p < S::kPasses; ++p) {
        const int d = PAD >= 64 ? lane + 64 * p : lane & 31;
#pragma unroll
        for (int i = 0; i < S::kSlots; ++i) {
            const int place = place0 + i;
            x[p][i] = place >= lo && place < hi && d < a.cache.width
                          ? T::to_float(base[int64_t(place - first) * a.vs.s[1] + d])
                          : 0.0f;
        }
        top = finite_largest(x[p], top);
    }
    const int byte = min(max(scale_byte(wave_largest(top)), was), kHighScale);
    const float inverse = power(254 - byte), limit = byte == kHighScale ? 240.0f : 448.0f;
    if (lane == 0) *scale = uint8_t(byte);
    const bool whole = lo == 16 * block && hi == 16 * block + 16;
#pragma unroll
    for (int p = 0; p < S::kPasses; ++p) {
        const int d = PAD >= 64 ? lane + 64 * p : lane & 31;
        uint8_t *const out = a.cache.v + ((pair * (a.cache.capacity / 64) + block / 4) * PAD + d) * 64 +
                             16 * (block % 4) + slot0;
        uint32_t c[S::kSlots / 4];
#pragma unroll
        for (int i = 0; i < S::kSlots / 4; ++i) {
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = in_range(x[p][4 * i + j], inverse, limit);
            c[i] = encode4(y[0], y[1], y[2], y[3]);
        }
        if (!whole) {  // the bytes around the new ones: lowered where older, left where behind
            uint32_t *const w = reinterpret_cast<uint32_t *>(out);
            const bool lower = begun && byte > was;
#pragma unroll
            for (int i = 0; i < S::kSlots / 4; ++i) {
                const int at = place0 + 4 * i;
                if (at + 4 <= lo ? !lower : at >= hi) continue;  // nothing of these four changes
                const uint32_t old = w[i], low = lower ? lowered4(old, byte - was) : old;
                uint32_t now = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t m = 0xffu << (8 * j);
                    now |= m & (at + j < lo ? low : at + j < hi ? c[i] : old);
                }
                w[i] = now;
            }
            continue;
        }
        if constexpr (S::kSlots == 16)
            *reinterpret_cast<uint4 *>(out) = uint4{c[0], c[1], c[2], c[3]};
        else
            *reinterpret_cast<uint2 *>(out) = uint2{c[0], c[1]};
    }
}

// One wave for the keys or the values of 16 tokens of a head; waves of the
// touched blocks of every (sequence, head).
template <class T, int PAD>
__global__ void __launch_bounds__(256) kv8_append_kernel(Kv8AppendArgs a, int blocks, uint32_t units) {
    const uint32_t u = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (u >= units) return;
    const uint32_t rest = u >> 1, pair = rest / uint32_t(blocks);
    const int seq = int(pair) / a.cache.heads, head = int(pair) - seq * a.cache.heads;
    const int length = a.lengths[seq], count = a.counts ? a.counts[seq] : a.count;
    if (length < 0 || length > a.cache.capacity || count < 0 || count > a.count || count > length) return;
    const int start = length - count, block = start / 16 + int(rest - pair * uint32_t(blocks));
    const int lo = max(start, 16 * block), hi = min(length, 16 * block + 16);
    if (lo >= hi) return;
    const int first = a.absolute ? 0 : start;
    if (u & 1)
        append_values<T, PAD>(a, seq, head, pair, block, lo, hi, first);
    else
        append_keys<T, PAD>(a, seq, head, pair, block, lo, hi, first);
}

template <class T, int PAD>
__device__ __forceinline__ void read_keys(const Kv8ReadArgs &a, int seq, int head, size_t pair, int block, int lo,
                                          int hi) {
    using S = Share<PAD>;
    const int lane = threadIdx.x & 63, place = 16 * block + (lane >> 2);
    if (place < lo || place >= hi) return;
    const float scale = power(a.cache.ks[pair * (a.cache.capacity / 16) + block]);
    const uint8_t *const in = a.cache.k + (pair * a.cache.capacity + place) * PAD;
    auto *row = static_cast<typename T::Raw *>(a.k) + seq * a.ks.s[0] + int64_t(place - a.first) * a.ks.s[1] +
                head * a.ks.s[2];
#pragma unroll
    for (int p = 0; p < S::kPasses; ++p) {
        const int d = S::kRun * (lane & 3) + 64 * p;
        const uint32_t *const w = reinterpret_cast<const uint32_t *>(in + d);
        float x[S::kRun];
#pragma unroll
        for (int i = 0; i < S::kRun / 4; ++i) {
            float y[4];
            decode4(w[i], y);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * i + j] = y[j] * scale;
        }
        store_run<T>(row + d, a.cache.width - d, a.aligned, x);
    }
}

template <class T, int PAD>
__device__ __forceinline__ void read_values(const Kv8ReadArgs &a, int seq, int head, size_t pair, int block, int lo,
                                            int hi) {
    using S = Share<PAD>;
    const int lane = threadIdx.x & 63, slot0 = PAD >= 64 ? 0 : 8 * (lane >> 5), place0 = 16 * block + slot0;
    const float scale = power(a.cache.vs[pair * (a.cache.capacity / 16) + block]);
    auto *base = static_cast<typename T::Raw *>(a.v) + seq * a.vs.s[0] + head * a.vs.s[2];
#pragma unroll
    for (int p = 0; p < S::kPasses; ++p) {
        const int d = PAD >= 64 ? lane + 64 * p : lane & 31;
        if (d >= a.cache.width) continue;
        const uint32_t *const w = reinterpret_cast<const uint32_t *>(
            a.cache.v + ((pair * (a.cache.capacity / 64) + block / 4) * PAD + d) * 64 + 16 * (block % 4) + slot0);
#pragma unroll
        for (int i = 0; i < S::kSlots / 4; ++i) {
            float y[4];
            decode4(w[i], y);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int place = place0 + 4 * i + j;
                if (place >= lo && place < hi)
                    base[int64_t(place - a.first) * a.vs.s[1] + d] = T::from_float(y[j] * scale);
            }
        }
    }
}

template <class T, int PAD>
__global__ void __launch_bounds__(256) kv8_read_kernel(Kv8ReadArgs a, int blocks, uint32_t units) {
    const uint32_t u = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (u >= units) return;
    const uint32_t rest = u >> 1, pair = rest / uint32_t(blocks);
    const int seq = int(pair) / a.cache.heads, head = int(pair) - seq * a.cache.heads;
    int last = a.first + a.count;
    if (a.lengths) last = min(last, a.lengths[seq]);
    const int block = a.first / 16 + int(rest - pair * uint32_t(blocks));
    const int lo = max(a.first, 16 * block), hi = min(last, 16 * block + 16);
    if (lo >= hi) return;
    if (u & 1)
        read_values<T, PAD>(a, seq, head, pair, block, lo, hi);
    else
        read_keys<T, PAD>(a, seq, head, pair, block, lo, hi);
}

template <class T, int PAD>
void launch_append(const Kv8AppendArgs &a, hipStream_t stream) {
    const int blocks = (a.count + 30) / 16;  // a run of n tokens touches at most so many
    const uint32_t units = 2u * uint32_t(a.cache.batch) * uint32_t(a.cache.heads) * uint32_t(blocks);
    hipLaunchKernelGGL((kv8_append_kernel<T, PAD>), dim3((units + 3) / 4), dim3(256), 0, stream, a, blocks, units);
}

template <class T, int PAD>
void launch_read(const Kv8ReadArgs &a, hipStream_t stream) {
    const int blocks = (a.first + a.count + 15) / 16 - a.first / 16;
    const uint32_t units = 2u * uint32_t(a.cache.batch) * uint32_t(a.cache.heads) * uint32_t(blocks);
    hipLaunchKernelGGL((kv8_read_kernel<T, PAD>), dim3((units + 3) / 4), dim3(256), 0, stream, a, blocks, units);
}

template <class T>
void append_of(const Kv8AppendArgs &a, hipStream_t stream) {
    switch (a.cache.pad) {
    case 32: return launch_append<T, 32>(a, stream);
    case 64: return launch_append<T, 64>(a, stream);
    case 128: return launch_append<T, 128>(a, stream);
    default: return launch_append<T, 256>(a, stream);
    }
}

template <class T>
void read_of(const Kv8ReadArgs &a, hipStream_t stream) {
    switch (a.cache.pad) {
    case 32: return launch_read<T, 32>(a, stream);
    case 64: return launch_read<T, 64>(a, stream);
    case 128: return launch_read<T, 128>(a, stream);
    default: return launch_read<T, 256>(a, stream);
    }
}

}  // namespace

void kv8_append(const Kv8AppendArgs &a, Type type, hipStream_t stream) {
    switch (type) {
    case Type::F32: return append_of<F32>(a, stream);
    case Type::F16: return append_of<F16>(a, stream);
    default: return append_of<BF16>(a, stream);
    }
}

void kv8_read(const Kv8ReadArgs &a, Type type, hipStream_t stream) {
    switch (type) {
    case Type::F32: return read_of<F32>(a, stream);
    case Type::F16: return read_of<F16>(a, stream);
    default: return read_of<BF16>(a, stream);
    }
}

}  // namespace meshgpt::kern
