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
// or of its values.  Keys are stored as they come; a lane takes 16 bytes of a
// token's inputs.  Values are stored transposed, 64 tokens of a channel in a row, the
// order in which the attention's matrix product reads them; a lane takes two
// channels of the 16 tokens.  Memory bounds both where there is enough of it: 8
// prompts of up to 4000 tokens, 8 heads of 128, BF16, are written in 37 us (3.3 TB/s
// read and written), or in 32 where the inputs lie in the Infinity Cache; 16 caches
// of 8000 tokens are read back as F16 in 135 us (5.8 TB/s); a step of 32 sequences
// takes 4.6 us.
#include <hip/hip_runtime.h>

#include <cfloat>

#include "dpp.hpp"
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

// N consecutive elements from p (N of 16 bytes, or two), those at or past `have`
// as 0.  Aligned: to 16 bytes, so that whole groups are aligned to their size, to
// 4, or (0) to the element.
template <class T, int N>
__device__ __forceinline__ void load_run(const typename T::Raw *p, int have, int aligned, float (&x)[N]) {
    if (aligned == 16 && have >= N) {
        if constexpr (N == T::kGroup) {
            T::unpack(*reinterpret_cast<const uint4 *>(p), x);
        } else if constexpr (sizeof(*p) == 4) {
            const uint2 w = *reinterpret_cast<const uint2 *>(p);
            x[0] = __builtin_bit_cast(float, w.x);
            x[1] = __builtin_bit_cast(float, w.y);
        } else {
            float y[8];
            T::unpack(uint4{*reinterpret_cast<const uint32_t *>(p), 0, 0, 0}, y);
            x[0] = y[0];
            x[1] = y[1];
        }
        return;
    }
    if constexpr (sizeof(*p) == 2) {
        if (aligned) {
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                uint32_t w = 0;
                if (i + 1 < have)
                    w = *reinterpret_cast<const uint32_t *>(p + i);
                else if (i < have)
                    w = __builtin_bit_cast(uint16_t, p[i]);
                float y[8];
                T::unpack(uint4{w, 0, 0, 0}, y);
                x[i] = y[0];
                x[i + 1] = y[1];
            }
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = i < have ? T::to_float(p[i]) : 0.0f;
}

template <class T, bool STREAM, int N>
__device__ __forceinline__ void store_run(typename T::Raw *p, int have, int aligned, const float (&x)[N]) {
    if (aligned == 16 && have >= N) {
        if constexpr (N == T::kGroup) {
            put<STREAM>(p, __builtin_bit_cast(u32x4, T::pack(x)));
        } else if constexpr (sizeof(*p) == 4) {
            put<STREAM>(p, f32x2{x[0], x[1]});
        } else {
            const float y[8] = {x[0], x[1], 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
            put<STREAM>(p, T::pack(y).x);
        }
        return;
    }
    if constexpr (sizeof(*p) == 2) {
        if (aligned) {
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                const float y[8] = {x[i], x[i + 1], 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
                if (i + 1 < have)
                    *reinterpret_cast<uint32_t *>(p + i) = T::pack(y).x;
                else if (i < have)
                    p[i] = T::from_float(x[i]);
            }
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (i < have) p[i] = T::from_float(x[i]);
}

__device__ __forceinline__ float finite_size(float x) { return fabsf(x) <= FLT_MAX ? fabsf(x) : 0.0f; }

// How a lane takes part in keys: kRun channels (16 bytes of the inputs) of tokens
// kRows apart, so that a wave's loads and stores are whole rows.
template <class T, int PAD>
struct KeyShare {
    static constexpr int kRun = T::kGroup, kLanes = PAD / kRun, kRows = 64 / kLanes, kPasses = 16 / kRows;
};
// In values: two channels of kSlots tokens, kPasses times 128 channels on.
template <int PAD>
struct ValueShare {
    static constexpr int kPasses = PAD >= 128 ? PAD / 128 : 1;
    static constexpr int kLanes = PAD >= 128 ? 64 : PAD / 2, kSlots = 16 * kLanes / 64;
};

// Positions [lo, hi) of the block's 16 are new; with lo past the block's first,
// the ones before it are older and keep their values.
template <class T, int PAD>
__device__ __forceinline__ void append_keys(const Kv8AppendArgs &a, int seq, int head, size_t pair, int block, int lo,
                                            int hi, int first) {
    using S = KeyShare<T, PAD>;
    const int lane = threadIdx.x & 63, d = S::kRun * (lane % S::kLanes), place0 = 16 * block + lane / S::kLanes;
    const bool begun = lo > 16 * block;
    const auto *base = static_cast<const typename T::Raw *>(a.k) + seq * a.ks.s[0] + head * a.ks.s[2] + d;
    uint8_t *const scale = a.cache.ks + pair * (a.cache.capacity / 16) + block;
    const int was = begun ? *scale : 0;
    float x[S::kPasses][S::kRun], top = 0.0f;
#pragma unroll
    for (int p = 0; p < S::kPasses; ++p) {
        const int place = place0 + p * S::kRows;
        const bool fresh = place >= lo && place < hi;
        load_run<T>(base + int64_t(place - first) * a.ks.s[1], fresh ? a.cache.width - d : 0, a.aligned, x[p]);
    }
#pragma unroll
    for (int p = 0; p < S::kPasses; ++p)
#pragma unroll
        for (int i = 0; i < S::kRun; ++i) top = fmaxf(top, finite_size(x[p][i]));
    const int byte = min(max(scale_byte(wave_largest(top)), was), kHighScale);
    const float inverse = power(254 - byte), limit = byte == kHighScale ? 240.0f : 448.0f;
    if (lane == 0) *scale = uint8_t(byte);
#pragma unroll
    for (int p = 0; p < S::kPasses; ++p) {
        const int place = place0 + p * S::kRows;
        const bool fresh = place >= lo && place < hi;
        if (!fresh && !(begun && byte > was && place < lo)) continue;
        uint32_t *const w = reinterpret_cast<uint32_t *>(a.cache.k + (pair * a.cache.capacity + place) * PAD + d);
        uint32_t c[S::kRun / 4];
#pragma unroll
        for (int i = 0; i < S::kRun / 4; ++i) {
            if (fresh) {
                float y[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = in_range(x[p][4 * i + j], inverse, limit);
                c[i] = encode4(y[0], y[1], y[2], y[3]);
            } else {
                c[i] = lowered4(w[i], byte - was);
            }
        }
        if constexpr (S::kRun == 8)
            *reinterpret_cast<uint2 *>(w) = uint2{c[0], c[1]};
        else
            *w = c[0];
    }
}

template <class T, int PAD>
__device__ __forceinline__ void append_values(const Kv8AppendArgs &a, int seq, int head, size_t pair, int block, int lo,
                                              int hi, int first) {
    using S = ValueShare<PAD>;
    const int lane = threadIdx.x & 63, slot0 = S::kSlots * (lane / S::kLanes), place0 = 16 * block + slot0;
    const bool begun = lo > 16 * block;
    const auto *base = static_cast<const typename T::Raw *>(a.v) + seq * a.vs.s[0] + head * a.vs.s[2];
    uint8_t *const scale = a.cache.vs + pair * (a.cache.capacity / 16) + block;
    const int was = begun ? *scale : 0;
    float x[S::kPasses][2][S::kSlots], top = 0.0f;
#pragma unroll
    for (int p = 0; p < S::kPasses; ++p) {
        const int d = 2 * (lane % S::kLanes) + 128 * p;
#pragma unroll
        for (int i = 0; i < S::kSlots; ++i) {
            const int place = place0 + i;
            const bool fresh = place >= lo && place < hi;
            float two[2];
            load_run<T>(base + int64_t(place - first) * a.vs.s[1] + d, fresh ? a.cache.width - d : 0, a.aligned, two);
            x[p][0][i] = two[0];
            x[p][1][i] = two[1];
        }
    }
#pragma unroll
    for (int p = 0; p < S::kPasses; ++p)
#pragma unroll
        for (int i = 0; i < S::kSlots; ++i)
            top = fmaxf(top, fmaxf(finite_size(x[p][0][i]), finite_size(x[p][1][i])));
    const int byte = min(max(scale_byte(wave_largest(top)), was), kHighScale);
    const float inverse = power(254 - byte), limit = byte == kHighScale ? 240.0f : 448.0f;
    if (lane == 0) *scale = uint8_t(byte);
    const bool whole = lo == 16 * block && hi == 16 * block + 16, lower = begun && byte > was;
#pragma unroll
    for (int p = 0; p < S::kPasses; ++p)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int d = 2 * (lane % S::kLanes) + 128 * p + q;
            uint32_t *const w = reinterpret_cast<uint32_t *>(
                a.cache.v + ((pair * (a.cache.capacity / 64) + block / 4) * PAD + d) * 64 + 16 * (block % 4) + slot0);
            uint32_t c[S::kSlots / 4];
#pragma unroll
            for (int i = 0; i < S::kSlots / 4; ++i) {
                float y[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = in_range(x[p][q][4 * i + j], inverse, limit);
                c[i] = encode4(y[0], y[1], y[2], y[3]);
            }
            if (!whole) {  // the bytes around the new ones: lowered where older, left where behind
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
                *reinterpret_cast<uint4 *>(w) = uint4{c[0], c[1], c[2], c[3]};
            else if constexpr (S::kSlots == 8)
                *reinterpret_cast<uint2 *>(w) = uint2{c[0], c[1]};
            else
                *w = c[0];
        }
}

// A wave's part of a launch: the keys or the values of one of the blocks of 16
// tokens of a head.  Four waves of a workgroup take the four blocks of a tile,
// whose lines of 64 values they fill together; the workgroups of a tile's heads,
// whose tokens lie side by side in most inputs, follow one another.  The values,
// which take longer, come first: keys and values in turn would give every other
// XCD the one kind (8 x 4000 tokens, 8 heads of 128, BF16: 53.8 us, against 43.7).
struct Unit {
    bool values;
    int seq, head, block;
    __device__ __forceinline__ Unit(int heads, int tiles) {
        const uint32_t half = gridDim.x / 2, u = blockIdx.x < half ? blockIdx.x : blockIdx.x - half;
        const uint32_t rest = u / uint32_t(heads);
        values = blockIdx.x < half;
        head = int(u - rest * uint32_t(heads));
        seq = int(rest / uint32_t(tiles));
        block = 4 * int(rest - uint32_t(seq) * uint32_t(tiles)) + int(threadIdx.x >> 6);
    }
};

// Of every (sequence, head), the tiles that a run of new tokens touches at most.
template <class T, int PAD>
__global__ void __launch_bounds__(256) kv8_append_kernel(Kv8AppendArgs a, int tiles) {
    const Unit u(a.cache.heads, tiles);
    const int seq = u.seq, head = u.head;
    const size_t pair = size_t(seq) * a.cache.heads + head;
    const int length = a.lengths[seq], count = a.counts ? a.counts[seq] : a.count;
    if (length < 0 || length > a.cache.capacity || count < 0 || count > a.count || count > length) return;
    const int start = length - count, block = start / 64 * 4 + u.block;
    const int lo = max(start, 16 * block), hi = min(length, 16 * block + 16);
    if (lo >= hi) return;
    const int first = a.absolute ? 0 : start;
    if (u.values)
        append_values<T, PAD>(a, seq, head, pair, block, lo, hi, first);
    else
        append_keys<T, PAD>(a, seq, head, pair, block, lo, hi, first);
}

template <class T, int PAD, bool STREAM>
__device__ __forceinline__ void read_keys(const Kv8ReadArgs &a, int seq, int head, size_t pair, int block, int lo,
                                          int hi) {
    using S = KeyShare<T, PAD>;
    const int lane = threadIdx.x & 63, d = S::kRun * (lane % S::kLanes), place0 = 16 * block + lane / S::kLanes;
    const float scale = power(a.cache.ks[pair * (a.cache.capacity / 16) + block]);
    auto *base = static_cast<typename T::Raw *>(a.k) + seq * a.ks.s[0] + head * a.ks.s[2] + d;
    const uint8_t *const in = a.cache.k + pair * a.cache.capacity * PAD + d;
    uint32_t w[S::kPasses][S::kRun / 4];
#pragma unroll
    for (int p = 0; p < S::kPasses; ++p) {
        const uint8_t *const row = in + size_t(place0 + p * S::kRows) * PAD;
        if constexpr (S::kRun == 8) {
            const uint2 v = *reinterpret_cast<const uint2 *>(row);
            w[p][0] = v.x;
            w[p][1] = v.y;
        } else {
            w[p][0] = *reinterpret_cast<const uint32_t *>(row);
        }
    }
#pragma unroll
    for (int p = 0; p < S::kPasses; ++p) {
        const int place = place0 + p * S::kRows;
        if (place < lo || place >= hi) continue;
        float x[S::kRun];
#pragma unroll
        for (int i = 0; i < S::kRun / 4; ++i) {
            float y[4];
            decode4(w[p][i], y);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * i + j] = y[j] * scale;
        }
        store_run<T, STREAM>(base + int64_t(place - a.first) * a.ks.s[1], a.cache.width - d, a.aligned, x);
    }
}

template <class T, int PAD, bool STREAM>
__device__ __forceinline__ void read_values(const Kv8ReadArgs &a, int seq, int head, size_t pair, int block, int lo,
                                            int hi) {
    using S = ValueShare<PAD>;
    const int lane = threadIdx.x & 63, slot0 = S::kSlots * (lane / S::kLanes), place0 = 16 * block + slot0;
    const float scale = power(a.cache.vs[pair * (a.cache.capacity / 16) + block]);
    auto *base = static_cast<typename T::Raw *>(a.v) + seq * a.vs.s[0] + head * a.vs.s[2];
#pragma unroll
    for (int p = 0; p < S::kPasses; ++p) {
        const int d = 2 * (lane % S::kLanes) + 128 * p;
        float x[2][S::kSlots];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const uint32_t *const w = reinterpret_cast<const uint32_t *>(
                a.cache.v + ((pair * (a.cache.capacity / 64) + block / 4) * PAD + d + q) * 64 + 16 * (block % 4) + slot0);
#pragma unroll
            for (int i = 0; i < S::kSlots / 4; ++i) {
                float y[4];
                decode4(w[i], y);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[q][4 * i + j] = y[j] * scale;
            }
        }
#pragma unroll
        for (int i = 0; i < S::kSlots; ++i) {
            const int place = place0 + i;
            const float two[2] = {x[0][i], x[1][i]};
            if (place >= lo && place < hi)
                store_run<T, STREAM>(base + int64_t(place - a.first) * a.vs.s[1] + d, a.cache.width - d, a.aligned, two);
        }
    }
}

template <class T, int PAD, bool STREAM>
__global__ void __launch_bounds__(256) kv8_read_kernel(Kv8ReadArgs a, int tiles) {
    const Unit u(a.cache.heads, tiles);
    const int seq = u.seq, head = u.head;
    const size_t pair = size_t(seq) * a.cache.heads + head;
    int last = a.first + a.count;
    if (a.lengths) last = min(last, a.lengths[seq]);
    const int block = a.first / 64 * 4 + u.block;
    const int lo = max(a.first, 16 * block), hi = min(last, 16 * block + 16);
    if (lo >= hi) return;
    if (u.values)
        read_values<T, PAD, STREAM>(a, seq, head, pair, block, lo, hi);
    else
        read_keys<T, PAD, STREAM>(a, seq, head, pair, block, lo, hi);
}

template <class T, int PAD>
void launch_append(const Kv8AppendArgs &a, hipStream_t stream) {
    const size_t groups = kv8_append_workgroups(size_t(a.cache.batch) * size_t(a.cache.heads), size_t(a.count));
    const int tiles = int(groups / (2 * size_t(a.cache.batch) * size_t(a.cache.heads)));
    hipLaunchKernelGGL((kv8_append_kernel<T, PAD>), dim3(uint32_t(groups)), dim3(256), 0, stream, a, tiles);
}

template <class T, int PAD>
void launch_read(const Kv8ReadArgs &a, hipStream_t stream) {
    const int tiles = (a.first + a.count + 63) / 64 - a.first / 64;
    const dim3 grid(2u * uint32_t(a.cache.batch * a.cache.heads) * uint32_t(tiles));
    // 524 MB of F16 take 135 us past the caches, 142 otherwise.
    if (2.0 * a.cache.batch * a.cache.heads * a.cache.width * double(a.count) * sizeof(typename T::Raw) > kCached)
        hipLaunchKernelGGL((kv8_read_kernel<T, PAD, true>), grid, dim3(256), 0, stream, a, tiles);
    else
        hipLaunchKernelGGL((kv8_read_kernel<T, PAD, false>), grid, dim3(256), 0, stream, a, tiles);
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
