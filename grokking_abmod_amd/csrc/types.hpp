// Element types of the device operators: 16-byte groups as floats and back.
#pragma once

#include <hip/hip_runtime.h>

namespace meshgpt::kern {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct F32 {
    using Raw = float;
    static constexpr int kGroup = 4;  // elements of 16 bytes
    static __device__ __forceinline__ float to_float(Raw x) { return x; }
    static __device__ __forceinline__ Raw from_float(float x) { return x; }
    static __device__ __forceinline__ void unpack(uint4 g, float (&x)[4]) {
        x[0] = __builtin_bit_cast(float, g.x);
        x[1] = __builtin_bit_cast(float, g.y);
        x[2] = __builtin_bit_cast(float, g.z);
        x[3] = __builtin_bit_cast(float, g.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&x)[4]) {
        return {__builtin_bit_cast(uint32_t, x[0]), __builtin_bit_cast(uint32_t, x[1]),
                __builtin_bit_cast(uint32_t, x[2]), __builtin_bit_cast(uint32_t, x[3])};
    }
};

struct F16 {
    using Raw = _Float16;
    static constexpr int kGroup = 8;
    static __device__ __forceinline__ float to_float(Raw x) { return float(x); }
    static __device__ __forceinline__ Raw from_float(float x) { return Raw(x); }
    static __device__ __forceinline__ void unpack(uint4 g, float (&x)[8]) {
        const uint32_t w[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f16x2 h = __builtin_bit_cast(f16x2, w[i]);
            x[2 * i] = float(h[0]);
            x[2 * i + 1] = float(h[1]);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(uint32_t, f16x2{Raw(x[2 * i]), Raw(x[2 * i + 1])});
        return {w[0], w[1], w[2], w[3]};
    }
};

struct BF16 {
    using Raw = __bf16;
    static constexpr int kGroup = 8;
    static __device__ __forceinline__ float to_float(Raw x) { return float(x); }
    static __device__ __forceinline__ Raw from_float(float x) { return Raw(x); }
    static __device__ __forceinline__ void unpack(uint4 g, float (&x)[8]) {
        const uint32_t w[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __builtin_bit_cast(float, w[i] << 16);
            x[2 * i + 1] = __builtin_bit_cast(float, w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x[2 * i], x[2 * i + 1]}, bf16x2));
        return {w[0], w[1], w[2], w[3]};
    }
};

// 16 bytes at any element: the compiler's loads and stores for this target allow it.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ uint4 get_any(const void *p) {
    return __builtin_bit_cast(uint4, u32x4(*static_cast<const u32x4_any *>(p)));
}
__device__ __forceinline__ void put_any(void *p, uint4 w) {
    *static_cast<u32x4_any *>(p) = __builtin_bit_cast(u32x4, w);
}

// A group's elements from the n-th on, moved to its begin, and zeros (n from 0 to all).  A
// row's end is read by a whole load that ends there, and moved.
template <class T>
__device__ __forceinline__ uint4 moved_down(uint4 w, int n) {
    const uint32_t bits = 8 * sizeof(typename T::Raw) * uint32_t(n);
    const uint64_t lo = uint64_t(w.y) << 32 | w.x, hi = uint64_t(w.w) << 32 | w.z;
    const uint64_t low = bits < 64 ? lo >> (bits & 63) | (bits ? hi << (64 - bits & 63) : 0) : bits < 128 ? hi >> (bits & 63) : 0;
    const uint64_t high = bits < 64 ? hi >> (bits & 63) : 0;
    return {uint32_t(low), uint32_t(low >> 32), uint32_t(high), uint32_t(high >> 32)};
}
// The first `have` elements of a group, fewer than it holds, the rest zero; and back.
template <class T>
__device__ __forceinline__ uint4 get_part(const typename T::Raw *p, int have) {
    constexpr int SIZE = sizeof(typename T::Raw);
    uint4 w{0, 0, 0, 0};
#pragma unroll 1
    for (int e = 0; e < have; ++e) {
        uint32_t x;
        if constexpr (SIZE == 4)
            x = __builtin_bit_cast(uint32_t, p[e]);
        else
            x = uint32_t(__builtin_bit_cast(uint16_t, p[e])) << (e % 2 * 16);
        const int word = e * SIZE / 4;
        w.x |= word == 0 ? x : 0;
        w.y |= word == 1 ? x : 0;
        w.z |= word == 2 ? x : 0;
        w.w |= word == 3 ? x : 0;
    }
    return w;
}
typedef uint32_t u32_any __attribute__((aligned(1)));
template <class T>
__device__ __forceinline__ void put_part(typename T::Raw *p, int have, uint4 w) {
    if (have <= 0) return;
    u32_any *const words = reinterpret_cast<u32_any *>(p);
    if constexpr (sizeof(*p) == 4) {
        words[0] = w.x;
        if (have > 1) words[1] = w.y;
        if (have > 2) words[2] = w.z;
    } else {
        if (have > 1) words[0] = w.x;
        if (have > 3) words[1] = w.y;
        if (have > 5) words[2] = w.z;
        const uint32_t last = have < 2 ? w.x : have < 4 ? w.y : have < 6 ? w.z : w.w;
        if (have % 2) p[have - 1] = __builtin_bit_cast(typename T::Raw, uint16_t(last));
    }
}

// Inputs and outputs of more than the Infinity Cache's 256 MB: whoever comes next
// does not find them there, so they are moved past the caches (STREAM).
constexpr double kCached = double(256u << 20);
template <bool STREAM, class W>
__device__ __forceinline__ void put(void *p, W w) {
    if constexpr (STREAM)
        __builtin_nontemporal_store(w, static_cast<W *>(p));
    else
        *static_cast<W *>(p) = w;
}
template <bool STREAM>
__device__ __forceinline__ void put_any(void *p, uint4 w) {
    if constexpr (STREAM)
        __builtin_nontemporal_store(__builtin_bit_cast(u32x4, w), static_cast<u32x4_any *>(p));
    else
        put_any(p, w);
}
template <bool STREAM>
__device__ __forceinline__ uint4 get(const uint4 *p) {
    if constexpr (STREAM)
        return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p)));
    else
        return *p;
}

}  // namespace meshgpt::kern
