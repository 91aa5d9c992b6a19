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
__device__ __forceinline__ uint4 get(const uint4 *p) {
    if constexpr (STREAM)
        return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p)));
    else
        return *p;
}

}  // namespace meshgpt::kern
