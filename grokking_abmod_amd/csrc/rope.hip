// Rotary positions of queries and keys, and their gradient.
//
// Pair i of a head (channels i and i + rotary / 2, or 2 i and 2 i + 1) at
// position p turns by the angle p f_i and is scaled by the magnitude m:
//   (a, b) -> m (a cos - b sin, b cos + a sin);
// the gradient turns back.  Channels from `rotary` on stay as they are.
//
// Angles are taken in FP64 as turns and reduced to an eighth of one, because at
// position 10^6 an FP32 product is off by a thirtieth of a radian; sine and
// cosine of what is left are FP32 series.  A workgroup makes them once for its
// tokens, in LDS, and applies them to all heads, 16 bytes of each half a thread.
#include "operators.hpp"
#include "types.hpp"

namespace meshgpt::kern {
namespace {

constexpr int kBlock = 256;
constexpr int kTokens = 16;    // of a workgroup, at most
constexpr int kPairs = 1024;   // angles of a workgroup, at most: half of the widest head times two

// cos and sin of 2 pi t.
__device__ __forceinline__ float2 turned(double t) {
    t -= rint(t);
    const double quarter = rint(4.0 * t);
    const float x = float((t - 0.25 * quarter) * 6.283185307179586), y = x * x;  // |x| <= pi / 4
    // The series to x^9 and x^10: the next terms are under 2e-9 and 2e-10.
    const float s = fmaf(x * y, fmaf(y, fmaf(y, fmaf(y, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), x);
    const float c = fmaf(y, fmaf(y, fmaf(y, fmaf(y, fmaf(y, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
    const int q = int(quarter) & 3;
    const float a = q & 1 ? s : c, b = q & 1 ? c : s;
    return {q == 1 || q == 2 ? -a : a, q >= 2 ? -b : b};
}

template <class T, int N>
__device__ __forceinline__ void load(const typename T::Raw *p, int have, float (&x)[N]) {
    if (have >= N) return T::unpack(get_any(p), x);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = i < have ? T::to_float(p[i]) : 0.0f;
}
template <class T, int N>
__device__ __forceinline__ void store(typename T::Raw *p, int have, const float (&x)[N]) {
    if (have >= N) return put_any(p, T::pack(x));
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (i < have) p[i] = T::from_float(x[i]);
}

template <class T>
__global__ void __launch_bounds__(kBlock) rope_kernel(RopeArgs a, int tile, int items, int slots) {
    using Raw = typename T::Raw;
    constexpr int G = T::kGroup;
    __shared__ float2 table[kPairs];
    __shared__ int64_t places[kTokens];  // sequence << 32 | token, -1: not there
    __shared__ int positions[kTokens];
    const int tid = threadIdx.x, half = a.rotary / 2;
    const int64_t first = int64_t(blockIdx.x) * tile, all = int64_t(a.batch) * a.count;
    if (tid < tile) {
        const int64_t t = first + tid;
        places[tid] = -1;
        if (t < all) {
            const int64_t s = t / a.count;
            const int i = int(t - s * a.count), n = a.counts ? a.counts[s] : a.count;
            const int length = a.lengths ? a.lengths[s] : n;
            if (n >= 0 && n <= a.count && length >= n && i < n) {
                places[tid] = s << 32 | i;
                positions[tid] = a.positions ? a.positions[t] : length - n + i;
            }
        }
    }
    __syncthreads();
    for (int i = tid; i < tile * half; i += kBlock) {
        const int t = i / half;
        if (places[t] < 0) continue;
        float2 cs = turned(double(positions[t]) * (a.frequencies[i - t * half] * 0.15915494309189535));
        if (a.backward) cs.y = -cs.y;
        table[i] = {cs.x * a.magnitude, cs.y * a.magnitude};
    }
    __syncthreads();

    // A thread has one group of a head, in every slots-th head of the tokens.
    const int slot = tid / items, item = tid - slot * items;
    if (slot >= slots) return;
    const int heads = a.side[0].heads + a.side[1].heads;
    const int groups = a.interleaved ? (a.rotary + G - 1) / G : (half + G - 1) / G;  // that turn
    int t = 0, h = slot;
    for (;;) {
        while (h >= heads) {
            h -= heads;
            ++t;
        }
        if (t >= tile) return;
        const int64_t place = places[t];
        if (place >= 0) {
            const bool second = h >= a.side[0].heads;
            const RopeSide &side = a.side[second];
            const int64_t s = place >> 32, i = place & 0xffffffff, head = second ? h - a.side[0].heads : h;
            const Raw *const x = static_cast<const Raw *>(side.x) + s * side.xs.s[0] + i * side.xs.s[1] + head * side.xs.s[2];
            Raw *const o = static_cast<Raw *>(side.out) + s * side.os.s[0] + i * side.os.s[1] + head * side.os.s[2];
            const float2 *const row = table + t * half;
            if (item >= groups) {  // stays as it is
                const int at = a.rotary + (item - groups) * G, have = a.width - at;
                if (have >= G) {
                    put_any(o + at, get_any(x + at));
                } else {
                    for (int e = 0; e < have; ++e) o[at + e] = x[at + e];
                }
            } else if (a.interleaved) {
                const int at = item * G, have = a.rotary - at;
                float v[G];
                load<T>(x + at, have, v);
#pragma unroll
                for (int e = 0; e < G; e += 2) {
                    const float2 cs = row[min(at + e, a.rotary - 2) / 2];
                    const float p = v[e], q = v[e + 1];
                    v[e] = p * cs.x - q * cs.y;
                    v[e + 1] = q * cs.x + p * cs.y;
                }
                store<T>(o + at, have, v);
            } else {
                const int at = item * G, have = half - at;
                float p[G], q[G];
                load<T>(x + at, have, p);
                load<T>(x + at + half, have, q);
#pragma unroll
                for (int e = 0; e < G; ++e) {
                    const float2 cs = row[min(at + e, half - 1)];
                    const float v = p[e], w = q[e];
                    p[e] = v * cs.x - w * cs.y;
                    q[e] = w * cs.x + v * cs.y;
                }
                store<T>(o + at, have, p);
                store<T>(o + at + half, have, q);
            }
        }
        h += slots;
    }
}

template <class T>
void launch(const RopeArgs &a, hipStream_t stream) {
    constexpr int G = T::kGroup;
    const int half = a.rotary / 2;
    bool same = true;  // what stays is there already
    for (const RopeSide &s : a.side)
        if (s.heads)
            same = same && s.x == s.out && s.xs.s[0] == s.os.s[0] && s.xs.s[1] == s.os.s[1] && s.xs.s[2] == s.os.s[2];
    const int turning = a.interleaved ? (a.rotary + G - 1) / G : (half + G - 1) / G;
    const int items = turning + (same ? 0 : (a.width - a.rotary + G - 1) / G);
    if (items == 0) return;
    const int64_t tokens = int64_t(a.batch) * a.count;
    const int most = half ? kPairs / half : kTokens;
    const int tile = int(std::max<int64_t>(1, std::min<int64_t>({tokens / 2048, kTokens, most})));
    rope_kernel<T><<<dim3(unsigned((tokens + tile - 1) / tile)), kBlock, 0, stream>>>(a, tile, items, kBlock / items);
}

}  // namespace

void rope(const RopeArgs &a, Type type, hipStream_t stream) {
    switch (type) {
        case Type::F32: return launch<F32>(a, stream);
        case Type::F16: return launch<F16>(a, stream);
        case Type::BF16: return launch<BF16>(a, stream);
    }
}

}  // namespace meshgpt::kern
