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
// tokens, in LDS, and applies them to all heads, 16 bytes of each half a thread, with the
// next head's loads under way.  Every element is read and written once, and memory bounds
// it: 32768 tokens of 40 heads of 128 BF16 115 us (5.8 TB/s), 16384 of 32 heads of 64 32
// (4.2); 3003 of 16 heads of 80 F16 7 us, which its few workgroups' chains bound.
#include <algorithm>

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

template <class T, bool STREAM>
__device__ __forceinline__ void store(typename T::Raw *p, int have, uint4 w) {
    if (have >= T::kGroup) return put_any<STREAM>(p, w);
    put_part<T>(p, have, w);
}

// A head's work is cut into items of 16 bytes: of neighbours that are pairs, all of the
// head; else of its first half of turning channels, with those of the second, and then of
// what stays.
template <class T, bool INTERLEAVED, bool STREAM>
__global__ void __launch_bounds__(kBlock) rope_kernel(RopeArgs a, int tile, int items, int slots) {
    using Raw = typename T::Raw;
    constexpr int G = T::kGroup;
    __shared__ float2 table[kPairs];
    __shared__ int tokens[kTokens];  // in its sequence, -1: not there
    __shared__ int sequences[kTokens], positions[kTokens];
    const int tid = threadIdx.x, half = a.rotary / 2;
    const uint32_t first = blockIdx.x * uint32_t(tile), all = uint32_t(a.batch) * uint32_t(a.count);
    if (tid < tile) {
        const uint32_t t = first + tid, s = min(t, all - 1) / uint32_t(a.count);
        const int i = int(t - s * uint32_t(a.count)), n = a.counts ? a.counts[s] : a.count;
        const int length = a.lengths ? a.lengths[s] : n;
        const bool there = t < all && n >= 0 && n <= a.count && length >= n && i < n;
        tokens[tid] = there ? i : -1;
        sequences[tid] = int(s);
        positions[tid] = there && a.positions ? a.positions[t] : length - n + i;
    }
    __syncthreads();

    // A thread has one item of a head, in every slots-th head of the tokens.
    const int slot = tid / items, item = tid - slot * items;
    const int heads = a.side[0].heads + a.side[1].heads;
    const int turning = INTERLEAVED ? items : (half + G - 1) / G;
    const bool turns = item < turning;
    const int at = turns ? item * G : a.rotary + (item - turning) * G;
    const int have = (INTERLEAVED || !turns ? a.width : half) - at;
    int t = 0, h = slot;
    struct Place {
        const Raw *x;
        Raw *o;
        int t;  // of the tile, or -1: nothing
    };
    const auto next = [&] {
        Place p{nullptr, nullptr, -1};
        for (;; h += slots) {
            while (h >= heads) {
                h -= heads;
                ++t;
            }
            if (slot >= slots || t >= tile) return p;
            if (tokens[t] < 0) continue;
            const bool second = h >= a.side[0].heads;
            const RopeSide &side = a.side[second];
            const int64_t s = sequences[t], i = tokens[t], head = second ? h - a.side[0].heads : h;
            p.x = static_cast<const Raw *>(side.x) + s * side.xs.s[0] + i * side.xs.s[1] + head * side.xs.s[2] + at;
            p.o = static_cast<Raw *>(side.out) + s * side.os.s[0] + i * side.os.s[1] + head * side.os.s[2] + at;
            p.t = t;
            h += slots;
            return p;
        }
    };
    // A group that an end cuts is read with other channels of the head, before it (and moved
    // once it is used) or behind it; a head of less than a group by its elements.
    const bool pairs = !INTERLEAVED && turns;
    const int end = at + (pairs ? half : 0), back = a.width >= G ? max(0, end + G - a.width) : 0;
    const int front = pairs ? (a.width >= G ? max(0, at + G - a.width) : 0) : back;
    const auto fetch = [&](const Place &p, uint4 &x, uint4 &y) {
        if (p.t < 0) return;
        x = a.width >= G ? get_any(p.x - front) : get_part<T>(p.x, have);
        if (pairs) y = a.width >= G ? get_any(p.x + half - back) : get_part<T>(p.x + half, have);
    };
    Place now = next();
    uint4 x{}, y{};
    fetch(now, x, y);  // under way while the angles are made
    for (int i = tid; i < tile * half; i += kBlock) {
        const int of = i / half;
        if (tokens[of] < 0) continue;
        float2 cs = turned(double(positions[of]) * (a.frequencies[i - of * half] * 0.15915494309189535));
        if (a.backward) cs.y = -cs.y;
        table[i] = {cs.x * a.magnitude, cs.y * a.magnitude};
    }
    __syncthreads();
    while (now.t >= 0) {
        const Place then = next();
        uint4 x2{}, y2{};
        fetch(then, x2, y2);
        if (front) x = moved_down<T>(x, front);
        if (pairs && back) y = moved_down<T>(y, back);
        const float2 *const row = table + now.t * half;
        float p[G], q[G];
        T::unpack(x, p);
        if constexpr (INTERLEAVED) {
#pragma unroll
            for (int e = 0; e < G; e += 2) {
                const float2 cs = row[max(0, min(at + e, a.rotary - 2)) / 2];
                const float v = p[e], w = p[e + 1];
                p[e] = v * cs.x - w * cs.y;
                p[e + 1] = w * cs.x + v * cs.y;
            }
            uint4 turned = T::pack(p);
            if (at + G > a.rotary) {  // some channels stay: whole words, for pairs turn
                const int words = (a.rotary - at) * int(sizeof(Raw)) / 4;
                turned = {words > 0 ? turned.x : x.x, words > 1 ? turned.y : x.y, words > 2 ? turned.z : x.z,
                          words > 3 ? turned.w : x.w};
            }
            store<T, STREAM>(now.o, have, turned);
        } else if (pairs) {
            T::unpack(y, q);
#pragma unroll
            for (int e = 0; e < G; ++e) {
                const float2 cs = row[min(at + e, half - 1)];
                const float v = p[e], w = q[e];
                p[e] = v * cs.x - w * cs.y;
                q[e] = w * cs.x + v * cs.y;
            }
            store<T, STREAM>(now.o, have, T::pack(p));
            store<T, STREAM>(now.o + half, have, T::pack(q));
        } else {
            store<T, STREAM>(now.o, have, x);
        }
        now = then;
        x = x2;
        y = y2;
    }
}

template <class T>
void launch(const RopeArgs &a, hipStream_t stream) {
    constexpr int G = T::kGroup;
    const int half = a.rotary / 2;
    const bool interleaved = a.interleaved || a.rotary == 2;  // one pair is the same in both
    bool same = true;  // what stays is there already
    for (const RopeSide &s : a.side)
        if (s.heads)
            same = same && s.x == s.out && s.xs.s[0] == s.os.s[0] && s.xs.s[1] == s.os.s[1] && s.xs.s[2] == s.os.s[2];
    const int turning = ((interleaved ? a.rotary : half) + G - 1) / G;
    const int items = same            ? turning
                      : interleaved   ? (a.width + G - 1) / G
                                      : turning + (a.width - a.rotary + G - 1) / G;
    if (items == 0) return;  // at most kBlock, for every width and rotary
    // Two or three heads a thread, where there are tokens enough for that: 32768 tokens of 40
    // heads of 128 BF16 took 128 us with 2 tokens a workgroup (2.5 heads), 142 with 1, 139
    // with 8 and 152 with 16; past the caches 121, with loads ahead 116 (5.8 TB/s).
    const int64_t tokens = int64_t(a.batch) * a.count, heads = a.side[0].heads + a.side[1].heads;
    const int slots = kBlock / items, most = half ? std::min(kTokens, kPairs / half) : kTokens;
    const int tile = int(std::max<int64_t>(1, std::min<int64_t>({tokens / 1024, 5 * slots / (2 * heads), most})));
    const dim3 grid(unsigned((tokens + tile - 1) / tile));
    const bool past = double(tokens) * double(heads) * a.width * sizeof(typename T::Raw) > kCached;
    if (interleaved && past)
        rope_kernel<T, true, true><<<grid, kBlock, 0, stream>>>(a, tile, items, slots);
    else if (interleaved)
        rope_kernel<T, true, false><<<grid, kBlock, 0, stream>>>(a, tile, items, slots);
    else if (past)
        rope_kernel<T, false, true><<<grid, kBlock, 0, stream>>>(a, tile, items, slots);
    else
        rope_kernel<T, false, false><<<grid, kBlock, 0, stream>>>(a, tile, items, slots);
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
