// Causal attention over the 8-bit KV cache: o_i = sum_j softmax_j(scale q_i.k_j) v_j
// over the keys j at or before query i's position.
//
// Every product runs on the BF16 matrix cores.  An E4M3 code is exact in BF16,
// so keys and values go there as codes, two an instruction, and their scales
// meet the scores in FP32 and the values, exactly, in their conversion.  Queries
// go there exactly: as one BF16 (BF16 calls), two (F16) or three (F32).
// Probabilities go there as two in 16-bit calls, which leaves 2^-16 of each, or as
// three in F32 calls, which leaves nothing.  Each piece is a product of its own.
// One BF16 would leave 2^-8 of each probability, as much as the output's own
// rounding: BF16 calls were then off by 0.0023 against 64 bits (root mean square),
// by 0.0017 with two, which is the output's rounding.  The second piece takes nothing
// where memory bounds (64 sequences of 2000 to 16000 tokens, 32 heads over 8 of 128:
// 229 us either way) and a third more where products do (4 prompts of 4096: 575 us
// with one, 758 with two).  Scores, maxima, sums and outputs are FP32.
//
// A wave takes tiles of 64 keys for 16 query rows at a time (few rows,
// kv8_rows_kernel) or 32 (prompts, kv8_tiles_kernel); query heads that share a
// cached head are rows of the same tile.  The scores are computed transposed,
// S^T = K Q^T: a lane then holds 16 keys of one row, all of them in one block of 16
// tokens, when the rows of K are taken in the right order: of 16 rows 16 (m / 4) +
// 4 t + m % 4 for matrix row m of product t, of 32 rows 16 (m / 4 % 2) + 4 (m / 8) +
// m % 4 for row m.  So one scale of the keys and one of the values serve a lane, the
// maximum needs two lane exchanges (one), and the probabilities are where the second
// product, O^T = V^T P^T, takes them: nothing moves between lanes.  Its values come
// in 16-byte loads because the cache holds them transposed.  The sums of 16 rows are
// a product with ones, those of 32 are added in each lane and exchanged once at the
// end.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "lds_dma.hpp"
#include "operators.hpp"
#include "types.hpp"

namespace meshgpt::kern {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kWaves = 4;

// Pieces of a query and of a probability in BF16.
template <class T>
constexpr int kQueryPieces = sizeof(typename T::Raw) == 4 ? 3 : 1;
template <>
constexpr int kQueryPieces<F16> = 2;
template <class T>
constexpr int kProbPieces = sizeof(typename T::Raw) == 4 ? 3 : 2;

__device__ __forceinline__ float bits(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ uint32_t bits(float f) { return __builtin_bit_cast(uint32_t, f); }
__device__ __forceinline__ float power(int byte) { return bits(uint32_t(byte) << 23); }

// Codes times a power of two as BF16.
template <bool HIGH>
__device__ __forceinline__ uint32_t codes2(uint32_t w, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HIGH));
}
__device__ __forceinline__ bf16x8 codes8(uint32_t a, uint32_t b, float scale = 1.0f) {
    return __builtin_bit_cast(bf16x8, u32x4{codes2<false>(a, scale), codes2<true>(a, scale), codes2<false>(b, scale),
                                            codes2<true>(b, scale)});
}

// x as a sum of NP BF16 values: all but the last cut off, the last rounded
// (and exact, for the third of an f32).
template <int NP>
__device__ __forceinline__ void pieces8(const float (&x)[8], bf16x8 (&out)[NP]) {
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
    for (int p = 0; p + 1 < NP; ++p) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = __builtin_amdgcn_perm(bits(r[2 * i + 1]), bits(r[2 * i]), 0x07060302);  // the two high halves
            r[2 * i] -= bits(bits(r[2 * i]) & 0xffff0000u);
            r[2 * i + 1] -= bits(bits(r[2 * i + 1]) & 0xffff0000u);
        }
        out[p] = __builtin_bit_cast(bf16x8, w);
    }
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{r[2 * i], r[2 * i + 1]}, bf16x2));
    out[NP - 1] = __builtin_bit_cast(bf16x8, w);
}

// The largest of the four lanes that hold a row.
__device__ __forceinline__ float row_max(float v) {
    const auto s = __builtin_amdgcn_permlane16_swap(int(bits(v)), int(bits(v)), false, false);
    v = fmaxf(bits(uint32_t(s[0])), bits(uint32_t(s[1])));
    const auto t = __builtin_amdgcn_permlane32_swap(int(bits(v)), int(bits(v)), false, false);
    return fmaxf(bits(uint32_t(t[0])), bits(uint32_t(t[1])));
}

// Rows keep a maximum that their scores may pass by up to 2^kSlack before sums
// and outputs are brought to a new one: nearly no tile after the first does, and
// nothing is lost, for probabilities are floating point.  Values past 2^80 take
// no slack: it would bring sums over 2^24 of them near the end of FP32's range.
constexpr float kSlack = 8.0f;
constexpr int kSlackByte = 127 + 80;

// The probabilities of a row's 16 scores in this lane against the row's maximum
// m (log2 units), as pieces.  Returns the factor that earlier sums and outputs
// take.  With `masked` only keys at or before `place` count, and the scores of
// the others may be anything.
template <int NP>
__device__ __forceinline__ float soften(f32x4 (&st)[4], bool masked, float kscale, float slack, int key0, int place,
                                        float &m, bf16x8 (&pf)[NP][2]) {
    if (masked) {
        __builtin_amdgcn_sched_barrier(0);  // a branch: few tiles are masked
#pragma unroll
        for (int j = 0; j < 16; ++j)  // scaled first: the scale may be 0, or anything where no key counts
            st[j / 4][j % 4] = key0 + j > place ? -INFINITY : st[j / 4][j % 4] * kscale;
        kscale = 1.0f;
    }
    float top = st[0][0];
#pragma unroll
    for (int j = 1; j < 16; ++j) top = fmaxf(top, st[j / 4][j % 4]);
    top = row_max(top * kscale);
    float drop = 1.0f;
    if (__any(top > m + slack)) {
        const float next = fmaxf(m, top);
        drop = __builtin_amdgcn_exp2f(m - (next == -INFINITY ? 0.0f : next));
        m = next;
    }
    // A row that has seen no key yet keeps -inf; 0 stands for it.
    const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            x[j] = __builtin_amdgcn_exp2f(fmaf(st[2 * h + j / 4][j % 4], kscale, -base));
        bf16x8 piece[NP];
        pieces8<NP>(x, piece);
#pragma unroll
        for (int p = 0; p < NP; ++p) pf[p][h] = piece[p];
    }
    return drop;
}

// A block's scale of the values, 1 behind the sequence, where the byte may be
// anything; and what scores may pass the maximum by with it.
__device__ __forceinline__ float value_scale(int byte, int key0, int length) {
    return key0 < length ? power(byte) : 1.0f;
}
__device__ __forceinline__ float slack_of(int byte) { return byte > kSlackByte ? 0.0f : kSlack; }

// The sums of the probabilities are a product with ones: row n's lands in every
// element of its lanes.
template <int NP>
__device__ __forceinline__ f32x4 add_sums(const bf16x8 (&pf)[NP][2], f32x4 l) {
    const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
#pragma unroll
    for (int p = NP - 1; p >= 0; --p)
#pragma unroll
        for (int h = 0; h < 2; ++h) l = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pf[p][h], l, 0, 0, 0);
    return l;
}

// A NaN value times a probability of 0 would reach rows that do not see its
// token.  So tiles that some row does not see whole are weighed with their NaN
// codes taken out (what lies behind a sequence may hold any), and where there
// were some, the outputs of the rows that see them are made NaN at the end.

// Bytes of a word that are NaN codes, as 1 each.
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) {
    return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
}
// Takes them out; the words in which there were some.
__device__ __forceinline__ uint32_t clean(uint4 &v) {
    const uint32_t x = nan_codes(v.x), y = nan_codes(v.y), z = nan_codes(v.z), w = nan_codes(v.w);
    v.x &= ~(x * 0xffu);
    v.y &= ~(y * 0xffu);
    v.z &= ~(z * 0xffu);
    v.w &= ~(w * 0xffu);
    return x | y | z | w;
}
// acc = NaN where a row sees a NaN of the tile: a product of the places
// of the NaN codes with those that a row sees counts them.
template <int PAD>
__device__ __forceinline__ void mark_nan(const uint8_t *vpair, int tile, int lane, int place, f32x4 (&acc)[PAD / 16]) {
    const int n = lane & 15, g = lane >> 4;
    const uint8_t *const vt = vpair + size_t(tile) * 64 * PAD + n * 64 + 16 * g;
#pragma unroll
    for (int d = 0; d < PAD / 16; ++d) {
        const uint4 v = *reinterpret_cast<const uint4 *>(vt + d * 16 * 64);
        // 0x38 is the code of 1.
        const u32x4 one{nan_codes(v.x) * 0x38u, nan_codes(v.y) * 0x38u, nan_codes(v.z) * 0x38u, nan_codes(v.w) * 0x38u};
        f32x4 hits{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            u32x4 see;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int key = tile * 64 + 16 * g + 8 * h + 2 * e;
                see[e] = (key <= place ? 0x3f80u : 0u) | (key + 1 <= place ? 0x3f800000u : 0u);
            }
            hits = __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes8(one[2 * h], one[2 * h + 1]),
                                                           __builtin_bit_cast(bf16x8, see), hits, 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (hits[e] > 0.0f) acc[d][e] = __builtin_nanf("");
    }
}

// The sequence of a pair (sequence, cached head), and whether its length and
// count are possible.
struct Sequence {
    int seq, head, length, count;
    bool valid;
    __device__ __forceinline__ Sequence(const Kv8AttnArgs &a, int pair) {
        seq = pair / a.cache.heads;
        head = pair - seq * a.cache.heads;
        length = a.lengths[seq];
        count = a.counts ? a.counts[seq] : a.count;
        valid = length >= 0 && length <= a.cache.capacity && count >= 0 && count <= a.count && count <= length;
        if (!valid) count = a.count;
    }
};

template <class T>
__device__ __forceinline__ typename T::Raw *out_row(const Kv8AttnArgs &a, const Sequence &s, int r) {
    const int i = r / a.group;
    return static_cast<typename T::Raw *>(a.out) + s.seq * a.os.s[0] + i * a.os.s[1] +
           (s.head * a.group + r - i * a.group) * a.os.s[2];
}

// Four outputs of a row from `at`, those inside the width.
template <class T>
__device__ __forceinline__ void store4(const Kv8AttnArgs &a, typename T::Raw *o, int at, f32x4 v) {
    if (a.o_aligned && at + 4 <= a.cache.width) {
        if constexpr (T::kGroup == 4) {
            *reinterpret_cast<f32x4 *>(o + at) = v;
        } else {
            const float x[8] = {v[0], v[1], v[2], v[3], 0.0f, 0.0f, 0.0f, 0.0f};
            const uint4 w = T::pack(x);
            *reinterpret_cast<uint2 *>(o + at) = uint2{w.x, w.y};
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (at + e < a.cache.width) o[at + e] = T::from_float(v[e]);
}

// Eight elements of a query from d as pieces, zeros where there are none.
template <class T>
__device__ __forceinline__ void query8(const Kv8AttnArgs &a, const typename T::Raw *q, bool real, int d,
                                       bf16x8 (&piece)[kQueryPieces<T>]) {
    float x[8];
    if (a.q_aligned && real && d + 8 <= a.cache.width) {
#pragma unroll
        for (int j = 0; j < 8 / T::kGroup; ++j) {
            float y[T::kGroup];
            T::unpack(reinterpret_cast<const uint4 *>(q + d)[j], y);
#pragma unroll
            for (int e = 0; e < T::kGroup; ++e) x[j * T::kGroup + e] = y[e];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = real && d + j < a.cache.width ? T::to_float(q[d + j]) : 0.0f;
    }
    pieces8<kQueryPieces<T>>(x, piece);
}

// The key tiles of a share for rows that see `keys` keys: equal shares, of a.least
// tiles or more.
struct Tiles {
    int first, last, each;
    __device__ __forceinline__ Tiles(const Kv8AttnArgs &a, int split, int keys) {
        const int tiles = (keys + 63) / 64;
        each = max(a.least, (tiles + a.splits - 1) / a.splits);
        first = split * each;
        last = min(tiles, first + each);
    }
};

template <class T>
__device__ __forceinline__ void fill_nan(const Kv8AttnArgs &a, const Sequence &s, int row0, int row_end, int from,
                                         int step) {
    for (int r = row0; r < row_end; ++r)
        for (int d = from; d < a.cache.width; d += step) out_row<T>(a, s, r)[d] = T::from_float(__builtin_nanf(""));
}

// Up to 16 rows of a pair a workgroup, as in single tokens: its waves take the
// key tiles in turn, straight from memory into operands, and join their states at
// the end.  The bytes of the cache bound it: 64 sequences of 2000 to 16000 tokens,
// 32 heads over 8 of 128, BF16, take 224 to 231 us (5.1 to 5.3 TB/s; each byte is
// fetched once, and the matrix units are busy for a ninth of the time).
template <class T, int PAD>
__global__ void __launch_bounds__(64 * kWaves) kv8_rows_kernel(Kv8AttnArgs a, int pairs) {
    constexpr int NQ = kQueryPieces<T>, NP = kProbPieces<T>, STEPS = PAD / 32, DT = PAD / 16;
    constexpr int WORDS = PAD >= 64 ? PAD / 16 : 2;  // 4-byte words of a key that a lane holds
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    const int id = int(blockIdx.x), pair = id % pairs, split = id / pairs % a.splits;
    const int row0 = id / pairs / a.splits * 16;
    const Sequence s(a, pair);
    const int rows = s.count * a.group, row_end = min(row0 + 16, rows);
    if (row0 >= rows) return;
    if (!s.valid) {
        if (a.out && a.splits == 1) fill_nan<T>(a, s, row0, row_end, int(threadIdx.x), 64 * kWaves);
        return;
    }
    const int begin = s.length - s.count;  // the first query's position
    const int seen = begin + row0 / a.group;
    const Tiles tiles(a, split, begin + (row_end - 1) / a.group + 1);
    if (tiles.first >= tiles.last && a.out) return;  // the join does not read it

    bf16x8 qf[NQ][STEPS];
    const int row = row0 + n, place = row < rows ? begin + row / a.group : -1;
    {
        const int i = row / a.group;
        const auto *q = static_cast<const typename T::Raw *>(a.q) + s.seq * a.qs.s[0] + i * a.qs.s[1] +
                        (s.head * a.group + row - i * a.group) * a.qs.s[2];
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
            bf16x8 piece[NQ];
            query8<T>(a, q, row < rows, PAD >= 64 ? 64 * (k / 2) + 16 * g + 8 * (k % 2) : 8 * g, piece);
#pragma unroll
            for (int p = 0; p < NQ; ++p) qf[p][k] = piece[p];
        }
    }

    const uint8_t *const kbase = a.cache.k + size_t(pair) * a.cache.capacity * PAD +
                                 (16 * (n >> 2) + (n & 3)) * PAD + (PAD >= 64 ? 16 : 8) * g;
    const uint8_t *const vbase = a.cache.v + size_t(pair) * a.cache.capacity * PAD + n * 64 + 16 * g;
    const uint8_t *const ksbase = a.cache.ks + size_t(pair) * (a.cache.capacity / 16) + g;
    const uint8_t *const vsbase = a.cache.vs + size_t(pair) * (a.cache.capacity / 16) + g;
    auto load_keys = [&](int tile, uint32_t (&k)[4][WORDS]) {
        const uint8_t *p = kbase + size_t(tile) * 64 * PAD;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if constexpr (PAD >= 64) {
#pragma unroll
                for (int c = 0; c < PAD / 64; ++c) {
                    const uint4 w = *reinterpret_cast<const uint4 *>(p + 4 * t * PAD + 64 * c);
                    k[t][4 * c] = w.x;
                    k[t][4 * c + 1] = w.y;
                    k[t][4 * c + 2] = w.z;
                    k[t][4 * c + 3] = w.w;
                }
            } else {
                const uint2 w = *reinterpret_cast<const uint2 *>(p + 4 * t * PAD);
                k[t][0] = w.x;
                k[t][1] = w.y;
            }
        }
    };

    float m = -INFINITY;
    f32x4 acc[DT], l{0.0f, 0.0f, 0.0f, 0.0f};
    uint32_t nans = 0;  // NaN codes were taken out
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    int tile = tiles.first + wave;
    uint32_t kw[4][WORDS];
    int kbyte = 0, vbyte = 0;
    if (tile < tiles.last) {
        load_keys(tile, kw);
        kbyte = ksbase[4 * tile];
        vbyte = vsbase[4 * tile];
    }
    for (; tile < tiles.last; tile += kWaves) {
        uint4 vw[DT];
        const uint8_t *const vt = vbase + size_t(tile) * 64 * PAD;
#pragma unroll
        for (int d = 0; d < DT; ++d) vw[d] = *reinterpret_cast<const uint4 *>(vt + d * 16 * 64);
        // The next tile's keys are under way during this one's products.
        const int next = min(tile + kWaves, tiles.last - 1);
        uint32_t kn[4][WORDS];
        load_keys(next, kn);
        const int kbyte_next = ksbase[4 * next], vbyte_next = vsbase[4 * next];

        f32x4 st[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            st[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < STEPS; ++k) {
                const bf16x8 kf = codes8(kw[t][2 * k], kw[t][2 * k + 1]);
#pragma unroll
                for (int p = NQ - 1; p >= 0; --p)
                    st[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[p][k], st[t], 0, 0, 0);
            }
        }
        const int key0 = tile * 64 + 16 * g;  // of the lane's 16 keys
        const bool masked = tile * 64 + 63 > seen;  // some row does not see all of the tile
        bf16x8 pf[NP][2];
        const float kscale = power(kbyte) * a.scale_log2, vscale = value_scale(vbyte, key0, s.length);
        const float drop = soften<NP>(st, masked, kscale, slack_of(vbyte), key0, place, m, pf);
        if (__any(drop != 1.0f)) {
            l *= drop;
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[d] *= drop;
        }
        l = add_sums<NP>(pf, l);
        if (masked) {
#pragma unroll
            for (int d = 0; d < DT; ++d) nans |= clean(vw[d]);
        }
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const bf16x8 vf = h ? codes8(vw[d].z, vw[d].w, vscale) : codes8(vw[d].x, vw[d].y, vscale);
#pragma unroll
                for (int p = NP - 1; p >= 0; --p)
                    acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[p][h], acc[d], 0, 0, 0);
            }
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int w = 0; w < WORDS; ++w) kw[t][w] = kn[t][w];
        kbyte = kbyte_next;
        vbyte = vbyte_next;
    }

    if (__any(nans != 0)) {
        // This wave's tiles from the first one masked.
        int from = tiles.first + wave;
        if (seen / 64 > from) from += (seen / 64 - from + kWaves - 1) / kWaves * kWaves;
        for (int t = from; t < tiles.last; t += kWaves)
            mark_nan<PAD>(a.cache.v + size_t(pair) * a.cache.capacity * PAD, t, lane, place, acc);
    }

    constexpr int PART = PAD < 128 ? PAD : 128;  // channels joined at a time
    __shared__ float wave_m[kWaves][16], wave_l[kWaves][16];
    __shared__ __align__(16) float wave_o[kWaves][16][PART + 4];
    if (g == 0) {
        wave_m[wave][n] = m;
        wave_l[wave][n] = l[0];
    }
    __syncthreads();
    float top = wave_m[0][n];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, wave_m[w][n]);
    const float base = top == -INFINITY ? 0.0f : top, mine = __builtin_amdgcn_exp2f(m - base);
    const int real = row_end - row0;
#pragma unroll
    for (int c = 0; c < PAD / PART; ++c) {
        if (c) __syncthreads();
#pragma unroll
        for (int d = 0; d < PART / 16; ++d)
            *reinterpret_cast<f32x4 *>(&wave_o[wave][n][16 * d + 4 * g]) = acc[c * (PART / 16) + d] * mine;
        __syncthreads();
        for (int i = int(threadIdx.x); i < real * PART; i += 64 * kWaves) {
            const int r = i / PART, d = i % PART, at = c * PART + d;
            float v = 0.0f, total = 0.0f, high = wave_m[0][r];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) high = fmaxf(high, wave_m[w][r]);
            const float from = high == -INFINITY ? 0.0f : high;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                v += wave_o[w][r][d];
                total += wave_l[w][r] * __builtin_amdgcn_exp2f(wave_m[w][r] - from);
            }
            if (a.out && a.splits == 1) {
                if (at < a.cache.width) out_row<T>(a, s, row0 + r)[at] = T::from_float(v / total);
            } else {
                float *o = a.part + ((size_t(pair) * a.rows + row0 + r) * a.splits + split) * a.stride;
                if (at < a.stride - 2) o[at] = v;
                if (at == 0) {
                    o[a.stride - 2] = high;
                    o[a.stride - 1] = total;
                }
            }
        }
    }
}

// The schedule of N operands read from LDS with NP products each: a few reads
// ahead of the products.
template <int N, int NP>
__device__ __forceinline__ void paced() {
    constexpr int AHEAD = N < 6 ? N : 6;
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, NP, 0);
        if (i + AHEAD < N) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
}

// As soften() and mark_nan() for the products of 32 x 32: a lane holds 16 keys of a
// row in each 32, one block of 16 tokens, and a row is two lanes.
template <int NP, int SUB>
__device__ __forceinline__ float soften32(f32x16 (&st)[SUB], bool masked, float (&kscale)[SUB], float slack,
                                          const int (&key0)[SUB], int place, float &m, float &l, bf16x8 (&pf)[SUB][NP][2]) {
    if (masked) {
        __builtin_amdgcn_sched_barrier(0);  // a branch: few tiles are masked
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
#pragma unroll
            for (int j = 0; j < 16; ++j) st[u][j] = key0[u] + j > place ? -INFINITY : st[u][j] * kscale[u];
            kscale[u] = 1.0f;
        }
    }
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
        float t = st[u][0];
#pragma unroll
        for (int j = 1; j < 16; ++j) t = fmaxf(t, st[u][j]);
        top = fmaxf(top, t * kscale[u]);
    }
    const auto both = __builtin_amdgcn_permlane32_swap(int(bits(top)), int(bits(top)), false, false);
    top = fmaxf(bits(uint32_t(both[0])), bits(uint32_t(both[1])));
    float drop = 1.0f;
    if (__any(top > m + slack)) {
        const float next = fmaxf(m, top);
        drop = __builtin_amdgcn_exp2f(m - (next == -INFINITY ? 0.0f : next));
        m = next;
        l *= drop;
    }
    const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = __builtin_amdgcn_exp2f(fmaf(st[u][8 * h + j], kscale[u], -base));
            l += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
            bf16x8 piece[NP];
            pieces8<NP>(x, piece);
#pragma unroll
            for (int p = 0; p < NP; ++p) pf[u][p][h] = piece[p];
        }
    return drop;
}

template <int PAD>
__device__ __forceinline__ void mark_nan32(const uint8_t *vpair, int from, int to, int lane, int place,
                                           f32x16 (&acc)[PAD / 32]) {
    for (int tile = from; tile < to; ++tile)
        for (int u = 0; u < 2; ++u) {
            const int key0 = tile * 64 + 32 * u + 16 * (lane >> 5);
            const uint8_t *const vt = vpair + size_t(tile) * 64 * PAD + (lane & 31) * 64 + 32 * u + 16 * (lane >> 5);
#pragma unroll
            for (int d = 0; d < PAD / 32; ++d) {
                const uint4 v = *reinterpret_cast<const uint4 *>(vt + d * 32 * 64);
                // 0x38 is the code of 1.
                const u32x4 one{nan_codes(v.x) * 0x38u, nan_codes(v.y) * 0x38u, nan_codes(v.z) * 0x38u,
                                nan_codes(v.w) * 0x38u};
                f32x16 hits{};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    u32x4 see;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = key0 + 8 * h + 2 * e;
                        see[e] = (key <= place ? 0x3f80u : 0u) | (key + 1 <= place ? 0x3f800000u : 0u);
                    }
                    hits = __builtin_amdgcn_mfma_f32_32x32x16_bf16(codes8(one[2 * h], one[2 * h + 1]),
                                                                   __builtin_bit_cast(bf16x8, see), hits, 0, 0, 0);
                }
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (hits[e] > 0.0f) acc[d][e] = __builtin_nanf("");
            }
        }
}

// Many rows of a pair a workgroup, as in prompts: every wave has 32 rows of its
// own, and the waves share the key tiles as BF16 in LDS.  Each converts its part of
// the next tile, which it has in registers since the tile before, into the other
// half of the LDS while the products run, so a code is converted once for 128 rows,
// with one barrier a tile; operands lie in LDS in the order of their readers, 16
// bytes a lane.  The products are of 32 x 32: the vector unit waits less for them
// than for 16 x 16 (beside as many exponentials a product of the same size took 12.9
// cycles against 22).  SUB times 32 keys are softened together, as the registers
// allow.  The matrix unit and the vector unit bound it, which two waves a SIMD hardly
// overlap: 4 prompts of 4096, 32 heads over 8 of 128, BF16, take 755 us, 1.09 PFLOP/s of
// the three products, with the matrix units busy for 52 % of the cycles and the
// vector units for about as many; 3 ragged ones of up to 1001 behind up to 500, 8
// heads of 64, F32 with three products each, 31 us.  Width 256 leaves one wave a SIMD
// and in F32 not registers enough even so: 48 of them are spilled (196 bytes a lane).
template <class T, int PAD, int SUB>
__global__ void __launch_bounds__(64 * kWaves, PAD == 256 ? 1 : 2)
kv8_tiles_kernel(Kv8AttnArgs a, int pairs, int pairs8, int row_tiles) {
    constexpr int NQ = kQueryPieces<T>, NP = kProbPieces<T>, DT = PAD / 32, ROWS = 32 * kWaves;
    // A tile's groups: 64 lanes' 16 codes of the keys (32 u + ..., 32 c + ...), then
    // of the values; in LDS two operands of 8 elements for each lane.
    static_assert(kWaves == 4, "two waves take the keys, two the values");
    __shared__ bf16x8 lds[2][4 * DT][2][64];
    __shared__ uint32_t nans;  // NaN codes were taken out
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, g = lane >> 5;
    // Workgroups of a pair lie 8 apart, on one XCD and its L2; long rows first.
    const int id = int(blockIdx.x), pair = id % pairs8;
    if (pair >= pairs) return;
    const int split = id / pairs8 % a.splits, tile0 = row_tiles - 1 - id / pairs8 / a.splits;
    const Sequence s(a, pair);
    const int rows = s.count * a.group, block0 = tile0 * ROWS, block_end = min(block0 + ROWS, rows);
    if (block0 >= rows) return;
    if (!s.valid) {
        if (a.out && a.splits == 1) fill_nan<T>(a, s, block0, block_end, int(threadIdx.x), 64 * kWaves);
        return;
    }
    const int begin = s.length - s.count;  // the first query's position
    const Tiles tiles(a, split, begin + (block_end - 1) / a.group + 1);
    if (tiles.first >= tiles.last) return;  // the join does not read it
    const int row0 = block0 + 32 * wave, row_end = min(row0 + 32, rows);
    const int seen = begin + row0 / a.group;
    const int cleaned = (begin + block0 / a.group) / 64;  // the first tile that some row may not see whole
    if (threadIdx.x == 0) nans = 0;
    // The wave's own keys end earlier than the workgroup's.
    const int mine = row0 < rows ? (begin + (row_end - 1) / a.group + 64) / 64 : 0;

    const uint8_t *const kpair = a.cache.k + size_t(pair) * a.cache.capacity * PAD;
    const uint8_t *const vpair = a.cache.v + size_t(pair) * a.cache.capacity * PAD;
    // A wave takes the keys or the values of 32 tokens.
    const bool values = wave >= 2;
    const int half = wave & 1;
    const uint8_t *const from = values ? vpair + n * 64 + 32 * half + 16 * g
                                       : kpair + (32 * half + 16 * (n >> 2 & 1) + 4 * (n >> 3) + (n & 3)) * PAD + 16 * g;
    const int apart = values ? 32 * 64 : 32;
    uint4 raw[DT];
    auto load_tile = [&](int tile) {
#pragma unroll
        for (int v = 0; v < DT; ++v) raw[v] = *reinterpret_cast<const uint4 *>(from + size_t(tile) * 64 * PAD + v * apart);
    };
    auto convert_tile = [&](int tile, uint32_t vword) {
        float scale = 1.0f;
        if (values) {
            const int block = 2 * half + g;
            scale = value_scale(vword >> (8 * block) & 0xff, tile * 64 + 16 * block, s.length);
            if (tile >= cleaned) {
                uint32_t any = 0;
#pragma unroll
                for (int v = 0; v < DT; ++v) any |= clean(raw[v]);
                if (any) nans = 1;
            }
        }
#pragma unroll
        for (int v = 0; v < DT; ++v) {
            lds[tile & 1][wave * DT + v][0][lane] = codes8(raw[v].x, raw[v].y, scale);
            lds[tile & 1][wave * DT + v][1][lane] = codes8(raw[v].z, raw[v].w, scale);
        }
    };
    load_tile(tiles.first);

    bf16x8 qf[NQ][DT][2];
    const int r = row0 + n, place = r < rows ? begin + r / a.group : -1;
    {
        const int i = r / a.group;
        const auto *q = static_cast<const typename T::Raw *>(a.q) + s.seq * a.qs.s[0] + i * a.qs.s[1] +
                        (s.head * a.group + r - i * a.group) * a.qs.s[2];
#pragma unroll
        for (int c = 0; c < DT; ++c)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                bf16x8 piece[NQ];
                query8<T>(a, q, r < rows, 32 * c + 16 * g + 8 * k, piece);
#pragma unroll
                for (int p = 0; p < NQ; ++p) qf[p][c][k] = piece[p];
            }
    }
    float m = -INFINITY, l = 0.0f;
    f32x16 acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = f32x16{};
    // Four scales of a tile are a word that all lanes read.
    typedef const __attribute__((address_space(4))) uint32_t *Words;
    const Words kscales = (Words)(a.cache.ks + size_t(pair) * (a.cache.capacity / 16));
    const Words vscales = (Words)(a.cache.vs + size_t(pair) * (a.cache.capacity / 16));

    uint32_t kword = kscales[tiles.first], vword = vscales[tiles.first];
    __syncthreads();  // nans is cleared
    convert_tile(tiles.first, vword);
    if (tiles.first + 1 < tiles.last) load_tile(tiles.first + 1);
    vword = vscales[min(tiles.first + 1, tiles.last - 1)];
    for (int tile = tiles.first; tile < tiles.last; ++tile) {
        barrier_lds();  // this tile is there, and everyone past the one before
        const uint32_t kbytes = kword, vbytes = vscales[tile];
        if (tile + 1 < tiles.last) {
            convert_tile(tile + 1, vword);
            kword = kscales[tile + 1];
            if (tile + 2 < tiles.last) {
                load_tile(tile + 2);
                vword = vscales[tile + 2];
            }
        }
        const auto &now = lds[tile & 1];
        if (tile >= mine) continue;
        const bool masked = tile * 64 + 63 > seen;
#pragma unroll
        for (int step = 0; step < 2; step += SUB) {
            f32x16 st[SUB];
#pragma unroll
            for (int u = 0; u < SUB; ++u) st[u] = f32x16{};
#pragma unroll
            for (int c = 0; c < DT; ++c)
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int u = 0; u < SUB; ++u) {
                        const bf16x8 kf = now[(step + u) * DT + c][k][lane];
#pragma unroll
                        for (int p = NQ - 1; p >= 0; --p)
                            st[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[p][c][k], st[u], 0, 0, 0);
                    }
            paced<2 * DT * SUB, NQ>();
            int key0[SUB];  // of the lane's 16 keys
            float kscale[SUB], slack = kSlack;
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                const int at = 8 * (2 * (step + u) + g), vbyte = vbytes >> at & 0xff;
                key0[u] = tile * 64 + 32 * (step + u) + 16 * g;
                kscale[u] = power(kbytes >> at & 0xff) * a.scale_log2;
                slack = fminf(slack, slack_of(vbyte));
            }
            bf16x8 pf[SUB][NP][2];
            const float drop = soften32<NP, SUB>(st, masked, kscale, slack, key0, place, m, l, pf);
            if (__any(drop != 1.0f)) {
#pragma unroll
                for (int d = 0; d < DT; ++d) acc[d] *= drop;
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        const bf16x8 vf = now[2 * DT + (step + u) * DT + d][h][lane];
#pragma unroll
                        for (int p = NP - 1; p >= 0; --p)
                            acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf[u][p][h], acc[d], 0, 0, 0);
                    }
            paced<2 * DT * SUB, NP>();
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (tiles.last > cleaned && nans)
        mark_nan32<PAD>(vpair, max(tiles.first, cleaned), min(tiles.last, mine), lane, place, acc);
    const auto both = __builtin_amdgcn_permlane32_swap(int(bits(l)), int(bits(l)), false, false);
    const float sum = bits(uint32_t(both[0])) + bits(uint32_t(both[1]));
    if (r >= rows) return;
    auto four = [&](int d, int e) { return f32x4{acc[d][4 * e], acc[d][4 * e + 1], acc[d][4 * e + 2], acc[d][4 * e + 3]}; };
    if (a.splits == 1) {
        auto *o = out_row<T>(a, s, r);
        const float inverse = 1.0f / sum;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) store4<T>(a, o, 32 * d + 8 * e + 4 * g, four(d, e) * inverse);
    } else {
        float *o = a.part + ((size_t(pair) * a.rows + r) * a.splits + split) * a.stride;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) *reinterpret_cast<f32x4 *>(o + 32 * d + 8 * e + 4 * g) = four(d, e);
        if (g == 0) {
            o[a.stride - 2] = m;
            o[a.stride - 1] = sum;
        }
    }
}

// Joins the shares of a row: a lane takes four of its channels.  5 us for 64 x 32
// rows of 128, 6 for 24000 of 64.
template <class T, int PAD>
__global__ void __launch_bounds__(256) kv8_join_kernel(Kv8AttnArgs a, int64_t total, int row_step) {
    constexpr int LANES = PAD / 4;
    const int64_t u = int64_t(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES;
    const int d = 4 * (threadIdx.x % LANES);
    if (u >= total) return;
    const int pair = int(u / a.rows), r = int(u - int64_t(pair) * a.rows);
    const Sequence s(a, pair);
    if (r >= s.count * a.group) return;
    auto *o = out_row<T>(a, s, r);
    f32x4 out;
    if (s.valid) {
        // The shares of this row's tile of rows reach to the tile's last row;
        // those past this row's own keys hold nothing of it.
        const int begin = s.length - s.count, end = min((r / row_step + 1) * row_step, s.count * a.group);
        const int each = Tiles(a, 0, begin + (end - 1) / a.group + 1).each;
        const int used = ((begin + r / a.group + 64) / 64 + each - 1) / each;
        const float *p = a.part + size_t(u) * a.splits * a.stride;
        float m = -INFINITY, l = 0.0f;
        f32x4 acc{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int k = 0; k < used; ++k, p += a.stride) {
            const f32x4 v = *reinterpret_cast<const f32x4 *>(p + d);
            const float mk = p[a.stride - 2], lk = p[a.stride - 1], top = fmaxf(m, mk);
            const float base = top == -INFINITY ? 0.0f : top;
            const float old = __builtin_amdgcn_exp2f(m - base), now = __builtin_amdgcn_exp2f(mk - base);
            acc = acc * old + v * now;
            l = l * old + lk * now;
            m = top;
        }
        out = acc * (1.0f / l);
    } else {
        out = f32x4{} + __builtin_nanf("");
    }
    store4<T>(a, o, d, out);
}

template <class T, int PAD>
void launch_attn(const Kv8AttnArgs &a, const Kv8Plan &plan, hipStream_t stream) {
    const int pairs = a.cache.batch * a.cache.heads;
    if (plan.wide) {
        constexpr int SUB = PAD <= 64 || (PAD == 128 && kQueryPieces<T> == 1) ? 2 : 1;
        const int pairs8 = (pairs + 7) / 8 * 8;
        hipLaunchKernelGGL((kv8_tiles_kernel<T, PAD, SUB>),
                           dim3(uint32_t(pairs8) * uint32_t(a.splits) * uint32_t(plan.row_tiles)), dim3(64 * kWaves), 0,
                           stream, a, pairs, pairs8, plan.row_tiles);
    } else {
        hipLaunchKernelGGL((kv8_rows_kernel<T, PAD>), dim3(uint32_t(pairs) * uint32_t(a.splits) * uint32_t(plan.row_tiles)),
                           dim3(64 * kWaves), 0, stream, a, pairs);
    }
    if (a.out && a.splits > 1)
        hipLaunchKernelGGL((kv8_join_kernel<T, PAD>), dim3(uint32_t((int64_t(pairs) * a.rows * (PAD / 4) + 255) / 256)),
                           dim3(256), 0, stream, a, int64_t(pairs) * a.rows, plan.wide ? 32 * kWaves : 16);
}

template <class T>
void attn_of(const Kv8AttnArgs &a, const Kv8Plan &plan, hipStream_t stream) {
    switch (a.cache.pad) {
    case 32: return launch_attn<T, 32>(a, plan, stream);
    case 64: return launch_attn<T, 64>(a, plan, stream);
    case 128: return launch_attn<T, 128>(a, plan, stream);
    default: return launch_attn<T, 256>(a, plan, stream);
    }
}

}  // namespace

Kv8Plan kv8_plan(const Kv8 &cache, Type type, int group, int count) {
    Kv8Plan p{};
    const int64_t rows = int64_t(count) * group;
    const int pairs = std::max(1, cache.batch * cache.heads);
    // Up to some rows the waves of a workgroup do better to split the keys of 16,
    // for all that several such workgroups read the same keys (us, split; not): 128 x
    // 8000 keys of 128, 20 rows BF16 90; 67, F16 89; 79, F32 91; 104, 64 rows BF16 163;
    // 96, F32 161; 153; 32 x 4000 keys of 64, 40 rows BF16 18.1; 22.7, F32 19.1; 25.9; 8 x
    // 16000, 64 rows BF16 20.3; 32.7.
    p.wide = rows > (cache.pad <= 64 ? 64 : type == Type::F32 ? 32 : 16);
    const int each = p.wide ? 32 * kWaves : 16;
    p.row_tiles = int((rows + each - 1) / each);
    const int64_t groups = int64_t(pairs) * p.row_tiles, tiles = cache.capacity / 64;
    if (p.wide) {
        // As many shares as the resident workgroups hold, two a CU, but one of width
        // 256 and three in F32 of width 64: fewer leave CUs without work, more go
        // over their rows' states again (us with 2; 3; 4; 5; 6 shares: 128 groups of
        // BF16 rows of 64, 4000 keys, 58.5; 54.3; 48.8; 50.6; 46.8, of F32 rows
        // 74.5; 72.5; 62.4; 63.4; 59.3; 152 of F16 rows of 128, 4000 keys, 102; 110;
        // 98; 99; 108; 64 of BF16 rows of 256, 1500 keys, 64.7; 53.4; 47.1; 61.0; 61.1).
        // The join is a launch of its own, some 6 us with what it waits for, so a
        // share is 4 tiles or more, and shares spare 10 or more (32 groups of
        // BF16 rows of 64, 1024 keys: 26.8 us in one, 18.9 in four; 256 of up to 1000:
        // 30.3 in one, 34.8 in two).
        const int64_t resident = 256 * (cache.pad == 256 ? 1 : cache.pad == 64 && type == Type::F32 ? 3 : 2);
        p.least = 4;
        p.splits = int(std::max<int64_t>(1, std::min(tiles / p.least, resident / groups)));
        if (tiles - tiles / p.splits < 10) p.splits = 1;
    } else {
        // Single tokens wait for memory, so they take up to 2048 workgroups; but a
        // share of 1024 keys or more (32 x 8 heads, up to 576 keys: 10.6 us in one
        // share, 16.6 in shares of 256), of width 256 of 512 (32 pairs of 4000 keys,
        // F16: 26.3 us, 29.4 in shares of 1024).
        p.least = cache.pad == 256 ? 8 : 16;
        p.splits = int(std::max<int64_t>(1, std::min<int64_t>({tiles / p.least, 256, (2048 + groups - 1) / groups})));
    }
    p.part_floats = p.splits > 1 ? size_t(pairs) * size_t(rows) * size_t(p.splits) * size_t(kv8_part_stride(cache.pad)) : 0;
    return p;
}

void kv8_attention(const Kv8AttnArgs &a, Type type, const Kv8Plan &plan, hipStream_t stream) {
    switch (type) {
    case Type::F32: return attn_of<F32>(a, plan, stream);
    case Type::F16: return attn_of<F16>(a, plan, stream);
    default: return attn_of<BF16>(a, plan, stream);
    }
}

}  // namespace meshgpt::kern
