// Operators on device buffers that the caller owns: the 8-bit KV cache with
// its attention (kv8.hip, kv8_attn.hip), the log probabilities of tokens with
// their gradient (logprobs.hip), sampling with filters (sample.hip), rotary
// positions (rope.hip) and the root-mean-square norm (norm.hip).  Host code
// (operators.cpp, step_operators.cpp, model.cpp) calls only these.
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>

namespace meshgpt {

enum class Type : int { F32 = 0, F16 = 1, BF16 = 2 };
inline size_t type_size(Type t) { return t == Type::F32 ? 4 : 2; }

constexpr int kKv8Tile = 64;   // tokens of a tile of transposed values
constexpr int kKv8Block = 16;  // tokens that share a scale

// An 8-bit KV cache.  Keys are [batch][heads][capacity][pad] and values
// [batch][heads][capacity / 64][pad][64] in E4M3 codes; the scale of 16 tokens
// of a head is 2^(byte - 127), [batch][heads][capacity / 16].
struct Kv8 {
    int batch, heads, width, pad, capacity;
    uint8_t *k, *v, *ks, *vs;
};
// The head width of the cache's rows: 32, 64, 128 or 256.
inline int kv8_pad(int width) { return width <= 32 ? 32 : width <= 64 ? 64 : width <= 128 ? 128 : 256; }

// Element (sequence, token, head, d) of a tensor lies at
// sequence * s[0] + token * s[1] + head * s[2] + d.
struct Strides {
    int64_t s[3];
};

namespace kern {

struct Kv8AppendArgs {
    Kv8 cache;
    const void *k, *v;
    Strides ks, vs;
    const int *lengths;  // tokens of each sequence, the new ones among them
    const int *counts;   // new tokens of each sequence (null: count)
    int count;
    int absolute;  // 1: token i of the inputs is position i of the sequence, 0: the first new token is token 0
    int aligned;   // of inputs and strides: 16 bytes, 4, or 0 for less
};
void kv8_append(const Kv8AppendArgs &a, Type type, hipStream_t stream);
// Workgroups of an append: a run of n tokens touches at most (n + 126) / 64 tiles.
inline size_t kv8_append_workgroups(size_t pairs, size_t count) { return 2 * pairs * ((count + 126) / kKv8Tile); }
// Workgroups of a launch at most: it counts its threads, 256 each, in 32 bits.
constexpr size_t kLaunchMost = (size_t(1) << 24) - 1;

struct Kv8ReadArgs {
    Kv8 cache;
    void *k, *v;
    Strides ks, vs;
    const int *lengths;  // positions behind a sequence's own are not written (null: all are)
    int first, count;
    int aligned;   // as above, of the outputs
};
void kv8_read(const Kv8ReadArgs &a, Type type, hipStream_t stream);

struct Kv8AttnArgs {
    Kv8 cache;
    const void *q;
    void *out;  // null: only the partial states are wanted
    Strides qs, os;
    const int *lengths, *counts;
    int count, group;  // queries of a sequence at most; query heads that share a cached head
    int rows;          // count * group
    float scale_log2;  // of the scores, times log2(e)
    int splits;        // shares of the keys
    int least;         // tiles of 64 keys of a share, at least
    // With out null or splits > 1: share s of row r of (sequence, head) p leaves
    // its unnormalised output, maximum (log2 units) and sum at
    // part[((p * rows + r) * splits + s) * stride + {d, stride - 2, stride - 1}].
    float *part;
    int stride;
    int q_aligned, o_aligned;
};
// Floats of a share's state: 16-byte groups, the last two elements the maximum
// and the sum.
inline int kv8_part_stride(int pad) { return pad + 4; }
// How a call is cut: the rows of a workgroup and the shares of the keys.
struct Kv8Plan {
    bool wide;  // a wave has rows of its own; else the waves share a workgroup's rows and split its keys
    int row_tiles, splits, least;
    size_t part_floats;
};
Kv8Plan kv8_plan(const Kv8 &cache, Type type, int group, int count);
void kv8_attention(const Kv8AttnArgs &a, Type type, const Kv8Plan &plan, hipStream_t stream);

struct LogprobArgs {
    const void *logits;
    size_t rows, vocab, stride;
    const uint32_t *tokens;
    float inv_temperature;
    float *logprob, *entropy, *stats;  // null: not wanted
    int top;
    uint32_t *top_tokens;
    float *top_logprobs;
    // Rows in several chunks: each one's maximum, sums and best tokens.
    int chunks, chunk;
    float *part_stats;   // [rows][chunks][3]
    uint64_t *part_top;  // [rows][chunks][top]
};
// Chunks of a row and their length (chunks == 1: no workspace).
void logprob_chunks(size_t rows, size_t vocab, int &chunks, int &chunk);
void token_logprobs(const LogprobArgs &a, Type type, hipStream_t stream);

struct LogprobBackwardArgs {
    const void *logits;
    size_t rows, vocab, stride;
    const uint32_t *tokens;
    float inv_temperature;
    const float *stats, *entropy, *d_logprob, *d_entropy;
    void *d_logits;
    size_t d_stride;
};
void token_logprobs_backward(const LogprobBackwardArgs &a, Type type, hipStream_t stream);

struct SampleArgs {
    const void *logits;
    size_t rows, vocab, stride;
    // One a row; null: temperature 1, no filter.
    const float *temperatures;
    const int *top_k;
    const float *top_p, *min_p;
    const float *uniforms;
    uint32_t *tokens;
    float *logprob;  // null: not wanted
};
void sample_filtered(const SampleArgs &a, Type type, hipStream_t stream);
// A model's step: `batch` rows of F32 logits drawn with one set of filters, a number of
// rng[r] each (advanced in place), the tokens appended at len[r].  scratch holds
// kSampledBytes a row.  flags[0] becomes 1 where a row holds a non-finite logit.
constexpr size_t kSampledBytes = 24;
void sample_step(const float *logits, size_t vocab, size_t batch, float temperature, uint32_t top_k, float top_p,
                 float min_p, uint64_t *rng, void *scratch, uint32_t *tokens, int token_stride, int *len, int *flags,
                 hipStream_t stream);

struct RopeSide {  // queries or keys
    const void *x;
    void *out;
    Strides xs, os;
    int heads;
};
struct RopeArgs {
    RopeSide side[2];
    const double *frequencies;  // radians a position, of each pair
    float magnitude;
    const int *lengths, *counts, *positions;  // null: none, `count` each, by the lengths
    int batch, count, width, rotary;
    bool interleaved, backward;
};
void rope(const RopeArgs &a, Type type, hipStream_t stream);

struct NormArgs {
    const void *x, *residual;  // residual null: none
    void *sum;                 // null: not kept
    const void *weight;        // null: 1
    void *out;                 // null: codes are wanted
    uint8_t *codes, *scales;
    float *rstd;  // null: not wanted
    size_t rows, xs, rs, ss, os, scs;
    int width;
    float epsilon;
};
void rms_norm(const NormArgs &a, Type type, hipStream_t stream);

struct NormBackwardArgs {
    const void *x, *weight, *d_out, *d_sum;  // weight and d_sum may be null
    const float *rstd;
    void *d_x;
    float *d_weight, *part;  // null: not wanted; parts x width
    size_t rows, xs, dos, dss, dxs;
    int width;
};
// Partial sums of the weight's gradient that a call makes.
size_t norm_parts(size_t rows, size_t width);
void rms_norm_backward(const NormBackwardArgs &a, Type type, hipStream_t stream);
constexpr size_t kNormWidth = 16384;  // at most

constexpr int kTopMax = 32;
constexpr int kSmallVocab = 1024;  // rows of so many logits take a wave, longer ones workgroups
constexpr int kGradRun = 736;      // F32 logits of a gradient's wave (twice as many in 16 bits)

}  // namespace kern

// The checked entry points (operators.cpp): work on `stream` of `device`,
// enqueued and not waited for; the caller's current device is restored.
void kv8_check(const Kv8 &cache);
size_t kv8_code_bytes(const Kv8 &cache);
size_t kv8_scale_bytes(const Kv8 &cache);
void kv8_append(int device, const Kv8 &cache, Type type, size_t count, const void *k, Strides ks, const void *v,
                Strides vs, const int *lengths, const int *counts, hipStream_t stream);
void kv8_read(int device, const Kv8 &cache, Type type, size_t first, size_t count, void *k, Strides ks, void *v,
              Strides vs, const int *lengths, hipStream_t stream);
size_t kv8_attention_workspace(const Kv8 &cache, size_t heads, size_t count);
void kv8_attention(int device, const Kv8 &cache, Type type, size_t heads, size_t count, const void *q, Strides qs,
                   void *out, Strides os, const int *lengths, const int *counts, float scale, void *workspace,
                   size_t workspace_bytes, hipStream_t stream);

size_t token_logprobs_workspace(size_t rows, size_t vocab, size_t top);
void token_logprobs_noalloc(int device, Type type, const void *logits, size_t rows, size_t vocab, size_t stride,
                            const uint32_t *tokens, float temperature, float *logprob, float *entropy, float *stats,
                            size_t top, uint32_t *top_tokens, float *top_logprobs, void *workspace,
                            size_t workspace_bytes, hipStream_t stream);
void token_logprobs_backward_noalloc(int device, Type type, const void *logits, size_t rows, size_t vocab,
                                     size_t stride, const uint32_t *tokens, float temperature, const float *stats,
                                     const float *entropy, const float *d_logprob, const float *d_entropy,
                                     void *d_logits, size_t d_stride, hipStream_t stream);
// On host arrays of f32 logits.
void token_logprobs(int device, const float *logits, size_t rows, size_t vocab, const uint32_t *tokens,
                    float temperature, float *logprob, float *entropy, size_t top, uint32_t *top_tokens,
                    float *top_logprobs);

// step_operators.cpp
void sample_filtered_noalloc(int device, Type type, const void *logits, size_t rows, size_t vocab, size_t stride,
                             const float *temperatures, const int *top_k, const float *top_p, const float *min_p,
                             const float *uniforms, uint32_t *tokens, float *logprob, hipStream_t stream);

struct Rope {
    size_t width, rotary;
    bool interleaved;
    float magnitude;
    const double *frequencies;
};
enum class RopeScaling : int { None = 0, Linear = 1, Base = 2, Bands = 3 };
void rope_frequencies(size_t rotary, double base, RopeScaling scaling, double factor, double context, double low,
                      double high, double *out);
void rope(int device, const Rope &r, Type type, size_t batch, size_t count, size_t heads, const void *q, Strides qs,
          void *q_out, Strides qos, size_t kv_heads, const void *k, Strides ks, void *k_out, Strides kos,
          const int *lengths, const int *counts, const int *positions, bool backward, hipStream_t stream);

// out, or codes and scales.
void rms_norm(int device, Type type, size_t rows, size_t width, const void *x, size_t x_stride, const void *residual,
              size_t residual_stride, void *sum, size_t sum_stride, const void *weight, float epsilon, void *out,
              size_t out_stride, float *rstd, hipStream_t stream);
void rms_norm_e4m3(int device, Type type, size_t rows, size_t width, const void *x, size_t x_stride,
                   const void *residual, size_t residual_stride, void *sum, size_t sum_stride, const void *weight,
                   float epsilon, uint8_t *codes, size_t codes_stride, uint8_t *scales, size_t scales_stride,
                   float *rstd, hipStream_t stream);
size_t rms_norm_backward_workspace(size_t rows, size_t width);
void rms_norm_backward(int device, Type type, size_t rows, size_t width, const void *sum, size_t sum_stride,
                       const void *weight, const float *rstd, const void *d_out, size_t d_out_stride, const void *d_sum,
                       size_t d_sum_stride, void *d_x, size_t d_x_stride, float *d_weight, void *workspace,
                       size_t workspace_bytes, hipStream_t stream);

}  // namespace meshgpt
