// The checked entry points of the operators on device buffers: arguments are
// looked at, the work is enqueued on the caller's stream, and the caller's
// current device is what it was.
#include "operators_host.hpp"

#include <algorithm>
#include <cmath>

namespace meshgpt {
namespace {

class Buffer {
  public:
    explicit Buffer(size_t bytes) { check(hipMalloc(&p_, std::max<size_t>(bytes, 16)), "hipMalloc"); }
    ~Buffer() { (void)hipFree(p_); }
    Buffer(const Buffer &) = delete;
    Buffer &operator=(const Buffer &) = delete;
    template <class T>
    T *as() const {
        return static_cast<T *>(p_);
    }

  private:
    void *p_ = nullptr;
};

void check_count(const Kv8 &cache, size_t count) {
    require(count <= size_t(cache.capacity), "count must not exceed the cache's capacity");
}

}  // namespace

void kv8_check(const Kv8 &cache) {
    require(cache.batch >= 0 && cache.batch <= 1 << 24, "cache batch must be in 0..2^24");
    require(cache.heads >= 1 && cache.heads <= 4096, "cache heads must be in 1..4096");
    require(cache.width >= 1 && cache.width <= 256, "cache head width must be in 1..256");
    require(cache.capacity >= kKv8Tile && cache.capacity <= 1 << 24 && cache.capacity % kKv8Tile == 0,
            "cache capacity must be a multiple of 64 in 64..2^24");
    require(int64_t(cache.batch) * cache.heads < int64_t(1) << 31, "cache batch times heads must stay below 2^31");
    require(cache.batch == 0 || (cache.k && cache.v && cache.ks && cache.vs), "cache buffers must not be null");
    require((reinterpret_cast<uintptr_t>(cache.k) | reinterpret_cast<uintptr_t>(cache.v)) % 16 == 0,
            "cache keys and values must be aligned to 16 bytes");
    require((reinterpret_cast<uintptr_t>(cache.ks) | reinterpret_cast<uintptr_t>(cache.vs)) % 4 == 0,
            "cache scales must be aligned to 4 bytes");
}

size_t kv8_code_bytes(const Kv8 &cache) {
    return size_t(cache.batch) * size_t(cache.heads) * size_t(cache.capacity) * size_t(cache.pad);
}
size_t kv8_scale_bytes(const Kv8 &cache) {
    return size_t(cache.batch) * size_t(cache.heads) * size_t(cache.capacity / kKv8Block);
}

void kv8_append(int device, const Kv8 &cache, Type type, size_t count, const void *k, Strides ks, const void *v,
                Strides vs, const int *lengths, const int *counts, hipStream_t stream) {
    kv8_check(cache);
    check_type(type);
    check_count(cache, count);
    if (cache.batch == 0 || count == 0) return;
    require(k && v && lengths, "keys, values and lengths must not be null");
    check_aligned(k, type, "keys must be aligned to their type");
    check_aligned(v, type, "values must be aligned to their type");
    check_grid(2.0 * cache.batch * cache.heads * ((double(count) + 126) / 64));
    const OnDevice on(device);
    kern::Kv8AppendArgs a{};
    a.cache = cache;
    a.k = k;
    a.v = v;
    a.ks = ks;
    a.vs = vs;
    a.lengths = lengths;
    a.counts = counts;
    a.count = int(count);
    a.aligned = alignment(k, ks, v, vs, type);
    kern::kv8_append(a, type, stream);
    check(hipGetLastError(), "append launch");
}

void kv8_read(int device, const Kv8 &cache, Type type, size_t first, size_t count, void *k, Strides ks, void *v,
              Strides vs, const int *lengths, hipStream_t stream) {
    kv8_check(cache);
    check_type(type);
    require(first <= size_t(cache.capacity) && count <= size_t(cache.capacity) - first,
            "positions must lie inside the cache's capacity");
    if (cache.batch == 0 || count == 0) return;
    require(k && v, "keys and values must not be null");
    check_aligned(k, type, "keys must be aligned to their type");
    check_aligned(v, type, "values must be aligned to their type");
    check_grid(2.0 * cache.batch * cache.heads * ((double(count) + 126) / 64));
    const OnDevice on(device);
    kern::Kv8ReadArgs a{};
    a.cache = cache;
    a.k = k;
    a.v = v;
    a.ks = ks;
    a.vs = vs;
    a.lengths = lengths;
    a.first = int(first);
    a.count = int(count);
    a.aligned = alignment(k, ks, v, vs, type);
    kern::kv8_read(a, type, stream);
    check(hipGetLastError(), "read launch");
}

namespace {
int group_of(const Kv8 &cache, size_t heads) {
    require(heads >= 1 && heads <= 65536 && heads % size_t(cache.heads) == 0,
            "query heads must be a multiple of the cache's heads, up to 65536");
    return int(heads / size_t(cache.heads));
}
}  // namespace

size_t kv8_attention_workspace(const Kv8 &cache, size_t heads, size_t count) {
    check_count(cache, count);
    const int group = group_of(cache, heads);
    require(double(count) * group < double(1u << 30), "the call is too large for one launch");
    if (cache.batch == 0 || count == 0) return 0;
    size_t floats = 0;
    for (Type t : {Type::F32, Type::F16, Type::BF16})
        floats = std::max(floats, kern::kv8_plan(cache, t, group, int(count)).part_floats);
    return floats * 4;
}

void kv8_attention(int device, const Kv8 &cache, Type type, size_t heads, size_t count, const void *q, Strides qs,
                   void *out, Strides os, const int *lengths, const int *counts, float scale, void *workspace,
                   size_t workspace_bytes, hipStream_t stream) {
    kv8_check(cache);
    check_type(type);
    check_count(cache, count);
    const int group = group_of(cache, heads);
    require(std::isfinite(2.0f * scale) && scale > 0.0f, "scale must be finite and positive");
    require(double(count) * group < double(1u << 30), "the call is too large for one launch");
    if (cache.batch == 0 || count == 0) return;
    require(q && out && lengths, "queries, output and lengths must not be null");
    check_aligned(q, type, "queries must be aligned to their type");
    check_aligned(out, type, "output must be aligned to its type");
    const kern::Kv8Plan plan = kern::kv8_plan(cache, type, group, int(count));
    require(plan.part_floats == 0 || (workspace && workspace_bytes >= plan.part_floats * 4),
            "the workspace is too small: mg_kv8_attention_workspace gives its size");
    require(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "the workspace must be aligned to 16 bytes");
    const double pairs = double(cache.batch) * cache.heads;
    check_grid((pairs + 7) * plan.splits * plan.row_tiles);
    if (plan.splits > 1) check_grid(pairs * double(count) * group * cache.pad / 1024 + 1);
    const OnDevice on(device);
    kern::Kv8AttnArgs a{};
    a.cache = cache;
    a.q = q;
    a.out = out;
    a.qs = qs;
    a.os = os;
    a.lengths = lengths;
    a.counts = counts;
    a.count = int(count);
    a.group = group;
    a.rows = int(count) * group;
    a.scale_log2 = float(double(scale) * 1.4426950408889634);
    a.splits = plan.splits;
    a.least = plan.least;
    a.part = static_cast<float *>(workspace);
    a.stride = kern::kv8_part_stride(cache.pad);
    a.q_aligned = aligned_to(16, q, qs, type);
    a.o_aligned = aligned_to(16, out, os, type);
    kern::kv8_attention(a, type, plan, stream);
    check(hipGetLastError(), "attention launch");
}

namespace {
void check_rows(size_t rows, size_t vocab, size_t top) {
    require(vocab >= 1 && vocab <= size_t(1) << 24, "vocabulary must hold 1..2^24 tokens");
    require(top <= size_t(kern::kTopMax), "at most 32 alternatives can be asked for");
    require(top <= vocab, "there are more alternatives than tokens");
    require(rows < size_t(1) << 31, "rows must stay below 2^31");
}
void check_temperature(float temperature) {
    // Its inverse is taken in log2 units too.
    require(std::isfinite(temperature) && temperature > 0.0f && std::isfinite(2.0f / temperature),
            "temperature must be finite and positive");
}
size_t stats_bytes(size_t rows, size_t chunks) { return (rows * chunks * 3 * 4 + 15) / 16 * 16; }
}  // namespace

size_t token_logprobs_workspace(size_t rows, size_t vocab, size_t top) {
    check_rows(rows, vocab, top);
    if (rows == 0) return 0;
    int chunks = 1, chunk = 0;
    kern::logprob_chunks(rows, vocab, chunks, chunk);
    return chunks == 1 ? 0 : stats_bytes(rows, size_t(chunks)) + rows * size_t(chunks) * top * 8;
}

void token_logprobs_noalloc(int device, Type type, const void *logits, size_t rows, size_t vocab, size_t stride,
                            const uint32_t *tokens, float temperature, float *logprob, float *entropy, float *stats,
                            size_t top, uint32_t *top_tokens, float *top_logprobs, void *workspace,
                            size_t workspace_bytes, hipStream_t stream) {
    check_type(type);
    const size_t need = token_logprobs_workspace(rows, vocab, top);
    require(stride >= vocab, "the row stride must be at least the vocabulary");
    check_temperature(temperature);
    if (rows == 0) return;
    require(logits, "logits must not be null");
    require(tokens || !logprob, "tokens must not be null");
    require(top == 0 || top_tokens, "the alternatives' tokens must not be null");
    check_aligned(logits, type, "logits must be aligned to their type");
    require(need == 0 || (workspace && workspace_bytes >= need),
            "the workspace is too small: mg_token_logprobs_workspace gives its size");
    require(reinterpret_cast<uintptr_t>(workspace) % 8 == 0, "the workspace must be aligned to 8 bytes");
    kern::LogprobArgs a{};
    kern::logprob_chunks(rows, vocab, a.chunks, a.chunk);
    check_grid(vocab <= kern::kSmallVocab ? double(rows) / 4 + 1 : double(rows) * a.chunks);  // small: a wave a row
    const OnDevice on(device);
    a.logits = logits;
    a.rows = rows;
    a.vocab = vocab;
    a.stride = stride;
    a.tokens = tokens;
    a.inv_temperature = 1.0f / temperature;
    a.logprob = logprob;
    a.entropy = entropy;
    a.stats = stats;
    a.top = int(top);
    a.top_tokens = top_tokens;
    a.top_logprobs = top_logprobs;
    if (a.chunks > 1) {
        a.part_stats = static_cast<float *>(workspace);
        a.part_top = reinterpret_cast<uint64_t *>(static_cast<char *>(workspace) + stats_bytes(rows, size_t(a.chunks)));
    }
    kern::token_logprobs(a, type, stream);
    check(hipGetLastError(), "log probability launch");
}

void token_logprobs_backward_noalloc(int device, Type type, const void *logits, size_t rows, size_t vocab,
                                     size_t stride, const uint32_t *tokens, float temperature, const float *stats,
                                     const float *entropy, const float *d_logprob, const float *d_entropy,
                                     void *d_logits, size_t d_stride, hipStream_t stream) {
    check_type(type);
    check_rows(rows, vocab, 0);
    require(stride >= vocab && d_stride >= vocab, "the row strides must be at least the vocabulary");
    check_temperature(temperature);
    if (rows == 0) return;
    require(logits && stats && d_logits, "logits, stats and the gradient must not be null");
    require(!d_logprob || tokens, "tokens must not be null");
    require(!d_entropy || entropy, "the gradient of the entropy needs the entropy");
    check_aligned(logits, type, "logits must be aligned to their type");
    check_aligned(d_logits, type, "the gradient must be aligned to its type");
    check_grid(double(rows) * std::ceil(double(vocab) / kern::kGradRun) / 4 + 1);
    const OnDevice on(device);
    kern::LogprobBackwardArgs a{};
    a.logits = logits;
    a.rows = rows;
    a.vocab = vocab;
    a.stride = stride;
    a.tokens = tokens;
    a.inv_temperature = 1.0f / temperature;
    a.stats = stats;
    a.entropy = entropy;
    a.d_logprob = d_logprob;
    a.d_entropy = d_entropy;
    a.d_logits = d_logits;
    a.d_stride = d_stride;
    kern::token_logprobs_backward(a, type, stream);
    check(hipGetLastError(), "log probability gradient launch");
}

void token_logprobs(int device, const float *logits, size_t rows, size_t vocab, const uint32_t *tokens,
                    float temperature, float *logprob, float *entropy, size_t top, uint32_t *top_tokens,
                    float *top_logprobs) {
    const size_t need = token_logprobs_workspace(rows, vocab, top);
    check_temperature(temperature);
    if (rows == 0) return;
    require(logits, "logits must not be null");
    require(tokens || !logprob, "tokens must not be null");
    require(top == 0 || top_tokens, "the alternatives' tokens must not be null");
    for (size_t i = 0; logprob && i < rows; ++i)
        require(tokens[i] < vocab || tokens[i] == 0xffffffffu, "token ID is outside the vocabulary");
    const OnDevice on(device);
    const Buffer z(rows * vocab * 4), t(rows * 4), out(rows * 8), ids(rows * top * 4), best(rows * top * 4), space(need);
    check(hipMemcpy(z.as<float>(), logits, rows * vocab * 4, hipMemcpyHostToDevice), "upload logits");
    if (logprob) check(hipMemcpy(t.as<float>(), tokens, rows * 4, hipMemcpyHostToDevice), "upload tokens");
    float *const lp = out.as<float>(), *const h = lp + rows;
    token_logprobs_noalloc(device, Type::F32, z.as<float>(), rows, vocab, vocab, t.as<uint32_t>(), temperature,
                           logprob ? lp : nullptr, entropy ? h : nullptr, nullptr, top, ids.as<uint32_t>(),
                           top_logprobs ? best.as<float>() : nullptr, space.as<void>(), need, nullptr);
    check(hipDeviceSynchronize(), "hipDeviceSynchronize");
    if (logprob) check(hipMemcpy(logprob, lp, rows * 4, hipMemcpyDeviceToHost), "download log probabilities");
    if (entropy) check(hipMemcpy(entropy, h, rows * 4, hipMemcpyDeviceToHost), "download entropies");
    if (top) {
        check(hipMemcpy(top_tokens, ids.as<float>(), rows * top * 4, hipMemcpyDeviceToHost), "download alternatives");
        if (top_logprobs)
            check(hipMemcpy(top_logprobs, best.as<float>(), rows * top * 4, hipMemcpyDeviceToHost),
                  "download alternatives");
    }
}

}  // namespace meshgpt
