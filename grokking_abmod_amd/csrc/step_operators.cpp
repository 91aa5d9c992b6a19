// The checked entry points of the operators around a step's matrix products:
// sampling with filters, rotary positions and the root-mean-square norm.
// Arguments are looked at, the work is enqueued on the caller's stream, and the
// caller's current device is what it was.
#include <algorithm>
#include <cmath>

#include "operators_host.hpp"

namespace meshgpt {

void sample_filtered_noalloc(int device, Type type, const void *logits, size_t rows, size_t vocab, size_t stride,
                             const float *temperatures, const int *top_k, const float *top_p, const float *min_p,
                             const float *uniforms, uint32_t *tokens, float *logprob, hipStream_t stream) {
    check_type(type);
    require(vocab >= 1 && vocab <= size_t(1) << 20, "vocabulary must hold 1..2^20 tokens");  // sums have 64 bits
    require(stride >= vocab, "the row stride must be at least the vocabulary");
    require(rows < size_t(1) << 22, "rows must stay below 2^22");  // of 1024 threads each, counted in 32 bits
    if (rows == 0) return;
    require(logits && uniforms && tokens, "logits, uniforms and tokens must not be null");
    check_aligned(logits, type, "logits must be aligned to their type");
    check_words({temperatures, top_k, top_p, min_p, uniforms, tokens, logprob},
                "settings, numbers, tokens and log probabilities must be aligned to 4 bytes");
    const OnDevice on(device);
    kern::SampleArgs a{};
    a.logits = logits;
    a.rows = rows;
    a.vocab = vocab;
    a.stride = stride;
    a.temperatures = temperatures;
    a.top_k = top_k;
    a.top_p = top_p;
    a.min_p = min_p;
    a.uniforms = uniforms;
    a.tokens = tokens;
    a.logprob = logprob;
    kern::sample_filtered(a, type, stream);
    check(hipGetLastError(), "sampling launch");
}

namespace {
void check_rope(size_t width, size_t rotary) {
    require(width >= 1 && width <= 1024, "head width must be in 1..1024");
    require(rotary % 2 == 0 && rotary <= width, "rotary channels must be an even number up to the head width");
}
}  // namespace

void rope_frequencies(size_t rotary, double base, RopeScaling scaling, double factor, double context, double low,
                      double high, double *out) {
    check_rope(1024, rotary);
    require(std::isfinite(base) && base > 1.0, "the base must be finite and over 1");
    const bool scaled = scaling != RopeScaling::None;
    require(scaling >= RopeScaling::None && scaling <= RopeScaling::Bands, "unknown rotary scaling code");
    require(!scaled || (std::isfinite(factor) && factor >= 1.0), "the scaling factor must be finite and at least 1");
    const bool bands = scaling == RopeScaling::Bands;
    require(!bands || (std::isfinite(context) && context > 0.0), "the original context must be finite and positive");
    require(!bands || (std::isfinite(low) && std::isfinite(high) && low >= 0.0 && low < high),
            "turns must rise from low to high");
    require(out != nullptr || rotary == 0, "output must not be null");
    if (scaling == RopeScaling::Base && rotary > 2) base *= std::pow(factor, double(rotary) / double(rotary - 2));
    for (size_t i = 0; i < rotary / 2; ++i) {
        const double f = std::pow(base, -2.0 * double(i) / double(rotary));
        out[i] = f;
        if (scaling == RopeScaling::Linear) out[i] = f / factor;
        if (bands) {
            const double turns = context * f / 6.283185307179586;
            const double kept = std::min(1.0, std::max(0.0, (turns - low) / (high - low)));
            out[i] = f * kept + f / factor * (1.0 - kept);
        }
    }
}

void rope(int device, const Rope &r, Type type, size_t batch, size_t count, size_t heads, const void *q, Strides qs,
          void *q_out, Strides qos, size_t kv_heads, const void *k, Strides ks, void *k_out, Strides kos,
          const int *lengths, const int *counts, const int *positions, bool backward, hipStream_t stream) {
    check_type(type);
    check_rope(r.width, r.rotary);
    require(std::isfinite(r.magnitude), "the magnitude must be finite");
    require(heads <= 65536 && kv_heads <= 65536, "heads must be at most 65536");
    check_grid(double(batch) * double(count));  // a token is a workgroup's, or several are
    if (batch == 0 || count == 0 || heads + kv_heads == 0) return;
    require((heads == 0 || (q && q_out)) && (kv_heads == 0 || (k && k_out)), "queries and keys must not be null");
    require(r.rotary == 0 || r.frequencies, "frequencies must not be null");
    if (heads)
        for (const void *p : {q, static_cast<const void *>(q_out)})
            check_aligned(p, type, "queries must be aligned to their type");
    if (kv_heads)
        for (const void *p : {k, static_cast<const void *>(k_out)})
            check_aligned(p, type, "keys must be aligned to their type");
    require(reinterpret_cast<uintptr_t>(r.frequencies) % 8 == 0, "frequencies must be aligned to 8 bytes");
    check_words({lengths, counts, positions}, "lengths, counts and positions must be aligned to 4 bytes");
    const OnDevice on(device);
    kern::RopeArgs a{};
    a.side[0] = {q, q_out, qs, qos, int(heads)};
    a.side[1] = {k, k_out, ks, kos, int(kv_heads)};
    a.frequencies = r.frequencies;
    a.magnitude = r.magnitude;
    a.lengths = lengths;
    a.counts = counts;
    a.positions = positions;
    a.batch = int(batch);
    a.count = int(count);
    a.width = int(r.width);
    a.rotary = int(r.rotary);
    a.interleaved = r.interleaved;
    a.backward = backward;
    kern::rope(a, type, stream);
    check(hipGetLastError(), "rotary launch");
}

namespace {
void check_norm(size_t rows, size_t width) {
    require(width >= 1 && width <= kern::kNormWidth, "width must be in 1..16384");
    require(rows < size_t(1) << 22, "rows must stay below 2^22");  // of up to 1024 threads each, counted in 32 bits
}

kern::NormArgs norm_args(Type type, size_t rows, size_t width, const void *x, size_t x_stride, const void *residual,
                         size_t residual_stride, void *sum, size_t sum_stride, const void *weight, float epsilon,
                         float *rstd) {
    check_type(type);
    check_norm(rows, width);
    require(x_stride >= width && (!residual || residual_stride >= width) && (!sum || sum_stride >= width),
            "the row strides must be at least the width");
    require(std::isfinite(epsilon) && epsilon > 0.0f, "epsilon must be finite and positive");
    require(rows == 0 || x, "rows must not be null");
    for (const void *p : {x, residual, static_cast<const void *>(sum), weight})
        check_aligned(p, type, "rows and weight must be aligned to their type");
    check_words({rstd}, "rstd must be aligned to 4 bytes");
    kern::NormArgs a{};
    a.x = x;
    a.residual = residual;
    a.sum = sum;
    a.weight = weight;
    a.rstd = rstd;
    a.rows = rows;
    a.xs = x_stride;
    a.rs = residual_stride;
    a.ss = sum_stride;
    a.width = int(width);
    a.epsilon = epsilon;
    return a;
}
}  // namespace

void rms_norm(int device, Type type, size_t rows, size_t width, const void *x, size_t x_stride, const void *residual,
              size_t residual_stride, void *sum, size_t sum_stride, const void *weight, float epsilon, void *out,
              size_t out_stride, float *rstd, hipStream_t stream) {
    kern::NormArgs a = norm_args(type, rows, width, x, x_stride, residual, residual_stride, sum, sum_stride, weight,
                                 epsilon, rstd);
    require(out_stride >= width, "the row strides must be at least the width");
    if (rows == 0) return;
    require(out, "output must not be null");
    check_aligned(out, type, "output must be aligned to its type");
    const OnDevice on(device);
    a.out = out;
    a.os = out_stride;
    kern::rms_norm(a, type, stream);
    check(hipGetLastError(), "norm launch");
}

void rms_norm_e4m3(int device, Type type, size_t rows, size_t width, const void *x, size_t x_stride,
                   const void *residual, size_t residual_stride, void *sum, size_t sum_stride, const void *weight,
                   float epsilon, uint8_t *codes, size_t codes_stride, uint8_t *scales, size_t scales_stride,
                   float *rstd, hipStream_t stream) {
    kern::NormArgs a = norm_args(type, rows, width, x, x_stride, residual, residual_stride, sum, sum_stride, weight,
                                 epsilon, rstd);
    require(codes_stride >= width && scales_stride >= (width + 31) / 32,
            "the strides of codes and scales must be at least a row's");
    if (rows == 0) return;
    require(codes && scales, "codes and scales must not be null");
    const OnDevice on(device);
    a.codes = codes;
    a.os = codes_stride;
    a.scales = scales;
    a.scs = scales_stride;
    kern::rms_norm(a, type, stream);
    check(hipGetLastError(), "norm launch");
}

size_t rms_norm_backward_workspace(size_t rows, size_t width) {
    check_norm(rows, width);
    return kern::norm_parts(rows, width) * width * 4;
}

void rms_norm_backward(int device, Type type, size_t rows, size_t width, const void *sum, size_t sum_stride,
                       const void *weight, const float *rstd, const void *d_out, size_t d_out_stride, const void *d_sum,
                       size_t d_sum_stride, void *d_x, size_t d_x_stride, float *d_weight, void *workspace,
                       size_t workspace_bytes, hipStream_t stream) {
    check_type(type);
    const size_t need = d_weight ? rms_norm_backward_workspace(rows, width) : 0;
    check_norm(rows, width);
    require(sum_stride >= width && d_out_stride >= width && (!d_sum || d_sum_stride >= width) && d_x_stride >= width,
            "the row strides must be at least the width");
    if (rows == 0 && !d_weight) return;
    require(rows == 0 || (sum && rstd && d_out && d_x), "rows, rstd and the gradients must not be null");
    for (const void *p : {sum, weight, d_out, d_sum, static_cast<const void *>(d_x)})
        check_aligned(p, type, "rows, weight and gradients must be aligned to their type");
    check_words({rstd, d_weight}, "rstd and the weight's gradient must be aligned to 4 bytes");
    require(need == 0 || (workspace && workspace_bytes >= need),
            "the workspace is too small: mg_rms_norm_backward_workspace gives its size");
    require(reinterpret_cast<uintptr_t>(workspace) % 4 == 0, "the workspace must be aligned to 4 bytes");
    const OnDevice on(device);
    kern::NormBackwardArgs a{};
    a.x = sum;
    a.weight = weight;
    a.d_out = d_out;
    a.d_sum = d_sum;
    a.rstd = rstd;
    a.d_x = d_x;
    a.d_weight = d_weight;
    a.part = d_weight ? static_cast<float *>(workspace) : nullptr;
    a.rows = rows;
    a.xs = sum_stride;
    a.dos = d_out_stride;
    a.dss = d_sum_stride;
    a.dxs = d_x_stride;
    a.width = int(width);
    kern::rms_norm_backward(a, type, stream);
    check(hipGetLastError(), "norm gradient launch");
}

}  // namespace meshgpt
