// Losses on a batch of logits [batch, seq, vocab] and their gradients.
//
// Log probability of a row's target: lp = z_y - lse(z).  A loss that depends
// on the logits through lp alone has d loss / d z = c (onehot(y) - p) with
// c = d loss / d lp and p = exp(z - max) / sum.  (The maximum and the sum are
// kept apart: a row of values as large as their type's lowest has no room for
// the sum's logarithm beside them.)
#include "common.h"

#include <algorithm>
#include <cmath>

namespace smx {

struct LogitRows {
  const void *z;
  const int64_t *targets;    // [batch, seq]
  const uint8_t *mask;       // [batch, seq] or null
  int64_t batch, seq, vocab, batch_stride, row_stride;
};

constexpr int kRowThreads = 256;

__device__ __forceinline__ float block_max(float v, float *scratch) {
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  for (int w = 0; w < static_cast<int>(blockDim.x >> 6); ++w) v = fmaxf(v, scratch[w]);
  return v;
}

struct RowLp {
  float top, sum;  // lse = top + log(sum)
  float lp;
};

template <int DT>
__device__ __forceinline__ RowLp row_lp(const LogitRows &a, int64_t at, int64_t y, float *scratch) {
  float top = -INFINITY;
  for (int64_t v = threadIdx.x; v < a.vocab; v += kRowThreads) top = fmaxf(top, load_elem<DT>(a.z, at + v));
  top = block_max(top, scratch);
  float sum = 0.f;
  for (int64_t v = threadIdx.x; v < a.vocab; v += kRowThreads) sum += expf(load_elem<DT>(a.z, at + v) - top);
  sum = block_sum(sum, scratch);
  const double z = y >= 0 && y < a.vocab ? static_cast<double>(load_elem<DT>(a.z, at + y)) : __builtin_nan("");
  return {top, sum, static_cast<float>((z - top) - log(static_cast<double>(sum)))};
}

// out[v] = c (onehot(y) - p).
template <int DT>
__device__ __forceinline__ void row_grad(const LogitRows &a, int64_t at, int64_t y, float top, float sum, float c,
                                         void *out, int64_t out_at) {
  const float inv = 1.f / sum;
  for (int64_t v = threadIdx.x; v < a.vocab; v += kRowThreads) {
    const float p = expf(load_elem<DT>(a.z, at + v) - top) * inv;
    store_any(out, DT, out_at + v, round_to(DT, v == y ? c - c * p : -c * p));
  }
}

template <int DT>
__device__ __forceinline__ void row_zero(void *out, int64_t out_at, int64_t vocab) {
  for (int64_t v = threadIdx.x; v < vocab; v += kRowThreads) store_any(out, DT, out_at + v, 0.f);
}

template <int DT>
__global__ void __launch_bounds__(kRowThreads) logprob_kernel(LogitRows a, float *logprobs, float2 *stats) {
  __shared__ float scratch[16];
  const int64_t r = blockIdx.x;
  if (a.mask && !a.mask[r]) {
    if (threadIdx.x == 0) {
      logprobs[r] = 0.f;
      if (stats) stats[r] = make_float2(0.f, 1.f);
    }
    return;
  }
  const RowLp o = row_lp<DT>(a, r / a.seq * a.batch_stride + r % a.seq * a.row_stride, a.targets[r], scratch);
  if (threadIdx.x == 0) {
    logprobs[r] = o.lp;
    if (stats) stats[r] = make_float2(o.top, o.sum);
  }
}

template <int DT>
__global__ void __launch_bounds__(kRowThreads) logprob_back_kernel(LogitRows a, const float2 *stats, const float *coef,
                                                                   int64_t coef_batch, int64_t coef_seq,
                                                                   const float *scale, void *dz) {
  const int64_t r = blockIdx.x, b = r / a.seq, t = r % a.seq;
  const bool live = !a.mask || a.mask[r];
  if (!live) return row_zero<DT>(dz, r * a.vocab, a.vocab);
  float c = coef[b * coef_batch + t * coef_seq];
  if (scale) c *= *scale;
  const int64_t y = a.targets[r];
  if (y < 0 || y >= a.vocab) c = __builtin_nanf("");
  row_grad<DT>(a, b * a.batch_stride + t * a.row_stride, y, stats[r].x, stats[r].y, c, dz, r * a.vocab);
}

// ---------------------------------------------------------- policy loss ---
struct PolicyArgs {
  LogitRows rows;
  const float *old_lp, *ref_lp, *adv;  // [batch, seq] (old, ref may be null); adv by its strides
  int64_t adv_batch, adv_seq;
  float low, high, kl, scale;  // the ratio's unclipped range
  int32_t per_sequence;
  float *logprobs, *weights, *terms;  // [batch, seq], [batch], [batch, seq]
  void *dz;
};

// A sequence's weight of each of its live tokens: 1 / live tokens of the
// batch, or 1 / (its live tokens * sequences with any).
__global__ void __launch_bounds__(1024) policy_weight_kernel(PolicyArgs a) {
  __shared__ double scratch[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double total = 0;
  for (int64_t b = wave; b < a.rows.batch; b += 16) {
    int64_t n = 0;
    if (a.rows.mask) {
      for (int64_t t = lane; t < a.rows.seq; t += 64) n += a.rows.mask[b * a.rows.seq + t] != 0;
      n = static_cast<int64_t>(wave_sum(static_cast<double>(n)));
    } else {
      n = a.rows.seq;
    }
    if (lane == 0) {
      a.weights[b] = static_cast<float>(n);
      total += a.per_sequence ? (n > 0) : static_cast<double>(n);
    }
  }
  total = block_sum(total, scratch);
  for (int64_t b = threadIdx.x; b < a.rows.batch; b += 1024) {
    const double n = a.weights[b], d = a.per_sequence ? n * total : total;
    a.weights[b] = n > 0 ? static_cast<float>(a.scale / d) : 0.f;
  }
}

template <int DT>
__global__ void __launch_bounds__(kRowThreads) policy_kernel(PolicyArgs a) {
  __shared__ float scratch[16];
  const LogitRows &q = a.rows;
  const int64_t r = blockIdx.x, b = r / q.seq, t = r % q.seq;
  if (q.mask && !q.mask[r]) {
    if (threadIdx.x == 0) a.logprobs[r] = a.terms[r] = 0.f;
    if (a.dz) row_zero<DT>(a.dz, r * q.vocab, q.vocab);
    return;
  }
  const int64_t at = b * q.batch_stride + t * q.row_stride, y = q.targets[r];
  const RowLp o = row_lp<DT>(q, at, y, scratch);
  const float w = a.weights[b], adv = a.adv[b * a.adv_batch + t * a.adv_seq];
  const float ratio = a.old_lp ? expf(o.lp - a.old_lp[r]) : 1.f;
  // (comparisons that keep a NaN, which fminf and fmaxf would drop)
  const float clipped = ratio < a.low ? a.low : ratio > a.high ? a.high : ratio;
  float term = -(clipped * adv < ratio * adv ? clipped * adv : ratio * adv);
  const bool moves = adv > 0.f ? ratio <= a.high : ratio >= a.low;
  float c = moves ? -ratio * adv : 0.f;
  if (a.ref_lp) {
    const float gap = a.ref_lp[r] - o.lp, em1 = expm1f(gap);
    term += a.kl * (em1 - gap);
    c -= a.kl * em1;
  }
  if (threadIdx.x == 0) {
    a.logprobs[r] = o.lp;
    a.terms[r] = w * term;
  }
  if (a.dz) row_grad<DT>(q, at, y, o.top, o.sum, w * c, a.dz, r * q.vocab);
}

__global__ void __launch_bounds__(1024) sum_kernel(const float *x, int64_t n, float *out) {
  __shared__ double scratch[16];
  double t = 0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) t += x[i];
  t = block_sum(t, scratch);
  if (threadIdx.x == 0) *out = static_cast<float>(t);
}

// ------------------------------------------------------ preference loss ---
struct PreferenceArgs {
  const float *lp, *ref;  // [2 pairs, seq], chosen first
  const uint8_t *mask;
  int64_t pairs, seq;
  double beta, smoothing;
  float *loss, *margins, *coef;  // [1], [pairs], [2 pairs]
};

// The gain of each sequence (sum of its live log ratios) in FP64, then a
// pair's margin, loss and d loss / d lp: a wave a pair, one block.
__global__ void __launch_bounds__(1024) preference_kernel(PreferenceArgs a) {
  __shared__ double scratch[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double loss = 0;
  for (int64_t p = wave; p < a.pairs; p += 16) {
    double gain = 0;
    for (int side = 0; side < 2; ++side) {
      const int64_t at = (p + side * a.pairs) * a.seq;
      double g = 0;
      for (int64_t t = lane; t < a.seq; t += 64)
        if (!a.mask || a.mask[at + t]) g += static_cast<double>(a.lp[at + t]) - a.ref[at + t];
      gain += side ? -g : g;
    }
    const double m = a.beta * wave_sum(gain);
    const double soft = log1p(exp(-fabs(m)));
    if (lane == 0) {
      loss += (1 - a.smoothing) * (soft - fmin(m, 0.)) + a.smoothing * (soft + fmax(m, 0.));
      a.margins[p] = static_cast<float>(m);
      const double slope = a.beta * (1 / (1 + exp(-m)) - (1 - a.smoothing)) / a.pairs;
      a.coef[p] = static_cast<float>(slope);
      a.coef[p + a.pairs] = static_cast<float>(-slope);
    }
  }
  loss = block_sum(loss, scratch);
  if (threadIdx.x == 0) *a.loss = static_cast<float>(a.pairs ? loss / a.pairs : 0.);
}

// x *= *scale, unless it is one.
template <int DT>
__global__ void __launch_bounds__(256) scale_kernel(void *x, int64_t n, const float *scale) {
  const float s = *scale;
  if (s == 1.f) return;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256)
    store_any(x, DT, i, round_to(DT, load_elem<DT>(x, i) * s));
}

// ----------------------------------------------------------------- host ---
static int logits_check(const char *what, const void *z, int dtype, int64_t batch, int64_t seq, int64_t vocab,
                        int64_t batch_stride, int64_t row_stride, const int64_t *targets) {
  const auto msg = [&](const char *m) { return std::string(what) + ": " + m; };
  SMX_REQUIRE(dtype == SMX_F32 || dtype == SMX_BF16 || dtype == SMX_F16, SMX_EDTYPE, msg("dtype must be f32, bf16 or f16"));
  SMX_REQUIRE(batch >= 0 && seq >= 0, SMX_ESHAPE, msg("negative size"));
  SMX_REQUIRE(vocab >= 1 && vocab <= (int64_t{1} << 30), SMX_ESHAPE, msg("vocabulary must be in [1, 2^30]"));
  if (batch == 0 || seq == 0) return SMX_OK;
  const int64_t most = int64_t{1} << 31;
  SMX_REQUIRE(batch < most && seq < most && batch * seq < most, SMX_ESHAPE, msg("more than 2^31 - 1 rows"));
  SMX_REQUIRE(z && targets, SMX_EINVAL, msg("null logits or targets"));
  SMX_REQUIRE(row_stride >= vocab || seq == 1, SMX_ESHAPE, msg("row stride smaller than the vocabulary"));
  SMX_REQUIRE(batch_stride >= 0, SMX_ESHAPE, msg("negative batch stride"));
  return SMX_OK;
}

#define LOGITS_BY_DTYPE(dtype, LAUNCH) \
  do {                                 \
    if ((dtype) == SMX_F32) {          \
      LAUNCH(SMX_F32);                 \
    } else if ((dtype) == SMX_BF16) {  \
      LAUNCH(SMX_BF16);                \
    } else {                           \
      LAUNCH(SMX_F16);                 \
    }                                  \
  } while (0)

}  // namespace smx

using namespace smx;

extern "C" int smx_token_logprobs(const void *logits, int dtype, int64_t batch, int64_t seq, int64_t vocab,
                                  int64_t batch_stride, int64_t row_stride, const int64_t *targets,
                                  const uint8_t *mask, float *logprobs, float *stats, void *stream) {
  const int rc = logits_check("token_logprobs", logits, dtype, batch, seq, vocab, batch_stride, row_stride, targets);
  if (rc != SMX_OK || batch * seq == 0) return rc;
  SMX_REQUIRE(logprobs, SMX_EINVAL, "token_logprobs: null output");
  const LogitRows a{logits, targets, mask, batch, seq, vocab, batch_stride, row_stride};
  const dim3 grid(static_cast<unsigned>(batch * seq));
#define LAUNCH(DT) \
  hipLaunchKernelGGL((logprob_kernel<DT>), grid, dim3(kRowThreads), 0, static_cast<hipStream_t>(stream), a, logprobs, \
                     reinterpret_cast<float2 *>(stats))
  LOGITS_BY_DTYPE(dtype, LAUNCH);
#undef LAUNCH
  return check_launch("token_logprobs");
}

extern "C" int smx_token_logprobs_backward(const void *logits, int dtype, int64_t batch, int64_t seq, int64_t vocab,
                                           int64_t batch_stride, int64_t row_stride, const int64_t *targets,
                                           const uint8_t *mask, const float *stats, const float *coef,
                                           int64_t coef_batch_stride, int64_t coef_row_stride, const float *scale,
                                           void *dlogits, void *stream) {
  const int rc = logits_check("token_logprobs_backward", logits, dtype, batch, seq, vocab, batch_stride, row_stride, targets);
  if (rc != SMX_OK || batch * seq == 0) return rc;
  SMX_REQUIRE(stats && coef && dlogits, SMX_EINVAL, "token_logprobs_backward: null pointer");
  const LogitRows a{logits, targets, mask, batch, seq, vocab, batch_stride, row_stride};
  const dim3 grid(static_cast<unsigned>(batch * seq));
#define LAUNCH(DT)                                                                                                    \
  hipLaunchKernelGGL((logprob_back_kernel<DT>), grid, dim3(kRowThreads), 0, static_cast<hipStream_t>(stream), a,    \
                     reinterpret_cast<const float2 *>(stats), coef, coef_batch_stride, coef_row_stride, scale, dlogits)
  LOGITS_BY_DTYPE(dtype, LAUNCH);
#undef LAUNCH
  return check_launch("token_logprobs_backward");
}

extern "C" int64_t smx_policy_loss_workspace_bytes(int64_t batch, int64_t seq) {
  if (batch < 0 || seq < 0) return SMX_EINVAL;
  return (batch + batch * seq) * static_cast<int64_t>(sizeof(float));
}

extern "C" int smx_policy_loss(const void *logits, int dtype, int64_t batch, int64_t seq, int64_t vocab,
                               int64_t batch_stride, int64_t row_stride, const int64_t *targets, const uint8_t *mask,
                               const float *old_logprobs, const float *ref_logprobs, const float *advantages,
                               int64_t adv_batch_stride, int64_t adv_row_stride, double clip_low, double clip_high,
                               double kl_coef, int reduction, double scale, float *loss, float *logprobs,
                               void *dlogits, void *workspace, int64_t workspace_bytes, void *stream) {
  const int rc = logits_check("policy_loss", logits, dtype, batch, seq, vocab, batch_stride, row_stride, targets);
  if (rc != SMX_OK) return rc;
  SMX_REQUIRE(reduction == SMX_MEAN_TOKEN || reduction == SMX_MEAN_SEQUENCE, SMX_EINVAL, "policy_loss: unknown reduction");
  SMX_REQUIRE(clip_low >= 0 && clip_low <= 1 && clip_high >= 0, SMX_EINVAL,
              "policy_loss: clip_low must be in [0, 1] and clip_high not negative");
  SMX_REQUIRE(loss, SMX_EINVAL, "policy_loss: null loss");
  const auto st = static_cast<hipStream_t>(stream);
  const int64_t rows = batch * seq;
  PolicyArgs a{};
  if (rows > 0) {
    SMX_REQUIRE(logprobs && advantages, SMX_EINVAL, "policy_loss: null pointer");
    SMX_REQUIRE(workspace && workspace_bytes >= smx_policy_loss_workspace_bytes(batch, seq), SMX_EWORKSPACE,
                "policy_loss: workspace too small");
    a.rows = {logits, targets, mask, batch, seq, vocab, batch_stride, row_stride};
    a.old_lp = old_logprobs, a.ref_lp = ref_logprobs, a.adv = advantages;
    a.adv_batch = adv_batch_stride, a.adv_seq = adv_row_stride;
    a.low = static_cast<float>(1 - clip_low), a.high = static_cast<float>(1 + clip_high);
    a.kl = static_cast<float>(kl_coef), a.scale = static_cast<float>(scale);
    a.per_sequence = reduction == SMX_MEAN_SEQUENCE;
    a.logprobs = logprobs, a.weights = static_cast<float *>(workspace), a.terms = a.weights + batch, a.dz = dlogits;
    hipLaunchKernelGGL(policy_weight_kernel, dim3(1), dim3(1024), 0, st, a);
    const dim3 grid(static_cast<unsigned>(rows));
#define LAUNCH(DT) hipLaunchKernelGGL((policy_kernel<DT>), grid, dim3(kRowThreads), 0, st, a)
    LOGITS_BY_DTYPE(dtype, LAUNCH);
#undef LAUNCH
  }
  hipLaunchKernelGGL(sum_kernel, dim3(1), dim3(1024), 0, st, static_cast<const float *>(a.terms), rows, loss);
  return check_launch("policy_loss");
}

extern "C" int smx_preference_loss(const float *logprobs, const float *ref_logprobs, const uint8_t *mask,
                                   int64_t pairs, int64_t seq, double beta, double label_smoothing, float *loss,
                                   float *margins, float *coef, void *stream) {
  SMX_REQUIRE(pairs >= 0 && seq >= 0, SMX_ESHAPE, "preference_loss: negative size");
  SMX_REQUIRE(label_smoothing >= 0 && label_smoothing <= 1, SMX_EINVAL, "preference_loss: label_smoothing must be in [0, 1]");
  SMX_REQUIRE(loss && (pairs == 0 || (margins && coef)), SMX_EINVAL, "preference_loss: null output");
  SMX_REQUIRE(pairs == 0 || seq == 0 || (logprobs && ref_logprobs), SMX_EINVAL, "preference_loss: null log probabilities");
  const PreferenceArgs a{logprobs, ref_logprobs, mask, pairs, seq, beta, label_smoothing, loss, margins, coef};
  hipLaunchKernelGGL(preference_kernel, dim3(1), dim3(1024), 0, static_cast<hipStream_t>(stream), a);
  return check_launch("preference_loss");
}

extern "C" int smx_scale(void *x, int dtype, int64_t n, const float *scale, void *stream) {
  SMX_REQUIRE(dtype == SMX_F32 || dtype == SMX_BF16 || dtype == SMX_F16, SMX_EDTYPE, "scale: dtype must be f32, bf16 or f16");
  SMX_REQUIRE(n >= 0, SMX_ESHAPE, "scale: negative size");
  if (n == 0) return SMX_OK;
  SMX_REQUIRE(x && scale, SMX_EINVAL, "scale: null pointer");
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(4096, ceil_div(n, 256))));
#define LAUNCH(DT) hipLaunchKernelGGL((scale_kernel<DT>), grid, dim3(256), 0, static_cast<hipStream_t>(stream), x, n, scale)
  LOGITS_BY_DTYPE(dtype, LAUNCH);
#undef LAUNCH
  return check_launch("scale");
}
