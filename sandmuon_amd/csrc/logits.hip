// Losses on a batch of logits [batch, seq, vocab] and their gradients.
//
// Log probability of a row's target: lp = z_y - lse(z).  A loss that depends
// on the logits through lp alone has d loss / d z = c (onehot(y) - p) with
// c = d loss / d lp and p = exp(z - max) / sum.  (The maximum and the sum are
// kept apart: a row of values as large as their type's lowest has no room for
// the sum's logarithm beside them.)
// Bound by HBM: every row is read once and its gradient written once; a row's
// exponentials are made twice, some 19 vector instructions an element, half of
// the time.  Measured at 8 x 1024 x 50257 bf16, 30% of the tokens masked: the
// policy loss with its gradient 285 us (1.40 GB, 4.9 TB/s), log probabilities
// alone 96-100 us (5.7-6 TB/s), their gradient 260 us (5.4 TB/s, part of it read
// from the last cache).  FP16 logits, whose policy gradient is made in the backward:
// 384 us for both.
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

// ------------------------------------------------------------- one row ---
// A row is held in registers from its one read to its gradient's one write:
// NT threads with up to NCH 16-byte chunks each, all of whose loads are in
// flight at once.  An odd vocabulary moves every row's start: the chunks of a
// long row begin at its first 16-byte boundary, since loads that straddle
// boundaries cost a tenth of the time (8 x 1024 x 50257 bf16: 333 us, 296 us
// with aligned ones), and which elements a thread sums then depends on where
// the row lies.  A row of one wave (NT = 64) is bound by latency, not by that,
// and takes its chunks from its first element, so that its sums are the same
// wherever it lies.  The elements before the first chunk and behind the last
// (at most 7 and 7 of 16 bits) are one of each of the first 16 threads.
typedef uint32_t v4u_any __attribute__((ext_vector_type(4), aligned(2)));

// Elements of a row before its first chunk.
template <int NT>
__device__ __forceinline__ int row_head(const char *row, int bytes, int vocab) {
  if constexpr (NT == 64) return 0;
  return min(static_cast<int>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / bytes, vocab);
}

template <int DT>
struct Logit {
  static constexpr int kBytes = DT == SMX_F32 ? 4 : 2, kPer = 16 / kBytes;  // elements of a chunk
  static constexpr uint32_t kNone = DT == SMX_F32 ? 0xff800000u : DT == SMX_BF16 ? 0xff80ff80u : 0xfc00fc00u;  // -inf
  static __device__ __forceinline__ float at(const uint4 &c, int k) {
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
    if constexpr (DT == SMX_F32) return __uint_as_float(w[k]);
    if constexpr (DT == SMX_BF16) return __uint_as_float(k & 1 ? w[k >> 1] & 0xffff0000u : w[k >> 1] << 16);
    return f16_bits_to_f32(static_cast<uint16_t>(w[k >> 1] >> (16 * (k & 1))));
  }
  static __device__ __forceinline__ uint4 pack(const float *v) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (DT == SMX_F32) {
        w[k] = __float_as_uint(v[k]);
      } else if constexpr (DT == SMX_BF16) {
        typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
        const v2bf h = {static_cast<__bf16>(v[2 * k]), static_cast<__bf16>(v[2 * k + 1])};
        __builtin_memcpy(&w[k], &h, 4);
      } else {
        const _Float16 h[2] = {static_cast<_Float16>(v[2 * k]), static_cast<_Float16>(v[2 * k + 1])};
        __builtin_memcpy(&w[k], h, 4);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// exp(d) for d <= 0, as exp2 of d log2 e in two parts: one rounding of the product,
// and no error of one sign, which the sum over a long sequence's tokens would not
// average out (the constant in one part is 1.3e-8 of d off: log probabilities of
// bf16 logits at a vocabulary of 50257 were -7.6e-8 off in the mean, in two parts
// they are -5e-9).  FP32 logits: the product's rounding is made good too.
template <int DT>
__device__ __forceinline__ float exp_of(float d) {
  constexpr float kHi = 1.44269504088896341f, kLo = 1.92596299112661e-8f;  // log2 e
  if constexpr (DT != SMX_F32) return __builtin_amdgcn_exp2f(fmaf(d, kHi, d * kLo));
  const float t = d * kHi, e = __builtin_amdgcn_exp2f(t);
  const float rest = fmaf(d, kLo, fmaf(d, kHi, -t));
  // (an infinite d has no rest)
  return t > -200.f ? fmaf(e, 0.6931471805599453f * rest, e) : e;
}

__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp_mov<0xB1>(v));
  v = fmaxf(v, dpp_mov<0x4E>(v));
  v = fmaxf(v, dpp_mov<0x141>(v));
  v = fmaxf(v, dpp_mov<0x140>(v));
  return fmaxf(fmaxf(read_lane(v, 0), read_lane(v, 16)), fmaxf(read_lane(v, 32), read_lane(v, 48)));
}

// What is left of sum * exp(m - top) where m may be top itself, infinite or not.
template <int DT>
__device__ __forceinline__ float moved(float sum, float m, float top) {
  return m == top ? sum : sum * exp_of<DT>(m - top);
}

struct RowStat {
  float top, sum;  // lse = top + log(sum)
};

template <int DT, int NT, int NCH>
struct Row {
  using L = Logit<DT>;
  uint4 c[NCH];
  float edge;       // this thread's element outside the whole chunks
  int edge_at;      // its place, or -1
  int chunks, head;  // whole chunks, elements before them
  int tid;
  const char *src;

  template <bool AGAIN>
  __device__ __forceinline__ void load(const void *z, int64_t at, int64_t vocab) {
    const char *row = src = static_cast<const char *>(z) + at * L::kBytes;
    tid = NT == 64 ? threadIdx.x & 63 : threadIdx.x;
    const int v = static_cast<int>(vocab);
    head = row_head<NT>(row, L::kBytes, v);
    chunks = (v - head) / L::kPer;
    const char *p = row + head * L::kBytes;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      c[i] = make_uint4(L::kNone, L::kNone, L::kNone, L::kNone);
      if (i * NT < chunks && tid + i * NT < chunks) {
        // (AGAIN: the row is read once more later, and may stay in a cache)
        const auto *at_i = reinterpret_cast<const v4u_any *>(p) + tid + i * NT;
        const v4u_any w = AGAIN ? *at_i : __builtin_nontemporal_load(at_i);
        c[i] = make_uint4(w.x, w.y, w.z, w.w);
      }
    }
    const int tail = head + chunks * L::kPer;
    edge_at = tid < 8 ? (tid < head ? tid : -1) : tid < 16 && tail + tid - 8 < v ? tail + tid - 8 : -1;
    edge = edge_at >= 0 ? load_elem<DT>(row, edge_at) : -INFINITY;
  }

  __device__ __forceinline__ RowStat stat(float2 *scratch) const {
    float m = edge;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (i * NT >= chunks) break;
#pragma unroll
      for (int k = 0; k < L::kPer; ++k) m = fmaxf(m, L::at(c[i], k));
    }
    // (a thread whose elements are all -inf adds nothing)
    const float from = m == -INFINITY ? 0.f : m;
    float s = exp_of<DT>(edge - from);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (i * NT >= chunks) break;
#pragma unroll
      for (int k = 0; k < L::kPer; ++k) s += exp_of<DT>(L::at(c[i], k) - from);
    }
    RowStat r;
    r.top = wave_max(m);
    r.sum = wave_sum(moved<DT>(s, m, r.top));
    if constexpr (NT > 64) {
      if ((tid & 63) == 0) scratch[tid >> 6] = make_float2(r.top, r.sum);
      __syncthreads();
      float2 w[NT / 64];
      float top = -INFINITY;
#pragma unroll
      for (int q = 0; q < NT / 64; ++q) {
        w[q] = scratch[q];
        top = fmaxf(top, w[q].x);
      }
      float sum = 0.f;
#pragma unroll
      for (int q = 0; q < NT / 64; ++q) sum += moved<DT>(w[q].y, w[q].x, top);
      r.top = top, r.sum = sum;
    }
    return r;
  }

  // out[v] = c (onehot(y) - p)
  __device__ __forceinline__ void grad(void *out, int64_t at, int64_t y, const RowStat &r, float coef) const {
    char *row = static_cast<char *>(out) + at * L::kBytes;
    const float scale = -coef / r.sum;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (i * NT >= chunks) break;
      if (tid + i * NT < chunks) {
        float v[L::kPer];
#pragma unroll
        for (int k = 0; k < L::kPer; ++k) v[k] = exp_of<DT>(L::at(c[i], k) - r.top) * scale;
        put(row, i, L::pack(v));
      }
    }
    if (edge_at >= 0) store_any(row, DT, edge_at, round_to(DT, exp_of<DT>(edge - r.top) * scale));
    // the target's element again, by the thread that wrote it
    const int t = static_cast<int>(y) - head;
    const bool mine = t < 0 || t >= chunks * L::kPer ? static_cast<int>(y) == edge_at : tid == t / L::kPer % NT;
    if (y >= 0 && mine)
      store_any(row, DT, y, round_to(DT, fmaf(exp_of<DT>(load_elem<DT>(src, y) - r.top), scale, coef)));
  }

  __device__ __forceinline__ void zero(void *out, int64_t at, int64_t vocab) {
    char *row = static_cast<char *>(out) + at * L::kBytes;
    tid = NT == 64 ? threadIdx.x & 63 : threadIdx.x;
    const int v = static_cast<int>(vocab);
    head = row_head<NT>(row, L::kBytes, v);
    chunks = (v - head) / L::kPer;
    for (int i = 0; i * NT < chunks; ++i)
      if (tid + i * NT < chunks) put(row, i, make_uint4(0, 0, 0, 0));
    const int tail = head + chunks * L::kPer;
    if (tid < head) store_any(row, DT, tid, 0.f);
    if (tid < v - tail) store_any(row, DT, tail + tid, 0.f);
  }

  // Chunk i of this thread, at the alignment of the output's row, which need
  // not be the input's.
  __device__ __forceinline__ void put(char *row, int i, const uint4 &w) const {
    __builtin_nontemporal_store(v4u_any{w.x, w.y, w.z, w.w}, reinterpret_cast<v4u_any *>(row + head * L::kBytes) + tid + i * NT);
  }
};

// A row of any length, read again for each use: first the maximum and sum,
// then the gradient.  For rows past 256 KB, which a block's registers do not hold;
// an element a thread at a time, bound by one load in flight and the running
// maximum's two exponentials an element: log probabilities of 4 x 512 x 151936 bf16
// 260 us (1.7 TB/s), their gradient 409 us (2.6 TB/s).
template <int DT>
struct LongRow {
  static constexpr int NT = 1024;
  const void *z;
  int64_t at, vocab;
  template <bool AGAIN>
  __device__ __forceinline__ void load(const void *p, int64_t i, int64_t v) { z = p, at = i, vocab = v; }
  __device__ __forceinline__ RowStat stat(float2 *scratch) const {
    float m = -INFINITY, s = 0.f;
    for (int64_t v = threadIdx.x; v < vocab; v += NT) {
      const float x = load_elem<DT>(z, at + v);
      const float top = fmaxf(m, x), from = top == -INFINITY ? 0.f : top;
      s = moved<DT>(s, m, top) + exp_of<DT>(x - from);
      m = top;
    }
    RowStat r;
    r.top = wave_max(m);
    r.sum = wave_sum(moved<DT>(s, m, r.top));
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = make_float2(r.top, r.sum);
    __syncthreads();
    float top = -INFINITY, sum = 0.f;
    for (int q = 0; q < NT / 64; ++q) top = fmaxf(top, scratch[q].x);
    for (int q = 0; q < NT / 64; ++q) sum += moved<DT>(scratch[q].y, scratch[q].x, top);
    return {top, sum};
  }
  __device__ __forceinline__ void grad(void *out, int64_t o, int64_t y, const RowStat &r, float coef) const {
    const float scale = -coef / r.sum;
    for (int64_t v = threadIdx.x; v < vocab; v += NT) {
      const float e = exp_of<DT>(load_elem<DT>(z, at + v) - r.top);
      store_any(out, DT, o + v, round_to(DT, v == y ? fmaf(e, scale, coef) : e * scale));
    }
  }
  __device__ __forceinline__ void zero(void *out, int64_t o, int64_t v) const {
    for (int64_t i = threadIdx.x; i < v; i += NT) store_any(out, DT, o + i, 0.f);
  }
};

// Rows of a block and this thread's one; -1 where there is none.
template <int NT>
__device__ __forceinline__ int64_t row_of(int64_t rows) {
  int64_t r = static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x;
  if constexpr (NT == 64) r = r * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  return r < rows ? r : -1;
}

// z_y - lse.  The logarithm as its exponent's part and its fraction's, so that
// only the result is rounded.
template <int DT>
__device__ __forceinline__ float target_lp(const LogitRows &a, int64_t at, int64_t y, const RowStat &r) {
  const float z = y >= 0 && y < a.vocab ? load_elem<DT>(a.z, at + y) : __builtin_nanf("");
  int e;
  float m = frexpf(r.sum, &e);
  if (m < 0.70710678f) m *= 2.f, --e;
  const float hi = static_cast<float>(e) * 0.693145751953125f;  // (15 bits of log 2: exact)
  const float lo = fmaf(static_cast<float>(e), 1.4286068203094172e-6f, logf(m));
  return ((z - r.top) - hi) - lo;
}

// The row kernels' form of a vocabulary: threads and chunks a row.
#define ROW_KERNEL(R, NT, NAME, ...) \
  template <int DT, class R, int NT>  \
  __global__ void __launch_bounds__(NT == 64 ? 256 : NT) NAME(__VA_ARGS__)

ROW_KERNEL(R, NT, logprob_kernel, LogitRows a, float *logprobs, float2 *stats) {
  __shared__ float2 scratch[16];
  const int64_t r = row_of<NT>(a.batch * a.seq);
  if (r < 0) return;
  const int lane = NT == 64 ? threadIdx.x & 63 : threadIdx.x;
  if (a.mask && !a.mask[r]) {
    if (lane == 0) {
      logprobs[r] = 0.f;
      if (stats) stats[r] = make_float2(0.f, 1.f);
    }
    return;
  }
  const int64_t at = r / a.seq * a.batch_stride + r % a.seq * a.row_stride, y = a.targets[r];
  R row;
  if (stats) {
    row.template load<true>(a.z, at, a.vocab);
  } else {
    row.template load<false>(a.z, at, a.vocab);
  }
  const RowStat o = row.stat(scratch);
  const float lp = target_lp<DT>(a, at, y, o);
  if (lane == 0) {
    logprobs[r] = lp;
    if (stats) stats[r] = make_float2(o.top, o.sum);
  }
}

struct CoefArgs {
  const float2 *stats;
  const float *coef, *scale;
  int64_t batch_stride, row_stride;
  void *dz;
};

ROW_KERNEL(R, NT, logprob_back_kernel, LogitRows a, CoefArgs k) {
  int64_t r = row_of<NT>(a.batch * a.seq);
  if (r < 0) return;
  // The rows that the forward read last first: what the last cache still holds
  // of them is read from it.
  r = a.batch * a.seq - 1 - r;
  const int64_t b = r / a.seq, t = r % a.seq;
  R row;
  if (a.mask && !a.mask[r]) {
    row.zero(k.dz, r * a.vocab, a.vocab);
    return;
  }
  float c = k.coef[b * k.batch_stride + t * k.row_stride];
  if (k.scale) c *= *k.scale;
  const int64_t y = a.targets[r];
  if (y < 0 || y >= a.vocab) c = __builtin_nanf("");
  row.template load<false>(a.z, b * a.batch_stride + t * a.row_stride, a.vocab);
  row.grad(k.dz, r * a.vocab, y < a.vocab ? y : -1, {k.stats[r].x, k.stats[r].y}, c);
}

// ---------------------------------------------------------- policy loss ---
struct PolicyArgs {
  LogitRows rows;
  const float *old_lp, *ref_lp, *adv;  // [batch, seq] (old, ref may be null); adv by its strides
  int64_t adv_batch, adv_seq;
  float low, high, kl, scale;  // the ratio's unclipped range
  int32_t per_sequence;
  float *logprobs, *weights, *terms;  // [batch, seq], [batch], [batch, seq]
  void *dz;                           // the gradient, or null
  float2 *stats;                      // or, for one made later, each row's maximum and sum
  float *coef;                        // and d loss / d lp
};

// Threads of a block of 1024 that share one of `items` sequences of `seq`
// tokens, `per` of them in flight in each: as many as leave none idle, at least
// `least`.
static int threads_of(int64_t items, int64_t seq, int per, int least) {
  int share = 1024;
  while (share > least && (1024 / share < items || share / 2 * per >= seq)) share /= 2;
  return share;
}

// A sequence's weight of each of its live tokens: 1 / live tokens of the
// batch, or 1 / (its live tokens * sequences with any).  One block, `share` of
// its threads (16 to 1024) to a sequence, eight tokens of each in flight at once:
// 131072 tokens take 11 us in one sequence.
__global__ void __launch_bounds__(1024) policy_weight_kernel(PolicyArgs a, int share) {
  __shared__ double scratch[16];
  __shared__ uint32_t part[16];
  const int wave = threadIdx.x >> 6, in = threadIdx.x & (share - 1), side = threadIdx.x / share;
  double total = 0;
  for (int64_t b0 = 0; b0 < a.rows.batch; b0 += 1024 / share) {
    const int64_t b = b0 + side;
    uint32_t n = static_cast<uint32_t>(a.rows.seq);
    if (a.rows.mask) {
      n = 0;
      if (b < a.rows.batch) {
        const uint8_t *mask = a.rows.mask + b * a.rows.seq;
        for (int64_t t0 = in; t0 < a.rows.seq; t0 += 8 * share) {
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const int64_t t = t0 + u * share;
            n += mask[t < a.rows.seq ? t : t0] != 0 && t < a.rows.seq;
          }
        }
      }
      n += dpp_mov<0xB1>(n);
      n += dpp_mov<0x4E>(n);
      n += dpp_mov<0x141>(n);
      n += dpp_mov<0x140>(n);
      if (share >= 32) n += __shfl_xor(n, 16);
      if (share >= 64) n += __shfl_xor(n, 32);
      if (share > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) part[wave] = n;
        __syncthreads();
        n = 0;
        for (int w = 0; w < share / 64; ++w) n += part[side * (share / 64) + w];
      }
    }
    if (b < a.rows.batch && in == 0) {
      a.weights[b] = static_cast<float>(n);
      total += a.per_sequence ? static_cast<double>(n > 0) : static_cast<double>(n);
    }
  }
  total = block_sum(total, scratch);
  for (int64_t b = threadIdx.x; b < a.rows.batch; b += 1024) {
    const double n = a.weights[b], d = a.per_sequence ? n * total : total;
    a.weights[b] = n > 0 ? static_cast<float>(a.scale / d) : 0.f;
  }
}

ROW_KERNEL(R, NT, policy_kernel, PolicyArgs a) {
  __shared__ float2 scratch[16];
  const LogitRows &q = a.rows;
  const int64_t r = row_of<NT>(q.batch * q.seq);
  if (r < 0) return;
  const int lane = NT == 64 ? threadIdx.x & 63 : threadIdx.x;
  const int64_t b = r / q.seq, t = r % q.seq;
  R row;
  if (q.mask && !q.mask[r]) {
    if (lane == 0) {
      a.logprobs[r] = a.terms[r] = 0.f;
      if (a.coef) a.stats[r] = make_float2(0.f, 1.f), a.coef[r] = 0.f;
    }
    if (a.dz) row.zero(a.dz, r * q.vocab, q.vocab);
    return;
  }
  const int64_t at = b * q.batch_stride + t * q.row_stride, y = q.targets[r];
  if (a.coef) {
    row.template load<true>(q.z, at, q.vocab);
  } else {
    row.template load<false>(q.z, at, q.vocab);
  }
  const RowStat o = row.stat(scratch);
  const float lp = target_lp<DT>(q, at, y, o);
  const float w = a.weights[b], adv = a.adv[b * a.adv_batch + t * a.adv_seq];
  const bool known = y >= 0 && y < q.vocab;
  const float ratio = a.old_lp ? expf(lp - a.old_lp[r]) : known ? 1.f : __builtin_nanf("");
  // (comparisons that keep a NaN, which fminf and fmaxf would drop)
  const float clipped = ratio < a.low ? a.low : ratio > a.high ? a.high : ratio;
  float term = -(clipped * adv < ratio * adv ? clipped * adv : ratio * adv);
  const bool moves = adv > 0.f ? ratio <= a.high : ratio >= a.low;
  float c = moves ? -ratio * adv : 0.f;
  if (a.ref_lp) {
    const float gap = a.ref_lp[r] - lp, em1 = expm1f(gap);
    term += a.kl * (em1 - gap);
    c -= a.kl * em1;
  }
  // (a comparison drops a NaN that the term has, or its part of c is zero)
  if (!known || term != term) c = __builtin_nanf("");
  if (lane == 0) {
    a.logprobs[r] = lp;
    a.terms[r] = w * term;
    if (a.coef) a.stats[r] = make_float2(o.top, o.sum), a.coef[r] = w * c;
  }
  if (a.dz) row.grad(a.dz, r * q.vocab, y < q.vocab ? y : -1, o, w * c);
}

__global__ void __launch_bounds__(1024) sum_kernel(const float *x, int64_t n, float *out) {
  __shared__ double scratch[16];
  double t = 0;
  for (int64_t i0 = threadIdx.x; i0 < n; i0 += 8 * 1024) {  // (eight loads in flight)
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = x[min(i0 + u * 1024, n - 1)];
#pragma unroll
    for (int u = 0; u < 8; ++u) t += i0 + u * 1024 < n ? v[u] : 0.f;
  }
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
// pair's margin, loss and d loss / d lp.  One block of 16 waves, `share` of them
// (a power of two) to a pair, four tokens of each lane in flight at once.
__global__ void __launch_bounds__(1024) preference_kernel(PreferenceArgs a, int share) {
  __shared__ double scratch[16], part[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lead = wave / share * share;
  double loss = 0;
  for (int64_t p0 = 0; p0 < a.pairs; p0 += 16 / share) {
    const int64_t p = p0 + wave / share;
    double gain = 0;
    if (p < a.pairs) {
      const int64_t at[2] = {p * a.seq, (p + a.pairs) * a.seq};
      for (int64_t t0 = (wave - lead) * 64 + lane; t0 < a.seq; t0 += 4 * 64 * share) {
        // (what a masked token's ref holds is loaded, not used)
        float lp[2][4], ref[2][4];
        bool live[2][4];
#pragma unroll
        for (int side = 0; side < 2; ++side)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int64_t t = t0 + u * 64 * share, i = at[side] + (t < a.seq ? t : t0);
            live[side][u] = t < a.seq && (!a.mask || a.mask[i]);
            lp[side][u] = a.lp[i], ref[side][u] = a.ref[i];
          }
        double g[2];
#pragma unroll
        for (int side = 0; side < 2; ++side) {
          float d[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) d[u] = live[side][u] ? lp[side][u] - ref[side][u] : 0.f;
          g[side] = (static_cast<double>(d[0]) + d[1]) + (static_cast<double>(d[2]) + d[3]);
        }
        gain += g[0] - g[1];
      }
    }
    gain = wave_sum(gain);
    __syncthreads();
    if (lane == 0) part[wave] = gain;
    __syncthreads();
    if (p < a.pairs && wave == lead && lane == 0) {
      for (int w = 1; w < share; ++w) gain += part[lead + w];
      // (the margin is rounded once; FP32 functions of it are within 2^-22)
      const float m = static_cast<float>(a.beta * gain), e = expf(-fabsf(m)), soft = log1pf(e);
      // (a term of weight zero is left out: it may be infinite)
      if (a.smoothing < 1) loss += (1 - a.smoothing) * (soft - (m > 0.f ? 0.f : m));
      if (a.smoothing > 0) loss += a.smoothing * (soft + (m < 0.f ? 0.f : m));
      a.margins[p] = m;
      // sigmoid(m) and sigmoid(-m) are 1 / (1 + e) and e / (1 + e) or the other way round
      const double up = static_cast<double>(m > 0.f ? 1.f : e) / (1.0 + e), down = static_cast<double>(m > 0.f ? e : 1.f) / (1.0 + e);
      const double slope = a.beta * (a.smoothing * up - (1 - a.smoothing) * down) / a.pairs;
      a.coef[p] = static_cast<float>(slope);
      a.coef[p + a.pairs] = static_cast<float>(-slope);
    }
  }
  loss = block_sum(loss, scratch);
  if (threadIdx.x == 0) *a.loss = static_cast<float>(a.pairs ? loss / a.pairs : 0.);
}

// x *= *scale, unless it is one, in 16-byte chunks and single elements behind
// them.  8 x 1024 x 50257 bf16: 339 us, the copy's rate (element by
// element 589 us).
template <int DT>
__global__ void __launch_bounds__(256) scale_kernel(void *x, int64_t n, int64_t chunks, const float *scale) {
  using L = Logit<DT>;
  const float s = *scale;
  if (s == 1.f) return;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, step = static_cast<int64_t>(gridDim.x) * 256;
  uint4 *p = static_cast<uint4 *>(x);
  for (int64_t i = first; i < chunks; i += step) {
    const uint4 c = p[i];
    float v[L::kPer];
#pragma unroll
    for (int k = 0; k < L::kPer; ++k) v[k] = L::at(c, k) * s;
    p[i] = L::pack(v);
  }
  for (int64_t i = chunks * L::kPer + first; i < n; i += step) store_any(x, DT, i, round_to(DT, load_elem<DT>(x, i) * s));
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

// A launch holds fewer than 2^32 threads along one axis, so the blocks of many
// rows lie along two.
static dim3 row_grid(int64_t blocks) {
  const int64_t x = std::min<int64_t>(blocks, int64_t{1} << 20);
  return dim3(static_cast<unsigned>(x), static_cast<unsigned>(ceil_div(blocks, x)));
}

// Threads and chunks by the row's length in 16-byte chunks: a wave a row (four
// rows a block) up to 8 KB, so that a short row waits for no other wave; then
// 256, 512 and 1024 threads with up to 16 chunks each, the fewest that hold
// the row, so that several rows share a CU; past 256 KB the row is read twice.
#define LOGITS_BY_ROW(DT, vocab, rows, NAME, ...)                                                                   \
  do {                                                                                                              \
    const int64_t chunks_ = ceil_div(vocab, Logit<DT>::kPer);                                                       \
    const dim3 grid_ = row_grid(chunks_ <= 512 ? ceil_div(rows, 4) : (rows));                                       \
    if (chunks_ <= 512) {                                                                                           \
      hipLaunchKernelGGL((NAME<DT, Row<DT, 64, 8>, 64>), grid_, dim3(256), 0, st, __VA_ARGS__);                     \
    } else if (chunks_ <= 4096) {                                                                                   \
      hipLaunchKernelGGL((NAME<DT, Row<DT, 256, 16>, 256>), grid_, dim3(256), 0, st, __VA_ARGS__);                  \
    } else if (chunks_ <= 8192) {                                                                                   \
      hipLaunchKernelGGL((NAME<DT, Row<DT, 512, 16>, 512>), grid_, dim3(512), 0, st, __VA_ARGS__);                  \
    } else if (chunks_ <= 16384) {                                                                                  \
      hipLaunchKernelGGL((NAME<DT, Row<DT, 1024, 16>, 1024>), grid_, dim3(1024), 0, st, __VA_ARGS__);               \
    } else {                                                                                                        \
      hipLaunchKernelGGL((NAME<DT, LongRow<DT>, 1024>), grid_, dim3(1024), 0, st, __VA_ARGS__);                     \
    }                                                                                                               \
  } while (0)

#define LOGITS_LAUNCH(dtype, vocab, rows, NAME, ...)                \
  do {                                                              \
    if ((dtype) == SMX_F32) {                                       \
      LOGITS_BY_ROW(SMX_F32, vocab, rows, NAME, __VA_ARGS__);       \
    } else if ((dtype) == SMX_BF16) {                               \
      LOGITS_BY_ROW(SMX_BF16, vocab, rows, NAME, __VA_ARGS__);      \
    } else {                                                        \
      LOGITS_BY_ROW(SMX_F16, vocab, rows, NAME, __VA_ARGS__);       \
    }                                                               \
  } while (0)

}  // namespace smx

using namespace smx;

extern "C" int smx_token_logprobs(const void *logits, int dtype, int64_t batch, int64_t seq, int64_t vocab,
                                  int64_t batch_stride, int64_t row_stride, const int64_t *targets,
                                  const uint8_t *mask, float *logprobs, float *stats, void *stream) {
  const int rc = logits_check("token_logprobs", logits, dtype, batch, seq, vocab, batch_stride, row_stride, targets);
  if (rc != SMX_OK || batch * seq == 0) return rc;
  SMX_REQUIRE(logprobs, SMX_EINVAL, "token_logprobs: null output");
  SMX_REQUIRE(reinterpret_cast<uintptr_t>(stats) % 8 == 0, SMX_EALIGN, "token_logprobs: stats must be 8-byte aligned");
  const LogitRows a{logits, targets, mask, batch, seq, vocab, batch_stride, row_stride};
  const auto st = static_cast<hipStream_t>(stream);
  LOGITS_LAUNCH(dtype, vocab, batch * seq, logprob_kernel, a, logprobs, reinterpret_cast<float2 *>(stats));
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
  SMX_REQUIRE(reinterpret_cast<uintptr_t>(stats) % 8 == 0, SMX_EALIGN,
              "token_logprobs_backward: stats must be 8-byte aligned");
  const LogitRows a{logits, targets, mask, batch, seq, vocab, batch_stride, row_stride};
  const CoefArgs k{reinterpret_cast<const float2 *>(stats), coef, scale, coef_batch_stride, coef_row_stride, dlogits};
  const auto st = static_cast<hipStream_t>(stream);
  LOGITS_LAUNCH(dtype, vocab, batch * seq, logprob_back_kernel, a, k);
  return check_launch("token_logprobs_backward");
}

extern "C" int64_t smx_policy_loss_workspace_bytes(int64_t batch, int64_t seq) {
  if (batch < 0 || seq < 0) return SMX_EINVAL;
  return (batch + batch * seq) * static_cast<int64_t>(sizeof(float));
}

namespace smx {
// What both entry points take: logits and targets, the policies' log probabilities, the loss.
struct PolicyCall {
  LogitRows rows;
  int dtype;
  const float *old_lp, *ref_lp, *adv;
  int64_t adv_batch, adv_seq;
  double clip_low, clip_high, kl, scale;
  int reduction;
  float *loss, *logprobs;
  void *workspace;
  int64_t workspace_bytes;
};

static int policy_run(const char *what, const PolicyCall &c, void *dz, float *stats, float *coef, hipStream_t st) {
  const auto msg = [&](const char *m) { return std::string(what) + ": " + m; };
  const LogitRows &q = c.rows;
  const int rc = logits_check(what, q.z, c.dtype, q.batch, q.seq, q.vocab, q.batch_stride, q.row_stride, q.targets);
  if (rc != SMX_OK) return rc;
  SMX_REQUIRE(c.reduction == SMX_MEAN_TOKEN || c.reduction == SMX_MEAN_SEQUENCE, SMX_EINVAL, msg("unknown reduction"));
  SMX_REQUIRE(c.clip_low >= 0 && c.clip_low <= 1 && c.clip_high >= 0, SMX_EINVAL,
              msg("clip_low must be in [0, 1] and clip_high not negative"));
  SMX_REQUIRE(c.loss, SMX_EINVAL, msg("null loss"));
  const int64_t rows = q.batch * q.seq;
  PolicyArgs a{};
  if (rows > 0) {
    SMX_REQUIRE(c.logprobs && c.adv, SMX_EINVAL, msg("null pointer"));
    SMX_REQUIRE(c.workspace && c.workspace_bytes >= smx_policy_loss_workspace_bytes(q.batch, q.seq), SMX_EWORKSPACE,
                msg("workspace too small"));
    a.rows = q, a.old_lp = c.old_lp, a.ref_lp = c.ref_lp, a.adv = c.adv;
    a.adv_batch = c.adv_batch, a.adv_seq = c.adv_seq;
    a.low = static_cast<float>(1 - c.clip_low), a.high = static_cast<float>(1 + c.clip_high);
    a.kl = static_cast<float>(c.kl), a.scale = static_cast<float>(c.scale);
    a.per_sequence = c.reduction == SMX_MEAN_SEQUENCE;
    a.logprobs = c.logprobs, a.weights = static_cast<float *>(c.workspace), a.terms = a.weights + q.batch;
    a.dz = dz, a.stats = reinterpret_cast<float2 *>(stats), a.coef = coef;
    hipLaunchKernelGGL(policy_weight_kernel, dim3(1), dim3(1024), 0, st, a, threads_of(q.batch, q.seq, 8, 16));
    LOGITS_LAUNCH(c.dtype, q.vocab, rows, policy_kernel, a);
    const int lrc = check_launch(what);
    if (lrc != SMX_OK) return lrc;
  }
  hipLaunchKernelGGL(sum_kernel, dim3(1), dim3(1024), 0, st, static_cast<const float *>(a.terms), rows, c.loss);
  return check_launch(what);
}
}  // namespace smx

extern "C" int smx_policy_loss(const void *logits, int dtype, int64_t batch, int64_t seq, int64_t vocab,
                               int64_t batch_stride, int64_t row_stride, const int64_t *targets, const uint8_t *mask,
                               const float *old_logprobs, const float *ref_logprobs, const float *advantages,
                               int64_t adv_batch_stride, int64_t adv_row_stride, double clip_low, double clip_high,
                               double kl_coef, int reduction, double scale, float *loss, float *logprobs,
                               void *dlogits, void *workspace, int64_t workspace_bytes, void *stream) {
  const PolicyCall c{{logits, targets, mask, batch, seq, vocab, batch_stride, row_stride}, dtype, old_logprobs,
                     ref_logprobs, advantages, adv_batch_stride, adv_row_stride, clip_low, clip_high, kl_coef, scale,
                     reduction, loss, logprobs, workspace, workspace_bytes};
  return policy_run("policy_loss", c, dlogits, nullptr, nullptr, static_cast<hipStream_t>(stream));
}

extern "C" int smx_policy_loss_coef(const void *logits, int dtype, int64_t batch, int64_t seq, int64_t vocab,
                                    int64_t batch_stride, int64_t row_stride, const int64_t *targets,
                                    const uint8_t *mask, const float *old_logprobs, const float *ref_logprobs,
                                    const float *advantages, int64_t adv_batch_stride, int64_t adv_row_stride,
                                    double clip_low, double clip_high, double kl_coef, int reduction, double scale,
                                    float *loss, float *logprobs, float *stats, float *coef, void *workspace,
                                    int64_t workspace_bytes, void *stream) {
  const PolicyCall c{{logits, targets, mask, batch, seq, vocab, batch_stride, row_stride}, dtype, old_logprobs,
                     ref_logprobs, advantages, adv_batch_stride, adv_row_stride, clip_low, clip_high, kl_coef, scale,
                     reduction, loss, logprobs, workspace, workspace_bytes};
  SMX_REQUIRE((stats && coef) || batch == 0 || seq == 0, SMX_EINVAL, "policy_loss_coef: null stats or coef");
  SMX_REQUIRE(reinterpret_cast<uintptr_t>(stats) % 8 == 0, SMX_EALIGN, "policy_loss_coef: stats must be 8-byte aligned");
  return policy_run("policy_loss_coef", c, nullptr, stats, coef, static_cast<hipStream_t>(stream));
}

extern "C" int smx_preference_loss(const float *logprobs, const float *ref_logprobs, const uint8_t *mask,
                                   int64_t pairs, int64_t seq, double beta, double label_smoothing, float *loss,
                                   float *margins, float *coef, void *stream) {
  SMX_REQUIRE(pairs >= 0 && seq >= 0, SMX_ESHAPE, "preference_loss: negative size");
  SMX_REQUIRE(label_smoothing >= 0 && label_smoothing <= 1, SMX_EINVAL, "preference_loss: label_smoothing must be in [0, 1]");
  SMX_REQUIRE(loss && (pairs == 0 || (margins && coef)), SMX_EINVAL, "preference_loss: null output");
  SMX_REQUIRE(pairs == 0 || seq == 0 || (logprobs && ref_logprobs), SMX_EINVAL, "preference_loss: null log probabilities");
  const PreferenceArgs a{logprobs, ref_logprobs, mask, pairs, seq, beta, label_smoothing, loss, margins, coef};
  hipLaunchKernelGGL(preference_kernel, dim3(1), dim3(1024), 0, static_cast<hipStream_t>(stream), a,
                     threads_of(pairs, seq, 4, 64) / 64);
  return check_launch("preference_loss");
}

extern "C" int smx_scale(void *x, int dtype, int64_t n, const float *scale, void *stream) {
  SMX_REQUIRE(dtype == SMX_F32 || dtype == SMX_BF16 || dtype == SMX_F16, SMX_EDTYPE, "scale: dtype must be f32, bf16 or f16");
  SMX_REQUIRE(n >= 0, SMX_ESHAPE, "scale: negative size");
  if (n == 0) return SMX_OK;
  SMX_REQUIRE(x && scale, SMX_EINVAL, "scale: null pointer");
  const int64_t per = dtype == SMX_F32 ? 4 : 8, chunks = reinterpret_cast<uintptr_t>(x) % 16 == 0 ? n / per : 0;
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(2048, ceil_div(chunks ? chunks : n, 256))));
  const auto st = static_cast<hipStream_t>(stream);
  if (dtype == SMX_F32) {
    hipLaunchKernelGGL((scale_kernel<SMX_F32>), grid, dim3(256), 0, st, x, n, chunks, scale);
  } else if (dtype == SMX_BF16) {
    hipLaunchKernelGGL((scale_kernel<SMX_BF16>), grid, dim3(256), 0, st, x, n, chunks, scale);
  } else {
    hipLaunchKernelGGL((scale_kernel<SMX_F16>), grid, dim3(256), 0, st, x, n, chunks, scale);
  }
  return check_launch("scale");
}
