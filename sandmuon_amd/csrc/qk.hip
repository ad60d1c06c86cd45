// RMS norm of every query and key head with its rotary position rotation, and
// the gradient, each in one pass over queries and keys together.
//
//   n = x * rsqrt(mean(x^2) + eps) * w;  each pair (a, b) of n's first `rot`
//   elements turns by the position's angle: (a c - b s, a s + b c).
// Backward: the pairs of dy turn back (g), gw = g w, u = x rsqrt(...):
//   dx = rsqrt(...) (gw - u mean(gw u)),   dw = sum over heads of g u.
//
// Bound by HBM: the vectors are read once and written once; the angle tables
// stay in cache.  A group of lanes owns one head's vector, 8 elements a lane,
// chosen so that both elements of a pair are in one lane: 8 neighbours where
// pairs are neighbours, 4 of each half where they are half a rotation apart.
// The norm is then a sum over the group in DPP moves, and nothing else
// crosses lanes.
//
// Measured at 16 x 1024 tokens of 12 + 12 heads of 64, bf16: forward 25 us (4.0
// TB/s of vectors read and written), backward 36 us (4.2 TB/s) and 4 us for the
// weights' gradients; more vectors a thread at once change neither.  64 x (16 +
// 4) heads of 128, one token: 3.5 us.
#include "common.h"

#include <algorithm>
#include <type_traits>

namespace smx {

struct QkSide {
  const void *x, *w, *dy;
  void *y;      // result (forward) or dx (backward)
  float *part;  // [blocks of this side, dim] partial dw, or null
  int64_t xs[3], ys[3], ds[3];
  uint32_t heads, heads_mul, heads_shift, items;
  int32_t w_dtype, blocks;
};

struct QkArgs {
  QkSide side[2];
  const float *cos, *sin;
  const int64_t *pos;
  int64_t pos_stride[2], pos0, table_rows;
  uint32_t seq, seq_mul, seq_shift;
  int32_t dim, rot, dtype;
  float eps, inv_dim;
};

// n / d for n < 2^31 by a multiplication (round-up method: m = ceil(2^(32+s) / d)).
static void fast_div(uint32_t d, uint32_t *mul, uint32_t *shift) {
  uint32_t s = 0;
  while ((uint64_t{1} << s) < d) ++s;
  if (s == 0) {
    *mul = 0, *shift = 0;
    return;
  }
  --s;
  *mul = static_cast<uint32_t>(((uint64_t{1} << (32 + s)) + d - 1) / d);
  *shift = s;
}
__device__ __forceinline__ uint32_t div_by(uint32_t n, uint32_t mul, uint32_t shift) {
  return mul ? __umulhi(n, mul) >> shift : n;
}

struct QkItem {
  int64_t b, t, h;
};

__device__ __forceinline__ QkItem qk_item(const QkArgs &a, const QkSide &s, uint32_t i) {
  const uint32_t token = div_by(i, s.heads_mul, s.heads_shift);
  const uint32_t b = div_by(token, a.seq_mul, a.seq_shift);
  return {b, token - b * a.seq, i - token * s.heads};
}

__device__ __forceinline__ int64_t qk_at(const int64_t *st, const QkItem &i) {
  return i.b * st[0] + i.t * st[1] + i.h * st[2];
}

// The item's position in the tables, or -1 where they do not hold it.
__device__ __forceinline__ int64_t qk_position(const QkArgs &a, const QkItem &i) {
  const int64_t p = a.pos ? a.pos[i.b * a.pos_stride[0] + i.t * a.pos_stride[1]] : a.pos0 + i.t;
  return p >= 0 && p < a.table_rows ? p : -1;
}

// ------------------------------------------------------- whole vectors ---
// Four elements at p + i.
template <int DT>
__device__ __forceinline__ void load4(const void *p, int64_t i, float *v) {
  if constexpr (DT == SMX_F32) {
    const float4 a = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  } else {
    const uint2 a = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + i);
    v[0] = load_elem<DT>(&a, 0), v[1] = load_elem<DT>(&a, 1);
    v[2] = load_elem<DT>(&a, 2), v[3] = load_elem<DT>(&a, 3);
  }
}

template <int DT>
__device__ __forceinline__ void store4(void *p, int64_t i, const float *v) {
  if constexpr (DT == SMX_F32) {
    *reinterpret_cast<float4 *>(static_cast<float *>(p) + i) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    typedef std::conditional_t<DT == SMX_BF16, __bf16, _Float16> T;
    typedef T v4t __attribute__((ext_vector_type(4)));
    *reinterpret_cast<v4t *>(static_cast<uint16_t *>(p) + i) =
        v4t{static_cast<T>(v[0]), static_cast<T>(v[1]), static_cast<T>(v[2]), static_cast<T>(v[3])};
  }
}

// Sum over groups of G lanes (a power of two), in every lane of the group.
template <int G>
__device__ __forceinline__ float group_sum(float v) {
  if constexpr (G >= 2) v += dpp_mov<0xB1>(v);
  if constexpr (G >= 4) v += dpp_mov<0x4E>(v);
  if constexpr (G >= 8) v += dpp_mov<0x141>(v);
  if constexpr (G >= 16) v += dpp_mov<0x140>(v);
  if constexpr (G >= 32) v += __shfl_xor(v, 16);
  if constexpr (G >= 64) v += __shfl_xor(v, 32);
  return v;
}

constexpr int kQkThreads = 256;

// A lane's 8 elements: v[0..3] at `lo`, v[4..7] at `hi`; where `turned`, pair
// k is (v[k], v[4 + k]) (HALF) or (v[2k], v[2k + 1]), at table column `col`.
struct QkLane {
  int lo, hi, col;
  bool active, turned;
};

template <bool HALF>
__device__ __forceinline__ QkLane qk_lane(const QkArgs &a, int j) {
  QkLane l;
  l.active = 8 * j < a.dim;
  l.turned = 8 * j < a.rot;
  l.col = 4 * j;
  const bool split = HALF && l.turned;
  l.lo = split ? 4 * j : 8 * j;
  l.hi = split ? a.rot / 2 + 4 * j : 8 * j + 4;
  return l;
}

template <bool HALF>
__device__ __forceinline__ void qk_turn(float *v, const float *c, const float *s, float sign) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float &x = HALF ? v[k] : v[2 * k], &y = HALF ? v[4 + k] : v[2 * k + 1];
    const float sk = sign * s[k], p = x * c[k] - y * sk, q = x * sk + y * c[k];
    x = p, y = q;
  }
}

template <int DT, int G, bool HALF, bool BACK>
__global__ void __launch_bounds__(kQkThreads) qk_kernel(QkArgs a) {
  const QkSide &s = a.side[blockIdx.y];
  const int nblocks = s.blocks, block = blockIdx.x;
  if (block >= nblocks) return;
  constexpr int kGroups = kQkThreads / G;
  const int j = threadIdx.x & (G - 1);
  const QkLane l = qk_lane<HALF>(a, j);
  float w[8], dw[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    w[k] = 1.f, dw[k] = 0.f;
    if (s.w && l.active) w[k] = load_any(s.w, s.w_dtype, (k < 4 ? l.lo : l.hi - 4) + k);
  }
  const uint32_t step = static_cast<uint32_t>(nblocks) * kGroups;
  for (uint32_t i = block * kGroups + threadIdx.x / G; i < s.items; i += step) {
    const QkItem it = qk_item(a, s, i);
    float x[8] = {}, g[8] = {}, c[4], sn[4];
    if (l.active) {
      const int64_t at = qk_at(s.xs, it);
      load4<DT>(s.x, at + l.lo, x);
      load4<DT>(s.x, at + l.hi, x + 4);
      if constexpr (BACK) {
        const int64_t dat = qk_at(s.ds, it);
        load4<DT>(s.dy, dat + l.lo, g);
        load4<DT>(s.dy, dat + l.hi, g + 4);
      }
    }
    if (l.turned) {
      const int64_t p = qk_position(a, it);
      if (p >= 0) {
        load4<SMX_F32>(a.cos, p * (a.rot / 2) + l.col, c);
        load4<SMX_F32>(a.sin, p * (a.rot / 2) + l.col, sn);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) c[k] = sn[k] = __builtin_nanf("");
      }
    }
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) sum = fmaf(x[k], x[k], sum);
    const float r = rsqrtf(group_sum<G>(sum) * a.inv_dim + a.eps);
    float y[8];
    if constexpr (!BACK) {
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] = x[k] * r * w[k];
      if (l.turned) qk_turn<HALF>(y, c, sn, 1.f);
    } else {
      if (l.turned) qk_turn<HALF>(g, c, sn, -1.f);
      float dot = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        x[k] *= r;
        dw[k] = fmaf(g[k], x[k], dw[k]);
        g[k] *= w[k];
        dot = fmaf(g[k], x[k], dot);
      }
      dot = group_sum<G>(dot) * a.inv_dim;
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] = r * (g[k] - x[k] * dot);
    }
    if (l.active) {
      const int64_t at = qk_at(s.ys, it);
      store4<DT>(s.y, at + l.lo, y);
      store4<DT>(s.y, at + l.hi, y + 4);
    }
  }
  if constexpr (BACK) {
    // dw over the groups of a wave, then over the waves, in a fixed order
    if (s.part) {
      __shared__ float red[kQkThreads / 64][G][8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
#pragma unroll
        for (int o = G; o < 64; o *= 2) dw[k] += __shfl_xor(dw[k], o);
        if ((threadIdx.x & 63) < G) red[threadIdx.x >> 6][j][k] = dw[k];
      }
      __syncthreads();
      float *part = s.part + static_cast<int64_t>(block) * a.dim;
      for (int e = threadIdx.x; e < 8 * G; e += kQkThreads) {
        const QkLane o = qk_lane<HALF>(a, e >> 3);
        const int k = e & 7;
        if (o.active)
          part[(k < 4 ? o.lo : o.hi - 4) + k] =
              (red[0][e >> 3][k] + red[1][e >> 3][k]) + (red[2][e >> 3][k] + red[3][e >> 3][k]);
      }
    }
  }
}

// --------------------------------------------------------- any geometry ---
// Dimensions, strides and addresses of any kind: a wave owns a vector and
// goes over its elements three times, one (or one pair) a lane.  16 x 1024 tokens of
// 12 + 12 heads of 60, bf16: forward 125 us, backward with weights 251 us (0.8 and
// 0.6 TB/s, bound by single-element accesses; heads of 64 take the kernel above).
template <int DT, bool BACK>
__global__ void __launch_bounds__(kQkThreads) qk_any_kernel(QkArgs a, int half) {
  const QkSide &s = a.side[blockIdx.y];
  const int nblocks = s.blocks, block = blockIdx.x;
  if (block >= nblocks) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int pairs = a.rot / 2, units = pairs + a.dim - a.rot;  // a unit: a pair, or an element that does not turn
  const uint32_t step = static_cast<uint32_t>(nblocks) * 4;
  for (uint32_t i = block * 4 + wave; i < s.items; i += step) {
    const QkItem it = qk_item(a, s, i);
    const int64_t at = qk_at(s.xs, it), yat = qk_at(s.ys, it), dat = qk_at(s.ds, it);
    float sum = 0.f;
    for (int e = lane; e < a.dim; e += 64) {
      const float v = load_elem<DT>(s.x, at + e);
      sum = fmaf(v, v, sum);
    }
    const float r = rsqrtf(wave_sum(sum) * a.inv_dim + a.eps);
    const int64_t p = qk_position(a, it);
    float dot = 0.f;
    for (int pass = BACK ? 0 : 1; pass < 2; ++pass) {
      for (int u = lane; u < units; u += 64) {
        const bool turned = u < pairs;
        int i0 = u + pairs, i1 = i0;  // (an element past the pairs: u - pairs + rot)
        float c = 1.f, sn = 0.f;
        if (turned) {
          i0 = half ? u : 2 * u;
          i1 = half ? u + pairs : 2 * u + 1;
          c = p >= 0 ? a.cos[p * pairs + u] : __builtin_nanf("");
          sn = p >= 0 ? a.sin[p * pairs + u] : __builtin_nanf("");
        }
        const float w0 = s.w ? load_any(s.w, s.w_dtype, i0) : 1.f, w1 = s.w ? load_any(s.w, s.w_dtype, i1) : 1.f;
        const float x0 = load_elem<DT>(s.x, at + i0) * r, x1 = load_elem<DT>(s.x, at + i1) * r;
        if constexpr (!BACK) {
          const float n0 = x0 * w0, n1 = x1 * w1;
          store_any(s.y, DT, yat + i0, round_to(DT, turned ? n0 * c - n1 * sn : n0));
          if (turned) store_any(s.y, DT, yat + i1, round_to(DT, n0 * sn + n1 * c));
        } else {
          const float d0 = load_elem<DT>(s.dy, dat + i0), d1 = load_elem<DT>(s.dy, dat + i1);
          const float g0 = turned ? d0 * c + d1 * sn : d0, g1 = turned ? d1 * c - d0 * sn : 0.f;
          if (pass == 0) {
            dot = fmaf(g0 * w0, x0, dot);
            if (turned) dot = fmaf(g1 * w1, x1, dot);
          } else {
            store_any(s.y, DT, yat + i0, round_to(DT, r * (g0 * w0 - x0 * dot)));
            if (turned) store_any(s.y, DT, yat + i1, round_to(DT, r * (g1 * w1 - x1 * dot)));
            if (s.part) {
              // each wave keeps its own partial row, each lane its own elements of it
              float *o = s.part + (static_cast<int64_t>(block) * 4 + wave) * a.dim;
              o[i0] += g0 * x0;
              if (turned) o[i1] += g1 * x1;
            }
          }
        }
      }
      if (BACK && pass == 0) dot = wave_sum(dot) * a.inv_dim;
    }
  }
}

// dw[e] = sum over the partial rows, in FP64 and a fixed order: a block per side
// and 16 elements, each from 64 threads.
struct QkDwArgs {
  const float *part[2];
  void *dw[2];
  int32_t rows[2], dtype[2], dim;
};
__global__ void __launch_bounds__(1024) qk_dw_kernel(QkDwArgs a) {
  __shared__ double red[64][17];
  const int which = blockIdx.y, col = threadIdx.x & 15, q = threadIdx.x >> 4, e = blockIdx.x * 16 + col;
  const float *part = a.part[which];
  if (!a.dw[which]) return;
  double t = 0;
  if (e < a.dim) {
    int r = q;
    for (; r + 7 * 64 < a.rows[which]; r += 8 * 64) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = part[static_cast<int64_t>(r + 64 * k) * a.dim + e];
#pragma unroll
      for (int k = 0; k < 8; ++k) t += v[k];
    }
    for (; r < a.rows[which]; r += 64) t += part[static_cast<int64_t>(r) * a.dim + e];
  }
  red[q][col] = t;
  __syncthreads();
  if (q < 8) {
    for (int k = 1; k < 8; ++k) t += red[q + 8 * k][col];
    red[q][col] = t;
  }
  __syncthreads();
  if (q == 0 && e < a.dim) {
    for (int k = 1; k < 8; ++k) t += red[k][col];
    store_any(a.dw[which], a.dtype[which], e, round_to(a.dtype[which], static_cast<float>(t)));
  }
}

__global__ void __launch_bounds__(256) qk_zero_kernel(float *p, int64_t n) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256)
    p[i] = 0.f;
}

// ----------------------------------------------------------------- host ---
static bool qk_float(int d) { return d == SMX_F32 || d == SMX_BF16 || d == SMX_F16; }

struct QkPlan {
  bool vec;
  int group, blocks[2];
  int rows[2];  // partial rows of dw
};

static bool qk_aligned(const void *p, const int64_t *st, int64_t e) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && st[0] * e % 16 == 0 && st[1] * e % 16 == 0 && st[2] * e % 16 == 0;
}

// Lane groups of 8 elements where the vectors and rotations divide into them
// and every vector starts on 16 bytes; a wave per vector otherwise.
static QkPlan qk_plan(const smx_qk_desc &d, bool back) {
  QkPlan p{};
  const int64_t e = d.dtype == SMX_F32 ? 4 : 2;
  p.vec = d.dim % 8 == 0 && d.rot % 8 == 0 && d.dim <= 512 &&
          (d.rot == 0 || (reinterpret_cast<uintptr_t>(d.cos) % 16 == 0 && reinterpret_cast<uintptr_t>(d.sin) % 16 == 0));
  for (const smx_qk_side &s : {d.q, d.k}) {
    if (s.heads == 0) continue;
    p.vec = p.vec && qk_aligned(s.x, s.x_stride, e) && qk_aligned(s.y, s.y_stride, e) &&
            (!back || qk_aligned(s.dy, s.dy_stride, e));
  }
  p.group = 64;
  if (p.vec)
    for (p.group = 4; p.group * 8 < d.dim;) p.group *= 2;
  const int per_block = kQkThreads / p.group;
  // as many blocks as fill every CU eight times over, shared by q and k
  const int64_t all = d.batch * d.seq * (d.q.heads + d.k.heads);
  const int64_t most = 2048;
  const int64_t want = std::max<int64_t>(1, std::min(most, ceil_div(all, per_block)));
  for (int i = 0; i < 2; ++i) {
    const smx_qk_side &s = i ? d.k : d.q;
    const int64_t items = d.batch * d.seq * s.heads;
    p.blocks[i] = items == 0 ? 0
                             : static_cast<int>(std::max<int64_t>(
                                   1, std::min(ceil_div(items, per_block), ceil_div(want * items, all))));
    p.rows[i] = p.vec ? p.blocks[i] : 4 * p.blocks[i];
  }
  return p;
}

static int qk_check(const char *what, const smx_qk_desc *d, bool back) {
  const auto msg = [&](const char *m) { return std::string(what) + ": " + m; };
  SMX_REQUIRE(d, SMX_EINVAL, msg("null descriptor"));
  SMX_REQUIRE(qk_float(d->dtype), SMX_EDTYPE, msg("dtype must be f32, bf16 or f16"));
  SMX_REQUIRE(d->style == SMX_ROTARY_HALF || d->style == SMX_ROTARY_INTERLEAVED, SMX_EINVAL, msg("unknown rotary style"));
  SMX_REQUIRE(d->batch >= 0 && d->seq >= 0 && d->q.heads >= 0 && d->k.heads >= 0, SMX_ESHAPE, msg("negative size"));
  SMX_REQUIRE(d->dim >= 1 && d->dim <= 65536, SMX_ESHAPE, msg("head dimension must be in [1, 65536]"));
  SMX_REQUIRE(d->rot >= 0 && d->rot <= d->dim && d->rot % 2 == 0, SMX_ESHAPE, msg("rot must be even and at most dim"));
  SMX_REQUIRE(d->rot == 0 || (d->cos && d->sin && d->table_rows >= 0), SMX_EINVAL, msg("null cos or sin table"));
  SMX_REQUIRE(d->eps >= 0, SMX_EINVAL, msg("eps must not be negative"));
  const int64_t most = int64_t{1} << 31;
  SMX_REQUIRE(d->batch < most && d->seq < most, SMX_ESHAPE, msg("more than 2^31 - 1 tokens"));
  const int64_t tokens = d->batch * d->seq;
  for (const smx_qk_side *s : {&d->q, &d->k}) {
    if (s->heads == 0 || tokens == 0) continue;
    // (half of 2^32: a group's index may step past the last vector)
    SMX_REQUIRE(tokens < most && s->heads < most && tokens * s->heads < most, SMX_ESHAPE, msg("more than 2^31 - 1 vectors"));
    SMX_REQUIRE(s->x && s->y, SMX_EINVAL, msg("null pointer"));
    SMX_REQUIRE(!back || s->dy, SMX_EINVAL, msg("null cotangent"));
    SMX_REQUIRE(!s->weight || qk_float(s->weight_dtype), SMX_EDTYPE, msg("weight dtype must be f32, bf16 or f16"));
    SMX_REQUIRE(!back || !s->dw || s->weight, SMX_EINVAL, msg("dw without a weight"));
  }
  return SMX_OK;
}

static QkArgs qk_args(const smx_qk_desc &d, const QkPlan &p, float *const part[2], bool back) {
  QkArgs a{};
  for (int i = 0; i < 2; ++i) {
    const smx_qk_side &s = i ? d.k : d.q;
    QkSide &o = a.side[i];
    o.x = s.x, o.w = s.weight, o.dy = back ? s.dy : nullptr, o.y = s.y, o.part = part[i];
    for (int k = 0; k < 3; ++k) o.xs[k] = s.x_stride[k], o.ys[k] = s.y_stride[k], o.ds[k] = back ? s.dy_stride[k] : 0;
    o.heads = static_cast<uint32_t>(std::max<int64_t>(1, s.heads));
    fast_div(o.heads, &o.heads_mul, &o.heads_shift);
    o.items = static_cast<uint32_t>(d.batch * d.seq * s.heads);
    o.w_dtype = s.weight_dtype, o.blocks = p.blocks[i];
  }
  a.cos = d.cos, a.sin = d.sin, a.pos = d.positions, a.pos0 = d.position0;
  a.pos_stride[0] = d.pos_stride[0], a.pos_stride[1] = d.pos_stride[1], a.table_rows = d.table_rows;
  a.seq = static_cast<uint32_t>(d.seq);
  fast_div(a.seq, &a.seq_mul, &a.seq_shift);
  a.dim = static_cast<int32_t>(d.dim), a.rot = static_cast<int32_t>(d.rot), a.dtype = d.dtype;
  a.eps = static_cast<float>(d.eps), a.inv_dim = static_cast<float>(1.0 / static_cast<double>(d.dim));
  return a;
}

template <int DT, bool BACK, bool HALF>
static void qk_launch_group(const QkArgs &a, int group, dim3 grid, hipStream_t st) {
  switch (group) {
    case 4: hipLaunchKernelGGL((qk_kernel<DT, 4, HALF, BACK>), grid, dim3(kQkThreads), 0, st, a); break;
    case 8: hipLaunchKernelGGL((qk_kernel<DT, 8, HALF, BACK>), grid, dim3(kQkThreads), 0, st, a); break;
    case 16: hipLaunchKernelGGL((qk_kernel<DT, 16, HALF, BACK>), grid, dim3(kQkThreads), 0, st, a); break;
    case 32: hipLaunchKernelGGL((qk_kernel<DT, 32, HALF, BACK>), grid, dim3(kQkThreads), 0, st, a); break;
    default: hipLaunchKernelGGL((qk_kernel<DT, 64, HALF, BACK>), grid, dim3(kQkThreads), 0, st, a); break;
  }
}

template <int DT, bool BACK>
static void qk_launch_as(const QkArgs &a, const QkPlan &p, bool half, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(std::max(p.blocks[0], p.blocks[1])), p.blocks[1] ? 2 : 1);
  if (!p.vec) {
    hipLaunchKernelGGL((qk_any_kernel<DT, BACK>), grid, dim3(kQkThreads), 0, st, a, half ? 1 : 0);
  } else if (half) {
    qk_launch_group<DT, BACK, true>(a, p.group, grid, st);
  } else {
    qk_launch_group<DT, BACK, false>(a, p.group, grid, st);
  }
}

template <bool BACK>
static int qk_launch(const QkArgs &a, const QkPlan &p, int dtype, bool half, hipStream_t st, const char *what) {
  if (p.blocks[0] + p.blocks[1] == 0) return SMX_OK;
  if (dtype == SMX_F32) {
    qk_launch_as<SMX_F32, BACK>(a, p, half, st);
  } else if (dtype == SMX_BF16) {
    qk_launch_as<SMX_BF16, BACK>(a, p, half, st);
  } else {
    qk_launch_as<SMX_F16, BACK>(a, p, half, st);
  }
  return check_launch(what);
}

}  // namespace smx

using namespace smx;

extern "C" int smx_qk_norm_rotary(const smx_qk_desc *desc, void *stream) {
  const int rc = qk_check("qk_norm_rotary", desc, false);
  if (rc != SMX_OK) return rc;
  if (desc->batch * desc->seq == 0) return SMX_OK;
  const QkPlan p = qk_plan(*desc, false);
  float *const none[2] = {nullptr, nullptr};
  return qk_launch<false>(qk_args(*desc, p, none, false), p, desc->dtype, desc->style == SMX_ROTARY_HALF,
                          static_cast<hipStream_t>(stream), "qk_norm_rotary");
}

extern "C" int64_t smx_qk_workspace_bytes(int64_t dim) {
  // partial rows of dw: at most 4 for each of 2048 blocks and one more
  return dim >= 1 && dim <= 65536 ? 4 * 2050 * dim * static_cast<int64_t>(sizeof(float)) : SMX_EINVAL;
}

extern "C" int smx_qk_norm_rotary_backward(const smx_qk_desc *desc, void *workspace, int64_t workspace_bytes,
                                           void *stream) {
  const int rc = qk_check("qk_norm_rotary_backward", desc, true);
  if (rc != SMX_OK) return rc;
  const bool empty = desc->batch * desc->seq == 0;
  const bool any_dw = desc->q.dw || desc->k.dw;
  if (empty && !any_dw) return SMX_OK;
  QkPlan p{};
  if (!empty) p = qk_plan(*desc, true);
  float *part[2] = {nullptr, nullptr};
  int64_t at = 0;
  if (any_dw) {
    SMX_REQUIRE(workspace && workspace_bytes >= smx_qk_workspace_bytes(desc->dim), SMX_EWORKSPACE,
                "qk_norm_rotary_backward: workspace too small");
    SMX_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, SMX_EALIGN,
                "qk_norm_rotary_backward: workspace must be 16-byte aligned");
    for (int i = 0; i < 2; ++i) {
      const smx_qk_side &s = i ? desc->k : desc->q;
      if (!s.dw || !s.heads) continue;
      part[i] = static_cast<float *>(workspace) + at;
      at += static_cast<int64_t>(p.rows[i]) * desc->dim;
    }
  }
  const auto st = static_cast<hipStream_t>(stream);
  if (at > 0 && !p.vec) {
    hipLaunchKernelGGL(qk_zero_kernel, dim3(static_cast<unsigned>(std::min<int64_t>(1024, ceil_div(at, 256)))), dim3(256), 0, st,
                       static_cast<float *>(workspace), at);
    const int zrc = check_launch("qk_norm_rotary_backward");
    if (zrc != SMX_OK) return zrc;
  }
  const int lrc = qk_launch<true>(qk_args(*desc, p, part, true), p, desc->dtype, desc->style == SMX_ROTARY_HALF, st,
                                  "qk_norm_rotary_backward");
  if (lrc != SMX_OK || !any_dw) return lrc;
  QkDwArgs w{};
  for (int i = 0; i < 2; ++i) {
    const smx_qk_side &s = i ? desc->k : desc->q;
    w.part[i] = part[i], w.dw[i] = s.dw, w.rows[i] = p.rows[i], w.dtype[i] = s.weight_dtype;
  }
  w.dim = static_cast<int32_t>(desc->dim);
  hipLaunchKernelGGL(qk_dw_kernel, dim3(static_cast<unsigned>(ceil_div(desc->dim, 16)), 2), dim3(1024), 0, st, w);
  return check_launch("qk_norm_rotary_backward");
}
