// The weight and bias gradients of a Linear whose input is kept in 8 bits:
//   dW[n, k] = sum_m delta[m, n] * held(x)[m, k],   db[n] = sum_m delta[m, n].
//
// One block owns a tile of dW (256 x 256 by eight waves, or 128 x 128 by four)
// over a range of rows m (a split) and goes over it in steps of kStep rows.  Both
// operands have the sum's index m as their slow axis, so each step is staged row
// by row in LDS as BF16 and read back transposed (ds_read_b64_tr_b16: four rows of
// one column per lane) as the operands of v_mfma_f32_32x32x16_bf16.  The codes
// become BF16 on the way into LDS: a code times its scale is exact in BF16, so its
// product with a BF16 cotangent is exact in FP32.  FP16 and FP32 cotangents are
// staged as the two or three BF16 parts that sum to them (down to 2^-133), with a
// product each.
//
// The two LDS buffers alternate: beside one step's MFMAs the next step is
// written to the other, and loads of a later step are in flight.  Splits of m
// write FP32 partial tiles that a second launch adds in order, so the result
// does not depend on timing.
//
// Measured, BF16 cotangents, with db, calls back to back: 8192 x 2048 -> 8192 246 us
// in e4m3 (1.12 PFLOP/s; 282-317 us among other kernels, at lower clocks) and 257 us
// in int8, whose codes take 2.5 vector instructions an element to widen where e4m3
// takes half of one; 16384 x 768 -> 3072 95 and 96 us; 16384 x 768 -> 768 (small
// tiles, 14 splits) 41 us, 7 of them the join.  The wide tile is bound by MFMA issue
// and the clock held under it (MFMAs busy 41% of the cycles, LDS 31%), the small one
// by staging (28%).
#include "act8.h"

#include <algorithm>

namespace smx {

typedef short v4s __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef float v16f __attribute__((ext_vector_type(16)));

struct WgradArgs {
  const void *delta;  // [rows, n] of its dtype
  const uint8_t *codes, *scales;
  void *dw;            // [n, k], or the splits' partial tiles [splits, n, k] in FP32
  float *db;           // partial column sums [splits, tiles_k, n], or null
  int64_t rows, n, k, pitch, delta_stride;
  int64_t split_rows;  // rows of a split, a multiple of the step
  int32_t tiles_k, tiles, splits, out;
};

constexpr int parts_of(int dt) { return dt == SMX_BF16 ? 1 : dt == SMX_F16 ? 2 : 3; }

// Tiles: rows and columns, the waves that share them, the rows of a step, and
// where in a step the next one is staged (MID: between its halves).
template <int TN, int TK, int WN, int WK, int STEP, int STEP_PARTS, int WPS, bool MID>
struct WgradTile {
  static constexpr bool kMid = MID;
  static constexpr int kTileN = TN, kTileK = TK, kWavesN = WN, kWavesK = WK, kThreads = 64 * WN * WK, kWavesPerSimd = WPS;
  static constexpr int step(int dt) { return dt == SMX_BF16 ? STEP : STEP_PARTS; }
};
using WgradWide = WgradTile<256, 256, 2, 4, 64, 32, 2, true>;
using WgradSmall = WgradTile<128, 128, 2, 2, 64, 32, 2, false>;

// 16 codes and their scale to 16 BF16 values (two uint4).
template <int FMT>
__device__ __forceinline__ void act8_to_bf16(const uint4 &c, int b, uint4 *o) {
  const float scale = act8_scale(b);
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  uint32_t r[8];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if constexpr (FMT == SMX_ACT8_INT8) {
      // code * scale, exact; the upper halves are the BF16 values
      float f[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) f[k] = static_cast<float>(static_cast<int8_t>(w[q] >> (8 * k))) * scale;
      r[2 * q] = __builtin_amdgcn_perm(__float_as_uint(f[1]), __float_as_uint(f[0]), 0x07060302u);
      r[2 * q + 1] = __builtin_amdgcn_perm(__float_as_uint(f[3]), __float_as_uint(f[2]), 0x07060302u);
    } else {
      const v2bf lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[q], scale, false);
      const v2bf hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[q], scale, true);
      __builtin_memcpy(&r[2 * q], &lo, 4);
      __builtin_memcpy(&r[2 * q + 1], &hi, 4);
    }
  }
  o[0] = make_uint4(r[0], r[1], r[2], r[3]);
  o[1] = make_uint4(r[4], r[5], r[6], r[7]);
}

// Eight cotangents as loaded.
template <int DT>
struct Cot8 {
  static constexpr int kWords = DT == SMX_F32 ? 8 : 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const void *p, int64_t i) {
    // (16-byte loads at the elements' own alignment)
    __builtin_memcpy(w, static_cast<const char *>(p) + i * (DT == SMX_F32 ? 4 : 2), sizeof(w));
  }
  __device__ __forceinline__ void load_some(const void *p, int64_t i, int n) {
#pragma unroll
    for (int k = 0; k < kWords; ++k) w[k] = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (k >= n) continue;
      if constexpr (DT == SMX_F32) {
        w[k] = static_cast<const uint32_t *>(p)[i + k];
      } else {
        w[k >> 1] |= static_cast<uint32_t>(static_cast<const uint16_t *>(p)[i + k]) << (16 * (k & 1));
      }
    }
  }
  __device__ __forceinline__ float value(int k) const {
    if constexpr (DT == SMX_F32) return __uint_as_float(w[k]);
    if constexpr (DT == SMX_BF16) return __uint_as_float(k & 1 ? w[k >> 1] & 0xffff0000u : w[k >> 1] << 16);
    return f16_bits_to_f32(static_cast<uint16_t>(w[k >> 1] >> (16 * (k & 1))));
  }
  // Its BF16 parts: each the leading eight bits of what is left (exact down to
  // 2^-133, BF16's smallest number), the rest of an infinity being nothing.
  __device__ __forceinline__ void parts(uint4 *o) const {
    if constexpr (DT == SMX_BF16) {
      o[0] = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      constexpr int P = parts_of(DT);
      uint32_t r[P][4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float a = value(2 * q), b = value(2 * q + 1);
#pragma unroll
        for (int p = 0; p < P; ++p) {
          const uint32_t ua = __float_as_uint(a) & 0xffff0000u, ub = __float_as_uint(b) & 0xffff0000u;
          r[p][q] = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
          a = fabsf(a) == INFINITY ? 0.f : a - __uint_as_float(ua);
          b = fabsf(b) == INFINITY ? 0.f : b - __uint_as_float(ub);
        }
      }
#pragma unroll
      for (int p = 0; p < P; ++p) o[p] = make_uint4(r[p][0], r[p][1], r[p][2], r[p][3]);
    }
  }
};

// LDS image of a step: [planes][kStep rows][T] BF16, where the 32-byte blocks
// of a row are exchanged by its row number (block ^ 2 (row mod 4)): the four
// rows that a transposing read takes from one column then lie in different banks.
template <int T>
__device__ __forceinline__ int lds_at(int row, int block) {
  return row * 2 * T + ((block ^ ((row & 3) << 1)) << 5);
}

// The first n of four neighbours of dw, at their own alignment.
__device__ __forceinline__ void store_row4(void *dw, int out, int64_t i, const float4 &v, int64_t n) {
  const float e[4] = {v.x, v.y, v.z, v.w};
  if (out == SMX_F32) {
    typedef float v4 __attribute__((ext_vector_type(4), aligned(4)));
    float *p = static_cast<float *>(dw) + i;
    if (n >= 4) {
      *reinterpret_cast<v4 *>(p) = v4{v.x, v.y, v.z, v.w};
    } else {
#pragma unroll
      for (int q = 0; q < 3; ++q)
        if (q < n) p[q] = e[q];
    }
  } else {
    uint16_t h[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const _Float16 half = static_cast<_Float16>(e[q]);
      h[q] = out == SMX_BF16 ? f32_to_bf16_bits(e[q]) : __builtin_bit_cast(uint16_t, half);
    }
    typedef uint32_t v2 __attribute__((ext_vector_type(2), aligned(2)));
    uint16_t *p = static_cast<uint16_t *>(dw) + i;
    if (n >= 4) {
      *reinterpret_cast<v2 *>(p) = v2{h[0] | static_cast<uint32_t>(h[1]) << 16, h[2] | static_cast<uint32_t>(h[3]) << 16};
    } else {
#pragma unroll
      for (int q = 0; q < 3; ++q)
        if (q < n) p[q] = h[q];
    }
  }
}

template <int DT, int FMT, class C>
__global__ void __launch_bounds__(C::kThreads, C::kWavesPerSimd) wgrad_kernel(WgradArgs a) {
  constexpr int P = parts_of(DT), kStep = C::step(DT), TN = C::kTileN, TK = C::kTileK;
  constexpr int kPlane = kStep * TN * 2, kBuffer = P * kPlane + kStep * TK * 2;
  constexpr int kDeltaRows = C::kThreads / (TN / 8), kCodeRows = C::kThreads / (TK / 16);  // rows of one pass of loads
  constexpr int kDeltaLoads = kStep / kDeltaRows, kCodeLoads = kStep / kCodeRows;
  static_assert(kDeltaLoads * kDeltaRows == kStep && kCodeLoads * kCodeRows == kStep, "whole passes");
  constexpr int FN = TN / C::kWavesN / 32, FK = TK / C::kWavesK / 32;  // a wave's MFMA tiles
  // dw's tile leaves through LDS too, in passes of a row of waves each where it is wide
  constexpr int kPasses = TN * TK * 4 > 65536 ? C::kWavesN : 1, kPassRows = TN / kPasses;
  __shared__ __attribute__((aligned(128))) char lds[kPassRows * TK * 4 > 2 * kBuffer ? kPassRows * TK * 4 : 2 * kBuffer];

  // Blocks of one split run on one XCD as far as they can, since they share its rows.
  const int64_t blocks = static_cast<int64_t>(a.tiles) * a.splits;
  const int64_t share = (blocks + 7) / 8;
  const int64_t id = (blockIdx.x & 7) * share + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= share || id >= blocks) return;
  const int split = static_cast<int>(id / a.tiles), tile = static_cast<int>(id % a.tiles);
  const int tile_k = tile % a.tiles_k;
  const int64_t n0 = static_cast<int64_t>(tile / a.tiles_k) * TN, k0 = static_cast<int64_t>(tile_k) * TK;
  const int64_t m_begin = split * a.split_rows, m_end = min(a.rows, m_begin + a.split_rows);
  const int steps = static_cast<int>((m_end - m_begin + kStep - 1) / kStep);

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave / C::kWavesK * (32 * FN), wk = wave % C::kWavesK * (32 * FK);

  // Staging: a thread loads 8 cotangents (16 codes) of the same columns in
  // every row of its own.  Columns past the end repeat others in bounds: what
  // they add to is not stored.
  const int d_row = tid / (TN / 8), d_col = tid % (TN / 8);
  const int c_row = tid / (TK / 16), c_col = tid % (TK / 16);
  const int64_t nc = min(n0 + 8 * d_col, (a.n - 1) & ~int64_t{7});
  const int nc_count = static_cast<int>(min<int64_t>(8, a.n - nc));
  const int64_t kc = min(k0 + 16 * c_col, a.pitch - 16);
  const int64_t scale_pitch = a.pitch >> 5;

  Cot8<DT> d[kDeltaLoads];
  uint4 c[kCodeLoads];
  int s[kCodeLoads];
  float sum[8] = {};

  const auto load = [&](int step) __attribute__((always_inline)) {
    const int64_t m0 = m_begin + static_cast<int64_t>(step) * kStep;
    // A load of 8 that begins in a row may end in the next: the tensor's last
    // row, and rows shorter than 8, are read one by one.  (No inputs, k = 0,
    // leave no codes to read.)
    if (m0 + kStep < a.rows && m0 + kStep <= m_end && a.n >= 8 && a.k > 0) {
#pragma unroll
      for (int i = 0; i < kDeltaLoads; ++i)
        d[i].load(a.delta, (m0 + d_row + i * kDeltaRows) * a.delta_stride + nc);
#pragma unroll
      for (int i = 0; i < kCodeLoads; ++i) {
        const int64_t m = m0 + c_row + i * kCodeRows;
        c[i] = *reinterpret_cast<const uint4 *>(a.codes + m * a.pitch + kc);
        s[i] = a.scales[m * scale_pitch + (kc >> 5)];
      }
    } else {
#pragma unroll
      for (int i = 0; i < kDeltaLoads; ++i) {
        const int64_t m = m0 + d_row + i * kDeltaRows;
        d[i].load_some(a.delta, m * a.delta_stride + nc, m < m_end ? nc_count : 0);
      }
#pragma unroll
      for (int i = 0; i < kCodeLoads; ++i) {
        const int64_t m = m0 + c_row + i * kCodeRows;
        c[i] = make_uint4(0, 0, 0, 0);
        s[i] = 1;
        if (m < m_end && a.k > 0) {
          c[i] = *reinterpret_cast<const uint4 *>(a.codes + m * a.pitch + kc);
          s[i] = a.scales[m * scale_pitch + (kc >> 5)];
        }
      }
    }
  };
  const auto stage_delta = [&](char *at, int i) __attribute__((always_inline)) {
    const int row = d_row + i * kDeltaRows;
    uint4 o[P];
    d[i].parts(o);
#pragma unroll
    for (int p = 0; p < P; ++p)
      *reinterpret_cast<uint4 *>(at + p * kPlane + lds_at<TN>(row, d_col >> 1) + (d_col & 1) * 16) = o[p];
  };
  const auto stage_codes = [&](char *at, int i) __attribute__((always_inline)) {
    const int row = c_row + i * kCodeRows;
    uint4 o[2];
    act8_to_bf16<FMT>(c[i], s[i], o);
    uint4 *to = reinterpret_cast<uint4 *>(at + P * kPlane + lds_at<TK>(row, c_col));
    to[0] = o[0], to[1] = o[1];
  };
  // The column sums for db, of the steps whose turn it is: each of the row of
  // tiles that share these cotangents takes its share.
  const auto add_bias = [&](int step) __attribute__((always_inline)) {
    if (!a.db || step % a.tiles_k != tile_k) return;
#pragma unroll
    for (int i = 0; i < kDeltaLoads; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) sum[k] += d[i].value(k);
  };

  // Transposing reads: lane i of a group of 16 names four columns of row
  // i / 4 and receives column i of four rows; groups 0 and 1 hold columns 0-15
  // and 16-31 of rows 0-7 of a 16-row operand, groups 2 and 3 rows 8-15.
  const int g = lane >> 4, i16 = lane & 15, r4 = i16 >> 2;
  const int tr_row = 8 * (g >> 1) + r4;
  int a_at[FN], b_at[FK];
#pragma unroll
  for (int f = 0; f < FN; ++f) a_at[f] = lds_at<TN>(tr_row, (wn >> 4) + 2 * f + (g & 1)) + (i16 & 3) * 8;
#pragma unroll
  for (int f = 0; f < FK; ++f) b_at[f] = P * kPlane + lds_at<TK>(tr_row, (wk >> 4) + 2 * f + (g & 1)) + (i16 & 3) * 8;
  const auto operand = [&](const char *at, int four_rows) __attribute__((always_inline)) {
    typedef __attribute__((address_space(3))) v4s *lds_ptr;
    const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(at));
    const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(at + four_rows));
    typedef short v8s __attribute__((ext_vector_type(8)));
    const v8s v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(v8bf, v);
  };

  v16f acc[FN][FK] = {};
  const auto stage = [&](char *to) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kDeltaLoads; ++i) stage_delta(to, i);
#pragma unroll
    for (int i = 0; i < kCodeLoads; ++i) stage_codes(to, i);
  };
  // The next step's registers are staged between the halves of a step, where
  // one block has the CU to itself (two waves a SIMD): what one wave stages,
  // the other covers with MFMAs.  Where two blocks share it, they do that for
  // each other, and staging behind a step's MFMAs leaves its loads more time.
  // (8192 x 2048 x 8192 e4m3, wide: 252 us, 265 us behind; 16384 x 768 x 768,
  // small: 42 us, 39 us behind.)
  if (steps > 0) {
    load(0);
    add_bias(0);
    stage(lds);
    if (C::kMid && steps > 1) load(1);
  }
  __syncthreads();
  constexpr int kHalf = kStep / 32;
  for (int t = 0; t < steps; ++t) {
    const char *at = lds + (t & 1) * kBuffer;
    char *next = lds + ((t & 1) ^ 1) * kBuffer;
    const auto products = [&](int ms) __attribute__((always_inline)) {
      v8bf bv[FK];
#pragma unroll
      for (int h = 0; h < FK; ++h) bv[h] = operand(at + ms * 16 * 2 * TK + b_at[h], 4 * 2 * TK);
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int f = 0; f < FN; ++f) {
          const v8bf av = operand(at + p * kPlane + ms * 16 * 2 * TN + a_at[f], 4 * 2 * TN);
#pragma unroll
          for (int h = 0; h < FK; ++h) acc[f][h] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(av, bv[h], acc[f][h], 0, 0, 0);
        }
    };
    if (!C::kMid && t + 1 < steps) load(t + 1);
#pragma unroll
    for (int ms = 0; ms < kHalf; ++ms) products(ms);
    if constexpr (C::kMid) {
      // (the last step stages registers that nobody reads)
      if (t + 1 < steps) add_bias(t + 1);
      stage(next);
      if (t + 2 < steps) load(t + 2);
    }
#pragma unroll
    for (int ms = kHalf; ms < kStep / 16; ++ms) products(ms);
    if (!C::kMid && t + 1 < steps) {
      add_bias(t + 1);
      stage(next);
    }
    __syncthreads();
  }

  // The tile goes out through LDS, row by row: lane l of a wave holds column l
  // mod 32 and rows 8 (r / 4) + 4 (l / 32) + r mod 4 of an MFMA tile.  (Stores
  // from there, one element a lane, took five times the code, which the first
  // blocks of a short launch wait for.)
  float *tile_out = reinterpret_cast<float *>(lds);
  const int64_t part = a.splits > 1 ? static_cast<int64_t>(split) * a.n * a.k : 0;
#pragma unroll 1
  for (int pass = 0; pass < kPasses; ++pass) {
    if (kPasses == 1 || wn == pass * kPassRows) {
      float *at = tile_out + (wn - pass * kPassRows + 4 * (lane >> 5)) * TK + wk + (lane & 31);
#pragma unroll
      for (int f = 0; f < FN; ++f)
#pragma unroll
        for (int h = 0; h < FK; ++h)
#pragma unroll
          for (int r = 0; r < 16; ++r) at[(32 * f + 8 * (r >> 2) + (r & 3)) * TK + 32 * h] = acc[f][h][r];
    }
    __syncthreads();
    constexpr int kPerRow = TK / 4, kAtOnce = C::kThreads / kPerRow;
    const int col = 4 * (tid % kPerRow);
    const int64_t k = k0 + col;
    const int64_t rows_here = min<int64_t>(kPassRows, a.n - n0 - pass * kPassRows);
#pragma unroll 4
    for (int row = tid / kPerRow; row < rows_here; row += kAtOnce) {
      const float4 v = *reinterpret_cast<const float4 *>(tile_out + row * TK + col);
      const int64_t o = part + (n0 + pass * kPassRows + row) * a.k + k;
      store_row4(a.dw, a.out, o, v, a.k - k);
    }
    if (kPasses > 1) __syncthreads();
  }
  if (kPasses == 1) __syncthreads();
  if (a.db) {
    float *red = reinterpret_cast<float *>(lds);  // [rows of threads][TN]
#pragma unroll
    for (int k = 0; k < 8; ++k) red[d_row * TN + 8 * d_col + k] = sum[k];
    __syncthreads();
    if (tid < TN && n0 + tid < a.n) {
      float t = 0.f;
      for (int q = 0; q < kDeltaRows; ++q) t += red[q * TN + tid];
      a.db[(static_cast<int64_t>(split) * a.tiles_k + tile_k) * a.n + n0 + tid] = t;
    }
  }
}

// The splits' partial sums added in order: dw (count = 0: it is whole), then db
// of `db_parts` parts: a block per 1024 elements of dw, then one per 16 of db.
__global__ void __launch_bounds__(256) wgrad_join_kernel(const float *part, int64_t count, int splits, void *out,
                                                         int out_dtype, const float *part_db, int64_t n, int db_parts,
                                                         void *db) {
  const int64_t dw_blocks = (count + 1023) / 1024;
  if (static_cast<int64_t>(blockIdx.x) >= dw_blocks) {
    // 16 columns of db, each from 16 threads
    __shared__ float red[16][17];
    const int col = threadIdx.x & 15, q = threadIdx.x >> 4;
    const int64_t j = (blockIdx.x - dw_blocks) * 16 + col;
    float t = 0.f;
    if (j < n) {
#pragma unroll 4
      for (int s = q; s < db_parts; s += 16) t += part_db[s * n + j];
    }
    red[q][col] = t;
    __syncthreads();
    if (q > 0 || j >= n) return;
    for (int s = 1; s < 16; ++s) t += red[s][col];
    store_any(db, out_dtype, j, round_to(out_dtype, t));
    return;
  }
  const int64_t i0 = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (i0 + 4 <= count && count % 4 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0) {
    float4 t = make_float4(0, 0, 0, 0);
    int s = 0;
    for (; s + 8 <= splits; s += 8) {  // (eight loads in flight, added in order)
      float4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = *reinterpret_cast<const float4 *>(part + (s + u) * count + i0);
#pragma unroll
      for (int u = 0; u < 8; ++u) t.x += v[u].x, t.y += v[u].y, t.z += v[u].z, t.w += v[u].w;
    }
#pragma unroll 4
    for (; s < splits; ++s) {
      const float4 v = *reinterpret_cast<const float4 *>(part + s * count + i0);
      t.x += v.x, t.y += v.y, t.z += v.z, t.w += v.w;
    }
    if (out_dtype == SMX_F32) {
      *reinterpret_cast<float4 *>(static_cast<float *>(out) + i0) = t;
    } else {
      store_any(out, out_dtype, i0, round_to(out_dtype, t.x));
      store_any(out, out_dtype, i0 + 1, round_to(out_dtype, t.y));
      store_any(out, out_dtype, i0 + 2, round_to(out_dtype, t.z));
      store_any(out, out_dtype, i0 + 3, round_to(out_dtype, t.w));
    }
  } else {
    for (int64_t i = i0; i < min(i0 + 4, count); ++i) {
      float t = 0.f;
      for (int s = 0; s < splits; ++s) t += part[s * count + i];
      store_any(out, out_dtype, i, round_to(out_dtype, t));
    }
  }
}

struct WgradPlan {
  bool wide;
  int tiles_n, tiles_k, splits;
  int64_t split_rows;
};

// The tile and the splits of the rows with the least expected time:
//   steps of 64 rows times what a step takes a CU (BF16 cotangents, measured:
//   2.0 us a wide tile, 1.2 us a small one alone on its CU, 1.6 us two small
//   ones together; each further part of the cotangents adds 0.8 of that), 7 or
//   2.5 us for a wide or small tile's first loads and last stores, and where
//   the rows are split the join's launch (4 us) and the partial tiles at 8 TB/s
//   written and read.
// (Measured on either tile: 2048 x 2048 x 2048 e4m3 45 us wide, 35 us small;
// 16384 x 768 x 3072 93 us wide, 110 us small; 64 x 2048 x 2048 16 and 10 us.)
static WgradPlan wgrad_plan(int dtype, int64_t rows, int64_t n, int64_t k) {
  constexpr int64_t kCus = 256;
  WgradPlan best{};
  double best_us = 0;
  for (const bool wide : {true, false}) {
    const int64_t tn = wide ? WgradWide::kTileN : WgradSmall::kTileN, tk = wide ? WgradWide::kTileK : WgradSmall::kTileK;
    const int64_t tiles_n = ceil_div(n, tn), tiles_k = std::max<int64_t>(1, ceil_div(k, tk)), tiles = tiles_n * tiles_k;
    const int64_t step = wide ? WgradWide::step(dtype) : WgradSmall::step(dtype);
    const int64_t most = std::min<int64_t>(64, std::max<int64_t>(1, 2 * kCus / tiles));
    for (int64_t s = 1; s <= most; ++s) {
      const int64_t split_rows = round_up(ceil_div(std::max<int64_t>(rows, 1), s), step);
      if (s > 1 && ceil_div(rows, split_rows) != s) continue;  // (as many splits with fewer rows each came before)
      const int64_t per_cu = ceil_div(tiles * s, kCus);
      const double steps = static_cast<double>(split_rows) / 64 * (0.2 + 0.8 * parts_of(dtype));
      const double small = per_cu == 1 ? 1.2 : 1.6 * static_cast<double>(ceil_div(per_cu, 2));
      double us = steps * (wide ? 2.0 * static_cast<double>(per_cu) : small) + (wide ? 7 : 2.5);
      if (s > 1) us += 4 + static_cast<double>(s * n * k) * 8 / 8e6;
      if (best_us == 0 || us < best_us) {
        best_us = us;
        best = {wide, static_cast<int>(tiles_n), static_cast<int>(tiles_k), static_cast<int>(s), split_rows};
      }
    }
  }
  return best;
}

template <int DT, int FMT>
static void wgrad_launch(const WgradArgs &a, bool wide, dim3 grid, hipStream_t st) {
  if (wide) {
    hipLaunchKernelGGL((wgrad_kernel<DT, FMT, WgradWide>), grid, dim3(WgradWide::kThreads), 0, st, a);
  } else {
    hipLaunchKernelGGL((wgrad_kernel<DT, FMT, WgradSmall>), grid, dim3(WgradSmall::kThreads), 0, st, a);
  }
}

}  // namespace smx

using namespace smx;

extern "C" int64_t smx_act8_wgrad_workspace_bytes(int64_t rows, int64_t n, int64_t k, int dtype) {
  if (rows < 0 || n < 0 || k < 0 || dtype < SMX_F32 || dtype > SMX_F16) return SMX_EINVAL;
  if (n > (int64_t{1} << 20) || k > (int64_t{1} << 20)) return SMX_ESHAPE;
  if (n == 0) return 0;  // (no tile, nothing to plan)
  const WgradPlan p = wgrad_plan(dtype, rows, n, k);
  // the splits' partial tiles where there are several, and the parts of db
  const int64_t tiles = p.splits > 1 ? p.splits * n * k : 0, db = static_cast<int64_t>(p.splits) * p.tiles_k * n;
  return round_up((tiles + db) * static_cast<int64_t>(sizeof(float)), 256);
}

extern "C" int smx_act8_wgrad(const void *delta, int dtype, int64_t rows, int64_t n, int64_t delta_stride,
                              const uint8_t *codes, const uint8_t *scales, int fmt, int64_t k, int64_t pitch, void *dw,
                              void *db, int out_dtype, void *workspace, int64_t workspace_bytes, void *stream) {
  const auto known = [](int d) { return d == SMX_F32 || d == SMX_BF16 || d == SMX_F16; };
  SMX_REQUIRE(known(dtype) && known(out_dtype), SMX_EDTYPE, "act8_wgrad: dtypes must be f32, bf16 or f16");
  SMX_REQUIRE(fmt == SMX_ACT8_INT8 || fmt == SMX_ACT8_E4M3, SMX_EINVAL, "act8_wgrad: unknown 8-bit format");
  SMX_REQUIRE(rows >= 0 && n >= 0 && k >= 0, SMX_ESHAPE, "act8_wgrad: negative size");
  SMX_REQUIRE(n <= (int64_t{1} << 20) && k <= (int64_t{1} << 20), SMX_ESHAPE, "act8_wgrad: more than 2^20 features");
  SMX_REQUIRE(pitch >= k && pitch % kAct8Block == 0 && pitch - k < kAct8Block, SMX_ESHAPE,
              "act8_wgrad: pitch must be k rounded up to a multiple of 32");
  if (n == 0 || (k == 0 && !db)) return SMX_OK;
  SMX_REQUIRE(dw || k == 0, SMX_EINVAL, "act8_wgrad: null dw");
  if (rows > 0) {
    SMX_REQUIRE(delta && ((codes && scales) || k == 0), SMX_EINVAL, "act8_wgrad: null pointer");
    SMX_REQUIRE(delta_stride >= n || rows == 1, SMX_ESHAPE, "act8_wgrad: delta's row stride smaller than n");
    SMX_REQUIRE(reinterpret_cast<uintptr_t>(codes) % 16 == 0, SMX_EALIGN, "act8_wgrad: codes must be 16-byte aligned");
  }
  const int64_t need = smx_act8_wgrad_workspace_bytes(rows, n, k, dtype);
  SMX_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), SMX_EWORKSPACE, "act8_wgrad: workspace too small");
  SMX_REQUIRE(need == 0 || reinterpret_cast<uintptr_t>(workspace) % 256 == 0, SMX_EALIGN,
              "act8_wgrad: workspace must be 256-byte aligned");
  const WgradPlan p = wgrad_plan(dtype, rows, n, k);
  WgradArgs a{};
  a.delta = delta, a.codes = codes, a.scales = scales, a.dw = dw;
  a.rows = rows, a.n = n, a.k = k, a.pitch = pitch, a.delta_stride = delta_stride;
  a.split_rows = p.split_rows, a.tiles_k = p.tiles_k, a.tiles = p.tiles_n * p.tiles_k, a.splits = p.splits, a.out = out_dtype;
  const int64_t tiles = p.splits > 1 ? p.splits * n * k : 0;
  if (p.splits > 1) a.dw = workspace, a.out = SMX_F32;
  if (db) a.db = static_cast<float *>(workspace) + tiles;
  const dim3 grid(static_cast<unsigned>(round_up(static_cast<int64_t>(a.tiles) * a.splits, 8)));
  const auto st = static_cast<hipStream_t>(stream);
  const bool i8 = fmt == SMX_ACT8_INT8;
  if (dtype == SMX_F32) {
    i8 ? wgrad_launch<SMX_F32, SMX_ACT8_INT8>(a, p.wide, grid, st) : wgrad_launch<SMX_F32, SMX_ACT8_E4M3>(a, p.wide, grid, st);
  } else if (dtype == SMX_BF16) {
    i8 ? wgrad_launch<SMX_BF16, SMX_ACT8_INT8>(a, p.wide, grid, st)
       : wgrad_launch<SMX_BF16, SMX_ACT8_E4M3>(a, p.wide, grid, st);
  } else {
    i8 ? wgrad_launch<SMX_F16, SMX_ACT8_INT8>(a, p.wide, grid, st) : wgrad_launch<SMX_F16, SMX_ACT8_E4M3>(a, p.wide, grid, st);
  }
  if (p.splits > 1 || db) {
    const int rc = check_launch("act8_wgrad");
    if (rc != SMX_OK) return rc;
    const int64_t count = p.splits > 1 ? n * k : 0, blocks = ceil_div(count, 1024) + (db ? ceil_div(n, 16) : 0);
    if (blocks == 0) return SMX_OK;
    hipLaunchKernelGGL(wgrad_join_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st,
                       static_cast<const float *>(workspace), count, p.splits, dw, out_dtype, a.db, n,
                       p.splits * p.tiles_k, db);
  }
  return check_launch("act8_wgrad");
}
