// The weight and bias gradients of a Linear whose input is kept in 8 bits:
//   dW[n, k] = sum_m delta[m, n] * held(x)[m, k],   db[n] = sum_m delta[m, n].
#include "act8.h"

#include <algorithm>

namespace smx {

struct WgradArgs {
  const void *delta;  // [rows, n] of its dtype
  const uint8_t *codes, *scales;
  void *dw;  // [n, k]
  void *db;  // [n] or null
  int64_t rows, n, k, pitch, delta_stride;
};

constexpr int kWgTile = 64, kWgStep = 16;

template <int DT, int FMT, int OUT>
__global__ void __launch_bounds__(256) wgrad_kernel(WgradArgs a) {
  __shared__ float sd[kWgStep][kWgTile], sx[kWgStep][kWgTile];
  const int64_t n0 = static_cast<int64_t>(blockIdx.y) * kWgTile, k0 = static_cast<int64_t>(blockIdx.x) * kWgTile;
  const int tn = threadIdx.x >> 4, tk = threadIdx.x & 15;
  float acc[4][4] = {}, sum[4] = {};
  for (int64_t m0 = 0; m0 < a.rows; m0 += kWgStep) {
    __syncthreads();
    for (int i = threadIdx.x; i < kWgStep * kWgTile; i += 256) {
      const int r = i >> 6, c = i & 63;
      const int64_t m = m0 + r;
      sd[r][c] = m < a.rows && n0 + c < a.n ? load_elem<DT>(a.delta, m * a.delta_stride + n0 + c) : 0.f;
      float x = 0.f;
      if (m < a.rows && k0 + c < a.k) {
        float v[4];
        act8_unpack4<FMT>(a.codes[m * a.pitch + k0 + c], act8_scale(a.scales[m * (a.pitch >> 5) + ((k0 + c) >> 5)]), v);
        x = v[0];
      }
      sx[r][c] = x;
    }
    __syncthreads();
    for (int r = 0; r < kWgStep; ++r) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float d = sd[r][4 * tn + i];
        sum[i] += d;
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(d, sx[r][4 * tk + j], acc[i][j]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t n = n0 + 4 * tn + i;
    if (n >= a.n) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t k = k0 + 4 * tk + j;
      if (k < a.k) store_any(a.dw, OUT, n * a.k + k, round_to(OUT, acc[i][j]));
    }
    if (a.db && blockIdx.x == 0 && tk == 0) store_any(a.db, OUT, n, round_to(OUT, sum[i]));
  }
}

template <int DT, int FMT>
static void wgrad_launch(const WgradArgs &a, int out, dim3 grid, hipStream_t st) {
  if (out == SMX_F32) {
    hipLaunchKernelGGL((wgrad_kernel<DT, FMT, SMX_F32>), grid, dim3(256), 0, st, a);
  } else if (out == SMX_BF16) {
    hipLaunchKernelGGL((wgrad_kernel<DT, FMT, SMX_BF16>), grid, dim3(256), 0, st, a);
  } else {
    hipLaunchKernelGGL((wgrad_kernel<DT, FMT, SMX_F16>), grid, dim3(256), 0, st, a);
  }
}

}  // namespace smx

using namespace smx;

extern "C" int64_t smx_act8_wgrad_workspace_bytes(int64_t rows, int64_t n, int64_t k, int dtype) {
  if (rows < 0 || n < 0 || k < 0 || dtype < SMX_F32 || dtype > SMX_F16) return SMX_EINVAL;
  return 0;
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
  const WgradArgs a{delta, codes, scales, dw, db, rows, n, k, pitch, delta_stride};
  const dim3 grid(static_cast<unsigned>(std::max<int64_t>(1, ceil_div(k, kWgTile))),
                  static_cast<unsigned>(ceil_div(n, kWgTile)));
  const auto st = static_cast<hipStream_t>(stream);
  const bool i8 = fmt == SMX_ACT8_INT8;
  if (dtype == SMX_F32) {
    i8 ? wgrad_launch<SMX_F32, SMX_ACT8_INT8>(a, out_dtype, grid, st)
       : wgrad_launch<SMX_F32, SMX_ACT8_E4M3>(a, out_dtype, grid, st);
  } else if (dtype == SMX_BF16) {
    i8 ? wgrad_launch<SMX_BF16, SMX_ACT8_INT8>(a, out_dtype, grid, st)
       : wgrad_launch<SMX_BF16, SMX_ACT8_E4M3>(a, out_dtype, grid, st);
  } else {
    i8 ? wgrad_launch<SMX_F16, SMX_ACT8_INT8>(a, out_dtype, grid, st)
       : wgrad_launch<SMX_F16, SMX_ACT8_E4M3>(a, out_dtype, grid, st);
  }
  return check_launch("act8_wgrad");
}
