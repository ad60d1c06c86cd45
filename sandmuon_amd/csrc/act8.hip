// Activations kept in 8 bits for the backward pass (format: act8.h): encode,
// decode, and the GELU of an MLP's hidden layer with its input and output
// kept in the same pass.  All are one pass over the data, bound by HBM.
//
// A thread owns 8 neighbours of a row, so that a 16-bit row is read in 16-byte
// loads, and four neighbouring lanes own a block of 32: the block's largest
// magnitude is two DPP moves away.  blockDim = (chunks of 8, rows), so no
// thread divides.  One row a thread: waves, not loads of a thread, hide the
// latency (four rows a thread took 68 us for the GELU of 16384 x 3072 bf16
// instead of 54, at half the waves).
//
// Measured at 16384 x 3072 bf16, int8: GELU with both sides kept 54 us (6 bytes
// an element: 5.6 TB/s), its gradient 58 us (5 bytes: 4.4 TB/s, bound by its 27
// vector instructions an element as much as by HBM), read back 24 us; 16384 x
// 768 bf16 kept 8 us (4.7 TB/s).
#include "act8.h"

#include <algorithm>

namespace smx {

// Two values rounded to nearest even in a 16-bit type.
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  uint32_t w;
  if constexpr (DT == SMX_BF16) {
    typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
    const v2bf h = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
    __builtin_memcpy(&w, &h, 4);
  } else {
    const _Float16 h[2] = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
    __builtin_memcpy(&w, h, 4);
  }
  return w;
}

template <int DT>
__device__ __forceinline__ void unpack2(uint32_t w, float *v) {
  if constexpr (DT == SMX_BF16) {
    v[0] = __uint_as_float(w << 16);
    v[1] = __uint_as_float(w & 0xffff0000u);
  } else {
    v[0] = f16_bits_to_f32(static_cast<uint16_t>(w));
    v[1] = f16_bits_to_f32(static_cast<uint16_t>(w >> 16));
  }
}

// Eight values as their type holds them.
template <int DT>
__device__ __forceinline__ void round8(float *v) {
  if constexpr (DT != SMX_F32) {
#pragma unroll
    for (int k = 0; k < 4; ++k) unpack2<DT>(pack2<DT>(v[2 * k], v[2 * k + 1]), v + 2 * k);
  }
}

// 16 bytes at the elements' own alignment: rows of an odd width are read and
// written like others.
typedef uint32_t act8_v4u __attribute__((ext_vector_type(4), aligned(2)));

template <int DT>
struct Elems8 {
  // Elements [i, i + n) of p, n <= 8; the rest are zero.
  static __device__ __forceinline__ void load(const void *p, int64_t i, int n, float *v) {
    if (n < 8) {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = k < n ? load_elem<DT>(p, i + k) : 0.f;
      return;
    }
    if constexpr (DT == SMX_F32) {
      const auto *at = reinterpret_cast<const act8_v4u *>(static_cast<const float *>(p) + i);
      const act8_v4u a = at[0], b = at[1];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = __uint_as_float(a[k]), v[4 + k] = __uint_as_float(b[k]);
    } else {
      const act8_v4u a = *reinterpret_cast<const act8_v4u *>(static_cast<const uint16_t *>(p) + i);
#pragma unroll
      for (int k = 0; k < 4; ++k) unpack2<DT>(a[k], v + 2 * k);
    }
  }
  static __device__ __forceinline__ void store(void *p, int64_t i, int n, const float *v) {
    if (n < 8) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < n) store_any(p, DT, i + k, round_to(DT, v[k]));
      return;
    }
    if constexpr (DT == SMX_F32) {
      auto *at = reinterpret_cast<act8_v4u *>(static_cast<float *>(p) + i);
#pragma unroll
      for (int q = 0; q < 2; ++q)
        at[q] = act8_v4u{__float_as_uint(v[4 * q]), __float_as_uint(v[4 * q + 1]), __float_as_uint(v[4 * q + 2]),
                         __float_as_uint(v[4 * q + 3])};
    } else {
      *reinterpret_cast<act8_v4u *>(static_cast<uint16_t *>(p) + i) =
          act8_v4u{pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]), pack2<DT>(v[4], v[5]), pack2<DT>(v[6], v[7])};
    }
  }
};

struct Act8Out {
  uint8_t *codes;   // [rows, pitch]
  uint8_t *scales;  // [rows, pitch / 32]
};

// Encodes 8 elements of every lane; `row`, `chunk` name them.
template <int FMT>
__device__ __forceinline__ void act8_put(const float *v, const Act8Out &o, int64_t row, int64_t pitch, int chunk) {
  // Magnitudes compare as whole numbers, a NaN above all (fmaxf would drop it).
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(v[k]) & 0x7fffffffu);
  top = max(top, dpp_mov<0xB1>(top));
  top = max(top, dpp_mov<0x4E>(top));
  const int b = act8_scale_byte<FMT>(static_cast<int>(top >> 23));
  uint2 w = make_uint2(0, 0);
  if (b != 255) {
    const float inv = act8_scale(254 - b);
    if (FMT == SMX_ACT8_E4M3 && (top >> 23) == 254) {
      // (the code 128 of this scale would stand for 2^128)
      float u[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) u[k] = __builtin_amdgcn_fmed3f(v[k] * inv, -120.f, 120.f);
      w = make_uint2(act8_pack4<FMT>(u, 1.f), act8_pack4<FMT>(u + 4, 1.f));
    } else {
      w = make_uint2(act8_pack4<FMT>(v, inv), act8_pack4<FMT>(v + 4, inv));
    }
  }
  *reinterpret_cast<uint2 *>(o.codes + row * pitch + 8 * chunk) = w;
  if ((chunk & 3) == 0) o.scales[row * (pitch >> 5) + (chunk >> 2)] = static_cast<uint8_t>(b);
}

struct Act8Args {
  const void *x;
  void *y;
  const void *dy;
  Act8Out x8, y8;
  int64_t rows, cols, pitch, x_stride, y_stride, dy_stride;
};

// FP32 in torch's order of operations: x * 0.5 * (1 + erf(x / sqrt 2)).
__device__ __forceinline__ float phi_f32(float x) { return 0.5f * (1.f + erff(x * 0.70710678118654752f)); }

// For 16-bit types, whose half place is 2^-12 at the least: the normal tail
// Q(x) = (1 - erf(x / sqrt 2)) / 2 of x >= 0 as exp(-x^2 / 2) times a polynomial
// of degree 8 in t = 1 / (1 + 0.3175 x), a least-squares fit of this file's own,
// reweighted towards the largest error, of exp(x^2 / 2) Q(x) on [0, 40] (Q
// underflows beyond 14): 3.5e-7 off, and 3e-7 as evaluated.  (Degree 6, 1.1e-5
// off, is not enough for the slope near its zero.)  About half of erff's vector
// instructions, which would bound the kernel, not HBM.
struct NormalTail {
  float e, q;  // exp(-x^2 / 2), Q(x)
};
__device__ __forceinline__ NormalTail normal_tail(float x) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.3175f, x, 1.f));
  float g = fmaf(t, 0.03485208749771118f, -0.1270199567079544f);
  g = fmaf(t, g, 0.11735344678163528f);
  g = fmaf(t, g, 0.009273595176637173f);
  g = fmaf(t, g, 0.09985337406396866f);
  g = fmaf(t, g, 0.11224232614040375f);
  g = fmaf(t, g, 0.12678450345993042f);
  g = fmaf(t, g, 0.1266608089208603f);
  const float e = __builtin_amdgcn_exp2f(x * x * -0.72134752044448170f);
  return {e, e * (t * g)};
}

// GELU(h) = max(h, 0) - |h| Q(|h|), keeping infinities and NaN as the formula
// h Phi(h) does (-inf gives NaN).
template <int DT>
__device__ __forceinline__ float gelu_of(float h) {
  if constexpr (DT == SMX_F32) return h * phi_f32(h);
  const float x = fminf(fabsf(h), 40.f);
  return fmaf(-x, normal_tail(x).q, fmaf(0.5f, fabsf(h), 0.5f * h));
}

// GELU'(h) = Phi(h) + h phi(h).
template <int DT>
__device__ __forceinline__ float gelu_slope(float h) {
  constexpr float kPhi0 = 0.3989422804014327f;
  if constexpr (DT == SMX_F32) return phi_f32(h) + h * (expf(-0.5f * h * h) * kPhi0);
  const NormalTail n = normal_tail(fminf(fabsf(h), 40.f));
  return fmaf(h, n.e * kPhi0, 0.5f + copysignf(0.5f - n.q, h));
}

// (the GELU that keeps no input is a kernel of its own: a branch on the pointer cost
// the other one 2%)
enum Act8Op : int { kActEncode = 0, kActGelu = 1, kActDecode = 2, kActGeluBack = 3, kActGeluOut = 4 };

template <int DT, int FMT, int OP>
__global__ void __launch_bounds__(256) act8_kernel(Act8Args a) {
  using E = Elems8<DT>;
  const int chunk = blockIdx.x * blockDim.x + threadIdx.x;
  if (8 * static_cast<int64_t>(chunk) >= a.pitch) return;
  const int n = static_cast<int>(min<int64_t>(8, max<int64_t>(0, a.cols - 8 * static_cast<int64_t>(chunk))));
  const int64_t step = static_cast<int64_t>(gridDim.y) * blockDim.y;
  for (int64_t r = static_cast<int64_t>(blockIdx.y) * blockDim.y + threadIdx.y; r < a.rows; r += step) {
    float v[8] = {};
    if constexpr (OP == kActEncode || OP == kActGelu || OP == kActGeluOut) {
      if (n > 0) E::load(a.x, r * a.x_stride + 8 * chunk, n, v);
      if constexpr (OP != kActGeluOut) act8_put<FMT>(v, a.x8, r, a.pitch, chunk);
      if constexpr (OP != kActEncode) {
        // (the output is kept as it is stored: rounded to its type first)
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = gelu_of<DT>(v[k]);
        round8<DT>(v);
        if (n > 0) E::store(a.y, r * a.y_stride + 8 * chunk, n, v);
        if (a.y8.codes) act8_put<FMT>(v, a.y8, r, a.pitch, chunk);
      }
    } else if (n > 0) {
      const uint2 codes = *reinterpret_cast<const uint2 *>(a.x8.codes + r * a.pitch + 8 * chunk);
      const float scale = act8_scale(a.x8.scales[r * (a.pitch >> 5) + (chunk >> 2)]);
      if constexpr (OP == kActGeluBack) E::load(a.dy, r * a.dy_stride + 8 * chunk, n, v);
      float h[8];
      act8_unpack4<FMT>(codes.x, scale, h);
      act8_unpack4<FMT>(codes.y, scale, h + 4);
      if constexpr (OP == kActGeluBack) {
#pragma unroll
        for (int k = 0; k < 8; ++k) h[k] = v[k] * gelu_slope<DT>(h[k]);
      }
      E::store(a.y, r * a.y_stride + 8 * chunk, n, h);
    }
  }
}

template <int DT, int FMT, int OP>
static int act8_launch_as(const Act8Args &a, hipStream_t st, const char *what) {
  const int64_t chunks = a.pitch / 8;
  const int64_t gx = ceil_div(chunks, 256);
  const int tx = static_cast<int>(round_up(ceil_div(chunks, gx), 4));
  const int ty = std::max(1, 256 / tx);
  const int64_t gy = std::min<int64_t>(ceil_div(a.rows, ty), 32768);
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(gy)), block(tx, ty);
  hipLaunchKernelGGL((act8_kernel<DT, FMT, OP>), grid, block, 0, st, a);
  return check_launch(what);
}

template <int OP>
static int act8_launch(const Act8Args &a, int dtype, int fmt, hipStream_t st, const char *what) {
  const bool i8 = fmt == SMX_ACT8_INT8;
  if (dtype == SMX_F32)
    return i8 ? act8_launch_as<SMX_F32, SMX_ACT8_INT8, OP>(a, st, what)
              : act8_launch_as<SMX_F32, SMX_ACT8_E4M3, OP>(a, st, what);
  if (dtype == SMX_BF16)
    return i8 ? act8_launch_as<SMX_BF16, SMX_ACT8_INT8, OP>(a, st, what)
              : act8_launch_as<SMX_BF16, SMX_ACT8_E4M3, OP>(a, st, what);
  return i8 ? act8_launch_as<SMX_F16, SMX_ACT8_INT8, OP>(a, st, what)
            : act8_launch_as<SMX_F16, SMX_ACT8_E4M3, OP>(a, st, what);
}

static std::string act8_name(const char *what, const char *msg) { return std::string(what) + ": " + msg; }

static int act8_check(const char *what, int dtype, int fmt, int64_t rows, int64_t cols, int64_t pitch) {
  SMX_REQUIRE(dtype == SMX_F32 || dtype == SMX_BF16 || dtype == SMX_F16, SMX_EDTYPE,
              act8_name(what, "dtype must be f32, bf16 or f16"));
  SMX_REQUIRE(fmt == SMX_ACT8_INT8 || fmt == SMX_ACT8_E4M3, SMX_EINVAL, act8_name(what, "unknown 8-bit format"));
  SMX_REQUIRE(rows >= 0 && cols >= 0, SMX_ESHAPE, act8_name(what, "negative rows or cols"));
  SMX_REQUIRE(cols <= (int64_t{1} << 30), SMX_ESHAPE, act8_name(what, "more than 2^30 columns"));
  SMX_REQUIRE(pitch >= cols && pitch % kAct8Block == 0 && pitch - cols < kAct8Block, SMX_ESHAPE,
              act8_name(what, "pitch must be cols rounded up to a multiple of 32"));
  return SMX_OK;
}

static int act8_check_tensor(const char *what, const void *p, int64_t rows, int64_t cols, int64_t stride) {
  SMX_REQUIRE(p, SMX_EINVAL, act8_name(what, "null pointer"));
  SMX_REQUIRE(stride >= cols || rows <= 1, SMX_ESHAPE, act8_name(what, "row stride smaller than cols"));
  return SMX_OK;
}

static int act8_check_codes(const char *what, const void *codes, const void *scales) {
  SMX_REQUIRE(codes && scales, SMX_EINVAL, act8_name(what, "null codes or scales"));
  SMX_REQUIRE(reinterpret_cast<uintptr_t>(codes) % 16 == 0, SMX_EALIGN, act8_name(what, "codes must be 16-byte aligned"));
  return SMX_OK;
}

}  // namespace smx

using namespace smx;

#define ACT8_TRY(call)           \
  do {                           \
    const int rc_ = (call);      \
    if (rc_ != SMX_OK) return rc_; \
  } while (0)

extern "C" int smx_act8_encode(const void *x, int dtype, int64_t rows, int64_t cols, int64_t row_stride, int fmt,
                               uint8_t *codes, uint8_t *scales, int64_t pitch, void *stream) {
  const char *what = "act8_encode";
  ACT8_TRY(act8_check(what, dtype, fmt, rows, cols, pitch));
  if (rows == 0 || cols == 0) return SMX_OK;
  ACT8_TRY(act8_check_tensor(what, x, rows, cols, row_stride));
  ACT8_TRY(act8_check_codes(what, codes, scales));
  Act8Args a{};
  a.x = x, a.x8 = {codes, scales}, a.rows = rows, a.cols = cols, a.pitch = pitch, a.x_stride = row_stride;
  return act8_launch<kActEncode>(a, dtype, fmt, static_cast<hipStream_t>(stream), what);
}

extern "C" int smx_act8_decode(const uint8_t *codes, const uint8_t *scales, int fmt, int64_t rows, int64_t cols,
                               int64_t pitch, void *out, int dtype, int64_t out_stride, void *stream) {
  const char *what = "act8_decode";
  ACT8_TRY(act8_check(what, dtype, fmt, rows, cols, pitch));
  if (rows == 0 || cols == 0) return SMX_OK;
  ACT8_TRY(act8_check_tensor(what, out, rows, cols, out_stride));
  ACT8_TRY(act8_check_codes(what, codes, scales));
  Act8Args a{};
  a.y = out, a.rows = rows, a.cols = cols, a.pitch = pitch, a.y_stride = out_stride;
  a.x8 = {const_cast<uint8_t *>(codes), const_cast<uint8_t *>(scales)};
  return act8_launch<kActDecode>(a, dtype, fmt, static_cast<hipStream_t>(stream), what);
}

extern "C" int smx_act8_gelu(const void *h, int dtype, int64_t rows, int64_t cols, int64_t row_stride, int fmt, void *y,
                             int64_t y_stride, uint8_t *h_codes, uint8_t *h_scales, uint8_t *y_codes,
                             uint8_t *y_scales, int64_t pitch, void *stream) {
  const char *what = "act8_gelu";
  ACT8_TRY(act8_check(what, dtype, fmt, rows, cols, pitch));
  if (rows == 0 || cols == 0) return SMX_OK;
  ACT8_TRY(act8_check_tensor(what, h, rows, cols, row_stride));
  ACT8_TRY(act8_check_tensor(what, y, rows, cols, y_stride));
  SMX_REQUIRE((h_codes == nullptr) == (h_scales == nullptr) && (y_codes == nullptr) == (y_scales == nullptr), SMX_EINVAL,
              "act8_gelu: codes and scales must both be given or both be null");
  if (h_codes) ACT8_TRY(act8_check_codes(what, h_codes, h_scales));
  if (y_codes) ACT8_TRY(act8_check_codes(what, y_codes, y_scales));
  Act8Args a{};
  a.x = h, a.y = y, a.x8 = {h_codes, h_scales}, a.y8 = {y_codes, y_scales};
  a.rows = rows, a.cols = cols, a.pitch = pitch, a.x_stride = row_stride, a.y_stride = y_stride;
  const auto st = static_cast<hipStream_t>(stream);
  return h_codes ? act8_launch<kActGelu>(a, dtype, fmt, st, what) : act8_launch<kActGeluOut>(a, dtype, fmt, st, what);
}

extern "C" int smx_act8_gelu_backward(const void *dy, int dtype, int64_t rows, int64_t cols, int64_t dy_stride,
                                      const uint8_t *h_codes, const uint8_t *h_scales, int fmt, int64_t pitch,
                                      void *dh, int64_t dh_stride, void *stream) {
  const char *what = "act8_gelu_backward";
  ACT8_TRY(act8_check(what, dtype, fmt, rows, cols, pitch));
  if (rows == 0 || cols == 0) return SMX_OK;
  ACT8_TRY(act8_check_tensor(what, dy, rows, cols, dy_stride));
  ACT8_TRY(act8_check_tensor(what, dh, rows, cols, dh_stride));
  ACT8_TRY(act8_check_codes(what, h_codes, h_scales));
  Act8Args a{};
  a.dy = dy, a.y = dh, a.x8 = {const_cast<uint8_t *>(h_codes), const_cast<uint8_t *>(h_scales)};
  a.rows = rows, a.cols = cols, a.pitch = pitch, a.dy_stride = dy_stride, a.y_stride = dh_stride;
  return act8_launch<kActGeluBack>(a, dtype, fmt, static_cast<hipStream_t>(stream), what);
}
