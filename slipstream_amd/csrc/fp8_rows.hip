// Rows quantized to 8-bit floating point (e4m3: 4 bits of exponent, 3 of mantissa, largest value 448)
// with an fp32 scale for every 128 columns, for gfx950: the inputs of the block-scaled product
// (fp8_gemm.hip).
//
// Mathematics, for a block x of a row (the last one may be shorter):
//   a = max |x|;  scale = a / 448;  q = e4m3(x * 448 / a), to the nearest, half to even;  x ~ q * scale.
//   q is that of the exact quotient. x and a have few bits, so quotients that lie halfway between
//   two e4m3 values are common (one in 700 of bf16 data), and the rounding of 448 / a alone would
//   move them to either side. With c = 448 * 2^-e(a) and m = a's mantissa in [1, 2): s = x c, y0 =
//   s / m by a rounded reciprocal, and one step y = y0 + (s - y0 m) / m in fused operations, whose
//   remainder is exact. For 16-bit x, s is exact and so every halfway quotient; others differ from
//   the halfway points by 2^-17 and more. For fp32 x, quotients within 1e-5 of a halfway point are
//   compared with it in 64 bits, where both sides' products are exact.
//   A block whose scale would be subnormal (a < 448 * 2^-126) is zeros with scale zero. A block that
//   holds a NaN or an infinity is zeros with scale NaN, so that every product with it is NaN.
//   The maximum is taken over the magnitudes' bit patterns as unsigned integers.
//
// Bound by the memory at a step's sizes (2240 x 14336 in bf16 19 to 24 us, 4.1 to 5.1 TB/s), by the launch at a
// decode's (197 x 4096 3.3 us).
#include "ss_common.h"

namespace {

using ss::u32x2;
using ss::u32x4;

struct Fp8RowArgs {
  const char* x;
  uint8_t* q;          // [rows, cols], contiguous
  float* scale;        // (row, block) at block * scale_stride + row
  int64_t x_stride;    // bytes
  int64_t scale_stride;
  int64_t rows;
  int cols, blocks, pairs;  // blocks of 128 columns, and pairs of them
};

constexpr uint32_t kInf = 0x7F800000u;
constexpr float kSmallest = 448.f * 1.17549435e-38f;  // 448 * 2^-126

// Largest of the sixteen lanes of a row, in all of them
template <int CTRL>
__device__ __forceinline__ uint32_t max_dpp(uint32_t x) {
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ uint32_t row_max(uint32_t x) {
  x = max_dpp<0x128>(x);    // row_ror:8
  x = max_dpp<0x124>(x);    // row_ror:4
  x = max_dpp<0x4E>(x);     // quad_perm [2, 3, 0, 1]
  return max_dpp<0xB1>(x);  // quad_perm [1, 0, 3, 2]
}

// Eight values from `at` of a row of `cols`, at any alignment (global accesses need none on this
// target); zeros past the end.
template <typename T>
__device__ __forceinline__ void load8(const char* row, int at, int cols, float (&v)[8]) {
  if (at + 8 <= cols) {
    if constexpr (sizeof(T) == 4) {
      __builtin_memcpy(v, row + 4 * (int64_t)at, 32);
    } else {
      u32x4 w;
      __builtin_memcpy(&w, row + 2 * (int64_t)at, 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[2 * e] = ss::Elem<T>::lo(w[e]);
        v[2 * e + 1] = ss::Elem<T>::hi(w[e]);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = at + e < cols ? (float)((const T*)row)[at + e] : 0.f;
  }
}

// y (fp32, near the quotient x * 448 / a), moved off a halfway point of e4m3 that the exact
// quotient does not lie on
__device__ __forceinline__ float settle(float y, float x, float a) {
  const float t = fabsf(y);
  const int e = max((int)(__builtin_bit_cast(uint32_t, t) >> 23) - 127, -6);
  const float u = ldexpf(t, 3 - e), whole = floorf(u);  // in steps of e4m3
  if (fabsf(u - whole - 0.5f) > 1e-5f) return y;
  const double exact = ldexp((double)fabsf(x) * 448.0, 3 - e), half = (double)(whole + 0.5f) * (double)a;
  const float off = exact < half ? 0.25f : exact > half ? 0.75f : 0.5f;
  return copysignf(ldexpf(whole + off, e - 3), y);
}

// Sixteen lanes take a block, eight columns each; a wave the same block of four rows, a workgroup of
// sixteen, so that the scales, kept block by block, are written 64 bytes at a time. Two blocks a
// lane, both requested before the first is used. Bound by memory.
template <typename T>
__global__ __launch_bounds__(256) void fp8_rows_kernel(const Fp8RowArgs a) {
  const int64_t tile = blockIdx.x / a.pairs;
  const int b0 = 2 * (int)(blockIdx.x - tile * a.pairs);
  const int64_t row = 16 * tile + (threadIdx.x >> 4);
  const int sub = 8 * (threadIdx.x & 15);
  const char* const xr = a.x + (row < a.rows ? row : a.rows - 1) * a.x_stride;
  float v[2][8];
#pragma unroll
  for (int u = 0; u < 2; ++u) load8<T>(xr, 128 * (b0 + u) + sub, a.cols, v[u]);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __builtin_bit_cast(uint32_t, v[u][e]) & 0x7FFFFFFFu);
    top = row_max(top);
    if (row >= a.rows || b0 + u >= a.blocks) continue;
    const float amax = __builtin_bit_cast(float, top);
    const bool live = top < kInf && amax >= kSmallest;
    uint32_t w[2] = {0, 0};
    if (live) {
      const float m = __builtin_bit_cast(float, (top & 0x7FFFFFu) | 0x3F800000u);
      const float c = __builtin_bit_cast(float, ((262u - (top >> 23)) << 23) | 0x600000u);  // 448 * 2^-e
      const float r = 1.f / m;
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float s = v[u][e] * c, y0 = s * r;
        y[e] = fmaf(fmaf(-y0, m, s), r, y0);
        if constexpr (sizeof(T) == 4) y[e] = settle(y[e], v[u][e], amax);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        int p = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h], y[4 * h + 1], 0, false);
        w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h + 2], y[4 * h + 3], p, true);
      }
    }
    const int at = 128 * (b0 + u) + sub;
    uint8_t* const q = a.q + row * a.cols + at;
    if (at + 8 <= a.cols) {
      __builtin_memcpy(q, w, 8);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (at + e < a.cols) q[e] = (uint8_t)(w[e >> 2] >> (8 * (e & 3)));
    }
    if (sub == 0)
      a.scale[(b0 + u) * a.scale_stride + row] = top >= kInf ? __builtin_nanf("") : live ? amax / 448.f : 0.f;
  }
}

}  // namespace

extern "C" int ss_quantize_fp8(const void* x, uint8_t* q, float* scale, int64_t rows, int64_t cols, int64_t x_stride,
                               int64_t scale_stride, int dtype, void* stream) {
  const char* who = "quantize_fp8";
  if (rows < 0 || cols < 0) {
    ss_host::set_error("%s: negative extent", who);
    return SS_ERR_INVALID;
  }
  if (dtype != SS_DTYPE_BF16 && dtype != SS_DTYPE_F16 && dtype != SS_DTYPE_F32) {
    ss_host::set_error("%s: dtype code %d not supported", who, dtype);
    return SS_ERR_UNSUPPORTED;
  }
  if (rows == 0 || cols == 0) return SS_OK;
  if (!x || !q || !scale) {
    ss_host::set_error("%s: null pointer", who);
    return SS_ERR_INVALID;
  }
  if ((rows > 1 && x_stride < cols) || scale_stride < rows) {
    ss_host::set_error("%s: row stride shorter than the rows, or scale stride than their number", who);
    return SS_ERR_INVALID;
  }
  const int64_t tiles = (rows + 15) / 16, pairs = (cols + 255) / 256;
  if (cols >= ((int64_t)1 << 30) || tiles * pairs >= (1 << 24)) {  // workgroups of 256 threads: below 2^32
    ss_host::set_error("%s: %lld x %lld are more than one launch holds", who, (long long)rows, (long long)cols);
    return SS_ERR_UNSUPPORTED;
  }
  const Fp8RowArgs a = {(const char*)x, q,         scale, x_stride * (dtype == SS_DTYPE_F32 ? 4 : 2),
                        scale_stride,   rows,      (int)cols, (int)((cols + 127) / 128), (int)pairs};
  const dim3 grid((unsigned)(tiles * pairs)), block(256);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == SS_DTYPE_BF16)
    hipLaunchKernelGGL(fp8_rows_kernel<ss::bf16_t>, grid, block, 0, s, a);
  else if (dtype == SS_DTYPE_F16)
    hipLaunchKernelGGL(fp8_rows_kernel<ss::f16_t>, grid, block, 0, s, a);
  else
    hipLaunchKernelGGL(fp8_rows_kernel<float>, grid, block, 0, s, a);
  return ss_host::launch_status(who);
}
