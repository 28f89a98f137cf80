// Device helpers shared by the W8A8 kernels: the call's parameters, the int8 matrix
// instruction and the scaled store of a result.
#pragma once

#include "ss_common.h"

namespace ss {

typedef int i32x4 __attribute__((ext_vector_type(4)));

struct W8Params {
  const int8_t* x;       // [m, k], row stride x_stride
  const int8_t* w;       // [n, k], row stride w_stride
  const float* x_scale;  // [m]
  const float* w_scale;  // [n]
  const void* bias;      // [n] or null
  void* out;             // [m, n], row stride o_stride
  int64_t m, n;
  int64_t x_stride, w_stride, o_stride;  // elements
  int k;
  int bias_dtype;
};

namespace {

// c += a b over 64 keys: lane l's sixteen bytes of a are keys 16 (l / 16) .. + 15 of row l % 16
// (of b: of column l % 16), its results rows 4 (l / 16) .. + 3 of column l % 16. Any order of
// the keys gives the same sums, so long as a and b share it.
__device__ __forceinline__ i32x4 mfma_i8(i32x4 a, i32x4 b, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ float load_as_f32(const void* p, int64_t i, int dtype) {
  if (dtype == SS_DTYPE_F16) return (float)((const f16_t*)p)[i];
  if (dtype == SS_DTYPE_BF16) return (float)((const bf16_t*)p)[i];
  return ((const float*)p)[i];
}

// The result of one output from its exact integer sum, before it is rounded to the output's
// type: three roundings in fp32 (four with a bias).
__device__ __forceinline__ float scaled(int sum, float xs, float ws, float bias) {
  return fmaf((float)sum * xs, ws, bias);
}

}  // namespace
}  // namespace ss
