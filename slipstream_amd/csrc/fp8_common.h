// Shared by the kernels of the product in 8-bit floating point: the call's parameters and the
// matrix instruction.
#pragma once

#include "w8a8_common.h"

namespace ss {

struct F8Params {
  const uint8_t* x;      // [m, k] e4m3, row stride x_stride
  const uint8_t* w;      // [n, k] e4m3, row stride w_stride
  const float* x_scale;  // (row, block of 128 k) at row * xs_row + block * xs_blk
  const float* w_scale;  // (block of 128 n, block of 128 k) at nb * ws_row + block * ws_blk
  const void* bias;      // [n] or null
  void* out;             // [m, n], row stride o_stride
  int64_t m, n;
  int64_t x_stride, w_stride, o_stride;  // elements
  int64_t xs_row, xs_blk, ws_row, ws_blk;
  int k;
  int bias_dtype;
};

// The tile kernel (fp8_tile.hip): a workgroup's tokens and channels, its grid and K split.
struct F8TilePlan {
  int bm, bn;
  int ks, per;  // K ranges and blocks of 128 keys per range
  int n_tiles, m_blocks;
};
// The stream kernel (fp8_stream.hip): a workgroup's 16-row tiles of tokens and channels, its waves and its grid.
struct F8StreamPlan {
  int mt, nt, waves;
  int n_tiles, m_blocks;
  bool once;  // the weights pass the caches by
};
double plan_fp8_stream(F8StreamPlan& pl, int64_t m, int64_t n, int64_t k);  // estimated us
int launch_fp8_stream(const F8Params& p, const F8StreamPlan& pl, int out_dtype, hipStream_t stream);

double plan_fp8_tile(F8TilePlan& pl, int64_t m, int64_t n, int64_t k, bool wide, bool may_split);  // estimated us
int launch_fp8_tile(const F8Params& p, const F8TilePlan& pl, int out_dtype, float* part, hipStream_t stream);

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// a b over 128 keys of e4m3: lane l holds 32 keys of row l % 16 of a (of b: of column l % 16), its
// results are rows 4 (l / 16) .. + 3 of column l % 16. Any order of the keys gives the same products,
// so long as a and b share it.
//
// Two ways to sum them. The instruction for e4m3 (5 PFLOP/s) does not keep fp32's bits between the
// products of one block: it aligns those of eight keys to the largest sum of exponents among them (a
// subnormal's counts as that of 2^-6, a product with zero does not count) and drops what lies below 2^-13
// of it (measured over every pair of values; the instruction of K = 32 gives the same bits). So 128 products
// of normal values are off by 2^-16 of themselves on average, eight by 7 * 2^-13 of the largest at most (eight
// times that where its smaller operand is subnormal: below 2^-14 of its block's largest value). bf16's half step is
// 2^-9 to 2^-8, and the instruction is taken for results in bf16 alone. For fp16 and fp32 the operands are widened to bf16, which holds
// every e4m3 value, and summed by that type's instruction (2.5 PFLOP/s; 2^-26.7 of itself on average).
__device__ __forceinline__ f32x4 sum_fp8(i32x8 a, i32x8 b) {
  // (its own scales, powers of two, are not used: with both zero the compiler takes the unscaled form)
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}

__device__ __forceinline__ uint32_t widen2(int word, int half) {
  const bf16x2 v = half ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, 1.f, true)
                        : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, 1.f, false);
  return __builtin_bit_cast(uint32_t, v);
}
// A lane's 32 keys in bf16, eight for each of four products
struct Wide {
  u32x4 v[4];
};
__device__ __forceinline__ Wide widen(i32x8 x) {
  Wide w;
#pragma unroll
  for (int s = 0; s < 4; ++s)
    w.v[s] = u32x4{widen2(x[2 * s], 0), widen2(x[2 * s], 1), widen2(x[2 * s + 1], 0), widen2(x[2 * s + 1], 1)};
  return w;
}
__device__ __forceinline__ f32x4 sum_wide(const Wide& a, const Wide& b) {
  f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < 4; ++s) c = Elem<bf16_t>::mfma(a.v[s], b.v[s], c);
  return c;
}

// The operand of a result type, and the sum of a block's products from two
template <typename TO>
struct Block {
  typedef Wide Operand;
  static __device__ __forceinline__ Operand operand(i32x8 x) { return widen(x); }
  static __device__ __forceinline__ f32x4 sum(const Operand& a, const Operand& b) { return sum_wide(a, b); }
};
template <>
struct Block<bf16_t> {
  typedef i32x8 Operand;
  static __device__ __forceinline__ Operand operand(i32x8 x) { return x; }
  static __device__ __forceinline__ f32x4 sum(Operand a, Operand b) { return sum_fp8(a, b); }
};

__device__ __forceinline__ i32x8 join8(i32x4 lo, i32x4 hi) {
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// 16-byte chunk c of row r of a 16-row tile lies at chunk c ^ f8_swizzle(r) of its 128 LDS bytes: a 16-byte
// read takes rows 0-3 and 12-15 of one key group with rows 4-11 of the next, whose chunk differs by 2, in a
// pass; rows 2p and 2p + 1 lie in different halves of the banks, and this value keeps the row pairs of a pass
// apart.
__device__ __forceinline__ int f8_swizzle(int r) {
  const int p = r >> 1;
  return (((p >> 2) ^ (p >> 1)) & 1) << 2 | ((p >> 2) & 1) << 1 | (p & 1);
}

// Sixteen keys of a row at any alignment, zeros past the row's end
__device__ __forceinline__ i32x4 load_keys8(const uint8_t* row, int at, int k) {
  i32x4 v = {0, 0, 0, 0};
  if (at + 16 <= k) {
    __builtin_memcpy(&v, row + at, 16);
  } else if (at < k) {
    uint32_t w[4] = {0, 0, 0, 0};
    for (int e = 0; e < k - at; ++e) w[e >> 2] |= (uint32_t)row[at + e] << (8 * (e & 3));
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (int)w[e];
  }
  return v;
}

}  // namespace
}  // namespace ss
