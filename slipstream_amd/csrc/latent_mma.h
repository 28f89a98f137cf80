// Device helpers shared by the matrix-core kernels of attention over latents: products of 32 x 32 x 16,
// the swizzle of rows in the LDS.
#pragma once

#include "latent_common.h"
#include "tile_order.h"

namespace ss {
namespace {

constexpr int kRopeDim = 64;
constexpr float kSlack = 8.f;  // by which (log2) a score may exceed the running maximum before that is raised

typedef short tr16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// Where the 16-byte chunk c of a row r of 256 bytes and more lies in the LDS: at c ^ lat_swizzle(r). The 16
// lanes of a pass of a 16-byte read have different rows (mod 16) and lie in different banks; of
// eight rows in order the low two bits and the highest differ, so that the 8-byte pieces of four
// chunks that differ in bit 2 (and their halves) do so too.
__device__ __forceinline__ int lat_swizzle(int r) { return (r & 3) | ((r & 4) << 1) | ((r & 8) >> 1); }

// s = a b (FIRST) or s += a b, chained; reading s is for the caller to wait for
template <typename T, bool FIRST>
__device__ __forceinline__ void mfma32_sum(f32x16& s, u32x4 a, u32x4 b) {
  if constexpr (std::is_same<T, bf16_t>::value) {
    if constexpr (FIRST)
      asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(s) : "v"(a), "v"(b));
    else
      asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(s) : "v"(a), "v"(b));
  } else {
    if constexpr (FIRST)
      asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, 0" : "=&v"(s) : "v"(a), "v"(b));
    else
      asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(s) : "v"(a), "v"(b));
  }
}
// (without the quieting of NaNs that fmaxf has: a score that is none makes its row one anyway)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// Probabilities are 2^(score - m) for a row's m, raised to its maximum score less kHeadroom: in fp16 they reach 2^15 (the
// largest value is below 2^16) and 2^-32 of the largest score's is left, where from 2^0 down to 2^8 it would be 2^-25:
// many keys that far below one may make up a row whose largest key's value is small. bf16 has fp32's range.
template <typename T>
constexpr float kHeadroom = std::is_same<T, f16_t>::value ? 7.f : 0.f;

// A row's sum goes over its probabilities as the product over keys takes them, rounded to the inputs' type: so the
// weights of its values sum to one, and of a key that outweighs all others the row is its value, whatever 2^x (x up to
// kSlack) its probability is. (Of the unrounded ones such a row is off by up to half a step.)
template <typename T>
__device__ __forceinline__ float pair_sum(uint32_t w) {
  return Elem<T>::lo(w) + Elem<T>::hi(w);
}

// The operand of 16 keys of a product over keys, from rows of the LDS: the lane's four keys at `lo`, and
// those eight rows on at `hi`. Within sixteen lanes, lane i receives element i % 4 of the 8-byte reads of
// lanes i / 4 + 4 e (e = 0 .. 3).
__device__ __forceinline__ u32x4 lds_keys(uint32_t lo, uint32_t hi) {
  typedef __attribute__((address_space(3))) tr16x4* Tr;
  const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Tr)(uintptr_t)lo));
  const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Tr)(uintptr_t)hi));
  return u32x4{a[0], a[1], b[0], b[1]};
}

}  // namespace
}  // namespace ss
