// Device helpers shared by the W8A8 kernels: the call's parameters, the int8 matrix
// instruction and the scaled store of a result.
#pragma once

#include <atomic>

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

// The tile kernel (w8a8_tile.hip): a workgroup's tokens and channels, its grid and K split.
struct TilePlan {
  int bm, bn;
  int ks, per;  // K ranges and 128-key stages per range
  int n_tiles, m_blocks;
  bool once;    // the weights pass the caches by
};
constexpr int64_t kMostGroups = 1 << 22;  // workgroups of a launch (of at most 512 threads: below 2^32)

// The stream kernel (w8a8_stream.hip): a workgroup's 16-row tiles of tokens and channels, its
// waves and its grid.
struct StreamPlan {
  int mt, nt, waves;
  int n_tiles, m_blocks;
  bool once;    // the weights pass the caches by
};
double plan_w8a8_stream(StreamPlan& pl, int64_t m, int64_t n, int64_t k);  // estimated us
int launch_w8a8_stream(const W8Params& p, const StreamPlan& pl, int out_dtype, hipStream_t stream);

double plan_w8a8_tile(TilePlan& pl, int64_t m, int64_t n, int64_t k, bool may_split);  // estimated us
int launch_w8a8_tile(const W8Params& p, const TilePlan& pl, int out_dtype, int* part, hipStream_t stream);

// Rows of bytes that are copied (w8a8.hip) to ones that begin on 16 bytes and end with 16, zeros behind them;
// 0 rows: none. As many rows a launch as its 32-bit piece numbers hold.
struct ByteRows {
  const int8_t* from;
  int8_t* to;
  int64_t stride;  // of `from`
  int rows;
};
int align_rows(ByteRows x, ByteRows w, int k, hipStream_t stream);

// Weights that one token block reads pass the caches by beyond this many bytes. Out of the memory that
// is 2 to 16 % faster at any size (24 x 28672 x 4096 25.1 -> 23.2 us, 24 x 4096 x 14336 18.0 ->
// 17.3, 64 x 28672 x 4096 30.8 -> 25.9, 64 x 14336 x 4096 20.5 -> 19.7), but up to 46 % slower for
// weights that the 256 MB cache still has from the call before (24 x 4096 x 14336 11.5 -> 14.5, 64 x
// 14336 x 4096 13.2 -> 19.3). A call does not know which it is. Three such weights in turn are
// kept at 59 MB and not at 117 (28672 x 4096 takes the same time either way: 25.0 and 25.1), so the
// size of one weight decides: a model whose weights are all below it and more than the cache
// altogether loses 2 to 8 %.
constexpr int64_t kKeptWeights = 64 << 20;

// Lets `kern` have `lds` bytes of dynamic LDS on the current device; `done` holds a bit for each
// device where it has them already (the attribute belongs to the function on a device).
inline int reserve_lds(const void* kern, int lds, std::atomic<uint64_t>& done) {
  int device = 0;
  const uint64_t bit = hipGetDevice(&device) == hipSuccess && device >= 0 && device < 64 ? 1ull << device : 0;
  if (lds <= 65536 || (done.load(std::memory_order_relaxed) & bit)) return SS_OK;
  if (hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) {
    ss_host::set_error("w8a8 gemm: cannot reserve %d bytes of LDS", lds);
    return SS_ERR_UNSUPPORTED;
  }
  done.fetch_or(bit, std::memory_order_relaxed);
  return SS_OK;
}

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

typedef int i32x16 __attribute__((ext_vector_type(16)));

// Position of 16-byte chunk c of row r within the row's 128 LDS bytes: c ^ tile_swizzle(r).
// A 16-byte LDS read runs in four passes of sixteen lanes, lanes 0-3, 12-15, 20-27 first,
// then 4-11, 16-19, 28-31, and the same of the upper half. The rows 2p and 2p + 1 lie in
// different halves of the 64 banks, and the row pairs of each pass differ in p % 8.
__device__ __forceinline__ int tile_swizzle(int r) { return (r >> 1) & 7; }

// The result of one output from its exact integer sum, before it is rounded to the output's
// type: three roundings in fp32, the sum's, the product's and that of the second product with the
// bias.
__device__ __forceinline__ float scaled(int sum, float xs, float ws, float bias) {
  return fmaf((float)sum * xs, ws, bias);
}

// N consecutive results (16 bytes) in the output's type
template <int N>
__device__ __forceinline__ void pack_results(float (&o)[N], const float (&y)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) o[e] = y[e];
}
template <int N, typename T>
__device__ __forceinline__ void pack_results(T (&o)[N], const float (&y)[N]) {
  static_assert(N == 8, "sixteen bytes");
  const u32x4 w = {Elem<T>::pack2(y[0], y[1]), Elem<T>::pack2(y[2], y[3]), Elem<T>::pack2(y[4], y[5]),
                   Elem<T>::pack2(y[6], y[7])};
  __builtin_memcpy(o, &w, 16);
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_over(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
}

// The biases of `chans` channels from n0 on, of whatever type, read without a branch on it (a
// load inside such a branch makes the compiler wait for every load before it, one channel
// after another): the aligned dword that holds a bias, through a descriptor that is empty where
// there are none, shifted so that its bits are the low ones, and decoded under bit masks.
struct BiasReader {
  __amdgpu_buffer_rsrc_t rs;
  uint32_t skew, size, f16_mask, bf16_mask;
};
__device__ __forceinline__ BiasReader bias_reader(const W8Params& p, int64_t n0, int chans) {
  BiasReader b;
  b.size = p.bias_dtype == SS_DTYPE_F32 ? 4 : 2;
  const uint64_t at = (uint64_t)p.bias + n0 * b.size;
  b.skew = (uint32_t)at & 3u;
  b.rs = buffer_over((const void*)(at & ~3ull), p.bias ? (b.skew + chans * b.size + 3) & ~3u : 0u);
  b.f16_mask = p.bias_dtype == SS_DTYPE_F16 ? ~0u : 0u;
  b.bf16_mask = p.bias_dtype == SS_DTYPE_BF16 ? ~0u : 0u;
  return b;
}
__device__ __forceinline__ uint32_t bias_bits(const BiasReader& b, int c) {  // c: from n0
  const uint32_t off = b.skew + c * b.size;
  return (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(b.rs, (int)(off & ~3u), 0, 0) >> (8 * (off & 2u));
}
__device__ __forceinline__ float bias_value(const BiasReader& b, uint32_t bits) {
  const uint32_t f16 = __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(f16_t, (uint16_t)(bits & 0xFFFFu)));
  const uint32_t bf16 = bits << 16;
  return __builtin_bit_cast(float, (f16 & b.f16_mask) | (bf16 & b.bf16_mask) | (bits & ~(b.f16_mask | b.bf16_mask)));
}

// A raw buffer descriptor over [base, base + bytes) as four scalars: offsets past the end read
// zeros without a memory access.
__device__ __forceinline__ i32x4 buffer_words(const void* base, uint32_t bytes) {
  const uint64_t a = (uint64_t)base;
  return i32x4{(int)(uint32_t)a, (int)((uint32_t)(a >> 32) & 0xFFFF), (int)bytes, 0x00020000};
}

// 16 bytes per lane from rs + voff + soff straight into LDS at lds + 16 * lane (M0 holds the
// LDS destination, written just before: the load may read it one wait state later). Written
// as asm, with no register to write, so that the compiler's waits do not count it: the
// kernel waits itself.
// STREAM: not kept in the caches, for what is read once.
typedef __attribute__((address_space(3))) char* LdsBytes;
template <bool STREAM = false>
__device__ __forceinline__ void dma_b128(i32x4 rs, LdsBytes lds, int voff, int soff) {
  const uint32_t m0 = (uint32_t)(uintptr_t)lds;
  if constexpr (STREAM)
    asm volatile("s_nop 1\n\tbuffer_load_dwordx4 %0, %1, %2 offen nt lds"
                 :
                 : "v"(voff), "s"(rs), "s"(soff), "{m0}"(m0)
                 : "memory");
  else
    asm volatile("s_nop 1\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds"
                 :
                 : "v"(voff), "s"(rs), "s"(soff), "{m0}"(m0)
                 : "memory");
}

}  // namespace
}  // namespace ss
