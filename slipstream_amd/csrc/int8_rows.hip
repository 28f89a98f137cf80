// Rows quantized to int8 with one fp32 scale each, for gfx950: the inputs of the W8A8 product
// (w8a8.hip). Plain rows, rows behind an RMSNorm with the residual's addition, and rows behind
// SwiGLU, each in one pass over memory.
//
// Mathematics, for a row y of fp32 values:
//   a = max |y|;  scale = a / 127;  q = rint(y * 127 / a), half to even;  y ~ q * scale.
//   Plain rows and SwiGLU: 1 / a, its product with 127 and the product with y are each rounded to
//   fp32, so that elementary operations on the same y give the same q. Norms: the exact q.
//   A row whose scale would be subnormal (a < 127 * 2^-126) is zeros with scale zero: 127 / a
//   stays finite, and what is dropped is below 1.5e-36. Norms go by p below, before r is known.
//   A row that holds a NaN or an infinity gets zeros and the scale NaN, so that every product
//   with it is NaN and none is silently finite. The maximum is taken over the magnitudes' bit
//   patterns as unsigned integers, in which infinity follows every number and NaN infinity.
// RMSNorm: s = x + residual, rounded to the inputs' type (it is also returned: the next
//   residual), r = 1 / sqrt(mean(s^2) + eps), y = s * w * r. Since r scales a whole row, q does
//   not depend on it: with p = s * w (exact in fp32 for 16-bit types) and a = max |p|,
//   q = rint(p * 127 / a) and scale = r * a / 127. So both reductions, the sum of squares and
//   the maximum, share one exchange between the waves, and q is the same whatever the order
//   of the sum. Nothing is rounded to 16 bits between the norm and its int8 values. A row whose
//   squares' sum fp32 does not hold has it taken again, of s times a power of two.
// SwiGLU: y = g / (1 + exp(-g)) * u, each operation rounded to fp32 and none to 16 bits.
#include "ss_common.h"

namespace {

using ss::u32x4;

enum Mode { kRows, kNorm, kNormRes, kSwiglu };

struct RowArgs {
  const char* x;    // rows; SwiGLU: gate
  const char* y;    // residual; SwiGLU: up
  const char* w;    // norm weight
  int8_t* q;        // [rows, cols], contiguous
  float* scale;     // [rows]
  char* s;          // x + residual, contiguous
  int64_t x_stride, y_stride;  // bytes
  int cols;
  float eps;
};

constexpr float kLevels = 127.f;
constexpr float kSmallest = 127.f * 1.17549435e-38f;  // 127 * 2^-126

template <typename T>
__device__ __forceinline__ void unpack(const u32x4& w, float (&f)[16 / sizeof(T)]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t u = w[e];
      f[e] = __builtin_bit_cast(float, u);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[2 * e] = ss::Elem<T>::lo(w[e]);
      f[2 * e + 1] = ss::Elem<T>::hi(w[e]);
    }
  }
}
template <typename T>
__device__ __forceinline__ u32x4 pack(const float (&f)[16 / sizeof(T)]) {
  u32x4 w;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (sizeof(T) == 4)
      w[e] = __builtin_bit_cast(uint32_t, f[e]);
    else
      w[e] = ss::Elem<T>::pack2(f[2 * e], f[2 * e + 1]);
  }
  return w;
}

// keeps the compiler from contracting x + r or s * w with what follows
__device__ __forceinline__ float pin(float x) {
  asm volatile("" : "+v"(x));
  return x;
}

__device__ __forceinline__ uint32_t magnitude(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu; }

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, true);
}
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t wave_umax(uint32_t x) {
  const auto s32 = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  x = umax(s32[0], s32[1]);
  const auto s16 = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = umax(s16[0], s16[1]);
  x = umax(x, dpp<0x128>(x));  // row_ror:8
  x = umax(x, dpp<0x124>(x));  // row_ror:4
  x = umax(x, dpp<0x4E>(x));   // quad_perm [2, 3, 0, 1]
  return umax(x, dpp<0xB1>(x));
}
template <int CTRL>
__device__ __forceinline__ float add_dpp(float x) {
  return x + __builtin_bit_cast(float, dpp<CTRL>(__builtin_bit_cast(uint32_t, x)));
}
__device__ __forceinline__ float wave_sum(float x) {
  x = ss::sum_across_rows(x);
  x = add_dpp<0x128>(x);
  x = add_dpp<0x124>(x);
  x = add_dpp<0x4E>(x);
  return add_dpp<0xB1>(x);
}

// g / d for a divisor d = 1 + exp(-g), rounded to nearest: a reciprocal refined by one Newton step, and
// Markstein's correction of the quotient by its remainder (the range scaling that a general
// division adds has nothing to do for a divisor from 1 to kFarDivisor, up to which the reciprocal is no
// subnormal: 2240 x 14336 38.1 us with it, 32.6 so, 28.0 with the hardware's exp2 and reciprocal
// alone, whose last bits moved some tens of q by a step).
constexpr float kFarDivisor = 0x1p126f;
__device__ __forceinline__ float silu_quotient(float g, float d) {
  const float r0 = __builtin_amdgcn_rcpf(d), r = fmaf(fmaf(-d, r0, 1.f), r0, r0), q = g * r;
  return fmaf(fmaf(-d, q, g), r, q);
}

// The low bytes of four words in a dword.
__device__ __forceinline__ uint32_t low_bytes(uint32_t b0, uint32_t b1, uint32_t b2, uint32_t b3) {
  return __builtin_amdgcn_perm(b1, b0, 0x0C0C0400u) | __builtin_amdgcn_perm(b3, b2, 0x04000C0Cu);
}
// Four values times 127 / a -> four int8 in a dword. A product plus 1.5 * 2^23 (2^52) is rounded to
// an integer, half to even, whose two's complement is the sum's low bits. Rows and SwiGLU round
// the product to fp32 first, as an elementary product does. Norms do it in 64 bits, where q is the
// exact quotient's nearest, half to even: the product is first rounded to multiples of 2^-40. With
// 24 bits in p and a, a quotient that is no half is 2^-33 away from one at least (|p| > a / 254 there,
// so p 254 - a (2 n + 1), over 2 a, counts units of a 2^-32), and the error of 127 / a moves it by
// 2^-46 at most. A step of one normalised value changes every output of its row behind the next
// product, and 16-bit rows hold many exact halves (2240 x 4096 10.69 us in 32 bits, 10.8 so).
__device__ __forceinline__ uint32_t quant4(const float* p, float inv) {
  uint32_t b[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) b[e] = __builtin_bit_cast(uint32_t, pin(p[e] * inv) + 12582912.f);
  return low_bytes(b[0], b[1], b[2], b[3]);
}
__device__ __forceinline__ uint32_t quant4(const float* p, double inv) {
  uint32_t b[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const double fine = fma((double)p[e], inv, 6144.0);  // 1.5 * 2^12
    b[e] = (uint32_t)__builtin_bit_cast(uint64_t, fine + (6755399441055744.0 - 6144.0));
  }
  return low_bytes(b[0], b[1], b[2], b[3]);
}
template <int MODE>
struct InvOf {
  typedef float type;
};
template <>
struct InvOf<kNorm> {
  typedef double type;
};
template <>
struct InvOf<kNormRes> {
  typedef double type;
};

// 16 bytes at any alignment (global accesses need none on this target). A row's last, partial
// piece is put together from the aligned words that hold its elements, read at the last one
// where they lie behind it, zeros past the row's end: loads that are each under their own
// condition wait for one another (SwiGLU of 11 x 4863 in fp16 3.96 us, so
// 3.54).
template <typename T>
__device__ __forceinline__ u32x4 load_piece(const char* row, int i, int cols) {
  constexpr int EPP = 16 / sizeof(T);
  u32x4 v = {0u, 0u, 0u, 0u};
  const char* const at = row + (int64_t)i * sizeof(T);
  if (i + EPP <= cols) {
    __builtin_memcpy(&v, at, 16);
  } else if (i < cols) {
    const int left = (cols - i) * (int)sizeof(T);
    const uint64_t from = (uint64_t)at, last = (from + left - 1) & ~3ull;
    uint32_t w[5];
#pragma unroll
    for (int e = 0; e < 5; ++e) {
      const uint64_t word = (from & ~3ull) + 4 * e;
      w[e] = *reinterpret_cast<const uint32_t*>(word < last ? word : last);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int bytes = left - 4 * e;  // that are left for this word
      const uint32_t mask = bytes >= 4 ? ~0u : bytes > 0 ? (1u << (8 * bytes)) - 1u : 0u;
      v[e] = __builtin_amdgcn_alignbyte(w[e + 1], w[e], (uint32_t)from & 3u) & mask;
    }
  }
  return v;
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_rsrc(const char* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p), 0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ u32x4 rsrc_piece(__amdgpu_buffer_rsrc_t r, int at) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0));
}

// What a piece contributes: its values y (norms: p), their largest magnitude, and for norms
// the sum of squares of s; with a residual `xw` becomes x + residual in T.
template <typename T, int MODE>
__device__ __forceinline__ void fold(u32x4& xw, const u32x4& yw, const u32x4& ww, float (&v)[16 / sizeof(T)],
                                     uint32_t& top, float& sq) {
  constexpr int EPP = 16 / sizeof(T);
  unpack<T>(xw, v);
  if constexpr (MODE == kNormRes) {
    float r[EPP];
    unpack<T>(yw, r);
#pragma unroll
    for (int e = 0; e < EPP; ++e) v[e] = pin(v[e] + r[e]);
    xw = pack<T>(v);
    unpack<T>(xw, v);
  }
  if constexpr (MODE == kNorm || MODE == kNormRes) {
    float w[EPP];
    unpack<T>(ww, w);
#pragma unroll
    for (int e = 0; e < EPP; ++e) {
      sq = fmaf(v[e], v[e], sq);
      v[e] = pin(v[e] * w[e]);
    }
  }
  if constexpr (MODE == kSwiglu) {
    float u[EPP], g[EPP], d[EPP], far = 0.f;
    unpack<T>(yw, u);
#pragma unroll
    for (int e = 0; e < EPP; ++e) {
      g[e] = v[e];
      d[e] = 1.f + expf(-g[e]);
      far = fmaxf(far, d[e]);
      v[e] = silu_quotient(g[e], d[e]) * u[e];
    }
    if (far > kFarDivisor) {  // gates below -87.3: the general division, in pieces that hold such a gate
#pragma unroll
      for (int e = 0; e < EPP; ++e) v[e] = g[e] / d[e] * u[e];
    }
  }
#pragma unroll
  for (int e = 0; e < EPP; ++e) top = umax(top, magnitude(v[e]));
}

template <int MODE>
struct RowEnd {
  typename InvOf<MODE>::type inv;  // 127 / a, zero where q is
  float peak;                      // a
  float by;                        // norms: not zero where the scale is still to be found, by scale_again
};

// The row's largest magnitude and sum over the workgroup, then 127 / a, and the scale written.
template <int MODE, int WAVES>
__device__ __forceinline__ RowEnd<MODE> finish_row(uint32_t top, float sq, const RowArgs& a, int64_t row) {
  __shared__ uint32_t s_top[WAVES];
  __shared__ float s_sq[WAVES];
  top = wave_umax(top);
  if constexpr (MODE == kNorm || MODE == kNormRes) sq = wave_sum(sq);
  if constexpr (WAVES > 1) {
    if ((threadIdx.x & 63) == 0) {
      s_top[threadIdx.x >> 6] = top;
      s_sq[threadIdx.x >> 6] = sq;
    }
    __syncthreads();
    top = s_top[0];
    sq = s_sq[0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) {
      top = umax(top, s_top[i]);
      sq += s_sq[i];
    }
  }
  RowEnd<MODE> end = {0, __builtin_bit_cast(float, top), 0.f};
  const bool finite = top < 0x7F800000u, live = finite && end.peak >= kSmallest;
  if (live) {
    if constexpr (__is_same(decltype(end.inv), double))
      end.inv = (double)kLevels / (double)end.peak;
    else  // 1 / a is subnormal, so short of bits, from 2^126 on
      end.inv = end.peak < 0x1p126f ? kLevels * (1.f / end.peak) : kLevels / end.peak;
  }
  if constexpr (MODE == kNorm || MODE == kNormRes)
    if (live) {
      if (sq > 0x1.fffffep127f) end.by = 0x1p-96f;
      if (sq < 0x1p-96f && a.eps < 0x1p-60f) end.by = 0x1p96f;
    }
  if (threadIdx.x == 0) {
    float scale = live ? end.peak / kLevels : 0.f;
    if constexpr (MODE == kNorm || MODE == kNormRes)
      if (live) scale *= 1.f / __builtin_sqrtf(sq / (float)a.cols + a.eps);
    a.scale[row] = finite ? scale : __builtin_nanf("");
  }
  return end;
}

// The scale of a norm's row whose sum of squares is not one that fp32 holds: infinite, or below 2^-96,
// where squares that were subnormal count (unless eps outweighs them all). Of s times 2^-96 (2^96) the
// squares that count are from 2^-106 on and their sum is below 2^125; the rest is done in
// doubles. It comes after the row's stores, where no registers are held for it, so the sum
// written there is read again, each thread what it wrote itself.
template <typename T, int MODE, int WAVES>
__device__ __forceinline__ void scale_again(const RowEnd<MODE>& end, const RowArgs& a, int64_t row) {
  constexpr int EPP = 16 / sizeof(T);
  __shared__ float s_sq[WAVES];
  const char* const s = MODE == kNormRes ? a.s + row * a.cols * (int64_t)sizeof(T) : a.x + row * a.x_stride;
  float sq = 0.f;
#pragma unroll 1
  for (int64_t i = (int64_t)threadIdx.x * EPP; i < a.cols; i += 64 * WAVES * EPP) {
    float v[EPP];
    unpack<T>(load_piece<T>(s, (int)i, a.cols), v);
#pragma unroll
    for (int e = 0; e < EPP; ++e) sq = fmaf(v[e] * end.by, v[e] * end.by, sq);
  }
  sq = wave_sum(sq);
  if constexpr (WAVES > 1) {
    if ((threadIdx.x & 63) == 0) s_sq[threadIdx.x >> 6] = sq;
    __syncthreads();
    sq = s_sq[0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) sq += s_sq[i];
  }
  if (threadIdx.x == 0) {
    const double mean = (double)sq / (double)a.cols / ((double)end.by * (double)end.by);
    a.scale[row] = (float)((double)end.peak / (double)kLevels / __builtin_sqrt(mean + (double)a.eps));
  }
}

template <typename T, typename Inv>
__device__ __forceinline__ void store_q(int8_t* q, int i, int cols, const float (&v)[16 / sizeof(T)], Inv inv) {
  constexpr int EPP = 16 / sizeof(T);
  uint32_t d[EPP / 4];
#pragma unroll
  for (int h = 0; h < EPP / 4; ++h) d[h] = inv != (Inv)0 ? quant4(v + 4 * h, inv) : 0u;
  if (i + EPP <= cols) {
    __builtin_memcpy(q + i, d, EPP);
  } else {
#pragma unroll
    for (int e = 0; e < EPP; ++e)
      if (i + e < cols) q[i + e] = (int8_t)(d[e >> 2] >> (8 * (e & 3)));
  }
}
template <typename T>
__device__ __forceinline__ void store_s(char* s, int i, int cols, const u32x4& w) {
  constexpr int EPP = 16 / sizeof(T);
  if (i + EPP <= cols) {
    __builtin_memcpy(s + (int64_t)i * sizeof(T), &w, 16);
  } else {
    T t[EPP];
    __builtin_memcpy(t, &w, 16);
#pragma unroll
    for (int e = 0; e < EPP; ++e)
      if (i + e < cols) reinterpret_cast<T*>(s)[i + e] = t[e];
  }
}

// One workgroup per row, PPT 16-byte pieces a thread, held in registers between the reduction
// and the write, so that the row is read once. Bound by memory for many rows and by its
// latency for few: with ALIGNED rows every piece is requested before the first is used, through
// descriptors that end with the row (a piece past it reads zeros without an access). Two waves a
// SIMD at least, which the compiler does not keep to by itself (fp16 norms of 2240 x 16384 62 us, so
// 45); of rows that are not aligned the longest would spill then.
template <typename T, int MODE, int TPB, int PPT, bool ALIGNED>
__global__ __launch_bounds__(TPB) __attribute__((amdgpu_waves_per_eu(ALIGNED ? 2 : 1))) void int8_rows_kernel(
    const RowArgs a) {
  constexpr int EPP = 16 / sizeof(T);
  const int64_t row = blockIdx.x;
  const char* const xr = a.x + row * a.x_stride;
  const char* const yr = MODE == kNormRes || MODE == kSwiglu ? a.y + row * a.y_stride : xr;
  u32x4 xw[PPT], yw[PPT], ww[PPT];
  if constexpr (ALIGNED) {
    const uint32_t bytes = (uint32_t)a.cols * (uint32_t)sizeof(T);
    const auto rx = row_rsrc(xr, bytes), ry = row_rsrc(yr, bytes);
    const auto rw = row_rsrc(MODE == kNorm || MODE == kNormRes ? a.w : xr, bytes);
    const int at = 16 * threadIdx.x;
#pragma unroll
    for (int u = 0; u < PPT; ++u) {
      xw[u] = rsrc_piece(rx, at + 16 * TPB * u);
      if constexpr (MODE == kNormRes || MODE == kSwiglu) yw[u] = rsrc_piece(ry, at + 16 * TPB * u);
    }
    if constexpr (MODE == kNorm || MODE == kNormRes) {
#pragma unroll
      for (int u = 0; u < PPT; ++u) ww[u] = rsrc_piece(rw, at + 16 * TPB * u);
    }
    __builtin_amdgcn_sched_barrier(0);
  } else {
#pragma unroll
    for (int u = 0; u < PPT; ++u) {
      const int i = (threadIdx.x + TPB * u) * EPP;
      xw[u] = load_piece<T>(xr, i, a.cols);
      if constexpr (MODE == kNormRes || MODE == kSwiglu) yw[u] = load_piece<T>(yr, i, a.cols);
      if constexpr (MODE == kNorm || MODE == kNormRes) ww[u] = load_piece<T>(a.w, i, a.cols);
    }
  }
  float v[PPT][EPP];
  uint32_t top = 0;
  float sq = 0.f;
#pragma unroll
  for (int u = 0; u < PPT; ++u) fold<T, MODE>(xw[u], yw[u], ww[u], v[u], top, sq);
  const auto end = finish_row<MODE, TPB / 64>(top, sq, a, row);
  int8_t* const q = a.q + row * a.cols;
  char* const s = a.s + row * a.cols * (int64_t)sizeof(T);
#pragma unroll
  for (int u = 0; u < PPT; ++u) {
    const int i = (threadIdx.x + TPB * u) * EPP;
    if (i < a.cols) {
      store_q<T>(q, i, a.cols, v[u], end.inv);
      if constexpr (MODE == kNormRes) store_s<T>(s, i, a.cols, xw[u]);
    }
  }
  if constexpr (MODE == kNorm || MODE == kNormRes)
    if (end.by != 0.f) scale_again<T, MODE, TPB / 64>(end, a, row);
}

// Rows longer than the registers hold: the same pieces in two passes over the row, the second
// reading it again (from the caches, mostly).
template <typename T, int MODE>
__global__ __launch_bounds__(256) void int8_rows_long_kernel(const RowArgs a) {
  constexpr int EPP = 16 / sizeof(T);
  const int64_t row = blockIdx.x;
  const char* const xr = a.x + row * a.x_stride;
  const char* const yr = MODE == kNormRes || MODE == kSwiglu ? a.y + row * a.y_stride : xr;
  auto piece = [&](int i, u32x4& xw, float (&v)[EPP], uint32_t& top, float& sq) {
    u32x4 yw = {}, ww = {};
    xw = load_piece<T>(xr, i, a.cols);
    if constexpr (MODE == kNormRes || MODE == kSwiglu) yw = load_piece<T>(yr, i, a.cols);
    if constexpr (MODE == kNorm || MODE == kNormRes) ww = load_piece<T>(a.w, i, a.cols);
    fold<T, MODE>(xw, yw, ww, v, top, sq);
  };
  uint32_t top = 0;
  float sq = 0.f;
  u32x4 xw;
  float v[EPP];
  for (int64_t i = (int64_t)threadIdx.x * EPP; i < a.cols; i += 256 * EPP) piece((int)i, xw, v, top, sq);
  const auto end = finish_row<MODE, 4>(top, sq, a, row);
  int8_t* const q = a.q + row * a.cols;
  char* const s = a.s + row * a.cols * (int64_t)sizeof(T);
  for (int64_t i = (int64_t)threadIdx.x * EPP; i < a.cols; i += 256 * EPP) {
    piece((int)i, xw, v, top, sq);
    store_q<T>(q, (int)i, a.cols, v, end.inv);
    if constexpr (MODE == kNormRes) store_s<T>(s, (int)i, a.cols, xw);
  }
  if constexpr (MODE == kNorm || MODE == kNormRes)
    if (end.by != 0.f) scale_again<T, MODE, 4>(end, a, row);
}

bool al16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

template <typename T, int MODE, bool ALIGNED>
int launch_part(const RowArgs& a, int64_t rows, hipStream_t stream, const char* who) {
  const int pieces = (int)(((int64_t)a.cols * sizeof(T) + 15) / 16);
  const dim3 grid((unsigned)rows);
  if (pieces <= 64)
    hipLaunchKernelGGL((int8_rows_kernel<T, MODE, 64, 1, ALIGNED>), grid, dim3(64), 0, stream, a);
  else if (pieces <= 256)
    hipLaunchKernelGGL((int8_rows_kernel<T, MODE, 256, 1, ALIGNED>), grid, dim3(256), 0, stream, a);
  else if (pieces <= 512)
    hipLaunchKernelGGL((int8_rows_kernel<T, MODE, 256, 2, ALIGNED>), grid, dim3(256), 0, stream, a);
  else if (pieces <= 1024)
    hipLaunchKernelGGL((int8_rows_kernel<T, MODE, 256, 4, ALIGNED>), grid, dim3(256), 0, stream, a);
  else if (pieces <= 2048)
    hipLaunchKernelGGL((int8_rows_kernel<T, MODE, 256, 8, ALIGNED>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((int8_rows_long_kernel<T, MODE>), grid, dim3(256), 0, stream, a);
  return ss_host::launch_status(who);
}

// As many rows a launch as keep its threads below 2^32
template <typename T, int MODE, bool ALIGNED>
int launch_rows(RowArgs a, int64_t rows, hipStream_t stream, const char* who) {
  constexpr int64_t kMost = 1 << 23;
  for (; rows > 0; rows -= kMost) {
    const int64_t part = rows < kMost ? rows : kMost;
    const int st = launch_part<T, MODE, ALIGNED>(a, part, stream, who);
    if (st != SS_OK) return st;
    a.x += part * a.x_stride;
    if (a.y) a.y += part * a.y_stride;
    a.q += part * a.cols;
    a.scale += part;
    if (a.s) a.s += part * a.cols * (int64_t)sizeof(T);
  }
  return SS_OK;
}

template <int MODE>
int launch_mode(const RowArgs& a, int64_t rows, int dtype, hipStream_t s, const char* who) {
  const int es = dtype == SS_DTYPE_F32 ? 4 : 2;
  const bool aligned = ((int64_t)a.cols * es) % 16 == 0 && al16(a.x) && a.x_stride % 16 == 0 &&
                       (!a.y || (al16(a.y) && a.y_stride % 16 == 0)) && (!a.w || al16(a.w));
  if (dtype == SS_DTYPE_BF16)
    return aligned ? launch_rows<ss::bf16_t, MODE, true>(a, rows, s, who) : launch_rows<ss::bf16_t, MODE, false>(a, rows, s, who);
  if (dtype == SS_DTYPE_F16)
    return aligned ? launch_rows<ss::f16_t, MODE, true>(a, rows, s, who) : launch_rows<ss::f16_t, MODE, false>(a, rows, s, who);
  return aligned ? launch_rows<float, MODE, true>(a, rows, s, who) : launch_rows<float, MODE, false>(a, rows, s, who);
}

// Extents, pointers and dtype of a call; `go` false: nothing to do, or an error. Element
// counts of a row stay below 2^29, so that byte offsets in it fit 31 bits.
int check_rows(const char* who, int64_t rows, int64_t cols, int dtype, bool null, int64_t x_stride, int64_t y_stride,
               bool& go) {
  go = false;
  if (rows < 0 || cols < 0) {
    ss_host::set_error("%s: negative extent", who);
    return SS_ERR_INVALID;
  }
  if (rows == 0 || cols == 0) return SS_OK;
  if (null) {
    ss_host::set_error("%s: null pointer", who);
    return SS_ERR_INVALID;
  }
  if (dtype != SS_DTYPE_BF16 && dtype != SS_DTYPE_F16 && dtype != SS_DTYPE_F32) {
    ss_host::set_error("%s: dtype code %d not supported", who, dtype);
    return SS_ERR_UNSUPPORTED;
  }
  if (x_stride < 0 || y_stride < 0) {
    ss_host::set_error("%s: negative row stride", who);
    return SS_ERR_INVALID;
  }
  if (rows > 0x7fffffff || cols >= (1 << 29)) {
    ss_host::set_error("%s: at most 2^31 - 1 rows of fewer than 2^29 elements", who);
    return SS_ERR_UNSUPPORTED;
  }
  go = true;
  return SS_OK;
}

}  // namespace

extern "C" int ss_quantize_int8(const void* x, int8_t* q, float* scale, int64_t rows, int64_t cols, int64_t x_stride,
                                int dtype, void* stream) {
  const char* who = "quantize_int8";
  bool go;
  const int st = check_rows(who, rows, cols, dtype, !x || !q || !scale, x_stride, 0, go);
  if (!go) return st;
  const int es = dtype == SS_DTYPE_F32 ? 4 : 2;
  const RowArgs a = {(const char*)x, nullptr, nullptr, q, scale, nullptr, x_stride * es, 0, (int)cols, 0.f};
  return launch_mode<kRows>(a, rows, dtype, (hipStream_t)stream, who);
}

extern "C" int ss_rmsnorm_int8(const void* x, const void* residual, const void* weight, int8_t* q, float* scale,
                               void* sum, int64_t rows, int64_t cols, int64_t x_stride, int64_t r_stride, float eps,
                               int dtype, void* stream) {
  const char* who = "rmsnorm_int8";
  bool go;
  const int st =
      check_rows(who, rows, cols, dtype, !x || !weight || !q || !scale || (residual && !sum), x_stride, r_stride, go);
  if (!go) return st;
  const int es = dtype == SS_DTYPE_F32 ? 4 : 2;
  const RowArgs a = {(const char*)x,    (const char*)residual, (const char*)weight, q, scale, (char*)sum, x_stride * es,
                     r_stride * es, (int)cols, eps};
  if (residual) return launch_mode<kNormRes>(a, rows, dtype, (hipStream_t)stream, who);
  return launch_mode<kNorm>(a, rows, dtype, (hipStream_t)stream, who);
}

extern "C" int ss_swiglu_int8(const void* gate, const void* up, int8_t* q, float* scale, int64_t rows, int64_t cols,
                              int64_t g_stride, int64_t u_stride, int dtype, void* stream) {
  const char* who = "swiglu_int8";
  bool go;
  const int st = check_rows(who, rows, cols, dtype, !gate || !up || !q || !scale, g_stride, u_stride, go);
  if (!go) return st;
  const int es = dtype == SS_DTYPE_F32 ? 4 : 2;
  const RowArgs a = {(const char*)gate, (const char*)up, nullptr, q, scale, nullptr, g_stride * es, u_stride * es,
                     (int)cols, 0.f};
  return launch_mode<kSwiglu>(a, rows, dtype, (hipStream_t)stream, who);
}
