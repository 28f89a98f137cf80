// The write of a paged cache of latents, for gfx950: for every new token one row [latent | key],
// shared by all heads, with the rotary embedding of the queries in the same launch.
//
//   c = latent * weight / sqrt(mean(latent^2) + eps)   (or latent as it is, without a weight)
//   rope(x) = x * cos + rotate_half(x) * sin, rotate_half(x) = cat(-x2, x1)
//   cache[slot] = [c | rope(k)],  q_out[h] = rope(q[h])
// Everything is computed in fp32 and rounded once to the tensors' type, so a row is as close to the
// formulas as its type allows (rope_cache.hip instead repeats the rounding of each torch operation).
//
// Work layout: a workgroup a token. Its first wave normalises the latent, all four rotate the heads
// and the key in 16-byte pieces of either half where the strides allow. The piece of the latent
// that a lane holds after the sum (all of a latent of 512 16-bit values) is written from registers.
//
// Bound by the memory at a step's sizes (2240 tokens of 128 heads of 64, latents of 512: 79 MB in 14.6 to 16 us, 4.9 to
// 5.4 TB/s), by the launch at a decode's (256 tokens of 16 heads 3.3 us).
#include "ss_common.h"

namespace {

using ss::u32x4;

struct LatentWriteArgs {
  const char* q;
  char* qo;
  const char* latent;
  const char* k;
  const char* cs;
  const char* sn;
  const char* w;  // or null: the latent is copied
  char* cache;
  const int64_t* slots;
  int64_t q_st, q_sh, o_st, o_sh, l_st, k_st, c_st, s_st;  // bytes: (token, head)
  int64_t c_sb, c_so;                                      // cache (block, position)
  int64_t num_slots;
  int heads, latent_dim, half;  // half the rotated values of a head
  int bs_shift, block_size;
  float eps;
};

template <typename T, int N>
struct Piece {
  float v[N];
  __device__ __forceinline__ void load(const char* p) {
    if constexpr (N == 1) {
      v[0] = (float)*reinterpret_cast<const T*>(p);
    } else {
      const u32x4 w = ss::load16(p);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t u = w[e];
        if constexpr (sizeof(T) == 4) {
          v[e] = __builtin_bit_cast(float, u);
        } else {
          v[2 * e] = ss::Elem<T>::lo(u);
          v[2 * e + 1] = ss::Elem<T>::hi(u);
        }
      }
    }
  }
  __device__ __forceinline__ void store(char* p) const {
    if constexpr (N == 1) {
      *reinterpret_cast<T*>(p) = (T)v[0];
    } else {
      u32x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(T) == 4)
          w[e] = __builtin_bit_cast(uint32_t, v[e]);
        else
          w[e] = ss::Elem<T>::pack2(v[2 * e], v[2 * e + 1]);
      }
      ss::store16(p, w);
    }
  }
};

// Its bits as they are: through fp32 a NaN that signals would be quieted
template <int BYTES>
__device__ __forceinline__ void copy_piece(char* to, const char* from) {
  if constexpr (BYTES == 16)
    ss::store16(to, ss::load16(from));
  else if constexpr (BYTES == 4)
    *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from);
  else
    *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(from);
}

// N values a piece: 16 bytes, or one where the strides or addresses do not allow it
template <typename T, int N>
__global__ __launch_bounds__(256) void latent_write_kernel(const LatentWriteArgs a) {
  typedef Piece<T, N> P;
  constexpr int kBytes = N * (int)sizeof(T);
  const int64_t tok = blockIdx.x;
  const int64_t slot = a.slots[tok];
  const bool kept = slot >= 0 && slot < a.num_slots;
  char* row = nullptr;
  if (kept) {
    const int64_t blk = a.bs_shift >= 0 ? slot >> a.bs_shift : slot / a.block_size;
    row = a.cache + blk * a.c_sb + (slot - blk * a.block_size) * a.c_so;
  }
  const int pieces = a.latent_dim / N;
  if (threadIdx.x < 64 && kept) {
    const char* const src = a.latent + tok * a.l_st;
    const int i0 = threadIdx.x;
    if (!a.w) {
      for (int i = i0; i < pieces; i += 64) copy_piece<kBytes>(row + i * kBytes, src + i * kBytes);
    } else {
      P x, w;
      if (i0 < pieces) {
        x.load(src + i0 * kBytes);
        w.load(a.w + i0 * kBytes);
      }
      float sum = 0.f;
      if (i0 < pieces) {
#pragma unroll
        for (int e = 0; e < N; ++e) sum = fmaf(x.v[e], x.v[e], sum);
      }
      for (int i = i0 + 64; i < pieces; i += 64) {
        P y;
        y.load(src + i * kBytes);
#pragma unroll
        for (int e = 0; e < N; ++e) sum = fmaf(y.v[e], y.v[e], sum);
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
      const float r = 1.f / sqrtf(sum / (float)a.latent_dim + a.eps);
      for (int i = i0; i < pieces; i += 64) {
        if (i != i0) {
          x.load(src + i * kBytes);
          w.load(a.w + i * kBytes);
        }
#pragma unroll
        for (int e = 0; e < N; ++e) x.v[e] = x.v[e] * r * w.v[e];
        x.store(row + i * kBytes);
      }
    }
  }
  // the heads, and behind them the key
  const int per = a.half / N, total = (a.heads + 1) * per;
  const int64_t half_bytes = (int64_t)a.half * (int)sizeof(T);
  for (int i = threadIdx.x; i < total; i += 256) {
    const int h = i / per, at = (i - h * per) * kBytes;
    const char* src = a.q + tok * a.q_st + h * a.q_sh + at;
    char* dst = a.qo + tok * a.o_st + h * a.o_sh + at;
    if (h == a.heads) {
      if (!kept) continue;
      src = a.k + tok * a.k_st + at;
      dst = row + (int64_t)a.latent_dim * (int)sizeof(T) + at;
    }
    const char* const c = a.cs + tok * a.c_st + at;
    const char* const s = a.sn + tok * a.s_st + at;
    P x1, x2, c1, c2, s1, s2;
    x1.load(src), x2.load(src + half_bytes);
    c1.load(c), c2.load(c + half_bytes);
    s1.load(s), s2.load(s + half_bytes);
    P y1, y2;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      y1.v[e] = fmaf(x1.v[e], c1.v[e], -x2.v[e] * s1.v[e]);
      y2.v[e] = fmaf(x2.v[e], c2.v[e], x1.v[e] * s2.v[e]);
    }
    y1.store(dst), y2.store(dst + half_bytes);
  }
}

template <typename T>
int launch_write(const LatentWriteArgs& a, int64_t n_tok, bool wide, hipStream_t stream) {
  const dim3 grid((unsigned)n_tok), block(256);
  if (wide)
    hipLaunchKernelGGL((latent_write_kernel<T, 16 / sizeof(T)>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((latent_write_kernel<T, 1>), grid, block, 0, stream, a);
  return ss_host::launch_status("latent_rope_and_cache");
}

}  // namespace

extern "C" int ss_latent_rope_and_cache(const void* q, void* q_out, const void* latent, const void* k_rope,
                                        const void* cos, const void* sin, const void* weight, void* cache,
                                        const int64_t* slot_mapping, int64_t n_tok, int heads, int latent_dim,
                                        int rope_dim, int block_size, int64_t num_slots, const int64_t q_strides[2],
                                        const int64_t o_strides[2], int64_t latent_stride, int64_t k_stride,
                                        int64_t cos_stride, int64_t sin_stride, const int64_t c_strides[2], float eps,
                                        int dtype, void* stream) {
  const char* who = "latent_rope_and_cache";
  if (n_tok < 0 || heads < 0 || latent_dim < 0 || rope_dim < 0) {
    ss_host::set_error("%s: negative extent", who);
    return SS_ERR_INVALID;
  }
  if (rope_dim % 2 != 0) {
    ss_host::set_error("%s: rope_dim must be even, got %d", who, rope_dim);
    return SS_ERR_INVALID;
  }
  if (block_size < 1) {
    ss_host::set_error("%s: block_size must be >= 1, got %d", who, block_size);
    return SS_ERR_INVALID;
  }
  if (dtype != SS_DTYPE_BF16 && dtype != SS_DTYPE_F16 && dtype != SS_DTYPE_F32) {
    ss_host::set_error("%s: dtype code %d not supported", who, dtype);
    return SS_ERR_UNSUPPORTED;
  }
  if (n_tok == 0 || latent_dim + rope_dim == 0) return SS_OK;
  if (n_tok >= (1 << 24) || heads >= (1 << 20) || latent_dim >= (1 << 20) || rope_dim > (1 << 10)) {
    ss_host::set_error("%s: %lld tokens of %d heads, latent_dim %d, rope_dim %d are more than one launch holds", who,
                       (long long)n_tok, heads, latent_dim, rope_dim);
    return SS_ERR_UNSUPPORTED;
  }
  if (!q_strides || !o_strides || !c_strides || !cache || !slot_mapping || (latent_dim > 0 && !latent) ||
      (rope_dim > 0 && (!k_rope || !cos || !sin)) || (heads > 0 && rope_dim > 0 && (!q || !q_out))) {
    ss_host::set_error("%s: null pointer", who);
    return SS_ERR_INVALID;
  }
  const int es = dtype == SS_DTYPE_F32 ? 4 : 2;
  LatentWriteArgs a;
  a.q = (const char*)q, a.qo = (char*)q_out, a.latent = (const char*)latent, a.k = (const char*)k_rope;
  a.cs = (const char*)cos, a.sn = (const char*)sin, a.w = (const char*)weight, a.cache = (char*)cache;
  a.slots = slot_mapping;
  a.q_st = q_strides[0] * es, a.q_sh = q_strides[1] * es, a.o_st = o_strides[0] * es, a.o_sh = o_strides[1] * es;
  a.l_st = latent_stride * es, a.k_st = k_stride * es, a.c_st = cos_stride * es, a.s_st = sin_stride * es;
  a.c_sb = c_strides[0] * es, a.c_so = c_strides[1] * es;
  a.num_slots = num_slots;
  a.heads = heads, a.latent_dim = latent_dim, a.half = rope_dim / 2;
  a.block_size = block_size;
  a.bs_shift = (block_size & (block_size - 1)) == 0 ? __builtin_ctz((unsigned)block_size) : -1;
  a.eps = eps;
  bool wide = (int64_t)latent_dim * es % 16 == 0 && (int64_t)a.half * es % 16 == 0;
  for (const void* ptr : {q, (const void*)q_out, latent, k_rope, cos, sin, weight, (const void*)cache})
    wide = wide && (uintptr_t)ptr % 16 == 0;
  for (int64_t st : {a.q_st, a.q_sh, a.o_st, a.o_sh, a.l_st, a.k_st, a.c_st, a.s_st, a.c_sb, a.c_so})
    wide = wide && st % 16 == 0;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == SS_DTYPE_BF16) return launch_write<ss::bf16_t>(a, n_tok, wide, s);
  if (dtype == SS_DTYPE_F16) return launch_write<ss::f16_t>(a, n_tok, wide, s);
  return launch_write<float>(a, n_tok, wide, s);
}
