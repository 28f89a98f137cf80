// Attention over latents for gfx950, both forms, for every shape and type: the entry points and the
// general kernel.
//
// A token's keys and values of all heads come from one latent c of R values and one rotated key r.
// With W_k and W_v a head's projections, its scores q_n . (W_k c) + q_r . r and outputs sum p W_v c:
//   absorbed: q_n W_k is multiplied out beforehand, so that the cached rows are keys and values
//     themselves, s = (q W_k) . c + q_r . r and o = sum p c, W_v applied to o. 4 R + 2 Dr operations
//     a (query, head, key), but the cache is all that is read: for few new tokens.
//   expanded: kv = [W_k c | W_v c] multiplied out for every token of the context: 2 (Dn + Dr + Dv)
//     operations (a third at R = 512, Dr = 64, Dn = Dv = 128): for chunks of many tokens.
#include "latent_common.h"
#include "w8a8_common.h"

namespace ss {
namespace {

// ---- the general kernel: fp32, any widths up to those below, any page size and strides ----
//
// A workgroup takes eight query rows that share their keys (absorbed: heads of a token; expanded:
// tokens of a head), its four waves the keys in turn, 64 at a time. Scores: lane = key, the query
// rows in LDS. Then o += p v with lane = value dimension, in registers. The waves' maxima, sums and
// outputs are merged at the end, in the order of the waves.
constexpr int kRows = 8;
constexpr int kMostValue = 512, kMostRope = 256, kMostKey = 512;

template <typename T>
__device__ __forceinline__ float dot_row(const T* row, const float* q, int n, float acc) {
  for (int d = 0; d < n; ++d) acc = fmaf((float)row[d], q[d], acc);
  return acc;
}

// NC: value dimensions a lane holds (64 apart)
template <typename T, int NC, bool ABSORBED>
__global__ __launch_bounds__(256) void latent_general_kernel(const LatentParams p, int tiles) {
  extern __shared__ __attribute__((aligned(16))) float s_mem[];
  const int qd = p.key_dim + p.rope_dim;
  float* const s_q = s_mem;                     // [kRows][qd]
  float* const s_p = s_q + kRows * qd;          // [4 waves][64 keys][kRows]
  float* const s_o = s_p + 4 * 64 * kRows;      // [kRows][value_dim]
  float* const s_ml = s_o + kRows * p.value_dim;  // [4][kRows][2]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // rows: absorbed: heads 8 tile .. of token `major`; expanded: tokens 8 tile .. of head `major`
  const int major = blockIdx.x / tiles, first = (blockIdx.x - major * tiles) * kRows;
  const int tokens = p.cu ? p.total : p.batch * p.tq;
  const int have = min(kRows, (ABSORBED ? p.heads : tokens) - first);
  for (int r0 = 0; r0 < have;) {
    // the sequence of row r0, and the rows of it: r0 .. r1 - 1
    const int tok0 = ABSORBED ? major : first + r0;
    int b = 0, count = 0, start = 0;
    if (p.cu) {
      for (; b < p.batch; ++b) {
        latent_queries(p, b, count, start);
        if (tok0 >= start && tok0 < start + count) break;
      }
    } else {
      b = tok0 / p.tq, count = p.tq, start = b * p.tq;
    }
    if (b >= p.batch) {  // of no sequence: left as it is
      ++r0;
      if (ABSORBED) break;
      continue;
    }
    const int r1 = ABSORBED ? have : min(have, start + count - first);
    int k0, length;
    const int keys = latent_keys(p, b, k0, length);
    int lim[kRows];
    int64_t qat[kRows], oat[kRows];
    int most = 0;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int tok = ABSORBED ? major : first + r, h = ABSORBED ? first + r : major;
      const int j = tok - start;
      lim[r] = r >= r0 && r < r1 ? min(keys, length - count + j + 1) : 0;
      most = max(most, lim[r]);
      const int64_t ob = p.cu ? 0 : b, ot = p.cu ? tok : j;
      qat[r] = ob * p.q_sb + ot * p.q_st + h * p.q_sh;
      oat[r] = ob * p.o_sb + ot * p.o_st + h * p.o_sh;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      if (r >= r0 && r < r1)
        for (int d = threadIdx.x; d < qd; d += 256) s_q[r * qd + d] = (float)((const T*)p.q)[qat[r] + d] * p.scale_log2;
    __syncthreads();
    float m[kRows], l[kRows], acc[kRows][NC];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      m[r] = kNegBig, l[r] = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) acc[r][c] = 0.f;
    }
    float* const mine = s_p + wave * 64 * kRows;
    for (int base = 64 * wave; base < most; base += 256) {
      const int i = base + lane;
      int64_t at = -1;  // of the key's row
      if (i < most) {
        if (ABSORBED) {
          const int blk = i / p.block_size, e = p.bt[(int64_t)b * p.bt_stride + blk];
          if (e >= 0 && e < p.num_blocks) at = e * p.kv_s0 + (i - blk * p.block_size) * p.kv_s1;
        } else {
          at = (int64_t)(k0 + i) * p.kv_s0 + major * p.kv_s1;
        }
      }
      const T* const key = (const T*)p.kv + at;
      const T* const rope = ABSORBED ? key + p.key_dim : (const T*)p.k_rope + (int64_t)(k0 + i) * p.k_st;
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        if (r < r0 || r >= r1) continue;
        const bool sees = at >= 0 && i < lim[r];
        float s = -__builtin_inff();
        if (sees) s = dot_row(rope, s_q + r * qd + p.key_dim, p.rope_dim, dot_row(key, s_q + r * qd, p.key_dim, 0.f));
        float top = s;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        const float mn = fmaxf(m[r], top), pr = sees ? fast_exp2(s - mn) : 0.f, alpha = fast_exp2(m[r] - mn);
        float sum = pr;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        l[r] = l[r] * alpha + sum;
        m[r] = mn;
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[r][c] *= alpha;
        mine[lane * kRows + r] = pr;
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      const int n = min(64, most - base);
      for (int t = 0; t < n; ++t) {
        const int64_t from = __shfl(at, t);
        if (from < 0) continue;
        const T* const v = (const T*)p.kv + from + (ABSORBED ? 0 : p.key_dim);
        float pr[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) pr[r] = r >= r0 && r < r1 ? mine[t * kRows + r] : 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int d = 64 * c + lane;
          if (d >= p.value_dim) continue;
          const float x = (float)v[d];
#pragma unroll
          for (int r = 0; r < kRows; ++r)
            if (pr[r] != 0.f) acc[r][c] = fmaf(pr[r], x, acc[r][c]);
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    // the waves one after another
    if (lane == 0) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) s_ml[(wave * kRows + r) * 2] = m[r], s_ml[(wave * kRows + r) * 2 + 1] = l[r];
    }
    __syncthreads();
    float total[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      float top = kNegBig, sum = 0.f;
      for (int w = 0; w < 4; ++w) top = fmaxf(top, s_ml[(w * kRows + r) * 2]);
      for (int w = 0; w < 4; ++w) sum += s_ml[(w * kRows + r) * 2 + 1] * fast_exp2(s_ml[(w * kRows + r) * 2] - top);
      const float mine_part = fast_exp2(m[r] - top);
      total[r] = sum;
#pragma unroll
      for (int c = 0; c < NC; ++c) acc[r][c] *= mine_part;
    }
    for (int w = 0; w < 4; ++w) {
      if (wave == w) {
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            const int d = 64 * c + lane;
            if (d >= p.value_dim || r < r0 || r >= r1) continue;
            float o = acc[r][c] + (w ? s_o[r * p.value_dim + d] : 0.f);
            if (w < 3)
              s_o[r * p.value_dim + d] = o;
            else
              ((T*)p.out)[oat[r] + d] = (T)(total[r] == 0.f ? 0.f : o / total[r]);
          }
      }
      __syncthreads();
    }
    r0 = r1;
  }
}

template <typename T, int NC, bool ABSORBED>
int launch_general_nc(const LatentParams& p, hipStream_t stream) {
  const int64_t tokens = p.cu ? p.total : (int64_t)p.batch * p.tq;
  const int64_t tiles = ((ABSORBED ? p.heads : tokens) + kRows - 1) / kRows, majors = ABSORBED ? tokens : p.heads;
  if (tokens >= INT32_MAX / 2 || tiles * majors >= (1 << 24)) {  // of 256 threads: below 2^32
    ss_host::set_error("latent attention: %lld query tokens of %d heads are more than one launch holds",
                       (long long)tokens, p.heads);
    return SS_ERR_UNSUPPORTED;
  }
  const int lds = 4 * (kRows * (p.key_dim + p.rope_dim) + 4 * 64 * kRows + kRows * p.value_dim + 4 * kRows * 2);
  auto kern = latent_general_kernel<T, NC, ABSORBED>;
  hipLaunchKernelGGL(kern, dim3((unsigned)(tiles * majors)), dim3(256), lds, stream, p, (int)tiles);
  return ss_host::launch_status("latent attention (general)");
}

template <bool ABSORBED>
int launch_general(const LatentParams& p, int dtype, hipStream_t stream) {
  const int nc = p.value_dim <= 128 ? 2 : p.value_dim <= 256 ? 4 : 8;
#define LATENT_GENERAL(T)                                                      \
  return nc == 2   ? launch_general_nc<T, 2, ABSORBED>(p, stream)              \
         : nc == 4 ? launch_general_nc<T, 4, ABSORBED>(p, stream)              \
                   : launch_general_nc<T, 8, ABSORBED>(p, stream)
  if (dtype == SS_DTYPE_BF16) LATENT_GENERAL(bf16_t);
  if (dtype == SS_DTYPE_F16) LATENT_GENERAL(f16_t);
  LATENT_GENERAL(float);
#undef LATENT_GENERAL
}

int check_call(const char* who, int64_t batch, int64_t total, int64_t keys, int heads, int key_dim, int rope_dim,
               int value_dim, int dtype) {
  if (batch < 0 || total < 0 || keys < 0 || heads < 0) {
    ss_host::set_error("%s: negative extent", who);
    return SS_ERR_INVALID;
  }
  if (dtype != SS_DTYPE_BF16 && dtype != SS_DTYPE_F16 && dtype != SS_DTYPE_F32) {
    ss_host::set_error("%s: dtype code %d not supported (bf16, fp16, fp32)", who, dtype);
    return SS_ERR_UNSUPPORTED;
  }
  if (key_dim < 1 || key_dim > kMostKey || rope_dim < 0 || rope_dim > kMostRope || value_dim < 1 ||
      value_dim > kMostValue) {
    ss_host::set_error("%s: widths %d + %d of keys and %d of values not supported (1..%d + 0..%d, 1..%d)", who, key_dim,
                       rope_dim, value_dim, kMostKey, kMostRope, kMostValue);
    return SS_ERR_UNSUPPORTED;
  }
  if (batch > (1 << 20) || heads > (1 << 16) || total > (1 << 28) || keys > (1 << 28)) {
    ss_host::set_error("%s: batch %lld, %d heads, %lld query tokens or %lld keys are more than one launch holds", who,
                       (long long)batch, heads, (long long)total, (long long)keys);
    return SS_ERR_UNSUPPORTED;
  }
  return SS_OK;
}

}  // namespace
}  // namespace ss

extern "C" int ss_latent_attention_workspace_size(int64_t batch, int64_t total_tokens, int tq, int heads,
                                                  int latent_dim, int rope_dim, int dtype, int64_t* bytes) {
  if (!bytes) {
    ss_host::set_error("latent attention workspace: null pointer");
    return SS_ERR_INVALID;
  }
  *bytes = 0;
  const int st = ss::check_call("latent attention workspace", batch, total_tokens, 0, heads, latent_dim, rope_dim,
                                latent_dim, dtype);
  if (st != SS_OK || batch == 0 || heads == 0 || total_tokens == 0) return st;
  if (dtype != SS_DTYPE_F32 && (latent_dim == 256 || latent_dim == 512))
    *bytes = ss::latent_tile_bytes(batch, total_tokens, tq, heads, latent_dim);
  return SS_OK;
}

extern "C" int ss_latent_attention(const void* q, void* out, const void* cache, const int32_t* block_tables,
                                   const int32_t* cu_seqlens, const int32_t* context_lens, int64_t batch,
                                   int64_t total_tokens, int tq, int heads, int latent_dim, int rope_dim,
                                   int max_blocks, int block_size, int64_t num_blocks, const int64_t q_strides[3],
                                   const int64_t o_strides[3], const int64_t c_strides[2], int64_t bt_stride,
                                   float scale, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "latent attention";
  const int st = ss::check_call(who, batch, cu_seqlens ? total_tokens : batch * (int64_t)(tq < 0 ? -1 : tq), 0, heads,
                                latent_dim, rope_dim, latent_dim, dtype);
  if (st != SS_OK) return st;
  if (block_size < 1 || max_blocks < 0 || num_blocks < 0) {
    ss_host::set_error("%s: block_size %d, table width %d or pool of %lld blocks", who, block_size, max_blocks,
                       (long long)num_blocks);
    return SS_ERR_INVALID;
  }
  if (batch == 0 || heads == 0 || (cu_seqlens ? total_tokens == 0 : tq == 0)) return SS_OK;
  if (!q || !out || !context_lens || !q_strides || !o_strides || !c_strides ||
      (max_blocks > 0 && num_blocks > 0 && (!cache || !block_tables))) {
    ss_host::set_error("%s: null pointer", who);
    return SS_ERR_INVALID;
  }
  ss::LatentParams p = {};
  p.q = q, p.out = out, p.kv = cache, p.bt = block_tables, p.ctx_lens = context_lens, p.cu = cu_seqlens;
  p.q_sb = cu_seqlens ? 0 : q_strides[0], p.q_st = q_strides[1], p.q_sh = q_strides[2];
  p.o_sb = cu_seqlens ? 0 : o_strides[0], p.o_st = o_strides[1], p.o_sh = o_strides[2];
  p.kv_s0 = c_strides[0], p.kv_s1 = c_strides[1];
  p.bt_stride = bt_stride, p.num_blocks = num_blocks;
  p.batch = (int)batch, p.heads = heads, p.tq = tq;
  p.key_dim = p.value_dim = latent_dim, p.rope_dim = rope_dim;
  p.max_blocks = num_blocks > 0 ? max_blocks : 0, p.block_size = block_size;
  p.total = (int)total_tokens;
  p.scale_log2 = scale * ss::kLog2e;
  if (ss::latent_tile_takes(p, dtype)) {
    const int64_t need = ss::latent_tile_bytes(batch, p.cu ? total_tokens : batch * tq, tq, heads, latent_dim);
    if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need) {
      ss_host::set_error("%s: workspace of %lld bytes, needs %lld (16-byte aligned)", who,
                         (long long)(workspace ? workspace_bytes : 0), (long long)need);
      return SS_ERR_WORKSPACE;
    }
    return ss::launch_latent_tile(p, dtype, (char*)workspace, (hipStream_t)stream);
  }
  return ss::launch_general<true>(p, dtype, (hipStream_t)stream);
}

extern "C" int ss_latent_attention_expanded(const void* q, void* out, const void* kv, const void* k_rope,
                                            const int32_t* cu_seqlens, const int32_t* cu_context, int64_t batch,
                                            int64_t total_tokens, int64_t total_keys, int max_query_len, int heads,
                                            int nope_dim, int rope_dim, int value_dim, const int64_t q_strides[2],
                                            const int64_t o_strides[2], const int64_t kv_strides[2], int64_t k_stride,
                                            float scale, int dtype, void* stream) {
  const char* who = "latent attention (expanded)";
  const int st = ss::check_call(who, batch, total_tokens, total_keys, heads, nope_dim, rope_dim, value_dim, dtype);
  if (st != SS_OK) return st;
  if (batch == 0 || heads == 0 || total_tokens == 0) return SS_OK;
  if (!q || !out || !cu_seqlens || !cu_context || !q_strides || !o_strides || !kv_strides ||
      (total_keys > 0 && (!kv || (rope_dim > 0 && !k_rope)))) {
    ss_host::set_error("%s: null pointer", who);
    return SS_ERR_INVALID;
  }
  ss::LatentParams p = {};
  p.q = q, p.out = out, p.kv = kv, p.k_rope = k_rope, p.cu = cu_seqlens, p.cu_ctx = cu_context;
  p.q_st = q_strides[0], p.q_sh = q_strides[1], p.o_st = o_strides[0], p.o_sh = o_strides[1];
  p.kv_s0 = kv_strides[0], p.kv_s1 = kv_strides[1], p.k_st = k_stride;
  p.batch = (int)batch, p.heads = heads, p.tq = max_query_len;
  p.key_dim = nope_dim, p.rope_dim = rope_dim, p.value_dim = value_dim;
  p.block_size = 1;
  p.total = (int)total_tokens, p.total_keys = (int)total_keys;
  p.scale_log2 = scale * ss::kLog2e;
  if (ss::latent_expanded_takes(p, dtype)) return ss::launch_latent_expanded(p, dtype, (hipStream_t)stream);
  return ss::launch_general<false>(p, dtype, (hipStream_t)stream);
}
