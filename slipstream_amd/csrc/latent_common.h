// Parameters shared by the kernels of attention over latents.
#pragma once

#include "ss_common.h"

namespace ss {

// A call of either form. A sequence b owns query tokens [start(b), start(b) + count(b)) and has
// ctx(b) keys; query j of them sees the keys [0, ctx - count + j].
//   absorbed: key i is the cache row [latent | rope] behind block_tables, its value the latent;
//     the heads of a token share it, and the query rows of a sequence are r = j * heads + h.
//   expanded: key i of head h is [kv(i, h)[:nope] | k_rope(i)], its value kv(i, h)[nope:], where i
//     counts from cu_ctx[b]; the query rows of a sequence and head are r = j.
struct LatentParams {
  const void* q;
  void* out;
  const void* kv;           // absorbed: the layer's pages
  const void* k_rope;       // expanded
  const int32_t* bt;        // absorbed
  const int32_t* ctx_lens;  // absorbed [batch]
  const int32_t* cu;        // [batch + 1], or null: tq query tokens each
  const int32_t* cu_ctx;    // expanded [batch + 1]
  int64_t q_sb, q_st, q_sh, o_sb, o_st, o_sh;  // elements; packed: q_sb = o_sb = 0
  int64_t kv_s0, kv_s1;  // absorbed: (block, position); expanded: (token, head)
  int64_t k_st;          // expanded: k_rope's token
  int64_t bt_stride, num_blocks;
  int batch, heads, tq;
  int key_dim, rope_dim, value_dim;  // absorbed: key_dim = value_dim = latent
  int max_blocks, block_size;
  int total, total_keys;  // packed: query tokens, and the expanded form's keys; cu's entries are clamped to them
  float scale_log2;       // softmax scale * log2(e)
};

typedef const __attribute__((address_space(4))) int32_t* ConstInts;

__device__ __forceinline__ void latent_queries(const LatentParams& p, int b, int& count, int& start) {
  if (p.cu) {
    const ConstInts cu = (ConstInts)p.cu;
    const int s = min(max(cu[b], 0), p.total), e = min(max(cu[b + 1], s), p.total);
    count = e - s, start = s;
  } else {
    count = p.tq, start = 0;
  }
}

// Keys of sequence b (those that the table reaches), the first one's row in the expanded form
// and by how many its length exceeds the keys
__device__ __forceinline__ int latent_keys(const LatentParams& p, int b, int& first, int& length) {
  first = 0;
  if (p.cu_ctx) {
    const ConstInts cu = (ConstInts)p.cu_ctx;
    const int s = min(max(cu[b], 0), p.total_keys), e = min(max(cu[b + 1], s), p.total_keys);
    first = s;
    length = e - s;
    return length;
  }
  length = max(((ConstInts)p.ctx_lens)[b], 0);
  return (int)min((int64_t)length, (int64_t)p.max_blocks * p.block_size);
}

// latent_tile.hip: whether the matrix-core kernels take a call of the absorbed form, the workspace they
// need for it, and the call
bool latent_tile_takes(const LatentParams& p, int dtype);
int64_t latent_tile_bytes(int64_t batch, int64_t total, int tq, int heads, int latent_dim);
int launch_latent_tile(const LatentParams& p, int dtype, char* ws, hipStream_t stream);

// latent_expanded.hip: the same of the expanded form (which needs no workspace)
bool latent_expanded_takes(const LatentParams& p, int dtype);
int launch_latent_expanded(const LatentParams& p, int dtype, hipStream_t stream);

}  // namespace ss
