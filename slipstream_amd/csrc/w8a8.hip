// W8A8 linear for gfx950: out[m, n] = (sum_k x[m, k] w[n, k]) x_scale[m] w_scale[n] (+ bias[n]),
// x and w in int8. The sum is exact in int32 for k < 2^17 (128 * 128 * k < 2^31, refused
// beyond), so a result does not depend on the kernel, the tile or the split that computed
// it: it is rounded in fp32 by the scales and once to the output's type.
#include <utility>

#include "w8a8_common.h"

namespace ss {
namespace {

// Sixteen keys of a row at any alignment (global accesses need none on this target), past the
// row's end zeros. A row's last, partial piece is put together from the aligned words that hold
// its keys, read at the last one where they lie behind it: sixteen loads of a byte, each under
// its own condition, wait for one another (the copies of 2000 rows of 1000: 6.5 us, so 4.0).
__device__ __forceinline__ i32x4 load_keys(const int8_t* row, int at, int k) {
  i32x4 v = {0, 0, 0, 0};
  if (at + 16 <= k) {
    __builtin_memcpy(&v, row + at, 16);
  } else if (at < k) {
    const uint64_t from = (uint64_t)(row + at), last = (uint64_t)(row + k - 1) & ~3ull;
    uint32_t w[5];
#pragma unroll
    for (int e = 0; e < 5; ++e) {
      const uint64_t word = (from & ~3ull) + 4 * e;
      w[e] = *reinterpret_cast<const uint32_t*>(word < last ? word : last);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int keys = k - at - 4 * e;  // that are left for this word
      const uint32_t mask = keys >= 4 ? ~0u : keys > 0 ? (1u << (8 * keys)) - 1u : 0u;
      v[e] = (int)(__builtin_amdgcn_alignbyte(w[e + 1], w[e], (uint32_t)from & 3u) & mask);
    }
  }
  return v;
}

// The other kernels' operands begin every row on 16 bytes and end it with 16. Rows that do not
// are copied to rows that do, zeros behind them, in the workspace: 333 x 4999 x 2051 (rows at any
// byte; bf16, no bias) 30.4 us in the general kernel, 20.8 so, of which 8 for the copies.
// Two pieces a thread, both on their way before the first is written.
struct Rows {
  const int8_t* from;
  int8_t* to;
  int64_t stride;  // of `from`
  int rows;
};
__global__ __launch_bounds__(256) void w8a8_align_kernel(Rows x, Rows w, int k, uint32_t pieces) {
  const uint32_t total = (uint32_t)(x.rows + w.rows) * pieces, half = (total + 1) >> 1;
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= half) return;
  i32x4 v[2];
  int8_t* to[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const uint32_t j = i + u * half;
    to[u] = nullptr;
    if (j >= total) continue;
    const uint32_t r = j / pieces, c = 16 * (j - r * pieces);
    const bool of_x = r < (uint32_t)x.rows;
    const int64_t row = of_x ? r : r - x.rows;
    to[u] = (of_x ? x.to : w.to) + row * (16 * (int64_t)pieces) + c;
    v[u] = load_keys((of_x ? x.from : w.from) + row * (of_x ? x.stride : w.stride), (int)c, k);
  }
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (to[u]) *reinterpret_cast<i32x4*>(to[u]) = v[u];
}

// The copies of both operands (0 rows: none), as many rows a launch as its 32-bit piece numbers hold
int align_rows(Rows x, Rows w, int k, hipStream_t stream) {
  const int pieces = (k + 15) / 16;
  const int most = (1 << 30) / pieces;
  for (int64_t left = (int64_t)x.rows + w.rows; left > 0;) {
    const Rows px = {x.from, x.to, x.stride, x.rows < most ? x.rows : most};
    const Rows pw = {w.from, w.to, w.stride, w.rows < most - px.rows ? w.rows : most - px.rows};
    const int64_t half = ((int64_t)(px.rows + pw.rows) * pieces + 1) / 2;
    hipLaunchKernelGGL(w8a8_align_kernel, dim3((unsigned)((half + 255) / 256)), dim3(256), 0, stream, px, pw, k,
                       (uint32_t)pieces);
    const int st = ss_host::launch_status("w8a8 gemm (align)");
    if (st != SS_OK) return st;
    for (auto [all, part] : {std::pair<Rows*, const Rows*>{&x, &px}, {&w, &pw}}) {
      all->from += part->rows * all->stride;
      all->to += part->rows * (16 * (int64_t)pieces);
      all->rows -= part->rows;
    }
    left -= px.rows + pw.rows;
  }
  return SS_OK;
}

// The kernel for every shape, stride and alignment, without a workspace: 64 x 64 results a
// workgroup, 64 keys at a time through LDS, rows of 80 bytes there so that sixteen lanes'
// 16-byte reads spread over the banks.
constexpr int kGenTile = 64;
constexpr int kGenRow = 80;

template <typename TO>
__global__ __launch_bounds__(256) void w8a8_general_kernel(const W8Params p, int n_tiles) {
  __shared__ __attribute__((aligned(16))) int8_t s_x[kGenTile * kGenRow];
  __shared__ __attribute__((aligned(16))) int8_t s_w[kGenTile * kGenRow];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int ln = lane & 15, kg = lane >> 4;
  const int64_t n0 = (int64_t)(blockIdx.x % n_tiles) * kGenTile, m0 = (int64_t)(blockIdx.x / n_tiles) * kGenTile;
  // staging: thread t brings 16 keys of row t / 4; rows past the end repeat the last one and
  // their results are not stored
  const int sr = threadIdx.x >> 2, sc = 16 * (threadIdx.x & 3);
  const int64_t xm = m0 + sr < p.m ? m0 + sr : p.m - 1, wn = n0 + sr < p.n ? n0 + sr : p.n - 1;
  const int8_t* const xr = p.x + xm * p.x_stride;
  const int8_t* const wr = p.w + wn * p.w_stride;
  const int wm = 32 * (wave & 1), wnn = 32 * (wave >> 1);  // this wave's 32 x 32 results
  i32x4 acc[2][2] = {};
  for (int k0 = 0; k0 < p.k; k0 += 64) {
    const i32x4 xv = load_keys(xr, k0 + sc, p.k), wv = load_keys(wr, k0 + sc, p.k);
    __syncthreads();
    *reinterpret_cast<i32x4*>(s_x + sr * kGenRow + sc) = xv;
    *reinterpret_cast<i32x4*>(s_w + sr * kGenRow + sc) = wv;
    __syncthreads();
    i32x4 a[2], b[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      a[t] = *reinterpret_cast<const i32x4*>(s_w + (wnn + 16 * t + ln) * kGenRow + 16 * kg);
      b[t] = *reinterpret_cast<const i32x4*>(s_x + (wm + 16 * t + ln) * kGenRow + 16 * kg);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = mfma_i8(a[i], b[j], acc[i][j]);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t m = m0 + wm + 16 * j + ln;
    if (m >= p.m) continue;
    const float xs = p.x_scale[m];
    TO* const o = (TO*)p.out + m * p.o_stride;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t n = n0 + wnn + 16 * i + 4 * kg + e;
        if (n < p.n) o[n] = (TO)scaled(acc[i][j][e], xs, p.w_scale[n], p.bias ? load_as_f32(p.bias, n, p.bias_dtype) : 0.f);
      }
  }
}

template <typename TO>
int launch_general(const W8Params& p, hipStream_t stream) {
  const int64_t n_tiles = (p.n + kGenTile - 1) / kGenTile, m_tiles = (p.m + kGenTile - 1) / kGenTile;
  if (n_tiles * m_tiles >= (1 << 24)) {  // of 256 threads: below 2^32
    ss_host::set_error("w8a8 gemm: %lld x %lld results are more than one launch holds", (long long)p.m, (long long)p.n);
    return SS_ERR_UNSUPPORTED;
  }
  hipLaunchKernelGGL(w8a8_general_kernel<TO>, dim3((unsigned)(n_tiles * m_tiles)), dim3(256), 0, stream, p, (int)n_tiles);
  return ss_host::launch_status("w8a8 gemm (general)");
}

// Rows that the DMA kernels can read in 16-byte pieces; a tile of 256 of them stays below a
// descriptor's 2^30 bytes.
bool whole_rows(const void* base, int64_t rows, int64_t stride, int64_t k) {
  return k % 16 == 0 && ((uintptr_t)base & 15) == 0 && (rows == 1 || stride % 16 == 0) && stride <= (1 << 21);
}
int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

// Which kernel a call takes: up to 32 tokens the stream kernel, which is the faster one there (at m =
// 32 28672 x 4096 22.9 us, in tiles 24.1; 4096 x 14336 12.1 and 14.9; 57344 x 8192 86 and 91),
// beyond that by the kernels' own estimates, fitted to measurements (at m = 64 4096 x 4096 6.3 us
// streamed and 10.8 in tiles, 28672 x 4096 31.2 and 25.0, 4096 x 14336 14.1 and 16.0; wrong where
// they are close: m = 48 4096 x 14336 goes in tiles, 15.9 us, streamed 13.4). Kept for the last
// shapes of the thread, as a plan is a few hundred estimates.
struct Plan {
  int64_t m = -1, n = 0, k = 0;
  bool may_split = false, stream = false;
  int device = -1;
  StreamPlan sp = {};
  TilePlan tp = {};
  int64_t workspace() const { return !stream && tp.ks > 1 ? (int64_t)tp.ks * m * n * 4 : 0; }
};
const Plan& plan_for(int64_t m, int64_t n, int64_t k, bool may_split) {
  static thread_local Plan kept[64];
  int device = 0;
  if (hipGetDevice(&device) != hipSuccess) device = 0;
  const uint64_t h = ((uint64_t)m * 0x9E3779B97F4A7C15ull) ^ ((uint64_t)n * 0xC2B2AE3D27D4EB4Full) ^
                     ((uint64_t)k * 0x165667B19E3779F9ull) ^ (may_split ? 0 : ~0ull);
  Plan& p = kept[h >> 58];
  if (p.m != m || p.n != n || p.k != k || p.may_split != may_split || p.device != device) {
    p.m = m, p.n = n, p.k = k, p.may_split = may_split, p.device = device;
    const double stream = plan_w8a8_stream(p.sp, m, n, k), tile = plan_w8a8_tile(p.tp, m, n, k, may_split);
    p.stream = stream < 1e29 && (m <= 32 || stream < tile);
    if (stream > 1e29 && tile > 1e29) p.tp.ks = 0;  // more results than one launch holds
  }
  return p;
}

bool known_dtype(int d) { return d == SS_DTYPE_BF16 || d == SS_DTYPE_F16 || d == SS_DTYPE_F32; }

int check_extents(int64_t m, int64_t n, int64_t k, int out_dtype) {
  if (m < 0 || n < 0 || k < 0) {
    ss_host::set_error("w8a8 gemm: negative extent");
    return SS_ERR_INVALID;
  }
  if (k >= (1 << 17)) {
    ss_host::set_error("w8a8 gemm: k = %lld: the int32 sum holds fewer than 131072 products", (long long)k);
    return SS_ERR_UNSUPPORTED;
  }
  if (!known_dtype(out_dtype)) {
    ss_host::set_error("w8a8 gemm: output dtype code %d not supported", out_dtype);
    return SS_ERR_UNSUPPORTED;
  }
  return SS_OK;
}

}  // namespace
}  // namespace ss

extern "C" int ss_w8a8_workspace_size(int64_t m, int64_t n, int64_t k, int x_whole, int w_whole, int64_t* bytes) {
  if (!bytes) {
    ss_host::set_error("w8a8 workspace: null pointer");
    return SS_ERR_INVALID;
  }
  *bytes = 0;
  const int st = ss::check_extents(m, n, k, SS_DTYPE_BF16);
  if (st != SS_OK || m == 0 || n == 0 || k == 0) return st;
  const int64_t kp = ss::round16(k);
  *bytes = ss::plan_for(m, n, kp, true).workspace() + (x_whole && kp == k ? 0 : m * kp) + (w_whole && kp == k ? 0 : n * kp);
  return st;
}

extern "C" int ss_w8a8_plan(int64_t m, int64_t n, int64_t k, int32_t* plan) {
  if (!plan) {
    ss_host::set_error("w8a8 plan: null pointer");
    return SS_ERR_INVALID;
  }
  for (int i = 0; i < 5; ++i) plan[i] = 0;
  const int st = ss::check_extents(m, n, k, SS_DTYPE_BF16);
  if (st != SS_OK || m == 0 || n == 0) return st;
  if (k == 0 || m > INT32_MAX || n > INT32_MAX) return SS_OK;
  const ss::Plan& p = ss::plan_for(m, n, ss::round16(k), true);
  if (p.stream) {
    const int32_t is[5] = {1, 16 * p.sp.mt, 16 * p.sp.nt, p.sp.waves, p.sp.once};
    for (int i = 0; i < 5; ++i) plan[i] = is[i];
  } else if (p.tp.ks > 0) {
    const int32_t is[5] = {2, p.tp.bm, p.tp.bn, p.tp.ks, p.tp.once};
    for (int i = 0; i < 5; ++i) plan[i] = is[i];
  }
  return SS_OK;
}

extern "C" int ss_w8a8_gemm(const int8_t* x, const float* x_scale, const int8_t* w, const float* w_scale,
                            const void* bias, void* out, int64_t m, int64_t n, int64_t k, int64_t x_stride,
                            int64_t w_stride, int64_t o_stride, int out_dtype, int bias_dtype, void* workspace,
                            int64_t workspace_bytes, void* stream) {
  const int st = ss::check_extents(m, n, k, out_dtype);
  if (st != SS_OK) return st;
  if (m == 0 || n == 0) return SS_OK;
  if (!x_scale || !w_scale || !out || (k > 0 && (!x || !w))) {
    ss_host::set_error("w8a8 gemm: null pointer");
    return SS_ERR_INVALID;
  }
  if (bias && !ss::known_dtype(bias_dtype)) {
    ss_host::set_error("w8a8 gemm: bias dtype code %d not supported", bias_dtype);
    return SS_ERR_UNSUPPORTED;
  }
  if ((m > 1 && (x_stride < k || o_stride < n)) || (n > 1 && w_stride < k)) {
    ss_host::set_error("w8a8 gemm: row strides shorter than the rows");
    return SS_ERR_INVALID;
  }
  ss::W8Params p = {x, w, x_scale, w_scale, bias, out, m, n, x_stride, w_stride, o_stride, (int)k, bias_dtype};
  if (m == 1) p.x_stride = ss::round16(k), p.o_stride = ss::round16(n);  // (not used to reach a row)
  if (n == 1) p.w_stride = ss::round16(k);
  hipStream_t s = (hipStream_t)stream;
  char* ws = (uintptr_t)workspace & 15 ? nullptr : (char*)workspace;
  int64_t left = ws ? workspace_bytes : 0;
  // rows that are not whole 16-byte pieces: their copies come first in the workspace
  const int64_t kp = ss::round16(k);
  const bool copy_x = !ss::whole_rows(p.x, m, p.x_stride, k), copy_w = !ss::whole_rows(p.w, n, p.w_stride, k);
  const int64_t x_bytes = copy_x ? m * kp : 0, w_bytes = copy_w ? n * kp : 0;
  if (k > 0 && x_bytes + w_bytes <= left && m <= INT32_MAX && n <= INT32_MAX) {
    if (copy_x || copy_w) {
      const ss::Rows rx = {p.x, (int8_t*)ws, p.x_stride, copy_x ? (int)m : 0};
      const ss::Rows rw = {p.w, (int8_t*)ws + x_bytes, p.w_stride, copy_w ? (int)n : 0};
      const int sa = ss::align_rows(rx, rw, (int)k, s);
      if (sa != SS_OK) return sa;
      if (copy_x) p.x = rx.to, p.x_stride = kp;
      if (copy_w) p.w = rw.to, p.w_stride = kp;
      p.k = (int)kp;
      ws += x_bytes + w_bytes;
      left -= x_bytes + w_bytes;
    }
    const ss::Plan* pl = &ss::plan_for(m, n, kp, true);
    if (pl->workspace() > left) pl = &ss::plan_for(m, n, kp, false);
    if (pl->stream) return ss::launch_w8a8_stream(p, pl->sp, out_dtype, s);
    if (pl->tp.ks > 0) return ss::launch_w8a8_tile(p, pl->tp, out_dtype, (int*)ws, s);
  }
  if (out_dtype == SS_DTYPE_BF16) return ss::launch_general<ss::bf16_t>(p, s);
  if (out_dtype == SS_DTYPE_F16) return ss::launch_general<ss::f16_t>(p, s);
  return ss::launch_general<float>(p, s);
}
