// W8A8 linear for gfx950: out[m, n] = (sum_k x[m, k] w[n, k]) x_scale[m] w_scale[n] (+ bias[n]),
// x and w in int8. The sum is exact in int32 for k < 2^17 (128 * 128 * k < 2^31, refused
// beyond), so a result does not depend on the kernel, the tile or the split that computed
// it: it is rounded in fp32 by the scales and once to the output's type.
#include "w8a8_common.h"

namespace ss {
namespace {

// The kernel for every shape, stride and alignment: 64 x 64 results a workgroup, 64 keys at a
// time through LDS, rows of 80 bytes there so that sixteen lanes' 16-byte reads spread over the
// banks. Sixteen bytes are read at any alignment (global accesses need none on this
// target); a row's last bytes one by one, zeros past its end.
constexpr int kGenTile = 64;
constexpr int kGenRow = 80;

__device__ __forceinline__ i32x4 load_keys(const int8_t* row, int at, int k) {
  i32x4 v = {0, 0, 0, 0};
  if (at + 16 <= k) {
    __builtin_memcpy(&v, row + at, 16);
  } else if (at < k) {
    int8_t b[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) b[e] = at + e < k ? row[at + e] : (int8_t)0;
    __builtin_memcpy(&v, b, 16);
  }
  return v;
}

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
  if (n_tiles * m_tiles > 0x7fffffff) {
    ss_host::set_error("w8a8 gemm: %lld x %lld results are more than one launch holds", (long long)p.m, (long long)p.n);
    return SS_ERR_UNSUPPORTED;
  }
  hipLaunchKernelGGL(w8a8_general_kernel<TO>, dim3((unsigned)(n_tiles * m_tiles)), dim3(256), 0, stream, p, (int)n_tiles);
  return ss_host::launch_status("w8a8 gemm (general)");
}

// Operands that the DMA kernels read in 16-byte pieces: every row starts on one and ends with
// one, and a tile of 256 rows stays below a descriptor's 2^30 bytes.
bool whole_pieces(const W8Params& p) {
  return p.k > 0 && p.k % 16 == 0 && ((uintptr_t)p.x & 15) == 0 && ((uintptr_t)p.w & 15) == 0 &&
         (p.m == 1 || p.x_stride % 16 == 0) && (p.n == 1 || p.w_stride % 16 == 0) && p.x_stride <= (1 << 21) &&
         p.w_stride <= (1 << 21);
}

// Which kernel a call of whole pieces takes, by the kernels' own estimates (fitted to
// measurements, see there): for example 64 x 4096 x 4096 6.4 us streamed and 12.2 in tiles, 64 x
// 28672 x 4096 36.7 and 28.5. Kept for the last shapes of the thread, as a plan is a few
// hundred estimates.
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
    p.stream = stream < tile;
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

extern "C" int ss_w8a8_workspace_size(int64_t m, int64_t n, int64_t k, int out_dtype, int64_t* bytes) {
  if (!bytes) {
    ss_host::set_error("w8a8 workspace: null pointer");
    return SS_ERR_INVALID;
  }
  *bytes = 0;
  const int st = ss::check_extents(m, n, k, out_dtype);
  if (st == SS_OK && m > 0 && n > 0 && k > 0 && k % 16 == 0) *bytes = ss::plan_for(m, n, k, true).workspace();
  return st;
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
  const ss::W8Params p = {x, w, x_scale, w_scale, bias, out, m, n, x_stride, w_stride, o_stride, (int)k, bias_dtype};
  hipStream_t s = (hipStream_t)stream;
  if (ss::whole_pieces(p)) {
    const ss::Plan* pl = &ss::plan_for(m, n, k, true);
    if (pl->workspace() > 0 && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < pl->workspace()))
      pl = &ss::plan_for(m, n, k, false);
    if (pl->stream) return ss::launch_w8a8_stream(p, pl->sp, out_dtype, s);
    if (pl->tp.ks > 0) return ss::launch_w8a8_tile(p, pl->tp, out_dtype, (int*)workspace, s);
  }
  if (out_dtype == SS_DTYPE_BF16) return ss::launch_general<ss::bf16_t>(p, s);
  if (out_dtype == SS_DTYPE_F16) return ss::launch_general<ss::f16_t>(p, s);
  return ss::launch_general<float>(p, s);
}
