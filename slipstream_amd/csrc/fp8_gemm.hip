// Linear layer in 8-bit floating point for gfx950: x [m, k] and w [n, k] in e4m3, with an fp32 scale
// for every 128 columns of a row of x and for every 128 x 128 values of w:
//   out[m, n] = sum_b x_scale[m, b] w_scale[n / 128, b] (sum_{k in block b} x[m, k] w[n, k]) (+ bias[n]).
// The matrix cores sum a block (fp8_common.h says in how many bits); its sum is multiplied with the
// product of its scales and added to an fp32 sum in one rounding. A result is rounded once to the
// output's type. Up to 32 tokens go to the stream kernel (fp8_stream.hip), which the weights' bytes bound, up to 128
// to it or the tile kernel (fp8_tile.hip) by whose estimate is the shorter (plan_for), more to the tile kernel; the
// kernel here takes what neither may read.
#include "fp8_common.h"

namespace ss {
namespace {

// The kernel for every shape, stride and alignment, without a workspace: 64 x 64 results a
// workgroup, a block of 128 keys at a time through LDS, rows of 144 bytes there so that sixteen
// lanes' 16-byte reads spread over the banks.
constexpr int kGenTile = 64;
constexpr int kGenRow = 144;

template <typename TO>
__global__ __launch_bounds__(256) void fp8_general_kernel(const F8Params p, int n_tiles) {
  __shared__ __attribute__((aligned(16))) uint8_t s_x[kGenTile * kGenRow];
  __shared__ __attribute__((aligned(16))) uint8_t s_w[kGenTile * kGenRow];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int ln = lane & 15, kg = lane >> 4;
  const int64_t n0 = (int64_t)(blockIdx.x % n_tiles) * kGenTile, m0 = (int64_t)(blockIdx.x / n_tiles) * kGenTile;
  // staging: thread t brings chunks of 16 keys t % 4 and t % 4 + 4 of row t / 4; rows past the end
  // repeat the last one and their results are not stored
  const int sr = threadIdx.x >> 2, sc = 16 * (threadIdx.x & 3);
  const int64_t xm = m0 + sr < p.m ? m0 + sr : p.m - 1, wn = n0 + sr < p.n ? n0 + sr : p.n - 1;
  const uint8_t* const xr = p.x + xm * p.x_stride;
  const uint8_t* const wr = p.w + wn * p.w_stride;
  const int wm = 32 * (wave & 1), wnn = 32 * (wave >> 1);  // this wave's 32 x 32 results
  const float* xs[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t m = m0 + wm + 16 * j + ln;
    xs[j] = p.x_scale + (m < p.m ? m : p.m - 1) * p.xs_row;
  }
  const float* const ws = p.w_scale + (n0 >> 7) * p.ws_row;
  f32x4 acc[2][2] = {};
  for (int k0 = 0; k0 < p.k; k0 += 128) {
    i32x4 xv[2], wv[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      xv[h] = load_keys8(xr, k0 + sc + 64 * h, p.k);
      wv[h] = load_keys8(wr, k0 + sc + 64 * h, p.k);
    }
    const int kb = k0 >> 7;
    const float wsc = ws[kb * p.ws_blk];
    const float sc2[2] = {xs[0][kb * p.xs_blk] * wsc, xs[1][kb * p.xs_blk] * wsc};
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      *reinterpret_cast<i32x4*>(s_x + sr * kGenRow + sc + 64 * h) = xv[h];
      *reinterpret_cast<i32x4*>(s_w + sr * kGenRow + sc + 64 * h) = wv[h];
    }
    __syncthreads();
    typename Block<TO>::Operand a[2], b[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint8_t* const ar = s_w + (wnn + 16 * t + ln) * kGenRow + 32 * kg;
      const uint8_t* const br = s_x + (wm + 16 * t + ln) * kGenRow + 32 * kg;
      a[t] = Block<TO>::operand(join8(*reinterpret_cast<const i32x4*>(ar), *reinterpret_cast<const i32x4*>(ar + 16)));
      b[t] = Block<TO>::operand(join8(*reinterpret_cast<const i32x4*>(br), *reinterpret_cast<const i32x4*>(br + 16)));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const f32x4 part = Block<TO>::sum(a[i], b[j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(part[e], sc2[j], acc[i][j][e]);
      }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t m = m0 + wm + 16 * j + ln;
    if (m >= p.m) continue;
    TO* const o = (TO*)p.out + m * p.o_stride;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t n = n0 + wnn + 16 * i + 4 * kg + e;
        if (n < p.n) o[n] = (TO)(acc[i][j][e] + (p.bias ? load_as_f32(p.bias, n, p.bias_dtype) : 0.f));
      }
  }
}

template <typename TO>
int launch_general(const F8Params& p, hipStream_t stream) {
  const int64_t n_tiles = (p.n + kGenTile - 1) / kGenTile, m_tiles = (p.m + kGenTile - 1) / kGenTile;
  if (n_tiles * m_tiles >= (1 << 24)) {  // of 256 threads: below 2^32
    ss_host::set_error("fp8 gemm: %lld x %lld results are more than one launch holds", (long long)p.m, (long long)p.n);
    return SS_ERR_UNSUPPORTED;
  }
  hipLaunchKernelGGL(fp8_general_kernel<TO>, dim3((unsigned)(n_tiles * m_tiles)), dim3(256), 0, stream, p, (int)n_tiles);
  return ss_host::launch_status("fp8 gemm (general)");
}

bool known_dtype(int d) { return d == SS_DTYPE_BF16 || d == SS_DTYPE_F16 || d == SS_DTYPE_F32; }

int check_extents(int64_t m, int64_t n, int64_t k, int out_dtype) {
  if (m < 0 || n < 0 || k < 0) {
    ss_host::set_error("fp8 gemm: negative extent");
    return SS_ERR_INVALID;
  }
  if (k >= ((int64_t)1 << 30)) {
    ss_host::set_error("fp8 gemm: k = %lld not supported (below 2^30)", (long long)k);
    return SS_ERR_UNSUPPORTED;
  }
  if (!known_dtype(out_dtype)) {
    ss_host::set_error("fp8 gemm: output dtype code %d not supported", out_dtype);
    return SS_ERR_UNSUPPORTED;
  }
  return SS_OK;
}

// Rows that the DMA kernels can read in 16-byte pieces; a tile of 256 of them stays below a descriptor's 2^30
// bytes.
constexpr int64_t kMostStride = 1 << 21;
bool whole_rows(const void* base, int64_t rows, int64_t stride, int64_t k) {
  return k % 16 == 0 && ((uintptr_t)base & 15) == 0 && (rows == 1 || stride % 16 == 0) && stride <= kMostStride;
}
int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

// What a call runs on the current device. Kept for the last shapes of the thread.
//
// Over 288 calls of 1 to 2240 tokens with weights of 1152 x 896 to 28672 x 4096, to bf16 and fp16, the plan is within
// 2.5 % of the best kernel, tile, split and waves on average (3.6 % up to 128 tokens, 1.1 % above) and 49 % off at worst
// (128 x 14336 x 512 to fp16: 11.8 us in the stream kernel, 7.8 in the tile kernel). Up to 32 tokens the tile kernel takes
// 1.6 times the stream kernel's time there and is never the faster, so the estimates are not asked: they agree, but
// for outputs of 131072 and more, where they err to either side (16 x 524288 x 512 85 us by the estimates, 68 so; 8 x
// 131072 x 128 12.4 and 14.6), and for rows of 65536 and more, which would be faster so (32 x 2048 x 65536 37.6 and 43.8).
struct Plan {
  int64_t m = -1, n = 0, k = 0;
  bool wide = false, may_split = false;
  int device = -1;
  bool stream = false;
  F8StreamPlan sp = {};
  F8TilePlan tp = {};
  int64_t workspace() const { return !stream && tp.ks > 1 ? (int64_t)tp.ks * m * n * 4 : 0; }
};
const Plan& plan_for(int64_t m, int64_t n, int64_t k, bool wide, bool may_split) {
  static thread_local Plan kept[64];
  int device = 0;
  if (hipGetDevice(&device) != hipSuccess) device = 0;
  const uint64_t h = ((uint64_t)m * 0x9E3779B97F4A7C15ull) ^ ((uint64_t)n * 0xC2B2AE3D27D4EB4Full) ^
                     ((uint64_t)k * 0x165667B19E3779F9ull) ^ (may_split ? 0 : ~0ull) ^ (wide ? 0xFFFFull << 40 : 0);
  Plan& p = kept[h >> 58];
  if (p.m != m || p.n != n || p.k != k || p.wide != wide || p.may_split != may_split || p.device != device) {
    p.m = m, p.n = n, p.k = k, p.wide = wide, p.may_split = may_split, p.device = device;
    const double stream = plan_fp8_stream(p.sp, m, n, k), tile = plan_fp8_tile(p.tp, m, n, k, wide, may_split);
    p.stream = stream < 1e29 && (m <= 32 || stream < tile);
  }
  return p;
}

}  // namespace
}  // namespace ss

extern "C" int ss_fp8_workspace_size(int64_t m, int64_t n, int64_t k, int x_whole, int w_whole, int out_dtype,
                                     int64_t* bytes) {
  if (!bytes) {
    ss_host::set_error("fp8 workspace: null pointer");
    return SS_ERR_INVALID;
  }
  *bytes = 0;
  const int st = ss::check_extents(m, n, k, out_dtype);
  if (st != SS_OK || m == 0 || n == 0 || k == 0) return st;
  const int64_t kp = ss::round16(k);
  if (kp > ss::kMostStride || m > INT32_MAX || n > INT32_MAX) return SS_OK;  // the general kernel's, without copies
  *bytes = ss::plan_for(m, n, kp, out_dtype != SS_DTYPE_BF16, true).workspace() + (x_whole && kp == k ? 0 : m * kp) +
           (w_whole && kp == k ? 0 : n * kp);
  return SS_OK;
}

extern "C" int ss_fp8_gemm(const uint8_t* x, const float* x_scale, const uint8_t* w, const float* w_scale,
                           const void* bias, void* out, int64_t m, int64_t n, int64_t k, int64_t x_stride,
                           int64_t w_stride, int64_t o_stride, const int64_t xs_strides[2], const int64_t ws_strides[2],
                           int out_dtype, int bias_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  const int st = ss::check_extents(m, n, k, out_dtype);
  if (st != SS_OK) return st;
  if (m == 0 || n == 0) return SS_OK;
  if (!out || !xs_strides || !ws_strides || (k > 0 && (!x || !w || !x_scale || !w_scale))) {
    ss_host::set_error("fp8 gemm: null pointer");
    return SS_ERR_INVALID;
  }
  if (bias && !ss::known_dtype(bias_dtype)) {
    ss_host::set_error("fp8 gemm: bias dtype code %d not supported", bias_dtype);
    return SS_ERR_UNSUPPORTED;
  }
  if ((m > 1 && (x_stride < k || o_stride < n)) || (n > 1 && w_stride < k)) {
    ss_host::set_error("fp8 gemm: row strides shorter than the rows");
    return SS_ERR_INVALID;
  }
  ss::F8Params p = {x,        w,        x_scale,       w_scale,       bias,          out,           m,      n,
                          x_stride, w_stride, o_stride,      xs_strides[0], xs_strides[1], ws_strides[0], ws_strides[1],
                          (int)k,   bias_dtype};
  if (m == 1) p.x_stride = ss::round16(k), p.o_stride = ss::round16(n), p.xs_row = 1;  // (not used to reach a row)
  if (n == 1) p.w_stride = ss::round16(k);
  if (n <= 128) p.ws_row = 1;
  hipStream_t s = (hipStream_t)stream;
  char* ws = (uintptr_t)workspace & 15 ? nullptr : (char*)workspace;
  int64_t left = ws ? workspace_bytes : 0;
  // rows that are not whole 16-byte pieces: their copies come first in the workspace
  const int64_t kp = ss::round16(k), blocks = (k + 127) / 128;
  const bool copy_x = !ss::whole_rows(p.x, m, p.x_stride, k), copy_w = !ss::whole_rows(p.w, n, p.w_stride, k);
  const int64_t x_bytes = copy_x ? m * kp : 0, w_bytes = copy_w ? n * kp : 0;
  // a tile's scales within a descriptor's reach
  const int64_t reach = (int64_t)1 << 27;
  const bool scales = p.xs_row >= 0 && p.xs_blk >= 0 && p.ws_row >= 0 && p.ws_blk >= 0 &&
                      256 * p.xs_row + blocks * p.xs_blk < reach && 2 * p.ws_row + blocks * p.ws_blk < reach;
  // (copies of longer rows would not lie within a descriptor's reach either)
  if (k > 0 && kp <= ss::kMostStride && scales && x_bytes + w_bytes <= left && m <= INT32_MAX && n <= INT32_MAX) {
    const bool wide = out_dtype != SS_DTYPE_BF16;
    const ss::Plan* pl = &ss::plan_for(m, n, kp, wide, true);
    if (pl->workspace() > left - x_bytes - w_bytes) pl = &ss::plan_for(m, n, kp, wide, false);
    if (pl->stream || pl->tp.ks > 0) {
      if (copy_x || copy_w) {
        const ss::ByteRows rx = {(const int8_t*)p.x, (int8_t*)ws, p.x_stride, copy_x ? (int)m : 0};
        const ss::ByteRows rw = {(const int8_t*)p.w, (int8_t*)ws + x_bytes, p.w_stride, copy_w ? (int)n : 0};
        if (const int sa = ss::align_rows(rx, rw, (int)k, s); sa != SS_OK) return sa;
        if (copy_x) p.x = (const uint8_t*)rx.to, p.x_stride = kp;
        if (copy_w) p.w = (const uint8_t*)rw.to, p.w_stride = kp;
        p.k = (int)kp;
      }
      if (pl->stream) return ss::launch_fp8_stream(p, pl->sp, out_dtype, s);
      return ss::launch_fp8_tile(p, pl->tp, out_dtype, (float*)(ws + x_bytes + w_bytes), s);
    }
  }
  if (out_dtype == SS_DTYPE_BF16) return ss::launch_general<ss::bf16_t>(p, s);
  if (out_dtype == SS_DTYPE_F16) return ss::launch_general<ss::f16_t>(p, s);
  return ss::launch_general<float>(p, s);
}
