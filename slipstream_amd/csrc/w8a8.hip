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
  return ss::check_extents(m, n, k, out_dtype);
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
  (void)workspace;
  (void)workspace_bytes;
  const ss::W8Params p = {x, w, x_scale, w_scale, bias, out, m, n, x_stride, w_stride, o_stride, (int)k, bias_dtype};
  hipStream_t s = (hipStream_t)stream;
  if (out_dtype == SS_DTYPE_BF16) return ss::launch_general<ss::bf16_t>(p, s);
  if (out_dtype == SS_DTYPE_F16) return ss::launch_general<ss::f16_t>(p, s);
  return ss::launch_general<float>(p, s);
}
