// W8A8 stream kernel: the int8 product for few tokens, where the weights' bytes set the time.
//
// A workgroup of up to eight waves multiplies 16 MT tokens with 16 NT channels; its waves share
// out the keys, 128 at a time in turn. A wave brings its 128 keys of every row by DMA into a
// part of the LDS that is its own, two blocks in turn, and reads the matrix
// instruction's operands from there: no wave waits for another before the end, where the
// integer sums are added in the LDS, in any order the same result. (Loaded straight into the
// operands' registers, sixteen lanes in a row touch sixteen cache lines, and the address
// unit, not the memory, sets the time: 16 x 4096 x 14336 15.0 us.)
#include "w8a8_common.h"

namespace ss {
namespace {

constexpr int kLdsBytes = 160 * 1024;
constexpr int kFar = 0x40000000;  // a byte offset past any operand tile (host-checked)
constexpr int kPlane = 68;        // LDS words of the 64 lanes' sums of one accumulator register

// 16-byte chunk c of row r of a 16-row tile lies at chunk c ^ swizzle of its 128 LDS bytes. A
// 16-byte LDS read takes lanes 0-3, 12-15, 20-27 first, then 4-11, 16-19, 28-31, and the same
// of the upper half: rows 0-3 and 12-15 of one key group and rows 4-11 of the next, whose
// chunk differs by 2. Rows 2p and 2p + 1 lie in different halves of the banks; this value
// keeps the row pairs of a pass apart.
__device__ __forceinline__ int stream_swizzle(int r) {
  const int p = r >> 1;
  return (((p >> 2) ^ (p >> 1)) & 1) << 2 | ((p >> 2) & 1) << 1 | (p & 1);
}

// a wave's blocks on their way, or in work
constexpr int D = 2;
// bytes of a block (128 keys of the weights' and tokens' rows), and of a workgroup's LDS
constexpr int block_bytes(int mt, int nt) { return (16 * nt + 16 * mt) * 128; }
constexpr int stream_lds_bytes(int mt, int nt, int waves) {
  return waves * D * block_bytes(mt, nt) + mt * nt * 4 * kPlane * 4 + 16 * mt * 4;
}

// Whether the weights pass the caches by, as what is read once does: where no second token block
// reads them, for 16 tokens at any size (4096 x 14336 from memory 12.7 -> 11.4 us, out of the
// 256 MB cache 10.2 and 10.0), beyond that above kKeptWeights.
inline bool read_once(int mt, int64_t m_blocks, int64_t n, int64_t k) {
  return m_blocks == 1 && (mt == 1 || n * k > kKeptWeights);
}

// XI: groups of eight tokens that are read (2 MT, or 1 of MT = 1); the rows of the others hold
// anything, and their sums are not stored.
template <typename TO, int MT, int NT, int XI>
__global__ __launch_bounds__(512) void w8a8_stream_kernel(const W8Params p, int n_tiles, int m_blocks, bool once) {
  constexpr int B = block_bytes(MT, NT), ND = 2 * NT + XI;
  extern __shared__ __attribute__((aligned(16))) char s_dyn[];  // [waves][D][B], then the sums
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int ln = lane & 15, kg = lane >> 4;
  int* const s_sum = reinterpret_cast<int*>(s_dyn + waves * D * B);
  float* const s_xs = reinterpret_cast<float*>(s_sum + MT * NT * 4 * kPlane);  // and the tokens' scales
  // each XCD (workgroups go round robin over the eight) takes a contiguous eighth of the list,
  // in which the token blocks of a channel tile follow each other: its L2 serves their weights
  const int total = n_tiles * m_blocks, per_xcd = (total + 7) >> 3;
  const int item = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per_xcd || item >= total) return;
  const int64_t n0 = (int64_t)(item / m_blocks) * (16 * NT), m0 = (int64_t)(item % m_blocks) * (16 * MT);
  const int rows = (int)min((int64_t)(16 * MT), p.m - m0), chans = (int)min((int64_t)(16 * NT), p.n - n0);

  // scales, requested first of all: the results wait for nothing then. Every thread's results are
  // of one channel (a multiple of 16 NT threads).
  const int tc = threadIdx.x % (16 * NT);
  const BiasReader rb = bias_reader(p, n0, chans);
  const uint32_t bias = bias_bits(rb, tc);
  const float ws = __builtin_bit_cast(
      float, __builtin_amdgcn_raw_buffer_load_b32(buffer_over(p.w_scale + n0, chans * 4), tc * 4, 0, 0));
  const uint32_t xs = __builtin_amdgcn_raw_buffer_load_b32(buffer_over(p.x_scale + m0, rows * 4),
                                                           (threadIdx.x % (16 * MT)) * 4, 0, 0);

  // a DMA instruction brings eight rows of 128 bytes; lane l byte 16 (l % 8) of row l / 8, which
  // holds chunk (l % 8) ^ swizzle. Rows past the end and, in the last 128 keys, chunks past k
  // get an offset outside the descriptors: zeros without an access.
  const i32x4 rx = buffer_words(p.x + m0 * p.x_stride, (uint32_t)((rows - 1) * (int)p.x_stride + p.k));
  const i32x4 rw = buffer_words(p.w + n0 * p.w_stride, (uint32_t)((chans - 1) * (int)p.w_stride + p.k));
  const int r8 = lane >> 3;
  const int chunk[2] = {16 * ((lane & 7) ^ stream_swizzle(r8)), 16 * ((lane & 7) ^ stream_swizzle(8 + r8))};
  int off[ND];
#pragma unroll
  for (int u = 0; u < 2 * NT; ++u) off[u] = 8 * u + r8 < chans ? (8 * u + r8) * (int)p.w_stride + chunk[u & 1] : kFar;
#pragma unroll
  for (int u = 0; u < XI; ++u)
    off[2 * NT + u] = 8 * u + r8 < rows ? (8 * u + r8) * (int)p.x_stride + chunk[u & 1] : kFar;
  const int blocks = (p.k + 127) >> 7, last = blocks - 1;
  // channel tiles begin at different keys, so that those that run at once on an XCD do not all
  // ask for the same cache lines (28672 x 4096 at m = 24 26.5 -> 23.1 us, at m = 1 21.3 -> 20.4)
  const int rotation = item / m_blocks % 32 * blocks / 32;
  const int past[2] = {last * 128 + chunk[0] >= p.k ? kFar : 0, last * 128 + chunk[1] >= p.k ? kFar : 0};
  const int count = wave < blocks ? (blocks - wave + waves - 1) / waves : 0;  // of this wave: wave, wave + waves, ...
  const LdsBytes ring = (LdsBytes)s_dyn + wave * D * B;
  asm volatile("s_nop 4");  // descriptor SGPRs written by VALU before the first asm load
  auto request = [&](int i, int slot) {  // the wave's block i
    const int turn = wave + i * waves + rotation, at = turn < blocks ? turn : turn - blocks;
    const int so = __builtin_amdgcn_readfirstlane(at * 128);
    const int base = __builtin_amdgcn_readfirstlane(slot * B);
    const int add[2] = {at == last ? past[0] : 0, at == last ? past[1] : 0};
    asm volatile("s_nop 4" : : "s"(so), "s"(base));  // VALU-written SGPRs: five wait states before a VMEM reads them
    if (once) {
#pragma unroll
      for (int u = 0; u < 2 * NT; ++u) dma_b128<true>(rw, ring + base + u * 1024, off[u] + add[u & 1], so);
    } else {
#pragma unroll
      for (int u = 0; u < 2 * NT; ++u) dma_b128(rw, ring + base + u * 1024, off[u] + add[u & 1], so);
    }
#pragma unroll
    for (int u = 2 * NT; u < ND; ++u) dma_b128(rx, ring + base + u * 1024, off[u] + add[u & 1], so);
  };
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (d < count) request(d, d);
  for (int i = threadIdx.x; i < MT * NT * 4 * kPlane; i += blockDim.x) s_sum[i] = 0;

  // fragment of lane (ln, kg): row ln, key step s: chunk 2 kg + s
  const int f[2] = {ln * 128 + 16 * ((2 * kg) ^ stream_swizzle(ln)), ln * 128 + 16 * ((2 * kg + 1) ^ stream_swizzle(ln))};
  const char* const mine = s_dyn + wave * D * B;
  i32x4 acc[NT][MT] = {};
  int slot = 0;
  for (int i = 0; i < count; ++i) {
    if (count - i >= D)
      asm volatile("s_waitcnt vmcnt(%0)" : : "n"((D - 1) * ND) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    i32x4 a[2][NT], b[2][MT];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int t = 0; t < NT; ++t) a[s][t] = *reinterpret_cast<const i32x4*>(mine + slot * B + t * 2048 + f[s]);
#pragma unroll
      for (int t = 0; t < MT; ++t) b[s][t] = *reinterpret_cast<const i32x4*>(mine + slot * B + (NT + t) * 2048 + f[s]);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read: the block's place is free
    if (i + D < count) request(i + D, slot);
    slot = slot + 1 == D ? 0 : slot + 1;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < MT; ++u) acc[t][u] = mfma_i8(a[s][t], b[s][u], acc[t][u]);
  }
  if (threadIdx.x < 16 * MT) s_xs[threadIdx.x] = __builtin_bit_cast(float, xs);
  __syncthreads();  // the sums are cleared
  if (count > 0) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int u = 0; u < MT; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          __hip_atomic_fetch_add(&s_sum[((t * MT + u) * 4 + e) * kPlane + lane], acc[t][u][e], __ATOMIC_RELAXED,
                                 __HIP_MEMORY_SCOPE_WORKGROUP);
  }
  __syncthreads();
  const float bf = bias_value(rb, bias);
  TO* const out = (TO*)p.out + m0 * p.o_stride + n0;
  for (int r = threadIdx.x / (16 * NT); r < rows; r += blockDim.x / (16 * NT))
    if (tc < chans) {
      const int sum = s_sum[(((tc >> 4) * MT + (r >> 4)) * 4 + (tc & 3)) * kPlane + 16 * ((tc & 15) >> 2) + (r & 15)];
      out[r * p.o_stride + tc] = (TO)scaled(sum, s_xs[r], ws, bf);
    }
}

template <typename TO, int MT, int NT, int XI>
int launch_stream(const W8Params& p, const StreamPlan& pl, hipStream_t stream) {
  auto kern = w8a8_stream_kernel<TO, MT, NT, XI>;
  const int lds = stream_lds_bytes(MT, NT, pl.waves);
  static std::atomic<uint64_t> done{0};
  constexpr int most = stream_lds_bytes(MT, NT, 8) < kLdsBytes ? stream_lds_bytes(MT, NT, 8) : kLdsBytes;
  if (const int st = reserve_lds((const void*)kern, most, done); st != SS_OK) return st;
  const int64_t grid = ((int64_t)pl.n_tiles * pl.m_blocks + 7) / 8 * 8;
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(64 * pl.waves), lds, stream, p, pl.n_tiles, pl.m_blocks,
                     pl.once);
  return ss_host::launch_status("w8a8 gemm (stream)");
}

// 16-row tiles of tokens and of channels of a workgroup
#define W8A8_STREAMS(X) X(1, 1) X(1, 2) X(2, 1) X(2, 2) X(4, 2) X(4, 4)

template <typename TO>
int launch_stream_typed(const W8Params& p, const StreamPlan& pl, hipStream_t stream) {
#define W8A8_LAUNCH(MT, NT)                                                      \
  if (pl.mt == MT && pl.nt == NT) {                                              \
    if (MT == 1 && p.m <= 8) return launch_stream<TO, MT, NT, 1>(p, pl, stream); \
    return launch_stream<TO, MT, NT, 2 * MT>(p, pl, stream);                     \
  }
  W8A8_STREAMS(W8A8_LAUNCH)
#undef W8A8_LAUNCH
  ss_host::set_error("w8a8 gemm: stream tile of %d x %d", pl.mt, pl.nt);
  return SS_ERR_UNSUPPORTED;
}

}  // namespace

// The tile and waves of least estimated time (us), fitted to the times of 3500 calls (every tile
// and number of waves at 240 shapes of up to 512 tokens); 8 % off on average over 3177 calls of the
// kernel as it is, too low for weights of hundreds of MB (8192 x 28672 at m = 32 36 us, takes 44;
// 57344 x 8192 73, takes 86 with the two waves so chosen and 76 with four): a round's
// start, a wave's blocks one after another, the adding of the sums and the results, the
// operands' way through a CU and out of the L2, and the weights' out of the memory.
double plan_w8a8_stream(StreamPlan& pl, int64_t m, int64_t n, int64_t k) {
#define W8A8_SIZE(MT, NT) {MT, NT},
  static const int kTiles[][2] = {W8A8_STREAMS(W8A8_SIZE)};
#undef W8A8_SIZE
  const int64_t cus = ss_host::device_cu_count(), blocks = (k + 127) / 128;
  double best = 1e30;
  if (m > 512) return best;
  for (const auto& t : kTiles) {
    const int mt = t[0], nt = t[1];
    if (mt > 1 && 8 * mt >= m) continue;
    const int64_t n_tiles = (n + 16 * nt - 1) / (16 * nt), m_blocks = (m + 16 * mt - 1) / (16 * mt);
    if (n_tiles * m_blocks > kMostGroups) continue;
    const int64_t groups = n_tiles * m_blocks, a_cu = (groups + cus - 1) / cus;
    const bool once = read_once(mt, m_blocks, n, k);
    const double bytes = (16.0 * nt + (m < 16 * mt ? m : 16 * mt)) * blocks * 128;
    // two waves only beyond 16 tokens (28672 x 4096 at m = 1 26.2 us with two, 22.3 with four)
    for (int waves = m > 16 ? 2 : 4; waves <= 8; waves *= 2) {
      const int64_t lds = stream_lds_bytes(mt, nt, waves);
      if (lds > kLdsBytes) continue;
      int64_t fit = kLdsBytes / lds;
      fit = fit < 32 / waves ? fit : 32 / waves;
      const double rounds = (double)((groups + cus * fit - 1) / (cus * fit)), each = (double)((blocks + waves - 1) / waves);
      const double us = 0.94 + rounds * (1.15 + each * (0.0141 * (mt + nt) + 0.0051 * mt * nt) +
                                         mt * nt * (0.103 + 0.416 / waves)) +
                        a_cu * (bytes * 5.32e-6 + 0.0005 * waves) + groups * bytes * 8.4e-9 + n * k * (once ? 7.4e-8 : 8.43e-8);
      if (us < best) {
        best = us;
        pl = {mt, nt, waves, (int)n_tiles, (int)m_blocks, once};
      }
    }
  }
  return best;
}

int launch_w8a8_stream(const W8Params& p, const StreamPlan& pl, int out_dtype, hipStream_t stream) {
  if (out_dtype == SS_DTYPE_BF16) return launch_stream_typed<bf16_t>(p, pl, stream);
  if (out_dtype == SS_DTYPE_F16) return launch_stream_typed<f16_t>(p, pl, stream);
  return launch_stream_typed<float>(p, pl, stream);
}

}  // namespace ss
