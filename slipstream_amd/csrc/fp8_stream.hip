// Stream kernel of the product in 8-bit floating point: few tokens, where the weights' bytes set the time.
//
// A workgroup of up to eight waves multiplies 16 MT tokens with 16 NT channels; its waves share out the blocks
// of 128 keys, one after another in turn. A wave brings its blocks' rows by DMA into a part of the LDS that is
// its own, two in turn, with their scales behind them, and reads the matrix instruction's operands from there: no
// wave waits for another before the end, where the waves' sums are added in their order.
//
// Bound by the weights' way out of the memory: 1 x 28672 x 4096 19.3 us a call, 24.2 over three sets of weights in
// turn (4.9 TB/s), 24 x 28672 x 4096 26.3 (4.5). With the scales of all blocks read into a table first, a wave of
// four blocks waits for the memory twice (0.7 us).
#include "fp8_common.h"
#include "tile_order.h"

namespace ss {
namespace {

constexpr int kLdsBytes = 160 * 1024;
constexpr int kFar = 0x40000000;  // a byte offset past any operand tile (host-checked)
constexpr int kPlane = 68;        // LDS words of the 64 lanes' sums of one accumulator register
constexpr int D = 2;              // a wave's blocks on their way, or in work

// bytes of a block (128 keys of the weights' and tokens' rows, the tokens' scales and the channels', 64 lanes
// each), and of a workgroup's LDS: the rings, or the waves' sums in their place
constexpr int block_bytes(int mt, int nt) { return (16 * nt + 16 * mt) * 128 + 512; }
constexpr int stream_lds_bytes(int mt, int nt, int waves) {
  const int ring = waves * D * block_bytes(mt, nt), sums = waves * mt * nt * 4 * kPlane * 4;
  return ring > sums ? ring : sums;
}

// Whether the weights pass the caches by, as what is read once does: where no second token block reads them
inline bool read_once(int mt, int64_t m_blocks, int64_t n, int64_t k) {
  return m_blocks == 1 && (mt == 1 || n * k > kKeptWeights);
}

// XI: groups of eight tokens that are read (2 MT, or 1 of MT = 1); the rows of the others hold anything, and their
// sums are not stored.
template <typename TO, int MT, int NT, int XI>
__global__ __launch_bounds__(512) void fp8_stream_kernel(const F8Params p, int n_tiles, int m_blocks, bool once) {
  constexpr int B = block_bytes(MT, NT), SC = B - 512, ND = 2 * NT + XI;  // DMA instructions of a block's rows
  extern __shared__ __attribute__((aligned(1024))) char s_dyn[];  // [waves][D][B], then the sums
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int ln = lane & 15, kg = lane >> 4;
  // each XCD (workgroups go round robin over the eight) takes a contiguous eighth of the list, in which the
  // token blocks of a channel tile follow each other: its L2 serves their weights
  const int total = n_tiles * m_blocks, per_xcd = (total + 7) >> 3;
  const int item = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per_xcd || item >= total) return;
  const int64_t n0 = (int64_t)(item / m_blocks) * (16 * NT), m0 = (int64_t)(item % m_blocks) * (16 * MT);
  const int rows = (int)min((int64_t)(16 * MT), p.m - m0), chans = (int)min((int64_t)(16 * NT), p.n - n0);
  const int blocks = (p.k + 127) >> 7, last = blocks - 1;

  // a DMA instruction brings eight rows of 128 bytes; lane l byte 16 (l % 8) of row l / 8, which holds chunk
  // (l % 8) ^ swizzle. Rows past the end and, in the last block, chunks past k get an offset outside the
  // descriptors: zeros without an access.
  const i32x4 rx = buffer_words(p.x + m0 * p.x_stride, (uint32_t)((rows - 1) * (int)p.x_stride + p.k));
  const i32x4 rw = buffer_words(p.w + n0 * p.w_stride, (uint32_t)((chans - 1) * (int)p.w_stride + p.k));
  const int r8 = lane >> 3;
  const int chunk[2] = {16 * ((lane & 7) ^ f8_swizzle(r8)), 16 * ((lane & 7) ^ f8_swizzle(8 + r8))};
  int off[ND];
#pragma unroll
  for (int u = 0; u < 2 * NT; ++u) off[u] = 8 * u + r8 < chans ? (8 * u + r8) * (int)p.w_stride + chunk[u & 1] : kFar;
#pragma unroll
  for (int u = 0; u < XI; ++u)
    off[2 * NT + u] = 8 * u + r8 < rows ? (8 * u + r8) * (int)p.x_stride + chunk[u & 1] : kFar;
  // channel tiles begin at different blocks, so that those that run at once on an XCD do not all ask for the same
  // cache lines
  const int rotation = item / m_blocks % 32 * blocks / 32;
  const int past[2] = {last * 128 + chunk[0] >= p.k ? kFar : 0, last * 128 + chunk[1] >= p.k ? kFar : 0};
  const int count = wave < blocks ? (blocks - wave + waves - 1) / waves : 0;  // of this wave: wave, wave + waves, ...
  const LdsBytes ring = (LdsBytes)s_dyn + wave * D * B;
  const i32x4 rxs = buffer_words(p.x_scale + m0 * p.xs_row, (uint32_t)(4 * ((rows - 1) * (int)p.xs_row + last * (int)p.xs_blk + 1)));
  const i32x4 rws = buffer_words(p.w_scale + (n0 >> 7) * p.ws_row, (uint32_t)(4 * (last * (int)p.ws_blk + 1)));
  const int off_xs = lane < rows ? 4 * lane * (int)p.xs_row : kFar;  // the channels' one: every lane the same
  asm volatile("s_nop 4");  // descriptor SGPRs written by VALU before the first asm load
  auto request = [&](int i, int slot) {  // the wave's block i
    const int turn = wave + i * waves + rotation, at = turn < blocks ? turn : turn - blocks;
    const int so = __builtin_amdgcn_readfirstlane(at * 128);
    const int base = __builtin_amdgcn_readfirstlane(slot * B);
    const int add[2] = {at == last ? past[0] : 0, at == last ? past[1] : 0};
    const int sx = __builtin_amdgcn_readfirstlane(4 * at * (int)p.xs_blk), sw = __builtin_amdgcn_readfirstlane(4 * at * (int)p.ws_blk);
    asm volatile("s_nop 4" : : "s"(so), "s"(base), "s"(sx), "s"(sw));  // VALU-written SGPRs: five wait states before a VMEM
    if (once) {
#pragma unroll
      for (int u = 0; u < 2 * NT; ++u) dma_b128<true>(rw, ring + base + u * 1024, off[u] + add[u & 1], so);
    } else {
#pragma unroll
      for (int u = 0; u < 2 * NT; ++u) dma_b128(rw, ring + base + u * 1024, off[u] + add[u & 1], so);
    }
#pragma unroll
    for (int u = 2 * NT; u < ND; ++u) dma_b128(rx, ring + base + u * 1024, off[u] + add[u & 1], so);
    dma_b32(rxs, (uint32_t)(uintptr_t)(ring + base + SC), off_xs, sx);
    dma_b32(rws, (uint32_t)(uintptr_t)(ring + base + SC + 256), 0, sw);
  };
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (d < count) request(d, d);

  // fragment of lane (ln, kg): row ln, chunks 2 kg and 2 kg + 1
  const uint32_t mine = lds_address(s_dyn) + wave * D * B;
  const uint32_t f0 = mine + ln * 128 + 16 * ((2 * kg) ^ f8_swizzle(ln)), f1 = mine + ln * 128 + 16 * ((2 * kg + 1) ^ f8_swizzle(ln));
  f32x4 acc[NT][MT] = {};
  int slot = 0;
  for (int i = 0; i < count; ++i) {
    if (count - i >= D)
      wait_dma<(D - 1) * (ND + 2)>();
    else
      wait_dma<0>();
    i32x4 a[NT][2], b[MT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      a[t][0] = __builtin_bit_cast(i32x4, lds_word(f0 + slot * B + t * 2048));
      a[t][1] = __builtin_bit_cast(i32x4, lds_word(f1 + slot * B + t * 2048));
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      b[t][0] = __builtin_bit_cast(i32x4, lds_word(f0 + slot * B + (NT + t) * 2048));
      b[t][1] = __builtin_bit_cast(i32x4, lds_word(f1 + slot * B + (NT + t) * 2048));
    }
    float sc[MT];
    const uint32_t at = mine + slot * B + SC;
    const float ws = lds_float(at + 256);
#pragma unroll
    for (int t = 0; t < MT; ++t) sc[t] = lds_float(at + 4 * (16 * t + ln)) * ws;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read: the block's place is free
    if (i + D < count) request(i + D, slot);
    slot = slot + 1 == D ? 0 : slot + 1;
    typename Block<TO>::Operand bo[MT];
#pragma unroll
    for (int u = 0; u < MT; ++u) bo[u] = Block<TO>::operand(join8(b[u][0], b[u][1]));
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const typename Block<TO>::Operand ao = Block<TO>::operand(join8(a[t][0], a[t][1]));
#pragma unroll
      for (int u = 0; u < MT; ++u) {
        const f32x4 part = Block<TO>::sum(ao, bo[u]);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][u][e] = fmaf(part[e], sc[u], acc[t][u][e]);
      }
    }
  }
  __syncthreads();  // every wave's blocks are read: the sums take their place
  float* const s_sum = reinterpret_cast<float*>(s_dyn);
  constexpr int REGS = MT * NT * 4;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int u = 0; u < MT; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) s_sum[(wave * REGS + (t * MT + u) * 4 + e) * kPlane + lane] = acc[t][u][e];
  __syncthreads();
  const int tc = threadIdx.x % (16 * NT);
  if (tc >= chans) return;
  const float bias = p.bias ? load_as_f32(p.bias, n0 + tc, p.bias_dtype) : 0.f;
  TO* const out = (TO*)p.out + m0 * p.o_stride + n0 + tc;
  for (int r = threadIdx.x / (16 * NT); r < rows; r += blockDim.x / (16 * NT)) {
    const int at = (((tc >> 4) * MT + (r >> 4)) * 4 + (tc & 3)) * kPlane + 16 * ((tc & 15) >> 2) + (r & 15);
    float y = s_sum[at];
    for (int w = 1; w < waves; ++w) y += s_sum[w * REGS * kPlane + at];
    out[r * p.o_stride] = (TO)(y + bias);
  }
}

template <typename TO, int MT, int NT, int XI>
int launch_stream(const F8Params& p, const F8StreamPlan& pl, hipStream_t stream) {
  auto kern = fp8_stream_kernel<TO, MT, NT, XI>;
  const int lds = stream_lds_bytes(MT, NT, pl.waves);
  static std::atomic<uint64_t> done{0};
  constexpr int most = stream_lds_bytes(MT, NT, 8) < kLdsBytes ? stream_lds_bytes(MT, NT, 8) : kLdsBytes;
  if (const int st = reserve_lds((const void*)kern, most, done); st != SS_OK) return st;
  const int64_t grid = ((int64_t)pl.n_tiles * pl.m_blocks + 7) / 8 * 8;
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(64 * pl.waves), lds, stream, p, pl.n_tiles, pl.m_blocks, pl.once);
  return ss_host::launch_status("fp8 gemm (stream)");
}

// 16-row tiles of tokens and of channels of a workgroup
#define FP8_STREAMS(X) X(1, 1) X(1, 2) X(2, 1) X(2, 2) X(4, 2)

template <typename TO>
int launch_stream_typed(const F8Params& p, const F8StreamPlan& pl, hipStream_t stream) {
#define FP8_LAUNCH(MT, NT)                                                       \
  if (pl.mt == MT && pl.nt == NT) {                                              \
    if (MT == 1 && p.m <= 8) return launch_stream<TO, MT, NT, 1>(p, pl, stream); \
    return launch_stream<TO, MT, NT, 2 * MT>(p, pl, stream);                     \
  }
  FP8_STREAMS(FP8_LAUNCH)
#undef FP8_LAUNCH
  ss_host::set_error("fp8 gemm: stream tile of %d x %d", pl.mt, pl.nt);
  return SS_ERR_UNSUPPORTED;
}

}  // namespace

// The tile and waves of least estimated time (us): a round's start, a wave's blocks one after another, the adding
// of the sums, the operands' way through a CU and the weights' out of the memory.
double plan_fp8_stream(F8StreamPlan& pl, int64_t m, int64_t n, int64_t k) {
#define FP8_SIZE(MT, NT) {MT, NT},
  static const int kTiles[][2] = {FP8_STREAMS(FP8_SIZE)};
#undef FP8_SIZE
  const int64_t cus = ss_host::device_cu_count(), blocks = (k + 127) / 128;
  double best = 1e30;
  if (m > 128) return best;
  for (const auto& t : kTiles) {
    const int mt = t[0], nt = t[1];
    if (mt > 1 && 8 * mt >= m) continue;
    const int64_t n_tiles = (n + 16 * nt - 1) / (16 * nt), m_blocks = (m + 16 * mt - 1) / (16 * mt);
    if (n_tiles * m_blocks > kMostGroups) continue;
    const int64_t groups = n_tiles * m_blocks, a_cu = (groups + cus - 1) / cus;
    const bool once = read_once(mt, m_blocks, n, k);
    const double bytes = (16.0 * nt + (m < 16 * mt ? m : 16 * mt)) * blocks * 128;
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

int launch_fp8_stream(const F8Params& p, const F8StreamPlan& pl, int out_dtype, hipStream_t stream) {
  if (out_dtype == SS_DTYPE_BF16) return launch_stream_typed<bf16_t>(p, pl, stream);
  if (out_dtype == SS_DTYPE_F16) return launch_stream_typed<f16_t>(p, pl, stream);
  return launch_stream_typed<float>(p, pl, stream);
}

}  // namespace ss
