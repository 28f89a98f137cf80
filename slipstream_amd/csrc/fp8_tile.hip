// Tile kernel of the product in 8-bit floating point: from some tens of tokens on, where the matrix cores or
// the operands' way into the LDS set the time.
//
// Eight waves multiply 16 JT WM tokens with 16 IT (8 / WM) channels, wave (wm, wn) 16 JT x 16 IT of them. A
// stage is a block of 128 keys: its rows (128 bytes) and its scales come by DMA into rings of D stages. An
// instruction of 16 x 16 x 128 sums a whole block, so a product's result is multiplied with its block's scales
// and added to the fp32 sums while the products after it run: four fused multiply-adds of 4 cycles against a
// product's 32.
//
// 2240 x 28672 x 4096: 234 to 253 us, 2.1 to 2.25 PFLOP/s (the card's library product with one scale 239), the matrix
// cores busy for half of the cycles at the 1.7 to 2 GHz that the card's power leaves; 197 x 4096 x 14336 29 us (keys
// split over workgroups, then the sums' way out and in). To fp16 and fp32 the operands' widening is the longer part: two halves of
// a dword in 8 cycles each, 333 x 4999 x 2064 19 us against 14.8 to bf16.
#include "fp8_common.h"
#include "tile_order.h"

namespace ss {
namespace {

constexpr int kLdsBytes = 160 * 1024;
constexpr int kFar = 0x40000000;  // a byte offset past any operand tile (host-checked)

constexpr int stage_bytes(int bm, int bn) { return (bm + bn) * 128 + bm * 4 + 256; }
constexpr int ring_depth(int bm, int bn) {
  int d = 2;
  while (d < 6 && (d + 1) * stage_bytes(bm, bn) <= kLdsBytes) ++d;
  return d;
}

__device__ __forceinline__ void mfma_block(f32x4& r, const i32x8& a, const i32x8& b) {
  asm volatile("v_mfma_f32_16x16x128_f8f6f4 %0, %1, %2, 0" : "=&v"(r) : "v"(a), "v"(b));
}

// TO: the results' type; PART: fp32 sums of a K range instead, for the reduce kernel
template <typename TO, bool PART, int JT, int IT, int WM>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void fp8_tile_kernel(
    const F8Params p, int per, int ks, int n_tiles, int m_blocks, int band) {
  constexpr int WN = 8 / WM, BM = 16 * JT * WM, BN = 16 * IT * WN;
  constexpr int D = ring_depth(BM, BN);
  constexpr int XB = BM * 128, WB = BN * 128, SB = stage_bytes(BM, BN);  // a stage: tokens, channels, their scales
  constexpr int NX = BM / 64, NW = BN / 64, ND = NX + NW + 1;            // DMA instructions of a wave and stage
  static_assert(BM % 64 == 0 && BN % 128 == 0 && BM <= 256 && JT <= 4, "tile");
  extern __shared__ __attribute__((aligned(1024))) char s_dyn[];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ln = lane & 15, kg = lane >> 4;
  const int wm = wave % WM, wn = wave / WM;
  // workgroup -> (K range, channel tile, token block) as in w8a8_tile.hip: each XCD takes a contiguous eighth
  // of a list in which the workgroups that run at once share few rows of both operands
  const int total = ks * n_tiles * m_blocks, per_xcd = (total + 7) >> 3;
  const int item = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per_xcd || item >= total) return;
  const int in_band = band * n_tiles * ks;
  const int mb0 = item / in_band * band, left = item - mb0 * n_tiles * ks;
  const int here = min(band, m_blocks - mb0);
  const int pair = left / here, zr = pair % ks;
  const int64_t n0 = (int64_t)(pair / ks) * BN, m0 = (int64_t)(mb0 + left - pair * here) * BM;
  const int rows = (int)min((int64_t)BM, p.m - m0), chans = (int)min((int64_t)BN, p.n - n0);
  const int stages = (p.k + 127) >> 7;
  const int i0 = zr * per, i1 = min(stages, i0 + per);

  // ---- operands: a DMA instruction brings eight LDS rows; lane l byte 16 (l % 8) of row l / 8, which holds
  // chunk (l % 8) ^ swizzle. Rows past the end and, in the last block, chunks past k get an offset outside
  // the descriptors: zeros without an access. One more brings four bytes a lane: the scales of 64 tokens
  // (the first waves), or those of the channels' blocks of 128.
  const i32x4 rx = buffer_words(p.x + m0 * p.x_stride, (uint32_t)((rows - 1) * (int)p.x_stride + p.k));
  const i32x4 rw = buffer_words(p.w + n0 * p.w_stride, (uint32_t)((chans - 1) * (int)p.w_stride + p.k));
  const int row8 = 8 * wave + (lane >> 3);
  const int chunk = 16 * ((lane & 7) ^ f8_swizzle(row8 & 15));
  int off[NX + NW];
#pragma unroll
  for (int u = 0; u < NX; ++u) off[u] = 64 * u + row8 < rows ? (64 * u + row8) * (int)p.x_stride + chunk : kFar;
#pragma unroll
  for (int u = 0; u < NW; ++u) off[NX + u] = 64 * u + row8 < chans ? (64 * u + row8) * (int)p.w_stride + chunk : kFar;
  const int past = (stages - 1) * 128 + chunk >= p.k ? kFar : 0;  // of the last stage
  const bool of_x = wave < NX;
  const int blocks_n = (chans + 127) >> 7;
  const int64_t sc_blk = of_x ? p.xs_blk : p.ws_blk;
  const i32x4 rs = of_x ? buffer_words(p.x_scale + m0 * p.xs_row,
                                       (uint32_t)(4 * ((rows - 1) * (int)p.xs_row + (stages - 1) * (int)p.xs_blk + 1)))
                        : buffer_words(p.w_scale + (n0 >> 7) * p.ws_row,
                                       (uint32_t)(4 * ((blocks_n - 1) * (int)p.ws_row + (stages - 1) * (int)p.ws_blk + 1)));
  const int off_s = of_x ? (64 * wave + lane < rows ? 4 * (64 * wave + lane) * (int)p.xs_row : kFar)
                         : (lane < blocks_n ? 4 * lane * (int)p.ws_row : kFar);
  const LdsBytes lds = (LdsBytes)s_dyn;
  const uint32_t base = lds_address(s_dyn);
  struct {
    int so, ss, slot;
  } to;
  auto aim = [&](int i, int slot) {  // stage i into ring slot `slot`; past the range zeros, which nobody reads
    const int at = min(i, stages - 1);
    to.so = __builtin_amdgcn_readfirstlane(at * 128);
    to.ss = __builtin_amdgcn_readfirstlane(4 * at * (int)sc_blk);
    to.slot = __builtin_amdgcn_readfirstlane(slot * SB);
    if (i >= min(i1, stages - 1)) {  // the last stage's chunks past k, and all past the range, from here on
      const int add = i >= i1 ? kFar : past;
#pragma unroll
      for (int u = 0; u < NX + NW; ++u) off[u] |= add;
    }
    asm volatile("s_nop 4" : : "s"(to.so), "s"(to.ss), "s"(to.slot));  // VALU-written SGPRs: five wait states
  };
  auto dma = [&](auto uc) __attribute__((always_inline)) {
    constexpr int u = decltype(uc)::value;
    if constexpr (u < NX) {
      dma_b128(rx, lds + to.slot + u * 8192 + wave * 1024, off[u], to.so);
    } else if constexpr (u < NX + NW) {
      dma_b128(rw, lds + to.slot + XB + (u - NX) * 8192 + wave * 1024, off[u], to.so);
    } else {
      dma_b32(rs, base + to.slot + XB + WB + (of_x ? wave * 256 : BM * 4), off_s, to.ss);
    }
  };

  // fragment of lane (ln, kg): row ln of a 16-row tile, chunks 2 kg and 2 kg + 1. The addresses of a stage's
  // first fragments and scales are kept; the others are a constant away.
  const uint32_t chunk0 = ln * 128 + 16 * ((2 * kg) ^ f8_swizzle(ln)), chunk1 = ln * 128 + 16 * ((2 * kg + 1) ^ f8_swizzle(ln));
  uint32_t x0, x1, w0, w1, sx, sw;
  auto look_at = [&](int slot) __attribute__((always_inline)) {
    const uint32_t at = base + slot * SB, xb = at + wm * JT * 2048, wb = at + XB + wn * IT * 2048;
    x0 = xb + chunk0, x1 = xb + chunk1, w0 = wb + chunk0, w1 = wb + chunk1;
    sx = at + XB + WB + 4 * (16 * JT * wm + ln), sw = at + XB + WB + BM * 4 + 4 * ((wn * IT * 16) >> 7);
    asm volatile("" : "+v"(x0), "+v"(x1), "+v"(w0), "+v"(w1), "+v"(sx), "+v"(sw));
  };
  auto frag = [&](uint32_t lo, uint32_t hi) __attribute__((always_inline)) {
    return join8(__builtin_bit_cast(i32x4, lds_word(lo)), __builtin_bit_cast(i32x4, lds_word(hi)));
  };

  f32x4 acc[IT][JT];
#pragma unroll
  for (int i = 0; i < IT; ++i)
#pragma unroll
    for (int j = 0; j < JT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  asm volatile("s_nop 4");  // descriptor SGPRs written by VALU before the first asm load
  static_for<D - 1>([&](auto jc) __attribute__((always_inline)) {
    constexpr int j = decltype(jc)::value;
    aim(i0 + j, j);
    static_for<ND>(dma);
  });

  // The products of a stage in the order of the channels' tiles. What the next stage begins with is read behind
  // the last channels' products, once it has landed for all waves (kReady); the DMAs of the stage D - 1 on
  // follow the first product, when all waves are past the stage whose place they take, and are through early,
  // so that most of the stage is left for them to land in. A product's results are added two products later, the
  // last two's in the next stage.
  constexpr int P = IT * JT, kReady = P - JT, kSent = P >= 16 ? P / 4 : 1;
  static_assert(P % 4 == 0 && IT % 2 == 0 && JT >= 2 && kSent <= kReady, "order");
  i32x8 next_a, next_b[JT];  // a stage's first operands and its scales, as they lie in the LDS
  float next_sc[JT], next_ws, sc[JT];
  f32x4 part[4];
#pragma unroll
  for (int j = 0; j < JT; ++j) sc[j] = 0.f;
  part[2] = part[3] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto add = [&](auto ic) __attribute__((always_inline)) {
    constexpr int q = decltype(ic)::value, i = q / JT, j = q % JT;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(part[q % 4][e], sc[j], acc[i][j][e]);
  };
  auto begin_a = [&]() __attribute__((always_inline)) {
    next_a = frag(w0, w1);
    next_ws = lds_float(sw);
  };
  auto begin_b = [&](int j) __attribute__((always_inline)) {
    next_b[j] = frag(x0 + j * 2048, x1 + j * 2048);
    next_sc[j] = lds_float(sx + 64 * j);
  };
  wait_dma<(D - 2) * ND>();
  __syncthreads();
  look_at(0);
  begin_a();
#pragma unroll
  for (int j = 0; j < JT; ++j) begin_b(j);
  int slot = 0;
  for (int st = i0; st < i1; ++st) {
    typename Block<TO>::Operand b[JT], a[2];
    a[0] = Block<TO>::operand(next_a);
#pragma unroll
    for (int j = 0; j < JT; ++j) b[j] = Block<TO>::operand(next_b[j]);
    const int before = slot == 0 ? D - 1 : slot - 1, after = slot + 1 == D ? 0 : slot + 1;
    __builtin_amdgcn_sched_barrier(0);
    static_for<P>([&](auto qc) __attribute__((always_inline)) {
      constexpr int q = decltype(qc)::value, i = q / JT, j = q % JT;
      if constexpr (__is_same(TO, bf16_t)) {
        mfma_block(part[q % 4], a[i & 1], b[j]);
      } else {
        part[q % 4] = Block<TO>::sum(a[i & 1], b[j]);
      }
      if constexpr (q == kReady) {
        wait_dma<(D - 2) * ND>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        look_at(after);
        begin_a();
      }
      if constexpr (j == 0 && i + 1 < IT) a[(i + 1) & 1] = Block<TO>::operand(frag(w0 + (i + 1) * 2048, w1 + (i + 1) * 2048));
      if constexpr (q >= kReady) begin_b(j);
      if constexpr (q == 0) {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        aim(st + D - 1, before);
      }
      constexpr int from = q < kSent ? q * ND / kSent : ND, to = q < kSent ? (q + 1) * ND / kSent : ND;
      static_for<to - from>([&](auto uc) __attribute__((always_inline)) {
        dma(std::integral_constant<int, from + decltype(uc)::value>{});
      });
      // not before this product's issue: it waits for the matrix cores to be done with the two before it. (Left
      // to the compiler, which does not know the asm's latency, the sums were read one product too early.)
      constexpr int done = (q + P - 2) % P;
      if constexpr (__is_same(TO, bf16_t)) asm volatile("" : "+v"(part[done % 4]));
      add(std::integral_constant<int, done>{});
      if constexpr (q == 1) {
#pragma unroll
        for (int t = 0; t < JT; ++t) sc[t] = next_sc[t] * next_ws;
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    slot = after;
  }
  asm volatile("s_nop 15\n\ts_nop 3" : "+v"(part[2]), "+v"(part[3]));  // the last products are through
  add(std::integral_constant<int, P - 2>{});
  add(std::integral_constant<int, P - 1>{});
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // no DMA and no read of the LDS is on its way,
  __syncthreads();                                              // of any wave

  // ---- results: 16 tokens at a time through the wave's own part of the LDS, so that lanes hold consecutive
  // channels and a store writes rows of the wave's 16 IT channels
  typedef typename std::conditional<PART, float, TO>::type TS;
  constexpr int CL = 16 / sizeof(TS), LR = 16 * IT / CL;  // channels of a lane, lanes of a token in the store
  constexpr int RS = 16 * IT * sizeof(TS) + 16;           // bytes of a token there
  static_assert(8 * 16 * RS <= D * SB && (LR & (LR - 1)) == 0 && LR <= 64, "the results fit where the operands were");
  char* const turn = s_dyn + wave * 16 * RS;
  TS* const out = (TS*)p.out + (PART ? (int64_t)zr * p.m * p.o_stride : 0);
  const int64_t mw = m0 + 16 * JT * wm, nw = n0 + 16 * IT * wn;
  const int left_rows = rows - 16 * JT * wm, left_chans = chans - 16 * IT * wn;
  float bias[IT][4];
#pragma unroll
  for (int i = 0; i < IT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = 16 * i + 4 * kg + e;
      bias[i][e] = !PART && p.bias && c < left_chans ? load_as_f32(p.bias, nw + c, p.bias_dtype) : 0.f;
    }
  const int c = lane % LR * CL;
  const bool pieces = p.n % CL == 0 && p.o_stride % CL == 0 && ((uintptr_t)p.out & 15) == 0;
#pragma unroll
  for (int j = 0; j < JT; ++j) {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = acc[i][j][e] + bias[i][e];
      char* const at = turn + ln * RS + (16 * i + 4 * kg) * sizeof(TS);
      if constexpr (sizeof(TS) == 4)
        *reinterpret_cast<f32x4*>(at) = f32x4{y[0], y[1], y[2], y[3]};
      else
        *reinterpret_cast<u32x2*>(at) = u32x2{Elem<TS>::pack2(y[0], y[1]), Elem<TS>::pack2(y[2], y[3])};
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int r0 = 0; r0 < 16; r0 += 64 / LR) {
      const int r = r0 + lane / LR;
      const u32x4 v = load16(turn + r * RS + c * sizeof(TS));
      if (r >= 16 || 16 * j + r >= left_rows || c >= left_chans) continue;
      TS* const o = out + (mw + 16 * j + r) * p.o_stride + nw + c;
      if (pieces || c + CL <= left_chans) {
        __builtin_memcpy(o, &v, 16);
      } else {
        TS y[CL];
        __builtin_memcpy(y, &v, 16);
#pragma unroll
        for (int e = 0; e < CL; ++e)
          if (c + e < left_chans) o[e] = y[e];
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the next tokens are written
  }
}

// The fp32 sums of ks K ranges added in order, with the bias, and rounded: a thread four channels of a token
template <typename TO>
__global__ __launch_bounds__(256) void fp8_reduce_kernel(const F8Params p, const float* __restrict__ part, int ks) {
  const uint32_t quads = (uint32_t)((p.n + 3) >> 2), total = (uint32_t)p.m * quads;  // m n below 2^29
  const int64_t plane = p.m * p.n;
  for (uint32_t q = blockIdx.x * 256 + threadIdx.x; q < total; q += gridDim.x * 256) {
    const int m = (int)(q / quads), n = 4 * (int)(q - m * quads);
    const float* const at = part + (int64_t)m * p.n + n;
    TO* const o = (TO*)p.out + m * p.o_stride + n;
    const int have = min(4, (int)p.n - n);
    float y[4] = {0.f, 0.f, 0.f, 0.f};
    if (p.n % 4 == 0) {
      for (int z = 0; z < ks; z += 4) {
        f32x4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const f32x4*>(at + min(z + j, ks - 1) * plane);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (z + j < ks)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] += v[j][e];
      }
    } else {
      for (int z = 0; z < ks; ++z)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < have) y[e] += at[z * plane + e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < have) o[e] = (TO)(y[e] + (p.bias ? load_as_f32(p.bias, n + e, p.bias_dtype) : 0.f));
  }
}

template <typename TO, bool PART, int JT, int IT, int WM>
int launch_tile(const F8Params& p, const F8TilePlan& pl, hipStream_t stream) {
  constexpr int bm = 16 * JT * WM, bn = 16 * IT * (8 / WM), lds = ring_depth(bm, bn) * stage_bytes(bm, bn);
  auto kern = fp8_tile_kernel<TO, PART, JT, IT, WM>;
  static std::atomic<uint64_t> done{0};
  if (const int st = reserve_lds((const void*)kern, lds, done); st != SS_OK) return st;
  // bands of at most 8 token blocks, of one size where they can be
  const int bands = (pl.m_blocks + 7) / 8, band = (pl.m_blocks + bands - 1) / bands;
  const int64_t grid = ((int64_t)pl.ks * pl.n_tiles * pl.m_blocks + 7) / 8 * 8;
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(512), lds, stream, p, pl.per, pl.ks, pl.n_tiles, pl.m_blocks, band);
  return ss_host::launch_status("fp8 gemm (tile)");
}

// A tile's tokens and channels, and its waves' tiles of 16 (JT, IT) and rows of waves (WM). The widest does
// not fit the registers with operands widened to bf16.
#define FP8_TILES(X) X(256, 256, 4, 8, 4) X(128, 256, 4, 4, 2) X(256, 128, 4, 4, 4) X(128, 128, 4, 2, 2) X(64, 128, 2, 2, 2)

template <typename TO, bool PART>
int launch_tile_typed(const F8Params& p, const F8TilePlan& pl, hipStream_t stream) {
#define FP8_LAUNCH(BM, BN, JT, IT, WM)                                                            \
  if (pl.bm == BM && pl.bn == BN)                                                                 \
    if constexpr (__is_same(TO, bf16_t) || IT < 8) return launch_tile<TO, PART, JT, IT, WM>(p, pl, stream);
  FP8_TILES(FP8_LAUNCH)
#undef FP8_LAUNCH
  ss_host::set_error("fp8 gemm: tile of %d x %d", pl.bm, pl.bn);
  return SS_ERR_UNSUPPORTED;
}

template <typename TO>
int launch_typed(const F8Params& p, const F8TilePlan& pl, float* part, hipStream_t stream) {
  if (pl.ks == 1) return launch_tile_typed<TO, false>(p, pl, stream);
  F8Params q = p;
  q.out = part;
  q.o_stride = p.n;
  if (const int st = launch_tile_typed<TO, true>(q, pl, stream); st != SS_OK) return st;
  const int64_t blocks = (p.m * ((p.n + 3) / 4) + 255) / 256, cap = (int64_t)ss_host::device_cu_count() * 8;
  hipLaunchKernelGGL(fp8_reduce_kernel<TO>, dim3((unsigned)(blocks < cap ? blocks : cap)), dim3(256), 0, stream, p, part,
                     pl.ks);
  return ss_host::launch_status("fp8 gemm (reduce)");
}

}  // namespace

double plan_fp8_tile(F8TilePlan& pl, int64_t m, int64_t n, int64_t k, bool wide, bool may_split) {
#define FP8_SIZE(BM, BN, JT, IT, WM) {BM, BN},
  static const int kTiles[][2] = {FP8_TILES(FP8_SIZE)};
#undef FP8_SIZE
  const int64_t stages = (k + 127) / 128, cus = ss_host::device_cu_count();
  double best = 1e30;
  pl.ks = 0;
  for (const auto& t : kTiles) {
    if (wide && t[0] == 256 && t[1] == 256) continue;
    const int64_t n_tiles = (n + t[1] - 1) / t[1], m_blocks = (m + t[0] - 1) / t[0];
    if (n_tiles * m_blocks > kMostGroups) continue;
    for (int64_t ks = 1; ks <= (may_split ? 14 : 1); ks += ks < 4 ? 1 : 2) {
      const int64_t per = (stages + ks - 1) / ks, groups = ks * n_tiles * m_blocks;
      if (ks > 1 && (per < 4 || groups > 600 || ks * m * n * 4 >= ((int64_t)1 << 31))) break;
      if ((stages + per - 1) / per != ks) continue;
      const double rounds = (double)((groups + cus - 1) / cus), area = t[0] * t[1] / 65536.0, edge = t[0] + t[1];
      double us = 4 + rounds * (per * ((wide ? 2.2 : 1.2) * area + 0.2 * edge / 512 + 0.1) + 3 * area + 1) +
                  groups * per * edge * 128 * 1.79e-8 + n * k * 4.2e-8 + m * n * 2.96e-7;
      if (ks > 1) us += 3 + ks * m * n * 4 * 2.79e-7;
      if (us < best) {
        best = us;
        pl = {t[0], t[1], (int)ks, (int)per, (int)n_tiles, (int)m_blocks};
      }
    }
  }
  return best;
}

int launch_fp8_tile(const F8Params& p, const F8TilePlan& pl, int out_dtype, float* part, hipStream_t stream) {
  if (out_dtype == SS_DTYPE_BF16) return launch_typed<bf16_t>(p, pl, part, stream);
  if (out_dtype == SS_DTYPE_F16) return launch_typed<f16_t>(p, pl, part, stream);
  return launch_typed<float>(p, pl, part, stream);
}

}  // namespace ss
