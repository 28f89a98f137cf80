// W8A8 tile kernel: the int8 product at the sizes where the matrix cores set the time (a prefill
// chunk's or a packed step's tokens).
//
// Four waves multiply 32 MT WM tokens with 32 NT (4 / WM) channels, wave (wm, wn) 32 MT x 32 NT
// of them. Both operands come into LDS by DMA, 128 keys of every row a stage, into rings of as
// many stages as fit (256 x 256: three of the tokens', two of the channels'). A wave holds the
// fragments of half a stage (64 keys) in registers while it multiplies them and reads the next
// half's beside the products, so a stage's LDS is free again once its second half has been
// read, long before it is multiplied:
//   first half's products:  the second half's fragments are read, then (barrier) the stage's
//                           LDS is free and the DMAs into it begin
//   second half's products: the DMAs go on; the next stage's, a stage or more old, have landed
//                           (wait, barrier) and its first half's fragments are read
// One wave per SIMD has nothing to hide behind, so the order is written out: every product is
// followed by at most a fragment read or two and a DMA, and the scheduler is held to that
// order. At 2240 x 28672 x 4096 (231 to 239 us) the products are under way in 61 % of the cycles
// and the card's power holds the clock at 1.85 GHz; the products alone, with nothing read, take
// 187 us. Small tiles are bound by their LDS reads: a 64 x 128 tile's 72 KB a stage take the 570
// cycles that a stage does.
#include <type_traits>
#include <utility>

#include "w8a8_common.h"

namespace ss {
namespace {

template <typename F, int... I>
__device__ __forceinline__ void static_for_impl(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void static_for(F&& f) {
  static_for_impl(f, std::make_integer_sequence<int, N>{});
}

// acc += a b on the matrix core over 32 keys, the accumulator in AGPRs: lane l's sixteen bytes of a are
// keys 16 (l / 32) .. + 15 of channel l % 32 (of b: of token l % 32); its result r is channel
// 8 (r / 4) + 4 (l / 32) + r % 4 of token l % 32. Written as asm because the
// compiler moves accumulators between the register files in every stage. What it therefore
// does not look after: the operands come from LDS reads, which it does wait for; an
// accumulator is touched once in MT NT products; and between the last product and what
// follows the loop stand the waits there.
__device__ __forceinline__ void mfma_acc(i32x16& acc, i32x4 a, i32x4 b) {
  asm volatile("v_mfma_i32_32x32x32_i8 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}

template <typename T, int N>
__device__ __forceinline__ u32x4 as_words(const T (&y)[N]) {
  u32x4 w;
  static_assert(sizeof(y) == 16, "sixteen bytes");
  __builtin_memcpy(&w, y, 16);
  return w;
}

constexpr int kFar = 0x40000000;  // a byte offset past any operand tile (host-checked)

// LDS stages of the tokens and of the channels (rows of 128 bytes) for a tile: as many as its part
// of the LDS holds, the tokens' first, at most six. Of small tiles two workgroups share a CU, so
// that a SIMD has two waves (one has nothing to do while it waits at a barrier: 128 x 28672 x
// 4096 33.5 us with one, 31.9 with two; 333 x 4992 x 2048 9.9 and 9.3).
constexpr int kLdsBytes = 160 * 1024;
constexpr int groups_of(int bm, int bn) { return bm + bn <= 256 ? 2 : 1; }
constexpr int channel_stages(int bm, int bn) {
  int d = 2;
  while (d < 6 && (d + 1) * (bm + bn) * 128 <= kLdsBytes / groups_of(bm, bn)) ++d;
  return d;
}
constexpr int token_stages(int bm, int bn) {
  const int d = channel_stages(bm, bn);
  return d < 6 && ((d + 1) * bm + d * bn) * 128 <= kLdsBytes / groups_of(bm, bn) ? d + 1 : d;
}
constexpr int ring_bytes(int bm, int bn) { return (token_stages(bm, bn) * bm + channel_stages(bm, bn) * bn) * 128; }

// TO int: a K range's sums, for the reduce kernel. ONCE: the only token block, and more than
// kKeptWeights: the weights pass the caches by, and the channel tiles begin at different
// stages, so that those that run at once on an XCD do not all ask for the same lines of the
// tokens (64 x 28672 x 4096 30.8 -> 25.9 us, 256 x 28672 x 4096 44.6 -> 41.6; with
// several token blocks, which share the weights' lines, either is slower: 512 x 4096 x 4096 14.9 us,
// past the caches 18.0, begun apart 16.0).
template <typename TO, int MT, int NT, int WM, int G, bool ONCE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(G, G))) void w8a8_tile_kernel(
    const W8Params p, int per, int ks, int n_tiles, int m_blocks, int band) {
  constexpr int WN = 4 / WM, BM = 32 * MT * WM, BN = 32 * NT * WN;
  constexpr int DX = token_stages(BM, BN), DW = channel_stages(BM, BN);
  constexpr int XB = BM * 128, WB = BN * 128;          // LDS bytes of a stage
  constexpr int NX = BM / 32, NW = BN / 32, ND = NX + NW;  // DMA instructions of a wave and stage
  constexpr int NF = 2 * (MT + NT);                    // fragments of half a stage
  extern __shared__ __attribute__((aligned(16))) char s_dyn[];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ln = lane & 31, kg = lane >> 5;
  const int wm = wave % WM, wn = wave / WM;
  // workgroup -> (K range, channel tile, token block): each XCD (workgroups go round robin over
  // the eight) takes a contiguous eighth of the list. In it bands of `band` token blocks
  // follow each other, in a band the (channel tile, K range) pairs, in those the band's blocks,
  // so that the workgroups that run at once on an XCD share few rows of both operands.
  const int total = ks * n_tiles * m_blocks, per_xcd = (total + 7) >> 3;
  const int item = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per_xcd || item >= total) return;
  const int in_band = band * n_tiles * ks;
  const int mb0 = item / in_band * band, left = item - mb0 * n_tiles * ks;
  const int here = min(band, m_blocks - mb0);
  const int pair = left / here;
  const int zr = pair % ks;
  const int64_t n0 = (int64_t)(pair / ks) * BN;
  const int64_t m0 = (int64_t)(mb0 + left - pair * here) * BM;
  const int rows = (int)min((int64_t)BM, p.m - m0), chans = (int)min((int64_t)BN, p.n - n0);
  const int stages = (p.k + 127) >> 7;
  const int i0 = zr * per, i1 = min(stages, i0 + per);

  // ---- operands: a DMA instruction brings eight LDS rows of 128 bytes; lane l byte 16 (l % 8)
  // of row l / 8, which holds chunk (l % 8) ^ swizzle. Instruction u of wave w: LDS rows
  // 8 (4 u + w) .. + 7. Rows past the end and, in the last stage, chunks past k get an offset
  // outside the descriptors: zeros without an access.
  const i32x4 rx = buffer_words(p.x + m0 * p.x_stride, (uint32_t)((rows - 1) * (int)p.x_stride + p.k));
  const i32x4 rw = buffer_words(p.w + n0 * p.w_stride, (uint32_t)((chans - 1) * (int)p.w_stride + p.k));
  const int row8 = 8 * wave + (lane >> 3);
  const int chunk = 16 * ((lane & 7) ^ tile_swizzle(row8));
  int off[ND];  // channels first
#pragma unroll
  for (int u = 0; u < NW; ++u) off[u] = 32 * u + row8 < chans ? (32 * u + row8) * (int)p.w_stride + chunk : kFar;
#pragma unroll
  for (int u = 0; u < NX; ++u) off[NW + u] = 32 * u + row8 < rows ? (32 * u + row8) * (int)p.x_stride + chunk : kFar;
  const int past = (stages - 1) * 128 + chunk >= p.k ? kFar : 0;  // of the last stage
  const LdsBytes lds = (LdsBytes)s_dyn + wave * 1024;
  // DMAs of one window: the channels of a stage into their slot, then the tokens of a stage
  struct Side {
    int so, add, slot;  // scalar offset, tail offset, LDS slot (bytes)
  } dw = {0, 0, 0}, dx = {0, 0, 0};
  const int apart = ONCE ? (pair / ks) % 16 * (i1 - i0) / 16 : 0;
  auto aim = [&](Side& d, int i, int next_slot) {  // stage i; past the range zeros, which nobody reads
    int at = min(i, stages - 1);
    if constexpr (ONCE)
      if (i < i1) at = i + apart < i1 ? i + apart : i + apart - (i1 - i0);
    d.so = __builtin_amdgcn_readfirstlane(at * 128);
    d.add = i >= i1 ? kFar : at == stages - 1 ? past : 0;
    d.slot = __builtin_amdgcn_readfirstlane(next_slot);
    asm volatile("s_nop 4" : : "s"(d.so), "s"(d.slot));  // VALU-written SGPRs: five wait states before a VMEM reads them
  };
  auto dma = [&](auto uc) __attribute__((always_inline)) {
    constexpr int u = uc;
    if constexpr (u < NW)
      dma_b128<ONCE>(rw, lds + DX * XB + dw.slot + u * 4096, off[u] + dw.add, dw.so);
    else
      dma_b128(rx, lds + dx.slot + (u - NW) * 4096, off[u] + dx.add, dx.so);
  };
  auto after = [](int slot, int bytes, int depth) { return slot + bytes == depth * bytes ? 0 : slot + bytes; };

  // ---- scales, requested first of all: the results wait for nothing then
  constexpr int CL = 16 / sizeof(TO), LR = 32 * NT / CL;  // channels of a lane, lanes of a token in the store
  const int c = lane % LR * CL, c0 = 32 * NT * wn + c;    // from the wave's first channel, and the workgroup's
  float xs[MT];
  u32x4 ws[CL / 4];
  uint32_t bias[CL];
  const BiasReader rb = bias_reader(p, n0, chans);
  if constexpr (!__is_same(TO, int)) {
    const __amdgpu_buffer_rsrc_t rxs = buffer_over(p.x_scale + m0, rows * 4), rws = buffer_over(p.w_scale + n0, chans * 4);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
      xs[mt] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rxs, (32 * (MT * wm + mt) + ln) * 4, 0, 0));
#pragma unroll
    for (int e = 0; e < CL / 4; ++e)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        ws[e][j] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rws, (c0 + 4 * e + j) * 4, 0, 0);
#pragma unroll
    for (int e = 0; e < CL; ++e) bias[e] = bias_bits(rb, c0 + e);
  }

  // fragment of lane (ln, kg): row ln of a 32-row tile; step s of the four of a stage: chunk
  // 2 s + kg. Half h of a stage: steps 2 h and 2 h + 1.
  int f[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) f[s] = ln * 128 + 16 * ((2 * s + kg) ^ tile_swizzle(ln));
  const int xb = wm * MT * 4096, wb = DX * XB + wn * NT * 4096;
  i32x4 a[2][2][NT], b[2][2][MT];  // channels' and tokens' fragments of the half in work and the next
  int rxs = 0, rws = 0;            // slots of the stage that is read
  auto read = [&](auto hc, auto uc) __attribute__((always_inline)) {
    constexpr int h = hc, s = uc / (MT + NT), u = uc % (MT + NT);
    const char* const at = (const char*)s_dyn + f[2 * h + s];
    if constexpr (u < NT)
      a[h][s][u] = *reinterpret_cast<const i32x4*>(at + wb + rws + u * 4096);
    else
      b[h][s][u - NT] = *reinterpret_cast<const i32x4*>(at + xb + rxs + (u - NT) * 4096);
  };

  i32x16 acc[NT][MT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[nt][mt] = i32x16{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};

  // Slots after the P products of each half: window DMAs run from kFree of the first half to
  // the end of the second, the channels' (whose LDS holds fewer stages) in the first P / 2.
  constexpr int P = 2 * MT * NT;
  constexpr int kFree = P * 5 / 8;     // the barrier after which the stage's LDS is free
  constexpr int kLanded = P * 7 / 16;  // of the second half: the next stage has landed
  constexpr int kSpan = 2 * P - kFree, kChan = P / 2, kRead1 = P - kLanded;
  constexpr auto issued = [](int v) constexpr {
    return v <= kChan ? v * NW / kChan : NW + (v - kChan) * NX / (kSpan - kChan);
  };
  // DMAs that may be on their way when stage i + 1 has to have landed, c of window i issued
  constexpr auto newer = [](int c) constexpr {
    const int w = (DW - 2) * ND + NX + c, x = (DX - 2) * ND + c;
    return w < x ? w : x;
  };

  asm volatile("s_nop 4");  // descriptor SGPRs written by VALU before the first asm load
  static_for<DX>([&](auto jc) __attribute__((always_inline)) {
    constexpr int j = jc - DX;  // the window of stage i0 + j
    if constexpr (j + DW >= 0) {
      aim(dw, i0 + j + DW, (j + DW) * WB);
      static_for<NW>(dma);
    }
    aim(dx, i0 + j + DX, (j + DX) * XB);
    static_for<NX>([&](auto uc) __attribute__((always_inline)) { dma(std::integral_constant<int, NW + uc>{}); });
  });
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(newer(ND)) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  static_for<NF>([&](auto uc) __attribute__((always_inline)) { read(std::integral_constant<int, 0>{}, uc); });
  int fx = 0, fw = 0;  // slots that the next window's DMAs fill: those of the stage in work

  for (int i = i0; i < i1; ++i) {
    static_for<P>([&](auto tc) __attribute__((always_inline)) {
      constexpr int t = tc, s = t / (MT * NT), nt = t / MT % NT, mt = t % MT;
      if constexpr (t < kFree)
        static_for<(t + 1) * NF / kFree - t * NF / kFree>([&](auto qc) __attribute__((always_inline)) {
          read(std::integral_constant<int, 1>{}, std::integral_constant<int, t * NF / kFree + qc>{});
        });
      if constexpr (t == kFree) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        aim(dw, i + DW, fw);
        aim(dx, i + DX, fx);
        rxs = fx = after(fx, XB, DX);
        rws = fw = after(fw, WB, DW);
      }
      if constexpr (t >= kFree) {
        constexpr int v = t - kFree;
        static_for<issued(v + 1) - issued(v)>([&](auto qc) __attribute__((always_inline)) {
          dma(std::integral_constant<int, issued(v) + qc>{});
        });
      }
      mfma_acc(acc[nt][mt], a[0][s][nt], b[0][s][mt]);
      __builtin_amdgcn_sched_barrier(0);
    });
    static_for<P>([&](auto tc) __attribute__((always_inline)) {
      constexpr int t = tc, v = t + P - kFree, s = t / (MT * NT), nt = t / MT % NT, mt = t % MT;
      if constexpr (t == kLanded) {
        asm volatile("s_waitcnt vmcnt(%0)" : : "n"(newer(issued(v))) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      }
      if constexpr (t >= kLanded) {
        constexpr int q0 = (t - kLanded) * NF / kRead1, q1 = (t - kLanded + 1) * NF / kRead1;
        static_for<q1 - q0>([&](auto qc) __attribute__((always_inline)) {
          read(std::integral_constant<int, 0>{}, std::integral_constant<int, q0 + qc>{});
        });
      }
      static_for<issued(v + 1) - issued(v)>([&](auto qc) __attribute__((always_inline)) {
        dma(std::integral_constant<int, issued(v) + qc>{});
      });
      mfma_acc(acc[nt][mt], a[1][s][nt], b[1][s][mt]);
      __builtin_amdgcn_sched_barrier(0);
    });
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // no DMA and no read of the LDS is on its way,
  __builtin_amdgcn_s_barrier();                                // of any wave
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");           // and the last products have landed

  // ---- results: 32 tokens at a time through the wave's own part of the LDS (as sum * x_scale, in
  // fp32), so that the lanes hold consecutive channels and a store writes rows of the wave's
  // 32 NT channels
  constexpr int RS = NT * 128 + 16;  // bytes of a token there
  static_assert(4 * 32 * RS <= ring_bytes(BM, BN), "the sums fit where the operands were");
  char* const turn = s_dyn + wave * 32 * RS;
  TO* const out = (TO*)p.out + (__is_same(TO, int) ? (int64_t)zr * p.m * p.o_stride : 0);
  // in 16-byte pieces, through a descriptor over the wave's rows: what lies outside it is not
  // written
  const bool pieces = p.n % CL == 0 && p.o_stride % CL == 0 && p.o_stride <= (1 << 20) && ((uintptr_t)p.out & 15) == 0;
  const int left_rows = rows - 32 * MT * wm, left_chans = chans - 32 * NT * wn;
  const int row_bytes = (int)p.o_stride * (int)sizeof(TO);
  const uint32_t bytes = left_rows > 0 && left_chans > 0 ? (min(left_rows, 32 * MT) - 1) * row_bytes +
                                                               min(left_chans, 32 * NT) * (int)sizeof(TO)
                                                         : 0;
  const __amdgpu_buffer_rsrc_t ro = __builtin_amdgcn_make_buffer_rsrc(
      out + (m0 + 32 * MT * wm) * p.o_stride + n0 + 32 * NT * wn, (short)0, (int)bytes, 0x00020000);
  const int o_at = c < left_chans ? lane / LR * row_bytes + c * (int)sizeof(TO) : kFar;
  int o_row = 0;  // bytes from the wave's first row
  float biasf[CL];
  if constexpr (!__is_same(TO, int)) {
#pragma unroll
    for (int e = 0; e < CL; ++e) biasf[e] = bias_value(rb, bias[e]);
  }
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      asm volatile("" : "+a"(acc[nt][mt]));  // read behind the waits above
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        u32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int sum = acc[nt][mt][4 * g + e];
          if constexpr (__is_same(TO, int))
            v[e] = (uint32_t)sum;
          else
            v[e] = __builtin_bit_cast(uint32_t, (float)sum * xs[mt]);
        }
        store16(turn + ln * RS + (32 * nt + 8 * g + 4 * kg) * 4, v);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    auto results = [&](int r, TO (&y)[CL]) __attribute__((always_inline)) {
      u32x4 v[CL / 4];
#pragma unroll
      for (int h = 0; h < CL / 4; ++h) v[h] = load16(turn + r * RS + (c + 4 * h) * 4);
      if constexpr (__is_same(TO, int)) {
#pragma unroll
        for (int e = 0; e < CL; ++e) y[e] = (int)v[0][e];
      } else {
        float y32[CL];
#pragma unroll
        for (int e = 0; e < CL; ++e)
          y32[e] = fmaf(__builtin_bit_cast(float, (uint32_t)v[e / 4][e % 4]),
                        __builtin_bit_cast(float, (uint32_t)ws[e / 4][e % 4]), biasf[e]);
        pack_results<CL>(y, y32);
      }
    };
    if (pieces) {
#pragma unroll
      for (int q = 0; q < LR / 2; ++q) {
        TO y[CL];
        results(q * (64 / LR) + lane / LR, y);
        __builtin_amdgcn_raw_buffer_store_b128(as_words(y), ro, o_at + o_row, 0, 0);
        o_row += 64 / LR * row_bytes;
      }
    } else {
      // at any alignment (global accesses need none on this target), a row's last ones one by one
#pragma unroll 2
      for (int r = lane / LR; r < 32; r += 64 / LR) {
        TO y[CL];
        results(r, y);
        if (32 * mt + r >= left_rows || c >= left_chans) continue;
        TO* const o = out + (m0 + 32 * (MT * wm + mt) + r) * p.o_stride + n0 + c0;
        if (c + CL <= left_chans) {
          __builtin_memcpy(o, y, sizeof(y));
        } else {
#pragma unroll
          for (int e = 0; e < CL; ++e)
            if (c + e < left_chans) o[e] = y[e];
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the next tokens are written
  }
}

// The sums of ks K ranges added, scaled and rounded: a thread four channels of a token. Every load
// that does not depend on the number of ranges is on its way before the first is waited for, and
// four ranges' at a time (past the last: outside the descriptor, zeros).
template <typename TO, bool VEC>
__global__ __launch_bounds__(256) void w8a8_reduce_kernel(const W8Params p, const int* __restrict__ part, int ks) {
  const uint32_t quads = (uint32_t)((p.n + 3) >> 2), total = (uint32_t)p.m * quads;  // m n below 2^29
  const int plane = (int)(p.m * p.n) * 4;  // bytes; ks of them below 2^31
  const __amdgpu_buffer_rsrc_t rp = buffer_over(part, (uint32_t)(ks * plane));
  const __amdgpu_buffer_rsrc_t rws = buffer_over(p.w_scale, (uint32_t)(p.n * 4));
  const BiasReader rb = bias_reader(p, 0, (int)p.n);
  for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < total; i += gridDim.x * 256) {
    const int m = (int)(i / quads), n = 4 * (int)(i - m * quads);
    const int at = (m * (int)p.n + n) * 4;
    const float xs = p.x_scale[m];
    uint32_t ws[4], bias[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      ws[e] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rws, (n + e) * 4, 0, 0);
      bias[e] = bias_bits(rb, n + e);
    }
    i32x4 sum = {0, 0, 0, 0};
    for (int z = 0; z < ks; z += 4) {
      i32x4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int off = z + j < ks ? at + (z + j) * plane : -16;
        if constexpr (VEC) {
          v[j] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rp, off, 0, 0));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[j][e] = __builtin_amdgcn_raw_buffer_load_b32(rp, off + 4 * e, 0, 0);
        }
      }
      sum += (v[0] + v[1]) + (v[2] + v[3]);
    }
    TO* const o = (TO*)p.out + m * p.o_stride + n;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (VEC || n + e < p.n)
        o[e] = (TO)scaled(sum[e], xs, __builtin_bit_cast(float, ws[e]), bias_value(rb, bias[e]));
  }
}

template <typename TO, int MT, int NT, int WM, bool ONCE>
int launch_tile(const W8Params& p, const TilePlan& pl, hipStream_t stream) {
  constexpr int bm = 32 * MT * WM, bn = 32 * NT * (4 / WM), lds = ring_bytes(bm, bn);
  auto kern = w8a8_tile_kernel<TO, MT, NT, WM, groups_of(bm, bn), ONCE>;
  static std::atomic<uint64_t> done{0};
  if (const int st = reserve_lds((const void*)kern, lds, done); st != SS_OK) return st;
  // bands of at most 8 token blocks, of one size where they can be
  const int bands = (pl.m_blocks + 7) / 8, band = (pl.m_blocks + bands - 1) / bands;
  const int64_t grid = ((int64_t)pl.ks * pl.n_tiles * pl.m_blocks + 7) / 8 * 8;
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(256), lds, stream, p, pl.per, pl.ks, pl.n_tiles, pl.m_blocks,
                     band);
  return ss_host::launch_status("w8a8 gemm (tile)");
}

// A tile's tokens and channels, and its waves' 32 x 32 tiles (MT, NT) and grid (WM x 4 / WM)
#define W8A8_TILES(X) \
  X(256, 256, 4, 4, 2) X(224, 256, 7, 2, 1) X(192, 256, 3, 4, 2) X(160, 256, 5, 2, 1) X(128, 256, 2, 4, 2) \
  X(256, 128, 4, 2, 2) X(192, 128, 3, 2, 2) X(128, 128, 2, 2, 2) \
  X(96, 128, 3, 1, 1) X(64, 128, 2, 1, 1)

inline bool read_once(int64_t m_blocks, int64_t ks, int64_t n, int64_t k) {
  return m_blocks == 1 && ks == 1 && n * k > kKeptWeights;
}

template <typename TO>
int launch_tile_typed(const W8Params& p, const TilePlan& pl, hipStream_t stream) {
#define W8A8_LAUNCH(BM, BN, MT, NT, WM) \
  if (pl.bm == BM && pl.bn == BN) {                                                             \
    if constexpr (!__is_same(TO, int))                                                         \
      if (pl.once) return launch_tile<TO, MT, NT, WM, true>(p, pl, stream); \
    return launch_tile<TO, MT, NT, WM, false>(p, pl, stream);                                  \
  }
  W8A8_TILES(W8A8_LAUNCH)
#undef W8A8_LAUNCH
  ss_host::set_error("w8a8 gemm: tile of %d x %d", pl.bm, pl.bn);
  return SS_ERR_UNSUPPORTED;
}

template <typename TO>
int launch_reduce(const W8Params& p, const int* part, int ks, hipStream_t stream) {
  const int64_t blocks = (p.m * ((p.n + 3) / 4) + 255) / 256, cap = (int64_t)ss_host::device_cu_count() * 8;
  const dim3 grid((unsigned)(blocks < cap ? blocks : cap));
  if (p.n % 4 == 0)
    hipLaunchKernelGGL((w8a8_reduce_kernel<TO, true>), grid, dim3(256), 0, stream, p, part, ks);
  else
    hipLaunchKernelGGL((w8a8_reduce_kernel<TO, false>), grid, dim3(256), 0, stream, p, part, ks);
  return ss_host::launch_status("w8a8 gemm (reduce)");
}

}  // namespace

// The tile and K split of least estimated time (us), fitted to the times of 4200 calls (tiles and
// splits of 290 shapes, 1 to 2240 tokens, 0.3 to 120 million weights); 7 % off on average over 5025
// calls of the kernel as it is, but 30 % too low for one token block of more than kKeptWeights,
// whose term was put in by hand (64 x 28672 x 4096 17 us, takes 25; among those the choice is
// mostly right, at worst 96 x 57344 x 8192 108 us in tiles of 96 x 128, 80 in 128 x 256): what a
// stage takes of a round of workgroups, the results of each round, the operands' way into the
// LDS, the memory's share, and for a split the sums' way out and back and the launch that adds
// them. (2240 x 4096 x 14336: 224 tiles of 160 x 256 117 us, 144 of 256 x 256 140; 197 x 4096 x
// 14336: four ranges of 128 x 128 tiles 24 us, whole rows 45.)
double plan_w8a8_tile(TilePlan& pl, int64_t m, int64_t n, int64_t k, bool may_split) {
#define W8A8_SIZE(BM, BN, MT, NT, WM) {BM, BN},
  static const int kTiles[][2] = {W8A8_TILES(W8A8_SIZE)};
#undef W8A8_SIZE
  const int64_t stages = (k + 127) / 128, cus = ss_host::device_cu_count();
  double best = 1e30;
  for (const auto& t : kTiles) {
    const int64_t n_tiles = (n + t[1] - 1) / t[1], m_blocks = (m + t[0] - 1) / t[0];
    const int64_t fit = groups_of(t[0], t[1]);
    if (n_tiles * m_blocks > kMostGroups) continue;
    for (int64_t ks = 1; ks <= (may_split ? 14 : 1); ks += ks < 4 ? 1 : 2) {
      const int64_t per = (stages + ks - 1) / ks, groups = ks * n_tiles * m_blocks;
      // a split of at least four stages each, for at most two rounds and a bit
      if (ks > 1 && (per < 4 || groups > 600 || ks * m * n * 4 >= ((int64_t)1 << 31))) break;
      if ((stages + per - 1) / per != ks) continue;
      const double rounds = (double)((groups + cus - 1) / cus), area = t[0] * t[1] / 65536.0, edge = t[0] + t[1];
      const double turns = (double)((groups + fit * cus - 1) / (fit * cus));
      double us = 3.13 + turns * per * 0.0844 + rounds * (per * (0.662 * area + 0.128 * edge / 512) + 0.21 + 6.33 * area) +
                  groups * per * edge * 128 * 1.79e-8 + n * k * 4.2e-8 + m * n * 2.96e-7;
      const bool once = read_once(m_blocks, ks, n, k);
      if (once) us -= n * k * 2e-8;
      if (ks > 1) us += 2.03 + ks * m * n * 4 * 2.79e-7;
      if (us < best) {
        best = us;
        pl = {t[0], t[1], (int)ks, (int)per, (int)n_tiles, (int)m_blocks, once};
      }
    }
  }
  return best;
}

int launch_w8a8_tile(const W8Params& p, const TilePlan& pl, int out_dtype, int* part, hipStream_t stream) {
  if (pl.ks > 1) {
    W8Params q = p;
    q.out = part;
    q.o_stride = p.n;
    const int st = launch_tile_typed<int>(q, pl, stream);
    if (st != SS_OK) return st;
    if (out_dtype == SS_DTYPE_BF16) return launch_reduce<bf16_t>(p, part, pl.ks, stream);
    if (out_dtype == SS_DTYPE_F16) return launch_reduce<f16_t>(p, part, pl.ks, stream);
    return launch_reduce<float>(p, part, pl.ks, stream);
  }
  if (out_dtype == SS_DTYPE_BF16) return launch_tile_typed<bf16_t>(p, pl, stream);
  if (out_dtype == SS_DTYPE_F16) return launch_tile_typed<f16_t>(p, pl, stream);
  return launch_tile_typed<float>(p, pl, stream);
}

}  // namespace ss
