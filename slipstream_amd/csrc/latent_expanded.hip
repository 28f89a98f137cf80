// Attention over latents, expanded form, on the matrix cores: bf16 and fp16, keys of 128 values of each
// head and 64 shared ones, values of 128.
//
// A workgroup takes 32 NW query tokens of one head and walks the keys in tiles of 64, a wave 32 rows:
//   S^T = K Q^T     two products of 32 x 32 x 192, the queries in registers
//   softmax         fp32; a row's keys lie in two lanes, so a maximum is one exchange
//   O^T += V^T P^T  the scores' layout is the operand's: probabilities stay in registers
// Keys (the heads' and the shared parts) and values come by DMA into rings in the LDS, whose 16-byte
// chunks are swizzled as in latent_mma.h. A step runs the scores of tile t + 1, then the outputs of tile t, with the
// softmax of either written between their products; two waves a SIMD.
// 4 chunks of 512 tokens over up to 4096, 128 heads: 445 to 472 us, 890 to 950 TFLOP/s; a step of 256 tokens and 64 keys
// takes 2.2 us, its products 1.4 of them at the 1.9 GHz that the card's power leaves. A turn of 77 tokens over 512, 16
// heads: 14.0 us, ten steps of 1 after 3.5 us of start; two groups of waves with half of the keys each took 0.5 us less.
#include "latent_mma.h"

namespace ss {
namespace {

constexpr int kNope = 128, kValue = 128;

// D: depth of the rings
template <int NW_, int D_>
struct LatExp {
  static constexpr int NW = NW_, D = D_, ROWS = 32 * NW, KT = 64;
  static constexpr int KP = KT * 2 * kNope, RP = KT * 2 * kRopeDim, VP = KT * 2 * kValue;  // bytes of a tile's planes
  static constexpr int kR = D * KP, kV = kR + D * RP, LDS = kV + D * VP;
  static constexpr int NK = 16 / NW, NR = 8 / NW;  // DMA instructions of a wave and tile: a head's keys (or values), shared keys
  static_assert(LDS <= 160 * 1024, "fits");
};

template <typename T, typename C>
__global__ __launch_bounds__(64 * C::NW) __attribute__((amdgpu_waves_per_eu(C::NW == 8 ? 2 : 1, C::NW == 8 ? 2 : 1))) void
latent_expanded_kernel(const LatentParams p) {
  extern __shared__ __attribute__((aligned(1024))) char s_exp[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, h = lane >> 5;
  // Workgroups go round robin over the eight XCDs, and a sequence's tiles of a head follow each other on one of
  // them, whose L2 then serves their keys. The sequences of the most keys come first, so that no long tile begins
  // when the others end (in the order of the batch: 4 chunks of 512 over up to 4096, 128 heads 540 us, then 464); of more than
  // 64 sequences each 64 are ordered. A sequence's first tile is the number of those of the ones before it.
  const int slot = blockIdx.x >> 3, groups = (p.heads + 7) >> 3;
  int left = slot, b = -1, count = 0, start = 0, head = 0, tile = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    int c = 0, s = 0, k = 0;
    if (b0 + lane < p.batch) {
      int first, length;
      latent_queries(p, b0 + lane, c, s);
      k = latent_keys(p, b0 + lane, first, length);
    }
    const int mine = (c + C::ROWS - 1) / C::ROWS;
    int before = 0, all = 0;
    for (int i = 0; i < min(64, p.batch - b0); ++i) {
      const int ki = __builtin_amdgcn_readlane(k, i), ti = __builtin_amdgcn_readlane(mine, i);
      before += ki > k || (ki == k && i < lane) ? ti : 0;
      all += ti;
    }
    if (left >= all * groups) {
      left -= all * groups;
      continue;
    }
    const int i = __builtin_ctzll(__ballot(left >= before * groups && left < (before + mine) * groups));
    b = b0 + i;
    count = __builtin_amdgcn_readlane(c, i);
    start = __builtin_amdgcn_readlane(s, i);
    const int tiles = __builtin_amdgcn_readlane(mine, i);
    left -= __builtin_amdgcn_readlane(before, i) * groups;
    head = 8 * (left / tiles) + (blockIdx.x & 7);
    tile = tiles - 1 - left % tiles;  // the last ones, which see the most keys, first
    break;
  }
  if (b < 0 || head >= p.heads) return;
  head = __builtin_amdgcn_readfirstlane(head), tile = __builtin_amdgcn_readfirstlane(tile);
  int k0, length;
  const int keys = latent_keys(p, b, k0, length);
  const int tok0 = tile * C::ROWS;
  const int kv_end = max(0, min(keys, keys - count + min(count, tok0 + C::ROWS)));
  const int tend = (kv_end + C::KT - 1) / C::KT;

  // ---- the tiles' way into the LDS: a DMA instruction brings four keys or values of a head, or eight shared
  // keys. One descriptor a plane and tile, which ends with the keys that are there.
  const uint32_t lds = lds_address(s_exp);
  const int kv_bytes = (int)(p.kv_s0 * 2), r_bytes = (int)(p.k_st * 2);
  const uint64_t kv0 = (uint64_t)p.kv + 2 * (k0 * p.kv_s0 + head * p.kv_s1), r0 = (uint64_t)p.k_rope + 2 * (k0 * p.k_st);
  // a lane's part of the offsets; the bits of the swizzle that an instruction's first row has are flipped in
  // the chunk's part (dma4, dma8)
  const int chunk4 = 16 * ((lane & 15) ^ (lane >> 4)), lane4 = (lane >> 4) * kv_bytes;
  const int chunk8 = 16 * ((lane & 7) ^ (lane >> 4)), lane8 = (lane >> 3) * r_bytes;
  auto plane = [&](uint64_t base, int t, int bytes, int width) {
    const int live = min(C::KT, kv_end - t * C::KT);
    const bool there = t >= 0 && live > 0;
    const uint64_t at = there ? base + (uint64_t)(t * C::KT) * (uint32_t)bytes : base;
    return i32x4{__builtin_amdgcn_readfirstlane((int)(uint32_t)at),
                 __builtin_amdgcn_readfirstlane((int)(uint32_t)(at >> 32) & 0xFFFF),
                 __builtin_amdgcn_readfirstlane(there ? (live - 1) * bytes + width : 0), 0x00020000};
  };
  auto dma4 = [&](i32x4 rs, uint32_t to, int u) __attribute__((always_inline)) {
    const int row = 4 * (C::NK * wave + u);
    dma_b128(rs, (LdsBytes)(uintptr_t)(to + row * 256), (chunk4 ^ 16 * lat_swizzle(row)) + (lane4 + row * kv_bytes), 0);
  };
  auto dma8 = [&](i32x4 rs, uint32_t to, int u) __attribute__((always_inline)) {
    const int row = 8 * (C::NR * wave + u);
    dma_b128(rs, (LdsBytes)(uintptr_t)(to + row * 128), (chunk8 ^ 16 * tile_swizzle(row)) + (lane8 + row * r_bytes), 0);
  };
  // always as many instructions, so that the waits can count them
  auto issue_keys = [&](int j, int slot) __attribute__((always_inline)) {
    const i32x4 rk = plane(kv0, j, kv_bytes, 2 * kNope), rr = plane(r0, j, r_bytes, 2 * kRopeDim);
    asm volatile("s_nop 4" : : "s"(rk), "s"(rr));  // SGPRs that a VALU wrote: five wait states before a VMEM
#pragma unroll
    for (int u = 0; u < C::NK; ++u) dma4(rk, lds + slot * C::KP, u);
#pragma unroll
    for (int u = 0; u < C::NR; ++u) dma8(rr, lds + C::kR + slot * C::RP, u);
  };
  auto issue_values = [&](int j, int slot) __attribute__((always_inline)) {
    const i32x4 rv = plane(kv0 + 2 * kNope, j, kv_bytes, 2 * kValue);
    asm volatile("s_nop 4" : : "s"(rv));
#pragma unroll
    for (int u = 0; u < C::NK; ++u) dma4(rv, lds + C::kV + slot * C::VP, u);
  };
  issue_keys(0, 0);

  // ---- the wave's rows
  const int tok = tok0 + 32 * wave + n;
  const bool ok = tok < count;
  const int lim = ok ? min(kv_end, keys - count + tok + 1) : kv_end;
  int least = lim, most = ok ? lim : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    least = min(least, __shfl_xor(least, o));
    most = max(most, __shfl_xor(most, o));
  }
  least = __builtin_amdgcn_readfirstlane(least);
  most = __builtin_amdgcn_readfirstlane(most);
  constexpr int NQ = (kNope + kRopeDim) / 16;
  u32x4 qop[NQ];
  {
    // a lane without a row reads the tile's first one and takes zeros; a negative scale is the query's sign
    const T* const q = (const T*)p.q + (start + (ok ? tok : tok0)) * p.q_st + head * p.q_sh + 8 * h;
    const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u, keep = ok ? ~0u : 0u;
#pragma unroll
    for (int s = 0; s < NQ; ++s)
      qop[s] = (load16(q + 16 * s) ^ u32x4{flip, flip, flip, flip}) & u32x4{keep, keep, keep, keep};
  }
  static_for<C::D - 1>([&](auto j) __attribute__((always_inline)) {
    constexpr int g = decltype(j)::value;
    issue_keys(g + 1, g + 1);
    issue_values(g, g);
  });
  const float cscale = fabsf(p.scale_log2);

  f32x16 acc[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[dt][e] = 0.f;
  float m = kNegBig, l = 0.f;

  const uint32_t kaddr = lds + n * 256 + 16 * (h ^ lat_swizzle(n));
  const uint32_t raddr = lds + C::kR + n * 128 + 16 * (h ^ tile_swizzle(n));
  const int sl = lane & 15, vrow = 4 * h + (sl >> 2), quad = 2 * ((lane >> 4) & 1) + ((sl & 3) >> 1);
  const uint32_t vaddr = lds + C::kV + vrow * 256 + 8 * (sl & 1) + 16 * ((4 * quad) ^ lat_swizzle(vrow));

  // A step of a wave in two parts: the scores of tile t + 1, then the outputs of tile t. A tile's softmax is written
  // between the products from the outputs of the tile before to its own, a few instructions that do not wait for each
  // other at a time: at two waves a SIMD one that waits for the instruction before it costs twice its own time.
  constexpr int AHEAD = 4;
  u32x4 vring[AHEAD];
  uint32_t pk[16], va = 0;
  float alpha = 1.f, mn = 0.f, sum[2], top[4], ex[2][2], fx[2][2];
  bool grew = false;
  // part i of the softmax of the scores x: the maximum (0 .. 6), the exponents of pair i - 7, the probabilities of
  // the pair before, the rounding of the one before that and the sum, of the rounded ones, of the one before that (a
  // part later than their rounding: in the same part, which waits for it, 453 us and not 445; of the unrounded ones 437),
  // and the row's new state
  constexpr int PARTS = 27, EARLY = 10;  // EARLY parts among the outputs of the tile before
  auto part = [&](auto ic, f32x16 (&x)[2]) __attribute__((always_inline)) {
    constexpr int i = ic;
    if constexpr (i < 4) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const f32x16& v = x[u >> 1];
        constexpr int at = i == 0 ? 0 : 2 * i + 1;  // three values, then two, two and one
        const int e = 8 * (u & 1) + at;
        top[u] = i == 0 ? max3(v[e], v[e + 1], v[e + 2]) : i < 3 ? max3(top[u], v[e], v[e + 1]) : max3(top[u], v[e], v[e]);
      }
    } else if constexpr (i == 4) {
      top[0] = max3(top[0], top[1], top[2]);
      top[0] = max3(top[0], top[3], top[3]);
    } else if constexpr (i == 5) {
      const uint32_t tb = __builtin_bit_cast(uint32_t, top[0]);
      auto sw = __builtin_amdgcn_permlane32_swap(tb, tb, false, false);
      top[0] = max3(__builtin_bit_cast(float, (uint32_t)sw[0]), __builtin_bit_cast(float, (uint32_t)sw[1]), kNegBig);
      top[0] = fmaxf(m, fmaf(top[0], cscale, -kHeadroom<T>));
    } else if constexpr (i == 6) {
      grew = __any(top[0] > m + kSlack);
      mn = grew ? top[0] : m;
      sum[0] = sum[1] = 0.f;
    } else if constexpr (i < PARTS - 1) {
      constexpr int q = i - 7;
      if constexpr (q >= 3) {
        constexpr int d = q - 3;
        sum[0] += Elem<T>::lo(pk[d]), sum[1] += Elem<T>::hi(pk[d]);
        asm volatile("" : "+v"(sum[0]), "+v"(sum[1]));  // made here
      }
      if constexpr (q >= 2 && q <= 17) {
        constexpr int d = q - 2;
        pk[d] = Elem<T>::pack2(ex[d & 1][0], ex[d & 1][1]);
        asm volatile("" : "+v"(pk[d]));
      }
      if constexpr (q >= 1 && q <= 16) {
        constexpr int d = q - 1;
        ex[d & 1][0] = fast_exp2(fx[d & 1][0]), ex[d & 1][1] = fast_exp2(fx[d & 1][1]);
        asm volatile("" : "+v"(ex[d & 1][0]), "+v"(ex[d & 1][1]));
      }
      if constexpr (q < 16) {
        constexpr int e = 2 * (q & 7);
        fx[q & 1][0] = fmaf(x[q >> 3][e], cscale, -mn), fx[q & 1][1] = fmaf(x[q >> 3][e + 1], cscale, -mn);
        asm volatile("" : "+v"(fx[q & 1][0]), "+v"(fx[q & 1][1]));
      }
    } else {
      alpha = fast_exp2(m - mn);
      l = fmaf(l, alpha, sum[0] + sum[1]);
      m = mn;
    }
  };
  auto vread = [&](auto ic) __attribute__((always_inline)) {  // output product i: 16 keys of i / 4, values of i % 4
    constexpr int i = ic, s = i >> 2, dt = i & 3;
    if constexpr (i < 16) {
      const uint32_t at = va ^ (16 * dt);
      vring[i % AHEAD] = lds_keys(at + 16 * s * 256, (at ^ 64) + (16 * s + 8) * 256);
    }
  };
  auto masked = [&](int t, f32x16 (&x)[2]) __attribute__((always_inline)) {
    if (t * C::KT + C::KT > least) {
      asm volatile("s_nop 15\n\ts_nop 7" : "+v"(x[0]), "+v"(x[1]));  // the last products are through
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (t * C::KT + 32 * y + 8 * (e >> 2) + 4 * h + (e & 3) >= lim) x[y][e] = -__builtin_inff();
    }
  };
  // the scores of the tile in key slot ks into `next`, with the later parts of `cur`'s softmax (OUT)
  auto scores = [&](auto outc, int ks, f32x16 (&cur)[2], f32x16 (&next)[2]) __attribute__((always_inline)) {
    constexpr bool OUT = decltype(outc)::value;
    u32x4 kring[AHEAD];
    const uint32_t ka = kaddr + ks * C::KP, ra = raddr + ks * C::RP;
    auto kread = [&](auto jc) __attribute__((always_inline)) {  // score product j: 32 keys x = j % 2, values of j / 2
      constexpr int j = jc, x = j & 1, s = j >> 1;
      if constexpr (s < kNope / 16)
        kring[j % AHEAD] = lds_word((ka ^ (32 * s)) + x * 8192);
      else if constexpr (s < NQ)
        kring[j % AHEAD] = lds_word((ra ^ (32 * (s - kNope / 16))) + x * 4096);
    };
    static_for<AHEAD>(kread);
    __builtin_amdgcn_sched_barrier(0);
    static_for<2 * NQ>([&](auto jc) __attribute__((always_inline)) {
      constexpr int j = jc, x = j & 1, s = j >> 1;
      mfma32_sum<T, s == 0>(next[x], kring[j % AHEAD], qop[s]);
      kread(std::integral_constant<int, j + AHEAD>{});
      if constexpr (OUT) {
        constexpr int from = EARLY + j * (PARTS - EARLY) / (2 * NQ), to = EARLY + (j + 1) * (PARTS - EARLY) / (2 * NQ);
        static_for<to - from>([&](auto qc) __attribute__((always_inline)) { part(std::integral_constant<int, from + qc>{}, cur); });
        if constexpr (j >= 2 * NQ - AHEAD) vread(std::integral_constant<int, j - (2 * NQ - AHEAD)>{});
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  // the outputs of tile t, with the first parts of the softmax of `next`, the scores of tile t + 1
  auto outputs = [&](int t, f32x16 (&next)[2]) __attribute__((always_inline)) {
    if (grew) {
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) acc[dt] *= alpha;
    }
    masked(t + 1, next);
    // what a VALU wrote is read by a product two wait states later at the earliest
    asm volatile("s_nop 1" : "+v"(acc[0]), "+v"(acc[1]), "+v"(acc[2]), "+v"(acc[3]));
    __builtin_amdgcn_sched_barrier(0);
    static_for<16>([&](auto ic) __attribute__((always_inline)) {
      constexpr int i = ic, s = i >> 2, dt = i & 3;
      mfma32_sum<T, false>(acc[dt], vring[i % AHEAD], u32x4{pk[4 * s], pk[4 * s + 1], pk[4 * s + 2], pk[4 * s + 3]});
      vread(std::integral_constant<int, i + AHEAD>{});
      if constexpr (i == 2) asm volatile("" : "+v"(next[0]), "+v"(next[1]));  // the scores are through by now
      constexpr int from = i < 3 ? 0 : (i - 3) * EARLY / 13, to = i < 3 ? 0 : (i - 2) * EARLY / 13;
      static_for<to - from>([&](auto qc) __attribute__((always_inline)) { part(std::integral_constant<int, from + qc>{}, next); });
      __builtin_amdgcn_sched_barrier(0);
    });
  };

  constexpr int PER = 2 * C::NK + C::NR;  // DMA instructions of a step
  f32x16 sa[2], sb[2];
  if (tend > 0) {
    wait_dma<(C::D - 1) * PER>();
    __syncthreads();
    if (most > 0) {
      scores(std::false_type{}, 0, sb, sa);
      asm volatile("s_nop 15\n\ts_nop 7" : "+v"(sa[0]), "+v"(sa[1]));  // the last products are through
      masked(0, sa);
      static_for<EARLY>([&](auto qc) __attribute__((always_inline)) { part(qc, sa); });
    }
    int slot = 0;  // of tile t
    // Keys of t + 1 and values of t have landed; tile t's keys and tile t - 1's values are done with: tile t + D's keys
    // and t + D - 1's values take their places. Waves whose rows see nothing of a tile do nothing else. (With half of
    // the waves half a step behind the others, so that a SIMD's two are not at the same part: no faster.)
    auto turn = [&](int t, f32x16 (&cur)[2], f32x16 (&next)[2]) __attribute__((always_inline)) {
      wait_dma<(C::D - 2) * PER>();
      __syncthreads();
      issue_keys(t + C::D, slot);
      issue_values(t + C::D - 1, slot == 0 ? C::D - 1 : slot - 1);
      const int after = slot + 1 == C::D ? 0 : slot + 1;
      va = vaddr + slot * C::VP;
      if (t * C::KT < most) {
        scores(std::true_type{}, after, cur, next);
        outputs(t, next);
      }
      slot = after;
    };
    for (int t = 0; t < tend; t += 2) {
      turn(t, sa, sb);
      if (t + 1 < tend) turn(t + 1, sb, sa);
    }
  }
  wait_dma<0>();  // no DMA may land after the workgroup has ended
  asm volatile("s_nop 15\n\ts_nop 7" : "+v"(acc[0]), "+v"(acc[1]), "+v"(acc[2]), "+v"(acc[3]));

  const uint32_t lb = __builtin_bit_cast(uint32_t, l);
  auto ls = __builtin_amdgcn_permlane32_swap(lb, lb, false, false);
  const float total = __builtin_bit_cast(float, (uint32_t)ls[0]) + __builtin_bit_cast(float, (uint32_t)ls[1]);
  const float inv = total == 0.f ? 0.f : 1.f / total;
  T* const o = (T*)p.out + (start + tok) * p.o_st + head * p.o_sh;
  // result r of output tile dt: value 8 (dt + 4 (r / 4)) + 4 h + r % 4 of row n. The halves of two chunks
  // change places so that a lane holds one whole.
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int x = 0; x < 4; x += 2) {
      uint32_t w[2][2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t even = Elem<T>::pack2(acc[dt][4 * x + 2 * e] * inv, acc[dt][4 * x + 2 * e + 1] * inv);
        const uint32_t odd = Elem<T>::pack2(acc[dt][4 * x + 4 + 2 * e] * inv, acc[dt][4 * x + 5 + 2 * e] * inv);
        auto sw = __builtin_amdgcn_permlane32_swap(even, odd, false, false);
        w[e][0] = sw[0], w[e][1] = sw[1];
      }
      if (ok) {
        const u32x4 y = {w[0][0], w[1][0], w[0][1], w[1][1]};
        __builtin_memcpy(o + 8 * (dt + 4 * (x + h)), &y, 16);
      }
    }
}

template <typename T, typename C>
int launch_rows(const LatentParams& p, hipStream_t stream) {
  const int64_t tiles = (p.total + C::ROWS - 1) / C::ROWS + p.batch, slots = (p.heads + 7) / 8;
  if (tiles * slots * 8 * 64 * C::NW >= (1ll << 32)) {
    ss_host::set_error("latent attention (expanded): %d tokens of %d heads are more than one launch holds", p.total, p.heads);
    return SS_ERR_UNSUPPORTED;
  }
  auto kern = latent_expanded_kernel<T, C>;
  static std::atomic<uint64_t> done{0};
  if (const int st = reserve_lds((const void*)kern, C::LDS, done); st != SS_OK) return st;
  hipLaunchKernelGGL(kern, dim3((unsigned)(tiles * slots * 8)), dim3(64 * C::NW), C::LDS, stream, p);
  return ss_host::launch_status("latent attention (expanded)");
}

// Eight waves share a tile's keys where there are enough tokens for a workgroup a CU; else four or two,
// whose workgroups are more.
template <typename T>
int launch_for(const LatentParams& p, hipStream_t stream) {
  const int64_t cus = ss_host::device_cu_count();
  if ((int64_t)p.total * p.heads >= 256 * cus) return launch_rows<T, LatExp<8, 3>>(p, stream);
  if ((int64_t)p.total * p.heads >= 128 * cus) return launch_rows<T, LatExp<4, 2>>(p, stream);
  return launch_rows<T, LatExp<2, 2>>(p, stream);
}

}  // namespace

bool latent_expanded_takes(const LatentParams& p, int dtype) {
  if (dtype != SS_DTYPE_BF16 && dtype != SS_DTYPE_F16) return false;
  if (p.key_dim != kNope || p.rope_dim != kRopeDim || p.value_dim != kValue || p.scale_log2 == 0.f) return false;
  for (int64_t s : {p.q_st, p.q_sh, p.kv_s0, p.kv_s1, p.k_st})
    if (s % 8) return false;
  return ((uintptr_t)p.q | (uintptr_t)p.kv | (uintptr_t)p.k_rope) % 16 == 0 && p.kv_s0 >= kNope + kValue &&
         p.kv_s0 < (1 << 23) && p.k_st >= kRopeDim && p.k_st < (1 << 23);
}

int launch_latent_expanded(const LatentParams& p, int dtype, hipStream_t stream) {
  return dtype == SS_DTYPE_BF16 ? launch_for<bf16_t>(p, stream) : launch_for<f16_t>(p, stream);
}

}  // namespace ss
