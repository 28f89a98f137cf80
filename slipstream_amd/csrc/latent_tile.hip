// Attention over latents, absorbed form, on the matrix cores: bf16 and fp16, latents of 256 or 512
// values, rotated keys of 64, pages of 8, 16, 32, ... tokens.
//
// All heads share a sequence's keys, so the query rows of a (sequence, few tokens) are its tokens' heads,
// and a tile of keys that is in the LDS serves them all. A workgroup takes 16, 32, 64 or 128 rows and walks the
// keys in tiles of 32:
//   S^T = K Q^T     a wave some of the rows against some of the keys; the queries stay in registers
//   softmax         in fp32 over the rows; P^T goes to the LDS in the order in which the next
//                   product's operand wants it (16 bytes a lane, no bank twice)
//   O^T += C^T P^T  a wave all the workgroup's rows, but a part of the latents' values: so a latent is
//                   read from the LDS once by each wave for the scores and once in all for the outputs
//                   (whole rows a wave would take twice the LDS reads, which bound the kernel then)
// The tiles come by DMA into rings in the LDS, two to four ahead (64 rows and fewer: a pair of tiles a step).
//
// In the LDS the 16-byte chunk c of a latent's row r lies at c ^ swizzle(r) (the four bits of r, two of
// them swapped): a score operand's sixteen rows then lie in different banks, and so do the 8-byte pieces of
// eight rows that a transposing read (ds_read_b64_tr_b16) takes of four chunks.
//
// Work: a sequence's tokens are cut into tiles of J (J heads <= ROWS, a power of two), one item each, or
// where there are more heads than rows into slices of heads. An item's length is its number of key
// tiles; the items in a row are cut into as many equal ranges as there are workgroups, so every
// workgroup has the same number of tiles whatever the lengths are. Each finds its range by a scan over the
// sequences' lengths in closed form. An item that is cut leaves fp32 partial rows, which
// latent_merge_kernel adds in order: results repeat themselves to the bit.
//
// Measured, with the merge. 256 decodes, 1024 tokens in the middle and 8192 at most, latents of 512 (64 rotated): 16 heads
// 126 us (3.7 TB/s), 32 147, 64 175, 128 heads 225 (488 TFLOP/s): bound by the memory, which has the partial
// rows of 128 heads to take too (some 100 MB beside 525; the merge 24 us). 4 chunks of 512 over up to 4096, 16
// heads 249 to 254 us (770 TFLOP/s; a step of 128 rows and 32 keys 1.9 us, its products 1.3). 8 decodes of 16 heads over
// some 256 18.4 us, one over some 4096 26 us: the start (lengths, page table, keys: 8 us), then the merge (4).
// Code that runs once counts: a workgroup's 8 KB of it took 8 us to come into the instruction cache.
#include "latent_mma.h"

namespace ss {
namespace {

// Ranges of a call of few tiles: a range of t tiles takes t steps, and its partial rows are written and read again. The
// least of tiles / ranges * kStep + ranges * rows * kRow, in us: a step takes 1.6 to 2, a row of 2 KB there and back 0.8
// ns by the memory's rate, less where the caches hold it (one decode of 128 heads over some 4096 tokens, of
// 59 ranges: 53 us with 0.5, 82 us with 0.35 of the merge's first form; 8 of them 80 and 86)
constexpr float kStep = 1.8f, kRow = 0.5e-3f;
// The same for 32 keys of 16 or 32 rows beside those, with its part of its items' starts (a step 1.1 to 1.25 then). Over
// eleven steps of 16 to 250 decodes beside 1 to 4 chunks (8, 16 and 32 heads, latents of 256 and 512) it is 5 % from the
// best of 1.0, 1.25, 1.5 and 1.8 on average, as 1.25 is (1.0 15 %, 1.8 6 %), and 36 % at worst: 250 decodes over some 300
// beside 2 chunks of 256, which would take 103 us with 1.0 and take 140. 32 heads would rather have 1.8 (192 decodes and 4
// chunks of 256: 316 us, and 328), 16 rather 1.25 (192 decodes and a chunk: 134 and 139).
constexpr float kFewStep = 1.5f;

template <int R_, int RT_, int NW_>
struct LatTile {
  static constexpr int R = R_, RT = RT_, NW = NW_;
  static constexpr int KT = 32, ROWS = 16 * RT;
  static constexpr int ROWB = 2 * R, LPLANE = KT * ROWB;  // latents of a tile in the LDS
  static constexpr int RPLANE = KT * 2 * kRopeDim;
  static constexpr int NS = 4, NR = 4;                    // rings: two pairs of tiles
  static constexpr int DT = R / (16 * NW);                // 16-value output tiles of a wave
  static constexpr int KQ = NW / 4, RW = 4 * RT / (NW * KQ);  // sixteens of a pair's keys and row tiles whose scores a wave has
  static constexpr int RPI = 1024 / ROWB;                 // latents a DMA instruction brings
  static constexpr int NL = KT / RPI / NW;                // DMA instructions of a wave and tile, latents
  static constexpr int kP = NS * LPLANE + NR * RPLANE, kTop = kP + 2 * RT * 1024, kSum = kTop + ROWS * 16,
                       kScan = kSum + ROWS * 16, LDS = kScan + 128;
  static_assert(LDS <= 160 * 1024, "one workgroup a CU");
  static_assert(KQ == 1 || (KQ == 2 && RW == 1), "scores");
};

// The same for 128 rows, four waves (one a SIMD, with all its registers) of 32 rows and R / 4 values
template <int R_>
struct LatWide {
  static constexpr int R = R_, NW = 4, ROWS = 128;
  static constexpr int KT = 32;
  static constexpr int ROWB = 2 * R, LPLANE = KT * ROWB, RPLANE = KT * 2 * kRopeDim;
  static constexpr int NS = 4, NR = 3;
  static constexpr int DT = R / 128;      // 32-value output tiles of a wave
  static constexpr int PB = 4 * 2048;     // bytes of a tile's P
  static constexpr int RPI = 1024 / ROWB, NL = KT / RPI / NW;
  static constexpr int kP = NS * LPLANE + NR * RPLANE, kAlpha = kP + 2 * PB, kMl = kAlpha + 2 * ROWS * 4,
                       kGrew = kMl + ROWS * 8, kScan = kGrew + 64, LDS = kScan + 128;
  static_assert(LDS <= 160 * 1024, "one workgroup a CU");
};

// The latents' chunk of 8 values that output tile dt of wave w takes for lanes of row group g: bit 2 from
// g >> 1, so that the four pieces of a transposing read lie in different banks whatever dt and w are
template <typename C>
__device__ __forceinline__ int out_chunk(int dt, int gh, int w) {
  if constexpr (C::DT == 8)
    return (dt & 3) + 4 * gh + 8 * (dt >> 2) + 16 * w;
  else if constexpr (C::DT == 4)
    return dt + 4 * gh + 8 * w;
  else
    return dt + 2 * (w & 1) + 4 * gh + 8 * (w >> 1);
}

// ---- items ----------------------------------------------------------------------------------

// How rows are made of tokens and heads: items of J tokens (1 << js), or HS slices of one token's heads
struct RowShape {
  int js, hs;
};
template <int ROWS>
__host__ __device__ inline RowShape row_shape(int heads) {
  RowShape s = {0, (heads + ROWS - 1) / ROWS};
  while ((heads << (s.js + 1)) <= ROWS) ++s.js;
  return s;
}

// A sequence as the items see it: n query tokens, `length` keys of which the table reaches `keys`
struct SeqView {
  int n, start, length, keys;
};
// lo < n heads <= hi, else the sequence counts as empty (another launch takes it)
__device__ __forceinline__ SeqView seq_view(const LatentParams& p, int b, int lo, int hi) {
  SeqView v;
  latent_queries(p, b, v.n, v.start);
  int first;
  v.keys = latent_keys(p, b, first, v.length);
  const int64_t rows = (int64_t)v.n * p.heads;
  if (rows <= lo || rows > hi) v.n = 0;
  return v;
}

// sum of floor(i / 2^s) over i < x
__device__ __forceinline__ int64_t steps_below(int64_t x, int s) {
  const int64_t q = x >> s;
  return ((q * (q - 1) / 2) << s) + q * (x - (q << s));
}
// Key tiles of the token tiles before the i-th of a sequence's nt: tile i ends at key length - n +
// (i + 1) J (the last one at `length`) and counts at least one. With a table that does not reach the
// length, all of them as long as the table.
__device__ __forceinline__ int64_t tiles_before(const SeqView& v, int i, int nt, int js) {
  if (v.length > v.keys) return (int64_t)i * max(1, (v.keys + 31) >> 5);
  const int m = min(i, nt - 1);  // of those that end with a whole tile of tokens
  const int base = v.length - v.n + (1 << js);
  const int none = base >= 1 ? 0 : min(m, (-base >> js) + 1);  // that see no key
  int64_t sum = none;
  const int64_t count = m - none, at = (int64_t)base + ((int64_t)none << js) + 31;
  if (count > 0) {
    if (js >= 5) {
      sum += count * (at >> 5) + ((count * (count - 1) / 2) << (js - 5));
    } else {
      const int64_t c = at >> js;
      sum += steps_below(c + count, 5 - js) - steps_below(c, 5 - js);
    }
  }
  return i > m ? sum + max(1, (v.length + 31) >> 5) : sum;
}
__device__ __forceinline__ int64_t seq_tiles(const SeqView& v, RowShape s) {
  if (v.n <= 0) return 0;
  const int nt = (v.n + (1 << s.js) - 1) >> s.js;
  return tiles_before(v, nt, nt, s.js) * s.hs;
}

// The same in every lane, kept in scalar registers
__device__ __forceinline__ int64_t uniform(int64_t x) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 |
                   (uint32_t)__builtin_amdgcn_readfirstlane((int)x));
}

struct LatentWork {
  float* o;   // [2 groups][ROWS][R] partial rows
  float* ml;  // [2 groups][ROWS][2] maximum (log2) and sum
  int* rec;   // [groups][4] the item that begins before a group's range and is merged there
  int lo, hi;  // the launch's sequences: lo < n heads <= hi
};

// ---- a wave's part of the tiles' way into the LDS ------------------------------------------------
//
// 32 / NW keys' latents, and waves 0 .. 3 eight rotated keys, of one page each (pages hold eight tokens at
// least): one descriptor a tile, which ends with the keys that are there; behind its end, for absent
// pages and for tiles past the last one the DMA writes zeros without an access. The page table is
// read 64 tiles at a time, an entry a lane.
template <typename C>
struct Feed {
  const LatentParams& p;
  const int32_t* table;
  uint32_t lds;
  int shift, kv_end, tend, key8, tok_bytes, base, at8;  // at8: the wave's first of the eight keys
  int entries;                                          // of tile base + lane
  int l16, first;
  int voff_r;
  i32x4 rsrc;
  uint32_t to_l, to_r;

  __device__ __forceinline__ Feed(const LatentParams& params, int b, char* mem, int kv_end_, int t0, int tend_)
      : p(params), kv_end(kv_end_), tend(tend_) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    table = p.bt + (int64_t)b * p.bt_stride;
    lds = (uint32_t)(uintptr_t)(LdsBytes)mem;
    shift = __builtin_ctz((unsigned)p.block_size);
    key8 = 8 * (wave & 3);
    at8 = C::NW == 8 ? 4 * (wave >> 2) : 0;
    tok_bytes = (int)(p.kv_s1 * 2);
    const int hi = lane / (C::R / 8);  // 0 where an instruction brings one latent
    l16 = 16 * ((lane & (C::R / 8 - 1)) ^ lat_swizzle(key8 + at8) ^ hi);
    first = (at8 + hi) * tok_bytes;
    voff_r = (lane >> 3) * tok_bytes + C::ROWB + 16 * ((lane & 7) ^ tile_swizzle(key8 + (lane >> 3)));
    load(t0);
  }
  __device__ __forceinline__ void load(int t) {
    base = t;
    const int i = (int)min(((int64_t)(t + (int)(threadIdx.x & 63)) * 32 + key8) >> shift, (int64_t)p.max_blocks - 1);
    entries = table[i];
    asm volatile("" : "+v"(entries));  // waited for here, not where every tile's entry is read
  }
  // tile t into ring slots ls and rs; ready for dma
  __device__ __forceinline__ void aim(int t, int ls, int rs) {
    if (t - base >= 64) load(t);
    const int e = __builtin_amdgcn_readlane(entries, t - base);
    const int key = t * 32 + key8, live = min(8, kv_end - key);
    const bool there = (uint32_t)e < (uint32_t)p.num_blocks && live > 0 && t < tend;
    const uint64_t off = 2 * (uint64_t)p.kv_s0 * (uint32_t)e + (uint32_t)((key & (p.block_size - 1)) * tok_bytes);
    const uint64_t at = (uint64_t)p.kv + (there ? off : 0);
    rsrc = i32x4{__builtin_amdgcn_readfirstlane((int)(uint32_t)at),
                 __builtin_amdgcn_readfirstlane((int)(uint32_t)(at >> 32) & 0xFFFF),
                 __builtin_amdgcn_readfirstlane(there ? (live - 1) * tok_bytes + C::ROWB + 2 * kRopeDim : 0), 0x00020000};
    to_l = lds + ls * C::LPLANE + (key8 + at8) * C::ROWB;
    to_r = lds + C::NS * C::LPLANE + rs * C::RPLANE + key8 * 2 * kRopeDim;
    asm volatile("s_nop 4" : : "s"(rsrc));  // SGPRs that a VALU wrote: five wait states before a VMEM reads them
  }
  // instruction u of C::NL (latents), and C::NL (rotated keys; waves 0 .. 3 alone)
  template <int u>
  __device__ __forceinline__ void dma() const {
    if constexpr (u < C::NL) {
      constexpr int k = u * C::RPI, sw = 16 * ((k & 3) | ((k & 4) << 1));
      int at = l16;
      asm volatile("" : "+v"(at));  // made anew each time: the offsets would take registers that the queries need
      dma_b128(rsrc, (LdsBytes)(uintptr_t)(to_l + k * C::ROWB), (at ^ sw) + (first + k * tok_bytes), 0);
    } else {
      dma_b128(rsrc, (LdsBytes)(uintptr_t)to_r, voff_r, 0);
    }
  }
  __device__ __forceinline__ void all() const {
    static_for<C::NL>([&](auto u) __attribute__((always_inline)) { dma<decltype(u)::value>(); });
    if (C::NW == 4 || threadIdx.x < 256) dma<C::NL>();
  }
};

// 16, 32 or 64 rows: a step takes a pair of tiles, 64 keys. A wave has the scores of sixteen of them for all rows (of
// eight waves, 32 for sixteen rows), writes their probabilities by the rows' maxima so far, and their own maxima; if one has grown by more than
// the slack, which all waves see then, the probabilities are written once more. So the scores, whose chain of products,
// maximum and exponents is what a step of few rows takes, are cut into four: 32 keys by one wave took 1.85 us
// on any number of CUs, 64 take 2.1 to 2.5 (256 decodes of 16 heads 138 -> 126 us, of 32 155 -> 147; of 64, whose
// eight waves had the scores of 32 keys and sixteen rows before too, 170 -> 175).
template <typename T, typename C>
__device__ __forceinline__ void latent_segment(const LatentParams& p, const LatentWork& work, char* const lds,
                                               const SeqView v, const int b, const int tok0, const int head0,
                                               const int js, const int t0, const int t1, const bool whole,
                                               const int slot) {
  constexpr int R = C::R, RT = C::RT, NW = C::NW, DT = C::DT, RW = C::RW, KQ = C::KQ, KS = R / 32, KR = kRopeDim / 32;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int quarter = KQ == 1 ? wave : 2 * (wave >> 2), rt0 = KQ == 1 ? 0 : wave & 3;  // its first sixteen keys and row tile
  const int heads = min(p.heads - head0, C::ROWS);       // of a token in this item
  const int tokens = min(1 << js, v.n - tok0);
  const int kv_end = max(0, min(v.keys, v.length - v.n + tok0 + tokens));
  const int tend = min(t1, (kv_end + 31) >> 5);

  // the row of this lane in row tile rt: token and head, or none
  auto row_of = [&](int rt, int& tok, int& head) {
    const int rr = 16 * rt + n, j = rr / heads;
    tok = tok0 + j;
    head = head0 + rr - j * heads;
    return j < tokens;
  };
  Feed<C> feed(p, b, lds, kv_end, t0, tend);
  auto send = [&](int t, int ring) {  // tiles t and t + 1 into ring slots ring and ring + 1
    for (int i = 0; i < 2; ++i) {
      feed.aim(t + i, ring + i, ring + i);
      feed.all();
    }
  };
  send(t0, 0);
  // queries: scaled inside the exponent, which needs a positive scale (a negative one is the query's sign)
  u32x4 qop[RW][KS + KR];
  int lim[RW], least = 0x7FFFFFFF;  // keys of a lane's rows up to here; of the wave's rows, tiles before it need no mask
#pragma unroll
  for (int rw = 0; rw < RW; ++rw) {
    int tok, head;
    const bool ok = row_of(rt0 + rw, tok, head);
    lim[rw] = min(kv_end, t1 * 32);
    if (ok) lim[rw] = min(lim[rw], v.length - v.n + tok + 1);
    least = min(least, lim[rw]);
    const T* const q = (const T*)p.q + (p.cu ? 0 : b * p.q_sb) + (v.start + (ok ? tok : tok0)) * p.q_st +
                       (ok ? head : head0) * p.q_sh + 8 * g;  // (a lane without a row: the item's first one, as zeros)
    const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u, keep = ok ? ~0u : 0u;
#pragma unroll
    for (int s = 0; s < KS + KR; ++s) qop[rw][s] = (load16(q + 32 * s) ^ u32x4{flip, flip, flip, flip}) & u32x4{keep, keep, keep, keep};
  }
  send(t0 + 2, 2);
  const float cscale = fabsf(p.scale_log2);
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) least = min(least, __shfl_xor(least, o));
  least = __builtin_amdgcn_readfirstlane(least);

  // absent pages among this item's: its tiles are masked key by key then
  bool bad = false;
  for (int i = ((t0 * 32) >> feed.shift) + threadIdx.x; (int64_t)i << feed.shift < min(kv_end, tend * 32); i += 64 * NW)
    bad |= (uint32_t)feed.table[i] >= (uint32_t)p.num_blocks;
  const bool holes = __syncthreads_or(bad);

  f32x4 acc[RT][DT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[rt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m[RT], own[RW], l[RW];  // of row n: the maxima of all row tiles and of the wave's; l: of this lane's keys
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) m[rt] = kNegBig;
#pragma unroll
  for (int rw = 0; rw < RW; ++rw) own[rw] = kNegBig, l[rw] = 0.f;
  const int sw = lat_swizzle(n), vrow = 4 * g + (n >> 2), vsw = lat_swizzle(vrow);

  for (int t = t0, ring = 0; t < tend; t += 2, ring ^= 2) {
    if (t == t0) {  // (the second pair may be on its way)
      if (wave < 4)
        wait_dma<2 * (C::NL + 1)>();
      else
        wait_dma<2 * C::NL>();
    } else {
      wait_dma<0>();
    }
    __syncthreads();  // the pair is there, and the one before is done with
    if (t > t0) send(t + 2, ring ^ 2);

    const char* const kl = lds + (ring + (quarter >> 1)) * C::LPLANE + (16 * (quarter & 1) + n) * C::ROWB;
    const char* const kr = lds + C::NS * C::LPLANE + (ring + (quarter >> 1)) * C::RPLANE + (16 * (quarter & 1) + n) * 2 * kRopeDim;
    constexpr int SC = KQ == 1 ? RW : KQ, CH = KQ == 1 ? 2 : 1;  // 16 x 16 scores, and sums of each that take turns
    f32x4 s2[SC][CH];
#pragma unroll
    for (int i = 0; i < SC; ++i)
#pragma unroll
      for (int h = 0; h < CH; ++h) s2[i][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < KS + KR; ++s)
#pragma unroll
      for (int x = 0; x < KQ; ++x) {
        const u32x4 k = s < KS ? load16(kl + 16 * x * C::ROWB + 16 * ((4 * s + g) ^ sw))
                               : load16(kr + 16 * x * 2 * kRopeDim + 16 * ((4 * (s - KS) + g) ^ tile_swizzle(n)));
#pragma unroll
        for (int rw = 0; rw < RW; ++rw) s2[KQ == 1 ? rw : x][s % CH] = Elem<T>::mfma(k, qop[rw][s], s2[KQ == 1 ? rw : x][s % CH]);
      }
    // the first tile's latents for the outputs, on their way beside the softmax
    auto latents = [&](int tile, u32x4 (&c)[DT]) {
      const uint32_t vp = lds_address(lds) + (ring + tile) * C::LPLANE + vrow * C::ROWB + 8 * (n & 1);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const uint32_t at = vp + 16 * (out_chunk<C>(dt, (n >> 1) & 1, wave) ^ vsw);
        c[dt] = lds_keys(at, at + 16 * C::ROWB);
      }
    };
    u32x4 c[2][DT];
    if constexpr (KQ == 1) latents(0, c[0]);  // (eight waves have no registers for it, and two a SIMD)
    f32x4 sv[RW][KQ];
#pragma unroll
    for (int rw = 0; rw < RW; ++rw)
#pragma unroll
      for (int x = 0; x < KQ; ++x) sv[rw][x] = KQ == 1 ? s2[rw][0] + s2[rw][CH - 1] : s2[x][0];
    if (holes || t * 32 + 64 > least) {
#pragma unroll
      for (int x = 0; x < KQ; ++x) {
        const int key = t * 32 + 16 * (quarter + x) + 4 * g;  // four keys of one page
        const bool there = !holes || key >= kv_end || (uint32_t)feed.table[key >> feed.shift] < (uint32_t)p.num_blocks;
#pragma unroll
        for (int rw = 0; rw < RW; ++rw)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!there || key + e >= lim[rw]) sv[rw][x][e] = -__builtin_inff();
      }
    }
    u32x2 pv[RW][KQ];  // as they are written
    auto probabilities = [&]() {
#pragma unroll
      for (int rw = 0; rw < RW; ++rw)
#pragma unroll
        for (int x = 0; x < KQ; ++x) {
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = fast_exp2(fmaf(sv[rw][x][e], cscale, -own[rw]));
          pv[rw][x] = u32x2{Elem<T>::pack2(y[0], y[1]), Elem<T>::pack2(y[2], y[3])};
          *reinterpret_cast<u32x2*>(lds + C::kP + ((quarter >> 1) * RT + rt0 + rw) * 1024 + lane * 16 + 8 * ((quarter + x) & 1)) =
              pv[rw][x];
        }
    };
#pragma unroll
    for (int rw = 0; rw < RW; ++rw) {
      float top = kNegBig;
#pragma unroll
      for (int x = 0; x < KQ; ++x) top = fmaxf(top, fmaxf(fmaxf(sv[rw][x][0], sv[rw][x][1]), fmaxf(sv[rw][x][2], sv[rw][x][3])));
      top = max_across_rows(top);
#pragma unroll
      for (int x = 0; x < KQ; ++x)
        if (g == x) *reinterpret_cast<float*>(lds + C::kTop + (16 * (rt0 + rw) + n) * 16 + 4 * (quarter + x)) = top;
    }
    probabilities();
    __syncthreads();
    float want[RT];
    bool grew = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const f32x4 top = *reinterpret_cast<const f32x4*>(lds + C::kTop + (16 * rt + n) * 16);
      want[rt] = fmaxf(m[rt], fmaf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), cscale, -kHeadroom<T>));
      grew |= want[rt] > m[rt] + kSlack;
    }
    if (__any(grew)) {  // the same in every wave
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const float alpha = fast_exp2(m[rt] - want[rt]);
        m[rt] = want[rt];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[rt][dt] *= alpha;
#pragma unroll
        for (int rw = 0; rw < RW; ++rw)
          if (rt == rt0 + rw) own[rw] = want[rt], l[rw] *= alpha;
      }
      probabilities();
      __syncthreads();
    }
#pragma unroll
    for (int rw = 0; rw < RW; ++rw)
#pragma unroll
      for (int x = 0; x < KQ; ++x) l[rw] += pair_sum<T>(pv[rw][x][0]) + pair_sum<T>(pv[rw][x][1]);
    if constexpr (KQ == 1) latents(1, c[1]);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if constexpr (KQ == 2) latents(x, c[x]);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const u32x4 pr = load16(lds + C::kP + (x * RT + rt) * 1024 + lane * 16);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[rt][dt] = Elem<T>::mfma(c[x][dt], pr, acc[rt][dt]);
      }
    }
  }
  wait_dma<0>();

  // ---- the rows' sums, then the rows themselves
#pragma unroll
  for (int rw = 0; rw < RW; ++rw) {
    const float sum = sum_across_rows(l[rw]);
#pragma unroll
    for (int x = 0; x < KQ; ++x)
      if (g == x) *reinterpret_cast<float*>(lds + C::kSum + (16 * (rt0 + rw) + n) * 16 + 4 * (quarter + x)) = x ? 0.f : sum;
  }
  __syncthreads();
  auto total_of = [&](int rt) {
    const f32x4 s = *reinterpret_cast<const f32x4*>(lds + C::kSum + (16 * rt + n) * 16);
    return (s[0] + s[1]) + (s[2] + s[3]);
  };
  if (whole) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      int tok, head;
      if (!row_of(rt, tok, head)) continue;
      const float total = total_of(rt);
      const float inv = total == 0.f ? 0.f : 1.f / total;
      T* const o = (T*)p.out + (p.cu ? 0 : b * p.o_sb) + (v.start + tok) * p.o_st + head * p.o_sh + 4 * (g & 1);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const f32x4 y = acc[rt][dt] * inv;
        const u32x2 w = {Elem<T>::pack2(y[0], y[1]), Elem<T>::pack2(y[2], y[3])};
        __builtin_memcpy(o + 8 * out_chunk<C>(dt, g >> 1, wave), &w, 8);  // (rows may begin at any value)
      }
    }
  } else {
    float* const o = work.o + (int64_t)slot * C::ROWS * R + 4 * (g & 1);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        *reinterpret_cast<f32x4*>(o + (16 * rt + n) * R + 8 * out_chunk<C>(dt, g >> 1, wave)) = acc[rt][dt];
      if (wave == 0 && g == 0)
        *reinterpret_cast<float2*>(work.ml + ((int64_t)slot * C::ROWS + 16 * rt + n) * 2) = float2{m[rt], total_of(rt)};
    }
  }
  __syncthreads();  // the LDS is free for the next item
}

// ---- 128 rows: 32 x 32 products --------------------------------------------------------------

// acc += a b, the accumulator in AGPRs. As asm, because the compiler moves accumulators between the register
// files when it needs more than half of the registers. What it therefore does not look after: the
// operands come from LDS reads, which it does wait for; an accumulator is touched again sixteen products
// later; and what reads the accumulators waits first (settled).
template <typename T>
__device__ __forceinline__ void mfma32_acc(f32x16& acc, u32x4 a, u32x4 b) {
  if constexpr (std::is_same<T, bf16_t>::value)
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
  else
    asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}
template <typename T>
__device__ __forceinline__ void clear_acc(f32x16& acc) {  // a product of zeros (two wait states after they are written): no other registers take part
  const u32x4 z = {0, 0, 0, 0};
  if constexpr (std::is_same<T, bf16_t>::value)
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %1, 0" : "=a"(acc) : "v"(z));
  else
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_f16 %0, %1, %1, 0" : "=a"(acc) : "v"(z));
}
template <int N>
__device__ __forceinline__ void settled(f32x16 (&acc)[4][N]) {
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
  for (int rt = 0; rt < 4; ++rt)
#pragma unroll
    for (int dt = 0; dt < N; ++dt) asm volatile("" : "+a"(acc[rt][dt]));
}


// A wave takes 32 rows' scores against all 32 keys (as S^T: lane l row l % 32, its result r key 8 (r / 4) +
// 4 (l / 32) + r % 4) and all 128 rows' outputs of R / 4 values. Four waves: with 32 rows each a key is
// read from the LDS four times for the scores instead of eight, which bound the kernel.
template <typename T, typename C>
__device__ __forceinline__ void latent_segment_wide(const LatentParams& p, const LatentWork& work, char* const lds,
                                                    const SeqView v, const int b, const int tok0, const int head0,
                                                    const int js, const int t0, const int t1, const bool whole,
                                                    const int slot) {
  constexpr int R = C::R, DT = C::DT, KS = R / 16, KR = kRopeDim / 16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, h = lane >> 5;
  const int heads = min(p.heads - head0, C::ROWS);
  const int tokens = min(1 << js, v.n - tok0);
  const int kv_end = max(0, min(v.keys, v.length - v.n + tok0 + tokens));
  const int tend = min(t1, (kv_end + 31) >> 5);
  auto row_of = [&](int rt, int& tok, int& head) {
    const int rr = 32 * rt + n, j = rr / heads;
    tok = tok0 + j;
    head = head0 + rr - j * heads;
    return j < tokens;
  };

  Feed<C> feed(p, b, lds, kv_end, t0, tend);
  feed.aim(t0, 0, 0);  // what the first scores need comes first: their keys, then the queries
  feed.all();

  u32x4 qop[KS + KR];
  int lim = min(kv_end, t1 * 32);  // keys of this lane's row up to here (its part of the item's)
  {
    int tok, head;
    const bool ok = row_of(wave, tok, head);
    if (ok) lim = min(lim, v.length - v.n + tok + 1);
    // a lane without a row reads the item's first one and takes zeros
    const T* const q = (const T*)p.q + (p.cu ? 0 : b * p.q_sb) + (v.start + (ok ? tok : tok0)) * p.q_st +
                       (ok ? head : head0) * p.q_sh + 8 * h;
    const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u, keep = ok ? ~0u : 0u;
#pragma unroll
    for (int s = 0; s < KS + KR; ++s) qop[s] = load16(q + 16 * s);
#pragma unroll
    for (int s = 0; s < KS + KR; ++s) qop[s] = (qop[s] ^ u32x4{flip, flip, flip, flip}) & u32x4{keep, keep, keep, keep};
    for (int i = 1; i < 3; ++i) {
      feed.aim(t0 + i, i, i);
      feed.all();
    }
  }
  const float cscale = fabsf(p.scale_log2);
  int least = lim;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) least = min(least, __shfl_xor(least, o));
  least = __builtin_amdgcn_readfirstlane(least);
  bool bad = false;
  for (int i = ((t0 * 32) >> feed.shift) + threadIdx.x; (int64_t)i << feed.shift < min(kv_end, tend * 32); i += 256)
    bad |= (uint32_t)feed.table[i] >= (uint32_t)p.num_blocks;
  const bool holes = __syncthreads_or(bad);

  f32x16 acc[4][DT];
#pragma unroll
  for (int rt = 0; rt < 4; ++rt)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) clear_acc<T>(acc[rt][dt]);
  float m = kNegBig, l = 0.f;

  const uint32_t lbase = (uint32_t)(uintptr_t)(LdsBytes)lds;
  // LDS addresses: the 16-byte chunk's bits 4 .. 7 under the swizzle are the low bits of an address (planes
  // begin on 512 bytes), so another chunk's address is an exclusive or away
  const uint32_t kaddr = lbase + n * C::ROWB + 16 * (h ^ lat_swizzle(n));
  const uint32_t raddr = lbase + C::NS * C::LPLANE + n * 2 * kRopeDim + 16 * (h ^ tile_swizzle(n));
  const int sl = lane & 15, vrow = 4 * h + (sl >> 2), quad = 2 * ((lane >> 4) & 1) + ((sl & 3) >> 1);
  const uint32_t vaddr = lbase + vrow * C::ROWB + 8 * (sl & 1) + 16 * ((4 * quad) ^ lat_swizzle(vrow)) +
                         (DT == 4 ? 256 * wave : 256 * (wave >> 1) + 0);
  const uint32_t vflip = DT == 4 ? 0 : 32 * (wave & 1);  // the wave's bit of the chunk
  const uint32_t paddr = lbase + C::kP;

  // a lane's number that the compiler cannot build addresses from ahead of time: they would take registers
  // that the queries need
  auto fresh = [&]() {
    int ln = lane;
    asm volatile("" : "+v"(ln));
    return ln;
  };
  auto word = [](uint32_t at) { return lds_word(at); };
  auto vread = [&](uint32_t slot, int s, int dt) {  // 16 keys from 16 s on, output tile dt
    const uint32_t at = (vaddr + slot) ^ (16 * dt) ^ vflip;
    return lds_keys(at + 16 * s * C::ROWB, (at ^ 64) + (16 * s + 8) * C::ROWB);
  };

  // One step: the scores of tile t + 1, then the outputs of tile t (OUT), whose latents are in ring slot vl and
  // whose probabilities in buffer `buf`, and between their products the softmax of t + 1, whose probabilities
  // go into the other buffer. One wave a SIMD has nothing to hide behind, so the order is written out: an
  // operand is read from the LDS a few products ahead of its own, and the two barriers stand where
  // products go on behind them:
  //   among the scores: the other waves are done with the step before. Their probabilities can be read, and
  //     the LDS of tile t - 1 is free: tile t + 3 is sent for.
  //   among the outputs: tile t + 2 has landed, and its first operands are read.
  constexpr int NQ = KS + KR, AHEAD = 4, P = 8 * DT;  // products of the scores and of the outputs
  constexpr int kShared = NQ / 3, kLanded = P / 2;    // where the barriers are
  static_assert(kShared + 3 + 2 * C::NL < NQ || C::NL < 8, "the DMAs fit among the scores");
  u32x4 kring[AHEAD];
  uint32_t ka = 0, ra = 0;
  auto kread = [&](auto sc) __attribute__((always_inline)) {
    constexpr int s = sc;
    if constexpr (s < KS)
      kring[s % AHEAD] = word((ka ^ (32 * (s & 7))) + 256 * (s >> 3));
    else if constexpr (s < NQ)
      kring[s % AHEAD] = word(ra ^ (32 * (s - KS)));
  };
  auto at_keys = [&](int kl, int kr) {  // of the tile in ring slots kl, kr
    ka = kaddr + kl * C::LPLANE;
    ra = raddr + kr * C::RPLANE;
  };
  auto step = [&](auto outc, int t, int vl, int vr, int buf) __attribute__((always_inline)) {
    constexpr bool OUT = decltype(outc)::value;
    f32x16 s16;
    u32x4 cv[DT], pr[2];
    int flags = 0;
    const uint32_t vslot = vl * C::LPLANE, pa = paddr + buf * C::PB + fresh() * 16;
    __builtin_amdgcn_sched_barrier(0);
    static_for<NQ>([&](auto sc) __attribute__((always_inline)) {
      constexpr int s = sc;
      mfma32_sum<T, s == 0>(s16, kring[s % AHEAD], qop[s]);
      kread(std::integral_constant<int, s + AHEAD>{});
      if constexpr (OUT) {
        if constexpr (s == kShared) {
          asm volatile("s_waitcnt lgkmcnt(%0)" : : "n"(AHEAD) : "memory");  // all but the scores' operands
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
        }
        if constexpr (s == kShared + 1) {
          flags = *reinterpret_cast<const int*>(lds + C::kGrew + (buf * 4 + (fresh() & 3)) * 4);
          feed.aim(t + 3, (vl + 3) & 3, vr);
        }
        constexpr int gap = C::NL < 8 ? 1 : 2, d = s - kShared - 3;
        if constexpr (d >= 0 && d % gap == 0 && d / gap <= C::NL) feed.template dma<d / gap>();
        constexpr int u = s - (NQ - DT - 1);  // the first outputs' operands behind the last scores'
        if constexpr (u >= 0 && u < DT) cv[u] = vread(vslot, 0, u);
        if constexpr (u == DT) pr[0] = word(pa);
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    if (OUT && __any(flags)) {  // some row's maximum grew with tile t
      settled(acc);
#pragma unroll
      for (int rt = 0; rt < 4; ++rt) {
        const float alpha = *reinterpret_cast<const float*>(lds + C::kAlpha + (buf * C::ROWS + 32 * rt + (fresh() & 31)) * 4);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          acc[rt][dt] *= alpha;
          asm volatile("" : "+a"(acc[rt][dt]));
        }
      }
      asm volatile("s_nop 4" ::: "memory");
    }
    if (holes || t * 32 + 64 > least) {
      asm volatile("s_nop 15\n\ts_nop 7" : "+v"(s16));  // the last product is through
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int key = (t + 1) * 32 + 8 * x + 4 * h;  // four keys of one page
        bool there = true;
        if (holes && key < kv_end) there = (uint32_t)feed.table[key >> feed.shift] < (uint32_t)p.num_blocks;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!there || key + e >= lim) s16[4 * x + e] = -__builtin_inff();
      }
    }
    float top = 0.f, mn = 0.f, sum = 0.f;
    bool grew = false;
    uint32_t pk[8];
    // the softmax in parts of a few instructions
    constexpr int kParts = 19;
    auto part = [&](auto ic) __attribute__((always_inline)) {
      constexpr int i = ic;
      if constexpr (i == 0) {
        asm volatile("s_nop 15\n\ts_nop 7" : "+v"(s16));  // the last score's product is through
        top = max3(max3(max3(s16[0], s16[1], s16[2]), s16[3], s16[4]), s16[5], s16[6]);
      } else if constexpr (i == 1) {
        top = max3(max3(max3(top, s16[7], s16[8]), s16[9], s16[10]), s16[11], s16[12]);
      } else if constexpr (i == 2) {
        top = max3(max3(top, s16[13], s16[14]), s16[15], s16[15]);
        const uint32_t tb = __builtin_bit_cast(uint32_t, top);
        auto sw = __builtin_amdgcn_permlane32_swap(tb, tb, false, false);
        top = max3(__builtin_bit_cast(float, (uint32_t)sw[0]), __builtin_bit_cast(float, (uint32_t)sw[1]),
                   __builtin_bit_cast(float, (uint32_t)sw[1]));
      } else if constexpr (i == 3) {
        top = fmaxf(m, fmaf(top, cscale, -kHeadroom<T>));
        grew = __any(top > m + kSlack);
        mn = grew ? top : m;
      } else if constexpr (i < 12) {
        constexpr int e = 2 * (i - 4);
        float a = fast_exp2(fmaf(s16[e], cscale, -mn)), c = fast_exp2(fmaf(s16[e + 1], cscale, -mn));
        asm volatile("" : "+v"(a), "+v"(c));  // made here
        s16[e] = a, s16[e + 1] = c;
      } else if constexpr (i < 16) {
        constexpr int e = 4 * (i - 12);
        pk[e / 2] = Elem<T>::pack2(s16[e], s16[e + 1]);
        pk[e / 2 + 1] = Elem<T>::pack2(s16[e + 2], s16[e + 3]);
        sum += pair_sum<T>(pk[e / 2]) + pair_sum<T>(pk[e / 2 + 1]);
      } else if constexpr (i == 16) {
        const float alpha = fast_exp2(m - mn);
        l = fmaf(l, alpha, sum);
        m = mn;
        // (by every lane, without a branch: behind one the compiler would gather the parts before it)
        *reinterpret_cast<float*>(lds + C::kAlpha + ((buf ^ 1) * C::ROWS + 32 * wave + (fresh() & 31)) * 4) = alpha;
        *reinterpret_cast<int*>(lds + C::kGrew + ((buf ^ 1) * 4 + wave) * 4) = OUT && grew;  // (before the first outputs are 0)
      } else if constexpr (i < kParts) {
        constexpr int q = i - 17;
        store16(lds + C::kP + (buf ^ 1) * C::PB + (2 * wave + q) * 1024 + fresh() * 16,
                u32x4{pk[4 * q], pk[4 * q + 1], pk[4 * q + 2], pk[4 * q + 3]});
      }
    };
    if constexpr (!OUT) {
      static_for<kParts>(part);
    } else {
      __builtin_amdgcn_sched_barrier(0);
      static_for<P>([&](auto ic) __attribute__((always_inline)) {
        constexpr int i = ic, q = i / (4 * DT), rt = i / DT % 4, dt = i % DT, g = i / DT;  // g: group of DT products
        if constexpr (dt == 0 && g + 1 < 8) pr[(g + 1) & 1] = word(pa + (2 * ((g + 1) & 3) + ((g + 1) >> 2)) * 1024);
        if constexpr (i == kLanded) {
          wait_dma<C::NL + 1>();
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
          at_keys((vl + 2) & 3, vr == 0 ? 2 : vr - 1);
        }
        mfma32_acc<T>(acc[rt][dt], cv[dt], pr[g & 1]);
        if constexpr (q == 0 && rt == 3) cv[dt] = vread(vslot, 1, dt);  // its last product of these 16 keys
        if constexpr (i >= P - AHEAD) kread(std::integral_constant<int, i - (P - AHEAD)>{});
        // from the third product on, in as many places as there are
        constexpr int from = i < 2 ? 0 : (i - 2) * kParts / (P - 2), to = i < 2 ? 0 : (i - 1) * kParts / (P - 2);
        static_for<to - from>(
            [&](auto jc) __attribute__((always_inline)) { part(std::integral_constant<int, from + jc>{}); });
        __builtin_amdgcn_sched_barrier(0);
      });
    }
  };

  if (t0 < tend) {
    wait_dma<2 * (C::NL + 1)>();
    __syncthreads();
    at_keys(0, 0);
    static_for<AHEAD>(kread);
    step(std::false_type{}, t0 - 1, 0, 0, 1);
    wait_dma<C::NL + 1>();
    __syncthreads();
    at_keys(1, 1);
    static_for<AHEAD>(kread);
    int ls = 0, rs = 0;
    for (int t = t0; t < tend; ++t) {
      // (the last step's scores are those of a tile of zeros behind every row's keys)
      step(std::true_type{}, t, ls, rs, (t - t0) & 1);
      ls = (ls + 1) & 3;
      rs = rs == 2 ? 0 : rs + 1;
    }
  }
  wait_dma<0>();
  settled(acc);

  {
    const uint32_t u = __builtin_bit_cast(uint32_t, l);
    auto sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const float sum = __builtin_bit_cast(float, (uint32_t)sw[0]) + __builtin_bit_cast(float, (uint32_t)sw[1]);
    if (h == 0) *reinterpret_cast<float2*>(lds + C::kMl + (32 * wave + n) * 8) = float2{m, sum};
  }
  __syncthreads();
  // Result r of output tile dt: value 8 chunk + 4 h + r % 4 of row n. The rows go through the LDS, where the tiles
  // were, 64 at a time, and are stored whole: a row's 16-byte pieces lie there at piece ^ (row % 16). (Stored as they
  // are in the registers, 32 bytes of 32 rows an instruction, 128 rows in fp32 took 16 us, now 9. Scaled and
  // rounded in the registers, whole ones took 9 as well, for the code's way into the instruction cache.)
  auto chunk = [&](int dt, int x) {
    return DT == 4 ? dt + 4 * x + 16 * wave : dt + 2 * (wave & 1) + 4 * x + 16 * (wave >> 1);
  };
  constexpr int B = 4 * R, L = R / 8;  // bytes of a row in the LDS, lanes of a row in the stores
  const int rows = tokens * heads, c = lane % L;
  T* const to = (T*)p.out + (p.cu ? 0 : b * p.o_sb) + (v.start + tok0) * p.o_st + head0 * p.o_sh + 8 * c;
  float* const o = work.o + (int64_t)slot * C::ROWS * R + 4 * c;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (half) __syncthreads();
    const uint32_t row = lbase + n * B;
#pragma unroll
    for (int rt = 0; rt < 2; ++rt)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const f32x16& a = acc[2 * half + rt][dt];
          *(__attribute__((address_space(3))) f32x4*)(uintptr_t)(row + 32 * rt * B + 16 * ((2 * chunk(dt, x) + h) ^ (n & 15))) =
              f32x4{a[4 * x], a[4 * x + 1], a[4 * x + 2], a[4 * x + 3]};
        }
    __syncthreads();
    if (whole) {
      const int end = min(64, rows - 64 * half);
#pragma unroll 4
      for (int r = (64 / L) * wave + lane / L; r < end; r += 256 / L) {
        const float total = reinterpret_cast<const float2*>(lds + C::kMl + (64 * half + r) * 8)->y;
        const float inv = total == 0.f ? 0.f : 1.f / total;
        const f32x4 lo = *reinterpret_cast<const f32x4*>(lds + r * B + 16 * ((2 * c) ^ (r & 15))) * inv;
        const f32x4 hi = *reinterpret_cast<const f32x4*>(lds + r * B + 16 * ((2 * c + 1) ^ (r & 15))) * inv;
        const u32x4 y = {Elem<T>::pack2(lo[0], lo[1]), Elem<T>::pack2(lo[2], lo[3]), Elem<T>::pack2(hi[0], hi[1]),
                         Elem<T>::pack2(hi[2], hi[3])};
        const int j = (64 * half + r) / heads;
        __builtin_memcpy(to + j * p.o_st + (64 * half + r - j * heads) * p.o_sh, &y, 16);
      }
    } else {
#pragma unroll 4
      for (int r = (64 / L) * wave + lane / L; r < 64; r += 256 / L)
#pragma unroll
        for (int u = 0; u < 2; ++u)
          store16(o + (64 * half + r) * R + 4 * u * L, load16(lds + r * B + 16 * ((u * L + c) ^ (r & 15))));
    }
  }
  if (!whole) {
    float* const ml = work.ml + (int64_t)slot * C::ROWS * 2;
    ml[threadIdx.x] = *reinterpret_cast<const float*>(lds + C::kMl + 4 * threadIdx.x);
  }
  __syncthreads();
}

extern __shared__ __attribute__((aligned(1024))) char s_lat[];

// Range w of at most `all` of the tiles of a launch's sequences
template <typename T, typename C>
__device__ __forceinline__ void latent_ranges(const LatentParams& p, const LatentWork& work, const int w, const int all) {
  constexpr int NT = 64 * C::NW;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const RowShape shape = row_shape<C::ROWS>(p.heads);
  // the sequences' lengths in tiles, summed: where this workgroup's range begins
  int64_t* const s_sum = reinterpret_cast<int64_t*>(s_lat + C::kScan);  // [NW], then what was found
  SeqView view = {0, 0, 0, 0};
  auto scan = [&](int b, int64_t& mine) {  // the sum up to and with sequence b, and that of the NT
    mine = 0;
    if (b < p.batch) view = seq_view(p, b, work.lo, work.hi), mine = seq_tiles(view, shape);
    int64_t sum = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t below = __shfl_up(sum, o);
      sum += lane >= o ? below : 0;
    }
    __syncthreads();
    if (lane == 63) s_sum[wave] = sum;
    __syncthreads();
    for (int i = 0; i < wave; ++i) sum += s_sum[i];
    return sum;
  };
  int64_t mine, upto = 0, total = 0;
  for (int b0 = 0; b0 < p.batch; b0 += NT) {
    upto = total + scan(b0 + threadIdx.x, mine);
    for (int i = 0; i < C::NW; ++i) total += s_sum[i];
  }
  total = uniform(total);
  const int64_t most = max((int64_t)sqrtf((float)total * (kStep / (kRow * C::ROWS))), min(total, (int64_t)p.batch));
  const int groups = (int)min(min((int64_t)all, total), most);
  int* const rec = work.rec + 4 * w;
  if (w >= groups) {
    if (threadIdx.x == 0) rec[0] = -1;
    return;
  }
  int64_t u = total * w / groups;
  const int64_t u1 = total * (w + 1) / groups;
  int64_t before = 0;  // tiles of the sequences before b
  int b = 0;
  for (int64_t b0 = 0, done = 0; b0 < p.batch; b0 += NT) {
    if (p.batch > NT) {
      upto = done + scan((int)b0 + threadIdx.x, mine);
      for (int i = 0; i < C::NW; ++i) done += s_sum[i];
    }
    if (upto - mine <= u && u < upto) {
      s_sum[C::NW] = b0 + threadIdx.x;
      s_sum[C::NW + 1] = upto - mine;
      *reinterpret_cast<SeqView*>(s_sum + C::NW + 2) = view;
    }
    __syncthreads();
    if (p.batch <= NT || u < done) break;
  }
  b = __builtin_amdgcn_readfirstlane((int)s_sum[C::NW]);
  before = uniform(s_sum[C::NW + 1]);
  SeqView v = *reinterpret_cast<SeqView*>(s_sum + C::NW + 2);
  v.n = __builtin_amdgcn_readfirstlane(v.n), v.start = __builtin_amdgcn_readfirstlane(v.start);
  v.length = __builtin_amdgcn_readfirstlane(v.length), v.keys = __builtin_amdgcn_readfirstlane(v.keys);
  __syncthreads();

  const int64_t u0 = u;
  for (;; v = seq_view(p, ++b, work.lo, work.hi)) {
    const int nt = (v.n + (1 << shape.js) - 1) >> shape.js;
    const int64_t end = before + seq_tiles(v, shape);
    if (u >= end) continue;  // no rows of this launch
    // the token tile that tile u is in: a search 64 at a time
    int i = 0;
    for (int span = nt; span > 1;) {
      const int step = (span + 63) >> 6, at = i + lane * step;
      const bool below = at < i + span && tiles_before(v, at, nt, shape.js) * shape.hs <= u - before;
      i += (__popcll(__ballot(below)) - 1) * step;
      span = min(step, nt - i);
    }
    i = __builtin_amdgcn_readfirstlane(i);
    for (; i < nt && u < u1; ++i) {
      const int64_t first = before + tiles_before(v, i, nt, shape.js) * shape.hs;
      const int64_t each = tiles_before(v, i + 1, nt, shape.js) - tiles_before(v, i, nt, shape.js);
      for (int h = shape.hs > 1 ? (int)((u - first) / each) : 0; h < shape.hs && u < u1; ++h) {
        const int64_t s = first + h * each, e = min(s + each, u1);
        const int t0 = (int)(u - s), t1 = (int)(e - s);
        if (u == u0 && threadIdx.x == 0) {  // an item begun in the range before: merged from here on
          const int from = (int)(((s + 1) * groups - 1) / total), to = (int)(((s + each) * groups - 1) / total);
          rec[0] = t0 > 0 && from + 1 == w ? b : -1;
          rec[1] = i * shape.hs + h;
          rec[2] = to;
        }
        if constexpr (std::is_same<C, LatWide<C::R>>::value)
          latent_segment_wide<T, C>(p, work, s_lat, v, b, i << shape.js, h * C::ROWS, shape.js, t0, t1,
                                    t0 == 0 && t1 == each, 2 * w + (t0 == 0));
        else
          latent_segment<T, C>(p, work, s_lat, v, b, i << shape.js, h * C::ROWS, shape.js, t0, t1,
                               t0 == 0 && t1 == each, 2 * w + (t0 == 0));
        u = e;
      }
    }
    if (u >= u1) break;
    before = end;
  }
}

template <typename T, typename C>
__global__ __launch_bounds__(64 * C::NW) __attribute__((amdgpu_waves_per_eu(C::NW / 4, C::NW / 4))) void latent_tile_kernel(
    const LatentParams p, const LatentWork work) {
  // workgroups go round robin over the eight XCDs: each XCD takes a contiguous eighth of the ranges, whose
  // items share keys
  const int all = gridDim.x, per_xcd = all >> 3;
  const int w = all & 7 ? (int)blockIdx.x : (int)(blockIdx.x & 7) * per_xcd + (int)(blockIdx.x >> 3);
  latent_ranges<T, C>(p, work, w, all);
}

// A step of decodes beside chunks: sequences of few rows in F's tiles and the others in M's, in one launch. Decodes wait
// for the memory and chunks for the matrix cores, so some workgroups of every XCD do the first while the others do
// the second, as many as the steps' times (kFewStep, kStep) ask for: 192 decodes and 4 chunks of 512 over up to
// 4096, 16 heads 284 to 301 us; in two launches 351, where one took 296.
template <typename T, typename F, typename M>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) void latent_mixed_kernel(
    const LatentParams p, const LatentWork few, const LatentWork many) {
  static_assert(F::NW == 4 && M::NW == 4, "workgroups of one size");
  float cost[2] = {0.f, 0.f};
  for (int b = threadIdx.x; b < p.batch; b += 256) {
    cost[0] += (float)seq_tiles(seq_view(p, b, few.lo, few.hi), row_shape<F::ROWS>(p.heads)) * kFewStep;
    cost[1] += (float)seq_tiles(seq_view(p, b, many.lo, many.hi), row_shape<M::ROWS>(p.heads)) * kStep;
  }
  float* const s_cost = reinterpret_cast<float*>(s_lat);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) cost[i] += __shfl_xor(cost[i], o);
    if ((threadIdx.x & 63) == 0) s_cost[4 * i + (threadIdx.x >> 6)] = cost[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) cost[i] = s_cost[4 * i] + s_cost[4 * i + 1] + s_cost[4 * i + 2] + s_cost[4 * i + 3];
  __syncthreads();
  // whole workgroups of each XCD (or of one that all are taken for), one at least for either where it has work
  const int xcds = gridDim.x & 7 ? 1 : 8, each = gridDim.x / xcds, xcd = blockIdx.x % xcds, at = blockIdx.x / xcds;
  int part = (int)(each * cost[0] / fmaxf(cost[0] + cost[1], 1.f) + 0.5f);
  part = min(max(part, cost[0] > 0.f ? 1 : 0), cost[1] > 0.f ? each - 1 : each);
  part = __builtin_amdgcn_readfirstlane(part);
  const int rest = each - part;
  if (at < part) {
    if (threadIdx.x == 0) many.rec[4 * (xcds * rest + xcd * part + at)] = -1;  // of no range
    latent_ranges<T, F>(p, few, xcd * part + at, xcds * part);
  } else {
    if (threadIdx.x == 0) few.rec[4 * (xcds * part + xcd * rest + at - part)] = -1;
    latent_ranges<T, M>(p, many, xcd * rest + at - part, xcds * rest);
  }
}

// The partial rows of an item that is cut, added in the order of its ranges: WPR waves one row of the item
// whose first cut is the begin of range w, each an equal part of the ranges. The parts' maxima and sums are read
// 64 at a time, a part a lane; then the rows, eight parts' on their way at once. With one wave a row blockIdx.x is w;
// else it counts the ranges at whose begin an item is merged, of which there are at most as many as items.
template <typename T, int R, int ROWS, int WPR>
__global__ __launch_bounds__(WPR == 1 ? 256 : 64 * WPR) void latent_merge_kernel(const LatentParams p, const LatentWork work,
                                                                                int groups) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int w = blockIdx.x;
  if constexpr (WPR > 1) {
    int left = w;
    w = -1;
    for (int w0 = 0; w0 < groups && w < 0; w0 += 64) {
      const bool here = w0 + lane < groups && work.rec[4 * (w0 + lane)] >= 0;
      uint64_t m = __ballot(here);
      if (__popcll(m) <= left) {
        left -= __popcll(m);
        continue;
      }
      for (; left > 0; --left) m &= m - 1;
      w = w0 + __builtin_ctzll(m);
    }
    if (w < 0) return;
  }
  const int* const rec = work.rec + 4 * w;
  const int b = rec[0];
  if (b < 0) return;
  const RowShape shape = row_shape<ROWS>(p.heads);
  const int item = rec[1], all = rec[2] - w + 2;  // ranges w - 1 .. rec[2]
  const int rr = WPR == 1 ? 4 * blockIdx.y + wave : blockIdx.y;
  constexpr int PER = R / 64, FIRST = 4;  // values of a lane; parts that are asked for at once
  const int each = (all + WPR - 1) / WPR, from = wave % WPR * each, parts = min(all - from, each);  // (none or less: none)
  auto row = [&](int i) { return (int64_t)(from + i == 0 ? 2 * w - 1 : 2 * (w - 1 + from + i)) * ROWS + rr; };
  // all that the first parts need is asked for before any of it is waited for (one after the other, 256 decodes of 128
  // heads: 29 us)
  float2 ml = {kNegBig, 0.f};
  f32x4 head[FIRST][PER / 4];
  if (parts > 0) {
    ml = *reinterpret_cast<const float2*>(work.ml + 2 * row(min(lane, parts - 1)));
#pragma unroll
    for (int k = 0; k < FIRST; ++k)
#pragma unroll
      for (int d = 0; d < PER / 4; ++d)
        head[k][d] = *reinterpret_cast<const f32x4*>(work.o + row(min(k, parts - 1)) * R + d * 256 + 4 * lane);
  }
  const SeqView v = seq_view(p, b, work.lo, work.hi);
  const int tok0 = item / shape.hs << shape.js, head0 = item % shape.hs * ROWS;
  const int heads = min(p.heads - head0, ROWS), tokens = min(1 << shape.js, v.n - tok0), j = rr / heads;
  if (j >= tokens) return;
  if (lane >= parts) ml = float2{kNegBig, 0.f};
  float top = kNegBig, sum = 0.f, o[PER] = {};
  for (int i0 = 0; i0 < parts; i0 += 64) {
    if (i0 > 0) {
      ml = float2{kNegBig, 0.f};
      if (i0 + lane < parts) ml = *reinterpret_cast<const float2*>(work.ml + 2 * row(i0 + lane));
    }
    float most = ml.x;
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) most = fmaxf(most, __shfl_xor(most, x));
    most = fmaxf(most, top);
    const float before = fast_exp2(top - most), f = fast_exp2(ml.x - most);
    float add = ml.y * f;
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) add += __shfl_xor(add, x);
    sum = fmaf(sum, before, add);
    top = most;
#pragma unroll
    for (int d = 0; d < PER; ++d) o[d] *= before;
    const int here = min(64, parts - i0);
    auto take = [&](int i, auto count) {
      constexpr int N = decltype(count)::value;
      f32x4 x[N][PER / 4];
#pragma unroll
      for (int k = 0; k < N; ++k)
#pragma unroll
        for (int d = 0; d < PER / 4; ++d)
          x[k][d] = *reinterpret_cast<const f32x4*>(work.o + row(i0 + i + k) * R + d * 256 + 4 * lane);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float fk = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), i + k));
#pragma unroll
        for (int d = 0; d < PER; ++d) o[d] = fmaf(x[k][d >> 2][d & 3], fk, o[d]);
      }
    };
    int i = 0;
    if (i0 == 0) {
#pragma unroll
      for (int k = 0; k < FIRST; ++k) {
        if (k >= here) continue;
        const float fk = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), k));
#pragma unroll
        for (int d = 0; d < PER; ++d) o[d] = fmaf(head[k][d >> 2][d & 3], fk, o[d]);
      }
      i = min(FIRST, here);
    }
    for (; i + 8 <= here; i += 8) take(i, std::integral_constant<int, 8>{});
    if (here - i >= 4) take(i, std::integral_constant<int, 4>{}), i += 4;
    if (here - i >= 2) take(i, std::integral_constant<int, 2>{}), i += 2;
    if (here > i) take(i, std::integral_constant<int, 1>{});
  }
  T* const out = (T*)p.out + (p.cu ? 0 : b * p.o_sb) + (v.start + tok0 + j) * p.o_st + (head0 + rr - j * heads) * p.o_sh;
  if constexpr (WPR > 1) {  // the waves' sums, in their order
    __shared__ float s_o[WPR][R];
    __shared__ float2 s_ml[WPR];
#pragma unroll
    for (int d = 0; d < PER; d += 4)
      *reinterpret_cast<f32x4*>(&s_o[wave][d * 64 + 4 * lane]) = f32x4{o[d], o[d + 1], o[d + 2], o[d + 3]};
    if (lane == 0) s_ml[wave] = float2{top, sum};
    __syncthreads();
    if ((int)threadIdx.x >= R / 2) return;
    float most = kNegBig;
#pragma unroll
    for (int k = 0; k < WPR; ++k) most = fmaxf(most, s_ml[k].x);
    float2 y = {0.f, 0.f};
    sum = 0.f;
#pragma unroll
    for (int k = 0; k < WPR; ++k) {
      const float f = fast_exp2(s_ml[k].x - most);
      const float2 x = *reinterpret_cast<const float2*>(&s_o[k][2 * threadIdx.x]);
      sum = fmaf(s_ml[k].y, f, sum);
      y.x = fmaf(x.x, f, y.x), y.y = fmaf(x.y, f, y.y);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const uint32_t w = Elem<T>::pack2(y.x * inv, y.y * inv);
    __builtin_memcpy(out + 2 * threadIdx.x, &w, 4);
  } else {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int d = 0; d < PER; d += 4) {
      const u32x2 w = {Elem<T>::pack2(o[d] * inv, o[d + 1] * inv), Elem<T>::pack2(o[d + 2] * inv, o[d + 3] * inv)};
      __builtin_memcpy(out + d * 64 + 4 * lane, &w, 8);
    }
  }
}

// ---- host ---------------------------------------------------------------------------------------

constexpr int64_t kAlign = 256, kFewRows = 2048;
int64_t up(int64_t n) { return (n + kAlign - 1) / kAlign * kAlign; }

int64_t part_bytes(int rows, int r) {
  const int64_t groups = ss_host::device_cu_count();
  return up(groups * 2 * rows * r * 4) + up(groups * 2 * rows * 2 * 4) + up(groups * 4 * 4);
}

template <typename C>
LatentWork work_of(char* ws, int lo, int hi) {
  const int64_t groups = ss_host::device_cu_count();
  LatentWork work;
  work.o = (float*)ws;
  work.ml = (float*)(ws + up(groups * 2 * C::ROWS * C::R * 4));
  work.rec = (int*)((char*)work.ml + up(groups * 2 * C::ROWS * 2 * 4));
  work.lo = lo, work.hi = hi;
  return work;
}

template <typename T, typename C>
int launch_merge(const LatentParams& p, const LatentWork& work, hipStream_t stream) {
  constexpr int R = C::R;
  const int64_t groups = ss_host::device_cu_count();
  // Many items are cut once or twice each: a wave a row (of 256 decodes of 128 heads). Few are cut often: sixteen
  // waves a row, and no more workgroups than there may be items.
  const RowShape shape = row_shape<C::ROWS>(p.heads);
  const int64_t tiles = p.cu ? (int64_t)p.batch + (p.total >> shape.js) : (int64_t)p.batch * (((p.tq - 1) >> shape.js) + 1);
  if (tiles * shape.hs * C::ROWS <= kFewRows)
    hipLaunchKernelGGL((latent_merge_kernel<T, R, C::ROWS, 16>), dim3((unsigned)(tiles * shape.hs), C::ROWS), dim3(1024), 0,
                       stream, p, work, (int)groups);
  else
    hipLaunchKernelGGL((latent_merge_kernel<T, R, C::ROWS, 1>), dim3((unsigned)groups, C::ROWS / 4), dim3(256), 0, stream,
                       p, work, (int)groups);
  return ss_host::launch_status("latent attention (merge)");
}

template <typename T, typename C>
int launch_rows(const LatentParams& p, int lo, int hi, char* ws, hipStream_t stream) {
  const LatentWork work = work_of<C>(ws, lo, hi);
  auto kern = latent_tile_kernel<T, C>;
  static std::atomic<uint64_t> done{0};
  if (const int st = reserve_lds((const void*)kern, C::LDS, done); st != SS_OK) return st;
  hipLaunchKernelGGL(kern, dim3((unsigned)ss_host::device_cu_count()), dim3(64 * C::NW), C::LDS, stream, p, work);
  if (const int st = ss_host::launch_status("latent attention"); st != SS_OK) return st;
  return launch_merge<T, C>(p, work, stream);
}

template <typename T, typename F, typename M>
int launch_mixed(const LatentParams& p, int lo, char* ws, hipStream_t stream) {
  const LatentWork few = work_of<F>(ws, 0, lo), many = work_of<M>(ws + part_bytes(F::ROWS, F::R), lo, 0x7FFFFFFF);
  constexpr int lds = F::LDS > M::LDS ? F::LDS : M::LDS;
  auto kern = latent_mixed_kernel<T, F, M>;
  static std::atomic<uint64_t> done{0};
  if (const int st = reserve_lds((const void*)kern, lds, done); st != SS_OK) return st;
  hipLaunchKernelGGL(kern, dim3((unsigned)ss_host::device_cu_count()), dim3(256), lds, stream, p, few, many);
  if (const int st = ss_host::launch_status("latent attention (mixed)"); st != SS_OK) return st;
  if (const int st = launch_merge<T, F>(p, few, stream); st != SS_OK) return st;
  return launch_merge<T, M>(p, many, stream);
}

template <typename T, int R>
int launch_for(const LatentParams& p, int rows, int lo, int hi, char* ws, hipStream_t stream) {
  if (rows <= 16) return launch_rows<T, LatTile<R, 1, 4>>(p, lo, hi, ws, stream);
  if (rows <= 32) return launch_rows<T, LatTile<R, 2, 4>>(p, lo, hi, ws, stream);
  if (rows <= 64) return launch_rows<T, LatTile<R, 4, 8>>(p, lo, hi, ws, stream);
  return launch_rows<T, LatWide<R>>(p, lo, hi, ws, stream);
}

// Rows of the launches of a call: of sequences of few rows (0: no such launch), and of the others. Where
// some sequences are shorter than the longest, those of one token take tiles of one token's heads.
void plan_rows(int64_t batch, int64_t total, int tq, int heads, int& few, int& many) {
  const int64_t rows = (int64_t)(tq < 1 ? 1 : tq) * heads;
  many = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
  few = tq > 1 && total < batch * tq && heads <= 64 ? (heads <= 16 ? 16 : heads <= 32 ? 32 : 64) : 0;
  if (few >= many) few = 0;
}

}  // namespace

bool latent_tile_takes(const LatentParams& p, int dtype) {
  const bool pow2 = (p.block_size & (p.block_size - 1)) == 0;
  if (dtype != SS_DTYPE_BF16 && dtype != SS_DTYPE_F16) return false;
  if ((p.key_dim != 512 && p.key_dim != 256) || p.rope_dim != kRopeDim || !pow2 || p.block_size < 8) return false;
  if (p.max_blocks < 1 || p.scale_log2 == 0.f) return false;  // (masked scores are -inf, times the scale)
  for (int64_t s : {p.q_sb, p.q_st, p.q_sh, p.kv_s0, p.kv_s1})
    if (s % 8) return false;
  return ((uintptr_t)p.q | (uintptr_t)p.kv) % 16 == 0 &&
         p.kv_s1 >= p.key_dim + p.rope_dim && p.block_size * p.kv_s1 < (1 << 29) && p.kv_s0 >= 0 &&
         p.num_blocks < (1ll << 31);
}

int64_t latent_tile_bytes(int64_t batch, int64_t total, int tq, int heads, int latent_dim) {
  int few, many;
  plan_rows(batch, total, tq, heads, few, many);
  return part_bytes(many, latent_dim) + (few ? part_bytes(few, latent_dim) : 0);
}

int launch_latent_tile(const LatentParams& p, int dtype, char* ws, hipStream_t stream) {
  int few, many;
  plan_rows(p.batch, p.cu ? p.total : (int64_t)p.batch * p.tq, p.tq, p.heads, few, many);
  constexpr int kAll = 0x7FFFFFFF;
  const int lo = few ? p.heads : 0;  // the first launch's sequences: of one token
#define LATENT_LAUNCH(T, R)                                                                           \
  do {                                                                                                \
    if (few == 16 && many == 128) return launch_mixed<T, LatTile<R, 1, 4>, LatWide<R>>(p, lo, ws, stream); \
    if (few == 32 && many == 128) return launch_mixed<T, LatTile<R, 2, 4>, LatWide<R>>(p, lo, ws, stream); \
    if (few)                                                                                          \
      if (const int st = launch_for<T, R>(p, few, 0, lo, ws, stream); st != SS_OK) return st;         \
    return launch_for<T, R>(p, many, lo, kAll, ws + (few ? part_bytes(few, R) : 0), stream);          \
  } while (0)
  if (dtype == SS_DTYPE_BF16) {
    if (p.key_dim == 512) LATENT_LAUNCH(bf16_t, 512);
    LATENT_LAUNCH(bf16_t, 256);
  }
  if (p.key_dim == 512) LATENT_LAUNCH(f16_t, 512);
  LATENT_LAUNCH(f16_t, 256);
#undef LATENT_LAUNCH
}

}  // namespace ss
