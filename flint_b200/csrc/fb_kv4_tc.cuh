// Attention of many query rows over the paged 4-bit cache on the 5th-generation tensor cores (tcgen05): prompts and large trees.
//
// A CTA takes 256 query rows (row = token * R + head of the group) of a sequence and kv head as two tiles of 128 (or 128 rows, where the SMs are not filled otherwise), and its
// task's positions in steps of 128 (two pages). Per step and tile: S[128 rows][128 positions] = Q K^T into tensor memory, softmax by a warpgroup (a thread a row: no shuffles), P back
// into tensor memory over S, O[128][HD] += P V. Tensor pipe and exponentials (16 a clock and SM) need the same 1024 clocks a tile and step at heads of 128, so the two
// tiles take turns: one multiplies while the other exponentiates. Keys and values are dequantised once for both tiles by six warps into the K-major
// 128-byte-swizzle layout that the MMA reads, K as [position][dim], V as [dim][position], each number (nib - 8) s + z rounded once. (Operands nib - 8, with s and z in the
// softmax as kv4_attn_few has them, would be exact, but cost the softmax, which is what bounds this kernel, twice its instructions.)
// Operands are fp16, half a step 2^-11: K times a power of two per step (per position where the keys of its 128 positions are more than 2^23 apart), Q times one per row, P times 2^7,
// V as it is. A page with a row of V whose values fp16 does not hold to 2^-11 of the largest one (below about 2^-13, and from 2^15 on) has its V and P in bf16, half a step 2^-8: there
// rows of any size stand side by side, whatever their weight. Outputs are off by 0.0017 of their 2-norm, which is the rounding of the output itself. (bf16 throughout takes 9 % less
// time: no look at the factors, no second form of P; but outputs are off by 0.0044. The factors converted in place by the warp that brings the pages: 10 % more, it has no
// more than a step's time.) Sums and maxima are fp32. The maximum is moved, and O rescaled, only when a score exceeds it by more than 2^8.
// 1000 tokens of 32 heads of 128 behind 7011 positions: 168 us, 735 TFLOP/s. No unit is full (tensor pipe 42 % of the time on a busy SM, exponentials 54 %): a tile's chain scores, maximum,
// exponentials, P, PV is longer than what the other tile hides. Times move by up to 5 % with where the compiler places code that never runs.
// Warps: 0..3 and 4..7 softmax of tiles 0 and 1 (and Q in, O out), 8..13 dequantise, 14 brings pages (one bulk copy each), 15 issues MMAs.
#pragma once
#include "fb_kv4.cuh"
#include "fb_kv4_geometry.hpp"
#include "fb_tcgen.cuh"

namespace fb {

constexpr int kManyThreads = 16 * 32;
constexpr float kManyLift = 7.f;                   // probabilities are 2^7 times what they are, 2^15 at most: in fp16 they lose nothing down to 2^-21
constexpr int kManyDequant = 6;                    // warps that dequantise

template <int HD>
struct Kv4Many {
  static constexpr int REC = Kv4<HD>::REC, NB = HD == 64 ? 1 : 2;           // blocks of 64 dims of a K-major tile
  static constexpr int QT = NB * 128 * 128, KT = NB * kManyStep * 128, VT = HD * 128;      // bytes: Q tile, K step, V page
  static constexpr int ND = 4;                                              // steps whose notes are kept: softmax may be at i when step i + 2 is dequantised
  static constexpr int NR = 4;                                              // pages: two being dequantised, two on their way
  static constexpr int Q = 0, K = Q + 2 * QT, V = K + 2 * KT, RAW = V + 4 * VT, BAR = RAW + NR * REC;
  static constexpr int BARS = 2 * NR + 17, TOTAL = BAR + BARS * 8 + 2 * ND * 8 + (2 + 2 + NR + 2 * ND) * 4 + ND * kManyStep;       // barriers, then what stands behind them in the kernel
  static constexpr int T_S = 0, T_O = 256, TCOLS = 512;                     // tensor memory columns: two S / P, two O
  static_assert(TOTAL <= 227 * 1024 && T_O + 2 * HD <= TCOLS && QT % 1024 == 0 && VT % 1024 == 0 && RAW % 16 == 0 && REC % 16 == 0, "plan");
};

__device__ __forceinline__ __nv_bfloat162 kv4_bf2(uint32_t v) { return *reinterpret_cast<const __nv_bfloat162*>(&v); }
// nibbles in bits 0..3 and 16..19. A row that reaches the largest number rounds past it: not to an infinity, which would be NaN where the probability is 0
__device__ __forceinline__ uint32_t kv4_dequant2(uint32_t w, __nv_bfloat162 s, __nv_bfloat162 z) {
  const __nv_bfloat162 r = __hfma2(__hsub2(kv4_bf2((w & 0x000F000Fu) | 0x43004300u), kv4_bf2(0x43084308u)), s, z),        // 128 + nib - 136
                       c = __hmax2(__hmin2(r, kv4_bf2(0x7f7f7f7fu)), kv4_bf2(0xff7fff7fu));
  return *reinterpret_cast<const uint32_t*>(&c);
}
// ... fp16, nibbles in bits 0..3 and 16..19, or 4..7 and 20..23 (nib - 8 is exact, one rounding follows)
__device__ __forceinline__ __half2 kv4_h2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
__device__ __forceinline__ uint32_t kv4_half_lo(uint32_t w, __half2 s, __half2 z) {
  const __half2 r = __hfma2(__hsub2(kv4_h2((w & 0x000F000Fu) | 0x64006400u), kv4_h2(0x64086408u)), s, z);
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t kv4_half_hi(uint32_t w, __half2 s, __half2 z) {
  const __half2 r = __hfma2(__hfma2(kv4_h2((w & 0x00F000F0u) | 0x64006400u), kv4_h2(0x2C002C00u), kv4_h2(0xD480D480u)), s, z);
  return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// two floats in a register pair, an instruction for both
__device__ __forceinline__ uint64_t f32x2(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float2 f32x2_of(uint64_t v) {
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(v));
  return d;
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// after a failure: the copies in flight, and the MMAs, half a step's that nothing was committed for among them
template <int NR>
inline __device__ __noinline__ void many_drain(uint64_t* raw_full, uint64_t* pv_done, volatile int* s_issued) {
  drain_ring<NR>(raw_full, (uint32_t)s_issued[0]);
  drain_commit_order((uint32_t)s_issued[1], [=](uint32_t parity) { drain_phase(pv_done, parity); __syncwarp(); },
                     [=] { if (elect_one()) tc_commit(pv_done); __syncwarp(); });
}

template <int HD, int ROWS>
__global__ void __launch_bounds__(kManyThreads, 1) kv4_attn_many(const Kv4Attend P) {
  using C = Kv4<HD>;
  using M = Kv4Many<HD>;
  constexpr int NR = M::NR, REC = M::REC, KS = HD / 16;
  extern __shared__ __align__(1024) uint8_t many_sm[];                // the swizzle is a function of the address: tiles start on 1024-byte boundaries
  uint8_t* const sm = many_sm;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + M::BAR);
  uint64_t *raw_full = bars, *raw_empty = raw_full + NR, *k_full = raw_empty + NR, *k_empty = k_full + 2, *v_full = k_empty + 2, *v_empty = v_full + 2,
           *s_full = v_empty + 2, *p_full = s_full + 2, *pv_done = p_full + 4, *q_full = pv_done + 2;
  unsigned long long* s_bad = reinterpret_cast<unsigned long long*>(bars + M::BARS);   // [ND steps][2 pages] positions whose V is NaN
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(s_bad + 2 * M::ND);
  volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
  volatile int* s_issued = s_abort + 1;                          // [2] pages, PV of tile 0
  volatile int* s_none = s_issued + 2;                           // [NR] the page does not exist
  volatile int* s_gone = s_none + NR;                            // [ND steps] bit p: page p of the step does not exist, bit 2 + p: it is wide, bit 4: keys have powers of two of their own
  volatile float* s_kscale = reinterpret_cast<volatile float*>(s_gone + M::ND);  // [ND steps] inverse of the power of two of the keys
  uint8_t* s_kown = reinterpret_cast<uint8_t*>(const_cast<float*>(s_kscale + M::ND));      // [ND steps][positions] bit 4: its exponent
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Kv4Seqs& S = P.S;
  pdl_begin(true);
  Kv4Task<ROWS, kManyStep> task;
  if (!task.template find<false>(P, blockIdx.x, lane, blockIdx.x == 0 && warp == 0) || (task.n <= 0 && task.parts == 1)) return;
  const Kv4Seq& seq = task.seq;
  const int rows = task.rows - task.r0, tiles = ROWS > 128 && rows > 128 ? 2 : 1, n = max(task.n, 0), kvh = task.kvh, total = task.total;
  if (tid == 0) {
    for (int i = 0; i < NR; i++) { mbar_init(&raw_full[i], 1); mbar_init(&raw_empty[i], kManyDequant); }
    for (int i = 0; i < 2; i++) {
      mbar_init(&k_full[i], kManyDequant); mbar_init(&k_empty[i], 1); mbar_init(&v_full[i], kManyDequant); mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1); mbar_init(&p_full[2 * i], 4); mbar_init(&p_full[2 * i + 1], 4); mbar_init(&pv_done[i], 1);
    }
    mbar_init(q_full, 4 * tiles);
    *s_abort = 0;
    s_issued[0] = s_issued[1] = 0;
    mbar_fence_init();
  }
  if (warp == 15) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_tmem)), "r"(M::TCOLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  const WaitCtl wc{S.status, s_abort, P.spin_limit};
  bool ok = true;

  // The block's 512 x 128 registers are dealt out anew, 256 x 176 + 256 x 80: the softmax keeps a row's 128 scores
  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
  if (warp == 14) {
    // ---------------- pages, two a step; a page behind the last position or that the table does not have is left out
    int r = 0, issued = 0, page = 0;
    uint32_t lap = 1;
    const int pages = 2 * n, p_end = (total + kPage - 1) / kPage;
    for (; issued < pages && ok; issued++) {
      if ((issued & 31) == 0) {
        const int p = 2 * task.unit + issued + lane;
        page = issued + lane < pages && p < p_end ? kv4_page(S, task.b, p * kPage, true) : -1;
      }
      const int now = __shfl_sync(0xffffffffu, page, issued & 31);
      ok = __all_sync(0xffffffffu, mbar_wait(&raw_empty[r], lap, wc, W_EMPTY, 40));
      if (!ok) break;
      if (lane == 0) {
        s_none[r] = now < 0;
        if (now < 0) {
          mbar_arrive(&raw_full[r]);
        } else {
          mbar_expect_tx(&raw_full[r], REC);
          bulk_g2s(sm + M::RAW + r * REC, kv4_block<HD>(S, now, kvh, 0), REC, &raw_full[r]);
        }
      }
      if (++r == NR) { r = 0; lap ^= 1u; }
    }
    if (lane == 0) s_issued[0] = issued;
  } else if (warp == 15) {
    // ---------------- MMA issue: per tile PV of a step, then QK of the next one once PV has read P, which lies over S
    constexpr uint32_t idesc = (1u << 4) | ((128u >> 4) << 24), bf16 = (1u << 7) | (1u << 10);        // fp16 x fp16 (or bf16 x bf16) -> fp32, 128 rows
    const uint64_t q0 = tc_desc(smem_u32(sm + M::Q)), k0 = tc_desc(smem_u32(sm + M::K)), v0 = tc_desc(smem_u32(sm + M::V));
    auto qk = [&](auto tile, int i) {
      constexpr int t = decltype(tile)::value;
      if (elect_one()) {
        const uint64_t kb = k0 + (uint64_t)((i & 1) * (M::KT >> 4));
#pragma unroll
        for (int k = 0; k < KS; k++) {
          constexpr uint32_t id = idesc | ((128u >> 3) << 17);
          const uint64_t off = (uint64_t)(((k >> 2) * (128 * 128) + (k & 3) * 32) >> 4);
          tc_mma_ss(tmem + M::T_S + t * 128, q0 + (uint64_t)(t * (M::QT >> 4)) + off, kb + off, id, k ? 1u : 0u);
        }
        tc_commit(&s_full[t]);
        if (t == tiles - 1 && i + 2 < n) tc_commit(&k_empty[i & 1]);       // step i + 2 waits for it: none is issued that nobody waits for before the CTA ends
      }
      __syncwarp();
    };
    auto pv = [&](auto tile, auto part, int i) {                 // of the step's first or second page
      constexpr int t = decltype(tile)::value, h = decltype(part)::value;
      const uint32_t id = idesc | (s_gone[i & (M::ND - 1)] >> h & 4 ? bf16 : 0u) | ((uint32_t)(HD >> 3) << 17);
      if (elect_one()) {
        const uint64_t vb = v0 + (uint64_t)((i & 1) * (M::VT >> 3) + h * (M::VT >> 4));
#pragma unroll
        for (int k = 0; k < 4; k++) {
          tc_mma_ts(tmem + M::T_O + t * HD, tmem + M::T_S + t * 128 + (4 * h + k) * 8, vb + (uint64_t)((k * 32) >> 4), id, i || h || k ? 1u : 0u);
        }
        if (h) {
          tc_commit(&pv_done[t]);
          if (t == tiles - 1 && i + 2 < n) tc_commit(&v_empty[i & 1]);
        }
      }
      __syncwarp();
      if (t == 0 && h && lane == 0) s_issued[1] = i + 1;
    };
    auto wait = [&](uint64_t* bar, int i, int where) {           // phase i of a barrier
      ok = ok && __all_sync(0xffffffffu, mbar_wait(bar, (uint32_t)i & 1u, wc, W_FULL, where));
      tc_fence_after();
      return ok;
    };
    const std::integral_constant<int, 0> first;
    const std::integral_constant<int, 1> second;
    if (n > 0 && wait(q_full, 0, 41) && wait(&k_full[0], 0, 42)) {
      qk(first, 0);
      if (tiles > 1) qk(second, 0);
    }
    auto turn = [&](auto tile, int i) {
      constexpr int t = decltype(tile)::value;
      if (!wait(&p_full[2 * t], i, 43) || (t == 0 && !wait(&v_full[i & 1], i >> 1, 44))) return;
      pv(tile, first, i);
      if (!wait(&p_full[2 * t + 1], i, 43)) return;
      pv(tile, second, i);
      if (i + 1 == n || (t == 0 && !wait(&k_full[(i + 1) & 1], (i + 1) >> 1, 45)) || !wait(&pv_done[t], i, 46)) return;
      qk(tile, i + 1);
    };
    for (int i = 0; i < n && ok; i++) {
      turn(first, i);
      if (tiles > 1 && ok) turn(second, i);
    }
  } else {
    // ---------------- dequantise: K of a step's two pages, then V, in turns of a warp. K: lanes of a turn take two words each, 16 dims of a position;
    // V: four words, four dims of eight positions. K's place is free once QK of two steps ago has read it, V's once PV has.
    // The turns of both pages are dealt out to the warps together. (Unrolled, they do not fit 80 registers: 160 us of 1000 tokens behind 7011 became 204.)
    const int dw = warp - 8;
    constexpr int QN = C::MAIN / 32, PT = 32 / QN, KTURNS = kPage / PT, VTURNS = C::MAIN / 16;       // lanes of a position, positions of a turn, turns of a page
    float kf = 1.f;                                              // the step's power of two of the keys
    auto key = [&](const uint8_t* rec, uint8_t* kt, int p, int w0, auto words, auto apart, uint8_t* own) {           // words w0 .. of position p
      constexpr int NWD = decltype(words)::value;
      const uint8_t* blk = rec + (p >> 4) * C::BLOCK;
      uint32_t x[NWD];
      if (NWD == 4) {
        const uint4 w = *reinterpret_cast<const uint4*>(blk + C::k_word(p & 15, w0));
        x[0] = w.x; x[1] = w.y; x[NWD - 2] = w.z; x[NWD - 1] = w.w;
      } else {
        const uint2 w = *reinterpret_cast<const uint2*>(blk + C::k_word(p & 15, w0));
        x[0] = w.x; x[1] = w.y;
      }
      const uint32_t sz = *reinterpret_cast<const uint32_t*>(blk + C::KSZ + (p & 15) * 4);
      float by = kf;
      if (decltype(apart)::value) {                              // a power of two of the position's own
        const float2 f = pow2_for(fmaf(8.f, fabsf(bflo(sz)), fabsf(bfhi(sz))));
        by = f.x;
        if (w0 == 0) own[p] = (uint8_t)(__float_as_uint(f.y) >> 23);
      }
      const uint32_t f = cvt_f16x2(bflo(sz) * by, bfhi(sz) * by);
      const __half2 s = kv4_h2(__byte_perm(f, f, 0x1010)), z = kv4_h2(__byte_perm(f, f, 0x3232));
      uint8_t* row = kt + (w0 >> 3) * (kManyStep * 128) + p * 128;
#pragma unroll
      for (int e = 0; e < NWD; e++)
        *reinterpret_cast<uint4*>(row + ((((w0 + e) & 7) ^ (p & 7)) << 4)) =
            make_uint4(kv4_half_lo(x[e], s, z), kv4_half_hi(x[e], s, z), kv4_half_lo(x[e] >> 8, s, z), kv4_half_hi(x[e] >> 8, s, z));
    };
    auto value = [&](const uint8_t* rec, uint8_t* vt, int c, int w, int left, bool wide, auto special) {        // dims 4w .. 4w+3 of positions 8c .. 8c+7
      const uint8_t* blk = rec + (c >> 1) * C::BLOCK;
      uint32_t out[4][4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int u = (c & 1) * 4 + k;
        const uint32_t x = *reinterpret_cast<const uint32_t*>(blk + C::v_word(u, w));
        uint2 sz = *reinterpret_cast<const uint2*>(blk + C::VSZ + u * 8);
        if (decltype(special)::value) {
          if (8 * c + 2 * k >= left || !(bflo(sz.x) < INFINITY)) sz.x = 0;
          if (8 * c + 2 * k + 1 >= left || !(bflo(sz.y) < INFINITY)) sz.y = 0;
        }
        if (decltype(special)::value && wide) {
          const __nv_bfloat162 s = kv4_bf2(__byte_perm(sz.x, sz.y, 0x5410)), z = kv4_bf2(__byte_perm(sz.x, sz.y, 0x7632));
#pragma unroll
          for (int e = 0; e < 4; e++) out[e][k] = kv4_dequant2(x >> (4 * e), s, z);
        } else {
          const __half2 s = kv4_h2(cvt_f16x2(bflo(sz.x), bflo(sz.y))), z = kv4_h2(cvt_f16x2(bfhi(sz.x), bfhi(sz.y)));
          out[0][k] = kv4_half_lo(x, s, z);
          out[1][k] = kv4_half_hi(x, s, z);
          out[2][k] = kv4_half_lo(x >> 8, s, z);
          out[3][k] = kv4_half_hi(x >> 8, s, z);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int d = 4 * w + e;
        *reinterpret_cast<uint4*>(vt + d * 128 + ((c ^ (d & 7)) << 4)) = make_uint4(out[e][0], out[e][1], out[e][2], out[e][3]);
      }
    };
    // a V turn: a phase of eight lanes stores to eight chunks; four chunks' lanes read words of different bank groups
    const int ci = (lane >> 1) & 3, wi = (lane & 1) | (lane >> 3) << 1;
    auto chunk_of = [&](int j) { return 4 * (j & 1) + ci; };
    auto word_of = [&](int j) { return 8 * (((j >> 1) + ci) & (VTURNS / 2 - 1)) + wi; };
    const std::integral_constant<int, 4> four;
    const std::integral_constant<int, 2> two;
    int r = 0;
    uint32_t lap = 0;
    for (int i = 0; i < n && ok; i++) {
      const int b = i & 1;
      const uint32_t before = (uint32_t)((i >> 1) - 1) & 1u;
      if (i >= 2) ok = __all_sync(0xffffffffu, mbar_wait(&k_empty[b], before, wc, W_EMPTY, 47));
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&raw_full[r], lap, wc, W_FULL, 49) && mbar_wait(&raw_full[r + 1], lap, wc, W_FULL, 49));
      if (!ok) break;
      const uint8_t *rec0 = sm + M::RAW + r * REC, *rec1 = rec0 + REC;
      uint8_t *kt = sm + M::K + b * M::KT, *vt = sm + M::V + 2 * b * M::VT;
      const int left0 = total - (task.unit + i) * kManyStep, left1 = left0 - kPage;                // positions of the pages that exist
      const bool none0 = s_none[r] != 0, none1 = s_none[r + 1] != 0 || left1 <= 0;
      // Positions whose V is NaN: those, and what lies behind the last position, become zeros, as every row of P multiplies them. A page is `wide`
      // whose rows of V have bounds 8 |s| + |z| (what a value may be at most, 17/15 of the largest one at most) beyond [2^-13, 2^15): half a step of fp16's smallest, 2^-25, is 2^-11
      // of a row's largest value there. s has to be exact in fp16, as it is from 2^-17 on; below, what it is off by counts eight times, and the bound starts at 2^-10. kmost, kleast: the largest bound of a key, the smallest but 0.
      uint32_t kmost = 0, kleast = 0x7f800000u;
      bool wide0 = false, wide1 = false;
      auto look = [&](const uint8_t* rec, int left, bool& wide) {
        uint32_t bad[2];
#pragma unroll
        for (int k = 0; k < 2; k++) {
          const uint8_t* at = rec + (2 * k + (lane >> 4)) * C::BLOCK + (lane & 15) * 4;
          const uint32_t a = *reinterpret_cast<const uint32_t*>(at + C::KSZ), c = *reinterpret_cast<const uint32_t*>(at + C::VSZ);
          const bool in = 32 * k + lane < left, num = bflo(c) < INFINITY;
          const float kb = fmaf(8.f, fabsf(bflo(a)), fabsf(bfhi(a))), vb = fmaf(8.f, fabsf(bflo(c)), fabsf(bfhi(c)));
          if (in && kb < INFINITY) {
            kmost = max(kmost, __float_as_uint(kb));
            if (kb > 0.f) kleast = min(kleast, __float_as_uint(kb));
          }
          bad[k] = __ballot_sync(0xffffffffu, in && !num);
          const float vsa = fabsf(bflo(c)), low = vsa == 0.f || vsa >= 0x1p-17f ? 0x1p-13f : 0x1p-10f;
          wide |= __any_sync(0xffffffffu, in && num && vb != 0.f && !(vb >= low && vb < 0x1p15f)) != 0;
        }
        return (unsigned long long)bad[0] | (unsigned long long)bad[1] << 32;
      };
      // The usual case at a glance: whole pages, all factors within narrower bounds than that: s of V from 2^-13 to below 2^11, |z| below 2^14, of K s from 2^-12 on and
      // the same above.
      unsigned long long bad0 = 0, bad1 = 0;
      bool looked = false;
      {
        const uint8_t* at = rec0 + (lane >> 4) * C::BLOCK + (lane & 15) * 4;
        uint32_t km = 0, vm = 0, ks = 0xffffu, vs = 0xffffu;
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const uint32_t a = *reinterpret_cast<const uint32_t*>(at + (k >> 1) * REC + 2 * (k & 1) * C::BLOCK + C::KSZ) & 0x7fff7fffu,
                         c = *reinterpret_cast<const uint32_t*>(at + (k >> 1) * REC + 2 * (k & 1) * C::BLOCK + C::VSZ) & 0x7fff7fffu;
          km = __vmaxu2(km, a);
          vm = __vmaxu2(vm, c);
          ks = min(ks, a & 0xffffu);
          vs = min(vs, c & 0xffffu);
        }
        const bool usual = __vmaxu2(__vmaxu2(km, vm), 0x467f44ffu) == 0x467f44ffu && vs >= 0x3900u && ks >= 0x3980u;
        if (__all_sync(0xffffffffu, usual) && !none0 && !none1 && left1 >= kPage) {
          kmost = __float_as_uint(fmaf(8.f, bflo(km), bfhi(km)));
        } else {
          looked = true;
          if (!none0) bad0 = look(rec0, left0, wide0);
          if (!none1) bad1 = look(rec1, left1, wide1);
        }
      }
      // One power of two does for keys whose bounds are 2^24 apart or less (fp16 then holds them from 2^-10 on); beyond that each has its own, so that a key
      // that is not seen, or as nothing to the softmax, takes no bits from the others.
      const uint32_t kmax = __reduce_max_sync(0xffffffffu, kmost);
      const bool apart = looked && __any_sync(0xffffffffu, (kmax >> 23) > (kleast >> 23) + 23u);
      const float2 kp = pow2_for(__uint_as_float(kmax));         // the largest into [2^14, 2^15)
      kf = kp.x;
      const bool special = none0 || none1 || bad0 || bad1 || left1 < kPage || wide0 || wide1;
      if (dw == 0 && lane == 0) {
        // Their place was step i - 4's: the softmax of that one has read it, as PV of step i - 3 has ended (the wait for V's place of the step before)
        const int note = i & (M::ND - 1);
        s_bad[2 * note] = bad0;
        s_bad[2 * note + 1] = bad1;
        s_gone[note] = (none0 ? 1 : 0) | (none1 ? 2 : 0) | (wide0 ? 4 : 0) | (wide1 ? 8 : 0) | (apart ? 16 : 0);
        s_kscale[note] = apart ? 1.f : kp.y;
      }
      if (!none0 && !none1 && !apart) {
#pragma unroll 1
        for (int it = dw; it < 2 * KTURNS; it += kManyDequant) {
          const int h = it / KTURNS, j = it % KTURNS;
          key(h ? rec1 : rec0, kt + h * (kPage * 128), j * PT + lane / QN, 4 * (lane & (QN - 1)), four, std::false_type(), nullptr);
        }
        if (HD == 80 && dw >= 2) key(dw < 4 ? rec0 : rec1, kt + (dw < 4 ? 0 : kPage * 128), (dw & 1) * 32 + lane, 8, two, std::false_type(), nullptr);
      } else {
        auto page = [&](int h, auto a) {
          uint8_t* own = s_kown + (i & (M::ND - 1)) * kManyStep + h * kPage;
#pragma unroll 1
          for (int j = dw; j < KTURNS; j += kManyDequant) key(h ? rec1 : rec0, kt + h * (kPage * 128), j * PT + lane / QN, 4 * (lane & (QN - 1)), four, a, own);
          if (HD == 80 && dw < 2) key(h ? rec1 : rec0, kt + h * (kPage * 128), dw * 32 + lane, 8, two, a, own);
        };
        for (int h = 0; h < 2; h++) {
          if (h ? none1 : none0) continue;
          if (apart) page(h, std::true_type());
          else page(h, std::false_type());
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&k_full[b]);
      if (i >= 2) ok = __all_sync(0xffffffffu, mbar_wait(&v_empty[b], before, wc, W_EMPTY, 48));
      if (!ok) break;
      if (!special) {
#pragma unroll 1
        for (int it = (dw + 4) % kManyDequant; it < 2 * VTURNS; it += kManyDequant) {                // who had one K turn less begins
          const int h = it / VTURNS, j = it % VTURNS;
          value(h ? rec1 : rec0, vt + h * M::VT, chunk_of(j), word_of(j), 0, false, std::false_type());
        }
        if (HD == 80 && dw < 2) value(dw ? rec1 : rec0, vt + dw * M::VT, (lane >> 1) & 7, 16 + ((lane & 1) | (lane >> 4) << 1), 0, false, std::false_type());
      } else {
        for (int h = 0; h < 2; h++) {
          const uint8_t* rec = h ? rec1 : rec0;
          if (h ? none1 : none0) {
            for (int k = tid - 256; k < M::VT / 16; k += kManyDequant * 32) *reinterpret_cast<uint4*>(vt + h * M::VT + k * 16) = make_uint4(0, 0, 0, 0);
            continue;
          }
          const int left = h ? left1 : left0;
          for (int j = dw; j < VTURNS; j += kManyDequant) value(rec, vt + h * M::VT, chunk_of(j), word_of(j), left, h ? wide1 : wide0, std::true_type());
          if (HD == 80 && dw == 5) value(rec, vt + h * M::VT, (lane >> 1) & 7, 16 + ((lane & 1) | (lane >> 4) << 1), left, h ? wide1 : wide0, std::true_type());
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) { mbar_arrive(&raw_empty[r]); mbar_arrive(&raw_empty[r + 1]); mbar_arrive(&v_full[b]); }
      r += 2;
      if (r == NR) { r = 0; lap ^= 1u; }
    }
  }
  } else {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
  if (warp >> 2 < tiles) {
    // ---------------- softmax of tile t: thread = row
    const int t = warp >> 2, row = tid & 127, lr = t * 128 + row, R = P.R;
    const uint32_t tl = tmem + ((uint32_t)((warp & 3) * 32) << 16), ts = tl + M::T_S + t * 128, to = tl + M::T_O + t * HD;
    const bool live = lr < rows;
    const int gr = task.r0 + min(lr, rows - 1), mq = gr / R, head = kvh * R + gr % R;
    float cs = fabsf(P.scale);
    {                                                            // Q: the row, as fp16 times a power of two, into the swizzled tile; a negative scale is a negative Q
      const uint16_t* src = P.q + (size_t)(seq.first + mq) * P.q_ld + (size_t)head * HD;
      const uint32_t flip = P.scale < 0.f ? 0x80008000u : 0u;
      uint8_t* qt = sm + M::Q + t * M::QT + row * 128;
      uint32_t w[HD / 2], most = 0;
#pragma unroll
      for (int c = 0; c < HD / 8; c++) {
        const uint4 v = live ? *reinterpret_cast<const uint4*>(src + 8 * c) : make_uint4(0, 0, 0, 0);
        w[4 * c] = v.x; w[4 * c + 1] = v.y; w[4 * c + 2] = v.z; w[4 * c + 3] = v.w;
      }
#pragma unroll
      for (int k = 0; k < HD / 2; k++) most = __vmaxu2(most, w[k] & 0x7fff7fffu);
      const float2 f = pow2_for(__uint_as_float(max(most & 0xffffu, most >> 16) << 16));
      cs *= f.y;
#pragma unroll
      for (int c = 0; c < HD / 8; c++) {
        auto half2_of = [&](uint32_t v) { return cvt_f16x2(bflo(v ^ flip) * f.x, bfhi(v ^ flip) * f.x); };
        *reinterpret_cast<uint4*>(qt + (c >> 3) * (128 * 128) + (((c & 7) ^ (row & 7)) << 4)) =
            make_uint4(half2_of(w[4 * c]), half2_of(w[4 * c + 1]), half2_of(w[4 * c + 2]), half2_of(w[4 * c + 3]));
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    const uint8_t* mask = P.amask ? P.amask + (size_t)(seq.first + mq) * P.mask_ld : nullptr;
    const int m_first = (task.r0 + min(t * 128 + (warp & 3) * 32, rows - 1)) / R;          // the warp's first token: what it sees, all rows see
    float m = kLowest, l = 0.f;
    // Exponents are a score's product with c2, not rounded, less m, which was: by less than half a power of two below 2^22. From there on products are rounded first.
    bool large = false;
    int plain = mask ? seq.cached : min(total, seq.cached + m_first + 1);                 // steps that end here or before need no look at what is seen; large: none
    for (int i = 0; i < n; i++) {
      ok = __all_sync(0xffffffffu, mbar_wait(&s_full[t], (uint32_t)i & 1u, wc, W_FULL, 50));
      if (!ok) break;
      tc_fence_after();
      uint32_t v[4][32];                                         // the row's scores, then its probabilities, stay in registers
#pragma unroll
      for (int c = 0; c < 4; c++) tc_ld32(ts + c * 32, v[c]);
      const int p0 = (task.unit + i) * kManyStep, note = i & (M::ND - 1), gone = s_gone[note];
      float c2 = fmaxf(cs * s_kscale[note], 1.2e-38f);           // not zero: a score that is not seen stays -inf
      const unsigned long long bad0 = s_bad[2 * note], bad1 = s_bad[2 * note + 1];
      tc_ld_wait();
      if (p0 + kManyStep > plain || (gone & 19) || (bad0 | bad1)) {
        if (__builtin_expect(gone & 16, 0)) {
#pragma unroll
          for (int c = 0; c < 4; c++)
#pragma unroll
            for (int e = 0; e < 32; e++) v[c][e] = __float_as_uint(__uint_as_float(v[c][e]) * __uint_as_float((uint32_t)s_kown[note * kManyStep + c * 32 + e] << 23));
        }
        if (__builtin_expect(large, 0)) {
#pragma unroll
          for (int c = 0; c < 4; c++)
#pragma unroll
            for (int e = 0; e < 32; e++) v[c][e] = __float_as_uint(__uint_as_float(v[c][e]) * c2);
          c2 = 1.f;
        }
        // what is not seen becomes -inf
        uint32_t vis[4];
#pragma unroll
        for (int c = 0; c < 4; c++) {
          const int q0 = p0 + 32 * c, lim = (mask ? min(total, seq.cached) : min(total, seq.cached + mq + 1)) - q0;
          vis[c] = lim >= 32 ? 0xffffffffu : (lim > 0 ? (1u << lim) - 1u : 0u);
          if (mask && lim < 32)
#pragma unroll 1
            for (int j = max(0, q0 - seq.cached); j < min(min(total, q0 + 32) - seq.cached, P.mask_ld); j++)
              vis[c] |= (mask[j] != 0 ? 1u : 0u) << (seq.cached + j - q0);
          if (gone >> (c >> 1) & 1) vis[c] = 0;
          if (vis[c] & (uint32_t)((c < 2 ? bad0 : bad1) >> (32 * (c & 1)))) l = __uint_as_float(0x7fc00000u);       // sees a row of V that is NaN
        }
#pragma unroll
        for (int c = 0; c < 4; c++)
#pragma unroll
          for (int e = 0; e < 32; e++)
            if (!(vis[c] & 1u << e)) v[c][e] = 0xff800000u;
        __syncwarp();
      }
      float mx[8];
#pragma unroll
      for (int k = 0; k < 8; k++) mx[k] = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; c++)
#pragma unroll
        for (int e = 0; e < 32; e += 2) mx[(e >> 1) & 7] = max3(mx[(e >> 1) & 7], __uint_as_float(v[c][e]), __uint_as_float(v[c][e + 1]));
      const float top = fmaxf(max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[4]), max3(mx[5], mx[6], mx[7])) * c2;
      if (__any_sync(0xffffffffu, top > m + 8.f)) {
        const float mn = fmaxf(m, top), corr = ex2(m - mn);
        if (!large && __any_sync(0xffffffffu, fabsf(mn) >= 0x1p22f && mn > kLowest)) {
          large = true;                                          // the step once more
          plain = 0;
          i--;
          continue;
        }
        if (i > 0) {                                             // O as the steps before left it
          ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[t], (uint32_t)(i - 1) & 1u, wc, W_FULL, 51));
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < HD; c += 8) {
            uint32_t x[8];
            tc_ld8(to + c, x);
            tc_ld_wait();
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = __float_as_uint(__uint_as_float(x[e]) * corr);
            tc_st8v(to + c, x);
          }
        }
        m = mn;
        l *= corr;
      }
      const uint64_t cs2 = f32x2(c2, c2), m2 = f32x2(kManyLift - m, kManyLift - m);
      uint64_t sum[4] = {0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < 4; c++) {
        uint32_t o[16];
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const float2 y = f32x2_of(fma_f32x2(f32x2(__uint_as_float(v[c][2 * e]), __uint_as_float(v[c][2 * e + 1])), cs2, m2));
          const float a = ex2(y.x), d = ex2(y.y);
          sum[e & 3] = add_f32x2(sum[e & 3], f32x2(a, d));
          o[e] = cvt_f16x2(a, d);
          v[c][2 * e] = __float_as_uint(a);
          v[c][2 * e + 1] = __float_as_uint(d);
        }
        tc_st16(ts + c * 16, o);
        if (c & 1) {                                             // a page's half of P is there
          tc_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0 && !(gone >> (c >> 1) & 4)) mbar_arrive(&p_full[2 * t + (c >> 1)]);
        }
      }
      if (gone & 12) {                                           // as bf16, by way of columns whose scores have been read: the usual path runs straight on (its second half's
                                                                 // exponentials during the first half's store)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          if (!(gone >> h & 4)) continue;
          tc_st32(ts + 64, v[2 * h]);
          tc_st32(ts + 96, v[2 * h + 1]);
          tc_st_wait();
#pragma unroll 1
          for (int k = 0; k < 64; k += 8) {
            uint32_t x[8];
            tc_ld8(ts + 64 + k, x);
            tc_ld_wait();
            tc_st4(ts + h * 32 + k / 2, pack_bf16(__uint_as_float(x[0]), __uint_as_float(x[1])), pack_bf16(__uint_as_float(x[2]), __uint_as_float(x[3])),
                   pack_bf16(__uint_as_float(x[4]), __uint_as_float(x[5])), pack_bf16(__uint_as_float(x[6]), __uint_as_float(x[7])));
          }
          tc_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[2 * t + h]);
        }
      }
      {
        const float2 y = f32x2_of(add_f32x2(add_f32x2(sum[0], sum[1]), add_f32x2(sum[2], sum[3])));
        l += y.x + y.y;
      }
    }
    if (ok && n > 0) ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[t], (uint32_t)(n - 1) & 1u, wc, W_FULL, 52));
    tc_fence_after();
    if (ok) {
      const float inv = task.parts > 1 ? 1.f : (l == 0.f ? 0.f : 1.f / l);
      uint16_t* out = P.out + (size_t)(seq.first + mq) * P.o_ld + (size_t)head * HD;
      float* w = task.parts > 1 ? P.work + ((size_t)blockIdx.x * ROWS + lr) * (HD + 4) : nullptr;
#pragma unroll 1
      for (int c = 0; c < HD; c += 16) {
        uint32_t v[16];
        if (n > 0) {
          tc_ld16(to + c, v);
          tc_ld_wait();
        } else {
#pragma unroll
          for (int e = 0; e < 16; e++) v[e] = 0;
        }
        float f[16];
#pragma unroll
        for (int e = 0; e < 16; e++) f[e] = l == 0.f ? 0.f : __uint_as_float(v[e]) * inv;
        if (!live) {
        } else if (w) {
#pragma unroll
          for (int e = 0; e < 16; e += 4) *reinterpret_cast<float4*>(w + c + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
        } else {
#pragma unroll
          for (int e = 0; e < 16; e += 8)
            *reinterpret_cast<uint4*>(out + c + e) =
                make_uint4(pack_bf16(f[e], f[e + 1]), pack_bf16(f[e + 2], f[e + 3]), pack_bf16(f[e + 4], f[e + 5]), pack_bf16(f[e + 6], f[e + 7]));
        }
        __syncwarp();
      }
      if (w && live) *reinterpret_cast<float2*>(w + HD) = make_float2(m - kManyLift, l);
    }
  }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 15) {
    if (*s_abort) many_drain<NR>(raw_full, pv_done, s_issued);
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(M::TCOLS));
  }
}

}  // namespace fb
