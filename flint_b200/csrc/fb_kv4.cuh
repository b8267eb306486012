// Paged K/V cache of 4 bits a number: layout, append (rotation and quantisation), read-back, moves, and the attention of few query rows over it.
//
// A row is the HD numbers of one position and kv head, of K or of V: HD nibbles and a bf16 pair (s, z). It stands for (nib - 8) * s + z, the int4
// weights' form (flint_b200/packing.py), with s = bf16((max - min) / 15), z = bf16(min + 8 s), nib = 8 + clamp(round((x - z) / s), -8, 7). A row that
// holds an infinity or a NaN, or whose range overflows, is a row of NaN (s = z = NaN).
// A page holds kPage positions: per kv head one record of four BLOCKS of 16 positions, each contiguous, so that one bulk copy brings any run of
// blocks of a page. A block: K's nibbles, V's nibbles, K's 16 pairs (s in the low half of a word), V's.
//   K  words of eight dims 8w .. 8w+7 of a position, the nibbles in the order that fb_vtc.cuh's conversion turns into ADJACENT pairs of dims; the words of a
//      position in a row, the main part (HD 128: all; else the first 64 dims) ahead of the tails of all positions. Four lanes of a quad read a position's row.
//   V  words of four dims 4w .. 4w+3 of TWO positions, the even one in the low half: the same conversion yields pairs of positions, which is what
//      the product with the probabilities contracts. Appending a position writes halves of words, never part of a byte that another position owns.
//      The words of a pair of positions in a row, tails behind, 16-byte (HD 128) or 32-byte (64) pieces exchanged by the pair's number so that the
//      lanes of a load, which hold four pairs each, meet no bank twice.
#pragma once
#include "fb_common.cuh"

namespace fb {

constexpr int kPage = 64;

template <int HD>
struct Kv4 {
  static_assert(HD == 64 || HD == 80 || HD == 128, "head sizes of the cache");
  static constexpr int MAIN = HD == 128 ? 128 : 64;                // dims whose words come first
  static constexpr int V = 8 * HD, KSZ = 16 * HD, VSZ = KSZ + 64, BLOCK = KSZ + 128, REC = BLOCK * (kPage / 16);
  // bytes inside a block (p: position 0..15)
  __host__ __device__ static constexpr int k_word(int p, int w) { return w < MAIN / 8 ? p * (MAIN / 2) + w * 4 : MAIN * 8 + p * ((HD - MAIN) / 2) + (w - MAIN / 8) * 4; }
  __host__ __device__ static constexpr int v_word(int u, int w) {  // u: pair of positions 0..7
    return V + (HD == 128 ? u * 128 + (((w >> 2) ^ (2 * (u & 3))) << 4) + (w & 3) * 4
                          : (w < 16 ? u * 64 + ((w * 4) ^ ((u >> 1 & 1) * 32)) : 512 + u * ((HD - MAIN) & 31) + (w - 16) * 4));
  }
};

// The sequences of a call. One sequence: start == nullptr, all T tokens are its. cached == nullptr: cached0 for every sequence.
struct Kv4Seqs {
  uint8_t* pool;             // [n_pages][nkv][record] of one layer
  const int* table;          // [n_seq][table_ld] pages
  const int *start, *cached;
  int cached0, n_pages, nkv, n_seq, table_ld, T;
  DevStatus* status;
};

enum Kv4Where { KV4_PAGE = 21, KV4_SLOT = 22, KV4_TOKENS = 23, KV4_PATH = 24 };

// a value from device memory that the call cannot use: reported (the first one stays), the access is left out
__device__ __forceinline__ void kv4_report(DevStatus* st, int where, int seq, int expected, int seen) {
  if (atomicCAS(&st->code, 0, 6 /*FB_ERR_RANGE*/) == 0) { st->where = where; st->layer = seq; st->block = (int)blockIdx.x; st->expected = expected; st->seen = seen; }
}

// What a sequence has: false where it has nothing to do or its numbers cannot be
struct Kv4Seq {
  int first, n, cached;
  __device__ __forceinline__ bool get(const Kv4Seqs& S, int b, bool report) {
    first = S.start ? S.start[b] : 0;
    const int end = S.start ? S.start[b + 1] : S.T;
    cached = S.cached ? S.cached[b] : S.cached0;
    n = end - first;
    if (first < 0 || end > S.T || end < first) {
      if (report) kv4_report(S.status, KV4_TOKENS, b, S.T, end);
      return false;
    }
    if (cached < 0 || (long long)cached + n > (long long)S.table_ld * kPage) {
      if (report) kv4_report(S.status, KV4_SLOT, b, S.table_ld * kPage, cached);
      return false;
    }
    return n > 0;
  }
};
// the page that holds a slot (below table_ld * kPage), or -1
__device__ __forceinline__ int kv4_page(const Kv4Seqs& S, int b, int slot, bool report) {
  const int page = __ldg(S.table + (size_t)b * S.table_ld + slot / kPage);
  if ((unsigned)page < (unsigned)S.n_pages) return page;
  if (report) kv4_report(S.status, KV4_PAGE, b, S.n_pages, page);
  return -1;
}
template <int HD>
__device__ __forceinline__ uint8_t* kv4_block(const Kv4Seqs& S, int page, int head, int slot) {
  return S.pool + ((size_t)page * S.nkv + head) * Kv4<HD>::REC + (slot % kPage / 16) * Kv4<HD>::BLOCK;
}
// The sequence of token m, found by a whole warp: how many sequences end at or before it. -1: behind the last one.
__device__ __forceinline__ int kv4_seq_of(const Kv4Seqs& S, int m, int lane) {
  if (!S.start) return 0;
  int b = 0;
  for (int i = 0; i < S.n_seq; i += 32) b += __popc(__ballot_sync(0xffffffffu, i + lane < S.n_seq && S.start[i + lane + 1] <= m));
  return b < S.n_seq ? b : -1;
}

// ------------------------------------------------------------------------------------------------ append
struct Kv4Append {
  Kv4Seqs S;
  const uint16_t *q, *k, *v;         // bf16 [T][heads][HD], tokens q_ld / k_ld / v_ld elements apart; q may be nullptr
  uint16_t* q_out;
  long long q_ld, k_ld, v_ld, qo_ld;
  const int* depth;                  // rotation position of a token behind its sequence's cached ones, or nullptr: its place
  const unsigned long long* freq;    // [HD / 2] turns per position in units of 2^-64, or nullptr: no rotation
  int nh;
};

// order-preserving integers of floats that are no NaN
__device__ __forceinline__ int kv4_key(float f) { const int i = __float_as_int(f); return i ^ ((i >> 31) & 0x7fffffff); }
__device__ __forceinline__ float kv4_of_key(int k) { return __int_as_float(k ^ ((k >> 31) & 0x7fffffff)); }

// A warp quantises one row: lane l < HD / 4 holds dims 4l .. 4l+3; returns the nibbles of the lane and the pair (s, z). Every operation rounds as
// IEEE single precision does, so that any program that follows the definition above gets the same bits.
template <int HD>
__device__ __forceinline__ uint32_t kv4_quantise(const float (&x)[4], int lane, int (&nib)[4]) {
  const bool on = lane < HD / 4;
  float lo = fminf(fminf(x[0], x[1]), fminf(x[2], x[3])), hi = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 4; e++) bad = bad || !(fabsf(x[e]) < INFINITY);
  lo = kv4_of_key(__reduce_min_sync(0xffffffffu, on && !bad ? kv4_key(lo) : 0x7f7fffff));
  hi = kv4_of_key(__reduce_max_sync(0xffffffffu, on && !bad ? kv4_key(hi) : (int)0x80800000));
  const float s = rbf(__fdiv_rn(__fsub_rn(hi, lo), 15.f)), z = rbf(__fadd_rn(lo, __fmul_rn(8.f, s)));
  if (__any_sync(0xffffffffu, on && bad) || !(s < INFINITY) || !(fabsf(z) < INFINITY)) {
#pragma unroll
    for (int e = 0; e < 4; e++) nib[e] = 8;
    return 0x7fc07fc0u;
  }
#pragma unroll
  for (int e = 0; e < 4; e++) nib[e] = s > 0.f ? 8 + (int)fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[e], z), s)), -8.f), 7.f) : 8;
  return (uint32_t)f2bf(s) | ((uint32_t)f2bf(z) << 16);
}

// grid (tokens, row groups), 256 threads; a warp takes a row (a head of q, k or v) of the token at a time.
// The angle of a far position needs more bits than a float has: pos * freq modulo one turn is exact in 64-bit integers, its sine and cosine are taken in double
// precision, once per token and pair, and k is rotated in double precision too, because a row's scale and nibbles hang on
// its last bits (q is rotated in single precision and rounded to bf16).
template <int HD>
__global__ void __launch_bounds__(256) kv4_append(const Kv4Append P) {
  using C = Kv4<HD>;
  constexpr int HP = HD / 2, LN = HD / 4;                        // rotation pairs, lanes that hold a row
  __shared__ double2 s_cs[HP];
  const Kv4Seqs& S = P.S;
  const int m = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nq = P.q ? P.nh : 0, rows = nq + 2 * S.nkv;
  pdl_begin(true);
  const int b = kv4_seq_of(S, m, lane);
  if (b < 0) return;
  Kv4Seq q;
  const bool first = blockIdx.y == 0 && tid == 0;
  if (!q.get(S, b, first) || m < q.first || m >= q.first + q.n) return;
  const int slot = q.cached + m - q.first;
  if (P.freq) {
    const long long pos = P.depth ? (long long)q.cached + P.depth[m] : slot;
    if (tid < HP) {
      double sn, cs;
      sincospi((double)(long long)((unsigned long long)pos * P.freq[tid]) * 0x1p-63, &sn, &cs);
      s_cs[tid] = make_double2(cs, sn);
    }
    __syncthreads();
  }
  const int page = kv4_page(S, b, slot, first);
  const bool on = lane < LN, low = lane < LN / 2;
  const int partner = on ? (low ? lane + LN / 2 : lane - LN / 2) : lane, i0 = 4 * (on ? (low ? lane : lane - LN / 2) : 0);
  for (int r = blockIdx.y * 8 + warp; r < rows; r += gridDim.y * 8) {
    const bool isq = r < nq, isv = r >= nq + S.nkv;
    const int head = isq ? r : (isv ? r - nq - S.nkv : r - nq);
    const uint16_t* src = isq ? P.q + (size_t)m * P.q_ld : (isv ? P.v + (size_t)m * P.v_ld : P.k + (size_t)m * P.k_ld);
    const uint2 w = on ? *reinterpret_cast<const uint2*>(src + head * HD + 4 * lane) : make_uint2(0, 0);
    float x[4] = {bflo(w.x), bfhi(w.x), bflo(w.y), bfhi(w.y)};
    if (P.freq && !isv) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float y = __shfl_sync(0xffffffffu, x[e], partner);
        const double2 cs = s_cs[i0 + e];
        if (isq) x[e] = low ? x[e] * (float)cs.x - y * (float)cs.y : x[e] * (float)cs.x + y * (float)cs.y;
        else x[e] = (float)(low ? (double)x[e] * cs.x - (double)y * cs.y : (double)x[e] * cs.x + (double)y * cs.y);
      }
    }
    if (isq) {
      if (on) *reinterpret_cast<uint2*>(P.q_out + (size_t)m * P.qo_ld + head * HD + 4 * lane) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
      continue;
    }
    int n[4];
    const uint32_t sz = kv4_quantise<HD>(x, lane, n);
    if (page < 0) continue;
    uint8_t* blk = kv4_block<HD>(S, page, head, slot);
    const int p = slot & 15;
    if (isv) {
      if (on) *reinterpret_cast<uint16_t*>(blk + C::v_word(p >> 1, lane) + (p & 1) * 2) = (uint16_t)(n[0] | n[1] << 4 | n[2] << 8 | n[3] << 12);
    } else {
      uint32_t word = (uint32_t)n[0] | (uint32_t)n[1] << 16 | (uint32_t)n[2] << 4 | (uint32_t)n[3] << 20;      // dims 0 .. 3 of the word, or 4 .. 7
      if (lane & 1) word <<= 8;
      word |= __shfl_xor_sync(0xffffffffu, word, 1);
      if (on && !(lane & 1)) *reinterpret_cast<uint32_t*>(blk + C::k_word(p, lane >> 1)) = word;
    }
    if (lane == 0) *reinterpret_cast<uint32_t*>(blk + (isv ? C::VSZ : C::KSZ) + p * 4) = sz;
  }
}

// ------------------------------------------------------------------------------------------------ read back, moves
// f32 [layers][T][nkv][HD]: (nib - 8) * s + z of the tokens' rows. grid (tokens, layers), 256 threads, a warp a row.
struct Kv4Read {
  Kv4Seqs S;
  float *k, *v;                      // either may be nullptr
  size_t layer;                      // bytes of a layer of the pool
};
template <int HD>
__global__ void __launch_bounds__(256) kv4_read(const Kv4Read P) {
  using C = Kv4<HD>;
  const Kv4Seqs& S = P.S;
  const int m = blockIdx.x, lane = threadIdx.x & 31;
  pdl_begin(true);
  const int b = kv4_seq_of(S, m, lane);
  if (b < 0) return;
  Kv4Seq q;
  if (!q.get(S, b, threadIdx.x == 0) || m < q.first || m >= q.first + q.n) return;
  const int slot = q.cached + m - q.first, page = kv4_page(S, b, slot, threadIdx.x == 0), p = slot & 15;
  if (page < 0 || lane >= HD / 4) return;
  for (int r = threadIdx.x >> 5; r < 2 * S.nkv; r += 8) {
    const bool isv = r >= S.nkv;
    const int head = isv ? r - S.nkv : r;
    float* out = isv ? P.v : P.k;
    if (!out) continue;
    const uint8_t* blk = kv4_block<HD>(S, page, head, slot) + blockIdx.y * P.layer;
    const uint32_t sz = *reinterpret_cast<const uint32_t*>(blk + (isv ? C::VSZ : C::KSZ) + p * 4);
    float x[4];
    if (isv) {
      const uint32_t h = *reinterpret_cast<const uint16_t*>(blk + C::v_word(p >> 1, lane) + (p & 1) * 2);
#pragma unroll
      for (int e = 0; e < 4; e++) x[e] = (float)((int)(h >> (4 * e) & 15u) - 8);
    } else {
      const uint32_t h = *reinterpret_cast<const uint32_t*>(blk + C::k_word(p, lane >> 1)) >> (8 * (lane & 1));
#pragma unroll
      for (int e = 0; e < 4; e++) x[e] = (float)((int)(h >> ((e & 1) * 16 + (e >> 1) * 4) & 15u) - 8);
    }
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = __fadd_rn(__fmul_rn(x[e], bflo(sz)), bfhi(sz));
    *reinterpret_cast<float4*>(out + (((size_t)blockIdx.y * S.T + m) * S.nkv + head) * HD + 4 * lane) = make_float4(x[0], x[1], x[2], x[3]);
  }
}

// Rows of a sequence from slots to slots, in order, in every layer. A thread owns the same piece of every row (a word of K, a half of V, a pair), so that a
// move that reads what an earlier one wrote finds it written without a wait between threads. grid (nkv, layers), 128 threads.
struct Kv4Move {
  Kv4Seqs S;
  size_t layer;
  const int* accept;                 // device: [0] = nodes on the path, [2 + i] = node of path step i: slot pos + i takes pos + path[i], 1 <= i
  int pos, most;                     // most: entries of accept's path
  int n;                             // or, accept == nullptr: n moves
  int src[64], dst[64];
};
template <int HD>
__global__ void __launch_bounds__(128) kv4_move(const Kv4Move P) {
  using C = Kv4<HD>;
  constexpr int KW = HD / 8, VH = HD / 4;
  static_assert(KW + VH + 2 <= 128, "a thread per piece of a row");
  const Kv4Seqs& S = P.S;
  const int tid = threadIdx.x, head = blockIdx.x;
  const bool first = tid == 0 && head == 0 && blockIdx.y == 0;
  pdl_begin(true);
  int len = P.n;
  if (P.accept) {
    len = P.accept[0];
    if (len < 0 || len > P.most) {
      if (first) kv4_report(S.status, KV4_PATH, 0, P.most, len);
      return;
    }
  }
  auto slots = [&](int i, int& from, int& to) {
    if (!P.accept) { from = P.src[i]; to = P.dst[i]; return true; }
    const int node = P.accept[2 + i];
    from = P.pos + node;
    to = P.pos + i;
    if (node >= 0 && (long long)P.pos + node < (long long)S.table_ld * kPage && to < S.table_ld * kPage) return true;
    if (first) kv4_report(S.status, KV4_PATH, i, S.table_ld * kPage, node);
    return false;
  };
  uint8_t* pool = S.pool + blockIdx.y * P.layer;
  auto at = [&](int page, int slot) {
    uint8_t* blk = pool + ((size_t)page * S.nkv + head) * C::REC + (slot % kPage / 16) * C::BLOCK;
    const int p = slot & 15;
    if (tid < KW) return blk + C::k_word(p, tid);
    if (tid < KW + VH) return blk + C::v_word(p >> 1, tid - KW) + (p & 1) * 2;
    return blk + (tid == KW + VH ? C::KSZ : C::VSZ) + p * 4;
  };
  const bool half = tid >= KW && tid < KW + VH;
  for (int i = P.accept ? 1 : 0; i < len; i++) {
    int from, to;
    if (!slots(i, from, to) || from == to) continue;
    const int pf = kv4_page(S, 0, from, first), pt = kv4_page(S, 0, to, first);
    if (pf < 0 || pt < 0 || tid >= KW + VH + 2) continue;
    const uint8_t* a = at(pf, from);
    uint8_t* d = at(pt, to);
    if (half) *reinterpret_cast<uint16_t*>(d) = *reinterpret_cast<const volatile uint16_t*>(a);
    else *reinterpret_cast<uint32_t*>(d) = *reinterpret_cast<const volatile uint32_t*>(a);
  }
}

// ------------------------------------------------------------------------------------------------ attention, few rows
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t cvt_f16x2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
// nibble pairs in bits (0..3, 16..19) / (4..7, 20..23) -> fp16 pair nib - 8, exact (fb_vtc.cuh's conversion without the scale)
__device__ __forceinline__ uint32_t kv4_lo(uint32_t w) {
  const uint32_t x = (w & 0x000F000Fu) | 0x64006400u;
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6408)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t kv4_hi(uint32_t w) {
  const uint32_t x = (w & 0x00F000F0u) | 0x64006400u;
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x2C00)), __half2half2(__ushort_as_half(0xD480)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t kv4_lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}

struct Kv4Attend {
  Kv4Seqs S;
  const uint16_t* q;         // bf16 [T][nh][HD], rotated, tokens q_ld elements apart
  uint16_t* out;             // bf16 [T][nh][HD], tokens o_ld apart
  long long q_ld, o_ld;
  const uint8_t* amask;      // [T][mask_ld]: token m sees new slot j of its sequence, or nullptr: causal
  int mask_ld, nh, R, max_new, groups, nsplit;
  float scale;               // times log2(e)
  unsigned spin_limit;
};

// Scores and outputs are computed TRANSPOSED: S^T[16 positions][8 query rows] = K Q^T and O^T[16 dims][8 query rows] += V^T P^T by mma.m16n8k16, so that
// the few query rows of a decode step (row = token * R + head of the group) fill the narrow side of the instruction and the cache the wide one. The cache's
// operands are nib - 8 in fp16, exact; a position's s and z join in fp32 behind the product, S = s (q . n) + z (sum q), and ahead of it,
// O += (p s) n, and sum p z apart. Q is fp16 times a power of two per row (exact for elements down to 2^-31 of the row's largest); p s is rounded to
// fp16 (half a step is 2^-11 of it, the output's bf16 rounding 2^-8), times a power of two that follows the largest p s of the row so far.
// A warp streams units of U positions through a ring of its own, one bulk copy each (lane 0 asks, all 32 lanes read), with a running maximum and sum;
// warps meet at the end, then the CTAs of a cluster that share a sequence's positions (partials pushed to the CTA that finishes the row).
template <int HD, int NQ, int W>
struct Kv4Few {
  static constexpr int U = 32, NST = 3, ROWS = 8 * NQ, PW = HD + 4;         // positions of a unit, stages of a warp, query rows, floats of a partial
  static constexpr int STAGE = U / 16 * Kv4<HD>::BLOCK, RING = W * NST * STAGE, PART = W * ROWS * PW * 4;
  static constexpr int INBOX = RING > PART ? RING : PART;
  static constexpr int BAR = INBOX + 16 * PW * 4, TOTAL = BAR + W * NST * 8 + 16;
  static_assert(TOTAL <= 227 * 1024, "shared memory");
};

// grid (clusters of nsplit over sequence x row group, nkv), W warps
template <int HD, int NQ, int W>
__global__ void __launch_bounds__(W * 32) kv4_attn_few(const Kv4Attend P) {
  using C = Kv4<HD>;
  using F = Kv4Few<HD, NQ, W>;
  constexpr int KS = HD / 16, MT = HD / 16, U = F::U, NST = F::NST, ROWS = F::ROWS, PW = F::PW;
  extern __shared__ __align__(128) uint8_t sm[];
  const Kv4Seqs& S = P.S;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int ns = P.nsplit, rank = (int)blockIdx.x % ns, idx = (int)blockIdx.x / ns, b = idx / P.groups, grp = idx % P.groups, kvh = blockIdx.y, R = P.R;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + F::BAR) + warp * NST;
  volatile int* s_abort = reinterpret_cast<volatile int*>(sm + F::BAR + W * NST * 8);
  pdl_begin(true);
  Kv4Seq seq;
  const bool told = kvh == 0 && rank == 0 && grp == 0 && tid == 0;
  if (!seq.get(S, b, told)) return;                              // the same for every CTA of a cluster
  if (told && seq.n > P.max_new) kv4_report(S.status, KV4_TOKENS, b, P.max_new, seq.n);
  const int rows = seq.n * R, r0 = grp * ROWS;
  if (r0 >= rows) return;
  if (ns > 1) cluster_arrive();                                  // partials are sent once every neighbour is known to run
  if (lane == 0) {
    for (int i = 0; i < NST; i++) mbar_init(&bars[i], 1);
    if (warp == 0) *s_abort = 0;
    mbar_fence_init();
  }
  __syncthreads();
  const WaitCtl wc{S.status, s_abort, P.spin_limit};
  const int m_last = min(seq.n - 1, (r0 + ROWS - 1) / R), total = seq.cached + seq.n, t_end = P.amask ? total : seq.cached + m_last + 1;
  const int nu = (t_end + U - 1) / U, u_begin = (int)((long long)nu * rank / ns), u_end = (int)((long long)nu * (rank + 1) / ns);
  const int mine = u_end - u_begin > warp ? (u_end - u_begin - warp + W - 1) / W : 0;      // units of this warp: u_begin + warp + i * W
  uint32_t skip = 0;                                             // stages whose unit has no page
  uint8_t* ring = sm + warp * NST * F::STAGE;
  auto page_of = [&](int i) { return i < mine ? kv4_page(S, b, (u_begin + warp + i * W) * U, lane == 0) : -1; };
  auto issue = [&](int i, int page, int st) {
    if (i >= mine) return;
    if (page < 0) {
      skip |= 1u << st;
      if (lane == 0) mbar_arrive(&bars[st]);
      return;
    }
    skip &= ~(1u << st);
    if (lane == 0) {
      const int slot = (u_begin + warp + i * W) * U;
      mbar_expect_tx(&bars[st], F::STAGE);
      bulk_g2s(ring + st * F::STAGE, kv4_block<HD>(S, page, kvh, slot), F::STAGE, &bars[st]);
    }
  };
  {
    int pg[NST];
#pragma unroll
    for (int i = 0; i < NST; i++) pg[i] = page_of(i);
#pragma unroll
    for (int i = 0; i < NST; i++) issue(i, pg[i], i);
  }
  int page_next = page_of(NST);

  // the query rows: lane (g, t) holds row g of each tile, the dims that it multiplies
  uint32_t qf[NQ][KS][2];
  float c2[NQ][2], qs[NQ][2];                                    // of columns 2t, 2t + 1: factor of the scores, sum of the row
#pragma unroll
  for (int nq = 0; nq < NQ; nq++) {
    const int r = r0 + nq * 8 + g;
    const uint16_t* src = P.q + (size_t)(seq.first + min(r, rows - 1) / R) * P.q_ld + (size_t)(kvh * R + min(r, rows - 1) % R) * HD;
    uint32_t w[KS * 2];
#pragma unroll
    for (int i = 0; i < C::MAIN / 32; i++) {
      const uint4 v = *reinterpret_cast<const uint4*>(src + C::MAIN / 4 * t + 8 * i);
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
    if constexpr (HD > C::MAIN) {
      const uint2 v = *reinterpret_cast<const uint2*>(src + C::MAIN + 4 * t);
      w[C::MAIN / 8] = v.x; w[C::MAIN / 8 + 1] = v.y;
    }
    float mx = 0.f, sum = 0.f;
    if (r >= rows)
#pragma unroll
      for (int i = 0; i < 2 * KS; i++) w[i] = 0;
#pragma unroll
    for (int i = 0; i < 2 * KS; i++) mx = fmaxf(mx, fmaxf(fabsf(bflo(w[i])), fabsf(bfhi(w[i]))));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const float2 f = pow2_for(mx);
#pragma unroll
    for (int i = 0; i < 2 * KS; i++) {
      const float a = bflo(w[i]) * f.x, c = bfhi(w[i]) * f.x;
      sum += a + c;
      qf[nq][i >> 1][i & 1] = cvt_f16x2(a, c);
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
    for (int e = 0; e < 2; e++) {
      c2[nq][e] = __shfl_sync(0xffffffffu, f.y, (2 * t + e) * 4) * P.scale;
      qs[nq][e] = __shfl_sync(0xffffffffu, sum, (2 * t + e) * 4);
    }
  }
  float o[NQ][MT][4], mrun[NQ][2], lrun[NQ][2], zrun[NQ][2], wrun[NQ][2];
  uint32_t erun[NQ][2];                                          // exponent field of wrun, the largest p s so far: o is in units of 2^(erun - 127)
#pragma unroll
  for (int nq = 0; nq < NQ; nq++) {
#pragma unroll
    for (int i = 0; i < MT; i++) o[nq][i][0] = o[nq][i][1] = o[nq][i][2] = o[nq][i][3] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; e++) { mrun[nq][e] = -1e30f; lrun[nq][e] = 0.f; zrun[nq][e] = 0.f; wrun[nq][e] = 0.f; erun[nq][e] = 1; }
  }
  bool ok = true;
  int st = 0;
  uint32_t lap = 0;
  int done = 0;
#pragma unroll 1
  for (int i = 0; i < mine; i++) {
    ok = __all_sync(0xffffffffu, mbar_wait(&bars[st], lap, wc, W_FULL, 30));
    if (!ok) break;
    done = i + 1;
    const int slot0 = (u_begin + warp + i * W) * U;
    if (!(skip >> st & 1)) {
      const uint32_t base = smem_u32(ring + st * F::STAGE);
      const bool edge = slot0 + U > seq.cached;                  // holds new tokens, or slots behind them
      float sc[NQ][U / 16][4], vs[U / 16][2], vz[U / 16][2];
#pragma unroll
      for (int k = 0; k < U / 16; k++) {
        const uint32_t blk = base + k * C::BLOCK;
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) sc[nq][k][0] = sc[nq][k][1] = sc[nq][k][2] = sc[nq][k][3] = 0.f;
        uint32_t wl[HD / 32 + (HD > C::MAIN)], wh[HD / 32 + (HD > C::MAIN)];       // words of positions g and g + 8
        if constexpr (HD == 128) {
          const uint4 x = lds128(blk + g * 64 + t * 16), y = lds128(blk + (g + 8) * 64 + t * 16);
          wl[0] = x.x; wl[1] = x.y; wl[2] = x.z; wl[3] = x.w;
          wh[0] = y.x; wh[1] = y.y; wh[2] = y.z; wh[3] = y.w;
        } else {
          const uint2 x = lds64(blk + g * 32 + t * 8), y = lds64(blk + (g + 8) * 32 + t * 8);
          wl[0] = x.x; wl[1] = x.y;
          wh[0] = y.x; wh[1] = y.y;
          if constexpr (HD > C::MAIN) {
            wl[2] = kv4_lds32(blk + 512 + g * 8 + (t >> 1) * 4) >> (8 * (t & 1));
            wh[2] = kv4_lds32(blk + 512 + (g + 8) * 8 + (t >> 1) * 4) >> (8 * (t & 1));
          }
        }
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
          const uint32_t a = wl[ks >> 1] >> (8 * (ks & 1)), c = wh[ks >> 1] >> (8 * (ks & 1));
          const uint32_t A[4] = {kv4_lo(a), kv4_lo(c), kv4_hi(a), kv4_hi(c)};
#pragma unroll
          for (int nq = 0; nq < NQ; nq++) mma_f16(sc[nq][k], A, qf[nq][ks][0], qf[nq][ks][1]);
        }
        const uint32_t k0 = kv4_lds32(blk + C::KSZ + g * 4), k1 = kv4_lds32(blk + C::KSZ + g * 4 + 32), v0 = kv4_lds32(blk + C::VSZ + g * 4),
                       v1 = kv4_lds32(blk + C::VSZ + g * 4 + 32);
        vs[k][0] = bflo(v0); vs[k][1] = bflo(v1); vz[k][0] = bfhi(v0); vz[k][1] = bfhi(v1);
        const float s0 = bflo(k0), s1 = bflo(k1), z0 = bfhi(k0), z1 = bfhi(k1);
#pragma unroll
        for (int nq = 0; nq < NQ; nq++)
#pragma unroll
          for (int e = 0; e < 4; e++) sc[nq][k][e] = fmaf(e < 2 ? z0 : z1, qs[nq][e & 1], sc[nq][k][e] * (e < 2 ? s0 : s1)) * c2[nq][e & 1];
        if (edge) {
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const int tp = slot0 + k * 16 + g + 8 * h;
            if (tp >= total) vs[k][h] = vz[k][h] = 0.f;          // what lies behind the last token may be anything
#pragma unroll
            for (int nq = 0; nq < NQ; nq++)
#pragma unroll
              for (int e = 0; e < 2; e++) {
                bool see = tp < total;
                if (see && tp >= seq.cached) {
                  const int mq = min(r0 + nq * 8 + 2 * t + e, rows - 1) / R, j = tp - seq.cached;
                  see = P.amask ? j < P.mask_ld && P.amask[(size_t)(seq.first + mq) * P.mask_ld + j] != 0 : j <= mq;
                }
                if (!see) sc[nq][k][2 * h + e] = -INFINITY;
              }
          }
        }
      }
      // running maximum, sums, and p s in place of the scores
      float corr[NQ][2];
      bool moved = false;
#pragma unroll
      for (int nq = 0; nq < NQ; nq++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float mx = -INFINITY;
#pragma unroll
          for (int k = 0; k < U / 16; k++) mx = fmaxf(mx, fmaxf(sc[nq][k][e], sc[nq][k][2 + e]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float mn = fmaxf(mrun[nq][e], mx);               // finite from below: the running maximum starts at -1e30
          const float cr = ex2(mrun[nq][e] - mn);
          mrun[nq][e] = mn;
          float ls = 0.f, zs = 0.f, wm = 0.f;
#pragma unroll
          for (int k = 0; k < U / 16; k++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
              float& x = sc[nq][k][2 * h + e];
              const float p = ex2(x - mn);
              float w = p * vs[k][h], pz = p * vz[k][h];
              if (edge && x == -INFINITY) w = pz = 0.f;          // an unseen row may be NaN
              ls += p;
              zs += pz;
              wm = fmaxf(wm, w);
              x = w;
            }
          wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, 4));
          wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, 8));
          wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, 16));
          lrun[nq][e] = fmaf(lrun[nq][e], cr, ls);
          zrun[nq][e] = fmaf(zrun[nq][e], cr, zs);
          wrun[nq][e] = fmaxf(wrun[nq][e] * cr, wm);
          const uint32_t en = min(max(__float_as_uint(wrun[nq][e]) >> 23, 1u), 253u);
          const int up = min(max((int)erun[nq][e] - (int)en, -126), 126);
          corr[nq][e] = cr * __uint_as_float((uint32_t)(127 + up) << 23);
          moved = moved || cr != 1.f || en != erun[nq][e];
          erun[nq][e] = en;
          const float vf = __uint_as_float((254u - en) << 23);
#pragma unroll
          for (int k = 0; k < U / 16; k++) { sc[nq][k][e] *= vf; sc[nq][k][2 + e] *= vf; }
        }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int nq = 0; nq < NQ; nq++)
#pragma unroll
          for (int j = 0; j < MT; j++) { o[nq][j][0] *= corr[nq][0]; o[nq][j][1] *= corr[nq][1]; o[nq][j][2] *= corr[nq][0]; o[nq][j][3] *= corr[nq][1]; }
      }
#pragma unroll
      for (int k = 0; k < U / 16; k++) {
        uint32_t pb[NQ][2];
#pragma unroll
        for (int nq = 0; nq < NQ; nq++)
#pragma unroll
          for (int h = 0; h < 2; h++) pb[nq][h] = movmatrix_trans(cvt_f16x2(sc[nq][k][2 * h], sc[nq][k][2 * h + 1]));
        const uint32_t vb = base + k * C::BLOCK + C::V;
        uint32_t x0[HD / 32 + (HD > C::MAIN)], x1[HD / 32 + (HD > C::MAIN)];      // words of pairs t and t + 4
        if constexpr (HD == 128) {
          const uint4 x = lds128(vb + t * 128 + ((g ^ (2 * t)) << 4)), y = lds128(vb + (t + 4) * 128 + ((g ^ (2 * t)) << 4));
          x0[0] = x.x; x0[1] = x.y; x0[2] = x.z; x0[3] = x.w;
          x1[0] = y.x; x1[1] = y.y; x1[2] = y.z; x1[3] = y.w;
        } else {
          const uint32_t off = (uint32_t)((g * 8) ^ ((t >> 1) * 32));
          const uint2 x = lds64(vb + t * 64 + off), y = lds64(vb + (t + 4) * 64 + off);
          x0[0] = x.x; x0[1] = x.y;
          x1[0] = y.x; x1[1] = y.y;
          if constexpr (HD > C::MAIN) {
            x0[2] = kv4_lds32(vb + 512 + t * 16 + (g >> 1) * 4) >> (8 * (g & 1));
            x1[2] = kv4_lds32(vb + 512 + (t + 4) * 16 + (g >> 1) * 4) >> (8 * (g & 1));
          }
        }
#pragma unroll
        for (int j = 0; j < MT; j++) {
          const uint32_t a = x0[j >> 1] >> (8 * (j & 1)), c = x1[j >> 1] >> (8 * (j & 1));
          const uint32_t A[4] = {kv4_lo(a), kv4_hi(a), kv4_lo(c), kv4_hi(c)};
#pragma unroll
          for (int nq = 0; nq < NQ; nq++) mma_f16(o[nq][j], A, pb[nq][0], pb[nq][1]);
        }
      }
    }
    __syncwarp();                                                // every lane has read the stage
    issue(i + NST, page_next, st);
    page_next = page_of(i + NST + 1);
    if (++st == NST) { st = 0; lap ^= 1u; }
  }
  if (!ok && lane == 0) {                                        // after a failure: this warp's copies in flight
    const int issued = min(mine, done + NST);
    for (int i = done; i < issued; i++) drain_phase(&bars[i % NST], (uint32_t)(i / NST) & 1u);
  }
#pragma unroll
  for (int nq = 0; nq < NQ; nq++)
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
      for (int s = 4; s < 32; s *= 2) {
        lrun[nq][e] += __shfl_xor_sync(0xffffffffu, lrun[nq][e], s);
        zrun[nq][e] += __shfl_xor_sync(0xffffffffu, zrun[nq][e], s);
      }
  __syncthreads();                                               // every warp has left its ring
  float* part = reinterpret_cast<float*>(sm);
  {
#pragma unroll
    for (int nq = 0; nq < NQ; nq++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float* pr = part + (size_t)(warp * ROWS + nq * 8 + 2 * t + e) * PW;
        const float back = __uint_as_float(erun[nq][e] << 23);   // 2^(erun - 127)
#pragma unroll
        for (int j = 0; j < MT; j++) {
          const int d = 8 * j < C::MAIN / 2 ? C::MAIN / 8 * g + 2 * j : C::MAIN + 2 * g;
          *reinterpret_cast<float2*>(pr + d) = make_float2(fmaf(o[nq][j][e], back, zrun[nq][e]), fmaf(o[nq][j][2 + e], back, zrun[nq][e]));
        }
        if (g == 0) *reinterpret_cast<float2*>(pr + HD) = make_float2(mrun[nq][e], lrun[nq][e]);
      }
  }
  __syncthreads();
  if (ns > 1) cluster_wait();
  auto merge = [&](const float* p0, int n, int stride, float4& acc, float& mm, float& den) {
    mm = -1e30f;
    for (int i = 0; i < n; i++) mm = fmaxf(mm, p0[(size_t)i * stride + HD]);
    den = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = 0; i < n; i++) {
      const float2 ml = *reinterpret_cast<const float2*>(p0 + (size_t)i * stride + HD);
      const float e = ex2(ml.x - mm);
      const float4 v = lane < HD / 4 ? *reinterpret_cast<const float4*>(p0 + (size_t)i * stride + lane * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
      den = fmaf(ml.y, e, den);
      acc.x = fmaf(v.x, e, acc.x); acc.y = fmaf(v.y, e, acc.y); acc.z = fmaf(v.z, e, acc.z); acc.w = fmaf(v.w, e, acc.w);
    }
  };
  auto finish = [&](int lr, const float4& acc, float den) {      // normalise and write local row lr; a row that sees nothing is zeros
    const int r = r0 + lr;
    if (r >= rows || lane >= HD / 4) return;
    const float inv = den == 0.f ? 0.f : 1.f / den;
    *reinterpret_cast<uint2*>(P.out + (size_t)(seq.first + r / R) * P.o_ld + (size_t)(kvh * R + r % R) * HD + lane * 4) =
        make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
  };
  for (int lr = warp; lr < ROWS; lr += W) {
    float4 acc;
    float mm, den;
    merge(part + (size_t)lr * PW, W, ROWS * PW, acc, mm, den);
    if (ns == 1) {
      finish(lr, acc, den);
    } else {                                                     // to the CTA that finishes the row
      const uint32_t to = (uint32_t)(lr % ns), slot = (uint32_t)(rank * ((ROWS + ns - 1) / ns) + lr / ns);
      const uint32_t a = cluster_map(smem_u32(sm + F::INBOX) + slot * PW * 4, to);
      if (lane < HD / 4) st_cluster(a + lane * 16, acc);
      if (lane == 0) st_cluster(a + HD * 4, make_float4(mm, den, 0.f, 0.f));
    }
  }
  if (ns > 1) {
    cluster_arrive();
    cluster_wait();
    const int own = (ROWS + ns - 1) / ns;
    for (int i = warp; i < own && i * ns + rank < ROWS; i += W) {
      float4 acc;
      float mm, den;
      merge(reinterpret_cast<const float*>(sm + F::INBOX) + (size_t)i * PW, ns, own * PW, acc, mm, den);
      finish(i * ns + rank, acc, den);
    }
  }
}

}  // namespace fb
