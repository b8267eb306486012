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
#include <type_traits>

#include "fb_common.cuh"
#include "fb_drain.hpp"
#include "fb_kv4_geometry.hpp"

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
// Does sequence b end ahead of its start? Then nothing of the call is done: tokens could be two sequences', and the tasks more than the grid and the scratch have room for.
__device__ __forceinline__ bool kv4_backward(const Kv4Seqs& S, int b, bool report) {
  const int first = S.start[b], end = S.start[b + 1];
  if (end < first && report) kv4_report(S.status, KV4_TOKENS, b, first, end);
  return end < first;
}
// The sequence of token m, found by a whole warp: how many sequences end at or before it. -1: behind the last one, or no call that can be.
__device__ __forceinline__ int kv4_seq_of(const Kv4Seqs& S, int m, int lane, bool report) {
  if (!S.start) return 0;
  int b = 0;
  for (int i = 0; i < S.n_seq; i += 32) {
    const bool in = i + lane < S.n_seq;
    const unsigned n = __reduce_add_sync(0xffffffffu, in ? (S.start[i + lane + 1] <= m) | (unsigned)kv4_backward(S, i + lane, report) << 8 : 0u);
    if (n >> 8) return -1;
    b += (int)n;
  }
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

// grid (tokens, row groups), 256 threads; a warp takes a row (a head of q, k or v) of the token at a time and loads the next one meanwhile. (Six rows loaded ahead and
// unrolled are six copies of the code, which the instruction cache pays for: one token 2.7 -> 3.8 us, 725 tokens 14.3 -> 18.1.)
// The angle of a far position needs more bits than a float has: pos * freq modulo one turn is exact in 64-bit integers, its sine and cosine are taken in double
// precision, once per token and pair, and k is rotated in double precision too, because a row's scale and nibbles hang on
// its last bits (q is rotated in single precision and rounded to bf16). Bound by latency for a few tokens (the load, the sines, the row's extremes).
template <int HD>
__global__ void __launch_bounds__(256) kv4_append(const Kv4Append P) {
  using C = Kv4<HD>;
  constexpr int HP = HD / 2, LN = HD / 4;                        // rotation pairs, lanes that hold a row
  __shared__ double2 s_cs[HP];
  __shared__ float2 s_csf[HP];
  const Kv4Seqs& S = P.S;
  const int m = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nq = P.q ? P.nh : 0, rows = nq + 2 * S.nkv;
  const bool on = lane < LN, low = lane < LN / 2;
  pdl_begin(true);
  auto load = [&](int r) {
    const uint16_t* src = r < nq ? P.q + (size_t)m * P.q_ld + r * HD
                                 : (r < nq + S.nkv ? P.k + (size_t)m * P.k_ld + (r - nq) * HD : P.v + (size_t)m * P.v_ld + (r - nq - S.nkv) * HD);
    return on && r < rows ? *reinterpret_cast<const uint2*>(src + 4 * lane) : make_uint2(0, 0);
  };
  const int step = gridDim.y * 8;
  uint2 w = load(blockIdx.y * 8 + warp);
  const int b = kv4_seq_of(S, m, lane, m == 0 && blockIdx.y == 0 && warp == 0);
  if (b < 0) return;
  Kv4Seq q;
  const bool first = blockIdx.y == 0 && tid == 0;
  if (!q.get(S, b, first) || m < q.first || m >= q.first + q.n) return;
  const int slot = q.cached + m - q.first, page = kv4_page(S, b, slot, first);
  if (P.freq) {
    const long long pos = P.depth ? (long long)q.cached + P.depth[m] : slot;
    if (tid < HP) {
      double sn, cs;
      sincospi((double)(long long)((unsigned long long)pos * P.freq[tid]) * 0x1p-63, &sn, &cs);
      s_cs[tid] = make_double2(cs, sn);
      s_csf[tid] = make_float2((float)cs, (float)sn);
    }
    __syncthreads();
  }
  const int partner = on ? (low ? lane + LN / 2 : lane - LN / 2) : lane, i0 = 4 * (on ? (low ? lane : lane - LN / 2) : 0);
  auto row = [&](int r, uint2 v) {
    const bool isq = r < nq, isv = r >= nq + S.nkv;
    float x[4] = {bflo(v.x), bfhi(v.x), bflo(v.y), bfhi(v.y)};
    if (P.freq && !isv) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float y = __shfl_sync(0xffffffffu, x[e], partner);
        if (isq) {
          const float2 cs = s_csf[i0 + e];
          x[e] = low ? x[e] * cs.x - y * cs.y : x[e] * cs.x + y * cs.y;
        } else {
          const double2 cs = s_cs[i0 + e];
          x[e] = (float)(low ? (double)x[e] * cs.x - (double)y * cs.y : (double)x[e] * cs.x + (double)y * cs.y);
        }
      }
    }
    if (isq) {
      if (on) *reinterpret_cast<uint2*>(P.q_out + (size_t)m * P.qo_ld + r * HD + 4 * lane) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
      return;
    }
    int n[4];
    const uint32_t sz = kv4_quantise<HD>(x, lane, n);
    if (page < 0) return;
    uint8_t* blk = kv4_block<HD>(S, page, isv ? r - nq - S.nkv : r - nq, slot);
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
  };
#pragma unroll 1
  for (int r = blockIdx.y * 8 + warp; r < rows; r += step) {
    const uint2 now = w;
    w = load(r + step);
    row(r, now);
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
  const int b = kv4_seq_of(S, m, lane, m == 0 && threadIdx.x < 32);
  Kv4Seq q;
  int page = -1, slot = 0;
  if (b >= 0 && q.get(S, b, threadIdx.x == 0) && m >= q.first && m < q.first + q.n) {
    slot = q.cached + m - q.first;
    page = kv4_page(S, b, slot, threadIdx.x == 0);
  }
  const int p = slot & 15;
  if (lane >= HD / 4) return;
  for (int r = threadIdx.x >> 5; r < 2 * S.nkv; r += 8) {
    const bool isv = r >= S.nkv;
    const int head = isv ? r - S.nkv : r;
    float* out = isv ? P.v : P.k;
    if (!out) continue;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (page >= 0) {
      const uint8_t* blk = kv4_block<HD>(S, page, head, slot) + blockIdx.y * P.layer;
      const uint32_t sz = *reinterpret_cast<const uint32_t*>(blk + (isv ? C::VSZ : C::KSZ) + p * 4);
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
    }
    *reinterpret_cast<float4*>(out + (((size_t)blockIdx.y * S.T + m) * S.nkv + head) * HD + 4 * lane) = make_float4(x[0], x[1], x[2], x[3]);
  }
}

// Rows of a sequence from slots to slots, in order, in every layer. A thread owns the same piece of every row (a word of K, a half of V, a pair), so that a
// move that reads what an earlier one wrote finds it written without a wait between threads. An accepted path never does (its rows lie behind the places that
// they go to), and then eight loads are under way side by side. grid (nkv, layers), 128 threads. Bound by latency: the path, the pages, the
// rows, one after the other.
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
  constexpr int KW = HD / 8, VH = HD / 4, N = 64;
  static_assert(KW + VH + 2 <= 128, "a thread per piece of a row");
  __shared__ int s_from[N], s_to[N], s_page_from[N], s_page_to[N];
  const Kv4Seqs& S = P.S;
  const int tid = threadIdx.x, head = blockIdx.x;
  const bool first = head == 0 && blockIdx.y == 0;
  pdl_begin(true);
  int len = P.n;
  if (P.accept) {
    len = P.accept[0];
    if (len < 0 || len > P.most) {
      if (first && tid == 0) kv4_report(S.status, KV4_PATH, 0, P.most, len);
      return;
    }
  }
  uint8_t* pool = S.pool + blockIdx.y * P.layer;
  auto at = [&](int page, int slot) {
    uint8_t* blk = pool + ((size_t)page * S.nkv + head) * C::REC + (slot % kPage / 16) * C::BLOCK;
    const int p = slot & 15;
    if (tid < KW) return blk + C::k_word(p, tid);
    if (tid < KW + VH) return blk + C::v_word(p >> 1, tid - KW) + (p & 1) * 2;
    return blk + (tid == KW + VH ? C::KSZ : C::VSZ) + p * 4;
  };
  const bool half = tid >= KW && tid < KW + VH, piece = tid < KW + VH + 2;
  auto load = [&](int i) -> uint32_t {
    const uint8_t* a = at(s_page_from[i], s_from[i]);
    return half ? *reinterpret_cast<const volatile uint16_t*>(a) : *reinterpret_cast<const volatile uint32_t*>(a);
  };
  auto store = [&](int i, uint32_t v) {
    uint8_t* d = at(s_page_to[i], s_to[i]);
    if (half) *reinterpret_cast<volatile uint16_t*>(d) = (uint16_t)v;
    else *reinterpret_cast<volatile uint32_t*>(d) = v;
  };
  for (int i0 = P.accept ? 1 : 0; i0 < len; i0 += N) {           // the same for all threads
    const int n = min(N, len - i0);
    bool chain = false;
    if (tid < n) {
      int from, to;
      bool ok = true;
      if (P.accept) {
        const int node = P.accept[2 + i0 + tid];
        ok = node >= 0 && (long long)P.pos + node < (long long)S.table_ld * kPage && (long long)P.pos + i0 + tid < (long long)S.table_ld * kPage;
        if (!ok && first) kv4_report(S.status, KV4_PATH, i0 + tid, S.table_ld * kPage, node);
        from = P.pos + node;
        to = P.pos + i0 + tid;
        chain = from < to;
      } else {
        from = P.src[tid];
        to = P.dst[tid];
        chain = true;
      }
      const int pf = ok && from != to ? kv4_page(S, 0, from, first) : -1, pt = pf >= 0 ? kv4_page(S, 0, to, first) : -1;
      s_from[tid] = from; s_to[tid] = to; s_page_from[tid] = pt >= 0 ? pf : -1; s_page_to[tid] = pt;
    }
    if (__syncthreads_or(chain)) {
      for (int i = 0; i < n && piece; i++)
        if (s_page_from[i] >= 0) store(i, load(i));
    } else {
      for (int i = 0; i < n && piece; i += 8) {
        uint32_t v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = i + k < n && s_page_from[i + k] >= 0 ? load(i + k) : 0;
#pragma unroll
        for (int k = 0; k < 8; k++)
          if (i + k < n && s_page_from[i + k] >= 0) store(i + k, v[k]);
      }
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------ attention, few rows
// (not volatile: independent products may pass one another)
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
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
constexpr float kLowest = -3.402823466e38f;        // a row's running maximum before any score: finite, so that differences from it are numbers, and below every score but -inf
struct Kv4Attend {
  Kv4Seqs S;
  const uint16_t* q;         // bf16 [T][nh][HD], rotated, tokens q_ld elements apart
  uint16_t* out;             // bf16 [T][nh][HD], tokens o_ld apart
  long long q_ld, o_ld;
  const uint8_t* amask;      // [T][mask_ld]: token m sees new slot j of its sequence, or nullptr: causal
  int mask_ld, nh, R;
  int nsplit;                // a cluster: its CTAs share the positions of a row group of the one sequence
  int slots, chunk;          // else: CTAs that the GPU holds, over which all positions are spread in pieces of `chunk` units or more; slots 0: whole
  float* work;               // partials of split row groups, [task][row][PW], for kv4_join
  float scale;               // times log2(e)
  unsigned spin_limit;
};

// What a CTA does: `n` units from `unit` on of the positions that query rows r0 .. of a sequence and kv head see; `parts` tasks share them, the first of
// them is task `first`. The lengths are the device's, so every CTA finds its own task: per = all units of all row groups / slots, a sequence's
// parts follow from that, and the task's sequence from the sum of the tasks ahead of it. A ragged batch is spread evenly whatever its lengths.
template <int ROWS, int U>
struct Kv4Task {
  Kv4Seq seq;
  int b, kvh, rows, r0, total, unit, n, parts;
  long long first;
  __device__ __forceinline__ int groups_of(const Kv4Attend& P, const Kv4Seq& q) const { return (int)(((long long)q.n * P.R + ROWS - 1) / ROWS); }
  __device__ __forceinline__ int units_of(const Kv4Seq& q) const { return (int)(((long long)q.cached + q.n + U - 1) / U); }
  __device__ __forceinline__ int parts_of(int units, int per) const { return (units - 1) / per + 1; }        // per may be the largest integer
  // group grp of the sequence in `seq`
  __device__ __forceinline__ int set(const Kv4Attend& P, int grp) {          // units that the group sees
    rows = seq.n * P.R;
    r0 = grp * ROWS;
    total = seq.cached + seq.n;
    const int t_end = P.amask ? total : seq.cached + min(seq.n - 1, (r0 + ROWS - 1) / P.R) + 1;
    return (t_end + U - 1) / U;
  }
  __device__ __forceinline__ int per_of(const Kv4Attend& P, long long units) const {
    if (!P.slots) return 0x7fffffff;
    const long long per = (units * P.S.nkv + P.slots - 1) / P.slots;
    return (int)min(max(per, (long long)P.chunk), 0x7fffffffll);
  }
  // task `idx`, or with JOIN row group `idx` of all sequences, all of its parts
  template <bool JOIN>
  __device__ __forceinline__ bool find(const Kv4Attend& P, long long idx, int lane, bool report) {
    const Kv4Seqs& S = P.S;
    int per, g = 0, part = 0;
    if (S.n_seq == 1) {
      b = 0;
      if (!seq.get(S, 0, report)) return false;
      const int groups = groups_of(P, seq), nu = units_of(seq);
      per = per_of(P, (long long)groups * nu);
      parts = parts_of(nu, per);
      first = 0;
      if (JOIN) {
        g = (int)idx;
        if (g >= groups) return false;
      } else {
        if (idx >= (long long)groups * parts * S.nkv) return false;
      }
    } else {
      long long units = 0;
      bool backward = false;
      for (int i = lane; i < S.n_seq; i += 32) {
        Kv4Seq q;
        backward = backward || kv4_backward(S, i, report);
        if (q.get(S, i, report)) units += (long long)groups_of(P, q) * units_of(q);
      }
      if (__any_sync(0xffffffffu, backward)) return false;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) units += __shfl_xor_sync(0xffffffffu, units, o);
      per = per_of(P, units);
      long long at = 0, tasks_ahead = 0;                         // what is counted (tasks, or row groups), and tasks, ahead of the 32 sequences
      int i0 = 0;
      for (;; i0 += 32) {
        if (i0 >= S.n_seq) return false;
        Kv4Seq q;
        long long tasks = 0, count = 0;
        if (i0 + lane < S.n_seq && q.get(S, i0 + lane, false)) {
          const int groups = groups_of(P, q), nu = units_of(q);
          tasks = (long long)groups * parts_of(nu, per) * S.nkv;
          count = JOIN ? groups : tasks;
        }
        long long sum = count, tsum = tasks;                     // inclusive sums over the lanes
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
          const long long x = __shfl_up_sync(0xffffffffu, sum, o), y = __shfl_up_sync(0xffffffffu, tsum, o);
          if (lane >= o) { sum += x; tsum += y; }
        }
        const unsigned past = __ballot_sync(0xffffffffu, idx < at + sum);
        if (past) {
          const int l = __ffs(past) - 1;
          b = i0 + l;
          idx -= at + __shfl_sync(0xffffffffu, sum - count, l);
          first = tasks_ahead + __shfl_sync(0xffffffffu, tsum - tasks, l);
          break;
        }
        at += __shfl_sync(0xffffffffu, sum, 31);
        tasks_ahead += __shfl_sync(0xffffffffu, tsum, 31);
      }
      seq.get(S, b, false);
      parts = parts_of(units_of(seq), per);
      g = (int)idx;
    }
    if (!JOIN) {                                                 // a sequence's tasks: parts, row groups, kv heads
      const int groups = groups_of(P, seq), i = (int)(idx / S.nkv);
      kvh = (int)(idx % S.nkv);
      part = i / groups;
      g = i % groups;
    }
    const int nu = set(P, g);
    unit = (int)min((long long)part * per, (long long)nu);       // a causal group may see less than the sequence's parts cover: it has empty ones
    n = (int)min((long long)per, (long long)nu - unit);
    return true;
  }
  __device__ __forceinline__ long long task_of(const Kv4Attend& P, int part) const {       // part `part` of this row group and kv head
    return first + ((long long)part * groups_of(P, seq) + r0 / ROWS) * P.S.nkv + kvh;
  }
};

// Partials of a row, n of them `stride` floats apart, eight loads side by side: lane < HD / 4 merges dims 4 lane .. 4 lane + 3
template <int HD>
__device__ __forceinline__ void kv4_merge(const float* p0, int n, size_t stride, int lane, float4& acc, float& mm, float& den) {
  mm = kLowest;
  den = 0.f;
  acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += 8) {
    float2 ml[8];
    float4 v[8];
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const float* p = p0 + (i0 + k < n ? i0 + k : i0) * stride;
      ml[k] = *reinterpret_cast<const float2*>(p + HD);
      v[k] = lane < HD / 4 ? *reinterpret_cast<const float4*>(p + lane * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
      if (i0 + k >= n) ml[k].x = -INFINITY;
    }
    float top = mm;
#pragma unroll
    for (int k = 0; k < 8; k++) top = fmaxf(top, ml[k].x);
    const float old = ex2(mm - top);
    mm = top;
    den *= old;
    acc.x *= old; acc.y *= old; acc.z *= old; acc.w *= old;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      if (i0 + k < n) {
        const float e = ex2(ml[k].x - mm);
        den = fmaf(ml[k].y, e, den);
        acc.x = fmaf(v[k].x, e, acc.x); acc.y = fmaf(v[k].y, e, acc.y); acc.z = fmaf(v[k].z, e, acc.z); acc.w = fmaf(v[k].w, e, acc.w);
      }
    }
  }
}
// normalise and write row r of a sequence; a row that sees nothing is zeros
template <int HD>
__device__ __forceinline__ void kv4_finish(const Kv4Attend& P, const Kv4Seq& seq, int kvh, int r, int lane, const float4& acc, float den) {
  if (lane >= HD / 4) return;
  const float inv = den == 0.f ? 0.f : 1.f / den;
  *reinterpret_cast<uint2*>(P.out + (size_t)(seq.first + r / P.R) * P.o_ld + (size_t)(kvh * P.R + r % P.R) * HD + lane * 4) =
      make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
}

// Scores and outputs are computed TRANSPOSED: S^T[16 positions][8 query rows] = K Q^T and O^T[16 dims][8 query rows] += V^T P^T by mma.m16n8k16, so that
// the few query rows of a decode step (row = token * R + head of the group) fill the narrow side of the instruction and the cache the wide one. The cache's
// operands are its nibbles as they lie, masked: nib 2^-24 and 16 nib 2^-24, subnormal fp16 numbers, which the tensor pipe multiplies exactly; the 16 is
// taken out of Q for the keys and of the outputs for the values. A position's s and z join in fp32, S = s (q . nib) + (z - 8 s) (sum q) behind the product, and
// (p s) ahead of it for O, with the sum of p (z - 8 s) apart. Q is fp16 times a power of two per row (exact for elements down to 2^-27 of the row's
// largest); p s is rounded to fp16 (half a step is 2^-11 of it, the output's bf16 rounding 2^-8) times a power of two that follows the row's largest p s.
// The maximum that p refers to and that power are looked at by votes and moved only when a score is more than 2^6 above the one or a p s 2^14 above the other.
// Warps 0 .. W-1 take the CTA's units of U positions in turn, each through NST stages of its own; lane w of warp W brings the units of warp w, one bulk copy
// each. They meet at the end, then the CTAs that share the positions: a cluster pushes its partials to the CTA that finishes the row, more CTAs
// than a cluster leave them to kv4_join.
template <int HD, int NQ, int W>
struct Kv4Few {
  static constexpr int U = kFewUnit, NST = 3, ROWS = 8 * NQ, PW = HD + 4;         // positions of a unit, stages of a warp, query rows, floats of a partial
  static constexpr int STAGE = U / 16 * Kv4<HD>::BLOCK, RING = W * NST * STAGE, PART = W * ROWS * PW * 4;
  static constexpr int INBOX = RING > PART ? RING : PART;
  static constexpr int BAR = INBOX + 16 * PW * 4, SKIP = BAR + 2 * W * NST * 8, TOTAL = SKIP + W * NST * 4 + 16;
  static_assert(TOTAL <= 227 * 1024 && W < 32, "shared memory, a lane per warp");
};

// W + 1 warps. CLUSTER: grid (nsplit x row groups, nkv) of one sequence, the nsplit CTAs are a cluster; else grid (tasks)
template <int HD, int NQ, int W, bool CLUSTER>
__global__ void __launch_bounds__(W * 32 + 32) kv4_attn_few(const Kv4Attend P) {
  using C = Kv4<HD>;
  using F = Kv4Few<HD, NQ, W>;
  constexpr int KS = HD / 16, MT = HD / 16, NW = HD / 32 + (HD > C::MAIN), U = F::U, NST = F::NST, ROWS = F::ROWS, PW = F::PW;
  extern __shared__ __align__(128) uint8_t sm[];
  const Kv4Seqs& S = P.S;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, R = P.R;
  uint64_t *full = reinterpret_cast<uint64_t*>(sm + F::BAR), *empty = full + W * NST;      // [stage][warp]
  volatile int* s_skip = reinterpret_cast<volatile int*>(sm + F::SKIP);                     // the stage's unit has no page
  volatile int* s_abort = s_skip + W * NST;
  pdl_begin(true);
  Kv4Task<ROWS, U> task;
  const int ns = CLUSTER ? P.nsplit : 1, rank = CLUSTER ? (int)blockIdx.x % ns : 0;
  if (CLUSTER) {
    task.b = 0;
    task.kvh = blockIdx.y;
    if (!task.seq.get(S, 0, blockIdx.x == 0 && blockIdx.y == 0 && tid == 0)) return;         // the same for every CTA of a cluster
    const int grp = (int)blockIdx.x / ns, nu = task.set(P, grp), per = (nu + ns - 1) / ns;
    task.unit = min(rank * per, nu);
    task.n = min(per, nu - task.unit);
  } else if (!task.template find<false>(P, blockIdx.x, lane, blockIdx.x == 0 && warp == 0)) {
    return;
  }
  const Kv4Seq& seq = task.seq;
  const int rows = task.rows, r0 = task.r0, total = task.total, kvh = task.kvh, b = task.b;
  if (CLUSTER) cluster_arrive();                                 // partials are sent once every neighbour is known to run
  const int u_begin = task.unit, n = task.n, rounds = (n + W - 1) / W;
  int page = warp == W && lane < min(W, n) ? kv4_page(S, b, (u_begin + lane) * U, true) : -1;
  if (tid < W * NST) {
    mbar_init(&full[tid], 1);
    mbar_init(&empty[tid], 1);
    mbar_fence_init();
  }
  if (tid == 0) *s_abort = 0;
  __syncthreads();
  const WaitCtl wc{S.status, s_abort, P.spin_limit};
  bool ok = true;
  uint32_t issued = 0;                                           // of the copying warp, a lane each: its copies (and pages that are none)
  if (warp == W) {
    int st = 0;
    uint32_t lap = 1;
    for (int round = 0; round < rounds && ok; round++) {
      const int i = round * W + lane;
      const bool mine = lane < W && i < n;
      const int now = page;
      if (mine && i + W < n) page = kv4_page(S, b, (u_begin + i + W) * U, true);
      if (mine) {
        const int k = st * W + lane;
        ok = mbar_wait(&empty[k], lap, wc, W_EMPTY, 31);
        if (ok) {
          s_skip[k] = now < 0;
          if (now < 0) {
            mbar_arrive(&full[k]);
          } else {
            mbar_expect_tx(&full[k], F::STAGE);
            bulk_g2s(sm + k * F::STAGE, kv4_block<HD>(S, now, kvh, (u_begin + i) * U), F::STAGE, &full[k]);
          }
          issued++;
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      if (++st == NST) { st = 0; lap ^= 1u; }
    }
  }
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
      const float a = bflo(w[i]) * f.x, c = bfhi(w[i]) * f.x, h = i & 1 ? 0.0625f : 1.f;
      sum += a + c;
      qf[nq][i >> 1][i & 1] = cvt_f16x2(a * h, c * h);
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
    for (int e = 0; e < 2; e++) {
      c2[nq][e] = __shfl_sync(0xffffffffu, f.y, (2 * t + e) * 4) * P.scale * 0x1p24f;
      qs[nq][e] = __shfl_sync(0xffffffffu, sum, (2 * t + e) * 4) * 0x1p-24f;
    }
  }
  float o[NQ][MT][4], mrun[NQ][2], lrun[NQ][2], zrun[NQ][2];
  float wtop[NQ][2], wlim[NQ][2], vf[NQ][2];                     // this lane's largest p s, how large one may be, the power of two that p s is multiplied by:
  uint32_t erun[NQ][2];                                          // 2^(127 - erun), o is in units of its inverse (and of 2^-24 or 2^-20)
#pragma unroll
  for (int nq = 0; nq < NQ; nq++) {
#pragma unroll
    for (int i = 0; i < MT; i++) o[nq][i][0] = o[nq][i][1] = o[nq][i][2] = o[nq][i][3] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; e++) {
      mrun[nq][e] = kLowest; lrun[nq][e] = 0.f; zrun[nq][e] = 0.f;
      wtop[nq][e] = 0.f; wlim[nq][e] = 0.f; vf[nq][e] = 1.f; erun[nq][e] = 127;
    }
  }
  auto scale_o = [&](int nq, float a, float c) {
#pragma unroll
    for (int j = 0; j < MT; j++) { o[nq][j][0] *= a; o[nq][j][1] *= c; o[nq][j][2] *= a; o[nq][j][3] *= c; }
  };
  auto top = [&](float x) {                                      // over the lanes of a column
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
    return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
  };
  // one unit; EDGE: it holds new tokens, or slots behind them
  auto unit = [&](const uint8_t* base, int slot0, auto edge) {
    constexpr bool EDGE = decltype(edge)::value;
    float sc[NQ][U / 16][4], vs[U / 16][2], vz[U / 16][2];
    uint32_t unseen[NQ];                                         // EDGE: bit 4 k + i: element i of block k is not seen
#pragma unroll
    for (int nq = 0; nq < NQ; nq++) unseen[nq] = 0;
    uint32_t wl[U / 16][NW], wh[U / 16][NW];                     // words of positions g and g + 8
#pragma unroll
    for (int k = 0; k < U / 16; k++) {
      const uint8_t* blk = base + k * C::BLOCK;
#pragma unroll
      for (int nq = 0; nq < NQ; nq++) sc[nq][k][0] = sc[nq][k][1] = sc[nq][k][2] = sc[nq][k][3] = 0.f;
      if constexpr (HD == 128) {
        const uint4 x = *reinterpret_cast<const uint4*>(blk + g * 64 + t * 16), y = *reinterpret_cast<const uint4*>(blk + (g + 8) * 64 + t * 16);
        wl[k][0] = x.x; wl[k][1] = x.y; wl[k][2] = x.z; wl[k][3] = x.w;
        wh[k][0] = y.x; wh[k][1] = y.y; wh[k][2] = y.z; wh[k][3] = y.w;
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(blk + g * 32 + t * 8), y = *reinterpret_cast<const uint2*>(blk + (g + 8) * 32 + t * 8);
        wl[k][0] = x.x; wl[k][1] = x.y;
        wh[k][0] = y.x; wh[k][1] = y.y;
        if constexpr (HD > C::MAIN) {
          wl[k][2] = *reinterpret_cast<const uint32_t*>(blk + 512 + g * 8 + (t >> 1) * 4) >> (8 * (t & 1));
          wh[k][2] = *reinterpret_cast<const uint32_t*>(blk + 512 + (g + 8) * 8 + (t >> 1) * 4) >> (8 * (t & 1));
        }
      }
    }
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
      for (int k = 0; k < U / 16; k++) {
        const uint32_t a = wl[k][ks >> 1] >> (8 * (ks & 1)), c = wh[k][ks >> 1] >> (8 * (ks & 1));
        const uint32_t A[4] = {a & 0x000F000Fu, c & 0x000F000Fu, a & 0x00F000F0u, c & 0x00F000F0u};
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) mma_f16(sc[nq][k], A, qf[nq][ks][0], qf[nq][ks][1]);
      }
#pragma unroll
    for (int k = 0; k < U / 16; k++) {
      const uint8_t* blk = base + k * C::BLOCK;
      auto pair = [&](int off) { return *reinterpret_cast<const uint32_t*>(blk + off + g * 4); };
      const uint32_t k0 = pair(C::KSZ), k1 = pair(C::KSZ + 32), v0 = pair(C::VSZ), v1 = pair(C::VSZ + 32);
      vs[k][0] = bflo(v0); vs[k][1] = bflo(v1); vz[k][0] = fmaf(-8.f, vs[k][0], bfhi(v0)); vz[k][1] = fmaf(-8.f, vs[k][1], bfhi(v1));
      const float s0 = bflo(k0), s1 = bflo(k1), z0 = fmaf(-8.f, s0, bfhi(k0)), z1 = fmaf(-8.f, s1, bfhi(k1));
#pragma unroll
      for (int nq = 0; nq < NQ; nq++)
#pragma unroll
        for (int e = 0; e < 4; e++) sc[nq][k][e] = fmaf(e < 2 ? z0 : z1, qs[nq][e & 1], sc[nq][k][e] * (e < 2 ? s0 : s1)) * c2[nq][e & 1];
      if (EDGE) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int tp = slot0 + k * 16 + g + 8 * h, j = tp - seq.cached;
#pragma unroll
          for (int nq = 0; nq < NQ; nq++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              bool see = tp < total;
              if (see && j >= 0) {
                const int mq = min(r0 + nq * 8 + 2 * t + e, rows - 1) / R;
                see = P.amask ? j < P.mask_ld && P.amask[(size_t)(seq.first + mq) * P.mask_ld + j] != 0 : j <= mq;
              }
              if (!see) { sc[nq][k][2 * h + e] = -INFINITY; unseen[nq] |= 1u << (4 * k + 2 * h + e); }
            }
        }
      }
    }
    bool far = false;
#pragma unroll
    for (int nq = 0; nq < NQ; nq++)
#pragma unroll
      for (int e = 0; e < 2; e++)
#pragma unroll
        for (int k = 0; k < U / 16; k++) far = far || fmaxf(sc[nq][k][e], sc[nq][k][2 + e]) > mrun[nq][e] + 6.f;
    const bool moved = __any_sync(0xffffffffu, far);
    if (moved) {
#pragma unroll
      for (int nq = 0; nq < NQ; nq++) {
        float cr[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float mx = -INFINITY;
#pragma unroll
          for (int k = 0; k < U / 16; k++) mx = fmaxf(mx, fmaxf(sc[nq][k][e], sc[nq][k][2 + e]));
          const float mn = fmaxf(mrun[nq][e], top(mx));          // finite from below
          cr[e] = ex2(mrun[nq][e] - mn);
          mrun[nq][e] = mn;
          lrun[nq][e] *= cr[e]; zrun[nq][e] *= cr[e]; wtop[nq][e] *= cr[e];
        }
        scale_o(nq, cr[0], cr[1]);
      }
    }
    bool large = false;
#pragma unroll
    for (int nq = 0; nq < NQ; nq++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
#pragma unroll
        for (int k = 0; k < U / 16; k++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const int i = 2 * h + e;
            const float p = ex2(sc[nq][k][i] - mrun[nq][e]);
            const bool out = EDGE && (unseen[nq] >> (4 * k + i) & 1);      // an unseen row may be NaN
            const float w = out ? 0.f : p * vs[k][h];
            lrun[nq][e] += p;
            zrun[nq][e] = fmaf(p, out ? 0.f : vz[k][h], zrun[nq][e]);
            wtop[nq][e] = fmaxf(wtop[nq][e], w);
            sc[nq][k][i] = w;
          }
        large = large || wtop[nq][e] > wlim[nq][e];
      }
    if (__any_sync(0xffffffffu, large) || moved) {
#pragma unroll
      for (int nq = 0; nq < NQ; nq++) {
        float up[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const uint32_t en = min(max(__float_as_uint(top(wtop[nq][e])) >> 23, 15u), 239u);
          up[e] = __uint_as_float((uint32_t)(127 + min(max((int)erun[nq][e] - (int)en, -126), 126)) << 23);
          erun[nq][e] = en;
          vf[nq][e] = __uint_as_float((254u - en) << 23);
          wlim[nq][e] = __uint_as_float((en + 14u) << 23);
        }
        scale_o(nq, up[0], up[1]);
      }
    }
#pragma unroll
    for (int k = 0; k < U / 16; k++) {
      uint32_t pb[NQ][2];
#pragma unroll
      for (int nq = 0; nq < NQ; nq++)
#pragma unroll
        for (int h = 0; h < 2; h++) pb[nq][h] = movmatrix_trans(cvt_f16x2(sc[nq][k][2 * h] * vf[nq][0], sc[nq][k][2 * h + 1] * vf[nq][1]));
      const uint8_t* vb = base + k * C::BLOCK + C::V;
      uint32_t x0[NW], x1[NW];                                   // words of pairs t and t + 4
      if constexpr (HD == 128) {
        const uint4 x = *reinterpret_cast<const uint4*>(vb + t * 128 + ((g ^ (2 * t)) << 4)),
                    y = *reinterpret_cast<const uint4*>(vb + (t + 4) * 128 + ((g ^ (2 * t)) << 4));
        x0[0] = x.x; x0[1] = x.y; x0[2] = x.z; x0[3] = x.w;
        x1[0] = y.x; x1[1] = y.y; x1[2] = y.z; x1[3] = y.w;
      } else {
        const uint32_t off = (uint32_t)((g * 8) ^ ((t >> 1) * 32));
        const uint2 x = *reinterpret_cast<const uint2*>(vb + t * 64 + off), y = *reinterpret_cast<const uint2*>(vb + (t + 4) * 64 + off);
        x0[0] = x.x; x0[1] = x.y;
        x1[0] = y.x; x1[1] = y.y;
        if constexpr (HD > C::MAIN) {
          x0[2] = *reinterpret_cast<const uint32_t*>(vb + 512 + t * 16 + (g >> 1) * 4) >> (8 * (g & 1));
          x1[2] = *reinterpret_cast<const uint32_t*>(vb + 512 + (t + 4) * 16 + (g >> 1) * 4) >> (8 * (g & 1));
        }
      }
#pragma unroll
      for (int j = 0; j < MT; j++) {
        const uint32_t a = x0[j >> 1] >> (8 * (j & 1)), c = x1[j >> 1] >> (8 * (j & 1));
        const uint32_t A[4] = {a & 0x000F000Fu, a & 0x00F000F0u, c & 0x000F000Fu, c & 0x00F000F0u};
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) mma_f16(o[nq][j], A, pb[nq][0], pb[nq][1]);
      }
    }
  };
  int st = 0;
  uint32_t lap = 0;
#pragma unroll 1
  for (int i = warp; i < n && warp < W; i += W) {
    const int k = st * W + warp;
    if (!mbar_try(&full[k], lap)) ok = mbar_wait(&full[k], lap, wc, W_FULL, 30);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) break;
    if (!s_skip[k]) {
      const uint8_t* base = sm + k * F::STAGE;
      const int slot0 = (u_begin + i) * U;
      if (slot0 + U > seq.cached) unit(base, slot0, std::true_type());
      else unit(base, slot0, std::false_type());
    }
    __syncwarp();                                                // every lane has read the stage
    if (lane == 0) mbar_arrive(&empty[k]);
    if (++st == NST) { st = 0; lap ^= 1u; }
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
  if (*s_abort && warp == W && lane < W)                         // after a failure: the copies in flight
    drain_ring_order<NST>(issued, [&](uint32_t stage, uint32_t parity) { drain_phase(&full[stage * W + lane], parity); });
  __syncthreads();
  float* part = reinterpret_cast<float*>(sm);
  if (warp < W) {
#pragma unroll
    for (int nq = 0; nq < NQ; nq++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float* pr = part + (size_t)(warp * ROWS + nq * 8 + 2 * t + e) * PW;
        const float back = __uint_as_float(erun[nq][e] << 23);   // 2^(erun - 127)
#pragma unroll
        for (int j = 0; j < MT; j++) {
          const int d = 8 * j < C::MAIN / 2 ? C::MAIN / 8 * g + 2 * j : C::MAIN + 2 * g;
          *reinterpret_cast<float2*>(pr + d) = make_float2(fmaf(o[nq][j][e] * 0x1p24f, back, zrun[nq][e]), fmaf(o[nq][j][2 + e] * 0x1p20f, back, zrun[nq][e]));
        }
        if (g == 0) *reinterpret_cast<float2*>(pr + HD) = make_float2(mrun[nq][e], lrun[nq][e]);
      }
  }
  __syncthreads();
  if (CLUSTER) cluster_wait();
  for (int lr = warp; lr < min(ROWS, rows - r0); lr += W + 1) {
    float4 acc;
    float mm, den;
    kv4_merge<HD>(part + (size_t)lr * PW, min(W, max(n, 1)), ROWS * PW, lane, acc, mm, den);
    if (!CLUSTER && task.parts == 1) {
      kv4_finish<HD>(P, seq, kvh, r0 + lr, lane, acc, den);
    } else if (CLUSTER) {                                        // to the CTA that finishes the row
      const uint32_t to = (uint32_t)(lr % ns), slot = (uint32_t)(rank * ((ROWS + ns - 1) / ns) + lr / ns);
      const uint32_t a = cluster_map(smem_u32(sm + F::INBOX) + slot * PW * 4, to);
      if (lane < HD / 4) st_cluster(a + lane * 16, acc);
      if (lane == 0) st_cluster(a + HD * 4, make_float4(mm, den, 0.f, 0.f));
    } else {
      float* w = P.work + ((size_t)blockIdx.x * ROWS + lr) * PW;
      if (lane < HD / 4) *reinterpret_cast<float4*>(w + lane * 4) = acc;
      if (lane == 0) *reinterpret_cast<float2*>(w + HD) = make_float2(mm, den);
    }
  }
  if (CLUSTER) {
    cluster_arrive();
    cluster_wait();
    const int own = (ROWS + ns - 1) / ns;
    for (int i = warp; i < own && i * ns + rank < min(ROWS, rows - r0); i += W + 1) {
      float4 acc;
      float mm, den;
      kv4_merge<HD>(reinterpret_cast<const float*>(sm + F::INBOX) + (size_t)i * PW, ns, own * PW, lane, acc, mm, den);
      kv4_finish<HD>(P, seq, kvh, r0 + i * ns + rank, lane, acc, den);
    }
  }
}

// The partials of rows whose positions were split. WARPS 8: as many warps share the parts of a row, grid (row groups, nkv, rows of a group): one long
// sequence, whose positions are in many parts (37 of 32 K positions by one warp: 5 us more). WARPS 1: a warp a row, eight rows a CTA, grid (row groups, nkv, rows /
// 8): a batch, whose sequences are in few (48 sequences with eight warps a row: 20 us more), and the many rows of kv4_attn_many.
template <int HD, int ROWS, int U, int WARPS>
__global__ void __launch_bounds__(256) kv4_join(const Kv4Attend P) {
  constexpr int PW = HD + 4;
  __shared__ __align__(16) float part[WARPS * PW];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lr = WARPS == 1 ? (int)blockIdx.z * 8 + warp : (int)blockIdx.z, w0 = WARPS == 1 ? 0 : warp;
  pdl_begin(true);
  Kv4Task<ROWS, U> task;
  task.kvh = blockIdx.y;
  if (!task.template find<true>(P, blockIdx.x, lane, false) || task.parts == 1 || task.r0 + lr >= task.rows) return;
  const long long t0 = task.task_of(P, 0), step = task.task_of(P, 1) - t0;
  float4 acc;
  float mm, den;
  kv4_merge<HD>(P.work + ((size_t)(t0 + w0 * step) * ROWS + lr) * PW, (task.parts - w0 + WARPS - 1) / WARPS, (size_t)step * WARPS * ROWS * PW, lane, acc, mm, den);
  if (WARPS > 1) {
    if (lane < HD / 4) *reinterpret_cast<float4*>(part + warp * PW + lane * 4) = acc;
    if (lane == 0) *reinterpret_cast<float2*>(part + warp * PW + HD) = make_float2(mm, den);
    __syncthreads();
    if (warp) return;
    kv4_merge<HD>(part, min(WARPS, task.parts), PW, lane, acc, mm, den);
  }
  kv4_finish<HD>(P, task.seq, task.kvh, task.r0 + lr, lane, acc, den);
}

}  // namespace fb
