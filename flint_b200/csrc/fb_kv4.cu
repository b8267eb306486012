// extern "C" entry points of the 4-bit paged K/V cache: append, attention, read-back, moves.
// No torch types, no CPU fallback: a failed CUDA call or an unsupported shape is an error code.
#include <string.h>

#include "../../include/flint_b200.h"
#include "fb_ctx.hpp"
#include "fb_kv4.cuh"
#include "fb_kv4_geometry.hpp"
#include "fb_kv4_tc.cuh"

using namespace fb;

namespace {

int device_sms(int dev) {
  static int sms[64] = {};
  if (dev < 0 || dev >= 64) return 0;
  if (!sms[dev] && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return sms[dev];
}

// The call's device, made current only where it is not (that alone takes half a microsecond)
struct OnDevice {
  int prev = 0;
  bool ok = false, moved = false;
  explicit OnDevice(int dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) return;
    ok = prev == dev || (moved = cudaSetDevice(dev) == cudaSuccess);
  }
  ~OnDevice() { if (moved) cudaSetDevice(prev); }
};

// FB_OK and the kernels' view of the sequences, or why not
int take_seqs(const fb_kv4_seqs* s, int rows_of_tokens, Kv4Seqs& S) {
  if (!s || !s->d_pool || !s->d_table || !s->d_status) return FB_ERR_ARG;
  if (((uintptr_t)s->d_pool & 15) || ((uintptr_t)s->d_table & 3) || ((uintptr_t)s->d_start & 3) || ((uintptr_t)s->d_cached & 3) || ((uintptr_t)s->d_status & 3))
    return FB_ERR_ARG;
  if (s->head_dim != 64 && s->head_dim != 80 && s->head_dim != 128) return FB_ERR_SHAPE;
  if (s->n_kv_head < 1 || s->n_kv_head > 65535 || s->n_pages < 1 || s->table_ld < 1 || s->n_seq < 0 || s->n_tokens < 0) return FB_ERR_ARG;
  if (s->table_ld > 0x7fffffff / kPage) return FB_ERR_RANGE;
  if (rows_of_tokens && s->n_seq > 1 && !s->d_start) return FB_ERR_ARG;
  if (!s->d_cached && (s->cached < 0 || (!s->d_start && (int64_t)s->cached + s->n_tokens > (int64_t)s->table_ld * kPage))) return FB_ERR_RANGE;
  S = Kv4Seqs{(uint8_t*)s->d_pool, s->d_table, s->d_start, s->d_cached, s->cached, s->n_pages, s->n_kv_head, s->n_seq, s->table_ld, s->n_tokens, (DevStatus*)s->d_status};
  return FB_OK;
}
int done(cudaError_t e) { return e == cudaSuccess ? FB_OK : FB_ERR_CUDA; }

// rows of 16-bit numbers that are read 16 bytes at a time
bool rows_ok(const void* p, int64_t ld, int64_t width) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0 && ld >= width; }

template <class K>
cudaError_t configure_few(K k, int smem, bool (&configured)[64]) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (configured[dev]) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  configured[dev] = e == cudaSuccess;
  return e;
}
template <int HD, int NQ, int W>
cudaError_t launch_few(Kv4Attend p, const Kv4Geometry& g, cudaStream_t st) {
  using F = Kv4Few<HD, NQ, W>;
  static bool done_c[64] = {}, done_s[64] = {};
  p.nsplit = g.nsplit; p.slots = g.slots; p.chunk = g.chunk;
  if (g.groups * g.nsplit > 0x7fffffff || g.ctas > 0x7fffffff) return cudaErrorInvalidValue;
  const dim3 block(W * 32 + 32);
  if (g.nsplit > 1) {
    const cudaError_t e = configure_few(kv4_attn_few<HD, NQ, W, true>, F::TOTAL, done_c);
    return e != cudaSuccess ? e : launch_pdl_cluster(kv4_attn_few<HD, NQ, W, true>, dim3((unsigned)(g.groups * g.nsplit), (unsigned)p.S.nkv), block,
                                                     (size_t)F::TOTAL, st, (unsigned)g.nsplit, p);
  }
  cudaError_t e = configure_few(kv4_attn_few<HD, NQ, W, false>, F::TOTAL, done_s);
  if (e == cudaSuccess) e = launch_pdl(kv4_attn_few<HD, NQ, W, false>, dim3((unsigned)g.ctas), block, (size_t)F::TOTAL, st, p);
  if (e != cudaSuccess || !g.slots) return e;
  if (p.S.n_seq == 1)
    return launch_pdl(kv4_join<HD, F::ROWS, F::U, 8>, dim3((unsigned)g.groups, (unsigned)p.S.nkv, F::ROWS), dim3(256), 0, st, p);
  return launch_pdl(kv4_join<HD, F::ROWS, F::U, 1>, dim3((unsigned)g.groups, (unsigned)p.S.nkv, F::ROWS / 8), dim3(256), 0, st, p);
}
// kv4_attn_many deals its registers out anew and counts on 128 a thread at launch
template <int HD, int ROWS>
bool configured_many() {
  static int regs = 0;
  cudaFuncAttributes a;
  if (!regs && cudaFuncGetAttributes(&a, kv4_attn_many<HD, ROWS>) == cudaSuccess) regs = a.numRegs;
  return regs == 128;
}
template <int HD, int ROWS>
cudaError_t launch_many(Kv4Attend p, const Kv4Geometry& g, cudaStream_t st) {
  static bool done[64] = {};
  p.nsplit = 1; p.slots = g.slots; p.chunk = g.chunk;
  if (g.groups > 0x7fffffff || g.ctas > 0x7fffffff) return cudaErrorInvalidValue;
  if (g.groups > 0 && !configured_many<HD, ROWS>()) return cudaErrorInvalidConfiguration;
  cudaError_t e = configure_few(kv4_attn_many<HD, ROWS>, Kv4Many<HD>::TOTAL, done);
  if (e == cudaSuccess) e = launch_pdl(kv4_attn_many<HD, ROWS>, dim3((unsigned)g.ctas), dim3(kManyThreads), (size_t)Kv4Many<HD>::TOTAL, st, p);
  if (e == cudaSuccess && g.slots)
    e = launch_pdl(kv4_join<HD, ROWS, kManyStep, 1>, dim3((unsigned)g.groups, (unsigned)p.S.nkv, ROWS / 8), dim3(256), 0, st, p);
  return e;
}
template <int HD>
cudaError_t launch_attend(const Kv4Attend& p, const Kv4Geometry& g, cudaStream_t st) {
  if (g.rows >= kManyRows / 2) return g.rows == kManyRows ? launch_many<HD, kManyRows>(p, g, st) : launch_many<HD, kManyRows / 2>(p, g, st);
  return (g.rows == 8 ? launch_few<HD, 1, kFewWarps>(p, g, st) : launch_few<HD, 2, kFewWarps>(p, g, st));
}

}  // namespace

extern "C" {

size_t fb_kv4_page_bytes(int32_t n_kv_head, int32_t head_dim) {
  if (n_kv_head < 1 || (head_dim != 64 && head_dim != 80 && head_dim != 128)) return 0;
  return (size_t)n_kv_head * (kPage / 16) * (16 * (size_t)head_dim + 128);
}

int fb_kv4_append(const fb_kv4_seqs* s, const void* d_q, int64_t q_ld, const void* d_k, int64_t k_ld, const void* d_v, int64_t v_ld, int32_t n_head,
                  const int32_t* d_depth, const uint64_t* d_freq, void* d_q_out, int64_t qo_ld, void* stream) {
  Kv4Append p;
  const int rc = take_seqs(s, 1, p.S);
  if (rc != FB_OK) return rc;
  if (s->n_tokens == 0 || s->n_seq == 0) return FB_OK;
  const int64_t hd = s->head_dim, kw = hd * s->n_kv_head, qw = hd * n_head;
  if (!d_k || !d_v || !rows_ok(d_k, k_ld, kw) || !rows_ok(d_v, v_ld, kw) || ((uintptr_t)d_freq & 7) || ((uintptr_t)d_depth & 3)) return FB_ERR_ARG;
  if (d_q && (!d_q_out || n_head < 1 || !rows_ok(d_q, q_ld, qw) || !rows_ok(d_q_out, qo_ld, qw))) return FB_ERR_ARG;
  OnDevice g(s->device);
  const int sms = device_sms(s->device);
  if (!g.ok || !sms) return FB_ERR_CUDA;
  p.q = (const uint16_t*)d_q; p.k = (const uint16_t*)d_k; p.v = (const uint16_t*)d_v; p.q_out = (uint16_t*)d_q_out;
  p.q_ld = q_ld; p.k_ld = k_ld; p.v_ld = v_ld; p.qo_ld = qo_ld;
  p.depth = d_depth; p.freq = (const unsigned long long*)d_freq; p.nh = n_head;
  const int groups = ((d_q ? n_head : 0) + 2 * s->n_kv_head + 7) / 8, room = 4 * sms / s->n_tokens;
  const dim3 grid(s->n_tokens, groups < room ? groups : (room > 1 ? room : 1)), block(256);
  cudaStream_t st = (cudaStream_t)stream;
  switch (s->head_dim) {
    case 64: return done(launch_pdl(kv4_append<64>, grid, block, 0, st, p));
    case 80: return done(launch_pdl(kv4_append<80>, grid, block, 0, st, p));
    default: return done(launch_pdl(kv4_append<128>, grid, block, 0, st, p));
  }
}

int fb_kv4_read(const fb_kv4_seqs* s, int32_t n_layer, int64_t layer_bytes, float* d_k, float* d_v, void* stream) {
  Kv4Read p;
  const int rc = take_seqs(s, 1, p.S);
  if (rc != FB_OK) return rc;
  if (n_layer < 1 || n_layer > 65535 || layer_bytes < 0 || layer_bytes % 16 || ((uintptr_t)d_k & 15) || ((uintptr_t)d_v & 15)) return FB_ERR_ARG;
  if (s->n_tokens == 0 || s->n_seq == 0 || (!d_k && !d_v)) return FB_OK;
  OnDevice g(s->device);
  if (!g.ok) return FB_ERR_CUDA;
  p.k = d_k; p.v = d_v; p.layer = (size_t)layer_bytes;
  const dim3 grid(s->n_tokens, n_layer), block(256);
  cudaStream_t st = (cudaStream_t)stream;
  switch (s->head_dim) {
    case 64: return done(launch_pdl(kv4_read<64>, grid, block, 0, st, p));
    case 80: return done(launch_pdl(kv4_read<80>, grid, block, 0, st, p));
    default: return done(launch_pdl(kv4_read<128>, grid, block, 0, st, p));
  }
}

static int launch_move(const fb_kv4_seqs* s, const Kv4Move& p, int32_t n_layer, cudaStream_t st) {
  const dim3 grid(s->n_kv_head, n_layer), block(128);
  switch (s->head_dim) {
    case 64: return done(launch_pdl(kv4_move<64>, grid, block, 0, st, p));
    case 80: return done(launch_pdl(kv4_move<80>, grid, block, 0, st, p));
    default: return done(launch_pdl(kv4_move<128>, grid, block, 0, st, p));
  }
}

int fb_kv4_compact(const fb_kv4_seqs* s, int32_t n_layer, int64_t layer_bytes, const int32_t* d_accept, int32_t most, void* stream) {
  Kv4Move p;
  memset(&p, 0, sizeof(p));
  const int rc = take_seqs(s, 0, p.S);
  if (rc != FB_OK) return rc;
  if (s->n_seq < 1 || !d_accept || ((uintptr_t)d_accept & 3) || most < 0 || n_layer < 1 || n_layer > 65535 || layer_bytes < 0 || layer_bytes % 16 || s->d_cached) return FB_ERR_ARG;
  if (s->cached > s->table_ld * kPage - 1) return FB_ERR_RANGE;
  OnDevice g(s->device);
  if (!g.ok) return FB_ERR_CUDA;
  p.layer = (size_t)layer_bytes; p.accept = d_accept; p.pos = s->cached; p.most = most;
  return launch_move(s, p, n_layer, (cudaStream_t)stream);
}

int fb_kv4_move(const fb_kv4_seqs* s, int32_t n_layer, int64_t layer_bytes, const int32_t* src, const int32_t* dst, int32_t n, void* stream) {
  Kv4Move p;
  memset(&p, 0, sizeof(p));
  const int rc = take_seqs(s, 0, p.S);
  if (rc != FB_OK) return rc;
  if (s->n_seq < 1 || n < 0 || (n > 0 && (!src || !dst)) || n_layer < 1 || n_layer > 65535 || layer_bytes < 0 || layer_bytes % 16) return FB_ERR_ARG;
  const int64_t slots = (int64_t)s->table_ld * kPage;
  for (int i = 0; i < n; i++)
    if (src[i] < 0 || dst[i] < 0 || src[i] >= slots || dst[i] >= slots) return FB_ERR_RANGE;
  OnDevice g(s->device);
  if (!g.ok) return FB_ERR_CUDA;
  p.layer = (size_t)layer_bytes;
  for (int i0 = 0; i0 < n; i0 += 64) {                           // the moves of a launch travel in its parameters
    p.n = n - i0 < 64 ? n - i0 : 64;
    memcpy(p.src, src + i0, p.n * sizeof(int));
    memcpy(p.dst, dst + i0, p.n * sizeof(int));
    const int e = launch_move(s, p, n_layer, (cudaStream_t)stream);
    if (e != FB_OK) return e;
  }
  return FB_OK;
}

int fb_kv4_attend(const fb_kv4_seqs* s, const void* d_q, int64_t q_ld, int32_t n_head, int32_t max_new, int32_t max_len, const uint8_t* d_amask,
                  int32_t mask_ld, float scale, void* d_out, int64_t o_ld, void* d_work, size_t work_bytes, void* stream) {
  return kv4_attend(s, d_q, q_ld, n_head, max_new, max_len, d_amask, mask_ld, scale, d_out, o_ld, (float*)d_work, work_bytes, false, 4000000u, (cudaStream_t)stream);
}

}  // extern "C"

int kv4_attend(const fb_kv4_seqs* s, const void* d_q, int64_t q_ld, int32_t n_head, int32_t max_new, int32_t max_len, const uint8_t* d_amask, int32_t mask_ld,
               float scale, void* d_out, int64_t o_ld, float* work, size_t work_bytes, bool fit, unsigned spin_limit, cudaStream_t st) {
  Kv4Attend p;
  const int rc = take_seqs(s, 1, p.S);
  if (rc != FB_OK) return rc;
  if (s->n_tokens == 0 || s->n_seq == 0) return FB_OK;
  const int64_t qw = (int64_t)s->head_dim * n_head;
  if (n_head < 1 || n_head % s->n_kv_head) return FB_ERR_SHAPE;
  if (!d_q || !d_out || !rows_ok(d_q, q_ld, qw) || !rows_ok(d_out, o_ld, qw) || max_new < 1 || max_len < 1 || (d_amask && mask_ld < 1)) return FB_ERR_ARG;
  if ((int64_t)s->n_tokens * (n_head / s->n_kv_head) > 0x7fffffff - 256) return FB_ERR_RANGE;      /* rows of a sequence */
  OnDevice g(s->device);
  const int sms = device_sms(s->device);
  if (!g.ok || !sms) return FB_ERR_CUDA;
  p.q = (const uint16_t*)d_q; p.out = (uint16_t*)d_out; p.q_ld = q_ld; p.o_ld = o_ld; p.amask = d_amask; p.mask_ld = mask_ld;
  p.nh = n_head; p.R = n_head / s->n_kv_head;
  p.scale = scale * 1.4426950408889634f; p.spin_limit = spin_limit;
  Kv4Geometry geo = attend_geometry(s->n_seq, s->n_tokens, s->n_kv_head, p.R, max_new < s->n_tokens ? max_new : s->n_tokens, max_len, sms);
  if (fit && attend_work(geo, s->head_dim) > work_bytes) geo = whole(geo, s->n_kv_head);
  if (attend_work(geo, s->head_dim) > work_bytes || ((uintptr_t)work & 15)) return FB_ERR_ARG;
  p.work = work;
  switch (s->head_dim) {
    case 64: return done(launch_attend<64>(p, geo, st));
    case 80: return done(launch_attend<80>(p, geo, st));
    default: return done(launch_attend<128>(p, geo, st));
  }
}

size_t fb_kv4_attend_bytes(const fb_kv4_seqs* s, int32_t n_head, int32_t max_new, int32_t max_len) {
  if (!s || s->n_kv_head < 1 || s->n_kv_head > 65535 || n_head < 1 || n_head % s->n_kv_head || max_new < 1 || max_len < 1 || s->n_seq < 0) return 0;
  const int sms = device_sms(s->device);
  if (!sms) return 0;
  return attend_work(attend_geometry(s->n_seq, s->n_tokens, s->n_kv_head, n_head / s->n_kv_head, max_new < s->n_tokens ? max_new : s->n_tokens, max_len, sms), s->head_dim);
}
