// Launch geometry of attention over the 4-bit cache as plain functions of the sizes: what fb_kv4.cu launches, what scratch that takes, and what a host-side test can ask. No CUDA here.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <initializer_list>

namespace fb {

constexpr int kFewRows = 64;                       // query rows of a kv head up to which kv4_attn_few does them
constexpr int kFewWarps = 7;                       // that compute, of a CTA of kv4_attn_few; an SM holds two CTAs
constexpr int kFewUnit = 32;                       // positions that a warp of it takes at a time
constexpr int kManyRows = 256, kManyStep = 128;    // of kv4_attn_many: most query rows of a task, positions of a step

// How an attention is cut. rows: query rows of a group; groups: of all sequences, at most; ctas: of a grid without clusters, at most.
// Up to kFewRows query rows a kv head: kv4_attn_few in groups of 8 or 16 rows, which dequantise the cache anew for each group. More: kv4_attn_many. Microseconds, few /
// many: 16 tokens of 4 heads (64 rows) behind 1024 positions 9.9 / 13.5, behind 4000 14.5 / 17.5, 12 (48 rows) behind 8000 24.2 / 23.9; 26 tokens (104 rows) behind
// 1024 13.5 / 13.2, behind 8000 44 / 26; 61 (244 rows) behind 3001 46 / 28.
// Few: a group's positions are shared by a cluster (one launch) while a warp of a cluster of eight has no more than six units; by as many CTAs as the GPU holds and a
// second launch that joins them, beyond that. (With one CTA of 16-row groups per SM the GPU holds 15 clusters of 8, but 36 of 4.) One sequence, eight
// kv heads, cluster / second launch: 1000 positions 5.5 / 8.2, 4000 6.7 / 8.5, 32768 20.5 / 13.1 (heads of 80). Of a batch no positions are shared until a
// warp would have more than 12 units: 48 sequences of up to 2000 positions 17.8 / 22.7, 24 of up to 8000 51 / 18.3 (over 148 parts; over 296 22.1).
// Many: a task has 128 or 256 query rows. A step of 128 positions takes about 2.5 us (1.6 with one tile of 128 rows), a task about two steps more, the second launch 5 us and what the
// partials take to write and read; rows and parts of the smallest sum are taken (all rows are counted with all positions, of which a prompt's first ones see fewer). 1000 tokens of
// 4 heads behind 7011 positions on 148 SMs: eight kv heads, 128 items of 256 rows, whole 168, two parts 206, with 128 rows 262; ten kv heads, 160 items, whole 307, three parts
// 277. Tree of 61 of 4 heads behind 3001, eight kv heads: 128 rows whole 58, eight parts 21.8, twelve 32; 256 rows in twelve parts 25.6. Tree of 26 behind 1024: whole 22.8,
// six parts 13.3. A prompt of 200 tokens: 11.1 with 128 rows, 13.1 with 256.
// rows of a group, groups, CTAs of a grid without clusters; CTAs of a cluster; tasks that all positions are cut into (0: they are not), of `chunk` units or more
struct Kv4Geometry { int rows; int64_t groups, ctas; int nsplit, slots, chunk; };
inline Kv4Geometry attend_geometry(int n_seq, int n_tokens, int nkv, int r, int max_new, int max_len, int sms) {
  Kv4Geometry g{(int64_t)max_new * r <= 8 ? 8 : 16, 0, 0, 1, 0, 8};
  auto groups_of = [&](int rows) { return n_seq == 1 ? ((int64_t)n_tokens * r + rows - 1) / rows : (int64_t)n_tokens * r / rows + n_seq; };
  const bool many = (int64_t)max_new * r > kFewRows;
  const int64_t units = ((int64_t)max_len + kFewUnit - 1) / kFewUnit, steps = ((int64_t)max_len + kManyStep - 1) / kManyStep;
  if (many) {
    g.chunk = 1;
    double best = 0;
    for (int rows : {kManyRows / 2, kManyRows}) {
      const double step_us = rows == kManyRows && (int64_t)max_new * r > kManyRows / 2 ? 2.5 : 1.6;
      const int64_t items = groups_of(rows) * nkv;
      for (int parts : {1, 2, 3, 4, 6, 8, 12, 16, 24}) {
        if (parts > steps || (parts > 1 && items * parts > 3 * sms)) break;
        const int64_t per = (steps + parts - 1) / parts, tasks = items * ((steps + per - 1) / per);
        const double us = (double)((tasks + sms - 1) / sms) * (double)(per + 2) * step_us + (parts > 1 ? 5.0 + (double)tasks * rows * 1056 / 3e6 : 0.0);
        if (best == 0 || us < best) { best = us; g.rows = rows; g.slots = parts > 1 ? (int)(items * parts) : 0; }
      }
    }
  }
  g.groups = groups_of(g.rows);
  const int64_t items = g.groups * nkv;
  if (!many && n_seq == 1) {
    while (g.nsplit < 8 && items * g.nsplit * 2 <= (g.nsplit == 4 ? sms * 2 / 3 : sms) && units >= g.nsplit * 2 * 4) g.nsplit *= 2;
    if (units > (int64_t)6 * kFewWarps * g.nsplit && items * g.nsplit <= sms) { g.nsplit = 1; g.slots = 2 * sms; }
  } else if (!many && units > 12 * kFewWarps && items <= 8 * (int64_t)sms) {
    g.slots = sms;
  }
  g.ctas = items + g.slots;
  return g;
}
inline size_t attend_work(const Kv4Geometry& g, int hd) { return g.slots ? (size_t)g.ctas * g.rows * (hd + 4) * 4 : 0; }
// the same without scratch: no positions are shared
inline Kv4Geometry whole(Kv4Geometry g, int nkv) {
  g.nsplit = 1; g.slots = 0;
  g.ctas = g.groups * nkv;
  return g;
}
// The most scratch that one sequence of up to `slots` positions asks for, at most `rows_max` new tokens a call. What is asked for goes by the number of groups of 128 rows and by steps
// (few rows: the longest sequence asks for most, as a sequence is split from some length on). Sequences of more than 4096 steps are looked at in strides: whoever has this much
// and needs more goes without (`whole`).
inline size_t attend_most(int nkv, int r, int head_dim, int64_t slots, int rows_max, int sms) {
  size_t most = 0;
  int64_t seen = -1;
  const int64_t steps = (slots + kManyStep - 1) / kManyStep, stride = steps > 4096 ? steps / 4096 : 1;
  for (int m = 1; m <= rows_max && m <= slots; m++) {
    const bool many = (int64_t)m * r > kFewRows;
    const int64_t groups = ((int64_t)m * r + kManyRows / 2 - 1) / (kManyRows / 2);
    if (many && groups == seen) continue;
    seen = many ? groups : -1;
    for (int64_t n = many ? (m + kManyStep - 1) / kManyStep : steps;; n = n + stride < steps ? n + stride : steps) {
      const int64_t len = n * kManyStep < slots ? n * kManyStep : slots;
      const size_t w = attend_work(attend_geometry(1, m, nkv, r, m, (int)len, sms), head_dim);
      if (w > most) most = w;
      if (n >= steps) break;
    }
  }
  return most;
}

}  // namespace fb
