// What the attention kernels on fp32 MFMAs (dce_attention.hip) and those on
// fp16 parts (dce_attention_parts.hip) share: the problem's description and the
// mask.
#pragma once
#include "dce_internal.h"

#include <algorithm>
#include <cmath>

namespace dce {

// Tokens come as [batch][token][head][dim].  `rep` query heads share one key
// head, so the problem of one (sequence, key head) pair is N = rep * S query
// rows against up to T keys: row n is query n / rep of head n % rep.
//
// Workgroups go through the problems first and their tiles next, the tiles with
// most work ahead: the last ones to start are the shortest, and as consecutive
// workgroups go to the 8 XCDs in turn, each XCD's L2 sees an eighth of the
// problems, or one of them where they are few.
struct Attn {
  const float *q, *k, *v, *len;  // len: keys of each sequence, or null
  float* o;
  float *m, *il;                 // row statistics [problem][N]; null: not kept
  float *pm, *pl, *po;           // partials of the key splits
  const float* dy;               // backward
  float *delta, *dq, *dk, *dv;
  uint32_t B, S, T, G, D, rep, N;
  uint32_t tiles, splits, perSplit;  // splits: of the keys (perSplit tiles each in the forward), or of the rows in dK, dV
  FastDiv dRep, dG;
  float c, scale;
  int causal;
};

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ uint32_t keys_of(const Attn& a, uint32_t b) {
  if (!a.len) return a.T;
  const float n = a.len[b];
  return n >= 1.f ? (n < float(a.T) ? uint32_t(n) : a.T) : 0u;  // NaN: none
}
// Keys that row n sees (row n of the problem, `len` keys in the sequence).
__device__ __forceinline__ uint32_t limit_of(const Attn& a, uint32_t n, uint32_t len) {
  if (!a.causal) return len;
  const int64_t e = int64_t(fdiv(n, a.dRep)) + int64_t(a.T) - int64_t(a.S) + 1;
  return e <= 0 ? 0u : uint32_t(min(e, int64_t(len)));
}
// Keys that `rows` rows from n on see, for a wave that holds them.
__device__ __forceinline__ uint32_t wave_limit(const Attn& a, uint32_t n, uint32_t rows, uint32_t len) {
  return __builtin_amdgcn_readfirstlane(n < a.N ? limit_of(a, min(n + rows, a.N) - 1, len) : 0u);
}
// First row that sees key k0.
__device__ __forceinline__ uint32_t first_row(const Attn& a, uint32_t k0) {
  const int64_t i = int64_t(k0) - (int64_t(a.T) - int64_t(a.S));
  return a.causal && i > 0 ? uint32_t(i) * a.rep : 0u;
}
// Rows [first, end) of split sp of those that see key k0 on, in whole 32-row tiles.
__device__ __forceinline__ void split_rows(const Attn& a, uint32_t k0, uint32_t len, uint32_t sp, uint32_t& first,
                                           uint32_t& end) {
  const uint32_t from = k0 < len ? min(first_row(a, k0), a.N) / 32 : 0u, to = k0 < len ? (a.N + 31) / 32 : 0u;
  first = (from + (to - from) * sp / a.splits) * 32;
  end = min((from + (to - from) * (sp + 1) / a.splits) * 32, a.N);
}
// Keys [first, end) of split sp of the `most` that a block of rows sees, in whole
// 32-key tiles, and the place of that split's dq.
__device__ __forceinline__ void split_keys(const Attn& a, uint32_t most, uint32_t sp, uint32_t& first, uint32_t& end) {
  const uint32_t tiles = (most + 31) / 32;
  first = tiles * sp / a.splits * 32;
  end = min(tiles * (sp + 1) / a.splits * 32, most);
}
__device__ __forceinline__ size_t dq_part(const Attn& a, uint32_t sp) {
  return size_t(sp) * a.B * a.G * a.N * a.D;
}
// First value of row n's vector in a [batch][seq][heads][dim] tensor.
__device__ __forceinline__ size_t q_at(const Attn& a, uint32_t b, uint32_t g, uint32_t n) {
  const uint32_t i = fdiv(n, a.dRep), h = g * a.rep + (n - i * a.rep);
  return ((size_t(b) * a.S + i) * (size_t(a.G) * a.rep) + h) * a.D;
}
__device__ __forceinline__ size_t k_at(const Attn& a, uint32_t b, uint32_t g, uint32_t j) {
  return ((size_t(b) * a.T + j) * a.G + g) * a.D;
}

inline uint32_t cdiv(uint64_t a, uint64_t b) { return uint32_t((a + b - 1) / b); }

// Pairs of a query and a key that the mask of full lengths leaves.
inline double pairs_of(const AttnArgs& x) {
  if (!x.causal) return double(x.S) * x.T;
  const double rows = std::min(x.S, x.T), last = x.T;
  return rows * last - rows * (rows - 1) / 2;
}

// Splits of a kernel's long side, `tiles` tiles of `us` microseconds each
// for each of `wgs` workgroups: the number of least time, where workgroups take
// the CUs in rounds (causal ones, longest first, fill them) and have some 8 us of
// their own, and each split's shares are written and read at 4 TB/s by a launch more.  10 x 1169 tokens, 3
// heads of 128 on one, 280 and 100 workgroups for 256 CUs: training 525 us with 1
// and 3 splits, 472 with 2 and 5; 1 x 6000 tokens, 2 heads of 96, 658 and 496.
inline uint32_t best_splits(double wgs, uint32_t tiles, double us, double shareBytes, bool causal) {
  const double cus = num_cus();
  const uint32_t most = uint32_t(std::min({256.0, (tiles + 7) / 8 + 0.0, std::max(1.0, 8 * cus / wgs)}));
  uint32_t best = 1;
  double least = INFINITY;
  for (uint32_t s = 1; s <= most; ++s) {
    const double one = tiles * us / s + 8;
    double t = causal ? std::max(one, 0.5 * wgs * (tiles * us + s * 8) / cus + one / 2) : std::ceil(wgs * s / cus) * one;
    if (s > 1) t += 5 + s * shareBytes * 2 / 4e6;
    if (t < 0.97 * least) {
      least = t;
      best = s;
    }
  }
  return best;
}
// Of the rows in a dK / dV kernel of `keys` keys per workgroup (64: on fp32, 128:
// on parts), and of the keys in a dQ kernel of `rows` rows: a tile's time is about
// proportional to the dims.
inline uint32_t row_splits(const Attn& a, uint32_t keys) {
  return best_splits(double(cdiv(a.T, keys)) * a.B * a.G, cdiv(a.N, 32), a.D * (keys == 64 ? 0.031 : 0.024),
                     8.0 * a.B * a.T * a.G * a.D, a.causal);
}
inline uint32_t key_splits(const Attn& a, uint32_t rows) {
  return best_splits(double(cdiv(a.N, rows)) * a.B * a.G, cdiv(a.T, 32), a.D * (rows == 64 ? 0.023 : 0.02),
                     4.0 * a.B * a.G * a.N * a.D, a.causal);
}

// Floats of the splits' shares of a backward, one kernel's after the other's.
inline size_t split_floats(const Attn& a, uint32_t rows, uint32_t keys) {
  const uint32_t sk = a.dq ? key_splits(a, rows) : 1, sr = a.dk || a.dv ? row_splits(a, keys) : 1;
  const size_t q = sk > 1 ? size_t(sk) * a.B * a.G * a.N * a.D : 0, k = sr > 1 ? 2 * size_t(sr) * a.B * a.T * a.G * a.D : 0;
  return std::max(q, k);
}

// Joins the key splits of a forward into o (and the statistics).
bool attn_join(const Attn& a);
// Adds the splits' shares of one or two results of n values each (null: none).
bool attn_sum(const float* p0, float* out0, const float* p1, float* out1, size_t n, uint32_t splits);
// On fp16 parts, where they are faster; `took` tells.
bool attn_fwd_parts(const AttnArgs& x, Attn a, bool* took);
bool attn_bwd_parts(const AttnArgs& x, Attn a, bool* took);

}  // namespace dce
