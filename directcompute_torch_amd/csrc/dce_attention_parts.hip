// Attention on fp16 parts: the products of large calls at a third of the fp16
// MFMA rate, which is 16 times the fp32 one, with fp32's accuracy.
//
// A value x is kept as x 2^e = h + l, two fp16 values rounded to nearest, and
// h h + (h l + l h) stands for a product: the parts carry 22 to 24 bits, and a
// dot product rounds its sum once per 16 terms instead of at every one.  The
// exponent e is one for each tile of 32 vectors, chosen so that the tile's
// largest value lies in [2^14, 2^15): l's half step is then 2^-25, so a vector
// whose own largest value is within 2^12 of the tile's keeps at least 24 bits of
// it.  A tile that has smaller vectors than that (zeros aside), values outside of
// 2^+-30 (gradients: 2^+-60) or any that is not finite is marked by the pass that
// splits, and the workgroups of its (sequence, key head) run the fp32 code.
//
// A tile's exponent costs a score nothing: c 2^-(eq + ek) is the factor that turns
// it into base 2 anyway.  P and dS are made into parts with an exponent of their
// own for every column of the transposed product (the row of O or dQ, the key of
// dK or dV) and the tile's exponent, so that a column's largest term so far lies
// in [2^12, 2^15): l's half step, 2^-25, is then 2^-37 of it.  Where it was made from
// a vector 2^-12 of its tile's largest that is 2^-25 of the term, fp32's half step.
// A larger term scales the column's sum down, which few tiles past the first need.
// (One exponent for all columns, from a bound on dS, left dK 8 bits where other
// rows' gradients were 2^18 larger.)
//
// The backward's 1 / l goes into dO (dO' = dO / l) when that is split, so that
// dV = P^T dO' and dS = scale P (dO' V^T - delta'), delta' = rowsum(dO' * O).
#include "dce_attention_fp32.h"

#include <type_traits>

namespace dce {

namespace {

constexpr int kT = 256;
constexpr int kRows = 32;         // vectors of a tile
constexpr int kRange = 30;        // exponents of values that parts are made of
constexpr int kRangeGrad = 60;    // and of gradients
constexpr float kWide = 4096.f;   // largest ratio of the vectors' sizes in a tile
constexpr int kZeros = 15 + kRange, kZerosGrad = 15 + kRangeGrad;  // exponents of tiles of zeros, larger than any other
// A column's parts of P or dS are made with its largest value in [2^kTop, 2^(kTop + 1));
// a later tile's may go up to 2^kFull before the column's sum is scaled down.
constexpr int kTop = 12, kFull = 15;
constexpr int kMost = 100;   // the largest factor that makes them, 2^kMost
constexpr int kNone = 1000;  // exponent of a sum that has no terms yet

using h2 = _Float16 __attribute__((ext_vector_type(2)));
using h4 = _Float16 __attribute__((ext_vector_type(4)));
using h8 = _Float16 __attribute__((ext_vector_type(8)));
using f16v = float __attribute__((ext_vector_type(16)));
using s4v = short __attribute__((ext_vector_type(4)));
using u4v = uint32_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f16v mma(const h8& a, const h8& b, const f16v& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ void zero(f16v& v) {
#pragma unroll
  for (int e = 0; e < 16; ++e) v[e] = 0.f;
}
// 2^e, for e < 128; no less than 2^-126.
__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + max(e, -126)) << 23); }

// The parts of one operand: [problem][vector][h | l], DP halves each, zero past
// D and past the last vector up to whole tiles; one exponent per tile.
struct Part {
  char* p;
  int* e;        // kBad: not made
  uint32_t pad;  // vectors of a problem, a multiple of 128
};
struct Parts {
  Part q, k, v, y;
  float* dl;  // delta' 2^e of dO's tile, [problem][q.pad]
};
constexpr int kBad = 1 << 20;
// Does problem pr have a tile that parts do not suit, or vectors whose scores might
// pass 2^24, past which they are no place to add an exponent to?  For all threads of
// the workgroup.
template <bool BWD>
__device__ __forceinline__ bool unsuited(const Attn& a, const Parts& ps, uint32_t pr) {
  __shared__ float ends[8][3];
  const uint32_t nq = ps.q.pad / kRows, nk = ps.k.pad / kRows;
  // kBad passes all others; of q and k the least exponents, negated, too
  float most = 0.f, q = -1000.f, k = q;
  auto take = [&](const int* e, uint32_t n, float* least) {
    for (uint32_t t = threadIdx.x; t < n; t += blockDim.x) {
      const float x = float(e[size_t(pr) * n + t]);
      most = fmaxf(most, x);
      if (least) *least = fmaxf(*least, -x);
    }
  };
  take(ps.q.e, nq, &q);
  take(ps.k.e, nk, &k);
  take(ps.v.e, nk, nullptr);
  if (BWD) take(ps.y.e, nq, nullptr);
  const float w[3] = {wave_reduce(most, OpMaxR()), wave_reduce(q, OpMaxR()), wave_reduce(k, OpMaxR())};
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int i = 0; i < 3; ++i) ends[threadIdx.x >> 6][i] = w[i];
  __syncthreads();
  for (uint32_t i = 0; i < blockDim.x / 64; ++i) {
    most = fmaxf(most, ends[i][0]);
    q = fmaxf(q, ends[i][1]);
    k = fmaxf(k, ends[i][2]);
  }
  return most >= float(kBad) || !(fabsf(a.c) * float(a.D) < pow2(24 - 30 - int(q + k)));
}

// ---------------------------------------------------------------------------
// The pass that splits: a workgroup per tile.  Bound by memory, 8 bytes per value
// (dO: 12): 2 x 4096 tokens, 16 heads of 128, forward 72 us, 5.6 TB/s; backward 105.
// ---------------------------------------------------------------------------
enum Which { QUERY, KEY, VALUE, GRAD };
template <int DP, bool VEC, int W>
__device__ __forceinline__ void split_tile(const Attn& a, const Part& P, const Parts& ps, uint32_t pr, uint32_t tile) {
  constexpr int CH = DP / 8, SLOTS = (kRows * CH + kT - 1) / kT;
  constexpr bool ROWS = W == QUERY || W == GRAD;
  __shared__ uint32_t top[kRows];
  __shared__ float dots[kRows];
  __shared__ int all[1];
  const uint32_t b = fdiv(pr, a.dG), g = pr - b * a.G;
  const uint32_t n0 = tile * kRows, have = ROWS ? a.N : keys_of(a, b);
  if (threadIdx.x < kRows) {
    top[threadIdx.x] = 0;
    dots[threadIdx.x] = 0.f;
  }
  __syncthreads();
  float v[SLOTS][8], o[SLOTS][8], by_row[SLOTS];
  float part[SLOTS];
  // Loads of clamped places: behind a branch each would wait for the one before.
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    const uint32_t slot = threadIdx.x + kT * i, d = slot % CH * 8, n = min(n0 + slot / CH, max(have, 1u) - 1);
    const size_t at = ROWS ? q_at(a, b, g, n) : k_at(a, b, g, n);
    const float* src = (W == QUERY ? a.q : W == KEY ? a.k : W == VALUE ? a.v : a.dy) + at;
    by_row[i] = W == GRAD ? a.il[size_t(pr) * a.N + n] : 1.f;
#pragma unroll
    for (int e = 0; e < 8; e += VEC ? 4 : 1) {
      const uint32_t k = min(d + e, a.D - (VEC ? 4 : 1));
      if constexpr (VEC) {
        *reinterpret_cast<f4*>(v[i] + e) = *reinterpret_cast<const f4*>(src + k);
        if (W == GRAD) *reinterpret_cast<f4*>(o[i] + e) = *reinterpret_cast<const f4*>(a.o + at + k);
      } else {
        v[i][e] = src[k];
        if (W == GRAD) o[i][e] = a.o[at + k];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    const uint32_t slot = threadIdx.x + kT * i, row = slot / CH, d = slot % CH * 8, n = n0 + row;
    part[i] = 0.f;
    const bool live = row < kRows && n < have;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool ok = live && d + e < a.D;
      if (W == GRAD) part[i] += ok ? v[i][e] * o[i][e] : 0.f;
      v[i][e] = ok ? v[i][e] * by_row[i] : 0.f;
    }
    if (!live) continue;
    float m = 0.f;
    bool fine = true;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      m = fmaxf(m, fabsf(v[i][e]));
      fine &= fabsf(v[i][e]) < INFINITY;  // false for NaN too
    }
    // The largest value of a vector, as bits (which order as the values do).
    atomicMax(&top[row], fine ? __float_as_uint(m) : 0x7f800000u);
  }
  if constexpr (W == GRAD) {
    // rowsum(dO * O), the partial sums of a row in a fixed order
    __shared__ float sums[kRows * CH];
#pragma unroll
    for (int i = 0; i < SLOTS; ++i)
      if (threadIdx.x + kT * i < kRows * CH) sums[threadIdx.x + kT * i] = part[i];
    __syncthreads();
    if (threadIdx.x < kRows) {
      float s = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c) s += sums[threadIdx.x * CH + c];
      dots[threadIdx.x] = s;
    }
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    const uint32_t mine = threadIdx.x < kRows ? top[threadIdx.x] : 0u;
    const float most = wave_reduce(__uint_as_float(mine), OpMaxR());
    const float least = -wave_reduce(mine ? -__uint_as_float(mine) : -INFINITY, OpMaxR());
    if (threadIdx.x == 0) {
      constexpr int range = W == GRAD ? kRangeGrad : kRange;
      int e = W == GRAD ? kZerosGrad : kZeros;
      if (most > 0.f) {
        const bool bad = !(most < pow2(range)) || most < pow2(-range) || most > kWide * least;
        e = bad ? kBad : 14 + 127 - int(__float_as_uint(most) >> 23);
      }
      all[0] = e == kBad ? 0 : e;
      P.e[size_t(pr) * (P.pad / kRows) + tile] = e;
    }
  }
  __syncthreads();
  const float by = pow2(all[0]);
  char* out = P.p + (size_t(pr) * P.pad + n0) * (DP * 4);
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    const uint32_t slot = threadIdx.x + kT * i, row = slot / CH, c = slot % CH;
    if (row >= kRows) continue;
    h8 h, l;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = v[i][e] * by;
      h[e] = _Float16(x);
      l[e] = _Float16(x - float(h[e]));
    }
    *reinterpret_cast<h8*>(out + row * (DP * 4) + c * 16) = h;
    *reinterpret_cast<h8*>(out + row * (DP * 4) + DP * 2 + c * 16) = l;
  }
  if (W == GRAD && threadIdx.x < kRows) {
    const uint32_t n = n0 + threadIdx.x;
    const size_t row = size_t(pr) * a.N + n;
    if (n < a.N) a.delta[row] = dots[threadIdx.x];
    ps.dl[size_t(pr) * P.pad + n] = n < a.N ? dots[threadIdx.x] * a.il[row] * by : 0.f;
  }
}
// Tiles of q (and dO), then of k and v, of each problem.
template <int DP, bool VEC, bool BWD>
__global__ void __launch_bounds__(kT) k_attn_split(const Attn a, const Parts ps) {
  const uint32_t tq = ps.q.pad / kRows, tk = ps.k.pad / kRows, per = (BWD ? 2 : 1) * tq + 2 * tk;
  const uint32_t pr = blockIdx.x / per;
  uint32_t t = blockIdx.x - pr * per;
  if (t < tq) return split_tile<DP, VEC, QUERY>(a, ps.q, ps, pr, t);
  t -= tq;
  if (t < tk) return split_tile<DP, VEC, KEY>(a, ps.k, ps, pr, t);
  t -= tk;
  if (t < tk) return split_tile<DP, VEC, VALUE>(a, ps.v, ps, pr, t);
  if constexpr (BWD) split_tile<DP, VEC, GRAD>(a, ps.y, ps, pr, t - tk);
}

// ---------------------------------------------------------------------------
// An LDS tile of 32 vectors' parts: the h plane, then the l plane, the 16-byte
// chunks of a row XORed by the row: a read of one chunk of 16 rows covers the 64
// banks once, and so does a transposed read, 64 bytes of each of four rows.
// ---------------------------------------------------------------------------
template <int DP, int NT = kT>
struct PTile {
  static constexpr int CH = DP / 8, PLANE = kRows * DP * 2, BYTES = 2 * PLANE, SLOTS = BYTES / 16;
  static constexpr int LOADS = (SLOTS + NT - 1) / NT;
  static constexpr bool WHOLE = SLOTS % NT == 0;  // else the last load is for some threads only
  __device__ static __forceinline__ int swz(int row) {
    const int low = (row >> 2) & 3;
    return CH % 16 == 0 ? ((row & 3) << 2) | low : CH % 8 == 0 ? ((row & 2) << 1) | low : low;
  }
  __device__ static __forceinline__ void load(const char* p, u4v (&r)[LOADS]) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      if (WHOLE || threadIdx.x + NT * i < SLOTS) r[i] = reinterpret_cast<const u4v*>(p)[threadIdx.x + NT * i];
  }
  __device__ static __forceinline__ void store(char* S, const u4v (&r)[LOADS]) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int m = threadIdx.x + NT * i, row = m / (2 * CH), pl = m / CH & 1, c = m % CH;
      if (WHOLE || m < SLOTS) *reinterpret_cast<u4v*>(S + pl * PLANE + (row * CH + (c ^ swz(row))) * 16) = r[i];
    }
  }
  // Row `row`, dims 8 c .. + 7.
  __device__ static __forceinline__ h8 rows(const char* S, int pl, int row, int c) {
    return *reinterpret_cast<const h8*>(S + pl * PLANE + (row * CH + (c ^ swz(row))) * 16);
  }
  // Dim 32 t + lane % 32, rows 16 k + 4 (lane / 32) + 0 .. 3 and the same + 8: the
  // rows that a lane's accumulator values 8 k .. 8 k + 7 belong to.
  __device__ static __forceinline__ h8 cols(const char* S, int pl, int k, int t, int lane) {
    const int j = lane & 15, d = 32 * t + (lane & 16) + 4 * (j & 3);
    h4 v[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = 16 * k + 8 * e + 4 * (lane >> 5) + (j >> 2);
      const s4v w = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s4v*)(S + pl * PLANE + (row * CH + ((d >> 3) ^ swz(row))) * 16 + (d & 7) * 2));
      v[e] = __builtin_bit_cast(h4, w);
    }
    return __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// A lane's vector as B operands: dims 16 i + 8 (lane / 32) + 0 .. 7.
template <int DP>
__device__ __forceinline__ void load_vec(const char* p, int half, h8 (&h)[DP / 16], h8 (&l)[DP / 16]) {
#pragma unroll
  for (int i = 0; i < DP / 16; ++i) {
    h[i] = *reinterpret_cast<const h8*>(p + i * 32 + half * 16);
    l[i] = *reinterpret_cast<const h8*>(p + DP * 2 + i * 32 + half * 16);
  }
}
// Accumulator values 8 k .. 8 k + 7 as parts.  x is made opaque: where it is a
// product, the compiler would round h from the unrounded product in one place
// and from the float in another, which differ by a step once in some 2^12 values.
__device__ __forceinline__ void split_acc(const f16v& s, int k, h8& h, h8& l) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    f2 x = {s[8 * k + e], s[8 * k + e + 1]};
    asm("" : "+v"(x));
    const h2 hh = __builtin_convertvector(x, h2);
    const f2 r = {__builtin_fmaf(float(hh[0]), -1.f, x[0]), __builtin_fmaf(float(hh[1]), -1.f, x[1])};
    const h2 ll = __builtin_convertvector(r, h2);
    h[e] = hh[0];
    h[e + 1] = hh[1];
    l[e] = ll[0];
    l[e + 1] = ll[1];
  }
}
// The tile's vectors times a lane's: out[e] is row 8 (e / 4) + 4 (lane / 32) + e % 4.
// QUERIES: the tile is the one of queries (or dO), and the small products are added
// in the order in which they are where it is the one of keys, so that all kernels
// have the same score to the last bit.
template <int DP, bool QUERIES = false>
__device__ __forceinline__ f16v scores(const char* S, const h8 (&h)[DP / 16], const h8 (&l)[DP / 16], int col, int half) {
  f16v big, small;
  zero(big);
  zero(small);
#pragma unroll
  for (int i = 0; i < DP / 16; ++i) {
    const h8 th = PTile<DP>::rows(S, 0, col, 2 * i + half), tl = PTile<DP>::rows(S, 1, col, 2 * i + half);
    big = mma(th, h[i], big);
    small = QUERIES ? mma(tl, h[i], small) : mma(th, l[i], small);
    small = QUERIES ? mma(th, l[i], small) : mma(tl, h[i], small);
  }
  return big + small;
}
// acc += (tile transposed) (parts of s).
template <int DP>
__device__ __forceinline__ void add_cols(const char* S, const f16v& s, f16v (&acc)[DP / 32], int lane) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    h8 h, l;
    split_acc(s, k, h, l);
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) {
      const h8 th = PTile<DP>::cols(S, 0, k, t, lane), tl = PTile<DP>::cols(S, 1, k, t, lane);
      acc[t] = mma(th, h, acc[t]);
      acc[t] = mma(th, l, acc[t]);
      acc[t] = mma(tl, h, acc[t]);
    }
  }
}
template <int N>
__device__ __forceinline__ void scale_acc(f16v (&acc)[N], float by) {
#pragma unroll
  for (int t = 0; t < N; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[t][i] *= by;
}
// A lane's vector from its accumulators: dims 32 t + 8 q + 4 half + 0 .. 3.
template <int DP, bool VEC>
__device__ __forceinline__ void write_vec(float* p, uint32_t D, int half, const f16v (&acc)[DP / 32], float by, float by2) {
#pragma unroll
  for (int t = 0; t < DP / 32; ++t)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t d = 32 * t + 8 * q + 4 * half;
      f4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = acc[t][4 * q + e] * by * by2;
      if constexpr (VEC) {
        if (d < D) *reinterpret_cast<f4*>(p + d) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d + e < D) p[d + e] = v[e];
      }
    }
}

// ---------------------------------------------------------------------------
// Forward: 128 query rows per workgroup, 32 per wave, in registers.  2 x 4096
// tokens, 16 heads of 128, causal: 442-450 us, 306-311 TFLOP/s of fp32 products; the
// MFMAs are busy 46 % of a clock that power holds at 1.95 GHz.
// ---------------------------------------------------------------------------
template <int DP, bool VEC>
__global__ void __launch_bounds__(kT, 2) k_attn_fwd_parts(const Attn a, const Parts ps) {
  using TL = PTile<DP>;
  __shared__ __attribute__((aligned(16))) char Ks[TL::BYTES], Vs[TL::BYTES];
  const uint32_t prob = a.B * a.G, rest = blockIdx.x / prob, pr = blockIdx.x - rest * prob;
  const uint32_t back = rest / a.splits, sp = rest - back * a.splits, tile = a.tiles - 1 - back;
  if (unsuited<false>(a, ps, pr)) {
    for (uint32_t n = tile * 128; n < min(tile * 128 + 128, a.N); n += 64)
      fwd_fp32<DP, VEC>(a, pr, n, sp, reinterpret_cast<float*>(Ks), reinterpret_cast<float*>(Vs));
    return;
  }
  const uint32_t b = fdiv(pr, a.dG), gh = pr - b * a.G;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, half = lane >> 5;
  const uint32_t n0 = tile * 128, n = n0 + wave * 32 + col, len = keys_of(a, b);
  const uint32_t least = limit_of(a, n0, len), most = limit_of(a, min(n0 + 128, a.N) - 1, len);
  const uint32_t lim = n < a.N ? limit_of(a, n, len) : 0u, mine = wave_limit(a, n0 + wave * 32, kRows, len);
  h8 qh[DP / 16], ql[DP / 16];
  load_vec<DP>(ps.q.p + (size_t(pr) * ps.q.pad + n) * (DP * 4), half, qh, ql);
  const float cq = a.c * pow2(-ps.q.e[size_t(pr) * (ps.q.pad / kRows) + n0 / kRows + wave]);
  const int* ek = ps.k.e + size_t(pr) * (ps.k.pad / kRows);
  const int* ev = ps.v.e + size_t(pr) * (ps.v.pad / kRows);
  const char* kp = ps.k.p + size_t(pr) * ps.k.pad * (DP * 4);
  const char* vp = ps.v.p + size_t(pr) * ps.v.pad * (DP * 4);
  f16v o[DP / 32];
#pragma unroll
  for (int t = 0; t < DP / 32; ++t) zero(o[t]);
  // o and l count in units of 2^C, a row's own: P's parts are 2^(s - C - e), which
  // the exponential's offset brings in
  float C = -3e38f, l = 0.f, most_s = -INFINITY;
  const uint32_t j0 = sp * a.perSplit * kRows, j1 = min(most, (sp + 1) * a.perSplit * kRows);
  u4v rk[TL::LOADS], rv[TL::LOADS];
  auto fetch = [&](uint32_t j) {
    TL::load(kp + size_t(j) * (DP * 4), rk);
    TL::load(vp + size_t(j) * (DP * 4), rv);
  };
  if (j0 < j1) fetch(j0);
  for (uint32_t j = j0; j < j1; j += kRows) {
    __syncthreads();
    TL::store(Ks, rk);
    TL::store(Vs, rv);
    __syncthreads();
    if (j + kRows < j1) fetch(j + kRows);
    if (j >= mine) continue;
    const float cs = cq * pow2(-ek[j / kRows]);
    const int e = ev[j / kRows];
    f16v s = scores<DP>(Ks, qh, ql, col, half);
    float top = -INFINITY;
    if (j + kRows > least) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t key = j + 8 * (i >> 2) + 4 * half + (i & 3);
        s[i] = key < lim ? scaled(s[i], cs) : -INFINITY;
        top = fmaxf(top, s[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = scaled(s[i], cs);
        top = fmaxf(top, s[i]);
      }
    }
    top = fmaxf(top, __shfl_xor(top, 32));
    most_s = fmaxf(most_s, top);
    float off = C + float(e);
    const bool full = top - off >= float(kFull);
    if (__any(full)) {
      const float next = full ? floorf(top) - float(kTop + e) : C;
      const float down = pow2(int(fmaxf(C - next, -126.f)));
      l *= down;
      scale_acc(o, down);
      C = next;
      off = C + float(e);
    }
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = exp2_(s[i] - off);
      sum += s[i];
    }
    l += sum * pow2(e);
    add_cols<DP>(Vs, s, o, lane);
  }
  l += __shfl_xor(l, 32);
  if (n >= a.N) return;
  // The statistics are relative to the largest score.
  const float up = most_s == -INFINITY ? 1.f : exp2_(C - most_s);
  if (a.splits > 1) {
    const size_t row = (size_t(sp) * a.B * a.G + pr) * a.N + n;
    if (half == 0) {
      a.pm[row] = most_s;
      a.pl[row] = l * up;
    }
    write_vec<DP, VEC>(a.po + row * a.D, a.D, half, o, up, 1.f);
    return;
  }
  if (a.m && half == 0) {
    a.m[size_t(pr) * a.N + n] = lim ? most_s : 0.f;
    a.il[size_t(pr) * a.N + n] = lim ? 1.f / (l * up) : 0.f;
  }
  write_vec<DP, VEC>(a.o + q_at(a, b, gh, n), a.D, half, o, lim ? 1.f / l : 0.f, 1.f);  // a row that sees nothing: zeros
}

// ---------------------------------------------------------------------------
// The backward kernels: eight waves, in pairs of one 32-vector block each.  The
// first of a pair computes P = exp(S - m) and leaves it in LDS; the second, a
// tile behind it, dP and dS.  Each holds only its own operand and sums, half of
// what one wave would need (over 256 registers at 128 dims, one wave per SIMD:
// 1400 and 784 us for dK, dV and dQ of 2 x 4096 tokens, 16 heads of 128), and a
// SIMD, which has one of each, multiplies for one while the other is at its
// exponentials.  Three LDS stages, one barrier per tile.
// ---------------------------------------------------------------------------
constexpr int kPair = 512;  // threads
constexpr int kStages = 3;

__device__ __forceinline__ void put_p(float* P, int lane, const f16v& s) {
#pragma unroll
  for (int q = 0; q < 4; ++q)
    *reinterpret_cast<f4*>(P + (q * 64 + lane) * 4) = f4{s[4 * q], s[4 * q + 1], s[4 * q + 2], s[4 * q + 3]};
}
__device__ __forceinline__ f4 get_p(const float* P, int lane, int q) {
  return *reinterpret_cast<const f4*>(P + (q * 64 + lane) * 4);
}
// f(t, stage) for t0 <= t <= t1, the stage (t - t0) % kStages a constant: the
// places in LDS are then offsets in the instructions (worked out per tile, they
// were a third of the vector instructions).
template <class F>
__device__ __forceinline__ void each_tile(uint32_t t0, uint32_t t1, F&& f) {
  for (uint32_t t = t0; t <= t1; t += kStages) {
    f(t, std::integral_constant<int, 0>{});
    if (t + 1 <= t1) f(t + 1, std::integral_constant<int, 1>{});
    if (t + 2 <= t1) f(t + 2, std::integral_constant<int, 2>{});
  }
}
// f's terms are f 2^-unit; f becomes what a column's sum adds, which counts in units
// of 2^-A (a lane and the one 32 further on hold a column).  A goes down, and the sum
// with it, where a value would pass 2^kFull or its factor 2^kMost.
template <int N>
__device__ __forceinline__ void fit_column(f16v& f, int unit, int& A, f16v (&acc)[N]) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(f[i]));
  top = fmaxf(top, __shfl_xor(top, 32));
  const int e = int(__float_as_uint(top) >> 23) - 127, room = A - unit;
  const bool full = top > 0.f && (e + room >= kFull || room > kMost);
  if (__any(full)) {
    const int next = full ? min(kTop - e, kMost) + unit : A;
    scale_acc(acc, pow2(next - A));
    A = next;
  }
  const float by = pow2(min(A - unit, kMost));
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] *= by;
}

// ---------------------------------------------------------------------------
// dQ (2 x 4096 tokens, 16 heads of 128, causal: 656-683 us, 302-314 TFLOP/s in three
// products): 128 query rows per workgroup; Q in the first waves' registers, dO' and the
// sums in the second ones'.  A row's exponent costs 2 % of a training pass.
// ---------------------------------------------------------------------------
template <int DP, bool VEC>
__global__ void __launch_bounds__(kPair, 2) k_attn_dq_parts(const Attn a, const Parts ps) {
  using TL = PTile<DP, kPair>;
  __shared__ __attribute__((aligned(16))) char Ks[kStages][TL::BYTES], Vs[kStages][TL::BYTES];
  __shared__ __attribute__((aligned(16))) float Ps[2][4][1024];
  const uint32_t prob = a.B * a.G, rest = blockIdx.x / prob, pr = blockIdx.x - rest * prob;
  const uint32_t back = rest / a.splits, sp = rest - back * a.splits, tile = a.tiles - 1 - back;
  if (unsuited<true>(a, ps, pr))
    return dq_fp32<DP, VEC, kPair>(a, pr, tile * 128, sp, reinterpret_cast<float*>(Ks[0]),
                                      reinterpret_cast<float*>(Vs[0]));
  const uint32_t b = fdiv(pr, a.dG), gh = pr - b * a.G;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, blk = wave & 3, col = lane & 31, half = lane >> 5;
  const bool first = __builtin_amdgcn_readfirstlane(wave) < 4;
  const uint32_t n0 = tile * 128, n = n0 + blk * 32 + col, len = keys_of(a, b);
  const uint32_t least = limit_of(a, n0, len), most = limit_of(a, min(n0 + 128, a.N) - 1, len);
  const uint32_t lim = n < a.N ? limit_of(a, n, len) : 0u, mine = wave_limit(a, n0 + blk * 32, kRows, len);
  const size_t row = size_t(pr) * ps.q.pad + n;
  const size_t et = size_t(pr) * (ps.q.pad / kRows) + n0 / kRows + blk;
  const int* ek = ps.k.e + size_t(pr) * (ps.k.pad / kRows);
  const int* ev = ps.v.e + size_t(pr) * (ps.v.pad / kRows);
  const char* kp = ps.k.p + size_t(pr) * ps.k.pad * (DP * 4);
  const char* vp = ps.v.p + size_t(pr) * ps.v.pad * (DP * 4);
  uint32_t j0, j1;
  split_keys(a, most, sp, j0, j1);
  const uint32_t t0 = j0 / kRows, t1 = max(t0, (j1 + kRows - 1) / kRows);
  u4v rk[TL::LOADS], rv[TL::LOADS];
  auto fetch = [&](uint32_t t) {
    TL::load(kp + size_t(t) * kRows * (DP * 4), rk);
    TL::load(vp + size_t(t) * kRows * (DP * 4), rv);
  };
  auto stage = [&](uint32_t t, auto place) {  // tile t from the registers, which then take t + 1
    if (t >= t1) return;
    TL::store(Ks[place], rk);
    TL::store(Vs[place], rv);
    if (t + 1 < t1) fetch(t + 1);
  };
  if (t0 < t1) fetch(t0);
  stage(t0, std::integral_constant<int, 0>{});
  __syncthreads();
  h8 xh[DP / 16], xl[DP / 16];
  if (first) {
    load_vec<DP>(ps.q.p + row * (DP * 4), half, xh, xl);
    const float cq = a.c * pow2(-ps.q.e[et]), m = n < a.N ? a.m[size_t(pr) * a.N + n] : 0.f;
    each_tile(t0, t1, [&](uint32_t t, auto st) {
      stage(t + 1, std::integral_constant<int, (st + 1) % kStages>{});
      const uint32_t j = t * kRows;
      if (t < t1 && j < mine) {
        const float cs = cq * pow2(-ek[t]);
        f16v s = scores<DP>(Ks[st], xh, xl, col, half);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = exp2_(scaled(s[i], cs) - m);
        if (j + kRows > least) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (j + 8 * (i >> 2) + 4 * half + (i & 3) >= lim) s[i] = 0.f;
        }
        put_p(Ps[t & 1][blk], lane, s);
      }
      __syncthreads();
    });
    return;
  }
  load_vec<DP>(ps.y.p + row * (DP * 4), half, xh, xl);
  const float delta = ps.dl[row];
  const int ey = ps.y.e[et];
  f16v dq[DP / 32];
#pragma unroll
  for (int t = 0; t < DP / 32; ++t) zero(dq[t]);
  int A = kNone;  // dq counts in units of 2^-A, a row's own
  each_tile(t0, t1, [&](uint32_t t, auto st) {
    stage(t + 1, std::integral_constant<int, (st + 1) % kStages>{});
    const uint32_t u = t - 1;  // the tile before the first waves'
    constexpr int su = (st + kStages - 1) % kStages;
    if (t > t0 && u * kRows < mine) {
      const int xk = ek[u], xv = ev[u];
      f16v dp = scores<DP>(Vs[su], xh, xl, col, half);
      const float dl = delta * pow2(xv);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f4 p = get_p(Ps[u & 1][blk], lane, q);
#pragma unroll
        for (int e = 0; e < 4; ++e) dp[4 * q + e] = p[e] * (dp[4 * q + e] - dl);
      }
      fit_column(dp, xk + xv + ey, A, dq);
      add_cols<DP>(Ks[su], dp, dq, lane);
    }
    __syncthreads();
  });
  if (n >= a.N) return;
  // 2^-A in two factors that stay in range
  write_vec<DP, VEC>(a.dq + dq_part(a, sp) + q_at(a, b, gh, n), a.D, half, dq, pow2(-(A / 2)) * a.scale,
                     pow2(A / 2 - A));
}

// ---------------------------------------------------------------------------
// dK, dV (likewise: 817-838 us, 328-336 TFLOP/s in four): 128 keys per workgroup; K
// and dV's sums in the first waves' registers, V and dK's in the second ones'; tiles
// of query rows of every head that shares the keys through LDS.
// ---------------------------------------------------------------------------
template <int DP, bool VEC>
__global__ void __launch_bounds__(kPair, 2) k_attn_dkv_parts(const Attn a, const Parts ps) {
  using TL = PTile<DP, kPair>;
  __shared__ __attribute__((aligned(16))) char Qs[kStages][TL::BYTES], Ys[kStages][TL::BYTES];
  __shared__ __attribute__((aligned(16))) float Ps[2][4][1024];
  __shared__ __attribute__((aligned(16))) float Ms[kStages][kRows], Ds[kStages][kRows];
  __shared__ uint32_t Ls[kStages][kRows];
  __shared__ int Up[2][4][64];  // the exponents of P's columns
  const uint32_t prob = a.B * a.G, rest = blockIdx.x / prob, pr = blockIdx.x - rest * prob;
  const uint32_t tile = rest / a.splits, sp = rest - tile * a.splits;
  if (unsuited<true>(a, ps, pr))
    return dkv_fp32<DP, VEC, kPair>(a, pr, tile * 128, sp, reinterpret_cast<float*>(Qs[0]),
                                    reinterpret_cast<float*>(Ys[0]), Ps[0][0], Ls[0]);
  const uint32_t b = fdiv(pr, a.dG), gh = pr - b * a.G;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, blk = wave & 3, col = lane & 31, half = lane >> 5;
  const bool first = __builtin_amdgcn_readfirstlane(wave) < 4;
  const uint32_t k0 = tile * 128, kw = __builtin_amdgcn_readfirstlane(k0 + blk * 32), key = kw + col;
  const uint32_t len = keys_of(a, b);
  const size_t row = size_t(pr) * ps.k.pad + key, kt = size_t(pr) * (ps.k.pad / kRows) + kw / kRows;
  const int* eq = ps.q.e + size_t(pr) * (ps.q.pad / kRows);
  const int* ey = ps.y.e + size_t(pr) * (ps.q.pad / kRows);
  const char* qp = ps.q.p + size_t(pr) * ps.q.pad * (DP * 4);
  const char* yp = ps.y.p + size_t(pr) * ps.q.pad * (DP * 4);
  uint32_t first_n, end_n;
  split_rows(a, k0, len, sp, first_n, end_n);
  const uint32_t t0 = first_n / kRows, t1 = max(t0, (end_n + kRows - 1) / kRows);
  const size_t part = size_t(sp) * a.B * a.T * a.G * a.D;
  u4v rq[TL::LOADS], ry[TL::LOADS];
  float rm = 0.f, rd = 0.f;
  uint32_t rl = 0;
  auto fetch = [&](uint32_t t) {
    TL::load(qp + size_t(t) * kRows * (DP * 4), rq);
    TL::load(yp + size_t(t) * kRows * (DP * 4), ry);
    if (threadIdx.x < kRows) {
      const uint32_t i = t * kRows + threadIdx.x;
      rm = i < a.N ? a.m[size_t(pr) * a.N + i] : 3e38f;  // P = 0 of rows past the last
      rl = i < a.N ? limit_of(a, i, len) : 0u;
      rd = ps.dl[size_t(pr) * ps.q.pad + i];
    }
  };
  auto stage = [&](uint32_t t, auto s) {  // tile t from the registers, which then take t + 1
    if (t >= t1) return;
    TL::store(Qs[s], rq);
    TL::store(Ys[s], ry);
    if (threadIdx.x < kRows) {
      Ms[s][threadIdx.x] = rm;
      Ds[s][threadIdx.x] = rd;
      Ls[s][threadIdx.x] = rl;
    }
    if (t + 1 < t1) fetch(t + 1);
  };
  if (t0 < t1) fetch(t0);
  stage(t0, std::integral_constant<int, 0>{});
  __syncthreads();
  h8 xh[DP / 16], xl[DP / 16];
  f16v acc[DP / 32];
#pragma unroll
  for (int t = 0; t < DP / 32; ++t) zero(acc[t]);
  int A = kNone;  // dv (second waves: dk) counts in units of 2^-A, a key's own
  if (first) {
    load_vec<DP>(ps.k.p + row * (DP * 4), half, xh, xl);
    const float ck = a.c * pow2(-ps.k.e[kt]);
    each_tile(t0, t1, [&](uint32_t t, auto st) {
      stage(t + 1, std::integral_constant<int, (st + 1) % kStages>{});
      if (t < t1 && wave_limit(a, t * kRows, kRows, len) > kw) {
        const int xy = ey[t];
        const float cs = ck * pow2(-eq[t]);
        f16v s = scores<DP, true>(Qs[st], xh, xl, col, half);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f4 m = *reinterpret_cast<const f4*>(Ms[st] + 8 * q + 4 * half);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[4 * q + e] = scaled(s[4 * q + e], cs) - m[e];
        }
        if (limit_of(a, t * kRows, len) < kw + kRows) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (key >= Ls[st][8 * (i >> 2) + 4 * half + (i & 3)]) s[i] = -INFINITY;
        }
        // As fit_column, on the logarithms
        float top = -kNone;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[i]);
        top = fmaxf(top, __shfl_xor(top, 32));
        const float room = float(A - xy);
        const bool full = top > -kNone / 2 && (top + room >= float(kFull) || room > float(kMost));
        if (__any(full)) {
          const int next = full ? min(kTop - int(floorf(top)), kMost) + xy : A;
          scale_acc(acc, pow2(next - A));
          A = next;
        }
        const int up = min(A - xy, kMost);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = exp2_(s[i] + float(up));
        put_p(Ps[t & 1][blk], lane, s);
        Up[t & 1][blk][lane] = up;
        add_cols<DP>(Ys[st], s, acc, lane);
      }
      __syncthreads();
    });
    if (key >= a.T || !a.dv) return;
    if (key >= len)  // keys past the length get zeros
#pragma unroll
      for (int t = 0; t < DP / 32; ++t) zero(acc[t]);
    write_vec<DP, VEC>(a.dv + part + k_at(a, b, gh, key), a.D, half, acc, pow2(-(A / 2)), pow2(A / 2 - A));
    return;
  }
  load_vec<DP>(ps.v.p + row * (DP * 4), half, xh, xl);
  const int xv = ps.v.e[kt];
  const float vs = pow2(xv);
  each_tile(t0, t1, [&](uint32_t t, auto sn) {
    stage(t + 1, std::integral_constant<int, (sn + 1) % kStages>{});
    const uint32_t u = t - 1;  // the tile before the first waves'
    if (t > t0 && wave_limit(a, u * kRows, kRows, len) > kw) {
      constexpr int st = (sn + kStages - 1) % kStages;
      f16v dp = scores<DP>(Ys[st], xh, xl, col, half);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f4 p = get_p(Ps[u & 1][blk], lane, q);
        const f4 d = *reinterpret_cast<const f4*>(Ds[st] + 8 * q + 4 * half);
#pragma unroll
        for (int e = 0; e < 4; ++e) dp[4 * q + e] = p[e] * (dp[4 * q + e] - d[e] * vs);
      }
      fit_column(dp, eq[u] + ey[u] + xv + Up[u & 1][blk][lane], A, acc);
      add_cols<DP>(Qs[st], dp, acc, lane);
    }
    __syncthreads();
  });
  if (key >= a.T || !a.dk) return;
  if (key >= len)
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) zero(acc[t]);
  write_vec<DP, VEC>(a.dk + part + k_at(a, b, gh, key), a.D, half, acc, pow2(-(A / 2)) * a.scale, pow2(A / 2 - A));
}

struct Places {
  size_t next = 0;
  size_t take(size_t floats) {
    const size_t p = next;
    next += (floats + 63) & ~size_t(63);
    return p;
  }
};

// The parts' places and the pass that fills them.
struct Prep {
  Attn a;
  Parts ps;
  bool bwd;
  size_t extra;   // floats behind the parts
  float* more;    // they
  template <int DP, bool VEC>
  bool run() {
    const uint32_t prob = a.B * a.G;
    const uint32_t nq = (a.N + 127) & ~127u, nk = (a.T + 127) & ~127u;
    Places at;
    const size_t q = at.take(size_t(prob) * nq * DP), qe = at.take(size_t(prob) * (nq / kRows));
    const size_t k = at.take(size_t(prob) * nk * DP), ke = at.take(size_t(prob) * (nk / kRows));
    const size_t v = at.take(size_t(prob) * nk * DP), ve = at.take(size_t(prob) * (nk / kRows));
    const size_t y = bwd ? at.take(size_t(prob) * nq * DP) : 0, ye = bwd ? at.take(size_t(prob) * (nq / kRows)) : 0;
    const size_t dl = bwd ? at.take(size_t(prob) * nq) : 0;
    const size_t ex = at.take(extra);
    float* ws = workspace(at.next);
    if (!ws) return false;
    auto part = [&](size_t p, size_t e, uint32_t pad) {
      return Part{reinterpret_cast<char*>(ws + p), reinterpret_cast<int*>(ws + e), pad};
    };
    ps.q = part(q, qe, nq);
    ps.k = part(k, ke, nk);
    ps.v = part(v, ve, nk);
    ps.y = part(y, ye, nq);
    ps.dl = ws + dl;
    more = ws + ex;
    if (bwd) a.delta = more;
    const uint32_t per = (bwd ? 2 : 1) * (nq / kRows) + 2 * (nk / kRows);
    if (bwd)
      hipLaunchKernelGGL((k_attn_split<DP, VEC, true>), dim3(per * prob), dim3(kT), 0, stream(), a, ps);
    else
      hipLaunchKernelGGL((k_attn_split<DP, VEC, false>), dim3(per * prob), dim3(kT), 0, stream(), a, ps);
    return check_launch("attention (parts)");
  }
};
struct Forward {
  Attn a;
  Parts ps;
  template <int DP, bool VEC>
  bool run() {
    hipLaunchKernelGGL((k_attn_fwd_parts<DP, VEC>), dim3(a.tiles * a.splits * a.B * a.G), dim3(kT), 0, stream(), a, ps);
    return check_launch("AttentionForward (parts)");
  }
};
struct Backward {
  Attn a;
  Parts ps;
  float* more;  // the splits' shares
  template <int DP, bool VEC>
  bool run() {
    const uint32_t prob = a.B * a.G;
    if (a.dq) {
      Attn q = a;
      q.tiles = cdiv(a.N, 128);
      q.splits = key_splits(a, 128);
      if (q.splits > 1) q.dq = more;
      hipLaunchKernelGGL((k_attn_dq_parts<DP, VEC>), dim3(q.tiles * q.splits * prob), dim3(kPair), 0, stream(), q, ps);
      if (q.splits > 1 && !attn_sum(q.dq, a.dq, nullptr, nullptr, size_t(prob) * a.N * a.D, q.splits)) return false;
    }
    if (a.dk || a.dv) {
      const size_t values = size_t(a.B) * a.T * a.G * a.D;
      Attn d = a;
      d.tiles = cdiv(a.T, 128);
      d.splits = row_splits(a, 128);
      if (d.splits > 1) {
        if (a.dk) d.dk = more;
        if (a.dv) d.dv = more + d.splits * values;
      }
      hipLaunchKernelGGL((k_attn_dkv_parts<DP, VEC>), dim3(d.tiles * d.splits * prob), dim3(kPair), 0, stream(), d, ps);
      if (d.splits > 1 && !attn_sum(d.dk, a.dk, d.dv, a.dv, values, d.splits)) return false;
    }
    return check_launch("AttentionBackward (parts)");
  }
};

template <class F>
bool by_dim(uint32_t D, F& f) {
  const bool vec = D % 4 == 0;
#define DCE_D(n) \
  if (D <= n) return vec ? f.template run<n, true>() : f.template run<n, false>();
  DCE_D(32) DCE_D(64) DCE_D(96) DCE_D(128)
#undef DCE_D
  return false;
}

// Parts cost a pass over the operands and its launch, and win the more the more
// keys a row goes over: taken from `least` products of operations and keys on.
// Forward, causal (us on fp32 / on parts): 4 x 512 tokens, 12 heads of 64, 35 / 44;
// 1 x 1024, 8 heads of 64, 38 / 34; 2 x 1024, 54 / 44; 1 x 2048, 4 heads of 128, 99 / 54.
// Backward: 32 x 64 tokens, 8 heads of 64, 20 / 37; 8 x 256 50 / 50; 16 x 197, 6
// heads, 69 / 48; 4 x 512, 8 heads, 90 / 63; 1 x 2048, 4 heads of 128, 410 / 208.
bool worth(const AttnArgs& x, double least) {
  return x.D <= 128 && x.S >= 32 && 4.0 * x.D * x.B * x.H * pairs_of(x) * x.T >= least &&
         uint64_t(x.B) * x.G * (uint64_t(x.H / x.G) * x.S + x.T + 256) < 0x08000000ull;  // threads below 2^32
}

}  // namespace

bool attn_fwd_parts(const AttnArgs& x, Attn a, bool* took) {
  if (!worth(x, 1e12)) return true;
  *took = true;
  const uint32_t prob = a.B * a.G, kt = cdiv(a.T, kRows);
  a.tiles = cdiv(a.N, 128);
  // Two workgroups live on a CU: keys are split to fill both (1 x 3000 tokens, 4
  // heads of 128: 108 us in 576 workgroups, 107 in 192, 86 in 480); from one per CU
  // on by the time of the longest (1 x 8192, 4 heads of 64, causal: 309 us unsplit,
  // 170 split).
  const uint32_t wgs = a.tiles * prob, cus = uint32_t(num_cus());
  a.splits = wgs < cus ? std::max(1u, std::min(cdiv(kt, 8), 2 * cus / wgs))
                       : best_splits(wgs, kt, a.D * 0.015, 4.0 * prob * a.N * (a.D + 2), a.causal);
  a.perSplit = cdiv(kt, a.splits);
  a.splits = cdiv(kt, a.perSplit);
  const size_t rows = size_t(prob) * a.N, stat = (rows * a.splits + 63) & ~size_t(63);
  Prep p{a, {}, false, a.splits > 1 ? 2 * stat + rows * a.splits * a.D : 0, nullptr};
  if (!by_dim(a.D, p)) return false;
  a.pm = p.more;
  a.pl = p.more + stat;
  a.po = p.more + 2 * stat;
  Forward f{a, p.ps};
  if (!by_dim(a.D, f)) return false;
  return a.splits == 1 || attn_join(a);
}

bool attn_bwd_parts(const AttnArgs& x, Attn a, bool* took) {
  if (!worth(x, 1e11)) return true;
  *took = true;
  const size_t rows = (size_t(a.B) * a.G * a.N + 63) & ~size_t(63);
  Prep p{a, {}, true, rows + split_floats(a, 128, 128), nullptr};
  if (!by_dim(a.D, p)) return false;
  a.delta = p.more;
  Backward f{a, p.ps, p.more + rows};
  return by_dim(a.D, f);
}

}  // namespace dce
