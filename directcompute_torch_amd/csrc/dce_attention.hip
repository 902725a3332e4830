// Attention: O = softmax(scale * Q K^T + mask) V and its gradients, without a
// matrix of scores in memory.
//
// Query i sees the keys below min(length, i + T - S + 1) when causal, else below
// length.
//
// Forward, per row, over tiles of keys with a running maximum m and sum l:
//   s_j = c q.k_j (c = scale * log2 e),  p_j = 2^(s_j - m),  l = sum p_j,
//   o = sum p_j v_j / l;   m and 1/l are kept for the backward.
// Backward, P computed again from m and 1/l:
//   dV = P^T dO,  dP = dO V^T,  delta = rowsum(dO * O),
//   dS = scale * P * (dP - delta),  dQ = dS K,  dK = dS^T Q.
//
// Every product runs on fp32 MFMAs (16 x 16 x 4).  Scores are computed
// transposed where queries stay in registers (S^T = K Q^T: a lane then holds
// four keys of one query) and as S = Q K^T where keys stay (four queries of one
// key); either way the accumulator's layout is that of the next product's B
// operand, so P goes from the exponential into the next MFMA without moving
// between lanes.  The order of a dot product's terms is free, so the K / Q
// fragments are read as 16 bytes (dims 16 j + 4 g + e feed step e of lane group
// g), and the transposed operands as up to 16 bytes too (row m of block e is
// dim 16 EG q + EG m + e).
#include "dce_attention.h"

namespace dce {

namespace {

constexpr int kT = 256;   // threads: four waves
constexpr int kKeys = 32; // keys (rows in the dK / dV kernel) of an LDS tile
constexpr int kFew = 64;  // and in the kernel for few rows

__device__ __forceinline__ f4 mfma4(float a, float b, const f4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
// A 16-lane fragment of vectors: lane group g takes dims 16 j + 4 g .. + 3.
template <int DP, bool VEC>
__device__ __forceinline__ void load_frag(const float* p, bool ok, uint32_t D, int g, f4 (&r)[DP / 16]) {
#pragma unroll
  for (int j = 0; j < DP / 16; ++j) {
    const uint32_t d = 16 * j + 4 * g;
    r[j] = f4{0.f, 0.f, 0.f, 0.f};
    if constexpr (VEC) {
      if (ok && d < D) r[j] = *reinterpret_cast<const f4*>(p + d);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (ok && d + e < D) r[j][e] = p[d + e];
    }
  }
}

template <int CH>
__device__ __forceinline__ int swz(int row) {
  return CH % 16 == 0 ? row & 15 : (row >> 1) & 7;
}
// An LDS tile of R vectors padded to DP dims, row pitch DP, the 16-byte chunks
// of a row XORed by the row so that a read of one chunk of 16 rows covers the 64
// banks once.  Loaded through registers; rows and dims past the ends read zeros
// (never what memory holds there, which may be NaN).
template <int DP, int R, bool VEC>
struct Tile {
  static constexpr int CH = DP / 4, LOADS = R * CH / kT;
  static_assert(R * CH % kT == 0, "whole slots");
  __device__ static __forceinline__ void load(const BRes& b, uint32_t stride, uint32_t D, f4 (&r)[LOADS]) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const uint32_t slot = threadIdx.x + kT * i, row = slot / CH, d = slot % CH * 4, off = row * stride + d;
      if constexpr (VEC) {
        r[i] = b.ld4(d < D ? off : kOob);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) r[i][e] = b.ld1(d + e < D ? off + e : kOob);
      }
    }
  }
  __device__ static __forceinline__ void store(float* S, const f4 (&r)[LOADS]) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const uint32_t slot = threadIdx.x + kT * i, row = slot / CH, c = slot % CH;
      *reinterpret_cast<f4*>(S + (row * CH + (c ^ swz<CH>(row))) * 4) = r[i];
    }
  }
  // Dims 4 c .. + 3 of a row.
  __device__ static __forceinline__ f4 chunk(const float* S, int row, int c) {
    return *reinterpret_cast<const f4*>(S + (row * CH + (c ^ swz<CH>(row))) * 4);
  }
};
// Blocks of a transposed operand read at once: 16 EG dims, lane m's are EG m .. + EG - 1.
template <int DP>
struct Cols {
  static constexpr int EG = DP % 64 == 0 ? 4 : 2, NG = DP / 16 / EG;
  typedef float V __attribute__((ext_vector_type(EG)));
  __device__ static __forceinline__ V read(const float* S, int row, int q, int m) {
    constexpr int CH = DP / 4;
    const int d = 16 * EG * q + EG * m;
    return *reinterpret_cast<const V*>(S + (row * CH + ((d >> 2) ^ swz<CH>(row))) * 4 + (d & 3));
  }
  // acc blocks of one vector (a lane's column): dims 16 EG q + EG (4 g + r) + e.
  template <bool VEC>
  __device__ static __forceinline__ void write(float* p, uint32_t D, int g, const f4 (&acc)[DP / 16], float by) {
#pragma unroll
    for (int q = 0; q < NG; ++q)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t d = 16 * EG * q + EG * (4 * g + r);
        V v;
#pragma unroll
        for (int e = 0; e < EG; ++e) v[e] = acc[q * EG + e][r] * by;
        if constexpr (VEC) {
          if (d < D) *reinterpret_cast<V*>(p + d) = v;
        } else {
#pragma unroll
          for (int e = 0; e < EG; ++e)
            if (d + e < D) p[d + e] = v[e];
        }
      }
  }
};

// Sum / maximum over the four lane groups that share a column.
__device__ __forceinline__ float sum_g(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}
__device__ __forceinline__ float max_g(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}

// The buffer view of `n` vectors from p on, `stride` floats apart.
__device__ __forceinline__ BRes rows_view(const float* p, uint32_t n, uint32_t stride, uint32_t D) {
  BRes b;
  b.init(p, n ? (n - 1) * stride + D : 0u);
  return b;
}

// ---------------------------------------------------------------------------
// Forward: 64 QT query rows per workgroup (16 QT per wave, in registers), key
// tiles through LDS, the next tile's loads in flight while one is multiplied.
// ---------------------------------------------------------------------------
template <int DP, int QT, bool VEC>
__global__ void __launch_bounds__(kT) k_attn_fwd(const Attn a) {
  using TL = Tile<DP, kKeys, VEC>;
  using CL = Cols<DP>;
  __shared__ __attribute__((aligned(16))) float Ks[kKeys * DP], Vs[kKeys * DP];
  const uint32_t prob = a.B * a.G, rest = blockIdx.x / prob, pr = blockIdx.x - rest * prob;
  const uint32_t back = rest / a.splits, sp = rest - back * a.splits, tile = a.tiles - 1 - back;
  if (a.only && !a.only[pr]) return;
  const uint32_t b = fdiv(pr, a.dG), gh = pr - b * a.G;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const uint32_t n0 = tile * 64 * QT, len = keys_of(a, b);
  const uint32_t least = limit_of(a, n0, len), most = limit_of(a, min(n0 + 64 * QT, a.N) - 1, len);
  const uint32_t mine = wave_limit(a, n0 + wave * 16 * QT, 16 * QT, len);

  f4 q[QT][DP / 16];
  uint32_t lim[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const uint32_t n = n0 + (wave * QT + t) * 16 + col;
    lim[t] = n < a.N ? limit_of(a, n, len) : 0u;
    load_frag<DP, VEC>(a.q + (n < a.N ? q_at(a, b, gh, n) : 0), n < a.N, a.D, g, q[t]);
  }
  f4 o[QT][DP / 16];
  float m[QT], l[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    m[t] = -INFINITY;
    l[t] = 0.f;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) o[t][i] = f4{0.f, 0.f, 0.f, 0.f};
  }
  const uint32_t stride = a.G * a.D;
  const uint32_t j0 = sp * a.perSplit * kKeys, j1 = min(most, (sp + 1) * a.perSplit * kKeys);
  f4 rk[TL::LOADS], rv[TL::LOADS];
  auto fetch = [&](uint32_t j) {
    const uint32_t n = min(len - j, uint32_t(kKeys));
    TL::load(rows_view(a.k + k_at(a, b, gh, j), n, stride, a.D), stride, a.D, rk);
    TL::load(rows_view(a.v + k_at(a, b, gh, j), n, stride, a.D), stride, a.D, rv);
  };
  if (j0 < j1) fetch(j0);
  for (uint32_t j = j0; j < j1; j += kKeys) {
    __syncthreads();
    TL::store(Ks, rk);
    TL::store(Vs, rv);
    __syncthreads();
    if (j + kKeys < j1) fetch(j + kKeys);
    if (j >= mine) continue;
    // S^T: keys 16 kt + 4 g + r of query `col`
    f4 s[QT][2];
#pragma unroll
    for (int t = 0; t < QT; ++t) s[t][0] = s[t][1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const f4 kf = TL::chunk(Ks, 16 * kt + col, 4 * i + g);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int t = 0; t < QT; ++t) s[t][kt] = mfma4(kf[e], q[t][i][e], s[t][kt]);
      }
    const bool masked = j + kKeys > least;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      float top = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float x = s[t][kt][r] * a.c;
          if (masked && j + 16 * kt + 4 * g + r >= lim[t]) x = -INFINITY;
          s[t][kt][r] = x;
          top = fmaxf(top, x);
        }
      top = fmaxf(m[t], max_g(top));
      const float base = top == -INFINITY ? 0.f : top;  // nothing seen yet: every p is 0
      if (__any(top > m[t])) {
        const float down = exp2_(m[t] - base);
        l[t] *= down;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[t][i][r] *= down;
        m[t] = top;
      }
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[t][kt][r] = exp2_(s[t][kt][r] - base);
          l[t] += s[t][kt][r];
        }
    }
    // O^T += V^T P^T
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int p = 0; p < CL::NG; ++p) {
          const typename CL::V vf = CL::read(Vs, 16 * kt + 4 * g + r, p, col);
#pragma unroll
          for (int e = 0; e < CL::EG; ++e)
#pragma unroll
            for (int t = 0; t < QT; ++t)
              o[t][p * CL::EG + e] = mfma4(vf[e], s[t][kt][r], o[t][p * CL::EG + e]);
        }
  }
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const uint32_t n = n0 + (wave * QT + t) * 16 + col;
    const float sum = sum_g(l[t]);
    if (n >= a.N) continue;
    if (a.splits > 1) {
      const size_t row = (size_t(sp) * a.B * a.G + pr) * a.N + n;
      if (g == 0) {
        a.pm[row] = m[t];
        a.pl[row] = sum;
      }
      CL::template write<VEC>(a.po + row * a.D, a.D, g, o[t], 1.f);
      continue;
    }
    const float il = lim[t] ? 1.f / sum : 0.f;  // a row that sees nothing: zeros
    if (a.m && g == 0) {
      a.m[size_t(pr) * a.N + n] = lim[t] ? m[t] : 0.f;
      a.il[size_t(pr) * a.N + n] = il;
    }
    CL::template write<VEC>(a.o + q_at(a, b, gh, n), a.D, g, o[t], il);
  }
}

// ---------------------------------------------------------------------------
// Forward of up to 16 rows (a new token or a few, all heads of a key head): bound
// by reading K and V once.  Tiles of 64 keys, 16 to each wave, which keeps sums of
// its own; the four waves' are joined at the end.  In the general kernel one wave
// would multiply for all four: 8 sequences of up to 8191 keys, 8 key heads of 128,
// took 114 us there and take 87 here, at the rate of a large copy.  Operands straight from memory, without LDS, took 155 us: the K
// fragment's 64 bytes of each of 16 rows keep the address unit busy.
// ---------------------------------------------------------------------------
template <int DP, bool VEC>
__global__ void __launch_bounds__(kT, 2) k_attn_few(const Attn a) {
  using CL = Cols<DP>;
  using TL = Tile<DP, kFew, VEC>;
  constexpr int EG = CL::EG, NG = CL::NG, NI = DP / 16;
  __shared__ __attribute__((aligned(16))) float Tiles[2][kFew * DP];
  float* Ks = Tiles[0];
  float* Vs = Tiles[1];
  float (*Os)[16][DP + 4] = reinterpret_cast<float (*)[16][DP + 4]>(Ks);  // after the last tile
  static_assert(4 * 16 * (DP + 4) <= 2 * kFew * DP, "the sums fit the tiles");
  __shared__ float Ms[4][16], Ss[4][16];
  const uint32_t prob = a.B * a.G, sp = blockIdx.x / prob, pr = blockIdx.x - sp * prob;
  const uint32_t b = fdiv(pr, a.dG), gh = pr - b * a.G;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t n = col, len = keys_of(a, b), lim = n < a.N ? limit_of(a, n, len) : 0u;
  const uint32_t least = limit_of(a, 0, len), most = limit_of(a, a.N - 1, len);
  f4 q[NI];
  load_frag<DP, VEC>(a.q + (n < a.N ? q_at(a, b, gh, n) : 0), n < a.N, a.D, g, q);
  f4 o[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) o[i] = f4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  const uint32_t stride = a.G * a.D, j0 = sp * a.perSplit * kFew, j1 = min(most, (sp + 1) * a.perSplit * kFew);
  f4 rk[TL::LOADS], rv[TL::LOADS];
  auto fetch = [&](uint32_t j) {
    const uint32_t n = min(len - j, uint32_t(kFew));
    TL::load(rows_view(a.k + k_at(a, b, gh, j), n, stride, a.D), stride, a.D, rk);
    TL::load(rows_view(a.v + k_at(a, b, gh, j), n, stride, a.D), stride, a.D, rv);
  };
  if (j0 < j1) fetch(j0);
  for (uint32_t j = j0; j < j1; j += kFew) {
    __syncthreads();
    TL::store(Ks, rk);
    TL::store(Vs, rv);
    __syncthreads();
    if (j + kFew < j1) fetch(j + kFew);
    const uint32_t jw = j + wave * 16;
    if (jw >= most) continue;
    f4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const f4 kf = TL::chunk(Ks, wave * 16 + col, 4 * i + g);
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        s0 = mfma4(kf[e], q[i][e], s0);
        s1 = mfma4(kf[e + 1], q[i][e + 1], s1);
      }
    }
    f4 s;
    float top = -INFINITY;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      s[r] = (s0[r] + s1[r]) * a.c;
      if (jw + 16 > least && jw + 4 * g + r >= lim) s[r] = -INFINITY;
      top = fmaxf(top, s[r]);
    }
    top = fmaxf(m, max_g(top));
    const float base = top == -INFINITY ? 0.f : top;
    if (__any(top > m)) {
      const float down = exp2_(m - base);
      l *= down;
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[i][r] *= down;
      m = top;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      s[r] = exp2_(s[r] - base);
      l += s[r];
#pragma unroll
      for (int p = 0; p < NG; ++p) {
        const typename CL::V vf = CL::read(Vs, wave * 16 + 4 * g + r, p, col);
#pragma unroll
        for (int e = 0; e < EG; ++e) o[p * EG + e] = mfma4(vf[e], s[r], o[p * EG + e]);
      }
    }
  }
  __syncthreads();
  l = sum_g(l);
  if (g == 0) {
    Ms[wave][col] = m;
    Ss[wave][col] = l;
  }
#pragma unroll
  for (int p = 0; p < NG; ++p)
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int e = 0; e < EG; ++e) Os[wave][col][16 * EG * p + EG * (4 * g + r) + e] = o[p * EG + e][r];
  __syncthreads();
  const bool one = a.splits == 1;
  for (uint32_t i = threadIdx.x; i < a.N * DP; i += kT) {
    const uint32_t row = i / DP, d = i % DP;
    float top = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, Ms[w][row]);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float by = exp2_(Ms[w][row] - base);
      sum += by * Ss[w][row];
      v += by * Os[w][row][d];
    }
    const size_t at = size_t(pr) * a.N + row, part = size_t(sp) * prob * a.N + at;
    const bool none = limit_of(a, row, len) == 0;
    const float il = none ? 0.f : 1.f / sum;
    if (d == 0 && !one) {
      a.pm[part] = top;
      a.pl[part] = sum;
    }
    if (d == 0 && one && a.m) {
      a.m[at] = none ? 0.f : top;
      a.il[at] = il;
    }
    if (d >= a.D) continue;
    if (one)
      a.o[q_at(a, b, gh, row) + d] = none ? 0.f : v * il;
    else
      a.po[part * a.D + d] = v;
  }
}

// Joins the key splits: a workgroup per row, a thread per value (or several).
__global__ void __launch_bounds__(kT) k_attn_join(const Attn a) {
  const uint32_t row = blockIdx.x, rows = a.B * a.G * a.N;
  const uint32_t pr = row / a.N, n = row - pr * a.N, b = fdiv(pr, a.dG), g = pr - b * a.G;
  const bool none = limit_of(a, n, keys_of(a, b)) == 0;
  float m = -INFINITY;
#pragma unroll 8
  for (uint32_t s = 0; s < a.splits; ++s) m = fmaxf(m, a.pm[size_t(s) * rows + row]);
  const float base = m == -INFINITY ? 0.f : m;
  for (uint32_t d = threadIdx.x; d < a.D; d += blockDim.x) {
    float l = 0.f, o = 0.f;
#pragma unroll 8
    for (uint32_t s = 0; s < a.splits; ++s) {
      const size_t i = size_t(s) * rows + row;
      const float w = exp2_(a.pm[i] - base);
      l += w * a.pl[i];
      o += w * a.po[i * a.D + d];
    }
    const float il = none ? 0.f : 1.f / l;
    if (a.m && d == 0) {
      a.m[row] = none ? 0.f : m;
      a.il[row] = il;
    }
    a.o[q_at(a, b, g, n) + d] = none ? 0.f : o * il;
  }
}

// ---------------------------------------------------------------------------
// dQ: as the forward, dQ^T += K^T dS^T.  Also leaves delta for the other kernel.
// ---------------------------------------------------------------------------
template <int DP, int QT, bool VEC>
__global__ void __launch_bounds__(kT) k_attn_dq(const Attn a) {
  using TL = Tile<DP, kKeys, VEC>;
  using CL = Cols<DP>;
  __shared__ __attribute__((aligned(16))) float Ks[kKeys * DP], Vs[kKeys * DP];
  const uint32_t prob = a.B * a.G, back = blockIdx.x / prob, pr = blockIdx.x - back * prob;
  const uint32_t tile = a.tiles - 1 - back;
  if (a.only && !a.only[pr]) return;
  const uint32_t b = fdiv(pr, a.dG), gh = pr - b * a.G;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const uint32_t n0 = tile * 64 * QT, len = keys_of(a, b);
  const uint32_t least = limit_of(a, n0, len), most = limit_of(a, min(n0 + 64 * QT, a.N) - 1, len);
  const uint32_t mine = wave_limit(a, n0 + wave * 16 * QT, 16 * QT, len);

  f4 q[QT][DP / 16], dy[QT][DP / 16], dq[QT][DP / 16];
  uint32_t lim[QT];
  float m[QT], il[QT], delta[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const uint32_t n = n0 + (wave * QT + t) * 16 + col;
    const bool ok = n < a.N;
    const size_t at = ok ? q_at(a, b, gh, n) : 0, row = size_t(pr) * a.N + n;
    lim[t] = ok ? limit_of(a, n, len) : 0u;
    m[t] = ok ? a.m[row] : 0.f;
    il[t] = ok ? a.il[row] : 0.f;
    load_frag<DP, VEC>(a.dy + at, ok, a.D, g, dy[t]);
    load_frag<DP, VEC>(a.o + at, ok, a.D, g, q[t]);
    float d = 0.f;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) d += dy[t][i][e] * q[t][i][e];
      dq[t][i] = f4{0.f, 0.f, 0.f, 0.f};
    }
    delta[t] = sum_g(d);
    if (ok && g == 0) a.delta[row] = delta[t];
    load_frag<DP, VEC>(a.q + at, ok, a.D, g, q[t]);
  }
  if (!a.dq) return;
  const uint32_t stride = a.G * a.D;
  f4 rk[TL::LOADS], rv[TL::LOADS];
  auto fetch = [&](uint32_t j) {
    const uint32_t n = min(len - j, uint32_t(kKeys));
    TL::load(rows_view(a.k + k_at(a, b, gh, j), n, stride, a.D), stride, a.D, rk);
    TL::load(rows_view(a.v + k_at(a, b, gh, j), n, stride, a.D), stride, a.D, rv);
  };
  if (most) fetch(0);
  for (uint32_t j = 0; j < most; j += kKeys) {
    __syncthreads();
    TL::store(Ks, rk);
    TL::store(Vs, rv);
    __syncthreads();
    if (j + kKeys < most) fetch(j + kKeys);
    if (j >= mine) continue;
    f4 s[QT][2], dp[QT][2];
#pragma unroll
    for (int t = 0; t < QT; ++t)
      s[t][0] = s[t][1] = dp[t][0] = dp[t][1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const f4 kf = TL::chunk(Ks, 16 * kt + col, 4 * i + g);
        const f4 vf = TL::chunk(Vs, 16 * kt + col, 4 * i + g);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int t = 0; t < QT; ++t) {
            s[t][kt] = mfma4(kf[e], q[t][i][e], s[t][kt]);
            dp[t][kt] = mfma4(vf[e], dy[t][i][e], dp[t][kt]);
          }
      }
    const bool masked = j + kKeys > least;
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = exp2_(s[t][kt][r] * a.c - m[t]) * il[t];
          const float ds = p * (dp[t][kt][r] - delta[t]) * a.scale;
          s[t][kt][r] = masked && j + 16 * kt + 4 * g + r >= lim[t] ? 0.f : ds;
        }
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int p = 0; p < CL::NG; ++p) {
          const typename CL::V kf = CL::read(Ks, 16 * kt + 4 * g + r, p, col);
#pragma unroll
          for (int e = 0; e < CL::EG; ++e)
#pragma unroll
            for (int t = 0; t < QT; ++t)
              dq[t][p * CL::EG + e] = mfma4(kf[e], s[t][kt][r], dq[t][p * CL::EG + e]);
        }
  }
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const uint32_t n = n0 + (wave * QT + t) * 16 + col;
    if (n < a.N) CL::template write<VEC>(a.dq + q_at(a, b, gh, n), a.D, g, dq[t], 1.f);
  }
}

// ---------------------------------------------------------------------------
// dK, dV: 64 keys per workgroup (16 per wave, K and V in registers), tiles of
// query rows of every head that shares them through LDS: the sum over the
// heads is part of the loop, in a fixed order.
// ---------------------------------------------------------------------------
template <int DP, bool VEC>
__global__ void __launch_bounds__(kT) k_attn_dkv(const Attn a) {
  using TL = Tile<DP, kKeys, VEC>;
  using CL = Cols<DP>;
  __shared__ __attribute__((aligned(16))) float Qs[kKeys * DP], Ys[kKeys * DP], St[3 * kKeys];
  __shared__ uint32_t Lim[kKeys];
  const uint32_t prob = a.B * a.G, tile = blockIdx.x / prob, pr = blockIdx.x - tile * prob;
  if (a.only && !a.only[pr]) return;
  const uint32_t b = fdiv(pr, a.dG), gh = pr - b * a.G;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const uint32_t k0 = tile * 64, len = keys_of(a, b), key = k0 + wave * 16 + col;
  const uint32_t kw = __builtin_amdgcn_readfirstlane(k0 + wave * 16);
  f4 kf[DP / 16], vf[DP / 16], dk[DP / 16], dv[DP / 16];
  load_frag<DP, VEC>(a.k + (key < len ? k_at(a, b, gh, key) : 0), key < len, a.D, g, kf);
  load_frag<DP, VEC>(a.v + (key < len ? k_at(a, b, gh, key) : 0), key < len, a.D, g, vf);
#pragma unroll
  for (int i = 0; i < DP / 16; ++i) dk[i] = dv[i] = f4{0.f, 0.f, 0.f, 0.f};
  const uint32_t first = k0 < len ? min(first_row(a, k0), a.N) : a.N;
  f4 rq[TL::LOADS], ry[TL::LOADS];
  float st = 0.f;
  uint32_t lm = 0;
  auto fetch = [&](uint32_t n0) {
    // Row slots: consecutive rows are not evenly spaced when heads share keys.
#pragma unroll
    for (int i = 0; i < TL::LOADS; ++i) {
      const uint32_t slot = threadIdx.x + kT * i, n = n0 + slot / TL::CH, d = slot % TL::CH * 4;
      const size_t at = n < a.N ? q_at(a, b, gh, n) + d : 0;
      rq[i] = ry[i] = f4{0.f, 0.f, 0.f, 0.f};
      if constexpr (VEC) {
        if (n < a.N && d < a.D) {
          rq[i] = *reinterpret_cast<const f4*>(a.q + at);
          ry[i] = *reinterpret_cast<const f4*>(a.dy + at);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n < a.N && d + e < a.D) {
            rq[i][e] = a.q[at + e];
            ry[i][e] = a.dy[at + e];
          }
      }
    }
    if (threadIdx.x < 3 * kKeys) {
      const uint32_t w = threadIdx.x / kKeys, n = n0 + threadIdx.x % kKeys;
      const float* src = w == 0 ? a.m : w == 1 ? a.il : a.delta;
      st = n < a.N ? src[size_t(pr) * a.N + n] : 0.f;
      lm = n < a.N ? limit_of(a, n, len) : 0u;
    }
  };
  if (first < a.N) fetch(first);
  for (uint32_t n0 = first; n0 < a.N; n0 += kKeys) {
    __syncthreads();
    TL::store(Qs, rq);
    TL::store(Ys, ry);
    if (threadIdx.x < 3 * kKeys) St[threadIdx.x] = st;
    if (threadIdx.x < kKeys) Lim[threadIdx.x] = lm;
    __syncthreads();
    if (n0 + kKeys < a.N) fetch(n0 + kKeys);
    if (wave_limit(a, n0, kKeys, len) <= kw) continue;
    // S: rows 16 t + 4 g + r of key `col`
    f4 s[2], dp[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) s[t] = dp[t] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const f4 qf = TL::chunk(Qs, 16 * t + col, 4 * i + g);
        const f4 yf = TL::chunk(Ys, 16 * t + col, 4 * i + g);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[t] = mfma4(qf[e], kf[i][e], s[t]);
          dp[t] = mfma4(yf[e], vf[i][e], dp[t]);
        }
      }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const f4 m = *reinterpret_cast<const f4*>(St + 16 * t + 4 * g);
      const f4 il = *reinterpret_cast<const f4*>(St + kKeys + 16 * t + 4 * g);
      const f4 delta = *reinterpret_cast<const f4*>(St + 2 * kKeys + 16 * t + 4 * g);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool sees = key < Lim[16 * t + 4 * g + r];
        const float p = sees ? exp2_(s[t][r] * a.c - m[r]) * il[r] : 0.f;
        s[t][r] = p;
        dp[t][r] = sees ? p * (dp[t][r] - delta[r]) * a.scale : 0.f;
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int p = 0; p < CL::NG; ++p) {
          const typename CL::V yf = CL::read(Ys, 16 * t + 4 * g + r, p, col);
          const typename CL::V qf = CL::read(Qs, 16 * t + 4 * g + r, p, col);
#pragma unroll
          for (int e = 0; e < CL::EG; ++e) {
            dv[p * CL::EG + e] = mfma4(yf[e], s[t][r], dv[p * CL::EG + e]);
            dk[p * CL::EG + e] = mfma4(qf[e], dp[t][r], dk[p * CL::EG + e]);
          }
        }
  }
  if (key < a.T) {  // keys past the length get zeros
    if (a.dk) CL::template write<VEC>(a.dk + k_at(a, b, gh, key), a.D, g, dk, 1.f);
    if (a.dv) CL::template write<VEC>(a.dv + k_at(a, b, gh, key), a.D, g, dv, 1.f);
  }
}

Attn params(const AttnArgs& x) {
  Attn a{};
  a.q = x.q;
  a.k = x.k;
  a.v = x.v;
  a.len = x.len;
  a.o = x.o;
  a.B = x.B;
  a.S = x.S;
  a.T = x.T;
  a.G = x.G;
  a.D = x.D;
  a.rep = x.H / x.G;
  a.N = a.rep * x.S;
  a.dRep = make_fastdiv(a.rep);
  a.dG = make_fastdiv(a.G);
  a.scale = x.scale;
  a.c = float(double(x.scale) * 1.4426950408889634);
  a.causal = x.causal;
  if (x.stats) {
    a.m = x.stats;
    a.il = x.stats + size_t(x.B) * x.G * a.N;
  }
  return a;
}

// The head dims a kernel is built for: the least that holds D.
template <class F>
bool by_dim(uint32_t D, bool vec, F f) {
#define DCE_D(n) \
  if (D <= n) return vec ? f.template run<n, true>() : f.template run<n, false>();
  DCE_D(32) DCE_D(64) DCE_D(96) DCE_D(128) DCE_D(256)
#undef DCE_D
  set_error("attention: a head has at most 256 values (got %u)", D);
  return false;
}

struct FwdRun {
  Attn a;
  template <int DP, bool VEC>
  bool run() {
    constexpr int QT = DP <= 128 ? 2 : 1;
    const uint32_t cus = uint32_t(num_cus()), prob = a.B * a.G;
    const bool few = a.N <= 16 && !a.only;
    const bool wide = QT == 2 && uint64_t(cdiv(a.N, 128)) * prob >= 2 * cus;
    a.tiles = cdiv(a.N, wide ? 128 : 64);
    const uint32_t kt = cdiv(a.T, few ? kFew : kKeys);
    a.splits = 1;
    if (few)
      a.splits = std::max(1u, std::min(cdiv(kt, 4), 4 * cus / prob));
    else if (!a.only && uint64_t(a.tiles) * prob < cus) {
      a.splits = std::min(cdiv(kt, 4), cdiv(4 * cus, a.tiles * prob));
      if (a.splits < 1) a.splits = 1;
    }
    a.perSplit = std::max(1u, cdiv(kt, a.splits));
    a.splits = std::max(1u, cdiv(kt, a.perSplit));
    const size_t rows = size_t(prob) * a.N;
    if (a.splits > 1) {
      const size_t stat = (rows * a.splits + 63) & ~size_t(63);
      float* ws = workspace(2 * stat + rows * a.splits * a.D);
      if (!ws) return false;
      a.pm = ws;
      a.pl = ws + stat;
      a.po = ws + 2 * stat;
    }
    const dim3 grid(a.tiles * a.splits * prob);
    if (few)
      hipLaunchKernelGGL((k_attn_few<DP, VEC>), grid, dim3(kT), 0, stream(), a);
    else if (wide)
      hipLaunchKernelGGL((k_attn_fwd<DP, QT, VEC>), grid, dim3(kT), 0, stream(), a);
    else
      hipLaunchKernelGGL((k_attn_fwd<DP, 1, VEC>), grid, dim3(kT), 0, stream(), a);
    if (!check_launch("AttentionForward")) return false;
    return a.splits == 1 || attn_join(a);
  }
};

struct BwdRun {
  Attn a;
  template <int DP, bool VEC>
  bool run() {
    constexpr int QT = DP <= 64 ? 2 : 1;
    const uint32_t prob = a.B * a.G;
    const bool wide = QT == 2 && uint64_t(cdiv(a.N, 128)) * prob >= 2 * uint32_t(num_cus());
    a.tiles = cdiv(a.N, wide ? 128 : 64);
    if (wide)
      hipLaunchKernelGGL((k_attn_dq<DP, QT, VEC>), dim3(a.tiles * prob), dim3(kT), 0, stream(), a);
    else
      hipLaunchKernelGGL((k_attn_dq<DP, 1, VEC>), dim3(a.tiles * prob), dim3(kT), 0, stream(), a);
    if (!check_launch("AttentionBackward (dQ)")) return false;
    if (!a.dk && !a.dv) return true;
    a.tiles = cdiv(a.T, 64);
    hipLaunchKernelGGL((k_attn_dkv<DP, VEC>), dim3(a.tiles * prob), dim3(kT), 0, stream(), a);
    return check_launch("AttentionBackward (dK, dV)");
  }
};

}  // namespace

bool attn_join(const Attn& a) {
  hipLaunchKernelGGL(k_attn_join, dim3(a.B * a.G * a.N), dim3(std::min(kT, int(a.D + 63) / 64 * 64)), 0, stream(), a);
  return check_launch("AttentionForward (join)");
}
bool attn_fwd_fp32(Attn a) { return by_dim(a.D, a.D % 4 == 0, FwdRun{a}); }
bool attn_bwd_fp32(Attn a) { return by_dim(a.D, a.D % 4 == 0, BwdRun{a}); }

bool attention_forward(const AttnArgs& x) {
  ProfScope prof("attention", 4.0 * x.D * x.B * x.H * pairs_of(x),
                 4.0 * x.D * (2.0 * x.B * x.S * x.H + 2.0 * x.B * x.T * x.G));
  const Attn a = params(x);
  bool took = false;
  return attn_fwd_parts(x, a, &took) && (took || attn_fwd_fp32(a));
}

bool attention_backward(const AttnArgs& x, const float* dy, float* dq, float* dk, float* dv) {
  ProfScope prof("attention_bwd", 10.0 * x.D * x.B * x.H * pairs_of(x),
                 4.0 * x.D * (4.0 * x.B * x.S * x.H + 4.0 * x.B * x.T * x.G));
  Attn a = params(x);
  a.dy = dy;
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  bool took = false;
  if (!attn_bwd_parts(x, a, &took)) return false;
  if (took) return true;
  a.delta = workspace(size_t(x.B) * x.H * x.S);
  return a.delta && attn_bwd_fp32(a);
}

}  // namespace dce
