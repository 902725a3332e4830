// The attention kernels' device code on fp32 MFMAs, which the kernels of
// dce_attention.hip are made of, and those of dce_attention_parts.hip where a
// problem's values do not suit parts.
#pragma once
#include "dce_attention.h"

namespace dce {

constexpr int kKeys = 32;  // keys (rows in the dK / dV kernel) of an LDS tile

__device__ __forceinline__ f4 mfma4(float a, float b, const f4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
// A 16-lane fragment of vectors: lane group g takes dims 16 j + 4 g .. + 3; zeros
// from D on and where not ok.  p is a vector in any case: the loads are of clamped
// places, for behind a branch each could wait for the one before.
template <int DP, bool VEC>
__device__ __forceinline__ void load_frag(const float* p, bool ok, uint32_t D, int g, f4 (&r)[DP / 16]) {
#pragma unroll
  for (int j = 0; j < DP / 16; ++j) {
    const uint32_t d = 16 * j + 4 * g;
    if constexpr (VEC) {
      r[j] = *reinterpret_cast<const f4*>(p + min(d, D - 4));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) r[j][e] = p[min(d + e, D - 1)];
    }
  }
#pragma unroll
  for (int j = 0; j < DP / 16; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) r[j][e] = ok && 16 * j + 4 * g + e < D ? r[j][e] : 0.f;
}

// A score times c, rounded before the row's maximum is taken off, here and in the
// backward: fused with the subtraction it would miss the (rounded) maximum by the
// product's rounding, which of large scores is a factor of P.  For the same reason
// the kernels multiply the terms of a score in one order.
__device__ __forceinline__ float scaled(float s, float c) {
#pragma clang fp contract(off)
  return s * c;
}

template <int CH>
__device__ __forceinline__ int swz(int row) {
  return CH % 16 == 0 ? row & 15 : (row >> 1) & 7;
}
// An LDS tile of R vectors padded to DP dims, row pitch DP, the 16-byte chunks
// of a row XORed by the row so that a read of one chunk of 16 rows covers the 64
// banks once.  Loaded through registers; rows and dims past the ends read zeros
// (never what memory holds there, which may be NaN).
template <int DP, int R, bool VEC, int NT>
struct Tile {
  static constexpr int CH = DP / 4, SLOTS = R * CH, LOADS = (SLOTS + NT - 1) / NT;
  static constexpr bool WHOLE = SLOTS % NT == 0;  // else the last load is for some threads only
  // NT: streaming, for what is read once and larger than the caches.
  template <bool NTL = false>
  __device__ static __forceinline__ void load(const BRes& b, uint32_t stride, uint32_t D, f4 (&r)[LOADS]) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const uint32_t slot = threadIdx.x + NT * i, row = slot / CH, d = slot % CH * 4, off = row * stride + d;
      if constexpr (VEC) {
        r[i] = NTL ? b.ld4nt(d < D ? off : kOob) : b.ld4(d < D ? off : kOob);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) r[i][e] = b.ld1(d + e < D ? off + e : kOob);
      }
    }
  }
  __device__ static __forceinline__ void store(float* S, const f4 (&r)[LOADS]) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const uint32_t slot = threadIdx.x + NT * i, row = slot / CH, c = slot % CH;
      if (WHOLE || slot < SLOTS) *reinterpret_cast<f4*>(S + (row * CH + (c ^ swz<CH>(row))) * 4) = r[i];
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
// Forward of the 64 query rows from n0 on (16 per wave, in registers): key tiles
// through LDS, the next tile's loads in flight while one is multiplied.  Twice the
// rows, which would reuse each fragment, hold the registers of two waves: 64 x 64
// tokens, 16 heads of 64, 27.7 us against 17.5; 64 x 24 rows over 4096 keys, 64
// heads of 64 on 8, 1195 against 1000.
// ---------------------------------------------------------------------------
template <int DP, bool VEC>
__device__ __forceinline__ void fwd_fp32(const Attn& a, uint32_t pr, uint32_t n0, uint32_t sp, float* Ks, float* Vs) {
  using TL = Tile<DP, kKeys, VEC, 256>;
  using CL = Cols<DP>;
  const uint32_t b = fdiv(pr, a.dG), gh = pr - b * a.G;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const uint32_t len = keys_of(a, b);
  const uint32_t least = limit_of(a, n0, len), most = limit_of(a, min(n0 + 64, a.N) - 1, len);
  const uint32_t mine = wave_limit(a, n0 + wave * 16, 16, len);
  const uint32_t n = n0 + wave * 16 + col, lim = n < a.N ? limit_of(a, n, len) : 0u;

  f4 q[DP / 16], o[DP / 16];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < DP / 16; ++i) o[i] = f4{0.f, 0.f, 0.f, 0.f};
  const uint32_t stride = a.G * a.D;
  const uint32_t j0 = sp * a.perSplit * kKeys, j1 = min(most, (sp + 1) * a.perSplit * kKeys);
  f4 rk[TL::LOADS], rv[TL::LOADS];
  auto fetch = [&](uint32_t j) {
    const uint32_t n = min(len - j, uint32_t(kKeys));
    TL::load(rows_view(a.k + k_at(a, b, gh, j), n, stride, a.D), stride, a.D, rk);
    TL::load(rows_view(a.v + k_at(a, b, gh, j), n, stride, a.D), stride, a.D, rv);
  };
  if (j0 < j1) fetch(j0);
  load_frag<DP, VEC>(a.q + q_at(a, b, gh, min(n, a.N - 1)), true, a.D, g, q);
  for (uint32_t j = j0; j < j1; j += kKeys) {
    __syncthreads();
    TL::store(Ks, rk);
    TL::store(Vs, rv);
    __syncthreads();
    if (j + kKeys < j1) fetch(j + kKeys);
    if (j >= mine) continue;
    // S^T: keys 16 kt + 4 g + r of query `col`
    f4 s[2];
    s[0] = s[1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const f4 kf = TL::chunk(Ks, 16 * kt + col, 4 * i + g);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[kt] = mfma4(kf[e], q[i][e], s[kt]);
      }
    const bool masked = j + kKeys > least;
    float top = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float x = scaled(s[kt][r], a.c);
        if (masked && j + 16 * kt + 4 * g + r >= lim) x = -INFINITY;
        s[kt][r] = x;
        top = fmaxf(top, x);
      }
    top = fmaxf(m, max_g(top));
    const float base = top == -INFINITY ? 0.f : top;  // nothing seen yet: every p is 0
    if (__any(top > m)) {
      const float down = exp2_(m - base);
      l *= down;
#pragma unroll
      for (int i = 0; i < DP / 16; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[i][r] *= down;
      m = top;
    }
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[kt][r] = exp2_(s[kt][r] - base);
        l += s[kt][r];
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
          for (int e = 0; e < CL::EG; ++e) o[p * CL::EG + e] = mfma4(vf[e], s[kt][r], o[p * CL::EG + e]);
        }
  }
  const float sum = sum_g(l);
  if (n >= a.N) return;
  if (a.splits > 1) {
    const size_t row = (size_t(sp) * a.B * a.G + pr) * a.N + n;
    if (g == 0) {
      a.pm[row] = m;
      a.pl[row] = sum;
    }
    CL::template write<VEC>(a.po + row * a.D, a.D, g, o, 1.f);
    return;
  }
  const float il = lim ? 1.f / sum : 0.f;  // a row that sees nothing: zeros
  if (a.m && g == 0) {
    a.m[size_t(pr) * a.N + n] = lim ? m : 0.f;
    a.il[size_t(pr) * a.N + n] = il;
  }
  CL::template write<VEC>(a.o + q_at(a, b, gh, n), a.D, g, o, il);
}

// ---------------------------------------------------------------------------
// dQ of NT / 4 rows: as the forward, dQ^T += K^T dS^T.  Also leaves delta for the
// other kernel.
// ---------------------------------------------------------------------------
template <int DP, bool VEC, int NT>
__device__ __forceinline__ void dq_fp32(const Attn& a, uint32_t pr, uint32_t n0, uint32_t sp, float* Ks, float* Vs) {
  using TL = Tile<DP, kKeys, VEC, NT>;
  using CL = Cols<DP>;
  constexpr uint32_t ROWS = NT / 4;
  const uint32_t b = fdiv(pr, a.dG), gh = pr - b * a.G;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const uint32_t len = keys_of(a, b);
  const uint32_t least = limit_of(a, n0, len), most = limit_of(a, min(n0 + ROWS, a.N) - 1, len);
  const uint32_t mine = wave_limit(a, n0 + wave * 16, 16, len);

  f4 q[DP / 16], dy[DP / 16], o[DP / 16], dq[DP / 16];
  // Rows past the last are computed as it (without a branch, behind which every
  // load would wait for the one before) and not written.
  const uint32_t n = n0 + wave * 16 + col, nn = min(n, a.N - 1), lim = limit_of(a, nn, len);
  const size_t at = q_at(a, b, gh, nn), row = size_t(pr) * a.N + nn;
  const float m = a.m[row], il = a.il[row];
  load_frag<DP, VEC>(a.dy + at, true, a.D, g, dy);
  load_frag<DP, VEC>(a.o + at, true, a.D, g, o);
  load_frag<DP, VEC>(a.q + at, true, a.D, g, q);
  uint32_t j0, j1;
  split_keys(a, most, sp, j0, j1);
  const uint32_t stride = a.G * a.D;
  f4 rk[TL::LOADS], rv[TL::LOADS];
  auto fetch = [&](uint32_t j) {
    const uint32_t n = min(len - j, uint32_t(kKeys));
    TL::load(rows_view(a.k + k_at(a, b, gh, j), n, stride, a.D), stride, a.D, rk);
    TL::load(rows_view(a.v + k_at(a, b, gh, j), n, stride, a.D), stride, a.D, rv);
  };
  if (a.dq && j0 < j1) fetch(j0);
  float d = 0.f;
#pragma unroll
  for (int i = 0; i < DP / 16; ++i) {
#pragma unroll
    for (int e = 0; e < 4; ++e) d += dy[i][e] * o[i][e];
    dq[i] = f4{0.f, 0.f, 0.f, 0.f};
  }
  const float delta = sum_g(d);
  if (n < a.N && g == 0) a.delta[size_t(pr) * a.N + n] = delta;
  if (!a.dq) return;
  for (uint32_t j = j0; j < j1; j += kKeys) {
    __syncthreads();
    TL::store(Ks, rk);
    TL::store(Vs, rv);
    __syncthreads();
    if (j + kKeys < j1) fetch(j + kKeys);
    if (j >= mine) continue;
    f4 s[2], dp[2];
    s[0] = s[1] = dp[0] = dp[1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const f4 kf = TL::chunk(Ks, 16 * kt + col, 4 * i + g);
        const f4 vf = TL::chunk(Vs, 16 * kt + col, 4 * i + g);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[kt] = mfma4(kf[e], q[i][e], s[kt]);
          dp[kt] = mfma4(vf[e], dy[i][e], dp[kt]);
        }
      }
    const bool masked = j + kKeys > least;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float p = exp2_(scaled(s[kt][r], a.c) - m) * il;
        const float ds = p * (dp[kt][r] - delta) * a.scale;
        s[kt][r] = masked && j + 16 * kt + 4 * g + r >= lim ? 0.f : ds;
      }
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int p = 0; p < CL::NG; ++p) {
          const typename CL::V kf = CL::read(Ks, 16 * kt + 4 * g + r, p, col);
#pragma unroll
          for (int e = 0; e < CL::EG; ++e) dq[p * CL::EG + e] = mfma4(kf[e], s[kt][r], dq[p * CL::EG + e]);
        }
  }
  if (n < a.N) CL::template write<VEC>(a.dq + dq_part(a, sp) + q_at(a, b, gh, n), a.D, g, dq, 1.f);
}

// ---------------------------------------------------------------------------
// dK, dV of NT / 4 keys (16 per wave, K and V in registers): tiles of query rows
// of every head that shares them through LDS: the sum over the heads is part of
// the loop, in a fixed order.
// ---------------------------------------------------------------------------
template <int DP, bool VEC, int NT>
__device__ __forceinline__ void dkv_fp32(const Attn& a, uint32_t pr, uint32_t k0, uint32_t sp, float* Qs, float* Ys,
                                         float* St, uint32_t* Lim) {
  using TL = Tile<DP, kKeys, VEC, NT>;
  using CL = Cols<DP>;
  const uint32_t b = fdiv(pr, a.dG), gh = pr - b * a.G;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const uint32_t len = keys_of(a, b), key = k0 + wave * 16 + col;
  const uint32_t kw = __builtin_amdgcn_readfirstlane(k0 + wave * 16);
  f4 kf[DP / 16], vf[DP / 16], dk[DP / 16], dv[DP / 16];
  load_frag<DP, VEC>(a.k + (key < len ? k_at(a, b, gh, key) : 0), key < len, a.D, g, kf);
  load_frag<DP, VEC>(a.v + (key < len ? k_at(a, b, gh, key) : 0), key < len, a.D, g, vf);
#pragma unroll
  for (int i = 0; i < DP / 16; ++i) dk[i] = dv[i] = f4{0.f, 0.f, 0.f, 0.f};
  uint32_t first, end;
  split_rows(a, k0, len, sp, first, end);
  const uint32_t sees = first_row(a, k0);
  const size_t part = size_t(sp) * a.B * a.T * a.G * a.D;
  f4 rq[TL::LOADS], ry[TL::LOADS];
  float st[3] = {0.f, 0.f, 0.f};
  uint32_t lm = 0;
  auto fetch = [&](uint32_t n0) {
    // Row by row: they are not evenly spaced when heads share keys.  Rows that see
    // no key from k0 on read as zeros, whatever they hold.
#pragma unroll
    for (int i = 0; i < TL::LOADS; ++i) {
      const uint32_t slot = threadIdx.x + NT * i, n = n0 + slot / TL::CH, d = slot % TL::CH * 4;
      const size_t at = n < a.N ? q_at(a, b, gh, n) + d : 0;
      rq[i] = ry[i] = f4{0.f, 0.f, 0.f, 0.f};
      if constexpr (VEC) {
        if (n >= sees && n < a.N && d < a.D) {
          rq[i] = *reinterpret_cast<const f4*>(a.q + at);
          ry[i] = *reinterpret_cast<const f4*>(a.dy + at);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n >= sees && n < a.N && d + e < a.D) {
            rq[i][e] = a.q[at + e];
            ry[i][e] = a.dy[at + e];
          }
      }
    }
    if (threadIdx.x < kKeys) {
      const uint32_t n = n0 + threadIdx.x;
      const size_t row = size_t(pr) * a.N + min(n, a.N - 1);
      st[0] = a.m[row];  // of rows past the last, which see nothing: any
      st[1] = a.il[row];
      st[2] = a.delta[row];
      lm = n < a.N ? limit_of(a, n, len) : 0u;
    }
  };
  if (first < end) fetch(first);
  for (uint32_t n0 = first; n0 < end; n0 += kKeys) {
    __syncthreads();
    TL::store(Qs, rq);
    TL::store(Ys, ry);
    if (threadIdx.x < kKeys) {
#pragma unroll
      for (int i = 0; i < 3; ++i) St[i * kKeys + threadIdx.x] = st[i];
      Lim[threadIdx.x] = lm;
    }
    __syncthreads();
    if (n0 + kKeys < end) fetch(n0 + kKeys);
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
        const float p = sees ? exp2_(scaled(s[t][r], a.c) - m[r]) * il[r] : 0.f;
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
    if (a.dk) CL::template write<VEC>(a.dk + part + k_at(a, b, gh, key), a.D, g, dk, 1.f);
    if (a.dv) CL::template write<VEC>(a.dv + part + k_at(a, b, gh, key), a.D, g, dv, 1.f);
  }
}

}  // namespace dce
