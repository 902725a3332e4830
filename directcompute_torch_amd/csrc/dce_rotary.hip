// Rotary positions: pairs of a head's values turned by an angle that grows with
// the token's position.  (a, b) -> (a c - b s, a s + b c) with c, s from the
// position's row of a table; the pairs are (2i, 2i + 1) when interleaved, else
// (i, i + rot / 2).  Values from `rot` on are copied.  The inverse (the
// gradient) turns the other way.
//
// Bound by memory: 8 bytes per value.  A thread keeps its pairs' c and s in
// registers over up to kHeads heads of the token, whose loads are all issued
// before the first store.
#include "dce_internal.h"

#include <algorithm>

namespace dce {

namespace {

constexpr int kT = 256;
constexpr uint32_t kHeads = 4;

struct Rot {
  const float *x, *table, *pos;
  float* y;
  uint32_t S, H, D, rot, rows, units, groups;  // units: threads of a head's vector
  FastDiv dU, dGr, dS;
  float sign;
  uint64_t total;
};

// The table row of token t (row t % S without positions); ~0: outside the
// table, which reads as zeros.
__device__ __forceinline__ uint32_t table_row(const Rot& a, uint32_t t) {
  if (!a.pos) {
    const uint32_t s = t - fdiv(t, a.dS) * a.S;
    return s < a.rows ? s : ~0u;
  }
  const float p = a.pos[t];
  return p >= 0.f && p < float(a.rows) ? uint32_t(p) : ~0u;
}

// Eight values per thread and head: four pairs, or a copy of up to eight.
template <bool INTER, bool NT>
__global__ void __launch_bounds__(kT) k_rotary4(const Rot a) {
  const uint64_t idx = uint64_t(xcd_block_id()) * kT + threadIdx.x;
  if (idx >= a.total) return;
  const uint32_t id = uint32_t(idx), tg = fdiv(id, a.dU), u = id - tg * a.units;
  const uint32_t t = fdiv(tg, a.dGr), h0 = (tg - t * a.groups) * kHeads;
  const uint32_t n = min(kHeads, a.H - h0);
  const float* x = a.x + (size_t(t) * a.H + h0) * a.D;
  float* y = a.y + (size_t(t) * a.H + h0) * a.D;
  const uint32_t turned = a.rot / 8;
  f4 A[kHeads], B[kHeads];
  if (u < turned) {
    const uint32_t i = INTER ? 8 * u : 4 * u, j = INTER ? 8 * u + 4 : 4 * u + a.rot / 2;
    const uint32_t row = table_row(a, t);
    f4 w0 = {0.f, 0.f, 0.f, 0.f}, w1 = w0;
    if (row != ~0u) {
      const f4* w = reinterpret_cast<const f4*>(a.table + size_t(row) * a.rot + 8 * u);
      w0 = w[0];
      w1 = w[1];
    }
    const f4 c = {w0[0], w0[2], w1[0], w1[2]};
    const f4 s = {w0[1] * a.sign, w0[3] * a.sign, w1[1] * a.sign, w1[3] * a.sign};
#pragma unroll
    for (uint32_t h = 0; h < kHeads; ++h)
      if (h < n) {
        A[h] = ld4s<NT>(x + size_t(h) * a.D + i);
        B[h] = ld4s<NT>(x + size_t(h) * a.D + j);
      }
#pragma unroll
    for (uint32_t h = 0; h < kHeads; ++h)
      if (h < n) {
        f4 p = A[h], q = B[h];
        if constexpr (INTER) {
          const f4 a0 = {p[0], p[2], q[0], q[2]}, b0 = {p[1], p[3], q[1], q[3]};
          f4 ya, yb;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            ya[e] = a0[e] * c[e] - b0[e] * s[e];
            yb[e] = a0[e] * s[e] + b0[e] * c[e];
          }
          p = f4{ya[0], yb[0], ya[1], yb[1]};
          q = f4{ya[2], yb[2], ya[3], yb[3]};
        } else {
          const f4 a0 = p, b0 = q;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            p[e] = a0[e] * c[e] - b0[e] * s[e];
            q[e] = a0[e] * s[e] + b0[e] * c[e];
          }
        }
        st4s<NT>(y + size_t(h) * a.D + i, p);
        st4s<NT>(y + size_t(h) * a.D + j, q);
      }
    return;
  }
  const uint32_t i = a.rot + 8 * (u - turned);
  const bool two = i + 4 < a.D;
#pragma unroll
  for (uint32_t h = 0; h < kHeads; ++h)
    if (h < n) {
      A[h] = ld4s<NT>(x + size_t(h) * a.D + i);
      if (two) B[h] = ld4s<NT>(x + size_t(h) * a.D + i + 4);
    }
#pragma unroll
  for (uint32_t h = 0; h < kHeads; ++h)
    if (h < n) {
      st4s<NT>(y + size_t(h) * a.D + i, A[h]);
      if (two) st4s<NT>(y + size_t(h) * a.D + i + 4, B[h]);
    }
}

// Any sizes: a pair, or one copied value, per thread.
template <bool INTER>
__global__ void __launch_bounds__(kT) k_rotary1(const Rot a) {
  const uint64_t idx = uint64_t(xcd_block_id()) * kT + threadIdx.x;
  if (idx >= a.total) return;
  const uint32_t id = uint32_t(idx), th = fdiv(id, a.dU), u = id - th * a.units;
  const uint32_t t = fdiv(th, a.dGr);
  const float* x = a.x + size_t(th) * a.D;
  float* y = a.y + size_t(th) * a.D;
  const uint32_t turned = a.rot / 2;
  if (u >= turned) {
    const uint32_t i = a.rot + (u - turned);
    y[i] = x[i];
    return;
  }
  const uint32_t i = INTER ? 2 * u : u, j = INTER ? 2 * u + 1 : u + turned;
  const uint32_t row = table_row(a, t);
  float c = 0.f, s = 0.f;
  if (row != ~0u) {
    c = a.table[size_t(row) * a.rot + 2 * u];
    s = a.table[size_t(row) * a.rot + 2 * u + 1] * a.sign;
  }
  const float p = x[i], q = x[j];
  y[i] = p * c - q * s;
  y[j] = p * s + q * c;
}

inline uint32_t cdiv(uint64_t a, uint64_t b) { return uint32_t((a + b - 1) / b); }

}  // namespace

bool rotary(const float* x, const float* table, const float* pos, float* y, uint32_t tokens, uint32_t S,
            uint32_t H, uint32_t D, uint32_t rot, uint32_t rows, bool interleaved, bool inverse) {
  Rot a{};
  a.x = x;
  a.table = table;
  a.pos = pos;
  a.y = y;
  a.S = S;
  a.H = H;
  a.D = D;
  a.rot = rot;
  a.rows = rows;
  a.dS = make_fastdiv(S);
  a.sign = inverse ? -1.f : 1.f;
  const double bytes = 8.0 * tokens * H * D;
  ProfScope prof("rotary", 3.0 * tokens * H * rot, bytes);
  const bool quads = rot % 8 == 0 && D % 4 == 0;
  a.groups = quads ? cdiv(H, kHeads) : H;
  a.units = quads ? rot / 8 + cdiv(D - rot, 8) : rot / 2 + (D - rot);
  a.dU = make_fastdiv(a.units);
  a.dGr = make_fastdiv(a.groups);
  a.total = uint64_t(tokens) * a.groups * a.units;
  if (a.total >= 0x80000000ull) {
    set_error("RotaryApply: %u tokens of %u heads of %u values are too many for one call", tokens, H, D);
    return false;
  }
  const dim3 grid(cdiv(a.total, kT)), block(kT);
  const bool nt = stream_nt(bytes);
#define DCE_ROT(I, N) hipLaunchKernelGGL((k_rotary4<I, N>), grid, block, 0, stream(), a)
  if (!quads) {
    if (interleaved)
      hipLaunchKernelGGL(k_rotary1<true>, grid, block, 0, stream(), a);
    else
      hipLaunchKernelGGL(k_rotary1<false>, grid, block, 0, stream(), a);
  } else if (interleaved) {
    if (nt) DCE_ROT(true, true); else DCE_ROT(true, false);
  } else {
    if (nt) DCE_ROT(false, true); else DCE_ROT(false, false);
  }
#undef DCE_ROT
  return check_launch("RotaryApply");
}

}  // namespace dce
