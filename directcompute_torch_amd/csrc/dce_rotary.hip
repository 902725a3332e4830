// Rotary positions: pairs of a head's values turned by an angle that grows with
// the token's position.  (a, b) -> (a c - b s, a s + b c) with c, s from the
// position's row of a table; the pairs are (2i, 2i + 1) when interleaved, else
// (i, i + rot / 2).  Values from `rot` on are copied.  The inverse (the
// gradient) turns the other way.
//
// Bound by memory: 8 bytes per value.  A wave loads whole vectors of neighbouring
// heads, 16 bytes per lane, contiguous; in the half layout the other value of a
// pair is then another lane's, and comes through the LDS crossbar.  (Loading both
// halves in each lane, whose runs of rot / 2 values start and end inside cache
// lines, ran at 4.7 TB/s over 4 x 4096 tokens of 32 heads of 128, 96 of them
// turned.)
#include "dce_internal.h"

#include <algorithm>

namespace dce {

namespace {

constexpr int kT = 256;
constexpr int kLoads = 4;  // vectors in flight per lane

struct Rot {
  const float *x, *table, *pos;
  float* y;
  uint32_t S, H, D, rot, rows;
  uint32_t units;      // lanes, or threads, of a head's vector
  uint32_t per;        // vectors of a wave's load
  FastDiv dU, dH, dS;
  float sign;
  uint64_t total;      // vectors, or threads
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

// Vectors of D / 4 lanes each, `per` of them to a load of a wave.
template <bool INTER, bool NT>
__global__ void __launch_bounds__(kT) k_rotary4(const Rot a) {
  const uint32_t lane = threadIdx.x & 63, own = fdiv(lane, a.dU), d = (lane - own * a.units) * 4;
  const bool live = own < a.per, turns = live && d < a.rot;
  const uint32_t half = a.rot / 2;
  // The pairs of this lane's values in a table row, and (half layout) the lane
  // of their other values.
  const uint32_t p = INTER ? d / 2 : d < half ? d : d - half;
  const int other = int(d < half ? lane + half / 4 : lane - half / 4) * 4;
  const float sign = INTER || d >= half ? a.sign : -a.sign;
  const uint64_t first = (uint64_t(blockIdx.x) * 4 + (threadIdx.x >> 6)) * (kLoads * a.per) + own;
  f4 x[kLoads], w0[kLoads], w1[kLoads];
#pragma unroll
  for (int k = 0; k < kLoads; ++k) {
    const uint64_t v = first + uint64_t(k) * a.per;
    x[k] = w0[k] = w1[k] = f4{0.f, 0.f, 0.f, 0.f};
    if (!live || v >= a.total) continue;
    x[k] = ld4s<NT>(a.x + v * a.D + d);
    if (!turns) continue;
    const uint32_t row = table_row(a, fdiv(uint32_t(v), a.dH));
    if (row == ~0u) continue;
    const f4* w = reinterpret_cast<const f4*>(a.table + size_t(row) * a.rot + 2 * p);
    w0[k] = w[0];
    if (!INTER) w1[k] = w[1];
  }
#pragma unroll
  for (int k = 0; k < kLoads; ++k) {
    const uint64_t v = first + uint64_t(k) * a.per;
    f4 y;
    if constexpr (INTER) {
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const float c = w0[k][e], s = w0[k][e + 1] * sign;
        y[e] = x[k][e] * c - x[k][e + 1] * s;
        y[e + 1] = x[k][e] * s + x[k][e + 1] * c;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float c = e < 2 ? w0[k][2 * e] : w1[k][2 * e - 4], s = e < 2 ? w0[k][2 * e + 1] : w1[k][2 * e - 3];
        const float o = __builtin_bit_cast(
            float, __builtin_amdgcn_ds_bpermute(other, __builtin_bit_cast(int, float(x[k][e]))));
        y[e] = x[k][e] * c + o * (s * sign);
      }
    }
    if (live && v < a.total) st4s<NT>(a.y + v * a.D + d, turns ? y : x[k]);
  }
}

// Any sizes: a pair, or one copied value, per thread.
template <bool INTER>
__global__ void __launch_bounds__(kT) k_rotary1(const Rot a) {
  const uint64_t idx = uint64_t(xcd_block_id()) * kT + threadIdx.x;
  if (idx >= a.total) return;
  const uint32_t id = uint32_t(idx), th = fdiv(id, a.dU), u = id - th * a.units;
  const uint32_t t = fdiv(th, a.dH);
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
  const uint64_t vectors = uint64_t(tokens) * H;
  // Whole quads of pairs' values, and vectors that fit a wave: 4 x 4096 tokens of 32
  // heads of 128, 96 turned, 83 us (212 pair by pair), interleaved 90 (158); one token
  // or 3 x 1001 the same.  Other widths run pair by pair: 60 of 80 turned 142 us, 2.4 TB/s.
  const bool quads = rot % (interleaved ? 4 : 8) == 0 && D % 4 == 0 && D <= 256;
  a.units = quads ? D / 4 : rot / 2 + (D - rot);
  a.per = 64 / (D / 4 ? D / 4 : 1);
  a.dU = make_fastdiv(a.units);
  a.dH = make_fastdiv(H);
  a.total = quads ? vectors : vectors * a.units;
  if (a.total >= 0x80000000ull) {
    set_error("RotaryApply: %u tokens of %u heads of %u values are too many for one call", tokens, H, D);
    return false;
  }
  const dim3 grid(quads ? cdiv(vectors, 4 * kLoads * a.per) : cdiv(a.total, kT)), block(kT);
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
