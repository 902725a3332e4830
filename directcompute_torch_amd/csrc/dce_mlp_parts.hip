// The gated feed-forward block on fp16 parts: the products of large calls at a
// third of the fp16 MFMA rate, which is 16 times the fp32 one, with fp32's accuracy.
//
// A value x is kept as x 2^e = h + l, two fp16 values rounded to nearest, and
// h h + (h l + l h) stands for a product.  The exponent is one for each row of an
// operand (a token's values, an output's weights), such that its largest value lies
// in [2^14, 2^15): l's half step is then 2^-25, 2^-39 of that, so that values down to
// 2^-15 of their row's largest keep 24 bits.  Rows only: the exponents are the product's
// factors of its rows and columns, and cost its loop nothing.  So a matrix that is
// summed over its rows in one product and over its columns in another is split twice.
//
// The steps, forward:  maxima -> parts of x, Wg, Wu, Wd -> g, u, m and m's maxima
// (one product over Wg and Wu, whose columns lie in turn, 32 by 32, so that a wave has
// g and u of one place) -> parts of m -> y.
// Backward:  maxima -> parts of dy, Wd, x, W -> dm, and from it dg, du, m and their
// maxima -> their parts -> dx, dWg, dWu, dWd.
#include "dce_mlp.h"

namespace dce {

namespace {

constexpr int kT = 256;
constexpr int kTile = 128, kStep = 32;

using h8 = _Float16 __attribute__((ext_vector_type(8)));
using f16v = float __attribute__((ext_vector_type(16)));

inline uint32_t cdiv(uint64_t a, uint64_t b) { return uint32_t((a + b - 1) / b); }
inline uint32_t pad(uint32_t v, uint32_t to) { return (v + to - 1) / to * to; }

// The exponent for a row whose largest value has these bits (sign aside).
__device__ __forceinline__ int exp_of(uint32_t bits) { return bits ? 14 + 127 - int(bits >> 23) : 0; }

// Parts in memory: 8 consecutive values of a row are 8 h, then 8 l (32 bytes).
__device__ __forceinline__ void put8(float* to, const float* x, int e) {
  h8 h, l;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = ldexpf(x[i], e);
    h[i] = _Float16(v);
    l[i] = _Float16(v - float(h[i]));
  }
  h8* p = reinterpret_cast<h8*>(to);
  p[0] = h;
  p[1] = l;
}

__global__ void __launch_bounds__(kT) k_mlp_clear(uint32_t* p, uint32_t n) {
  for (uint32_t i = blockIdx.x * kT + threadIdx.x; i < n; i += gridDim.x * kT) p[i] = 0;
}

// ---------------------------------------------------------------------------
// Maxima and parts of up to six matrices, [rows][pitch] of which rows x cols count.
// ---------------------------------------------------------------------------
struct Job {
  float* src;
  uint32_t rows, cols, pitch;
  uint32_t* rowMax;  // bits of the largest value of each row; null: not wanted
  uint32_t* colMax;  // of each column; at place col, or with columns in turn at lane(col)
  float *straight, *across;          // parts of the rows, of the columns; null: none
  uint32_t sPitch, aPitch, sRows, aRows;  // in values; rows to write (zeros from the matrix's end on)
  int turn;  // -1: no; 0, 1: its columns are those of Wg, Wu in turn
};
constexpr int kJobs = 6;
struct Jobs {
  Job j[kJobs];
  uint32_t start[kJobs + 1];
  uint32_t count;
};
__device__ __forceinline__ int find_job(const Jobs& t, uint32_t blk) {
  int i = 0;
  while (i + 1 < int(t.count) && t.start[i + 1] <= blk) ++i;
  return i;
}
__device__ __forceinline__ uint32_t in_turn(uint32_t c, int turn) {
  return turn < 0 ? c : (c >> 5) * 64 + uint32_t(turn) * 32 + (c & 31);
}
// In a tile of 32 rows and 256 columns for each workgroup.
constexpr uint32_t kMaxRows = 32;
__global__ void __launch_bounds__(kT) k_mlp_max(const Jobs t) {
  const int k = find_job(t, blockIdx.x);
  const Job J = t.j[k];
  const uint32_t id = blockIdx.x - t.start[k], across = (J.cols + kT - 1) / kT;
  const uint32_t r0 = id / across * kMaxRows, c = (id % across) * kT + threadIdx.x;
  const bool in = c < J.cols;
  const float* p = J.src + size_t(r0) * J.pitch + min(c, J.cols - 1);
  uint32_t v[kMaxRows], top = 0;
#pragma unroll
  for (uint32_t i = 0; i < kMaxRows; ++i) v[i] = __float_as_uint(p[size_t(min(i, J.rows - 1 - r0)) * J.pitch]) & 0x7fffffffu;
#pragma unroll
  for (uint32_t i = 0; i < kMaxRows; ++i) top = max(top, v[i]);
  if (J.colMax && in && top) atomicMax(J.colMax + in_turn(c, J.turn), top);
  if (!J.rowMax) return;
#pragma unroll
  for (uint32_t i = 0; i < kMaxRows; ++i) {
    // as floats, which order as their bits do; one that is not finite is infinity here
    const float f = in ? (v[i] > 0x7f800000u ? INFINITY : __uint_as_float(v[i])) : 0.f;
    const uint32_t m = __float_as_uint(wave_reduce(f, OpMaxR()));
    if ((threadIdx.x & 63) == 0 && r0 + i < J.rows && m) atomicMax(J.rowMax + r0 + i, m);
  }
}

// A 64 x 64 tile through LDS.  `straight` may be the matrix itself.
constexpr int kSq = 64, kPitch = 68;
__global__ void __launch_bounds__(kT) k_mlp_split(const Jobs t) {
  __shared__ float S[kSq * kPitch];
  const int k = find_job(t, blockIdx.x);
  const Job J = t.j[k];
  const uint32_t across = max(J.straight ? J.sPitch / (J.turn < 0 ? 1 : 2) : 0u, J.across ? J.aRows / (J.turn < 0 ? 1 : 2) : 0u);
  const uint32_t tc = (across + kSq - 1) / kSq;
  const uint32_t id = blockIdx.x - t.start[k], i0 = id / tc * kSq, j0 = id % tc * kSq;
#pragma unroll
  for (int u = 0; u < kSq * kSq / kT; ++u) {
    const uint32_t s = threadIdx.x + kT * u, r = s / kSq, c = s % kSq;
    const float v = J.src[size_t(min(i0 + r, J.rows - 1)) * J.pitch + min(j0 + c, J.cols - 1)];
    S[r * kPitch + c] = i0 + r < J.rows && j0 + c < J.cols ? v : 0.f;
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kSq * kSq / 8 / kT; ++u) {
    const uint32_t slot = threadIdx.x + kT * u;
    float v[8];
    if (J.straight) {
      const uint32_t r = slot / 8, c = slot % 8 * 8, to = in_turn(j0 + c, J.turn);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = S[r * kPitch + c + e];
      if (i0 + r < J.sRows && to < J.sPitch)
        put8(J.straight + size_t(i0 + r) * J.sPitch + to, v, i0 + r < J.rows ? exp_of(J.rowMax[i0 + r]) : 0);
    }
    if (J.across) {
      const uint32_t c = slot % 64, r = slot / 64 * 8, to = in_turn(j0 + c, J.turn);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = S[(r + e) * kPitch + c];
      if (to < J.aRows && i0 + r < J.aPitch)
        put8(J.across + size_t(to) * J.aPitch + i0 + r, v, j0 + c < J.cols ? exp_of(J.colMax[to]) : 0);
    }
  }
}

// ---------------------------------------------------------------------------
// Products C = P Q^T of parts, both along their rows, in 128 x 128 tiles of four
// waves, 64 x 64 each (2 x 2 blocks of 32 x 32).  The depth goes in steps of 32 through
// two LDS stages, the next one's direct loads in flight while one is multiplied.  A
// stage's rows are eight 16-byte slots, h and l of 8 values in turn, XORed by the row
// so that a read of one slot of 16 rows covers the 64 banks once.  The two small
// products have an accumulator of their own: an MFMA cuts what it adds off at the
// scale of the largest addend, always downwards.
// ---------------------------------------------------------------------------
enum Op { STORE, GATE, GRAD };
struct Prod {
  const float *p, *q;              // parts, padded to whole tiles
  const uint32_t *pMax, *qMax;
  uint32_t tm, tn, depth;          // tiles; values of a row
  uint32_t rows, cols;             // of the result
  float* out;                      // STORE; GATE: m; GRAD: dg, du in turn
  float* out2;                     // STORE with columns in turn: the second matrix; GRAD: m
  uint32_t pitch;                  // of out
  int turn;                        // STORE: columns in turn
  float *g, *u;                    // GATE: kept (null: not); GRAD: read
  uint32_t hidden;                 // their pitch
  uint32_t *rowMax, *colMax, *colMax2;  // GATE: m's rows; GRAD: rows and columns of dg, du; columns of m
};

constexpr int kStageBytes = kTile * kStep * 4;
__device__ __forceinline__ int swz(int row) { return (row >> 1) & 7; }
__device__ __forceinline__ void load_stage(const BRes& b, uint32_t pitchBytes, uint32_t k, char* S) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
  for (int i = 0; i < kStageBytes / 16 / kT; ++i) {
    const uint32_t slot = threadIdx.x + kT * i, row = slot / 8, c = (slot % 8) ^ swz(row);
    b.ld16_lds(row * pitchBytes + k * 4 + c * 16, S + (wave * 64 + i * kT) * 16);
  }
}
__device__ __forceinline__ h8 frag(const char* S, int row, int c) {
  return *reinterpret_cast<const h8*>(S + (row * 8 + (c ^ swz(row))) * 16);
}
__device__ __forceinline__ float max32(float v) {  // over the 32 lanes of a half
  v = group8_reduce(v, OpMaxR());
  v = fmaxf(v, xl::dpp<xl::kRowMirror>(v));
  return fmaxf(v, xl::swz(v));
}
// |v| for a maximum: fmaxf drops NaN, which then counts as infinity.
__device__ __forceinline__ float size_of(float v) { return v == v ? fabsf(v) : INFINITY; }

template <Op OP, MlpAct ACT>
__global__ void __launch_bounds__(kT) __attribute__((amdgpu_waves_per_eu(2))) k_mlp_product(const Prod a) {
  __shared__ __attribute__((aligned(16))) char S[4 * kStageBytes];
  // bands of 8 rows of tiles: what an XCD runs at once reads few rows of either side
  const uint32_t id = xcd_block_id(), band = id / (8 * a.tn), in = id - band * 8 * a.tn, high = min(8u, a.tm - band * 8);
  const uint32_t tj = in / high, ti = band * 8 + (in - tj * high);
  const uint32_t pitch = a.depth * 4;
  BRes bp, bq;
  bp.init(a.p + size_t(ti) * kTile * a.depth, kTile * a.depth);
  bq.init(a.q + size_t(tj) * kTile * a.depth, kTile * a.depth);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  const int col = lane & 31, half = lane >> 5;
  f16v big[2][2], small[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) big[i][j][e] = small[i][j][e] = 0.f;
  load_stage(bp, pitch, 0, S);
  load_stage(bq, pitch, 0, S + kStageBytes);
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  int s = 0;
  for (uint32_t k = 0; k < a.depth; k += kStep, s ^= 1) {
    const char* St = S + s * 2 * kStageBytes;
    // Fragments first: a direct load in flight would make the compiler wait for it
    // before any LDS read.
    h8 p[2][2][2], q[2][2][2];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          p[kk][i][e] = frag(St, wm + 32 * i + col, 2 * (2 * kk + half) + e);
          q[kk][i][e] = frag(St + kStageBytes, wn + 32 * i + col, 2 * (2 * kk + half) + e);
        }
    if (k + kStep < a.depth) {
      char* N = S + (s ^ 1) * 2 * kStageBytes;
      load_stage(bp, pitch, k + kStep, N);
      load_stage(bq, pitch, k + kStep, N + kStageBytes);
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          big[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[kk][i][0], q[kk][j][0], big[i][j], 0, 0, 0);
          small[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[kk][i][0], q[kk][j][1], small[i][j], 0, 0, 0);
          small[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[kk][i][1], q[kk][j][0], small[i][j], 0, 0, 0);
        }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
  }
  // Row 8 (e / 4) + 4 half + e % 4 of a block, column `col`.
  const uint32_t r0 = ti * kTile + wm, c0 = tj * kTile + wn;
  int eq[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint32_t n = c0 + 32 * j + col;
    eq[j] = exp_of(a.qMax[n]);
  }
  float top[2][3] = {};  // GRAD: of dg, du, m in the lane's columns
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const uint32_t r = r0 + 32 * i + 8 * (e >> 2) + 4 * half + (e & 3);
      const int ep = exp_of(a.pMax[r]);
      float v[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) v[j] = ldexpf(big[i][j][e] + small[i][j][e], -(ep + eq[j]));
      if constexpr (OP == STORE) {
        if (r >= a.rows) continue;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t n = c0 + 32 * j + col;
          float* to = a.out;
          if (a.turn) {
            to = j ? a.out2 : a.out;
            n = (c0 >> 1) + col;
          }
          if (n < a.cols && to) to[size_t(r) * a.pitch + n] = v[j];
        }
      }
      if constexpr (OP == GATE) {
        const uint32_t f = (c0 >> 1) + col;
        const float m = act<ACT>(v[0]) * v[1];
        a.out[size_t(r) * a.pitch + f] = m;
        if (a.g && r < a.rows && f < a.hidden) {
          a.g[size_t(r) * a.hidden + f] = v[0];
          a.u[size_t(r) * a.hidden + f] = v[1];
        }
        const float most = max32(size_of(m));
        if (col == 0 && most > 0.f) atomicMax(a.rowMax + r, __float_as_uint(most));
      }
      if constexpr (OP == GRAD) {
        float most = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t f = c0 + 32 * j + col;
          const bool live = r < a.rows && f < a.hidden;
          const size_t at = size_t(min(r, a.rows - 1)) * a.hidden + min(f, a.hidden - 1);
          float d;
          const float g = a.g[at], u = a.u[at], y = act_grad<ACT>(g, d);
          const float dg = live ? v[j] * u * d : 0.f, du = live ? v[j] * y : 0.f, m = live ? y * u : 0.f;
          float* to = a.out + size_t(r) * a.pitch + in_turn(f, 0);
          to[0] = dg;
          to[32] = du;
          a.out2[size_t(r) * (a.pitch / 2) + f] = m;
          top[j][0] = fmaxf(top[j][0], size_of(dg));
          top[j][1] = fmaxf(top[j][1], size_of(du));
          top[j][2] = fmaxf(top[j][2], size_of(m));
          most = fmaxf(most, fmaxf(size_of(dg), size_of(du)));
        }
        most = max32(most);
        if (col == 0 && most > 0.f) atomicMax(a.rowMax + r, __float_as_uint(most));
      }
    }
  if constexpr (OP == GRAD) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t f = c0 + 32 * j + col;
      uint32_t* to[3] = {a.colMax + in_turn(f, 0), a.colMax + in_turn(f, 1), a.colMax2 + f};
#pragma unroll
      for (int w = 0; w < 3; ++w)
        if (top[j][w] > 0.f) atomicMax(to[w], __float_as_uint(top[j][w]));
    }
  }
}

// Places in the workspace.
struct Places {
  size_t next = 0;
  size_t take(size_t floats) {
    const size_t p = next;
    next += (floats + 63) & ~size_t(63);
    return p;
  }
};

template <class F>
uint32_t job_blocks(Jobs& t, F&& f) {
  uint32_t n = 0;
  for (uint32_t i = 0; i < t.count; ++i) {
    t.start[i] = n;
    n += f(t.j[i]);
  }
  t.start[t.count] = n;
  return n;
}
bool run_max(Jobs& t) {
  const uint32_t n = job_blocks(t, [](const Job& j) { return cdiv(j.rows, kMaxRows) * cdiv(j.cols, kT); });
  hipLaunchKernelGGL(k_mlp_max, dim3(n), dim3(kT), 0, stream(), t);
  return check_launch("gated_mlp");
}
bool run_split(Jobs& t) {
  const uint32_t n = job_blocks(t, [](const Job& j) {
    const uint32_t by = j.turn < 0 ? 1 : 2, high = std::max(j.straight ? j.sRows : 0, j.across ? j.aPitch : 0);
    const uint32_t wide = std::max(j.straight ? j.sPitch / by : 0, j.across ? j.aRows / by : 0);
    return cdiv(high, kSq) * cdiv(wide, kSq);
  });
  hipLaunchKernelGGL(k_mlp_split, dim3(n), dim3(kT), 0, stream(), t);
  return check_launch("gated_mlp");
}
template <Op OP>
bool run_product(const Prod& a, MlpAct act = kSilu) {
  by_act(act, [&](auto k) {
    hipLaunchKernelGGL((k_mlp_product<OP, OP == STORE ? kSilu : decltype(k)::value>), dim3(a.tm * a.tn), dim3(kT), 0, stream(), a);
  });
  return check_launch("gated_mlp");
}
bool clear(uint32_t* p, size_t n) {
  hipLaunchKernelGGL(k_mlp_clear, dim3(std::min(cdiv(n, kT), 256u)), dim3(kT), 0, stream(), p, uint32_t(n));
  return check_launch("gated_mlp");
}

Job job(const float* src, uint32_t rows, uint32_t cols, uint32_t pitch, int turn = -1) {
  Job j{};
  j.src = const_cast<float*>(src);
  j.rows = rows;
  j.cols = cols;
  j.pitch = pitch;
  j.turn = turn;
  return j;
}

}  // namespace

bool mlp_forward_parts(const MlpArgs& a) {
  const uint32_t M = pad(a.rows, kTile), C = pad(a.cols, 64), F = pad(a.hidden, 64), O = pad(a.out, kTile);
  Places at;
  const size_t px = at.take(size_t(M) * C), pw = at.take(size_t(2) * F * C), pd = at.take(size_t(O) * F), pm = at.take(size_t(M) * F);
  const size_t top = at.take(0), xMax = at.take(M), wMax = at.take(2 * size_t(F)), dMax = at.take(O), mMax = at.take(M), end = at.next;
  float* ws = workspace(end);
  if (!ws) return false;
  auto bits = [&](size_t p) { return reinterpret_cast<uint32_t*>(ws + p); };
  ProfScope prof("mlp", 6.0 * a.rows * a.cols * a.hidden, 4.0 * (2.0 * a.rows * a.cols + 3.0 * a.cols * a.hidden));
  if (!clear(bits(top), end - top)) return false;
  Jobs t{};
  t.count = 4;
  t.j[0] = job(a.x, a.rows, a.cols, a.cols);
  t.j[0].rowMax = bits(xMax);
  for (int w = 0; w < 2; ++w) {
    t.j[1 + w] = job(w ? a.wu : a.wg, a.cols, a.hidden, a.hidden, w);
    t.j[1 + w].colMax = bits(wMax);
  }
  t.j[3] = job(a.wd, a.hidden, a.out, a.out);
  t.j[3].colMax = bits(dMax);
  if (!run_max(t)) return false;
  t.j[0].straight = ws + px;
  t.j[0].sPitch = C;
  t.j[0].sRows = M;
  for (int w = 1; w < 3; ++w) {
    t.j[w].across = ws + pw;
    t.j[w].aPitch = C;
    t.j[w].aRows = 2 * F;
  }
  t.j[3].across = ws + pd;
  t.j[3].aPitch = F;
  t.j[3].aRows = O;
  if (!run_split(t)) return false;
  Prod g{};
  g.p = ws + px;
  g.q = ws + pw;
  g.pMax = bits(xMax);
  g.qMax = bits(wMax);
  g.tm = M / kTile;
  g.tn = 2 * F / kTile;
  g.depth = C;
  g.rows = a.rows;
  g.out = ws + pm;
  g.pitch = F;
  g.hidden = a.hidden;
  g.rowMax = bits(mMax);
  if (a.saved) {
    g.g = a.saved;
    g.u = a.saved + size_t(a.rows) * a.hidden;
  }
  if (!run_product<GATE>(g, a.act)) return false;
  t.count = 1;
  t.j[0] = job(ws + pm, M, F, F);
  t.j[0].rowMax = bits(mMax);
  t.j[0].straight = ws + pm;
  t.j[0].sPitch = F;
  t.j[0].sRows = M;
  if (!run_split(t)) return false;
  Prod y{};
  y.p = ws + pm;
  y.q = ws + pd;
  y.pMax = bits(mMax);
  y.qMax = bits(dMax);
  y.tm = M / kTile;
  y.tn = O / kTile;
  y.depth = F;
  y.rows = a.rows;
  y.cols = a.out;
  y.out = a.y;
  y.pitch = a.out;
  return run_product<STORE>(y);
}

bool mlp_backward_parts(const MlpArgs& a, const float* dy, float* dx, float* dwg, float* dwu, float* dwd) {
  const bool weights = dwg || dwu;
  // Each side of a product is padded to whole tiles, whichever it is.
  const uint32_t M = pad(a.rows, kTile), C = pad(a.cols, kTile), F = pad(a.hidden, kTile), O = pad(a.out, kTile);
  Places at;
  const size_t pyr = at.take(size_t(M) * O), pyc = dwd ? at.take(size_t(O) * M) : 0, pd = at.take(size_t(F) * O);
  const size_t pxc = weights ? at.take(size_t(C) * M) : 0, pw = dx ? at.take(size_t(C) * 2 * F) : 0;
  const size_t pg = at.take(size_t(M) * 2 * F), pgc = weights ? at.take(size_t(2) * F * M) : 0;
  const size_t pm = at.take(size_t(M) * F), pmc = dwd ? at.take(size_t(F) * M) : 0;
  const size_t top = at.take(0), yrMax = at.take(M), ycMax = at.take(O), dMax = at.take(F), xMax = at.take(C), wMax = at.take(C),
               grMax = at.take(M), gcMax = at.take(2 * size_t(F)), mMax = at.take(F), end = at.next;
  float* ws = workspace(end);
  if (!ws) return false;
  auto bits = [&](size_t p) { return reinterpret_cast<uint32_t*>(ws + p); };
  ProfScope prof("mlp", 12.0 * a.rows * a.cols * a.hidden, 8.0 * (2.0 * a.rows * a.cols + 3.0 * a.cols * a.hidden));
  if (!clear(bits(top), end - top)) return false;
  Jobs t{};
  auto add = [&](const Job& j) -> Job& { return t.j[t.count++] = j; };
  {
    Job& j = add(job(dy, a.rows, a.out, a.out));
    j.rowMax = bits(yrMax);
    j.colMax = dwd ? bits(ycMax) : nullptr;
    add(job(a.wd, a.hidden, a.out, a.out)).rowMax = bits(dMax);
    if (weights) add(job(a.x, a.rows, a.cols, a.cols)).colMax = bits(xMax);
    if (dx)
      for (int w = 0; w < 2; ++w) add(job(w ? a.wu : a.wg, a.cols, a.hidden, a.hidden, w)).rowMax = bits(wMax);
  }
  if (!run_max(t)) return false;
  for (uint32_t i = 0; i < t.count; ++i) {
    Job& j = t.j[i];
    auto straight = [&](size_t p, uint32_t rows, uint32_t pitch) {
      j.straight = ws + p;
      j.sRows = rows;
      j.sPitch = pitch;
    };
    auto across = [&](size_t p, uint32_t rows, uint32_t pitch) {
      j.across = ws + p;
      j.aRows = rows;
      j.aPitch = pitch;
    };
    if (j.src == dy) {
      straight(pyr, M, O);
      if (dwd) across(pyc, O, M);
    } else if (j.turn >= 0) {
      straight(pw, C, 2 * F);
    } else if (j.rowMax == bits(dMax)) {
      straight(pd, F, O);
    } else {
      across(pxc, C, M);
    }
  }
  if (!run_split(t)) return false;
  Prod g{};
  g.p = ws + pyr;
  g.q = ws + pd;
  g.pMax = bits(yrMax);
  g.qMax = bits(dMax);
  g.tm = M / kTile;
  g.tn = F / kTile;
  g.depth = O;
  g.rows = a.rows;
  g.out = ws + pg;
  g.out2 = ws + pm;
  g.pitch = 2 * F;
  g.hidden = a.hidden;
  g.g = a.saved;
  g.u = a.saved + size_t(a.rows) * a.hidden;
  g.rowMax = bits(grMax);
  g.colMax = bits(gcMax);
  g.colMax2 = bits(mMax);
  if (!run_product<GRAD>(g, a.act)) return false;
  t.count = 0;
  if (dx || weights) {
    Job& j = add(job(ws + pg, M, 2 * F, 2 * F));
    j.rowMax = bits(grMax);
    j.colMax = bits(gcMax);
    if (dx) {
      j.straight = ws + pg;
      j.sRows = M;
      j.sPitch = 2 * F;
    }
    if (weights) {
      j.across = ws + pgc;
      j.aRows = 2 * F;
      j.aPitch = M;
    }
  }
  if (dwd) {
    Job& j = add(job(ws + pm, M, F, F));
    j.colMax = bits(mMax);
    j.across = ws + pmc;
    j.aRows = F;
    j.aPitch = M;
  }
  if (!run_split(t)) return false;
  auto product = [&](size_t p, const uint32_t* pMax, uint32_t rows, uint32_t tm, size_t q, const uint32_t* qMax, uint32_t cols,
                     uint32_t tn, uint32_t depth, float* out, float* out2, bool turn) {
    Prod r{};
    r.p = ws + p;
    r.q = ws + q;
    r.pMax = pMax;
    r.qMax = qMax;
    r.tm = tm;
    r.tn = tn;
    r.depth = depth;
    r.rows = rows;
    r.cols = cols;
    r.out = out;
    r.out2 = out2;
    r.pitch = cols;
    r.turn = turn;
    return run_product<STORE>(r);
  };
  if (dwd && !product(pmc, bits(mMax), a.hidden, F / kTile, pyc, bits(ycMax), a.out, O / kTile, M, dwd, nullptr, false)) return false;
  if (weights && !product(pxc, bits(xMax), a.cols, C / kTile, pgc, bits(gcMax), a.hidden, 2 * F / kTile, M, dwg, dwu, true)) return false;
  return !dx || product(pg, bits(grMax), a.rows, M / kTile, pw, bits(wMax), a.cols, C / kTile, 2 * F, dx, nullptr, false);
}

bool mlp_on_parts(const MlpArgs& a) {
  // a tile's rows are reached with 32-bit offsets
  return std::max({a.rows, a.cols, a.hidden, a.out}) <= (1u << 21) && double(a.rows) * a.cols * a.hidden >= 1e8;
}

}  // namespace dce
