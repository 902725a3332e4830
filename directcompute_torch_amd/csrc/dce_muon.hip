// The orthogonalised momentum update of many matrices at once.
//
//   m <- mu m + g,  d = g + mu m (or m),  X = d / (|d| + eps),
//   five times:  A = X X^T,  B = b A + c A^2,  X <- a X + B X,
//   w <- w - decay w - step X.
//
// The quintic a s + b s^3 + c s^5 takes every singular value s of X towards 1
// (K. Jordan, "Muon: an optimizer for hidden layers in neural networks", 2024,
// whose coefficients these are): X tends to the orthogonal factor of d.  A
// matrix with more rows than columns is worked on transposed, so that A is the
// smaller Gram matrix.
//
// Every matrix of a call runs in the same launches: a workgroup finds its
// matrix and tile in a table that travels as a kernel argument.  A and A^2 are
// symmetric: only tiles on or above the diagonal are multiplied, and stored
// twice.  A Gram product with long dot products and few tiles is split over
// them and summed by a pass of its own.
//
// Products: a value is kept as two fp16 parts, x 2^e = h + l, each rounded to
// nearest, and h h + (h l + l h) stands for the product: 22 to 24 bits at a
// third of the fp16 MFMA rate, which is 16 times the fp32 one.  Ranges are
// known, so the exponents are fixed: |X| <= 1.21 (|d| bounds its singular
// values by 1, and the quintic's largest value on [0, 1.21] is 1.21), |A| <=
// 1.47, |B| <= 2.81.  X is normalised, so its typical value is at least 2^-16
// and l's smallest step, 2^-39, is below the fp32 rounding of such a value.  X
// itself stays in fp32, for the term a X.  Errors are fp32's relative to the whole
// matrix, and to each row down to rows 2^-16 of the largest; one of 2^-20 is off by
// 2e-5 of its own length, one of 2^-24 by 3e-4, in an update that is as much smaller
// than the other rows'.  The two small products have an
// accumulator of their own: an MFMA cuts what it adds off at the scale of the
// largest addend, always downwards.
#include "dce_internal.h"

#include <algorithm>
#include <cmath>
#include <set>
#include <vector>

namespace dce {

namespace {

constexpr int kT = 256;
constexpr int kStep = 32;     // depth of an LDS stage of the 128 x 128 tiles
constexpr int kDepth = 128;   // and of the 64 x 64 tiles' only one
constexpr int kMaxM = 40;     // matrices of a launch
constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr int kExpX = 15, kExpA = 14;  // parts hold X 2^15, A 2^14, B 2^14

using h8 = _Float16 __attribute__((ext_vector_type(8)));
using f16v = float __attribute__((ext_vector_type(16)));

// One matrix, r x c as the caller has it; m <= n after the transposition.
struct Mat {
  float *w, *g, *mom;
  uint32_t m, n, mp, np;  // padded to whole tiles (zeros)
  uint32_t tall, splits;
  uint32_t chunk, chunks, sums;  // values of a momentum workgroup, their number, their sums' place
  float step;
  uint32_t x, xp, xt0, xt1, a, b, part;  // places in the workspace, in units of 64 floats
};
struct Mats {
  Mat t[kMaxM];
  uint32_t start[kMaxM + 1];  // first workgroup of each
  uint32_t count;
};
__device__ __forceinline__ int find_mat(const Mats& t, uint32_t blk) {
  int lo = 0, hi = int(t.count) - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.start[mid] <= blk) lo = mid; else hi = mid - 1;
  }
  return lo;
}
__device__ __forceinline__ float* at(float* ws, uint32_t place) { return ws + size_t(place) * 64; }

// Parts in memory: 8 consecutive values of a row are 8 h, then 8 l (32 bytes).
__device__ __forceinline__ void split8(const float* x, float by, h8& h, h8& l) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float v = x[e] * by;
    h[e] = _Float16(v);
    l[e] = _Float16(v - float(h[e]));
  }
}
__device__ __forceinline__ void put8(float* row, uint32_t k, const float* x, float by) {
  h8 h, l;
  split8(x, by, h, l);
  h8* p = reinterpret_cast<h8*>(row + k);
  p[0] = h;
  p[1] = l;
}

// ---------------------------------------------------------------------------
// d = g + mu m, m <- mu m + g, and the sums of d^2 (in double, one per
// workgroup: 4096 values, more where that would be over 1024 of them); d goes to
// X's place, as the caller's matrix lies.  16 bytes per value: AlexNet's
// 61 million 166 us, 5.9 TB/s.
// ---------------------------------------------------------------------------
constexpr uint32_t kChunk = 4096, kMaxChunks = 1024;
__global__ void __launch_bounds__(kT)
    k_muon_momentum(const Mats t, float* ws, double* sums, float mu, float clip, int nesterov) {
  __shared__ double sh[4];
  const int i = find_mat(t, blockIdx.x);
  const Mat M = t.t[i];
  const uint32_t id = blockIdx.x - t.start[i], n = M.m * M.n, end = min(n, (id + 1) * M.chunk);
  float* d = at(ws, M.xt1);  // free until the first step
  double sum = 0;
  auto one = [&](float g, float& m) {
    if (g > clip) g = clip;
    if (g < -clip) g = -clip;
    m = mu * m + g;
    const float v = nesterov ? mu * m + g : m;
    sum += double(v) * v;
    return v;
  };
  uint32_t c0 = id * M.chunk;
  for (; c0 + kChunk <= end; c0 += kChunk) {
    f4 G[4], V[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t k = c0 + (j * kT + threadIdx.x) * 4;
      G[j] = *reinterpret_cast<const f4*>(M.g + k);
      V[j] = *reinterpret_cast<const f4*>(M.mom + k);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t k = c0 + (j * kT + threadIdx.x) * 4;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float m = V[j][e];
        G[j][e] = one(G[j][e], m);
        V[j][e] = m;
      }
      *reinterpret_cast<f4*>(M.mom + k) = V[j];
      *reinterpret_cast<f4*>(d + k) = G[j];
    }
  }
  if (c0 < end) {  // the loads ahead of everything that depends on them
    constexpr int W = kChunk / kT;
    float G[W], V[W];
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const uint32_t k = min(c0 + j * kT + threadIdx.x, end - 1);
      G[j] = M.g[k];
      V[j] = M.mom[k];
    }
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const uint32_t k = c0 + j * kT + threadIdx.x;
      if (k >= end) break;
      d[k] = one(G[j], V[j]);
      M.mom[k] = V[j];
    }
  }
  sum = block_sum256(sum, sh);
  if (threadIdx.x == 0) sums[M.sums + id] = sum;
}

// X = d / (|d| + eps), 16 bytes per value too (221 us there, 4.4 TB/s).
// A 64 x 64 tile through LDS: X in fp32 and as parts, along rows and columns.
constexpr int kSq = 64, kPitch = 68;
__device__ __forceinline__ void put_tile(const float (&S)[kSq * kPitch], float* rows, uint32_t rowPitch,
                                         float* cols, uint32_t colPitch, uint32_t i0, uint32_t j0) {
#pragma unroll
  for (int u = 0; u < kSq * kSq / 8 / kT; ++u) {
    const uint32_t slot = threadIdx.x + kT * u;
    float v[8];
    {
      const uint32_t r = slot / 8, k = slot % 8 * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = S[r * kPitch + k + e];
      put8(rows + size_t(i0 + r) * rowPitch, j0 + k, v, ldexpf(1.f, kExpX));
    }
    {
      const uint32_t r = slot % 64, k = slot / 64 * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = S[(k + e) * kPitch + r];
      put8(cols + size_t(j0 + r) * colPitch, i0 + k, v, ldexpf(1.f, kExpX));
    }
  }
}
__global__ void __launch_bounds__(kT) k_muon_scale(const Mats t, float* ws, const double* sums) {
  __shared__ float S[kSq * kPitch];
  __shared__ double sh[4];
  __shared__ float norm[1];
  const int i = find_mat(t, blockIdx.x);
  const Mat M = t.t[i];
  const uint32_t tn = M.np / kSq, id = blockIdx.x - t.start[i], i0 = id / tn * kSq, j0 = id % tn * kSq;
  const float* d = at(ws, M.xt1);
  float* x = at(ws, M.x);
  const uint32_t si = M.tall ? 1 : M.n, sj = M.tall ? M.m : 1;
  float v[kSq * kSq / kT];
  // Loads of clamped places: behind a branch each would wait for the one before.
#pragma unroll
  for (int u = 0; u < kSq * kSq / kT; ++u) {
    const uint32_t s = threadIdx.x + kT * u;
    // consecutive threads along the caller's rows
    const uint32_t r = M.tall ? s % kSq : s / kSq, c = M.tall ? s / kSq : s % kSq;
    v[u] = d[min(i0 + r, M.m - 1) * si + min(j0 + c, M.n - 1) * sj];
  }
  // 1 / (|d| + eps), which every workgroup works out again: a launch less
  double sum = 0;
#pragma unroll
  for (uint32_t k = 0; k < kMaxChunks / kT; ++k) {
    const double more = sums[M.sums + min(k * kT + threadIdx.x, M.chunks - 1)];
    sum += k * kT + threadIdx.x < M.chunks ? more : 0.0;
  }
  sum = block_sum256(sum, sh);
  if (threadIdx.x == 0) norm[0] = float(1.0 / (sqrt(sum) + 1e-7));
  __syncthreads();
  const float by = norm[0];
#pragma unroll
  for (int u = 0; u < kSq * kSq / kT; ++u) {
    const uint32_t s = threadIdx.x + kT * u, r = M.tall ? s % kSq : s / kSq, c = M.tall ? s / kSq : s % kSq;
    v[u] = i0 + r < M.m && j0 + c < M.n ? v[u] * by : 0.f;
  }
#pragma unroll
  for (int u = 0; u < kSq * kSq / kT; ++u) {
    const uint32_t s = threadIdx.x + kT * u;
    S[(M.tall ? s % kSq : s / kSq) * kPitch + (M.tall ? s / kSq : s % kSq)] = v[u];
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kSq * kSq / 4 / kT; ++u) {
    const uint32_t s = threadIdx.x + kT * u, r = s / (kSq / 4), c = s % (kSq / 4) * 4;
    *reinterpret_cast<f4*>(x + size_t(i0 + r) * M.np + j0 + c) = *reinterpret_cast<const f4*>(S + r * kPitch + c);
  }
  put_tile(S, at(ws, M.xp), M.np, at(ws, M.xt0), M.mp, i0, j0);
}

// ---------------------------------------------------------------------------
// Products C = P Q^T of parts, both along their rows, in BLK x BLK tiles of four
// waves.
//   128: 64 x 64 per wave (2 x 2 blocks of 32 x 32), the depth in steps of 32
//        through two LDS stages, the next one's direct loads in flight while one
//        is multiplied; two workgroups per CU.  For launches that fill the chip.
//        AlexNet's eight matrices: A 709 us, B 462, X 1486, 310 TFLOP/s of fp32
//        products; power holds the clock at 1.8 GHz.
//   64:  32 x 32 per wave, depths of 128 loaded at once.  A step of the other
//        kernel takes a load's latency where a CU has one workgroup (about 1 us);
//        here one latency covers four times the depth, over four times the
//        workgroups.
// A stage's rows are 16-byte slots, h and l of 8 values in turn, XORed by the row
// so that a read of one slot of 16 rows covers the 64 banks once.
// ---------------------------------------------------------------------------
enum Op { GRAM, POLY, APPLY, LAST };
template <int BLK>
struct Lds {
  static constexpr int DEPTH = BLK == 128 ? kStep : kDepth, SLOTS = DEPTH / 4;  // slots of a row
  static constexpr int STAGE = BLK * DEPTH * 4;   // bytes of one operand's stage
  static constexpr int CP = BLK + 4;              // pitch of the result tile
  static constexpr int IN = (BLK == 128 ? 4 : 2) * STAGE, OUT = BLK * CP * 4;
  static constexpr int BYTES = IN > OUT ? IN : OUT;
  __device__ static __forceinline__ int swz(int row) { return SLOTS == 8 ? (row >> 1) & 7 : row & 15; }
  // A slot from `end` on is zeros.
  __device__ static __forceinline__ void load(const BRes& b, uint32_t pitchBytes, uint32_t k, uint32_t end, char* S) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < STAGE / 16 / kT; ++i) {
      const uint32_t slot = threadIdx.x + kT * i, row = slot / SLOTS, c = (slot % SLOTS) ^ swz(row);
      const uint32_t off = row * pitchBytes + k * 4 + c * 16;
      b.ld16_lds(SLOTS == 8 || k + c * 4 < end ? off : kOob * 4u, S + (wave * 64 + i * kT) * 16);
    }
  }
  __device__ static __forceinline__ h8 frag(const char* S, int row, int c) {
    return *reinterpret_cast<const h8*>(S + (row * SLOTS + (c ^ swz(row))) * 16);
  }
};
// Tile (i, j), i <= j, of the upper triangle in row order.
__device__ __forceinline__ void triangle(uint32_t id, uint32_t n, uint32_t& i, uint32_t& j) {
  i = 0;
  while (id >= n - i) {
    id -= n - i;
    ++i;
  }
  j = i + id;
}

template <Op OP, int BLK>
__global__ void __launch_bounds__(kT) __attribute__((amdgpu_waves_per_eu(2)))
    k_muon_product(const Mats t, float* ws, uint32_t cur, float decay) {
  using L = Lds<BLK>;
  constexpr int F = BLK / 64;  // blocks of a wave, each way
  __shared__ __attribute__((aligned(16))) char S[L::BYTES];
  const uint32_t blk = xcd_block_id();
  const int mi = find_mat(t, blk);
  const Mat M = t.t[mi];
  uint32_t id = blk - t.start[mi], ti, tj, sp = 0;
  const uint32_t tm = M.mp / BLK;
  uint32_t end = OP == GRAM ? M.np : M.mp, k0 = 0;
  if constexpr (OP == GRAM) {
    const uint32_t tiles = tm * (tm + 1) / 2, steps = (end + L::DEPTH - 1) / L::DEPTH;
    sp = id / tiles;
    id -= sp * tiles;
    k0 = uint32_t(uint64_t(steps) * sp / M.splits) * L::DEPTH;
    end = min(end, uint32_t(uint64_t(steps) * (sp + 1) / M.splits) * L::DEPTH);
  }
  if constexpr (OP == GRAM || OP == POLY) {
    triangle(id, tm, ti, tj);
  } else {
    ti = id % tm;
    tj = id / tm;
  }
  const float* P = at(ws, OP == GRAM ? M.xp : OP == POLY ? M.a : M.b);
  const float* Q = at(ws, OP == GRAM ? M.xp : OP == POLY ? M.a : cur ? M.xt1 : M.xt0);
  const uint32_t pitch = OP == GRAM ? M.np : M.mp;
  BRes bp, bq;
  bp.init(P + size_t(ti) * BLK * pitch, BLK * pitch);
  bq.init(Q + size_t(tj) * BLK * pitch, BLK * pitch);

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = (wave >> 1) * 32 * F, wn = (wave & 1) * 32 * F;
  const int col = lane & 31, half = lane >> 5;
  f16v big[F][F], small[F][F];
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) big[i][j][e] = small[i][j][e] = 0.f;
  auto mul = [&](const h8 (&p)[F][2], const h8 (&q)[F][2]) {
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
      for (int j = 0; j < F; ++j) {
        big[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[i][0], q[j][0], big[i][j], 0, 0, 0);
        small[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[i][0], q[j][1], small[i][j], 0, 0, 0);
        small[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[i][1], q[j][0], small[i][j], 0, 0, 0);
      }
  };
  auto frags = [&](const char* St, int w, int kk, h8 (&f)[F][2]) {
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) f[i][e] = L::frag(St, w + 32 * i + col, 2 * (2 * kk + half) + e);
  };

  // What the epilogue reads, in flight with the operands where registers allow.
  constexpr bool EARLY = BLK == 64;
  constexpr int NU = BLK * BLK / 8 / kT, NW = EARLY && OP == LAST ? BLK * BLK / kT : 1;
  const uint32_t i0 = ti * BLK, j0 = tj * BLK;
  f4 x0[EARLY ? NU : 1], x1[EARLY ? NU : 1];
  float w0[NW];
  auto epilogue_loads = [&](int u, f4& a, f4& b) {
    const uint32_t slot = threadIdx.x + kT * u, r = slot / (BLK / 8), k = slot % (BLK / 8) * 8;
    const float* p = OP == POLY ? at(ws, M.a) + size_t(i0 + r) * M.mp : at(ws, M.x) + size_t(i0 + r) * M.np;
    a = reinterpret_cast<const f4*>(p + j0 + k)[0];
    b = reinterpret_cast<const f4*>(p + j0 + k)[1];
  };
  // Consecutive threads along the caller's rows; of clamped places, as in k_muon_scale.
  const uint32_t si = M.tall ? 1 : M.n, sj = M.tall ? M.m : 1;
  auto weight = [&](int u) {
    const uint32_t s = threadIdx.x + kT * u, r = M.tall ? s % BLK : s / BLK, c = M.tall ? s / BLK : s % BLK;
    return M.w[min(i0 + r, M.m - 1) * si + min(j0 + c, M.n - 1) * sj];
  };
  L::load(bp, pitch * 4, k0, end, S);
  L::load(bq, pitch * 4, k0, end, S + L::STAGE);
  if constexpr (EARLY && OP != GRAM) {
#pragma unroll
    for (int u = 0; u < NU; ++u) epilogue_loads(u, x0[u], x1[u]);
  }
  if constexpr (EARLY && OP == LAST) {
#pragma unroll
    for (int u = 0; u < NW; ++u) w0[u] = weight(u);
  }
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if constexpr (BLK == 128) {
    int s = 0;
    for (uint32_t k = k0; k < end; k += kStep, s ^= 1) {
      const char* Sp = S + s * 2 * L::STAGE;
      // Fragments first: a direct load in flight would make the compiler wait
      // for it before any LDS read.
      h8 p[2][F][2], q[2][F][2];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        frags(Sp, wm, kk, p[kk]);
        frags(Sp + L::STAGE, wn, kk, q[kk]);
      }
      if (k + kStep < end) {
        char* N = S + (s ^ 1) * 2 * L::STAGE;
        L::load(bp, pitch * 4, k + kStep, end, N);
        L::load(bq, pitch * 4, k + kStep, end, N + L::STAGE);
      }
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) mul(p[kk], q[kk]);
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
    }
  } else {
    for (uint32_t k = k0;;) {
#pragma unroll
      for (int kk = 0; kk < kDepth / 16; ++kk) {
        if (kk == 4 && end - k <= 64) break;  // the depth is a multiple of 64
        h8 p[F][2], q[F][2];
        frags(S, wm, kk, p);
        frags(S + L::STAGE, wn, kk, q);
        mul(p, q);
      }
      __syncthreads();
      k += kDepth;
      if (k >= end) break;
      L::load(bp, pitch * 4, k, end, S);
      L::load(bq, pitch * 4, k, end, S + L::STAGE);
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
    }
  }
  // The tile in LDS, in its own scale.
  float* C = reinterpret_cast<float*>(S);
  constexpr int CP = L::CP;
  const float unit = OP == GRAM ? ldexpf(1.f, -2 * kExpX) : OP == POLY ? ldexpf(1.f, -2 * kExpA)
                                                                       : ldexpf(1.f, -kExpX - kExpA);
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        C[(wm + 32 * i + 8 * (e >> 2) + 4 * half + (e & 3)) * CP + wn + 32 * j + col] =
            (big[i][j][e] + small[i][j][e]) * unit;
  __syncthreads();
  if constexpr (OP == GRAM) {
    if (M.splits > 1) {  // summed by k_muon_sum
      float* out = at(ws, M.part) + (size_t(sp) * (tm * (tm + 1) / 2) + id) * (BLK * BLK);
#pragma unroll 4
      for (int u = 0; u < BLK * BLK / 4 / kT; ++u) {
        const uint32_t slot = threadIdx.x + kT * u, r = slot / (BLK / 4), c = slot % (BLK / 4) * 4;
        *reinterpret_cast<f4*>(out + slot * 4) = *reinterpret_cast<const f4*>(C + r * CP + c);
      }
      return;
    }
  }
  constexpr int UNROLL = BLK == 128 ? 1 : 2;
  float* out = at(ws, OP == GRAM ? M.a : OP == POLY ? M.b : M.xp);
#pragma unroll UNROLL
  for (int u = 0; u < NU; ++u) {
    const uint32_t slot = threadIdx.x + kT * u, r = slot / (BLK / 8), k = slot % (BLK / 8) * 8;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = C[r * CP + k + e];
    f4 p = {0.f, 0.f, 0.f, 0.f}, q = p;
    if constexpr (EARLY && OP != GRAM) {
      p = x0[u];
      q = x1[u];
    } else if constexpr (OP != GRAM) {
      epilogue_loads(u, p, q);
    }
    if constexpr (OP == POLY) {  // B = b A + c A^2
      const h8 ah = __builtin_bit_cast(h8, p), al = __builtin_bit_cast(h8, q);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        v[e] = kB * ((float(ah[e]) + float(al[e])) * ldexpf(1.f, -kExpA)) + kC * v[e];
    }
    if constexpr (OP == APPLY || OP == LAST) {  // X <- a X + B X
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = p[e] = kA * p[e] + v[e];
        v[4 + e] = q[e] = kA * q[e] + v[4 + e];
      }
      if constexpr (OP == APPLY) {
        float* x = at(ws, M.x) + size_t(i0 + r) * M.np + j0 + k;
        reinterpret_cast<f4*>(x)[0] = p;
        reinterpret_cast<f4*>(x)[1] = q;
      }
    }
    if constexpr (OP != LAST)
      put8(out + size_t(i0 + r) * (OP == APPLY ? M.np : M.mp), j0 + k, v, ldexpf(1.f, OP == APPLY ? kExpX : kExpA));
    if constexpr (OP != GRAM) {  // for the pass over columns
#pragma unroll
      for (int e = 0; e < 8; ++e) C[r * CP + k + e] = v[e];
    }
  }
  if ((OP == GRAM || OP == POLY) && ti == tj) return;
  __syncthreads();
  if constexpr (OP == LAST) {  // w <- w - decay w - step X, along the caller's rows
    constexpr int W = EARLY ? NW : 8;
#pragma unroll 1
    for (int u = 0; u < BLK * BLK / kT; u += W) {
      float w[W];
#pragma unroll
      for (int e = 0; e < W; ++e) w[e] = EARLY ? w0[e] : weight(u + e);
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const uint32_t s = threadIdx.x + kT * (u + e), r = M.tall ? s % BLK : s / BLK, c = M.tall ? s / BLK : s % BLK;
        const float next = w[e] - decay * w[e] - M.step * C[r * CP + c];
        if (i0 + r < M.m && j0 + c < M.n) M.w[(i0 + r) * si + (j0 + c) * sj] = next;
      }
    }
    return;
  }
  float* tr = OP == APPLY ? at(ws, cur ? M.xt0 : M.xt1) : out;
#pragma unroll UNROLL
  for (int u = 0; u < BLK * BLK / 8 / kT; ++u) {
    const uint32_t slot = threadIdx.x + kT * u, r = slot % BLK, k = slot / BLK * 8;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = C[(k + e) * CP + r];
    put8(tr + size_t(j0 + r) * M.mp, i0 + k, v, ldexpf(1.f, OP == APPLY ? kExpX : kExpA));
  }
}

// A from the partial tiles of a split Gram product: a workgroup per 16 rows of a
// tile.
template <int BLK>
__global__ void __launch_bounds__(kT) k_muon_sum(const Mats t, float* ws) {
  constexpr int RW = 16, CP = BLK + 4, PIECES = BLK / RW;
  __shared__ float C[RW * CP];
  const int mi = find_mat(t, blockIdx.x);
  const Mat M = t.t[mi];
  const uint32_t id = blockIdx.x - t.start[mi], piece = id % PIECES, tile = id / PIECES, tm = M.mp / BLK;
  const uint32_t tiles = tm * (tm + 1) / 2;
  uint32_t ti, tj;
  triangle(tile, tm, ti, tj);
  const float* part = at(ws, M.part) + size_t(tile) * (BLK * BLK) + piece * RW * BLK;
  float* a = at(ws, M.a);
  const uint32_t i0 = ti * BLK + piece * RW, j0 = tj * BLK;
  const uint32_t r = threadIdx.x / (BLK / 8), k = threadIdx.x % (BLK / 8) * 8;
  if (r < RW) {
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (uint32_t s = 0; s < M.splits; ++s) {
      const f4* p = reinterpret_cast<const f4*>(part + size_t(s) * tiles * (BLK * BLK) + threadIdx.x * 8);
      const f4 p0 = p[0], p1 = p[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] += p0[e];
        v[4 + e] += p1[e];
      }
    }
    put8(a + size_t(i0 + r) * M.mp, j0 + k, v, ldexpf(1.f, kExpA));
#pragma unroll
    for (int e = 0; e < 8; ++e) C[r * CP + k + e] = v[e];
  }
  if (ti == tj) return;
  __syncthreads();
  const uint32_t c = threadIdx.x % BLK, q = threadIdx.x / BLK * 8;
  if (q < RW) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = C[(q + e) * CP + c];
    put8(a + size_t(j0 + c) * M.mp, i0 + q, v, ldexpf(1.f, kExpA));
  }
}

inline uint32_t cdiv(uint64_t a, uint64_t b) { return uint32_t((a + b - 1) / b); }
inline uint32_t pad(uint32_t v, uint32_t to) { return (v + to - 1) / to * to; }

// start[] for `f(matrix)` workgroups each; returns their number.
template <class F>
uint32_t blocks(Mats& t, F&& f) {
  uint32_t n = 0;
  for (uint32_t i = 0; i < t.count; ++i) {
    t.start[i] = n;
    n += f(t.t[i]);
  }
  t.start[t.count] = n;
  return n;
}

struct Places {
  size_t next = 0;  // in units of 64 floats
  uint32_t take(size_t floats) {
    const size_t p = next;
    next += (floats + 63) / 64;
    return uint32_t(p);
  }
};

// The matrices of one set of launches.
struct Group {
  Mats t{};
  bool big = false, split = false;  // on 128 x 128 tiles; with a Gram product that is split
  size_t sums = 0, floats = 0;      // the sums' place in the workspace, its size
};

// Places in the workspace, and splits.
template <int BLK>
void plan_group(Group& gr) {
  Mats& t = gr.t;
  constexpr uint32_t depth = Lds<BLK>::DEPTH;
  // A Gram product is split so that no workgroup has more than a quarter of a CU's
  // share of the launch's depth, and none less than 256 (AlexNet's matrices: half a
  // share 14.7 ms, a third 14.7, a quarter or a sixth 13.4, an eighth 13.8).
  auto tri = [](const Mat& m) { return m.mp / BLK * (m.mp / BLK + 1) / 2; };
  double all = 0;
  for (uint32_t i = 0; i < t.count; ++i) {
    t.t[i].mp = pad(t.t[i].m, BLK);
    t.t[i].np = pad(t.t[i].n, BLK);
    all += double(tri(t.t[i])) * t.t[i].np;
  }
  const double most = std::max(256.0, all / (4.0 * num_cus()));
  Places at;
  uint32_t chunks = 0;
  for (uint32_t i = 0; i < t.count; ++i) {
    Mat& m = t.t[i];
    m.splits = std::min<uint32_t>(cdiv(m.np, depth), std::max<uint32_t>(1, uint32_t(std::ceil(m.np / most))));
    gr.split |= m.splits > 1;
    const size_t xn = size_t(m.mp) * m.np, an = size_t(m.mp) * m.mp;
    m.x = at.take(xn);
    m.xp = at.take(xn);
    m.xt0 = at.take(xn);
    m.xt1 = at.take(xn);
    m.a = at.take(an);
    m.b = at.take(an);
    m.part = m.splits > 1 ? at.take(size_t(m.splits) * tri(m) * BLK * BLK) : 0;
    const size_t size = size_t(m.m) * m.n;
    m.chunk = cdiv(cdiv(size, kMaxChunks), kChunk) * kChunk;
    m.chunks = cdiv(size, m.chunk);
    m.sums = chunks;
    chunks += m.chunks;
  }
  gr.sums = size_t(at.take(size_t(2) * chunks)) * 64;
  gr.floats = at.next * 64;
}

template <int BLK>
bool run_group(Group& gr, float* ws, float mu, bool nesterov, float decay, float clip, uint32_t steps) {
  Mats& t = gr.t;
  auto tri = [](const Mat& m) { return m.mp / BLK * (m.mp / BLK + 1) / 2; };
  double* dsum = reinterpret_cast<double*>(ws + gr.sums);
  uint32_t n = blocks(t, [](const Mat& m) { return m.chunks; });
  hipLaunchKernelGGL(k_muon_momentum, dim3(n), dim3(kT), 0, stream(), t, ws, dsum, mu, clip, int(nesterov));
  n = blocks(t, [](const Mat& m) { return m.mp / kSq * (m.np / kSq); });
  hipLaunchKernelGGL(k_muon_scale, dim3(n), dim3(kT), 0, stream(), t, ws, dsum);
  for (uint32_t s = 0; s < steps; ++s) {
    n = blocks(t, [&](const Mat& m) { return tri(m) * m.splits; });
    hipLaunchKernelGGL((k_muon_product<GRAM, BLK>), dim3(n), dim3(kT), 0, stream(), t, ws, s & 1, decay);
    if (gr.split) {
      n = blocks(t, [&](const Mat& m) { return m.splits > 1 ? tri(m) * (BLK / 16) : 0; });
      hipLaunchKernelGGL(k_muon_sum<BLK>, dim3(n), dim3(kT), 0, stream(), t, ws);
    }
    n = blocks(t, tri);
    hipLaunchKernelGGL((k_muon_product<POLY, BLK>), dim3(n), dim3(kT), 0, stream(), t, ws, s & 1, decay);
    n = blocks(t, [](const Mat& m) { return m.mp / BLK * (m.np / BLK); });
    if (s + 1 < steps)
      hipLaunchKernelGGL((k_muon_product<APPLY, BLK>), dim3(n), dim3(kT), 0, stream(), t, ws, s & 1, decay);
    else
      hipLaunchKernelGGL((k_muon_product<LAST, BLK>), dim3(n), dim3(kT), 0, stream(), t, ws, s & 1, decay);
  }
  return check_launch("MuonBatch");
}

}  // namespace

bool muon_multi(void** params, void** grads, void** momenta, const uint32_t* rows, const uint32_t* cols,
                const float* stepSizes, uint32_t n, float mu, bool nesterov, float decay, float clip,
                uint32_t steps) {
  std::vector<Mat> all;
  std::set<const void*> written, read;
  double bytes = 0, flops = 0;
  for (uint32_t i = 0; i < n; ++i) {
    if (!params[i] || !grads[i]) continue;
    Buffer* W = as_buffer(params[i], "MuonBatch(param)");
    Buffer* G = as_buffer(grads[i], "MuonBatch(grad)");
    Buffer* V = as_buffer(momenta[i], "MuonBatch(momentum)");
    if (!W || !G || !V) return false;
    const uint64_t size = uint64_t(rows[i]) * cols[i];
    if (!size || size >= 0x80000000ull || W->count < size || G->count < size || V->count < size) {
      set_error("MuonBatch: matrix %u of %u x %u does not fit its buffers", i, rows[i], cols[i]);
      return false;
    }
    if (!written.insert(W).second || !written.insert(V).second) {
      set_error("MuonBatch: the parameter or momentum of matrix %u is another one's too", i);
      return false;
    }
    read.insert(G);
    Mat m{};
    m.w = W->ptr;
    m.g = G->ptr;
    m.mom = V->ptr;
    m.tall = rows[i] > cols[i];
    m.m = std::min(rows[i], cols[i]);
    m.n = std::max(rows[i], cols[i]);
    m.step = stepSizes[i];
    // a tile's operand rows are reached with 32-bit offsets
    if (uint64_t(m.n) * 128 + (1u << 14) >= kOob) {
      set_error("MuonBatch: matrix %u is %u long (4 million at most)", i, m.n);
      return false;
    }
    all.push_back(m);
    bytes += 20.0 * size;
    flops += steps * (3.0 * m.m * m.m * m.n + double(m.m) * m.m * m.m);
  }
  if (all.empty()) return true;
  for (const void* g : read)
    if (written.count(g)) {
      set_error("MuonBatch: a gradient is a parameter or momentum too");
      return false;
    }
  ProfScope prof("muon", flops, bytes);
  // Groups of up to kMaxM matrices, and of up to 2^28 values (padded to whole tiles, a
  // thin matrix being up to 128 times its size) unless one is larger.
  // Tiles by the operations of a step (us on 128 / on 64): 1024 x 1024 435 / 281,
  // 1536 x 1536 (1.4e10) 649 / 571, four 768 x 768 with two 768 x 2000 (1.5e10)
  // 631 / 578, 2048 x 2048 (3.4e10) 914 / 1032, 2048 x 4096 1336 / 1652.
  std::vector<Group> groups;
  size_t floats = 0;
  auto padded = [](const Mat& m) { return size_t(pad(m.m, 128)) * pad(m.n, 128); };
  for (size_t i = 0; i < all.size();) {
    Group gr;
    Mats& t = gr.t;
    size_t values = 0;
    double work = 0;  // of a step
    while (i < all.size() && t.count < uint32_t(kMaxM) &&
           (!t.count || values + padded(all[i]) <= (size_t(1) << 28))) {
      values += padded(all[i]);
      work += (3.0 * all[i].n + all[i].m) * all[i].m * all[i].m;
      t.t[t.count++] = all[i++];
    }
    gr.big = work >= 2.2e10;
    (gr.big ? plan_group<128> : plan_group<64>)(gr);
    floats = std::max(floats, gr.floats);
    groups.push_back(gr);
  }
  // The largest group's, before any launch: a call that it does not fit changes nothing.
  float* ws = workspace(floats);
  if (!ws) return false;
  for (Group& gr : groups)
    if (!(gr.big ? run_group<128> : run_group<64>)(gr, ws, mu, nesterov, decay, clip, steps)) return false;
  return true;
}

}  // namespace dce
