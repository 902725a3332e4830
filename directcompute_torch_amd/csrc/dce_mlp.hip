// The gated feed-forward block:
//
//   g = x Wg,  u = x Wu,  m = act(g) u,  y = m Wd,
//
// and its gradients:
//
//   dm = dy Wd^T,  dg = dm u act'(g),  du = dm act(g),
//   dWd = m^T dy,  dWg = x^T dg,  dWu = x^T du,  dx = dg Wg^T + du Wu^T.
#include "dce_mlp.h"

namespace dce {

namespace {

using f16v = float __attribute__((ext_vector_type(16)));
inline uint32_t cdiv(uint64_t a, uint64_t b) { return uint32_t((a + b - 1) / b); }

// ---------------------------------------------------------------------------
// Products of small calls on fp32 MFMAs, C[r][c] = sum over k of A(r, k) B(c, k), in
// tiles of 32 x 32 (T = 1), or 64 x 64 of large ones (T = 2).  1, 2, 4 or 8 of a workgroup's eight waves share a tile's depth and add
// up their sums in LDS, in order; of a deep product with few tiles workgroups do, too, whose
// sums a pass brings together, in order.  No stage in between: an operand whose depth is
// contiguous comes by 16 bytes a lane, 4 k of its row, the other one by a dword of each k,
// 32 neighbours together.  The MFMA's two k of a step are then 4 apart, for both.  Rows and
// columns outside are the last ones again; what comes of them is not stored.  Tiles go down a
// column first, and those next to each other run on one XCD: rows of odd length share cache
// lines (100 x 2000 x 8001 forward 226 us without that, 179 with it).
//
// Bound by memory latency: a wave has four octets of k in flight and then multiplies them,
// and most calls have a wave or two of each SIMD only.  154 x 384 x 1001, training
// (1.07 GFLOP, 7 us at the rate of a large fp32 product): the gate's product 10 us, y 6 and 3
// for its sums, the gradient's 9, the four others 18.5 and 4; 64 x 1024 x 2816, training: 81
// us (with eight waves for each tile and no splits 102).  Eight octets in flight, with twice
// the code, took 10 % more.  Many rows of large weights (96 x 2048 x 8192 training: 465 us, 62
// TFLOP/s, more than the plain form's 391) wait for L2 as much as they multiply: MFMAs busy 22 to 48 %, 7 to 12
// TB/s from L2, dm's product 22; each weight is read once for 32 rows.
// ---------------------------------------------------------------------------
enum Op { STORE, GATE, GRAD };
struct Side {
  const float* p;
  uint32_t n, pitch;  // rows or columns of the result; from one row (contiguous: of the depth) to the next
};
struct Prod {
  Side a, b, b2;   // b2: GATE: Wu; STORE: of the second part
  const float* a2; // STORE: a second part of the depth, as long as the first (null: none)
  uint32_t depth, start, down, tiles;  // first workgroup; tiles of a column, in all
  uint32_t waves, splits;  // log2 of the waves that share a tile's depth, workgroups that do
  uint32_t aDeep, bDeep;  // is the depth contiguous
  float *out, *g, *u, *du, *m;
};
struct Prods {
  Prod p[4];
  uint32_t count, side;  // side of a tile, in 32
  const uint32_t* again; // AGAIN: set for the rows that are wanted (null: all)
};

// Octet o of the depth, k = 8 o + 4 half + i; WHOLE: all of it is there, else zeros past the
// depth.  `off`: bytes of the lane's row (or column) and its half.
template <bool DEEP, bool WHOLE>
__device__ __forceinline__ void octet(const float* p, uint32_t pitch, uint32_t off, uint32_t o, uint32_t depth, int half, float (&v)[4]) {
  if constexpr (WHOLE && DEEP) {
    const f4u q = ldus<false, f4u>(reinterpret_cast<const char*>(p + 8 * o) + off);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = q[i];
  } else if constexpr (WHOLE) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const float*>(reinterpret_cast<const char*>(p + size_t(8 * o + i) * pitch) + off);
  } else {
    const float* row = reinterpret_cast<const float*>(reinterpret_cast<const char*>(p) + off) - (DEEP ? 4 * half : size_t(4 * half) * pitch);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t k = 8 * o + 4 * half + i;
      const float x = row[size_t(min(k, depth - 1)) * (DEEP ? 1 : pitch)];
      v[i] = k < depth ? x : 0.f;
    }
  }
}

constexpr int kWaves = 8;
template <Op OP>
using SumsOf = float[OP == GATE ? 2 : 1][kWaves][32 * 32];
// Workgroup id of a launch's; sums start at `start`.
template <Op OP, MlpAct ACT, int T, bool AGAIN>
__device__ __forceinline__ void small_tiles(const Prods& all, uint32_t id, SumsOf<OP>& S, float start) {
  constexpr int NW = kWaves, D = OP == GATE ? 2 : 1;
  int which = 0;
  while (which + 1 < int(all.count) && all.p[which + 1].start <= id) ++which;
  const Prod& P = all.p[which];
  id -= P.start;
  const uint32_t each = NW >> P.waves, groups = (P.tiles + each - 1) >> (3 - P.waves);  // tiles of a workgroup
  id = xcd_place(id, groups * P.splits);
  const uint32_t sp = id / groups, first = (id - sp * groups) * each;
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  auto wanted = [&](uint32_t r) { return r < P.a.n && (!AGAIN || !all.again || all.again[r]); };
  if (AGAIN && all.again) {  // the same in each wave
    bool any = false;
    for (uint32_t t = lane; t < each * T * 32; t += 64) any |= wanted(min(first + t / (T * 32), P.tiles - 1) % P.down * (T * 32) + t % (T * 32));
    if (!__any(any)) return;
  }
  const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t tile = min(first + (w >> P.waves), P.tiles - 1), share = (sp << P.waves) + (w & ((1u << P.waves) - 1)), shares = P.splits << P.waves;
  static_assert(T == 1 || OP == STORE);
  constexpr int N = D * T;  // blocks side by side
  f16v acc[T][N];
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int d = 0; d < N; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[t][d][e] = start;
  const uint32_t tj = tile / P.down, ti = tile - tj * P.down;
  uint32_t ar[T], bc[T];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    ar[t] = min((ti * T + t) * 32 + col, P.a.n - 1);
    bc[t] = min((tj * T + t) * 32 + col, P.b.n - 1);
  }
  const uint32_t octets = P.depth / 8, few = octets / shares, more = octets - few * shares;
  const uint32_t lo = share * few + min(share, more), hi = lo + few + (share < more);
  const bool tail = P.depth % 8 && share + 1 == shares;
  // This thread's places in block (bi, bj) of the group's tile i; GRAD: g and u there, the first ones' ahead of the product.
  size_t at[2];
  bool in[2];
  float g[2], u[2];
  auto at_of = [&](uint32_t i, int bi, int bj) __attribute__((always_inline)) {
    const uint32_t now = min(first + i, P.tiles - 1), nj = now / P.down, ni = now - nj * P.down;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t t = threadIdx.x + h * NW * 64, r = (ni * T + bi) * 32 + t / 32, c = (nj * T + bj) * 32 + t % 32;
      in[h] = first + i < P.tiles && wanted(r) && c < P.b.n;
      at[h] = in[h] ? size_t(r) * P.b.n + c : 0;
      if constexpr (OP == GRAD) {
        g[h] = P.g[at[h]];
        u[h] = P.u[at[h]];
      }
    }
  };
  if (OP == GRAD) at_of(0, 0, 0);
  auto run = [&](auto aDeep, auto bDeep, const float* a, const float* b, const float* b2) __attribute__((always_inline)) {
    constexpr bool AD = decltype(aDeep)::value, BD = decltype(bDeep)::value;
    uint32_t ao[T], bo[T];
#pragma unroll
    for (int t = 0; t < T; ++t) {
      ao[t] = (AD ? ar[t] * P.a.pitch + 4 * half : 4 * half * P.a.pitch + ar[t]) * 4;
      bo[t] = (BD ? bc[t] * P.b.pitch + 4 * half : 4 * half * P.b.pitch + bc[t]) * 4;
    }
    constexpr int U = 4 / T;  // octets in flight
    float x[U][T][4], y[U][N][4];
    auto mul = [&](int j) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
          for (int d = 0; d < N; ++d) acc[t][d] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j][t][i], y[j][d][i], acc[t][d], 0, 0, 0);
    };
    uint32_t o = lo;
    auto fetch = [&](int j, uint32_t at) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < T; ++t) {
        octet<AD, true>(a, P.a.pitch, ao[t], at, P.depth, half, x[j][t]);
        octet<BD, true>(b, P.b.pitch, bo[t], at, P.depth, half, y[j][t]);
      }
      if constexpr (D == 2) octet<BD, true>(b2, P.b.pitch, bo[0], at, P.depth, half, y[j][N - 1]);
    };
    for (; o + U <= hi; o += U) {
#pragma unroll
      for (int j = 0; j < U; ++j) fetch(j, o + j);
#pragma unroll
      for (int j = 0; j < U; ++j) mul(j);
    }
    if (o < hi) {  // fewer
#pragma unroll
      for (int j = 0; j < U - 1; ++j) fetch(j, min(o + j, hi - 1));
      mul(0);
#pragma unroll
      for (int j = 1; j < U - 1; ++j)
        if (o + j < hi) mul(j);
    }
    if (tail) {
#pragma unroll
      for (int t = 0; t < T; ++t) {
        octet<AD, false>(a, P.a.pitch, ao[t], octets, P.depth, half, x[0][t]);
        octet<BD, false>(b, P.b.pitch, bo[t], octets, P.depth, half, y[0][t]);
      }
      if constexpr (D == 2) octet<BD, false>(b2, P.b.pitch, bo[0], octets, P.depth, half, y[0][N - 1]);
      mul(0);
    }
  };
  auto pass = [&](const float* a, const float* b, const float* b2) __attribute__((always_inline)) {
    if constexpr (OP == GATE)
      run(std::true_type{}, std::false_type{}, a, b, b2);
    else if constexpr (OP == GRAD)
      run(std::true_type{}, std::true_type{}, a, b, b2);
    else if (!P.aDeep)
      run(std::false_type{}, std::false_type{}, a, b, b2);
    else if (P.bDeep)
      run(std::true_type{}, std::true_type{}, a, b, b2);
    else
      run(std::true_type{}, std::false_type{}, a, b, b2);
  };
  pass(P.a.p, P.b.p, P.b2.p);
  if (OP == STORE && P.a2) pass(P.a2, P.b2.p, nullptr);
  float* out = P.out + (OP == STORE ? size_t(sp) * P.a.n * P.b.n : 0);
  if (OP == STORE && P.waves == 0) {  // nothing to add up (24 x 2048 x 8192 training 204 us through LDS, 186 without)
    if (first + w >= P.tiles) return;
#pragma unroll
    for (int bi = 0; bi < T; ++bi)
#pragma unroll
      for (int bj = 0; bj < T; ++bj) {
        const uint32_t c = (tj * T + bj) * 32 + col;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint32_t r = (ti * T + bi) * 32 + 8 * (e >> 2) + 4 * half + (e & 3);
          if (wanted(r) && c < P.b.n) out[size_t(r) * P.b.n + c] = acc[bi][bj][e];
        }
      }
    return;
  }
  // The waves' sums, block by block, a thread two values of each tile's.
#pragma unroll
  for (int b = 0; b < T * T; ++b) {
    if (b) __syncthreads();
#pragma unroll
    for (int d = 0; d < D; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) S[d][w][(8 * (e >> 2) + 4 * half + (e & 3)) * 32 + col] = acc[b / T][D == 2 ? d : b % T][e];
    __syncthreads();
    for (uint32_t i = 0; i < each; ++i) {
      if (OP != GRAD || i || b) at_of(i, b / T, b % T);
      float v[2][D];
      auto sum = [&](auto waves) __attribute__((always_inline)) {
        constexpr int W = decltype(waves)::value;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int d = 0; d < D; ++d) {
            v[h][d] = 0.f;
#pragma unroll
            for (int n = 0; n < W; ++n) v[h][d] += S[d][i * W + n][threadIdx.x + h * NW * 64];
          }
      };
      if (P.waves == 3)
        sum(std::integral_constant<int, 8>{});
      else if (P.waves == 2)
        sum(std::integral_constant<int, 4>{});
      else if (P.waves == 1)
        sum(std::integral_constant<int, 2>{});
      else
        sum(std::integral_constant<int, 1>{});
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (!in[h]) continue;
        if constexpr (OP == STORE) out[at[h]] = v[h][0];
        if constexpr (OP == GATE) {
          out[at[h]] = act<ACT>(v[h][0]) * v[h][D - 1];
          if (P.g) {
            P.g[at[h]] = v[h][0];
            P.u[at[h]] = v[h][D - 1];
          }
        }
        if constexpr (OP == GRAD) {
          float d;
          const float y = act_grad<ACT>(g[h], d);
          out[at[h]] = v[h][0] * u[h] * d;
          P.du[at[h]] = v[h][0] * y;
          P.m[at[h]] = y * u[h];
        }
      }
    }
  }
}

template <Op OP, MlpAct ACT, int T>
__global__ void __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(T == 2 ? 2 : 4, T == 2 ? 2 : 4))) k_mlp_small(const Prods all) {
  __shared__ SumsOf<OP> S;
  small_tiles<OP, ACT, T, false>(all, blockIdx.x, S, 0.f);
}

__global__ void __launch_bounds__(256) k_mlp_sum(const MlpSums t) {
  int k;
  uint32_t at;
  const f4u v = mlp_sum_of(t, blockIdx.x * 256 + threadIdx.x, &k, &at);
  if (k >= 0) stus<false>(t.s[k].out + at, v);
}
void mlp_sum(const MlpSums& t) {
  if (t.count) hipLaunchKernelGGL(k_mlp_sum, dim3(t.blocks), dim3(256), 0, stream(), t);
}

// The last launch of a call on parts: adds up the splits' sums, and works out again what the products
// marked, first m (dg, du and m), then the products of them.  Most often there is nothing marked, and
// the workgroups beyond those of the sums (all, of a call without splits: 3 us) end at once.  Else they
// take places one by one: a second product waits for all of the first ones, which have been taken by
// workgroups that run.
template <bool BWD>
struct Again {
  Prods first, second;
  MlpSums sums;
  MlpAgain g;
  uint32_t sumBlocks, n1, n2;  // workgroups for the sums; places of the first and the second products
  uint32_t cols;               // of y
  Waits waits;
};
template <bool BWD, MlpAct ACT>
__global__ void __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(4, 4))) k_mlp_again(const Again<BWD> t) {
  constexpr Op FIRST = BWD ? GRAD : GATE;
  __shared__ SumsOf<FIRST> S;
  __shared__ uint32_t mine;
  const uint32_t any = __hip_atomic_load(t.g.any, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (blockIdx.x < t.sumBlocks) {
    int k;
    uint32_t at;
    const f4u v = mlp_sum_of(t.sums, blockIdx.x * (kWaves * 64) + threadIdx.x, &k, &at);
    if (k < 0 || (BWD && any)) return;
    if (!any) {
      stus<false>(t.sums.s[k].out + at, v);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (!t.g.rows[(at + e) / t.cols]) t.sums.s[k].out[at + e] = v[e];
    }
    return;
  }
  if (!any) return;
  for (;;) {
    __syncthreads();
    if (threadIdx.x == 0) mine = __hip_atomic_fetch_add(t.g.counts, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const uint32_t id = __builtin_amdgcn_readfirstlane(mine);
    if (id >= t.n1 + t.n2) return;
    if (id < t.n1) {
      small_tiles<FIRST, ACT, 1, true>(t.first, id, S, 0.f);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "agent");
      __syncthreads();
      if (threadIdx.x == 0) __hip_atomic_fetch_add(t.g.counts + 1, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      continue;
    }
    auto done = [&] { return __hip_atomic_load(t.g.counts + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == t.n1; };
    bool there = done();
    for (uint32_t spin = 0; !there && spin < t.waits.spins; ++spin) {
      __builtin_amdgcn_s_sleep(8);
      there = done();
    }
    if (!there) t.waits.report();
    __syncthreads();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    small_tiles<STORE, kSilu, 1, true>(t.second, id - t.n1, reinterpret_cast<SumsOf<STORE>&>(S), there ? 0.f : NAN);
  }
}

// How the products of a launch share their depths, such that every wave has about as many
// octets (4096 waves are 16 for each CU, all that run at once); floats of what splits leave.
// More than a workgroup's eight waves for a tile only where each of those would have three times
// its share, or 12 octets: the sums are one more launch (training us without splits and with them,
// 20 x 2048 x 8192 384 and 205, 40 x 512 x 2048 67 and 44, 154 x 384 x 1001 54 and 46; from
// twice the share on, 300 x 256 x 512 35 for 33).
size_t share(Prods& t, bool split) {
  size_t floats = 0;
  auto octets = [](const Prod& p) { return (p.a2 ? 2.0 : 1.0) * p.depth / 8; };
  auto work = [&](uint32_t side) {  // of blocks of 32 x 32
    double all = 0;
    for (uint32_t i = 0; i < t.count; ++i) all += double(cdiv(t.p[i].a.n, 32 * side)) * cdiv(t.p[i].b.n, 32 * side) * side * side * octets(t.p[i]);
    return all;
  };
  // Tiles of 64 x 64, which halve the reads and are a quarter as many, from 64 octets of 32 x 32 for each
  // wave on, unless their edges are much more (training us with 32 and 64, 48 x 2048 x 8192 323 and
  // 284, 64 of them 344 and 311; from 16 octets on 64 x 1024 x 2816 89 for 81).
  t.side = split && work(1) >= 4096 * 64 && work(2) <= 1.15 * work(1) ? 2 : 1;
  const double all = work(t.side) / (t.side * t.side);
  for (uint32_t i = 0; i < t.count; ++i) {
    Prod& p = t.p[i];
    p.down = cdiv(p.a.n, 32 * t.side);
    p.tiles = p.down * cdiv(p.b.n, 32 * t.side);
  }
  const double most = std::max(1.0, all / 4096);
  for (uint32_t i = 0; i < t.count; ++i) {
    Prod& p = t.p[i];
    const double depth = octets(p), want = depth / std::max(most, 4.0);
    p.waves = 0;
    while ((1 << p.waves) < std::min<double>(depth / most, kWaves)) ++p.waves;
    const size_t n = size_t(p.a.n) * p.b.n;
    p.splits = split && n >= 4 && want > 3 * kWaves ? cdiv(uint64_t(want), kWaves) : 1;
    if (p.splits > 1) floats += (p.splits * n + 63) & ~size_t(63);
  }
  return floats;
}
// The products' first workgroups, and those of all of them.
uint32_t lay_out(Prods& t) {
  uint32_t n = 0;
  for (uint32_t i = 0; i < t.count; ++i) {
    t.p[i].start = n;
    n += cdiv(t.p[i].tiles, kWaves >> t.p[i].waves) * t.p[i].splits;
  }
  return n;
}
template <Op OP>
bool run_small(Prods& t, MlpAct act = kSilu, float* part = nullptr) {
  const uint32_t n = lay_out(t);
  MlpSums sums{};
  for (uint32_t i = 0; i < t.count; ++i) {
    Prod& p = t.p[i];
    if (p.splits == 1) continue;
    const size_t values = size_t(p.a.n) * p.b.n;
    sums.add(part, p.out, uint32_t(values), p.splits);
    p.out = part;
    part += (p.splits * values + 63) & ~size_t(63);
  }
  by_act(act, [&](auto k) {
    constexpr MlpAct A = OP == STORE ? kSilu : decltype(k)::value;
    if (OP == STORE && t.side == 2)
      hipLaunchKernelGGL((k_mlp_small<OP, A, OP == STORE ? 2 : 1>), dim3(n), dim3(kWaves * 64), 0, stream(), t);
    else
      hipLaunchKernelGGL((k_mlp_small<OP, A, 1>), dim3(n), dim3(kWaves * 64), 0, stream(), t);
  });
  mlp_sum(sums);
  return check_launch("gated_mlp");
}
Prod& add(Prods& t, const float* a, uint32_t rows, uint32_t aPitch, bool aDeep, const float* b, uint32_t cols, uint32_t bPitch, bool bDeep,
          uint32_t depth, float* out) {
  Prod& p = t.p[t.count++];
  p.a = {a, rows, aPitch};
  p.b = {b, cols, bPitch};
  p.depth = depth;
  p.aDeep = aDeep;
  p.bDeep = bDeep;
  p.out = out;
  return p;
}

// Floats of m, or of dg or du.
size_t third(const MlpArgs& a) { return (size_t(a.rows) * a.hidden + 63) & ~size_t(63); }

// y's product, whose m comes from the gate's.
Prods down_product(const MlpArgs& a) {
  Prods y{};
  add(y, nullptr, a.rows, a.hidden, true, a.wd, a.out, a.out, false, a.hidden, a.y);
  return y;
}
// The gate's, which leaves m.
Prods gate_product(const MlpArgs& a, float* m) {
  Prods t{};
  Prod& p = add(t, a.x, a.rows, a.cols, true, a.wg, a.hidden, a.hidden, false, a.cols, m);
  p.b2.p = a.wu;
  p.g = a.saved;
  p.u = a.saved ? a.saved + size_t(a.rows) * a.hidden : nullptr;
  share(t, false);
  return t;
}

bool forward_small(const MlpArgs& a) {
  const size_t at = third(a);
  Prods y = down_product(a);
  float* m = workspace(at + share(y, true));
  if (!m) return false;
  ProfScope prof("mlp", 6.0 * a.rows * a.cols * a.hidden, 4.0 * (2.0 * a.rows * a.cols + 3.0 * a.cols * a.hidden));
  Prods t = gate_product(a, m);
  if (!run_small<GATE>(t, a.act)) return false;
  y.p[0].a.p = m;
  return run_small<STORE>(y, kSilu, m + at);
}

// The four products that follow dm's; dg, du and m lie one after the other, `at` floats each (null: not yet).
Prods rest_products(const MlpArgs& a, const float* dy, float* dx, float* dwg, float* dwu, float* dwd, float* dg, size_t at) {
  float *du = dg ? dg + at : nullptr, *m = dg ? du + at : nullptr;
  Prods r{};
  if (dx) {
    Prod& q = add(r, dg, a.rows, a.hidden, true, a.wg, a.cols, a.hidden, true, a.hidden, dx);
    q.a2 = dg ? du : a.x;
    q.b2.p = a.wu;
  }
  if (dwd) add(r, m, a.hidden, a.hidden, false, dy, a.out, a.out, false, a.rows, dwd);
  if (dwg) add(r, a.x, a.cols, a.cols, false, dg, a.hidden, a.hidden, false, a.rows, dwg);
  if (dwu) add(r, a.x, a.cols, a.cols, false, du, a.hidden, a.hidden, false, a.rows, dwu);
  return r;
}
// dm's, which leaves dg, du and m.
Prods grad_product(const MlpArgs& a, const float* dy, float* dg, size_t at) {
  Prods t{};
  Prod& p = add(t, dy, a.rows, a.out, true, a.wd, a.hidden, a.out, true, a.out, dg);
  p.g = a.saved;
  p.u = a.saved + size_t(a.rows) * a.hidden;
  p.du = dg + at;
  p.m = p.du + at;
  share(t, false);
  return t;
}

bool backward_small(const MlpArgs& a, const float* dy, float* dx, float* dwg, float* dwu, float* dwd) {
  const size_t at = third(a);
  // Twice: how the products share first, their places once there is a workspace.
  Prods r = rest_products(a, dy, dx, dwg, dwu, dwd, nullptr, at);
  float* dg = workspace(3 * at + share(r, true));
  if (!dg) return false;
  r = rest_products(a, dy, dx, dwg, dwu, dwd, dg, at);
  share(r, true);
  ProfScope prof("mlp", 12.0 * a.rows * a.cols * a.hidden, 8.0 * (2.0 * a.rows * a.cols + 3.0 * a.cols * a.hidden));
  Prods t = grad_product(a, dy, dg, at);
  return run_small<GRAD>(t, a.act) && run_small<STORE>(r, kSilu, dg + 3 * at);
}

template <bool BWD>
bool run_again(Again<BWD>& t, MlpAct act) {
  share(t.second, false);
  t.first.again = t.second.again = t.g.rows;
  t.waits = g_waits;
  t.n1 = lay_out(t.first);
  t.n2 = lay_out(t.second);
  t.sumBlocks = (t.sums.blocks + 1) / 2;
  const uint32_t n = t.sumBlocks + std::min(t.n1 + t.n2, uint32_t(num_cus()));
  by_act(act, [&](auto k) { hipLaunchKernelGGL((k_mlp_again<BWD, decltype(k)::value>), dim3(n), dim3(kWaves * 64), 0, stream(), t); });
  return check_launch("gated_mlp");
}

// ---------------------------------------------------------------------------
// Up to 16 rows (new tokens): the weights are read once, on vector units.  A lane has one
// column (of each of Wg, Wu) and sums for all rows; a workgroup has 64 columns and a share
// of the depth, 128 k at a time, 16 for each of its 8 waves, all of whose loads are in
// flight at once.  Sums of the shares are left in memory and added up, in order, by what
// reads them: those of g and u by the second product's workgroups, each for its own
// share, those of y by a pass of its own.
//
// Bound by memory.  8 rows, 1024 x 2816: 8.7, 6.8 and 3.0 us for 34.6 MB of weights, a
// launch's own time each not far below that (on MFMAs as above 62 in all); 2048 x 8192:
// 41 us, 4.8 TB/s; 4096 x 11008: 122 us, 4.4 TB/s.  The next step's weights loaded ahead
// gained nothing: two workgroups a CU cover each other.
// ---------------------------------------------------------------------------
constexpr int kFew = 16, kFewWaves = 8, kFewDepth = 16 * kFewWaves;
struct Few {
  const float *x, *w, *w2;  // w2: Wu, or null
  float* part;              // [shares][1 or 2][rows][cols]
  uint32_t rows, depth, cols, blocks, steps, each;  // steps of 128 k in all, and of a share
  // second product: x from g's and u's sums of `shares` shares
  const float* gu;
  uint32_t shares;
  float *g, *u;  // kept (or null)
};
template <int R, bool FIRST, MlpAct ACT>
__global__ void __launch_bounds__(kFewWaves * 64) k_mlp_few(const Few a) {
  constexpr int T = kFewWaves * 64, D = FIRST ? 2 : 1, KW = kFewDepth / kFewWaves;
  __shared__ __attribute__((aligned(16))) float X[R][kFewDepth];
  __shared__ float S[kFewWaves][D * R * 64];
  const uint32_t share = blockIdx.x / a.blocks, block = blockIdx.x - share * a.blocks;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t c = block * 64 + lane, col = min(c, a.cols - 1);
  float acc[D][R];
#pragma unroll
  for (int d = 0; d < D; ++d)
#pragma unroll
    for (int r = 0; r < R; ++r) acc[d][r] = 0.f;
  const uint32_t end = min((share + 1) * a.each, a.steps);
  for (uint32_t step = share * a.each; step < end; ++step) {
    const uint32_t k0 = step * kFewDepth;
    float y[D][KW];
#pragma unroll
    for (int i = 0; i < KW; ++i) {
      const size_t at = size_t(min(k0 + w * KW + i, a.depth - 1)) * a.cols + col;
      y[0][i] = a.w[at];
      if constexpr (FIRST) y[D - 1][i] = a.w2[at];
    }
    if (step != share * a.each) __syncthreads();
    // The rows' values, zeros past the depth, as the weights' there.
    constexpr int EACH = (R * kFewDepth + T - 1) / T;
    float v[EACH];
    size_t at[EACH];
    bool in[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      const uint32_t t = threadIdx.x + j * T, r = t / kFewDepth, k = k0 + t % kFewDepth;
      in[j] = r < a.rows && k < a.depth;
      at[j] = size_t(in[j] ? r : 0) * a.depth + min(k, a.depth - 1);
      if constexpr (FIRST) v[j] = a.x[at[j]];
    }
    if constexpr (!FIRST) {
      const size_t n = size_t(a.rows) * a.depth;
      float g[EACH], u[EACH];
#pragma unroll
      for (int j = 0; j < EACH; ++j) g[j] = u[j] = 0.f;
      constexpr uint32_t U = EACH > 2 ? 2 : 4;  // shares in flight
      for (uint32_t s = 0; s < a.shares; s += U) {
        float p[EACH][U], q[EACH][U];
#pragma unroll
        for (uint32_t i = 0; i < U; ++i)
#pragma unroll
          for (int j = 0; j < EACH; ++j) {
            const size_t from = 2 * min(s + i, a.shares - 1) * n + at[j];
            p[j][i] = a.gu[from];
            q[j][i] = a.gu[from + n];
          }
#pragma unroll
        for (uint32_t i = 0; i < U; ++i)
#pragma unroll
          for (int j = 0; j < EACH; ++j) {
            g[j] += s + i < a.shares ? p[j][i] : 0.f;
            u[j] += s + i < a.shares ? q[j][i] : 0.f;
          }
      }
#pragma unroll
      for (int j = 0; j < EACH; ++j) {
        v[j] = act<ACT>(g[j]) * u[j];
        if (a.g && block == 0 && in[j]) {
          a.g[at[j]] = g[j];
          a.u[at[j]] = u[j];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      const uint32_t t = threadIdx.x + j * T;
      if (R * kFewDepth >= T || t < R * kFewDepth) X[t / kFewDepth][t % kFewDepth] = in[j] ? v[j] : 0.f;
    }
    __syncthreads();
    if (k0 + kFewDepth > a.depth) {
#pragma unroll
      for (int i = 0; i < KW; ++i)
#pragma unroll
        for (int d = 0; d < D; ++d) y[d][i] = k0 + w * KW + i < a.depth ? y[d][i] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < KW; i += 4)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const f4 x = *reinterpret_cast<const f4*>(&X[r][w * KW + i]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int d = 0; d < D; ++d) acc[d][r] = fmaf(x[e], y[d][i + e], acc[d][r]);
      }
  }
#pragma unroll
  for (int d = 0; d < D; ++d)
#pragma unroll
    for (int r = 0; r < R; ++r) S[w][(d * R + r) * 64 + lane] = acc[d][r];
  __syncthreads();
  for (int t = threadIdx.x; t < D * R * 64; t += T) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < kFewWaves; ++i) v += S[i][t];
    const uint32_t d = t / (R * 64), r = t / 64 % R, n = block * 64 + t % 64;
    if (r < a.rows && n < a.cols) a.part[((size_t(share) * D + d) * a.rows + r) * a.cols + n] = v;
  }
}
__global__ void __launch_bounds__(256) k_mlp_few_sum(const float* part, float* y, uint32_t n, uint32_t shares) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float v = 0.f;
#pragma unroll 8
  for (uint32_t s = 0; s < shares; ++s) v += part[size_t(s) * n + i];
  y[i] = v;
}

bool forward_few(const MlpArgs& a) {
  Few f{}, s{};
  auto size = [](Few& t, uint32_t depth, uint32_t cols) {
    t.depth = depth;
    t.cols = cols;
    t.blocks = cdiv(cols, 64);
    t.steps = cdiv(depth, kFewDepth);
    // Some 512 workgroups, two a CU, and shares of 128 k only where there are fewer than one:
    // what shares leave has to be read again (16 rows of 2048 x 8192: 76 us with shares of 128
    // everywhere, 64 with 1024 workgroups, 53 with 512, 68 with 256; 8 of 1024 x 2816: 19.4 with
    // shares of 128, 17.5 of 256, 19.3 of 384; of 512 x 2048: 11.2, 13.8, 18.4).
    const uint32_t all = t.blocks * t.steps;
    t.each = all <= 256 ? 1 : std::max(2u, cdiv(t.steps, cdiv(512, t.blocks)));
    return cdiv(t.steps, t.each);
  };
  const uint32_t s1 = size(f, a.cols, a.hidden), s2 = size(s, a.hidden, a.out);
  const size_t gu = 2 * size_t(s1) * a.rows * a.hidden, ny = size_t(s2) * a.rows * a.out;
  float* ws = workspace(((gu + 63) & ~size_t(63)) + (s2 > 1 ? ny : 0));
  if (!ws) return false;
  float* part = s2 > 1 ? ws + ((gu + 63) & ~size_t(63)) : a.y;
  ProfScope prof("mlp", 6.0 * a.rows * a.cols * a.hidden, 4.0 * (2.0 * a.rows * a.cols + 3.0 * a.cols * a.hidden));
  f.x = a.x;
  f.w = a.wg;
  f.w2 = a.wu;
  f.part = ws;
  f.rows = a.rows;
  s.w = a.wd;
  s.part = part;
  s.rows = a.rows;
  s.gu = ws;
  s.shares = s1;
  s.g = a.saved;
  s.u = a.saved ? a.saved + size_t(a.rows) * a.hidden : nullptr;
  auto run = [&](auto rows) {
    constexpr int R = decltype(rows)::value;
    hipLaunchKernelGGL((k_mlp_few<R, true, kSilu>), dim3(f.blocks * s1), dim3(kFewWaves * 64), 0, stream(), f);
    by_act(a.act, [&](auto k) {
      hipLaunchKernelGGL((k_mlp_few<R, false, decltype(k)::value>), dim3(s.blocks * s2), dim3(kFewWaves * 64), 0, stream(), s);
    });
  };
  if (a.rows == 1)
    run(std::integral_constant<int, 1>{});
  else if (a.rows <= 4)
    run(std::integral_constant<int, 4>{});
  else if (a.rows <= 8)
    run(std::integral_constant<int, 8>{});
  else
    run(std::integral_constant<int, 16>{});
  if (s2 > 1)
    hipLaunchKernelGGL(k_mlp_few_sum, dim3(cdiv(a.rows * a.out, 256)), dim3(256), 0, stream(), part, a.y, a.rows * a.out, s2);
  return check_launch("GatedMlpForward");
}

}  // namespace

bool mlp_forward_again(const MlpArgs& a, const MlpAgain& g, const MlpSums& sums) {
  Again<false> t{};
  t.first = gate_product(a, g.ws);
  t.second = down_product(a);
  t.second.p[0].a.p = g.ws;
  t.sums = sums;
  t.g = g;
  t.cols = a.out;
  return run_again(t, a.act);
}
size_t mlp_again_floats(const MlpArgs& a) { return 3 * third(a); }
bool mlp_backward_again(const MlpArgs& a, const float* dy, float* dx, float* dwg, float* dwu, float* dwd, const MlpAgain& g, const MlpSums& sums) {
  Again<true> t{};
  t.first = grad_product(a, dy, g.ws, third(a));
  t.second = rest_products(a, dy, dx, dwg, dwu, dwd, g.ws, third(a));
  t.sums = sums;
  t.g = g;
  return run_again(t, a.act);
}

bool mlp_forward(const MlpArgs& a) {
  if (a.rows <= uint32_t(kFew)) return forward_few(a);
  return mlp_on_parts(a, false) ? mlp_forward_parts(a) : forward_small(a);
}

bool mlp_backward(const MlpArgs& a, const float* dy, float* dx, float* dwg, float* dwu, float* dwd) {
  return mlp_on_parts(a, true) ? mlp_backward_parts(a, dy, dx, dwg, dwu, dwd) : backward_small(a, dy, dx, dwg, dwu, dwd);
}

}  // namespace dce
