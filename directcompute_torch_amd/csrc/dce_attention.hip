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
#include "dce_attention_fp32.h"

namespace dce {

namespace {

constexpr int kT = 256;   // threads: four waves
constexpr int kFew = 64;  // keys of a tile in the kernel for few rows

template <int DP, bool VEC>
__global__ void __launch_bounds__(kT) k_attn_fwd(const Attn a) {
  __shared__ __attribute__((aligned(16))) float Ks[kKeys * DP], Vs[kKeys * DP];
  const uint32_t prob = a.B * a.G, rest = blockIdx.x / prob, pr = blockIdx.x - rest * prob;
  const uint32_t back = rest / a.splits, sp = rest - back * a.splits;
  fwd_fp32<DP, VEC>(a, pr, (a.tiles - 1 - back) * 64, sp, Ks, Vs);
}
template <int DP, bool VEC>
__global__ void __launch_bounds__(kT) k_attn_dq(const Attn a) {
  __shared__ __attribute__((aligned(16))) float Ks[kKeys * DP], Vs[kKeys * DP];
  const uint32_t prob = a.B * a.G, rest = blockIdx.x / prob, pr = blockIdx.x - rest * prob;
  const uint32_t back = rest / a.splits, sp = rest - back * a.splits;
  dq_fp32<DP, VEC, kT>(a, pr, (a.tiles - 1 - back) * 64, sp, Ks, Vs);
}
template <int DP, bool VEC>
__global__ void __launch_bounds__(kT) k_attn_dkv(const Attn a) {
  __shared__ __attribute__((aligned(16))) float Qs[kKeys * DP], Ys[kKeys * DP], St[3 * kKeys];
  __shared__ uint32_t Lim[kKeys];
  const uint32_t prob = a.B * a.G, rest = blockIdx.x / prob, pr = blockIdx.x - rest * prob;
  const uint32_t tile = rest / a.splits, sp = rest - tile * a.splits;
  dkv_fp32<DP, VEC, kT>(a, pr, tile * 64, sp, Qs, Ys, St, Lim);
}

// Gradients from the splits' shares (`values` of each, in a row), added in order;
// V: f4 or float.
template <typename V>
__global__ void __launch_bounds__(kT)
    k_attn_sum(const V* pk, V* dk, const V* pv, V* dv, size_t values, uint32_t splits) {
  const size_t i = size_t(blockIdx.x) * kT + threadIdx.x;
  if (i >= values) return;
  V x = pk[i], y = dv ? pv[i] : x;
#pragma unroll 4
  for (uint32_t s = 1; s < splits; ++s) {
    x += pk[s * values + i];
    if (dv) y += pv[s * values + i];
  }
  dk[i] = x;
  if (dv) dv[i] = y;
}

// ---------------------------------------------------------------------------
// Forward of up to 16 rows (a new token or a few, all heads of a key head): bound
// by reading K and V once.  Tiles of 64 keys, 16 to each wave, which keeps sums of
// its own; the four waves' are joined at the end.  In the general kernel one wave
// would multiply for all four: 8 sequences of up to 8191 keys, 8 key heads of 128,
// took 114 us there and take 81 here (5.2 TB/s; 87 without streaming loads).
// Operands straight from memory, without LDS, took 155 us: the K fragment's 64
// bytes of each of 16 rows keep the address unit busy.
// ---------------------------------------------------------------------------
template <int DP, bool VEC, bool NT>
__global__ void __launch_bounds__(kT, DP <= 128 ? 2 : 1) k_attn_few(const Attn a) {
  using CL = Cols<DP>;
  using TL = Tile<DP, kFew, VEC, kT>;
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
  f4 q[NI], o[NI];
  load_frag<DP, VEC>(a.q + q_at(a, b, gh, min(n, a.N - 1)), true, a.D, g, q);
#pragma unroll
  for (int i = 0; i < NI; ++i) o[i] = f4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  const uint32_t stride = a.G * a.D, j0 = sp * a.perSplit * kFew, j1 = min(most, (sp + 1) * a.perSplit * kFew);
  f4 rk[TL::LOADS], rv[TL::LOADS];
  auto fetch = [&](uint32_t j) {
    const uint32_t n = min(len - j, uint32_t(kFew));
    TL::template load<NT>(rows_view(a.k + k_at(a, b, gh, j), n, stride, a.D), stride, a.D, rk);
    TL::template load<NT>(rows_view(a.v + k_at(a, b, gh, j), n, stride, a.D), stride, a.D, rv);
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
    f4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const f4 kf = TL::chunk(Ks, wave * 16 + col, 4 * i + g);
#pragma unroll
      for (int e = 0; e < 4; ++e) s = mfma4(kf[e], q[i][e], s);
    }
    float top = -INFINITY;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      s[r] = scaled(s[r], a.c);
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

// Joins the key splits: a row per `lanes` threads of a wave, 4 values each (or, of
// dims that are no multiple of 4, one at a time).  ONE: a row per workgroup, for
// few rows: its statistics are then scalar loads (256 rows of 128 in 16 splits 4.9
// us, two rows to a wave 6.8).
template <bool VEC, bool ONE>
__global__ void __launch_bounds__(64) k_attn_join(const Attn a, uint32_t lanes) {
  const uint32_t own = ONE ? 0 : threadIdx.x / lanes, lane = threadIdx.x - own * lanes, rows = a.B * a.G * a.N;
  const uint32_t row = ONE ? blockIdx.x : blockIdx.x * (64 / lanes) + own;
  if (!ONE && (own >= 64 / lanes || row >= rows)) return;
  const uint32_t pr = row / a.N, n = row - pr * a.N, b = fdiv(pr, a.dG), g = pr - b * a.G;
  const bool none = limit_of(a, n, keys_of(a, b)) == 0;
  float m = -INFINITY;
#pragma unroll 8
  for (uint32_t s = 0; s < a.splits; ++s) m = fmaxf(m, a.pm[size_t(s) * rows + row]);
  const float base = m == -INFINITY ? 0.f : m;
  constexpr uint32_t W = VEC ? 4 : 1;
  using V = float __attribute__((ext_vector_type(W)));
  for (uint32_t d = lane * W; d < a.D; d += (ONE ? 64 : lanes) * W) {
    float l = 0.f;
    V o = {};
#pragma unroll 8
    for (uint32_t s = 0; s < a.splits; ++s) {
      const size_t i = size_t(s) * rows + row;
      const float w = exp2_(a.pm[i] - base);
      l += w * a.pl[i];
      o += w * *reinterpret_cast<const V*>(a.po + i * a.D + d);
    }
    const float il = none ? 0.f : 1.f / l;
    if (a.m && d == 0) {
      a.m[row] = none ? 0.f : m;
      a.il[row] = il;
    }
    *reinterpret_cast<V*>(a.o + q_at(a, b, g, n) + d) = none ? V{} : o * il;
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
    const uint32_t cus = uint32_t(num_cus()), prob = a.B * a.G;
    const bool few = a.N <= 16;
    a.tiles = cdiv(a.N, 64);
    const uint32_t kt = cdiv(a.T, few ? kFew : kKeys);
    a.splits = 1;
    if (few)
      a.splits = std::max(1u, std::min(cdiv(kt, 4), 4 * cus / prob));
    else if (uint64_t(a.tiles) * prob < cus) {
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
    if (few && stream_nt(8.0 * a.B * a.T * a.G * a.D))
      hipLaunchKernelGGL((k_attn_few<DP, VEC, true>), grid, dim3(kT), 0, stream(), a);
    else if (few)
      hipLaunchKernelGGL((k_attn_few<DP, VEC, false>), grid, dim3(kT), 0, stream(), a);
    else
      hipLaunchKernelGGL((k_attn_fwd<DP, VEC>), grid, dim3(kT), 0, stream(), a);
    if (!check_launch("AttentionForward")) return false;
    return a.splits == 1 || attn_join(a);
  }
};

struct BwdRun {
  Attn a;
  float* more;  // the splits' shares
  template <int DP, bool VEC>
  bool run() {
    const uint32_t prob = a.B * a.G;
    Attn q = a;
    q.tiles = cdiv(a.N, 64);
    q.splits = a.dq ? key_splits(a, 64) : 1;
    if (q.splits > 1) q.dq = more;
    const dim3 grid(q.tiles * q.splits * prob);
    hipLaunchKernelGGL((k_attn_dq<DP, VEC>), grid, dim3(kT), 0, stream(), q);
    if (!check_launch("AttentionBackward (dQ)")) return false;
    if (q.splits > 1 && !attn_sum(q.dq, a.dq, nullptr, nullptr, size_t(prob) * a.N * a.D, q.splits)) return false;
    if (!a.dk && !a.dv) return true;
    const size_t values = size_t(a.B) * a.T * a.G * a.D;
    Attn d = a;
    d.tiles = cdiv(a.T, 64);
    d.splits = row_splits(a, 64);
    if (d.splits > 1) {
      if (a.dk) d.dk = more;
      if (a.dv) d.dv = more + d.splits * values;
    }
    hipLaunchKernelGGL((k_attn_dkv<DP, VEC>), dim3(d.tiles * d.splits * prob), dim3(kT), 0, stream(), d);
    return check_launch("AttentionBackward (dK, dV)") &&
           (d.splits == 1 || attn_sum(d.dk, a.dk, d.dv, a.dv, values, d.splits));
  }
};

}  // namespace

bool attn_join(const Attn& a) {
  const bool vec = a.D % 4 == 0;
  const uint32_t lanes = vec ? a.D / 4 : std::min(64u, a.D);
  const uint32_t rows = a.B * a.G * a.N;
  const bool one = rows <= 4 * uint32_t(num_cus());
  const dim3 grid(one ? rows : cdiv(rows, 64 / lanes));
  if (vec && one)
    hipLaunchKernelGGL((k_attn_join<true, true>), grid, dim3(64), 0, stream(), a, lanes);
  else if (vec)
    hipLaunchKernelGGL((k_attn_join<true, false>), grid, dim3(64), 0, stream(), a, lanes);
  else if (one)
    hipLaunchKernelGGL((k_attn_join<false, true>), grid, dim3(64), 0, stream(), a, lanes);
  else
    hipLaunchKernelGGL((k_attn_join<false, false>), grid, dim3(64), 0, stream(), a, lanes);
  return check_launch("AttentionForward (join)");
}

bool attn_sum(const float* p0, float* out0, const float* p1, float* out1, size_t n, uint32_t splits) {
  if (!out0) {
    p0 = p1;
    out0 = out1;
    out1 = nullptr;
  }
  if (n % 4 == 0)
    hipLaunchKernelGGL(k_attn_sum<f4>, dim3(cdiv(n / 4, kT)), dim3(kT), 0, stream(), reinterpret_cast<const f4*>(p0),
                       reinterpret_cast<f4*>(out0), reinterpret_cast<const f4*>(p1), reinterpret_cast<f4*>(out1),
                       n / 4, splits);
  else
    hipLaunchKernelGGL(k_attn_sum<float>, dim3(cdiv(n, kT)), dim3(kT), 0, stream(), p0, out0, p1, out1, n, splits);
  return check_launch("AttentionBackward (splits)");
}

bool attention_forward(const AttnArgs& x) {
  ProfScope prof("attention", 4.0 * x.D * x.B * x.H * pairs_of(x),
                 4.0 * x.D * (2.0 * x.B * x.S * x.H + 2.0 * x.B * x.T * x.G));
  const Attn a = params(x);
  bool took = false;
  return attn_fwd_parts(x, a, &took) && (took || by_dim(a.D, a.D % 4 == 0, FwdRun{a}));
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
  const size_t rows = (size_t(x.B) * x.H * x.S + 63) & ~size_t(63);
  a.delta = workspace(rows + split_floats(a, 64, 64));
  return a.delta && by_dim(a.D, a.D % 4 == 0, BwdRun{a, a.delta + rows});
}

}  // namespace dce
