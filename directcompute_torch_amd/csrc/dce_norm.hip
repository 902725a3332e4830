// The norms around a block's residual stream, in one pass over a row:
//
//   u = post ? block r1 post : block,       r1 = 1 / sqrt(mean(block^2) + eps)
//   h = scale x + gate u,                   gate: a row for each `per` rows, or none
//   n = h r2 pre,                           r2 = 1 / sqrt(mean(h^2) + eps)
//
// and, from dh and dn,
//
//   t = dh + r2 (pre dn - h r2^2 mean(pre dn h)),   dx = scale t,   du = gate t,
//   dblock = r1 (post du - block r1^2 mean(post du block)),
//   dgate = sum t u,  dpost = sum du block r1,  dpre = sum dn h r2.
//
// The plain norm (y = x r2 pre) is the same without a block.
//
// A row lies in the registers of `TPR` threads, in quads of 4 values.  A width
// that is no multiple of 4 has its last quad end with the row, so that some of
// its values are the quad's before it too: they are computed twice, to the same
// bits, and left out of the sums.
//
// Bound by memory.  8192 x 2048, a gate for each channel: forward (16 bytes a value) 44
// to 48 us, 6.1 to 5.6 TB/s; backward (24) 74 us, 5.4 TB/s, and 6 us for the sums over rows.  8191 x
// 4096 with a gate for each value: 97 and 170 us, 6.9 and 6.3 TB/s.  Passes over more
// than the last cache go past it (nontemporal), which is worth 20 to 25 % there.  The
// next row's loads ahead of time, and gains held in registers, gained nothing.
#include "dce_internal.h"

#include <algorithm>

namespace dce {

namespace {

inline uint32_t cdiv(uint64_t a, uint64_t b) { return uint32_t((a + b - 1) / b); }

struct Norm {
  const float *x, *block, *gate, *post, *pre;
  float *h, *n, *r1, *r2;  // r1, r2: null where not kept
  const float *dh, *dn;
  float *dx, *db, *dgate, *dpost, *dpre;  // dgate .. dpre: partial sums of the workgroups
  uint32_t rows, cols;
  uint32_t first;   // of this launch's rows (forward)
  uint32_t per;     // rows of a gate row
  uint32_t each;    // every row has a gate row of its own (per then counts all rows)
  uint32_t pieces;  // workgroups of a gate row's rows (backward)
  uint32_t groups;  // gate rows of a workgroup (backward)
  float scale, eps;
};

// W values of a row from column c on, of which the first `dup` belong to the quad
// before, too; none where c lies past the row.
template <int W>
struct Span {
  uint32_t at;
  int dup;  // W: nothing
  __device__ __forceinline__ void init(uint32_t c, uint32_t cols) {
    at = min(c, cols - W);
    dup = int(min(c - at, uint32_t(W)));
  }
  template <bool NT = false>
  __device__ __forceinline__ void load(const float* row, float* v) const {
    if constexpr (W == 4) {
      const f4u q = ldus<NT, f4u>(row + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = q[e];
    } else {
      v[0] = ldus<NT, float>(row + at);
    }
  }
  template <bool NT = false>
  __device__ __forceinline__ void store(float* row, const float* v) const {
    if (dup == W) return;
    if constexpr (W == 4) {
      stus<NT>(row + at, f4u{v[0], v[1], v[2], v[3]});
    } else {
      stus<NT>(row + at, v[0]);
    }
  }
};

// Sum over the TPR threads of a row, in every one of them.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* sh) {
  if constexpr (TPR < 64) {
    v = group8_reduce(v);
    v += xl::dpp<xl::kRowMirror>(v);
    if constexpr (TPR == 32) v += xl::swz(v);
    return v;
  }
  v = wave_reduce(v);
  if constexpr (TPR > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) v += sh[i];
  }
  return v;
}

// 1 / sqrt(mean of a row's squares + eps).  Rows whose squares would leave fp32's range (and, where eps
// does not hide it, fall below it) are added up scaled.
template <int TPR, int NV, int W>
__device__ __forceinline__ float inv_rms(const Span<W> (&s)[NV], const float (&v)[NV][W], uint32_t cols, float eps, float* sh) {
  auto squares = [&](float by) {
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const float x = v[j][e] * by;
        sum += e >= s[j].dup ? x * x : 0.f;
      }
    return row_sum<TPR>(sum, sh);
  };
  float sum = squares(1.f), by = 1.f;
  if (!(sum < 0x1p120f)) by = 0x1p-64f;
  if (sum < 0x1p-70f && eps < 0x1p-70f) by = 0x1p64f;
  if (by != 1.f) sum = squares(by);
  return by / sqrtf(sum / float(cols) + eps * by * by);
}

template <int TPR>
constexpr int threads_of = TPR < 256 ? 256 : TPR;

template <int TPR, int NV, int W, bool NT>
__global__ void __launch_bounds__(threads_of<TPR>) k_norm_fwd(const Norm a) {
  constexpr int T = threads_of<TPR>, RPB = T / TPR;
  __shared__ float sh[T / 64];
  const uint32_t lane = threadIdx.x % TPR, row = a.first + blockIdx.x * RPB + threadIdx.x / TPR;
  if (RPB > 1 && row >= a.rows) return;
  const size_t base = size_t(row) * a.cols;
  Span<W> s[NV];
  float x[NV][W], b[NV][W], t[W];
#pragma unroll
  for (int j = 0; j < NV; ++j) s[j].init((j * TPR + lane) * W, a.cols);
#pragma unroll
  for (int j = 0; j < NV; ++j) s[j].template load<NT>(a.x + base, x[j]);
  if (a.block) {
#pragma unroll
    for (int j = 0; j < NV; ++j) s[j].template load<NT>(a.block + base, b[j]);
    if (a.post) {
      const float r = inv_rms<TPR>(s, b, a.cols, a.eps, sh);
      if (a.r1 && lane == 0) a.r1[row] = r;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        s[j].load(a.post, t);
#pragma unroll
        for (int e = 0; e < W; ++e) b[j][e] = b[j][e] * r * t[e];
      }
    }
    const float* gate = a.gate ? a.gate + size_t(a.each ? row : row / a.per) * a.cols : nullptr;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (gate) {
        s[j].load(gate, t);
#pragma unroll
        for (int e = 0; e < W; ++e) x[j][e] = a.scale * x[j][e] + t[e] * b[j][e];
      } else {
#pragma unroll
        for (int e = 0; e < W; ++e) x[j][e] = a.scale * x[j][e] + b[j][e];
      }
      s[j].template store<NT>(a.h + base, x[j]);
    }
  }
  if (!a.n) return;
  const float r = inv_rms<TPR>(s, x, a.cols, a.eps, sh);
  if (a.r2 && lane == 0) a.r2[row] = r;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    s[j].load(a.pre, t);
#pragma unroll
    for (int e = 0; e < W; ++e) x[j][e] = x[j][e] * r * t[e];
    s[j].template store<NT>(a.n + base, x[j]);
  }
}

// Rows of a workgroup: `groups` whole gate rows, or the piece blockIdx % pieces of
// one.  The sums over rows stay in registers until the last one; a workgroup
// leaves one row of each in dpost and dpre, and one of dgate for each gate row it
// has rows of.
template <int TPR, int NV, int W, bool NT>
__global__ void __launch_bounds__(threads_of<TPR>) k_norm_bwd(const Norm a) {
  constexpr int T = threads_of<TPR>, RPB = T / TPR;
  __shared__ float sh[T / 64];
  __shared__ float acc[RPB > 1 ? RPB * TPR * NV * W : 1];
  const uint32_t lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const uint32_t gates = (a.rows + a.per - 1) / a.per;
  const uint32_t g0 = a.pieces > 1 ? blockIdx.x / a.pieces : blockIdx.x * a.groups;
  const uint32_t g1 = a.pieces > 1 ? g0 + 1 : min(g0 + a.groups, gates);
  const uint32_t piece = a.pieces > 1 ? blockIdx.x % a.pieces : 0;
  Span<W> s[NV];
  float dpost[NV][W], dpre[NV][W], dgate[NV][W];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    s[j].init((j * TPR + lane) * W, a.cols);
#pragma unroll
    for (int e = 0; e < W; ++e) dpost[j][e] = dpre[j][e] = 0.f;
  }
  const float inv = 1.f / float(a.cols);
  auto fetch = [&](uint32_t row, float (&t)[NV][W], float (&h)[NV][W], float (&w)[NV][W], float (&b)[NV][W]) {
    const size_t base = size_t(row) * a.cols;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (a.dh) {
        s[j].template load<NT>(a.dh + base, t[j]);
      } else {
#pragma unroll
        for (int e = 0; e < W; ++e) t[j][e] = 0.f;
      }
      if (a.dn) {
        s[j].template load<NT>(a.h + base, h[j]);
        s[j].template load<NT>(a.dn + base, w[j]);
      }
      if (a.post || a.dgate) s[j].template load<NT>(a.block + base, b[j]);
    }
  };
  // The threads' sums to one row of `to`.
  auto put = [&](float (&v)[NV][W], float* to) {
    if constexpr (RPB > 1) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < W; ++e) acc[((j * W + e) * RPB + sub) * TPR + lane] = v[j][e];
      __syncthreads();
      if (sub) return;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < W; ++e) {
          v[j][e] = 0.f;
#pragma unroll
          for (int i = 0; i < RPB; ++i) v[j][e] += acc[((j * W + e) * RPB + i) * TPR + lane];
        }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) s[j].store(to, v[j]);
  };
  for (uint32_t g = g0; g < g1; ++g) {
    const uint64_t first = uint64_t(g) * a.per, have = min(uint64_t(a.per), a.rows - first);
    const uint32_t r0 = uint32_t(first + have * piece / a.pieces), r1 = uint32_t(first + have * (piece + 1) / a.pieces);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < W; ++e) dgate[j][e] = 0.f;
    // Every thread of the workgroup goes through the same number of rounds.
    for (uint32_t at = r0; at < r1; at += RPB) {
      const uint32_t row = min(at + sub, r1 - 1);
      const bool live = at + sub < r1;
      const size_t base = size_t(row) * a.cols;
      const float* gate = a.gate ? a.gate + (a.each ? base : size_t(g) * a.cols) : nullptr;
      float t[NV][W], h[NV][W], b[NV][W], w[NV][W], gain[W];
      fetch(row, t, h, w, b);
      if (a.dn) {
        const float r = a.r2[row];
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          s[j].load(a.pre, gain);
#pragma unroll
          for (int e = 0; e < W; ++e) {
            if (live) dpre[j][e] += w[j][e] * h[j][e] * r;
            w[j][e] *= gain[e];
            sum += e >= s[j].dup ? w[j][e] * h[j][e] : 0.f;
          }
        }
        const float m = row_sum<TPR>(sum, sh) * inv * r * r;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int e = 0; e < W; ++e) t[j][e] += r * (w[j][e] - h[j][e] * m);
      }
      if (a.dx && live) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
          for (int e = 0; e < W; ++e) w[j][e] = a.scale * t[j][e];
          s[j].template store<NT>(a.dx + base, w[j]);
        }
      }
      if (!a.db && !a.dgate && !a.dpost) continue;
      const float r = a.post ? a.r1[row] : 1.f;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float gt[W];
#pragma unroll
        for (int e = 0; e < W; ++e) gain[e] = gt[e] = 1.f;
        if (a.post) s[j].load(a.post, gain);
        if (gate) s[j].load(gate, gt);
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const float bn = (a.post || a.dgate) ? b[j][e] * r : 0.f;
          if (a.each)
            dgate[j][e] = t[j][e] * bn * gain[e];
          else if (live)
            dgate[j][e] += t[j][e] * bn * gain[e];
          w[j][e] = gt[e] * t[j][e];
          if (live) dpost[j][e] += w[j][e] * bn;
          w[j][e] *= gain[e];
          if (a.post) sum += e >= s[j].dup ? w[j][e] * b[j][e] : 0.f;
        }
      }
      if (a.each && a.dgate && live) {
#pragma unroll
        for (int j = 0; j < NV; ++j) s[j].store(a.dgate + base, dgate[j]);
      }
      if (a.post) {
        const float m = row_sum<TPR>(sum, sh) * inv * r * r;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int e = 0; e < W; ++e) w[j][e] = r * (w[j][e] - b[j][e] * m);
      }
      if (a.db && live) {
#pragma unroll
        for (int j = 0; j < NV; ++j) s[j].template store<NT>(a.db + base, w[j]);
      }
    }
    if (a.dgate && !a.each) put(dgate, a.dgate + (size_t(g) * a.pieces + piece) * a.cols);
  }
  if (a.dpost) put(dpost, a.dpost + size_t(blockIdx.x) * a.cols);
  if (a.dpre) put(dpre, a.dpre + size_t(blockIdx.x) * a.cols);
}

// out[g][c] = sum over i < count of part[g][i][c], in order; up to three sums.
struct Cols {
  const float* part[3];
  float* out[3];
  uint32_t count[3], groups[3];
  uint32_t cols, blocks;  // blocks: of 64 columns
};
constexpr int kColWaves = 16;
__global__ void __launch_bounds__(kColWaves * 64) k_norm_cols(const Cols a) {
  __shared__ float sh[kColWaves][64];
  uint32_t id = blockIdx.x;
  int k = 0;
  while (id >= a.blocks * a.groups[k]) id -= a.blocks * a.groups[k++];
  const uint32_t g = id / a.blocks, lane = threadIdx.x & 63, c = id % a.blocks * 64 + lane, w = threadIdx.x >> 6;
  const uint32_t n = a.count[k], lo = n * w / kColWaves, hi = n * (w + 1) / kColWaves;
  float v = 0.f;
  if (c < a.cols) {
    const float* p = a.part[k] + size_t(g) * n * a.cols + c;
    float part[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    uint32_t i = lo;
    for (; i + 8 <= hi; i += 8)
#pragma unroll
      for (int e = 0; e < 8; ++e) part[e] += p[size_t(i + e) * a.cols];
    for (; i < hi; ++i) v += p[size_t(i) * a.cols];
#pragma unroll
    for (int e = 0; e < 8; ++e) v += part[e];
  }
  sh[w][lane] = v;
  __syncthreads();
  if (w || c >= a.cols) return;
  v = 0.f;
#pragma unroll
  for (int i = 0; i < kColWaves; ++i) v += sh[i][lane];
  a.out[k][size_t(g) * a.cols + c] = v;
}

// f.run<TPR, NV, W>() for a width.
template <class F>
bool dispatch(uint32_t cols, const F& f) {
  if (cols < 4) return f.template run<16, 1, 1>();
  if (cols <= 64) return f.template run<16, 1, 4>();
  if (cols <= 128) return f.template run<32, 1, 4>();
  if (cols <= 256) return f.template run<64, 1, 4>();
  if (cols <= 512) return f.template run<64, 2, 4>();
  if (cols <= 1024) return f.template run<256, 1, 4>();
  if (cols <= 2048) return f.template run<256, 2, 4>();
  if (cols <= 4096) return f.template run<512, 2, 4>();
  if (cols <= 8192) return f.template run<512, 4, 4>();
  return f.template run<1024, 4, 4>();
}

struct Fwd {
  Norm& a;
  bool nt;
  template <int TPR, int NV, int W>
  bool run() const {
    constexpr int T = threads_of<TPR>, RPB = T / TPR;
    constexpr uint32_t most = 1u << 21;  // workgroups: fewer than 2^32 threads in a launch
    for (uint64_t first = 0; first < a.rows; first += uint64_t(most) * RPB) {
      a.first = uint32_t(first);
      hipLaunchKernelGGL((nt ? k_norm_fwd<TPR, NV, W, true> : k_norm_fwd<TPR, NV, W, false>),
                         dim3(std::min(cdiv(a.rows - first, RPB), most)), dim3(T), 0, stream(), a);
    }
    return check_launch("norm");
  }
};

struct Bwd {
  Norm& a;
  const NormGrads& g;
  bool nt;
  template <int TPR, int NV, int W>
  bool run() const {
    constexpr int T = threads_of<TPR>, RPB = T / TPR;
    // 1024 threads a CU: more leave more partial sums, fewer less in flight (8192 x 2048:
    // 84 us with 512 or 1024, 94 with 1536, 88 with 2048; 4096 x 8192: 169, 173, 193, 185).
    const uint32_t gates = cdiv(a.rows, a.per), want = std::min(cdiv(a.rows, RPB), uint32_t(num_cus()) * 1024 / T);
    uint32_t wgs;
    if (gates >= want) {
      a.pieces = 1;
      a.groups = cdiv(gates, want);
      wgs = cdiv(gates, a.groups);
    } else {
      a.groups = 1;
      a.pieces = std::max(1u, std::min(cdiv(want, gates), cdiv(a.per, RPB)));
      wgs = gates * a.pieces;
    }
    Cols c{};
    c.cols = a.cols;
    c.blocks = cdiv(a.cols, 64);
    size_t floats = 0;
    auto take = [&](size_t rows) {
      const size_t at = floats;
      floats += (rows * a.cols + 63) & ~size_t(63);
      return at;
    };
    const bool gatePart = g.dgate && !a.each && a.pieces > 1;
    const size_t pGate = gatePart ? take(wgs) : 0, pPost = g.dpost && wgs > 1 ? take(wgs) : 0,
                 pPre = g.dpre && wgs > 1 ? take(wgs) : 0;
    float* ws = floats ? workspace(floats) : nullptr;
    if (floats && !ws) return false;
    a.dgate = gatePart ? ws + pGate : g.dgate;
    a.dpost = g.dpost && wgs > 1 ? ws + pPost : g.dpost;
    a.dpre = g.dpre && wgs > 1 ? ws + pPre : g.dpre;
    hipLaunchKernelGGL((nt ? k_norm_bwd<TPR, NV, W, true> : k_norm_bwd<TPR, NV, W, false>), dim3(wgs), dim3(T), 0, stream(), a);
    if (!check_launch("norm")) return false;
    uint32_t sums = 0, blocks = 0;
    auto add = [&](const float* part, float* out, uint32_t count, uint32_t groups) {
      c.part[sums] = part;
      c.out[sums] = out;
      c.count[sums] = count;
      c.groups[sums++] = groups;
      blocks += groups * c.blocks;
    };
    if (gatePart) add(a.dgate, g.dgate, a.pieces, gates);
    if (g.dpost && wgs > 1) add(a.dpost, g.dpost, wgs, 1);
    if (g.dpre && wgs > 1) add(a.dpre, g.dpre, wgs, 1);
    if (!sums) return true;
    hipLaunchKernelGGL(k_norm_cols, dim3(blocks), dim3(kColWaves * 64), 0, stream(), c);
    return check_launch("norm");
  }
};

Norm norm_of(const NormArgs& x) {
  Norm a{};
  a.x = x.x;
  a.block = x.block;
  a.gate = x.gate;
  a.post = x.post;
  a.pre = x.pre;
  a.h = x.h;
  a.n = x.n;
  a.r1 = x.r1;
  a.r2 = x.r2;
  a.rows = x.rows;
  a.cols = x.cols;
  a.each = x.gate && x.gateRows == x.rows;
  a.per = x.gate && !a.each ? x.rows / x.gateRows : x.rows;
  a.scale = x.scale;
  a.eps = x.eps;
  return a;
}

}  // namespace

bool norm_forward(const NormArgs& x) {
  Norm a = norm_of(x);
  const double n = double(x.rows) * x.cols, bytes = 4 * n * (x.block ? (x.n ? 4 : 3) : 2);
  ProfScope prof("norm", 10 * n, bytes);
  return dispatch(x.cols, Fwd{a, stream_nt(bytes)});
}

bool norm_backward(const NormArgs& x, const NormGrads& g) {
  Norm a = norm_of(x);
  a.dh = g.dh;
  a.dn = g.dn;
  a.dx = g.dx;
  a.db = g.db;
  const double n = double(x.rows) * x.cols;
  const double bytes = 4 * n * ((g.dh ? 1 : 0) + (g.dn ? 2 : 0) + (x.block ? 1 : 0) + (g.dx ? 1 : 0) + (g.db ? 1 : 0));
  ProfScope prof("norm", 20 * n, bytes);
  return dispatch(x.cols, Bwd{a, g, stream_nt(bytes)});
}

}  // namespace dce
