// The gated linear recurrence of a sequence's channels, each by itself:
//
//   f_t = sigmoid(z_t),   h_t = f_t h_(t-1) + (1 - f_t) x_t,   y = h,
//
// from a state h_0 (or zeros), and its gradients, which run the other way:
//
//   D_t = dy_t + f_(t+1) D_(t+1),   dx_t = (1 - f_t) D_t,
//   dz_t = D_t (h_(t-1) - x_t) f_t (1 - f_t),   dh_0 = f_1 D_1.
//
// Tokens from a sequence's length on leave the state as it is.
//
// A run of tokens maps the state that comes in to A state + H, A the product of
// its f, and two runs in a row to another such pair.  A lane holds L tokens of one
// channel in registers (of the batch's channels taken together, so that narrow
// ones fill waves), a workgroup NW waves of such runs, and where a sequence is
// longer than that, workgroups go one after the other along it.  Each reads its
// tokens once, leaves its pair in memory, waits for the pairs of those before it,
// and then goes through its tokens again, in registers, from the state that they
// make.  (Every 64th leaves its last state, too, where those after it start: no more
// than 63 pairs are read.)  So every value moves once: 12 bytes a value forward, 24
// backward.  4 x 4096
// tokens of 1024 channels: forward 42 us, 4.8 TB/s, backward 72 us, 5.6 TB/s, with
// about a third of that time's vector instructions; the pass that clears the pairs 2 to
// 4 us each.  (A thread for each channel: 6.0 ms.)
//
// Runs of 16 tokens and 16 waves: of 32 the backward's registers spill (190 us for 80),
// of 8 the pairs of twice as many workgroups are read (forward over 1 x 32768 tokens of
// 512 channels 51 us for 43; 8 waves of 16: 52).  Two channels a lane changed nothing.
// Small calls take runs of 8, for more workgroups (2 x 2048 tokens of 256 channels:
// forward 10.5 -> 9.9, backward 13.1 -> 11.6 us).
//
// Waiting: a workgroup takes its place from a counter, so those before it run
// already (a wait that ends all the same is reported).  Each leaves its pair before it waits for any, and a state waits for pairs
// and an earlier state only, so the first that lacks something gets it.  A pair, or a state,
// is one 64-bit word, whose value tells whether it is there, so no other word has to be
// ordered with it.  They are combined in one order, whoever came first.
#include "dce_internal.h"

#include <algorithm>

namespace dce {

namespace {

inline uint32_t cdiv(uint64_t a, uint64_t b) { return uint32_t((a + b - 1) / b); }

struct Scan {
  ScanArgs a;
  uint32_t per, across;     // sequences of a wave; waves across a sequence's channels
  uint32_t blocks, chunks;  // workgroups of one run of tokens; of a sequence
  unsigned long long* pairs;   // [chunks][blocks][64]
  unsigned long long* states;  // [chunks / kGroup][blocks][64]
  uint32_t* count;
  Waits waits;
};

// A lane's channel.  Tokens are reached from a place that a wave's lanes share, with
// 32-bit offsets of their own.
struct Lane {
  uint32_t off;    // bytes from the wave's first value of a token
  uint32_t n;      // tokens that count
  uint32_t state;  // place in [B][C]
  bool live;
  size_t first;    // the wave's first value of token 0
  __device__ __forceinline__ void init(const Scan& s, uint32_t block);
  // of token t, the wave's own
  template <bool NT>
  __device__ __forceinline__ float load(const float* p, size_t token) const {
    return ldus<NT, float>(reinterpret_cast<const char*>(p + first + token) + off);
  }
  template <bool NT>
  __device__ __forceinline__ void store(float* p, size_t token, float v) const {
    stus<NT>(reinterpret_cast<char*>(p + first + token) + off, v);
  }
};

__device__ __forceinline__ uint32_t tokens_of(const ScanArgs& a, uint32_t b) {
  if (!a.len) return a.S;
  const float n = a.len[b];
  return n >= 1.f ? min(uint32_t(fminf(n, 0x1p31f)), a.S) : 0u;  // NaN: none; S may be no float
}

__device__ __forceinline__ void Lane::init(const Scan& s, uint32_t block) {
  const ScanArgs& a = s.a;
  const uint32_t lane = threadIdx.x & 63, part = block / s.across;
  const uint32_t b0 = __builtin_amdgcn_readfirstlane(part * s.per);
  const uint32_t c0 = __builtin_amdgcn_readfirstlane((block - part * s.across) * 64);
  uint32_t i = 0, c = lane;
  if (s.per > 1) {
    i = lane / a.C;
    c = lane - i * a.C;
  }
  live = i < s.per && b0 + i < a.B && c0 + c < a.C;
  i = live ? i : 0;
  c = live ? c : 0;
  first = (size_t(b0) * a.S) * a.C + c0;
  off = (i * a.S * a.C + c) * 4;
  state = (b0 + i) * a.C + c0 + c;
  n = tokens_of(a, b0 + i);
}

constexpr uint32_t kGroup = 64;  // workgroups from one state to the next

// A pair that is not there yet: all bits set, as the pass before leaves them.  (A
// product of gates has that value only as a NaN, which is then written as another.)
constexpr unsigned long long kAbsent = ~0ull;
__device__ __forceinline__ unsigned long long pack(float A, float H) {
  const unsigned long long v = (static_cast<unsigned long long>(__float_as_uint(A)) << 32) | __float_as_uint(H);
  return v == kAbsent ? 0x7fc000007fc00000ull : v;
}
__device__ __forceinline__ unsigned long long look(const unsigned long long* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// (A, H) <- (A, H) then (A2, H2).
__device__ __forceinline__ void then(float& A, float& H, float A2, float H2) {
  H = A2 * H + H2;
  A = A2 * A;
}

// What is there at p, when it is there (where a wait ends before, NaN).
__device__ __forceinline__ unsigned long long await(const Waits& waits, const unsigned long long* p, unsigned long long v) {
  for (uint32_t spin = 0; v == kAbsent && spin < waits.spins; ++spin) {
    __builtin_amdgcn_s_sleep(1);
    v = look(p);
  }
  if (v == kAbsent) waits.report();
  return v;
}

// The state that comes into this wave's run, from `first` at the sequence's
// start; f: the run's gates, v(j): its inputs (h <- f h + v).
template <int NW, int L, class V>
__device__ __forceinline__ float state_in(const Scan& s, uint32_t chunk, uint32_t block, const float (&f)[L],
                                          const V& v, float first) {
  if constexpr (NW == 1) return first;
  __shared__ float run[2][NW][64], before[2][NW][64], start[64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const size_t next = size_t(s.blocks) * 64;
  unsigned long long* mine = s.pairs + block * 64 + lane;
  float A = 1.f, H = 0.f;
#pragma unroll
  for (int j = 0; j < L; ++j) then(A, H, f[j], v(j));
  run[0][w][lane] = A;
  run[1][w][lane] = H;
  __syncthreads();
  if (chunk + 1 < s.chunks && w == 0) {
    float a = 1.f, h = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) then(a, h, run[0][i][lane], run[1][i][lane]);
    __hip_atomic_store(mine + chunk * next, pack(a, h), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  float h = first;
  const uint32_t group = chunk / kGroup, from = group * kGroup, ahead = chunk - from;
  if (chunk) {
    // each wave a share of the group's workgroups before, four loads in flight
    const uint32_t lo = from + ahead * w / NW, hi = from + ahead * (w + 1) / NW;
    float a = 1.f, b = 0.f;
    for (uint32_t i = lo; i < hi; i += 4) {
      unsigned long long p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) p[e] = look(mine + min(i + e, hi - 1) * next);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[e] = await(s.waits, mine + min(i + e, hi - 1) * next, p[e]);
        if (i + e < hi) then(a, b, __uint_as_float(uint32_t(p[e] >> 32)), __uint_as_float(uint32_t(p[e])));
      }
    }
    before[0][w][lane] = a;
    before[1][w][lane] = b;
    if (group && w == 0) {
      const unsigned long long* p = s.states + (group - 1) * next + block * 64 + lane;
      start[lane] = __uint_as_float(uint32_t(await(s.waits, p, look(p))));
    }
    __syncthreads();
    if (group) h = start[lane];
#pragma unroll
    for (int i = 0; i < NW; ++i) h = before[0][i][lane] * h + before[1][i][lane];
  }
#pragma unroll
  for (int i = 0; i < NW; ++i)
    if (i < w) h = run[0][i][lane] * h + run[1][i][lane];
  return h;
}
// The state after the last wave's run, left where the next group starts.
template <int NW>
__device__ __forceinline__ void state_out(const Scan& s, uint32_t chunk, uint32_t block, uint32_t w, float h) {
  if (NW > 1 && w == NW - 1 && (chunk + 1) % kGroup == 0 && chunk + 1 < s.chunks)
    __hip_atomic_store(s.states + size_t(chunk / kGroup) * s.blocks * 64 + block * 64 + (threadIdx.x & 63), pack(1.f, h),
                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The workgroup's place: block of columns, and chunk along the sequence.
template <int NW>
__device__ __forceinline__ void place(const Scan& s, uint32_t& block, uint32_t& chunk) {
  uint32_t id = blockIdx.x;
  if (NW > 1 && s.chunks > 1) {
    __shared__ uint32_t mine;
    if (threadIdx.x == 0)  // the counter starts at 2^32 - 1
      mine = __hip_atomic_fetch_add(s.count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1;
    __syncthreads();
    id = __builtin_amdgcn_readfirstlane(mine);
  }
  chunk = id / s.blocks;
  block = id - chunk * s.blocks;
}

template <int NW, int L, bool NT>
__global__ void __launch_bounds__(NW * 64) k_scan_fwd(const Scan s) {
  const ScanArgs& a = s.a;
  uint32_t block, chunk;
  place<NW>(s, block, chunk);
  Lane at;
  at.init(s, block);
  const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t0 = (chunk * NW + w) * L;
  float f[L], v[L];
#pragma unroll
  for (int j = 0; j < L; ++j) {
    const size_t t = size_t(min(t0 + j, a.S - 1)) * a.C;
    f[j] = at.load<NT>(a.z, t);
    v[j] = at.load<NT>(a.x, t);
  }
  const float first = a.state ? a.state[at.state] : 0.f;
  // Most waves' tokens count for all of their channels.
  const bool whole = __all(t0 + L <= at.n);
#pragma unroll
  for (int j = 0; j < L; ++j) {
    float k;
    sigmoid_pair(f[j], f[j], k);
    v[j] *= k;
  }
  if (!whole) {
#pragma unroll
    for (int j = 0; j < L; ++j) {
      const bool in = t0 + j < at.n;
      f[j] = in ? f[j] : 1.f;
      v[j] = in ? v[j] : 0.f;
    }
  }
  float h = state_in<NW, L>(s, chunk, block, f, [&](int j) { return v[j]; }, first);
#pragma unroll
  for (int j = 0; j < L; ++j) v[j] = h = f[j] * h + v[j];
  state_out<NW>(s, chunk, block, w, h);
  if (!at.live) return;
  if (whole) {
#pragma unroll
    for (int j = 0; j < L; ++j) at.store<NT>(a.y, size_t(t0 + j) * a.C, v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < L; ++j)
      if (t0 + j < a.S) at.store<NT>(a.y, size_t(t0 + j) * a.C, t0 + j < at.n ? v[j] : 0.f);
  }
  if (a.last && chunk + 1 == s.chunks && w == NW - 1) a.last[at.state] = h;
}

// Token t = S - 1 - r, r counting up as above; the state is f_t D_t, and v = f dy.
template <int NW, int L, bool NT>
__global__ void __launch_bounds__(NW * 64) k_scan_bwd(const Scan s) {
  const ScanArgs& a = s.a;
  uint32_t block, chunk;
  place<NW>(s, block, chunk);
  Lane at;
  at.init(s, block);
  const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r0 = (chunk * NW + w) * L;
  float f[L], k[L], dy[L], u[L];
#pragma unroll
  for (int j = 0; j < L; ++j) {
    const size_t t = size_t(a.S - 1 - min(r0 + j, a.S - 1)) * a.C;
    f[j] = at.load<NT>(a.z, t);
    dy[j] = at.load<NT>(a.dy, t);
  }
  if (a.dz) {  // h_(t-1) - x_t
    float x[L];
#pragma unroll
    for (int j = 0; j < L; ++j) {
      const uint32_t t = a.S - 1 - min(r0 + j, a.S - 1);
      x[j] = at.load<NT>(a.x, size_t(t) * a.C);
      u[j] = at.load<NT>(a.y, size_t(max(t, 1u) - 1) * a.C);
    }
    const float first = a.state ? a.state[at.state] : 0.f;
#pragma unroll
    for (int j = 0; j < L; ++j) u[j] = (r0 + j + 1 < a.S ? u[j] : first) - x[j];
  }
  const bool whole = r0 + L <= a.S && __all(a.S - r0 <= at.n);
#pragma unroll
  for (int j = 0; j < L; ++j) sigmoid_pair(f[j], f[j], k[j]);
  if (!whole) {
#pragma unroll
    for (int j = 0; j < L; ++j) {
      const bool in = r0 + j < a.S && a.S - 1 - (r0 + j) < at.n;
      f[j] = in ? f[j] : 1.f;
      dy[j] = in ? dy[j] : 0.f;
    }
  }
  float h = state_in<NW, L>(s, chunk, block, f, [&](int j) { return f[j] * dy[j]; }, 0.f);
#pragma unroll
  for (int j = 0; j < L; ++j) {
    const float d = dy[j] + h;
    h = f[j] * d;
    u[j] = d * u[j] * (f[j] * k[j]);
    k[j] *= d;
  }
  state_out<NW>(s, chunk, block, w, h);
  if (!at.live) return;
  if (!whole) {
#pragma unroll
    for (int j = 0; j < L; ++j) {
      const bool in = a.S - 1 - (r0 + j) < at.n;
      u[j] = in ? u[j] : 0.f;
      k[j] = in ? k[j] : 0.f;
    }
  }
#pragma unroll
  for (int j = 0; j < L; ++j) {
    if (r0 + j >= a.S) break;
    const size_t t = size_t(a.S - 1 - (r0 + j)) * a.C;
    if (a.dx) at.store<NT>(a.dx, t, k[j]);
    if (a.dz) at.store<NT>(a.dz, t, u[j]);
  }
  if (a.dstate && chunk + 1 == s.chunks && w == NW - 1) a.dstate[at.state] = h;
}

__global__ void __launch_bounds__(256) k_scan_clear(unsigned long long* p, size_t n) {
  for (size_t i = size_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += size_t(gridDim.x) * 256) p[i] = kAbsent;
}

template <bool BWD, int NW, int L>
bool run(const ScanArgs& a, const char* what) {
  Scan s{};
  s.a = a;
  // Whole sequences side by side where they are narrow (and their offsets fit).
  s.per = a.C < 64 && uint64_t(a.S) * 64 < (1u << 30) ? 64 / a.C : 1;
  s.across = cdiv(a.C, 64);
  s.blocks = cdiv(a.B, s.per) * s.across;
  s.chunks = cdiv(a.S, NW * L);
  s.waits = g_waits;
  if (s.chunks > 1) {
    const size_t pairs = size_t(s.chunks) * s.blocks * 64, words = pairs + size_t(s.chunks / kGroup) * s.blocks * 64 + 1;
    float* ws = workspace(2 * words);
    if (!ws) return false;
    s.pairs = reinterpret_cast<unsigned long long*>(ws);
    s.states = s.pairs + pairs;
    s.count = reinterpret_cast<uint32_t*>(s.pairs + words - 1);
    hipLaunchKernelGGL(k_scan_clear, dim3(std::min(cdiv(words, 256), 1024u)), dim3(256), 0, stream(), s.pairs, words);
  }
  const bool nt = stream_nt((BWD ? 24.0 : 12.0) * a.B * a.S * a.C);
  auto* kernel = BWD ? (nt ? k_scan_bwd<NW, L, true> : k_scan_bwd<NW, L, false>)
                     : (nt ? k_scan_fwd<NW, L, true> : k_scan_fwd<NW, L, false>);
  hipLaunchKernelGGL(kernel, dim3(s.blocks * s.chunks), dim3(NW * 64), 0, stream(), s);
  return check_launch(what);
}

template <bool BWD>
bool scan(const ScanArgs& a, const char* what) {
  if (a.S == 1) return run<BWD, 1, 1>(a, what);
  if (a.S <= 8) return run<BWD, 1, 8>(a, what);
  if (a.S <= 32) return run<BWD, 4, 8>(a, what);
  const uint64_t wgs = cdiv(uint64_t(a.B) * a.C, 64) * uint64_t(cdiv(a.S, 256));
  return wgs < 100 ? run<BWD, 16, 8>(a, what) : run<BWD, 16, 16>(a, what);
}

}  // namespace

bool scan_forward(const ScanArgs& a) {
  const double n = double(a.B) * a.S * a.C;
  ProfScope prof("scan", 6 * n, 12 * n);
  return scan<false>(a, "GatedScanForward");
}

bool scan_backward(const ScanArgs& a) {
  const double n = double(a.B) * a.S * a.C;
  ProfScope prof("scan", 10 * n, 24 * n);
  return scan<true>(a, "GatedScanBackward");
}

}  // namespace dce
