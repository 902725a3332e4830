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
#include "dce_internal.h"

namespace dce {

namespace {

constexpr int kT = 256;
inline uint32_t cdiv(uint64_t a, uint64_t b) { return uint32_t((a + b - 1) / b); }

__device__ __forceinline__ uint32_t tokens_of(const ScanArgs& a, uint32_t b) {
  if (!a.len) return a.S;
  const float n = a.len[b];
  return n >= 1.f ? (n < float(a.S) ? uint32_t(n) : a.S) : 0u;  // NaN: none
}

// f = sigmoid(z) and k = 1 - f, each to fp32's accuracy of its own.
__device__ __forceinline__ void gates(float z, float& f, float& k) {
  const float e = expf(-fabsf(z)), big = 1.f / (1.f + e), small = e * big;
  f = z >= 0.f ? big : small;
  k = z >= 0.f ? small : big;
  if (z != z) f = k = z;
}

__global__ void __launch_bounds__(kT) k_scan_fwd(const ScanArgs a) {
  const uint64_t id = uint64_t(blockIdx.x) * kT + threadIdx.x;
  if (id >= uint64_t(a.B) * a.C) return;
  const uint32_t b = uint32_t(id / a.C), c = uint32_t(id % a.C), n = tokens_of(a, b);
  float h = a.state ? a.state[id] : 0.f;
  const size_t base = size_t(b) * a.S * a.C + c;
  for (uint32_t t = 0; t < n; ++t) {
    float f, k;
    gates(a.z[base + size_t(t) * a.C], f, k);
    h = f * h + k * a.x[base + size_t(t) * a.C];
    a.y[base + size_t(t) * a.C] = h;
  }
  for (uint32_t t = n; t < a.S; ++t) a.y[base + size_t(t) * a.C] = 0.f;
  if (a.last) a.last[id] = h;
}

__global__ void __launch_bounds__(kT) k_scan_bwd(const ScanArgs a) {
  const uint64_t id = uint64_t(blockIdx.x) * kT + threadIdx.x;
  if (id >= uint64_t(a.B) * a.C) return;
  const uint32_t b = uint32_t(id / a.C), c = uint32_t(id % a.C), n = tokens_of(a, b);
  const size_t base = size_t(b) * a.S * a.C + c;
  for (uint32_t t = a.S; t-- > n;) {
    if (a.dx) a.dx[base + size_t(t) * a.C] = 0.f;
    if (a.dz) a.dz[base + size_t(t) * a.C] = 0.f;
  }
  float back = 0.f;
  for (uint32_t t = n; t-- > 0;) {
    const size_t at = base + size_t(t) * a.C;
    float f, k;
    gates(a.z[at], f, k);
    const float d = a.dy[at] + back, before = t ? a.y[at - a.C] : a.state ? a.state[id] : 0.f;
    if (a.dx) a.dx[at] = k * d;
    if (a.dz) a.dz[at] = d * (before - a.x[at]) * f * k;
    back = f * d;
  }
  if (a.dstate) a.dstate[id] = back;
}

}  // namespace

bool scan_forward(const ScanArgs& a) {
  const double n = double(a.B) * a.S * a.C;
  ProfScope prof("scan", 6 * n, 12 * n);
  hipLaunchKernelGGL(k_scan_fwd, dim3(cdiv(uint64_t(a.B) * a.C, kT)), dim3(kT), 0, stream(), a);
  return check_launch("GatedScanForward");
}

bool scan_backward(const ScanArgs& a) {
  const double n = double(a.B) * a.S * a.C;
  ProfScope prof("scan", 10 * n, 24 * n);
  hipLaunchKernelGGL(k_scan_bwd, dim3(cdiv(uint64_t(a.B) * a.C, kT)), dim3(kT), 0, stream(), a);
  return check_launch("GatedScanBackward");
}

}  // namespace dce
