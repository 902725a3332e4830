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

constexpr int kT = 256;
inline uint32_t cdiv(uint64_t a, uint64_t b) { return uint32_t((a + b - 1) / b); }

// m = act(g) u, n values.
template <MlpAct ACT>
__global__ void __launch_bounds__(kT) k_mlp_gate(const float* g, const float* u, float* m, uint32_t n) {
  for (uint32_t i = blockIdx.x * kT + threadIdx.x; i < n; i += gridDim.x * kT) m[i] = act<ACT>(g[i]) * u[i];
}
// dg, du and m from dm; dg may be dm.
template <MlpAct ACT>
__global__ void __launch_bounds__(kT)
    k_mlp_gate_grad(const float* dm, const float* g, const float* u, float* dg, float* du, float* m, uint32_t n) {
  for (uint32_t i = blockIdx.x * kT + threadIdx.x; i < n; i += gridDim.x * kT) {
    float d;
    const float a = act_grad<ACT>(g[i], d), t = dm[i], v = u[i];
    dg[i] = t * v * d;
    du[i] = t * a;
    m[i] = a * v;
  }
}
__global__ void __launch_bounds__(kT) k_mlp_add(const float* a, float* to, uint32_t n) {
  for (uint32_t i = blockIdx.x * kT + threadIdx.x; i < n; i += gridDim.x * kT) to[i] += a[i];
}

// A buffer that goes back to the pool with the scope: calls on the stream that
// follow may take it over, in order.
struct Temp {
  void* h;
  explicit Temp(size_t floats) : h(create_buffer(nullptr, uint32_t(floats))) {}
  ~Temp() { release_buffer(h); }
  Temp(const Temp&) = delete;
  Temp& operator=(const Temp&) = delete;
  float* ptr() const { return h ? static_cast<Buffer*>(h)->ptr : nullptr; }
};

inline dim3 grid_of(uint32_t n) { return dim3(std::min(cdiv(n, kT), uint32_t(num_cus()) * 32)); }

bool forward_plain(const MlpArgs& a) {
  const uint32_t n = a.rows * a.hidden;
  const Temp m(n), gu(a.saved ? 1 : 2 * size_t(n));
  float* g = a.saved ? a.saved : gu.ptr();
  if (!m.h || !gu.h) return false;
  if (!gemm(a.x, a.wg, g, a.rows, a.cols, a.hidden, 0) || !gemm(a.x, a.wu, g + n, a.rows, a.cols, a.hidden, 0)) return false;
  by_act(a.act, [&](auto k) {
    hipLaunchKernelGGL(k_mlp_gate<decltype(k)::value>, grid_of(n), dim3(kT), 0, stream(), g, g + n, m.ptr(), n);
  });
  return check_launch("GatedMlpForward") && gemm(m.ptr(), a.wd, a.y, a.rows, a.hidden, a.out, 0);
}

bool backward_plain(const MlpArgs& a, const float* dy, float* dx, float* dwg, float* dwu, float* dwd) {
  const uint32_t n = a.rows * a.hidden;
  const Temp dg(n), du(n), m(n), part(dx ? size_t(a.rows) * a.cols : 1);
  if (!dg.h || !du.h || !m.h || !part.h) return false;
  if (!gemm(dy, a.wd, dg.ptr(), a.rows, a.out, a.hidden, 2)) return false;
  by_act(a.act, [&](auto k) {
    hipLaunchKernelGGL(k_mlp_gate_grad<decltype(k)::value>, grid_of(n), dim3(kT), 0, stream(), dg.ptr(), a.saved,
                       a.saved + n, dg.ptr(), du.ptr(), m.ptr(), n);
  });
  if (!check_launch("GatedMlpBackward")) return false;
  if (dwd && !gemm(m.ptr(), dy, dwd, a.hidden, a.rows, a.out, 1)) return false;
  if (dwg && !gemm(a.x, dg.ptr(), dwg, a.cols, a.rows, a.hidden, 1)) return false;
  if (dwu && !gemm(a.x, du.ptr(), dwu, a.cols, a.rows, a.hidden, 1)) return false;
  if (!dx) return true;
  const uint32_t nx = a.rows * a.cols;
  if (!gemm(dg.ptr(), a.wg, dx, a.rows, a.hidden, a.cols, 2) || !gemm(du.ptr(), a.wu, part.ptr(), a.rows, a.hidden, a.cols, 2))
    return false;
  hipLaunchKernelGGL(k_mlp_add, grid_of(nx), dim3(kT), 0, stream(), part.ptr(), dx, nx);
  return check_launch("GatedMlpBackward");
}

}  // namespace

bool mlp_forward(const MlpArgs& a) { return mlp_on_parts(a) ? mlp_forward_parts(a) : forward_plain(a); }

bool mlp_backward(const MlpArgs& a, const float* dy, float* dx, float* dwg, float* dwu, float* dwd) {
  return mlp_on_parts(a) ? mlp_backward_parts(a, dy, dx, dwg, dwu, dwd) : backward_plain(a, dy, dx, dwg, dwu, dwd);
}

}  // namespace dce
