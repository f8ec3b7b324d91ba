// AdamW over flat f32 buffers (parameters that are not matrices beside Muon, or a whole model).
//
// Seven streams of n floats (read p g m v, write p m v) and a dozen operations an element: bound by HBM alone.
#include <algorithm>
#include <cmath>

#include "common.h"
#include "prof.h"

namespace {
constexpr int TPB = 256;
constexpr long long MOST = 1LL << 31;   // elements of a launch (a grid has fewer than 2^32 threads; a multiple of 4: alignment stays)

struct AdamW {
  float keep, step_size, beta1, omb1, beta2, omb2, inv_bc2, eps;   // 1 - lr wd, lr / (1 - beta1^t), ..., 1 / (1 - beta2^t)
  float grad_scale, max_norm;
};

__device__ __forceinline__ void adamw_one(float& p, float g, float& m, float& v, const AdamW& a, float coef) {
  g *= coef;
  m = fmaf(a.omb1, g, a.beta1 * m);   // (fused by hand: both forms of the kernel give the same bits)
  v = fmaf(a.omb2 * g, g, a.beta2 * v);
  p = fmaf(-a.step_size, m / (sqrtf(v * a.inv_bc2) + a.eps), a.keep * p);
}

// VEC: 16-byte accesses, four elements a thread and the last n % 4 by the last workgroup; else one element at a time (buffers that
// start anywhere). 66.4 M elements: 4.8 TB/s one element at a time.
template <bool VEC>
__global__ __launch_bounds__(TPB) void adamw_kernel(float* __restrict__ p, const float* __restrict__ g, float* __restrict__ m,
                                                    float* __restrict__ v, long long n, AdamW a, const float* __restrict__ sumsq) {
  float coef = a.grad_scale;
  if (a.max_norm > 0.f) {
    const float k = a.max_norm / (sqrtf(*sumsq) * a.grad_scale + 1e-6f);
    coef *= k > 1.f ? 1.f : k;   // (a NaN norm stays NaN)
  }
  const long long at = (long long)blockIdx.x * TPB + threadIdx.x;
  if constexpr (VEC) {
    if (at < n / 4) {
      float4 q = reinterpret_cast<float4*>(p)[at], w = reinterpret_cast<float4*>(m)[at], x = reinterpret_cast<float4*>(v)[at];
      const float4 y = reinterpret_cast<const float4*>(g)[at];
      adamw_one(q.x, y.x, w.x, x.x, a, coef);
      adamw_one(q.y, y.y, w.y, x.y, a, coef);
      adamw_one(q.z, y.z, w.z, x.z, a, coef);
      adamw_one(q.w, y.w, w.w, x.w, a, coef);
      reinterpret_cast<float4*>(p)[at] = q;
      reinterpret_cast<float4*>(m)[at] = w;
      reinterpret_cast<float4*>(v)[at] = x;
    }
    const long long i = n / 4 * 4 + threadIdx.x;
    if (blockIdx.x + 1 == gridDim.x && i < n) adamw_one(p[i], g[i], m[i], v[i], a, coef);
  } else {
    if (at < n) adamw_one(p[at], g[at], m[at], v[at], a, coef);
  }
}
}  // namespace

extern "C" int das_adamw_step(float* p, const float* g, float* m, float* v, long long n, double lr, double beta1, double beta2,
                              double eps, double weight_decay, long long step, float grad_scale, float max_norm,
                              const float* grad_sumsq, void* stream) {
  DAS_PROF(stream);
  if (!p || !g || !m || !v || n <= 0 || step < 1 || !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) || !(eps >= 0) ||
      !(lr >= 0) || !(weight_decay >= 0) || (max_norm > 0.f && !grad_sumsq))
    return DAS_ERR_ARG;
  if ((((uintptr_t)p | (uintptr_t)g | (uintptr_t)m | (uintptr_t)v) & 3) || n > (1LL << 60)) return DAS_ERR_ARG;
  const void* const buffers[4] = {p, g, m, v};
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < i; ++j)
      if (buffers_overlap(buffers[i], buffers[j], 4 * n)) return DAS_ERR_ARG;
  const double bc1 = 1.0 - std::pow(beta1, (double)step), bc2 = 1.0 - std::pow(beta2, (double)step);
  const AdamW a = {(float)(1.0 - lr * weight_decay), (float)(lr / bc1), (float)beta1, (float)(1.0 - beta1), (float)beta2,
                   (float)(1.0 - beta2), (float)(1.0 / bc2), (float)eps, grad_scale, max_norm};
  const bool vec = !(((uintptr_t)p | (uintptr_t)g | (uintptr_t)m | (uintptr_t)v) & 15);
  for (long long at = 0; at < n; at += MOST) {
    const long long k = std::min(MOST, n - at), threads = vec ? std::max(1LL, k / 4) : k;
    hipLaunchKernelGGL(vec ? adamw_kernel<true> : adamw_kernel<false>, dim3((unsigned)((threads + TPB - 1) / TPB)), dim3(TPB), 0,
                       (hipStream_t)stream, p + at, g + at, m + at, v + at, k, a, grad_sumsq);
    DAS_CHECK_LAUNCH();
  }
  return DAS_OK;
}
