// AdamW over flat f32 buffers (parameters that are not matrices beside Muon, or a whole model).
//
// Seven streams of n floats (read p g m v, write p m v) and a dozen operations an element: bound by HBM alone.
#include <cmath>

#include "common.h"
#include "prof.h"

namespace {
constexpr int TPB = 256;

struct AdamW {
  float keep, step_size, beta1, omb1, beta2, omb2, inv_bc2, eps;   // 1 - lr wd, lr / (1 - beta1^t), ..., 1 / (1 - beta2^t)
  float grad_scale, max_norm;
};

__device__ __forceinline__ void adamw_one(float& p, float g, float& m, float& v, const AdamW& a, float coef) {
  g *= coef;
  m = a.beta1 * m + a.omb1 * g;
  v = a.beta2 * v + a.omb2 * (g * g);
  p = a.keep * p - a.step_size * m / (sqrtf(v * a.inv_bc2) + a.eps);
}

__global__ __launch_bounds__(TPB) void adamw_kernel(float* __restrict__ p, const float* __restrict__ g, float* __restrict__ m,
                                                    float* __restrict__ v, long long n, AdamW a, const float* __restrict__ sumsq) {
  float coef = a.grad_scale;
  if (a.max_norm > 0.f) {
    const float k = a.max_norm / (sqrtf(*sumsq) * a.grad_scale + 1e-6f);
    coef *= k > 1.f ? 1.f : k;   // (a NaN norm stays NaN)
  }
  for (long long i = (long long)blockIdx.x * TPB + threadIdx.x; i < n; i += (long long)gridDim.x * TPB)
    adamw_one(p[i], g[i], m[i], v[i], a, coef);
}
}  // namespace

extern "C" int das_adamw_step(float* p, const float* g, float* m, float* v, long long n, double lr, double beta1, double beta2,
                              double eps, double weight_decay, long long step, float grad_scale, float max_norm,
                              const float* grad_sumsq, void* stream) {
  DAS_PROF(stream);
  if (!p || !g || !m || !v || n <= 0 || step < 1 || !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) || !(eps >= 0) ||
      !(lr >= 0) || !(weight_decay >= 0) || (max_norm > 0.f && !grad_sumsq))
    return DAS_ERR_ARG;
  if (((uintptr_t)p | (uintptr_t)g | (uintptr_t)m | (uintptr_t)v) & 3) return DAS_ERR_ARG;
  const double bc1 = 1.0 - std::pow(beta1, (double)step), bc2 = 1.0 - std::pow(beta2, (double)step);
  const AdamW a = {(float)(1.0 - lr * weight_decay), (float)(lr / bc1), (float)beta1, (float)(1.0 - beta1), (float)beta2,
                   (float)(1.0 - beta2), (float)(1.0 / bc2), (float)eps, grad_scale, max_norm};
  const long long blocks = (n + TPB - 1) / TPB;
  hipLaunchKernelGGL(adamw_kernel, dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(TPB), 0, (hipStream_t)stream, p, g, m, v,
                     n, a, grad_sumsq);
  DAS_CHECK_LAUNCH();
  return DAS_OK;
}
