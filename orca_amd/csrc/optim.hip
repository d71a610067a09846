// Adam over a list of tensors in one launch (train.py:180,238: torch.optim.Adam(tgn.parameters(), lr) /
// optimizer.step()).  The model has ~35 parameter tensors of 100 .. 141,600 floats: torch's foreach implementation is
// seven launches and 0.3 ms of host time per step, a third of what is left of the training step.  Arithmetic in the
// order of torch's _multi_tensor_adam (no weight decay, no amsgrad):
//   m += (1 - b1) (g - m);  v = b2 v + (1 - b2) g g;  p -= (lr / (1 - b1^t)) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
#include "adam.h"

namespace {
__global__ __launch_bounds__(256) void k_adam(AdamGroup grp, AdamScalars k) {
  int t = 0;
#pragma unroll
  for (int i = 1; i < ADAM_MAX; ++i) t += (i < grp.n && (int)blockIdx.x >= grp.first[i]) ? 1 : 0;
  t = __builtin_amdgcn_readfirstlane(t);
  float* __restrict__ p = grp.p[t];
  const float* __restrict__ g = grp.g[t];
  float* __restrict__ m = grp.m[t];
  float* __restrict__ v = grp.v[t];
  const int64_t n = grp.size[t];
  const int64_t base = (int64_t)((int)blockIdx.x - grp.first[t]) * 1024 + threadIdx.x;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t i = base + 256 * u;
    if (i < n) adam_element(g[i], p + i, m + i, v + i, k);
  }
}
}  // namespace

ORCA_API int orca_adam_step(int n, float* const* params, const float* const* grads, float* const* exp_avg,
                            float* const* exp_avg_sq, const int64_t* sizes, double lr, double beta1, double beta2, double eps,
                            int64_t step, void* stream) {
  const AdamScalars k = adam_scalars(lr, beta1, beta2, eps, step < 1 ? 1 : step);
  return adam_groups(n, params, grads, exp_avg, exp_avg_sq, sizes, step, [&](const AdamGroup& grp, unsigned blocks) {
    k_adam<<<blocks, 256, 0, (hipStream_t)stream>>>(grp, k);
  });
}
