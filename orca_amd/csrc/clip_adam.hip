// Adam steps that k_adam (optim.hip) has no form for: with the gradients scaled by a device value on the way (the clipping coefficient of
// orca_grad_norm: no pass of its own over the gradients, no host read), and for the rows of a row-sparse gradient.
//   m += (1 - b1) (g - m);  v = b2 v + (1 - b2) g g;  p -= (lr / (1 - b1^t)) * m / (sqrt(v) / sqrt(1 - b2^t) + eps),   g = s * gradient
// The arithmetic is k_adam's (adam.h), so that a coefficient of 1 gives k_adam's bits.  Bound by the HBM, 28 bytes an element: 100 million of
// them 456 us (6.1 TB/s; k_adam 473 to 483), 37,663 rows of 100 out of ten million 21.8 us (4.8 TB/s); a TGN's 35 parameters 6.8 us (k_adam
// 6.4), 3391 rows 4.1 us, both by the latency of one round of workgroups.
#include "adam.h"

namespace {
__global__ __launch_bounds__(256) void k_adam_scaled(AdamGroup grp, AdamScalars k, const float* __restrict__ scale) {
  int t = 0;
#pragma unroll
  for (int i = 1; i < ADAM_MAX; ++i) t += (i < grp.n && (int)blockIdx.x >= grp.first[i]) ? 1 : 0;
  t = __builtin_amdgcn_readfirstlane(t);
  const float* __restrict__ g = grp.g[t];
  const float s = *scale;
  const int64_t n = grp.size[t], base = (int64_t)((int)blockIdx.x - grp.first[t]) * 1024 + threadIdx.x;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t i = base + 256 * u;
    if (i < n) adam_element(g[i] * s, grp.p[t] + i, grp.m[t] + i, grp.v[t] + i, k);
  }
}

// a wave per row; 28 bytes an element, whole rows at a time
__global__ __launch_bounds__(256) void k_adam_rows(const int64_t* __restrict__ ids, const float* __restrict__ g, const int32_t* __restrict__ count,
                                                   int64_t room, int64_t num_rows, int64_t width, float* __restrict__ p, float* __restrict__ m,
                                                   float* __restrict__ v, AdamScalars k, const float* __restrict__ scale) {
  const int64_t n = *count < room ? *count : room;
  const float s = scale ? *scale : 1.0f;
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < n; r += (int64_t)gridDim.x * 4) {
    const int64_t id = ids[r];
    if (id < 0 || id >= num_rows) continue;
    for (int64_t c = threadIdx.x & 63; c < width; c += 64) {
      const int64_t at = id * width + c;
      adam_element(g[r * width + c] * s, p + at, m + at, v + at, k);
    }
  }
}
}  // namespace

ORCA_API int orca_adam_step_scaled(int n, float* const* params, const float* const* grads, float* const* exp_avg, float* const* exp_avg_sq,
                                   const int64_t* sizes, double lr, double beta1, double beta2, double eps, int64_t step,
                                   const float* grad_scale, void* stream) {
  if (!grad_scale) return orca_adam_step(n, params, grads, exp_avg, exp_avg_sq, sizes, lr, beta1, beta2, eps, step, stream);
  const AdamScalars k = adam_scalars(lr, beta1, beta2, eps, step < 1 ? 1 : step);
  return adam_groups(n, params, grads, exp_avg, exp_avg_sq, sizes, step, [&](const AdamGroup& grp, unsigned blocks) {
    k_adam_scaled<<<blocks, 256, 0, (hipStream_t)stream>>>(grp, k, grad_scale);
  });
}

ORCA_API int orca_adam_rows(const int64_t* ids, const float* rows, const int32_t* count, int64_t room, int64_t num_rows, int64_t width, float* param,
                            float* exp_avg, float* exp_avg_sq, double lr, double beta1, double beta2, double eps, int64_t step,
                            const float* grad_scale, void* stream) {
  ORCA_REQUIRE(room >= 0 && num_rows >= 0 && width >= 1 && step >= 1 && room < (1LL << 31), "orca_adam_rows: bad sizes");
  if (room == 0 || num_rows == 0) return ORCA_OK;
  ORCA_REQUIRE(ids && rows && count && param && exp_avg && exp_avg_sq, "orca_adam_rows: null argument");
  const AdamScalars k = adam_scalars(lr, beta1, beta2, eps, step);
  const int64_t blocks = ceil_div64(room, 4);
  k_adam_rows<<<(unsigned)(blocks < 8192 ? blocks : 8192), 256, 0, (hipStream_t)stream>>>(ids, rows, count, room, num_rows, width, param, exp_avg,
                                                                                          exp_avg_sq, k, grad_scale);
  ORCA_LAUNCH_CHECK();
  return ORCA_OK;
}
