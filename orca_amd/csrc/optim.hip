// Adam over a list of tensors in one launch (train.py:180,238: torch.optim.Adam(tgn.parameters(), lr) /
// optimizer.step()).  The model has ~35 parameter tensors of 100 .. 141,600 floats: torch's foreach implementation is
// seven launches and 0.3 ms of host time per step, a third of what is left of the training step.  Arithmetic in the
// order of torch's _multi_tensor_adam (no weight decay, no amsgrad):
//   m += (1 - b1) (g - m);  v = b2 v + (1 - b2) g g;  p -= (lr / (1 - b1^t)) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// With a device scalar s (the clipping coefficient of orca_grad_norm) g is s times the gradient: clipping costs no pass of its own and
// no host read.
#include <cmath>
#include "common.h"

namespace {
constexpr int ADAM_MAX = 48;       // tensors per launch (the TGN of the bench has 35: one launch)
struct AdamGroup {
  int n;
  int first[ADAM_MAX + 1];         // first block of each tensor (1024 elements per block)
  float* p[ADAM_MAX];
  const float* g[ADAM_MAX];
  float* m[ADAM_MAX];
  float* v[ADAM_MAX];
  int64_t size[ADAM_MAX];
};

// one element: g -> p, m, v
__device__ __forceinline__ void adam_element(float gi, float* p, float* m, float* v, float w1, float b2, float w2, float step_size, float bc2_sqrt,
                                             float eps) {
  const float mi = *m + w1 * (gi - *m);
  const float vi = *v * b2 + w2 * gi * gi;
  *m = mi;
  *v = vi;
  *p -= step_size * (mi / (sqrtf(vi) / bc2_sqrt + eps));
}

template <bool SCALED>
__global__ __launch_bounds__(256) void k_adam(AdamGroup grp, float w1, float b2, float w2, float step_size, float bc2_sqrt,
                                              float eps, const float* __restrict__ scale) {
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
    if (i >= n) continue;
    const float gi = SCALED ? g[i] * *scale : g[i];
    adam_element(gi, p + i, m + i, v + i, w1, b2, w2, step_size, bc2_sqrt, eps);
  }
}

// the rows of a row-sparse gradient: a wave per row, bound by 7 accesses per element (28 bytes) at the rows' own width
__global__ __launch_bounds__(256) void k_adam_rows(const int64_t* __restrict__ ids, const float* __restrict__ g, const int32_t* __restrict__ count,
                                                   int64_t room, int64_t num_rows, int64_t width, float* __restrict__ p, float* __restrict__ m,
                                                   float* __restrict__ v, float w1, float b2, float w2, float step_size, float bc2_sqrt, float eps,
                                                   const float* __restrict__ scale) {
  const int64_t n = *count < room ? *count : room;
  const float s = scale ? *scale : 1.0f;
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < n; r += (int64_t)gridDim.x * 4) {
    const int64_t id = ids[r];
    if (id < 0 || id >= num_rows) continue;
    for (int64_t c = threadIdx.x & 63; c < width; c += 64) {
      const int64_t at = id * width + c;
      adam_element(g[r * width + c] * s, p + at, m + at, v + at, w1, b2, w2, step_size, bc2_sqrt, eps);
    }
  }
}

struct adam_scalars { float w1, b2, w2, step_size, bc2_sqrt, eps; };
adam_scalars scalars(double lr, double beta1, double beta2, double eps, int64_t step) {
  const double bc1 = 1.0 - std::pow(beta1, (double)step), bc2 = 1.0 - std::pow(beta2, (double)step);
  return adam_scalars{(float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)(lr / bc1), (float)std::sqrt(bc2), (float)eps};
}
}  // namespace

ORCA_API int orca_adam_step_scaled(int n, float* const* params, const float* const* grads, float* const* exp_avg,
                                   float* const* exp_avg_sq, const int64_t* sizes, double lr, double beta1, double beta2, double eps,
                                   int64_t step, const float* grad_scale, void* stream) {
  ORCA_REQUIRE(n >= 0 && step >= 1 && (n == 0 || (params && grads && exp_avg && exp_avg_sq && sizes)),
               "orca_adam_step: bad arguments");
  const adam_scalars k = scalars(lr, beta1, beta2, eps, step);
  for (int i0 = 0; i0 < n; i0 += ADAM_MAX) {
    AdamGroup grp{};
    int first = 0, t = 0;
    for (int i = i0; i < n && i < i0 + ADAM_MAX; ++i) {
      if (sizes[i] <= 0) continue;
      ORCA_REQUIRE(params[i] && grads[i] && exp_avg[i] && exp_avg_sq[i], "orca_adam_step: null tensor %d", i);
      ORCA_REQUIRE(sizes[i] < (1LL << 40), "orca_adam_step: tensor %d too large", i);
      grp.first[t] = first;
      grp.p[t] = params[i]; grp.g[t] = grads[i]; grp.m[t] = exp_avg[i]; grp.v[t] = exp_avg_sq[i]; grp.size[t] = sizes[i];
      first += (int)ceil_div64(sizes[i], 1024);
      ++t;
    }
    if (t == 0) continue;
    grp.n = t;
    grp.first[t] = first;
    auto* kernel = grad_scale ? k_adam<true> : k_adam<false>;
    kernel<<<(unsigned)first, 256, 0, (hipStream_t)stream>>>(grp, k.w1, k.b2, k.w2, k.step_size, k.bc2_sqrt, k.eps, grad_scale);
  }
  ORCA_LAUNCH_CHECK();
  return ORCA_OK;
}

ORCA_API int orca_adam_step(int n, float* const* params, const float* const* grads, float* const* exp_avg,
                            float* const* exp_avg_sq, const int64_t* sizes, double lr, double beta1, double beta2, double eps,
                            int64_t step, void* stream) {
  return orca_adam_step_scaled(n, params, grads, exp_avg, exp_avg_sq, sizes, lr, beta1, beta2, eps, step, nullptr, stream);
}

ORCA_API int orca_adam_rows(const int64_t* ids, const float* rows, const int32_t* count, int64_t room, int64_t num_rows, int64_t width, float* param,
                            float* exp_avg, float* exp_avg_sq, double lr, double beta1, double beta2, double eps, int64_t step,
                            const float* grad_scale, void* stream) {
  ORCA_REQUIRE(room >= 0 && num_rows >= 0 && width >= 1 && step >= 1 && room < (1LL << 31), "orca_adam_rows: bad sizes");
  if (room == 0 || num_rows == 0) return ORCA_OK;
  ORCA_REQUIRE(ids && rows && count && param && exp_avg && exp_avg_sq, "orca_adam_rows: null argument");
  const adam_scalars k = scalars(lr, beta1, beta2, eps, step);
  const int64_t blocks = ceil_div64(room, 4);
  k_adam_rows<<<(unsigned)(blocks < 8192 ? blocks : 8192), 256, 0, (hipStream_t)stream>>>(ids, rows, count, room, num_rows, width, param, exp_avg, exp_avg_sq,
                                                                                         k.w1, k.b2, k.w2, k.step_size, k.bc2_sqrt, k.eps, grad_scale);
  ORCA_LAUNCH_CHECK();
  return ORCA_OK;
}
