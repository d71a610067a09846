// A list of tensors as one Adam launch takes it (optim.hip, clip_adam.hip).
#pragma once
#include <cmath>
#include "common.h"

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

struct AdamScalars { float w1, b2, w2, step_size, bc2_sqrt, eps; };
inline AdamScalars adam_scalars(double lr, double beta1, double beta2, double eps, int64_t step) {
  const double bc1 = 1.0 - std::pow(beta1, (double)step), bc2 = 1.0 - std::pow(beta2, (double)step);
  return AdamScalars{(float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)(lr / bc1), (float)std::sqrt(bc2), (float)eps};
}

// launch(group, its blocks) for every ADAM_MAX tensors
template <class F>
int adam_groups(int n, float* const* params, const float* const* grads, float* const* exp_avg, float* const* exp_avg_sq,
                const int64_t* sizes, int64_t step, F launch) {
  ORCA_REQUIRE(n >= 0 && step >= 1 && (n == 0 || (params && grads && exp_avg && exp_avg_sq && sizes)),
               "orca_adam_step: bad arguments");
  for (int i0 = 0; i0 < n; i0 += ADAM_MAX) {
    AdamGroup grp{};
    int64_t first = 0;
    int k = 0;
    for (int i = i0; i < n && i < i0 + ADAM_MAX; ++i) {
      if (sizes[i] <= 0) continue;
      ORCA_REQUIRE(params[i] && grads[i] && exp_avg[i] && exp_avg_sq[i], "orca_adam_step: null tensor %d", i);
      ORCA_REQUIRE(sizes[i] < (1LL << 40), "orca_adam_step: tensor %d too large", i);
      grp.first[k] = (int)first;
      grp.p[k] = params[i]; grp.g[k] = grads[i]; grp.m[k] = exp_avg[i]; grp.v[k] = exp_avg_sq[i]; grp.size[k] = sizes[i];
      first += ceil_div64(sizes[i], 1024);
      ORCA_REQUIRE(first < (1 << 24), "orca_adam_step: too many elements for one call");      // (a launch has under 2^32 threads)
      ++k;
    }
    if (k == 0) continue;
    grp.n = k;
    grp.first[k] = (int)first;
    launch(grp, (unsigned)first);
  }
  ORCA_LAUNCH_CHECK();
  return ORCA_OK;
}

// One element of the step.  Which products are fused with their sums is written out: the compiler's choice changes with its flags.
__device__ __forceinline__ void adam_element(float gi, float* p, float* m, float* v, const AdamScalars& k) {
#pragma clang fp contract(off)
  const float mi = fmaf(k.w1, gi - *m, *m);
  const float vi = *v * k.b2 + k.w2 * gi * gi;
  *m = mi;
  *v = vi;
  *p = fmaf(-k.step_size, mi / (sqrtf(vi) / k.bc2_sqrt + k.eps), *p);
}
