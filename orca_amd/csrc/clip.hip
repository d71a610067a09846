// The global 2-norm of a list of gradient tensors and their scaling to a largest norm (torch.nn.utils.clip_grad_norm_'s formula):
//   N = sqrt(sum g^2),  c = min(1, max_norm / (N + 1e-6)),  g <- c * g
// Two launches per GROUP_MAX tensors, no atomics and no host read: k_norm_partial leaves one fp64 sum per workgroup, and every
// workgroup of k_clip adds those sums up in the same order before it scales its share.  Squares and sums are fp64: neither
// overflows nor vanishes for any fp32 input, and the conversion is hidden behind the loads (4.5 elements per clock and CU at the
// HBM rate for 16-bit gradients).
#include <algorithm>
#include "elem.h"

namespace {
constexpr int GROUP_MAX = 96;         // tensors per launch: the group travels in the kernel's arguments (under 4 KB)
constexpr int TILE = 8192;            // elements a workgroup takes at a time
constexpr int PARTS = 2048;           // most partial sums of a call

struct grad_group {
  int n;
  int first[GROUP_MAX + 1];           // first tile of each tensor
  uint8_t dtype[GROUP_MAX];
  int32_t width[GROUP_MAX];           // of a row-sparse tensor
  const int32_t* rows[GROUP_MAX];     // its device count, or null
  void* g[GROUP_MAX];
  void* out[GROUP_MAX];               // k_clip: where the products go
  int64_t size[GROUP_MAX];
};
static_assert(sizeof(grad_group) <= 4000, "kernel arguments");

// the tensor that tile belongs to (uniform), its size now, and the tile's first element
__device__ __forceinline__ int locate(const grad_group& grp, int tile, int64_t* base, int64_t* size) {
  int lo = 0, hi = grp.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tile >= grp.first[mid]) lo = mid; else hi = mid;
  }
  *base = (int64_t)(tile - grp.first[lo]) * TILE;
  int64_t s = grp.size[lo];
  if (grp.rows[lo]) {
    const int64_t have = (int64_t)*grp.rows[lo] * grp.width[lo];
    s = have < s ? (have > 0 ? have : 0) : s;
  }
  *size = s;
  return lo;
}

template <class T>
__device__ __forceinline__ double tile_squares(const T* __restrict__ g, int64_t base, int64_t size) {
  constexpr int VEC = elems16<T>, STEPS = TILE / (256 * VEC);
  double acc = 0.0;
  if (base + TILE <= size) {
    u32x4 r[STEPS];
#pragma unroll
    for (int k = 0; k < STEPS; ++k) r[k] = load16(g + base + (threadIdx.x + 256 * k) * VEC);
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      float f[VEC];
      unpack16<T>(r[k], f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const double d = (double)f[j];
        acc = fma(d, d, acc);
      }
    }
  } else {
    for (int64_t i = base + threadIdx.x; i < size; i += 256) {
      const double d = (double)(float)g[i];
      acc = fma(d, d, acc);
    }
  }
  return acc;
}

// sum over the workgroup's 256 threads, the same bits in every thread
__device__ __forceinline__ double block_sum(double v, double* lds) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

__global__ __launch_bounds__(256) void k_norm_partial(grad_group grp, double* __restrict__ part) {
  __shared__ double lds[4];
  double acc = 0.0;
  const int tiles = grp.first[grp.n];
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    int64_t base, size;
    const int t = locate(grp, tile, &base, &size);
    if (base >= size) continue;
    if (grp.dtype[t] == ORCA_F32) acc += tile_squares((const float*)grp.g[t], base, size);
    else if (grp.dtype[t] == ORCA_BF16) acc += tile_squares((const __bf16*)grp.g[t], base, size);
    else acc += tile_squares((const _Float16*)grp.g[t], base, size);
  }
  const double s = block_sum(acc, lds);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// the coefficient from the partial sums: every workgroup adds them in the same order
__device__ __forceinline__ float coefficient(const double* __restrict__ part, int parts, double max_norm, double* lds, double* norm) {
  double acc = 0.0;
#pragma unroll
  for (int k = 0; k < PARTS / 256; ++k) {
    const int i = threadIdx.x + 256 * k;
    acc += i < parts ? part[i] : 0.0;
  }
  *norm = sqrt(block_sum(acc, lds));
  const double c = max_norm / (*norm + 1e-6);
  return c > 1.0 ? 1.0f : (float)c;       // (a NaN stays one)
}

__global__ __launch_bounds__(256) void k_norm_finish(const double* __restrict__ part, int parts, double max_norm, float* __restrict__ norm,
                                                     float* __restrict__ coef) {
  __shared__ double lds[4];
  double n;
  const float c = coefficient(part, parts, max_norm, lds, &n);
  if (threadIdx.x == 0) {
    *norm = (float)n;
    if (coef) *coef = c;
  }
}

template <class T>
__device__ __forceinline__ void tile_scale(const T* g, T* out, int64_t base, int64_t size, float c) {
  constexpr int VEC = elems16<T>, STEPS = TILE / (256 * VEC);
  if (base + TILE <= size) {
    u32x4 r[STEPS];
#pragma unroll
    for (int k = 0; k < STEPS; ++k) r[k] = load16(g + base + (threadIdx.x + 256 * k) * VEC);
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      float f[VEC];
      unpack16<T>(r[k], f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] *= c;
      store16(out + base + (threadIdx.x + 256 * k) * VEC, pack16<T>(f));
    }
  } else {
    for (int64_t i = base + threadIdx.x; i < size; i += 256) out[i] = (T)((float)g[i] * c);
  }
}

__global__ __launch_bounds__(256) void k_clip(grad_group grp, const double* __restrict__ part, int parts, double max_norm, int in_place,
                                              float* __restrict__ norm) {
  __shared__ double lds[4];
  double n;
  const float c = coefficient(part, parts, max_norm, lds, &n);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
  if (in_place && c == 1.0f) return;
  const int tiles = grp.first[grp.n];
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    int64_t base, size;
    const int t = locate(grp, tile, &base, &size);
    if (base >= size) continue;
    if (grp.dtype[t] == ORCA_F32) tile_scale((const float*)grp.g[t], (float*)grp.out[t], base, size, c);
    else if (grp.dtype[t] == ORCA_BF16) tile_scale((const __bf16*)grp.g[t], (__bf16*)grp.out[t], base, size, c);
    else tile_scale((const _Float16*)grp.g[t], (_Float16*)grp.out[t], base, size, c);
  }
}

int check_list(const char* who, int n, void* const* grads, const int64_t* sizes, const uint8_t* dtypes, const int32_t* const* rows, const int32_t* widths,
               double max_norm, const float* norm, const void* workspace, int64_t* tiles) {
  ORCA_REQUIRE(n >= 0 && n <= 65536 && norm && workspace && (n == 0 || (grads && sizes && dtypes)) && (!rows || widths), "%s: null argument, or not 0 to 65536 tensors", who);
  ORCA_REQUIRE(max_norm >= 0.0, "%s: max_norm %g (not negative, not NaN)", who, max_norm);
  *tiles = 0;
  for (int i = 0; i < n; ++i) {
    ORCA_REQUIRE(sizes[i] >= 0 && sizes[i] < (1LL << 40) && (sizes[i] == 0 || grads[i]), "%s: tensor %d: null, or a bad size", who, i);
    ORCA_REQUIRE(dtypes[i] <= ORCA_F16, "%s: tensor %d: unknown type %d", who, i, dtypes[i]);
    ORCA_REQUIRE(!rows || !rows[i] || widths[i] >= 1, "%s: tensor %d: width %d", who, i, rows && rows[i] ? widths[i] : 0);
    *tiles += ceil_div64(sizes[i], TILE);
  }
  ORCA_REQUIRE(*tiles < (1LL << 31), "%s: too many elements for one call", who);
  return ORCA_OK;
}

// calls f(group, its tiles) for each GROUP_MAX tensors that hold anything
template <class F>
int each_group(int n, void* const* grads, const int64_t* sizes, const uint8_t* dtypes, const int32_t* const* rows, const int32_t* widths,
               void* const* flat, F f) {
  int64_t used[3] = {0, 0, 0};
  for (int i = 0; i < n;) {
    grad_group grp{};
    int64_t tiles = 0;
    for (; i < n && grp.n < GROUP_MAX; ++i) {
      const int k = grp.n, dt = dtypes[i];
      if (sizes[i] == 0) continue;
      grp.first[k] = (int)tiles;
      grp.dtype[k] = (uint8_t)dt;
      grp.rows[k] = rows ? rows[i] : nullptr;
      grp.width[k] = grp.rows[k] ? widths[i] : 0;
      grp.g[k] = grads[i];
      grp.out[k] = flat ? (char*)flat[dt] + used[dt] : grads[i];
      grp.size[k] = sizes[i];
      used[dt] += sizes[i] * (dt == ORCA_F32 ? 4 : 2);
      tiles += ceil_div64(sizes[i], TILE);
      grp.first[++grp.n] = (int)tiles;
    }
    if (grp.n) {
      if (int rc = f(grp, tiles)) return rc;
    }
  }
  return ORCA_OK;
}

// k_norm_partial over the list: *parts sums, at most PARTS (each group gets its share of them)
int partial_sums(int n, void* const* grads, const int64_t* sizes, const uint8_t* dtypes, const int32_t* const* rows, const int32_t* widths, int64_t tiles,
                 double* part, int* parts, hipStream_t stream) {
  *parts = 0;
  const int64_t room = PARTS - ceil_div64(n, GROUP_MAX);
  return each_group(n, grads, sizes, dtypes, rows, widths, nullptr, [&](const grad_group& grp, int64_t mine) {
    const int64_t grid = std::min(mine, mine * room / tiles + 1);
    k_norm_partial<<<(unsigned)grid, 256, 0, stream>>>(grp, part + *parts);
    *parts += (int)grid;
    ORCA_LAUNCH_CHECK();
    return ORCA_OK;
  });
}
}  // namespace

ORCA_API int64_t orca_grad_norm_workspace_bytes(void) { return PARTS * 8; }

ORCA_API int orca_grad_norm(int n, void* const* grads, const int64_t* sizes, const uint8_t* dtypes, const int32_t* const* rows, const int32_t* widths,
                            double max_norm, float* norm, float* coef, void* workspace, void* stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  int64_t tiles = 0;
  int parts = 0;
  if (int rc = check_list("orca_grad_norm", n, grads, sizes, dtypes, rows, widths, max_norm, norm, workspace, &tiles)) return rc;
  if (int rc = partial_sums(n, grads, sizes, dtypes, rows, widths, tiles, (double*)workspace, &parts, stream)) return rc;
  k_norm_finish<<<1, 256, 0, stream>>>((const double*)workspace, parts, max_norm, norm, coef);
  ORCA_LAUNCH_CHECK();
  return ORCA_OK;
}

ORCA_API int orca_clip_grads(int n, void* const* grads, const int64_t* sizes, const uint8_t* dtypes, const int32_t* const* rows, const int32_t* widths,
                             double max_norm, void* const* flat, float* norm, void* workspace, void* stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  int64_t tiles = 0;
  int parts = 0;
  if (int rc = check_list("orca_clip_grads", n, grads, sizes, dtypes, rows, widths, max_norm, norm, workspace, &tiles)) return rc;
  for (int i = 0; flat && i < n; ++i) ORCA_REQUIRE(sizes[i] == 0 || flat[dtypes[i]], "orca_clip_grads: no flat buffer for type %d", dtypes[i]);
  if (int rc = partial_sums(n, grads, sizes, dtypes, rows, widths, tiles, (double*)workspace, &parts, stream)) return rc;
  if (tiles == 0) {
    k_norm_finish<<<1, 256, 0, stream>>>((const double*)workspace, 0, max_norm, norm, nullptr);
    ORCA_LAUNCH_CHECK();
    return ORCA_OK;
  }
  float* norm_out = norm;         // the first group's launch writes it
  return each_group(n, grads, sizes, dtypes, rows, widths, flat, [&](const grad_group& grp, int64_t mine) {
    k_clip<<<(unsigned)std::min<int64_t>(mine, 2048), 256, 0, stream>>>(grp, (const double*)workspace, parts, max_norm, flat == nullptr, norm_out);
    norm_out = nullptr;
    ORCA_LAUNCH_CHECK();
    return ORCA_OK;
  });
}
