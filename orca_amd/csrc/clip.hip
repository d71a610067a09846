// The global 2-norm of a list of gradient tensors and their scaling to a largest norm (torch.nn.utils.clip_grad_norm_'s formula):
//   N = sqrt(sum g^2),  c = min(1, max_norm / (N + 1e-6)),  g <- c * g
// No atomics and no host read.  Short lists, two launches: k_norm_partial leaves one fp64 sum per workgroup, and every workgroup of k_clip
// adds those sums up in the same order (while its first piece is on its way) before it scales its share.  Long ones, where that time
// shows: k_norm_finish adds them up in between, and a workgroup of k_clip takes a piece or four and ends.  Squares and sums are fp64:
// neither overflows nor vanishes for any fp32 input, and the conversions hide behind the loads (5 elements per clock and CU at the
// HBM rate for 16-bit gradients).  Bound by the HBM: 400 million elements in 300 tensors, 871 MB, 425 us = 138 (6.3 TB/s) + 5 + 282 (6.2
// TB/s; torch's copy of 1 GiB runs at 5.0); short lists by the two launches: 35 tensors of 2.9 MB 3.5 + 4.6 us.
//   A list travels in the kernel's arguments, under 4 KB: 12 bytes per tensor (16 with flat buffers), so that a few hundred tensors
// are one launch.  With a search by scalar loads through 41 bytes per tensor, k_norm_partial took 6.4 us for 32 tensors of 2.9 MB.
#include <algorithm>
#include "elem.h"

namespace {
// Bytes a workgroup takes at a time: small pieces spread a short list over more workgroups.
constexpr int PIECE = 16384, SMALL_PIECE = 4096, LONG_PIECE = 8192;
// From here on a list is long, us for fp32 and both ways: into flat buffers 80 MB 41.0 (long: 45.6), 100 MB 54.9 (54.5), 120 MB 72.0 (63.2),
// 500 MB 286 (246); in place 120 MB 55.6 (62.9), 160 MB 80.9 (80.1), 240 MB 133 (115), 1 GB 545 (466).
constexpr int64_t LONG_FLAT = 100000000, LONG_IN_PLACE = 160000000;
// The products of long lists are written past the caches (non-temporal; 871 MB, most of it in 16 bits, flat: 425, with plain stores 502)
// and their gradients read so by k_clip (439 with plain loads), by k_norm_partial from here on: below, the last-level cache keeps some of
// them for k_clip (300 tensors of both widths, flat, plain and past: 120 MB 69.8 and 73.6, 300 MB 147 and 156, 500 MB 245 and 251, 600 MB 295
// and 296, 700 MB 346 and 341, 800 MB 398 and 391, 1 GB 500 and 487; all fp32 500 MB 241 and 247, 700 MB 343 and 344, 800 MB 394 and 393).
constexpr int64_t PAST_NORM = 650000000;
// Workgroups of a launch of k_norm_partial, and the most partial sums of a call.
constexpr int GRID = 2048, LONG_GRID = 1024, PARTS = 2048, LONG_PARTS = 8192;
// Pieces of a workgroup of k_clip on a long list in place: when the coefficient is 1 they all only come and go (500 MB of fp32 with one
// piece, four, sixteen: 107, 91, 87 us; with a coefficient below 1 233, 226, 238).
constexpr int IN_PLACE_PIECES = 4;
constexpr unsigned MOST_BLOCKS = 1 << 22;       // (a launch has under 2^32 threads; more pieces go round)
constexpr int SPARSE_MAX = 4;         // row-sparse tensors per launch

struct sparse_grad {
  const int32_t* rows;                // the device count
  int32_t width, dtype;
};
// Tensor t: its address in the low 48 bits, the bytes of its last piece / 2 - 1 in the next 13, 1 for a row-sparse one, its type in the top 2
// (row-sparse: its number in `sparse` is in `which`).
template <int N, bool FLAT> struct grad_list {
  int n, n_sparse;
  uint64_t at[N];
  int first[N + 1];                   // first piece of each tensor
  int which[SPARSE_MAX];              // the tensors that are row-sparse
  sparse_grad sparse[SPARSE_MAX];
  uint32_t to[FLAT ? N : 1];          // flat: where the tensor begins in its type's buffer, in elements from flat[type]
  char* flat[3];                      // (the buffers, moved on to this list's first tensor of the type)
};
constexpr int IN_PLACE_MAX = 310, FLAT_MAX = 235;
typedef grad_list<IN_PLACE_MAX, false> in_place_list;
typedef grad_list<FLAT_MAX, true> flat_list;
static_assert(sizeof(in_place_list) <= 4000 && sizeof(flat_list) <= 4000, "kernel arguments");

struct piece { char* p; int64_t offset; int len, dtype, tensor; };       // offset: bytes from the tensor's beginning
// the lanes hold the first pieces of all tensors: those at or before a piece are counted in one go
template <class L> struct locator {
  static constexpr int K = (int)(sizeof(L::first) / 4 + 62) / 64;
  int first[K];
  __device__ __forceinline__ explicit locator(const L& list) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int k = 0; k < K; ++k) first[k] = 64 * k + lane < list.n ? list.first[64 * k + lane] : 0x7fffffff;
  }
  __device__ __forceinline__ piece find(const L& list, int i, int bytes) const {
    int t = -1;
#pragma unroll
    for (int k = 0; k < K; ++k) t += __popcll(__ballot(first[k] <= i));
    t = __builtin_amdgcn_readfirstlane(t);
    const uint64_t at = list.at[t];
    const int begin = list.first[t], end = list.first[t + 1];
    piece q;
    q.tensor = t;
    q.p = reinterpret_cast<char*>(at & 0xffffffffffffULL);
    q.dtype = (int)(at >> 62);
    q.offset = (int64_t)(i - begin) * bytes;
    q.len = i + 1 == end ? (((int)(at >> 48) & 0x1fff) + 1) * 2 : bytes;
    if ((at >> 61) & 1) {
      for (int s = 0; s < list.n_sparse; ++s)
        if (list.which[s] == t) {
          const int rows = *list.sparse[s].rows;
          const int64_t have = (int64_t)(rows > 0 ? rows : 0) * list.sparse[s].width * (q.dtype == ORCA_F32 ? 4 : 2) - q.offset;
          q.len = have < q.len ? (have > 0 ? (int)have : 0) : q.len;
        }
    }
    return q;
  }
};

template <class T, int STEPS>
__device__ __forceinline__ double squares(const u32x4 (&r)[STEPS], const piece& q) {
  double acc = 0.0;
  auto add = [&](float f) { acc = fma((double)f, (double)f, acc); };
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    const int b = ((int)threadIdx.x + 256 * k) * 16;
    if (b + 16 <= q.len) {
      float f[elems16<T>];
      unpack16<T>(r[k], f);
#pragma unroll
      for (int j = 0; j < elems16<T>; ++j) add(f[j]);
    } else {
      for (int e = b; e < q.len; e += (int)sizeof(T)) add((float)*reinterpret_cast<const T*>(q.p + q.offset + e));
    }
  }
  return acc;
}
template <bool PAST, class T, int STEPS>
__device__ __forceinline__ void scale(const u32x4 (&r)[STEPS], const piece& q, char* out, float c) {
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    const int b = ((int)threadIdx.x + 256 * k) * 16;
    if (b + 16 <= q.len) {
      float f[elems16<T>];
      unpack16<T>(r[k], f);
#pragma unroll
      for (int j = 0; j < elems16<T>; ++j) f[j] *= c;
      if constexpr (PAST) store16_past(out + b, pack16<T>(f));
      else store16(out + b, pack16<T>(f));
    } else {
      for (int e = b; e < q.len; e += (int)sizeof(T))
        *reinterpret_cast<T*>(out + e) = (T)((float)*reinterpret_cast<const T*>(q.p + q.offset + e) * c);
    }
  }
}
template <bool PAST, int STEPS>
__device__ __forceinline__ void request(u32x4 (&r)[STEPS], const piece& q) {
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    const int b = ((int)threadIdx.x + 256 * k) * 16;
    if (b + 16 <= q.len) {
      if constexpr (PAST) r[k] = load16_past(q.p + q.offset + b);
      else r[k] = load16(q.p + q.offset + b);
    }
  }
}

// sum over the workgroup's 256 threads, the same bits in every thread
__device__ __forceinline__ double block_sum(double v, double* lds) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// The pieces are taken from the last to the first: what was read last is still in the 256 MB last-level cache when k_clip begins.
template <int BYTES, bool PAST>
__global__ __launch_bounds__(256) void k_norm_partial(in_place_list list, double* __restrict__ part) {
  constexpr int STEPS = BYTES / 4096;
  __shared__ double lds[4];
  const locator<in_place_list> where(list);
  const int pieces = list.first[list.n];
  double acc = 0.0;
  for (int i = pieces - 1 - (int)blockIdx.x; i >= 0; i -= (int)gridDim.x) {
    const piece q = where.find(list, i, BYTES);
    u32x4 r[STEPS];
    request<PAST>(r, q);
    if (q.dtype == ORCA_F32) acc += squares<float>(r, q);
    else if (q.dtype == ORCA_BF16) acc += squares<__bf16>(r, q);
    else acc += squares<_Float16>(r, q);
  }
  const double s = block_sum(acc, lds);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// the coefficient from the partial sums: every workgroup adds them in the same order
__device__ __forceinline__ float coefficient(const double* __restrict__ part, int parts, double max_norm, double* lds, double* norm) {
  double acc = 0.0;
  for (int i0 = 0; i0 < parts; i0 += PARTS) {
    double v[PARTS / 256];
#pragma unroll
    for (int k = 0; k < PARTS / 256; ++k) {
      const int i = i0 + (int)threadIdx.x + 256 * k;
      v[k] = i < parts ? part[i] : 0.0;
    }
#pragma unroll
    for (int k = 0; k < PARTS / 256; ++k) acc += v[k];
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

// coef (long lists): what k_norm_finish left; else the coefficient is made here
template <int BYTES, bool PAST, class L, bool FLAT>
__global__ __launch_bounds__(256) void k_clip(L list, const float* __restrict__ coef, const double* __restrict__ part, int parts, double max_norm,
                                              float* __restrict__ norm) {
  constexpr int STEPS = BYTES / 4096;
  __shared__ double lds[4];
  const locator<L> where(list);
  const int pieces = list.first[list.n];
  int i = blockIdx.x;
  piece q = where.find(list, i, BYTES);                   // (there are at least as many pieces as workgroups)
  u32x4 r[STEPS];
  float c;
  if constexpr (BYTES == LONG_PIECE) {
    c = *coef;
    if (!FLAT && c == 1.0f) return;
  }
  request<PAST>(r, q);
  if constexpr (BYTES != LONG_PIECE) {
    double n;
    c = coefficient(part, parts, max_norm, lds, &n);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
  }
  if (!FLAT && c == 1.0f) return;
  for (;;) {
    char* out = q.p + q.offset;
    if constexpr (FLAT) out = list.flat[q.dtype] + (int64_t)list.to[q.tensor] * (q.dtype == ORCA_F32 ? 4 : 2) + q.offset;
    if (q.dtype == ORCA_F32) scale<PAST, float>(r, q, out, c);
    else if (q.dtype == ORCA_BF16) scale<PAST, __bf16>(r, q, out, c);
    else scale<PAST, _Float16>(r, q, out, c);
    i += (int)gridDim.x;
    if (i >= pieces) break;
    q = where.find(list, i, BYTES);
    request<PAST>(r, q);
  }
}

struct host_list {
  int n;
  void* const* grads;
  const int64_t* sizes;
  const uint8_t* dtypes;
  const int32_t* const* rows;
  const int32_t* widths;
  int piece;                          // bytes, for the whole call
  int64_t pieces;
};
int64_t bytes_of(const host_list& h, int i) { return h.sizes[i] * (h.dtypes[i] == ORCA_F32 ? 4 : 2); }

int check_list(const char* who, host_list* h, int64_t long_from, double max_norm, const float* norm, const void* workspace) {
  ORCA_REQUIRE(h->n >= 0 && h->n <= 65536 && norm && workspace && (h->n == 0 || (h->grads && h->sizes && h->dtypes)) && (!h->rows || h->widths),
               "%s: null argument, or not 0 to 65536 tensors", who);
  ORCA_REQUIRE(((uintptr_t)workspace & 7) == 0, "%s: the workspace is not 8-byte aligned", who);
  ORCA_REQUIRE(max_norm >= 0.0, "%s: max_norm %g (not negative, not NaN)", who, max_norm);
  int64_t total = 0;
  for (int i = 0; i < h->n; ++i) {
    ORCA_REQUIRE(h->sizes[i] >= 0 && h->sizes[i] < (1LL << 40) && (h->sizes[i] == 0 || h->grads[i]), "%s: tensor %d: null, or a bad size", who, i);
    ORCA_REQUIRE(h->dtypes[i] <= ORCA_F16, "%s: tensor %d: unknown type %d", who, i, h->dtypes[i]);
    ORCA_REQUIRE(!h->rows || !h->rows[i] || h->widths[i] >= 1, "%s: tensor %d: width %d", who, i, h->rows && h->rows[i] ? h->widths[i] : 0);
    ORCA_REQUIRE(((uint64_t)(uintptr_t)h->grads[i] >> 48) == 0 && ((uintptr_t)h->grads[i] & 1) == 0, "%s: tensor %d: not a device address", who, i);
    total += bytes_of(*h, i);
  }
  // small pieces up to four workgroups per CU of them
  h->piece = total <= 1024LL * SMALL_PIECE ? SMALL_PIECE : total <= long_from ? PIECE : LONG_PIECE;
  h->pieces = 0;
  for (int i = 0; i < h->n; ++i) h->pieces += ceil_div64(bytes_of(*h, i), h->piece);
  ORCA_REQUIRE(h->pieces < (1LL << 31), "%s: too many elements for one call", who);
  return ORCA_OK;
}

// The list from tensor *i on, as much of it as a launch takes.  `to`: elements of each type so far, moved on.
template <class L, bool FLAT> void take(const host_list& h, int* i, int64_t* to, L* list) {
  constexpr int N = (int)(sizeof(L::at) / 8);
  list->n = list->n_sparse = 0;
  int64_t pieces = 0, from[3] = {0, 0, 0};
  if constexpr (FLAT) std::copy(to, to + 3, from);
  for (; *i < h.n && list->n < N; ++*i) {
    if (h.sizes[*i] == 0) continue;
    const int t = list->n, dt = h.dtypes[*i];
    const bool sparse = h.rows && h.rows[*i];
    if (sparse && list->n_sparse == SPARSE_MAX) break;
    if (FLAT && to[dt] - from[dt] >= (1LL << 32)) break;
    const int64_t bytes = bytes_of(h, *i), mine = ceil_div64(bytes, h.piece);
    const uint64_t tail = (uint64_t)(bytes - (mine - 1) * h.piece);
    list->at[t] = (uint64_t)(uintptr_t)h.grads[*i] | (tail / 2 - 1) << 48 | (uint64_t)sparse << 61 | (uint64_t)dt << 62;
    if (sparse) {
      list->which[list->n_sparse] = t;
      list->sparse[list->n_sparse++] = sparse_grad{h.rows[*i], h.widths[*i], dt};
    }
    if constexpr (FLAT) {
      list->to[t] = (uint32_t)(to[dt] - from[dt]);
      to[dt] += h.sizes[*i];
    }
    list->first[t] = (int)pieces;
    pieces += mine;
    list->first[t + 1] = (int)pieces;
    list->n = t + 1;
  }
}

int launches_of(const host_list& h) {             // how many lists take() makes of it, without flat buffers
  int launches = 0, n = 0, sparse = 0;
  for (int i = 0; i < h.n; ++i) {
    if (h.sizes[i] == 0) continue;
    const int s = h.rows && h.rows[i];
    if (launches == 0 || n == IN_PLACE_MAX || sparse + s > SPARSE_MAX) {
      ++launches;
      n = sparse = 0;
    }
    ++n;
    sparse += s;
  }
  return launches;
}

// k_norm_partial over the list: *parts sums
int partial_sums(const char* who, const host_list& h, double* part, int* parts, hipStream_t stream) {
  *parts = 0;
  const bool is_long = h.piece == LONG_PIECE;
  const int64_t most = is_long ? LONG_PARTS : PARTS, launches = launches_of(h);
  ORCA_REQUIRE(launches <= most / 2, "%s: too many row-sparse gradients for one call", who);
  for (int i = 0; i < h.n;) {
    in_place_list list;
    take<in_place_list, false>(h, &i, nullptr, &list);
    if (list.n == 0) continue;
    // (shares of what is left when every launch has one)
    const int64_t mine = list.first[list.n], wanted = is_long ? LONG_GRID : GRID;
    const unsigned grid = (unsigned)std::min({mine, wanted, launches * wanted <= most ? wanted : mine * (most - launches) / h.pieces + 1});
    if (is_long && h.pieces * LONG_PIECE >= PAST_NORM) k_norm_partial<LONG_PIECE, true><<<grid, 256, 0, stream>>>(list, part + *parts);
    else if (is_long) k_norm_partial<LONG_PIECE, false><<<grid, 256, 0, stream>>>(list, part + *parts);
    else if (h.piece == PIECE) k_norm_partial<PIECE, false><<<grid, 256, 0, stream>>>(list, part + *parts);
    else k_norm_partial<SMALL_PIECE, false><<<grid, 256, 0, stream>>>(list, part + *parts);
    ORCA_LAUNCH_CHECK();
    *parts += (int)grid;
  }
  return ORCA_OK;
}

template <class L, bool FLAT>
int clip(const host_list& h, void* const* flat, const float* coef, const double* part, int parts, double max_norm, float* norm, hipStream_t stream) {
  int64_t to[3] = {0, 0, 0};
  for (int i = 0; i < h.n;) {
    L list;
    if constexpr (FLAT)
      for (int k = 0; k < 3; ++k) list.flat[k] = (char*)flat[k] + to[k] * (k == ORCA_F32 ? 4 : 2);
    take<L, FLAT>(h, &i, to, &list);
    if (list.n == 0) continue;
    const unsigned pieces = (unsigned)list.first[list.n], grid = std::min<unsigned>(pieces, GRID),
                   many = std::min(FLAT ? pieces : (pieces - 1) / IN_PLACE_PIECES + 1, MOST_BLOCKS);
    if (h.piece == LONG_PIECE) k_clip<LONG_PIECE, true, L, FLAT><<<many, 256, 0, stream>>>(list, coef, part, parts, max_norm, norm);
    else if (h.piece == PIECE) k_clip<PIECE, false, L, FLAT><<<grid, 256, 0, stream>>>(list, coef, part, parts, max_norm, norm);
    else k_clip<SMALL_PIECE, false, L, FLAT><<<grid, 256, 0, stream>>>(list, coef, part, parts, max_norm, norm);
    ORCA_LAUNCH_CHECK();
    norm = nullptr;             // (the first launch writes it)
  }
  return ORCA_OK;
}
}  // namespace

ORCA_API int64_t orca_grad_norm_workspace_bytes(void) { return LONG_PARTS * 8 + 8; }

ORCA_API int orca_grad_norm(int n, void* const* grads, const int64_t* sizes, const uint8_t* dtypes, const int32_t* const* rows, const int32_t* widths,
                            double max_norm, float* norm, float* coef, void* workspace, void* stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  host_list h{n, grads, sizes, dtypes, rows, widths, 0, 0};
  int parts = 0;
  if (int rc = check_list("orca_grad_norm", &h, LONG_IN_PLACE, max_norm, norm, workspace)) return rc;
  if (int rc = partial_sums("orca_grad_norm", h, (double*)workspace, &parts, stream)) return rc;
  k_norm_finish<<<1, 256, 0, stream>>>((const double*)workspace, parts, max_norm, norm, coef);
  ORCA_LAUNCH_CHECK();
  return ORCA_OK;
}

ORCA_API int orca_clip_grads(int n, void* const* grads, const int64_t* sizes, const uint8_t* dtypes, const int32_t* const* rows, const int32_t* widths,
                             double max_norm, void* const* flat, float* norm, void* workspace, void* stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  host_list h{n, grads, sizes, dtypes, rows, widths, 0, 0};
  int parts = 0;
  if (int rc = check_list("orca_clip_grads", &h, flat ? LONG_FLAT : LONG_IN_PLACE, max_norm, norm, workspace)) return rc;
  for (int i = 0; flat && i < n; ++i) ORCA_REQUIRE(sizes[i] == 0 || flat[dtypes[i]], "orca_clip_grads: no flat buffer for type %d", dtypes[i]);
  if (int rc = partial_sums("orca_clip_grads", h, (double*)workspace, &parts, stream)) return rc;
  const double* part = (const double*)workspace;
  float* coef = (float*)((double*)workspace + LONG_PARTS);
  if (h.pieces == 0 || h.piece == LONG_PIECE) {
    k_norm_finish<<<1, 256, 0, stream>>>(part, parts, max_norm, norm, coef);
    ORCA_LAUNCH_CHECK();
  }
  return flat ? clip<flat_list, true>(h, flat, coef, part, parts, max_norm, norm, stream)
              : clip<in_place_list, false>(h, flat, coef, part, parts, max_norm, norm, stream);
}
