// Embedding rows and their gradient: out[p] = scale * table[ids[p]], and for the table
//   G[v] = round(scale * sum over {p : ids[p] = v} of g[p])
// as a dense table or as (ascending distinct ids, their rows, their number).  The sums are fp32 (each g is 16 or 32 bits wide; the
// one rounding to the output's type is the last step) and their order is fixed by (id, position) alone: the positions are sorted
// by id with a stable radix sort and the sorted list is cut into windows of equal length, so that a hub id with thousands of
// occurrences is spread over as many windows as it needs and two runs give the same bits.  (orca_scatter_add_flagged adds with
// fp32 atomics in whatever order they arrive.)
#include <algorithm>
#include <atomic>
#include <type_traits>
#include "elem.h"

namespace {
// VEC consecutive elements of a row as floats: one 16-byte access, or single elements (VEC = 1) where a row is shorter than that
template <int VEC, class T> __device__ __forceinline__ void load_chunk(const T* p, float (&f)[VEC]) {
  if constexpr (VEC == 1) f[0] = (float)p[0];
  else unpack16<T>(load16(p), f);
}
template <int VEC, class T, bool PAST = false> __device__ __forceinline__ void store_chunk(T* p, const float (&f)[VEC]) {
  if constexpr (VEC * sizeof(T) < 16) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) p[j] = (T)f[j];
  } else {
#pragma unroll
    for (int k = 0; k < VEC; k += elems16<T>) {
      if constexpr (PAST) store16_past(p + k, pack16<T>(f + k));
      else store16(p + k, pack16<T>(f + k));
    }
  }
}

// Where accesses go past the caches, by the bytes they cover.  Measured with the pass that reads or writes them next to it (us, plain
// -> past), since in between the 256 MB last-level cache hands the bytes to the neighbour:
//   lookup (100 and 172 fp32, 512 and 2048 bf16) with a product, a row maximum, a matrix product and a layer norm over its output, geometric
//     mean of past / plain: 0.25 to 2 MB 1.02 to 1.10, 4 to 8 MB 1.00 to 1.05, 12 MB 0.99 to 1.02, 18 MB 1.04 to 1.06, 200 MB 0.99 to 1.02, 256 MB
//     0.98 to 1.01, 300 MB 0.96 to 1.00, 400 MB 0.96 to 0.99.  (The lookup by itself is faster past the caches from 4 MB on, 18 MB 8.7 -> 8.0,
//     and its reader slower by more.)
//   dense gradient and the norm of it: 256 MB 104 -> 112, 400 MB 164 -> 162, 800 MB 318 -> 302
//   a product over grad_out and the gradient's pass over it: 96 MB 70 -> 73, 128 MB 86.5 -> 85.8, 256 MB 156 -> 147
constexpr int64_t MB = 1000000;
bool past_lookup(int64_t bytes) { return bytes >= 256 * MB; }
bool past_zeros(int64_t bytes) { return bytes >= 384 * MB; }
bool past_gradient(int64_t bytes) { return bytes >= 128 * MB; }

constexpr int64_t MAX_WIDTH = 65536;      // x * C of the division below stays under 2^32
// A launch has under 2^32 threads (the runtime's limit for blocks * threads).
bool fits_launch(int64_t blocks, int threads) { return blocks * threads < (1LL << 32); }

// ---- lookup ----------------------------------------------------------------------------------------------------------
// The output is a list of n * C chunks of 16 bytes; the last chunk of a row starts at width - VEC, so that every access is
// whole (it overlaps the one before it: both write the same values).  Rows narrower than a chunk go element by element.
// Bound by the id -> row latency of one round of workgroups (45,045 rows of 100 fp32: 7.2 us, 3.5 TB/s), large ones by the HBM (65,536 rows
// of 2048 bf16: 59.8 us, 5.8 TB/s: repeated rows come out of the caches); small ones by the launch (600 rows: 3.2 us).
constexpr int LOOK_U = 4;                 // chunks per thread: that many independent id -> row chains
template <class T, int VEC, bool PAST, class I>
__global__ __launch_bounds__(256) void k_embedding(const T* __restrict__ table, int64_t n_rows, int64_t ld,
                                                   const I* __restrict__ ids, int64_t total, int width, uint32_t C,
                                                   uint32_t magic, float scale, T* __restrict__ out) {
  const int64_t base = (int64_t)blockIdx.x * (256 * LOOK_U);
  const int64_t p0 = base / C;
  const uint32_t c0 = (uint32_t)(base - p0 * C) + threadIdx.x;
  int64_t at[LOOK_U], row[LOOK_U];
  int col[LOOK_U];
#pragma unroll
  for (int u = 0; u < LOOK_U; ++u) {
    const uint32_t x = c0 + 256 * u;
    const uint32_t q = C == 1 ? x : __umulhi(x, magic);
    const bool in = base + threadIdx.x + 256 * u < total;
    const int64_t p = p0 + q;
    const int c = (int)(x - q * C) * VEC;
    col[u] = VEC == 1 ? c : min(c, width - VEC);
    at[u] = in ? p * width + col[u] : -1;
    row[u] = in ? (int64_t)ids[p] : -1;
  }
  float v[LOOK_U][VEC];
#pragma unroll
  for (int u = 0; u < LOOK_U; ++u) {
    if (row[u] >= 0 && row[u] < n_rows) {
      load_chunk<VEC, T>(table + row[u] * ld + col[u], v[u]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[u][j] = 0.f;        // an id outside the table reads as zeros
    }
  }
#pragma unroll
  for (int u = 0; u < LOOK_U; ++u) {
    if (at[u] < 0) continue;
    if (row[u] >= 0 && row[u] < n_rows)
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[u][j] *= scale;
    store_chunk<VEC, T, PAST>(out + at[u], v[u]);
  }
}

template <class T, int VEC, class I>
int launch_embedding(const void* table, int64_t n_rows, int64_t width, int64_t ld, const I* ids, int64_t n, float scale, void* out,
                     hipStream_t stream) {
  const int64_t C = ceil_div64(width, VEC), total = n * C, blocks = ceil_div64(total, 256 * LOOK_U);
  ORCA_REQUIRE(fits_launch(blocks, 256), "orca_embedding_forward: %lld rows of %lld values are too many for one call", (long long)n, (long long)width);
  const uint32_t magic = C == 1 ? 0 : (uint32_t)(((1ULL << 32) + C - 1) / C);
  auto* kernel = VEC > 1 && past_lookup(n * width * (int64_t)sizeof(T)) ? k_embedding<T, VEC, VEC != 1, I> : k_embedding<T, VEC, false, I>;
  kernel<<<(unsigned)blocks, 256, 0, stream>>>((const T*)table, n_rows, ld, ids, total, (int)width, (uint32_t)C, magic, scale, (T*)out);
  ORCA_LAUNCH_CHECK();
  return ORCA_OK;
}

template <class T>
int embedding_typed(const void* table, int64_t n_rows, int64_t width, int64_t ld, const int64_t* idx64, const int32_t* idx32, int64_t n,
                    float scale, void* out, hipStream_t stream) {
  constexpr int VEC = elems16<T>;
  if (width >= VEC)
    return idx64 ? launch_embedding<T, VEC>(table, n_rows, width, ld, idx64, n, scale, out, stream)
                 : launch_embedding<T, VEC>(table, n_rows, width, ld, idx32, n, scale, out, stream);
  return idx64 ? launch_embedding<T, 1>(table, n_rows, width, ld, idx64, n, scale, out, stream)
               : launch_embedding<T, 1>(table, n_rows, width, ld, idx32, n, scale, out, stream);
}

// ---- zeros ahead of the sums -----------------------------------------------------------------------------------------
// A dense gradient starts as zeros; nothing before the sums reads it, so the launches of the sort carry the zero fill in extra
// workgroups: the sort waits on latency with a few dozen workgroups, the fill on the HBM, and the longer of the two is what counts.
// A piece is one 16-byte store for each of 256 threads: 640 MB in workgroups of 256 threads 94 us, 512 100, 1024 104, several stores a
// thread 105 to 107, a grid of 2048 that goes round 118.
constexpr int FILL_PIECE = 4096;
struct fill_job {
  char* p;                      // `rows` rows of `bytes` bytes, `pitch` bytes apart (a table without gaps is one row, pitch 0)
  int64_t bytes, pitch, per_row, from, to;      // pieces of a row; this launch's pieces
  int past;
};
template <int THREADS, bool PAST> __device__ __forceinline__ void fill_loop(const fill_job& f, int64_t block, int64_t blocks) {
  const u32x4 zero = {0, 0, 0, 0};
  for (int64_t i = f.from + block * (THREADS / 256) + (threadIdx.x >> 8); i < f.to; i += blocks * (THREADS / 256)) {
    const int64_t r = f.pitch ? i / f.per_row : 0, at = (i - r * f.per_row) * FILL_PIECE;
    char* p = f.p + r * f.pitch + at;
    const int len = (int)(f.bytes - at < FILL_PIECE ? f.bytes - at : FILL_PIECE), b = (int)(threadIdx.x & 255) * 16;
    if (b + 16 <= len) {
      if constexpr (PAST) store16_past(p + b, zero);
      else store16(p + b, zero);
    } else {
      for (int e = b; e < len; e += 2) *reinterpret_cast<uint16_t*>(p + e) = 0;
    }
  }
}
template <int THREADS> __device__ __forceinline__ void fill_pieces(const fill_job& f, int64_t block, int64_t blocks) {
  if (f.past) fill_loop<THREADS, true>(f, block, blocks);
  else fill_loop<THREADS, false>(f, block, blocks);
}
__global__ __launch_bounds__(256) void k_fill(fill_job f) { fill_pieces<256>(f, blockIdx.x, gridDim.x); }

// ---- sort of the positions by id -------------------------------------------------------------------------------------
// Stable least-significant-digit radix sort of (key, position) pairs; key = the id, or num_rows for what has no row (the padding
// id, ids outside the table): those end up last and are dropped.  A tile is 512 * ITEMS consecutive pairs of one workgroup; within it
// a wave owns 64 * ITEMS consecutive pairs and ranks them 64 at a time: the lanes with the same digit find each other with one
// ballot per digit bit.  Two launches per pass (count, scatter); with many tiles a third one adds the counts up.  Bound by latency: 85,995
// pairs in digits of 8 bits 4.1 and 7.6 us a pass; with 100 MB of zeros on board 16.4 and 16.0 (6.2 TB/s).
constexpr int SORT_THREADS = 512, SORT_WAVES = SORT_THREADS / 64;
constexpr int MIN_DIGIT = 2, MAX_DIGIT = 11, MAX_BINS = 1 << MAX_DIGIT;
// Up to this many tiles every workgroup adds the tiles' counts up itself; it takes the fewest pairs per thread whose counts stay below the
// bytes for one and for two.  One, two and four, us, row-sparse: 12,000 pairs in digits of 7 bits 29 31 36, 20,000 of 10 bits 38 39 43, 45,000 of
// 10 42 40 43, 86,000 of 8 52 53 57, 131,072 of 11 93 67 58, 300,000 of 10 133 93 75.
constexpr int DIRECT_TILES = 64;
constexpr int64_t ONE_BYTES = 192000, TWO_BYTES = 256000;
static_assert(4 * SORT_THREADS <= 65536, "16-bit counts within a tile");
static_assert(2 * SORT_THREADS * 16 <= SORT_WAVES * MAX_BINS * 2, "the slices' sums fit where the counts lie");
static_assert(MAX_BINS == 4 * SORT_THREADS, "a thread takes four neighbouring bins");
struct pair32 { uint32_t pos, key; };

struct sort_src {               // where a pass reads: the caller's ids (first pass) or the pairs of the pass before
  const int64_t* idx64;
  const int32_t* idx32;
  const pair32* pairs;
  int64_t n, num_rows, padding;
};
__device__ __forceinline__ pair32 sort_read(const sort_src& s, int64_t i) {
  if (s.pairs) return s.pairs[i];
  const int64_t id = s.idx64 ? s.idx64[i] : (int64_t)s.idx32[i];
  const bool ok = id >= 0 && id < s.num_rows && id != s.padding;
  return pair32{(uint32_t)i, ok ? (uint32_t)id : (uint32_t)s.num_rows};
}

// counts[tile][bin] of this pass' digit
template <int ITEMS>
__global__ __launch_bounds__(SORT_THREADS) void k_sort_count(sort_src src, int shift, int bins, uint32_t* __restrict__ counts, int tiles, fill_job fill) {
  __shared__ uint32_t h[MAX_BINS];
  if ((int)blockIdx.x >= tiles) {
    fill_pieces<SORT_THREADS>(fill, (int)blockIdx.x - tiles, (int)gridDim.x - tiles);
    return;
  }
  pair32 p[ITEMS];
  const int64_t base = (int64_t)blockIdx.x * (SORT_THREADS * ITEMS);
#pragma unroll
  for (int u = 0; u < ITEMS; ++u) {
    const int64_t i = base + threadIdx.x + SORT_THREADS * u;
    p[u] = i < src.n ? sort_read(src, i) : pair32{0u, 0u};
  }
  for (int b = threadIdx.x; b < bins; b += SORT_THREADS) h[b] = 0;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < ITEMS; ++u)
    if (base + threadIdx.x + SORT_THREADS * u < src.n) atomicAdd(&h[(p[u].key >> shift) & (bins - 1)], 1u);
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += SORT_THREADS) counts[(int64_t)blockIdx.x * bins + b] = h[b];
}

// counts[tile][bin] -> the number in the tiles before; totals[bin].  Bound by its round trips, eight tiles in each (a million pairs, 489
// tiles: 34 us a pass; four million: 136).
__global__ __launch_bounds__(64) void k_sort_columns(uint32_t* __restrict__ counts, int64_t tiles, int bins, uint32_t* __restrict__ totals) {
  const int b = blockIdx.x * 64 + threadIdx.x;
  if (b >= bins) return;
  uint32_t run = 0;
  for (int64_t t0 = 0; t0 < tiles; t0 += 8) {
    uint32_t c[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) c[u] = t0 + u < tiles ? counts[(t0 + u) * bins + b] : 0u;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (t0 + u < tiles) counts[(t0 + u) * bins + b] = run;
      run += c[u];
    }
  }
  totals[b] = run;
}

// inclusive prefix sums over the wave: within rows of 16 by row shifts, then the rows' last lanes broadcast (no LDS round trips)
__device__ __forceinline__ uint32_t wave_inclusive(uint32_t v) {
  int x = (int)v;
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  return (uint32_t)x;
}

// the lanes of `in` whose digit equals this lane's: per bit one compare, and one three-operand bit operation per half of the mask
__device__ __forceinline__ uint64_t same_digit(uint32_t d, int digit_bits, bool in) {
  const uint64_t all = __ballot(in);
  uint32_t lo = (uint32_t)all, hi = (uint32_t)(all >> 32);
#pragma unroll
  for (int k = 0; k < MAX_DIGIT; ++k) {
    if (k >= digit_bits) break;
    const int bit = (int)(d << (31 - k)) >> 31;          // 0 or all ones
    const uint64_t m = __ballot(bit != 0);
    lo &= ~((uint32_t)m ^ (uint32_t)bit);
    hi &= ~((uint32_t)(m >> 32) ^ (uint32_t)bit);
  }
  return ((uint64_t)hi << 32) | lo;
}

// totals == null: counts holds every tile's counts, which this workgroup adds up itself
template <int ITEMS>
__global__ __launch_bounds__(SORT_THREADS) void k_sort_scatter(sort_src src, int shift, int digit_bits, const uint32_t* __restrict__ counts,
                                                               const uint32_t* __restrict__ totals, pair32* __restrict__ out, int tiles, fill_job fill) {
  __shared__ uint32_t place[MAX_BINS];                   // where the tile's first pair of a digit goes
  __shared__ uint16_t part[SORT_WAVES][MAX_BINS];        // the wave's counts of a digit, then those of the waves before it
  __shared__ uint32_t wave_sum[SORT_WAVES];
  if ((int)blockIdx.x >= tiles) {
    fill_pieces<SORT_THREADS>(fill, (int)blockIdx.x - tiles, (int)gridDim.x - tiles);
    return;
  }
  const int bins = 1 << digit_bits, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int64_t base = (int64_t)blockIdx.x * (SORT_THREADS * ITEMS) + wave * (64 * ITEMS);
  pair32 p[ITEMS];
#pragma unroll
  for (int u = 0; u < ITEMS; ++u) {
    const int64_t i = base + 64 * u + lane;
    p[u] = i < src.n ? sort_read(src, i) : pair32{0u, 0u};
  }
  // pairs of each bin in the tiles before this one, and in all: a thread takes four bins and every `slices`-th tile
  u32x4 before = {0, 0, 0, 0}, total = {0, 0, 0, 0};
  const int quads = bins / 4, slices = SORT_THREADS / quads, quad = t & (quads - 1), slice = t / quads;
  if (totals) {
    if (slice == 0) {
      before = load16(counts + (int64_t)blockIdx.x * bins + 4 * quad);
      total = load16(totals + 4 * quad);
    }
  } else {
    for (int k0 = slice; k0 < tiles; k0 += 8 * slices) {
      u32x4 c[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) c[u] = k0 + u * slices < tiles ? load16(counts + (int64_t)(k0 + u * slices) * bins + 4 * quad) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (k0 + u * slices < (int)blockIdx.x) before += c[u];
        total += c[u];
      }
    }
    if (slices > 1) {           // the slices' sums meet in LDS (`part` is not in use yet)
      u32x4* meet = reinterpret_cast<u32x4*>(&part[0][0]);
      meet[t] = before;
      meet[SORT_THREADS + t] = total;
      __syncthreads();
      if (slice == 0)
        for (int k = 1; k < slices; ++k) {
          before += meet[quad + k * quads];
          total += meet[SORT_THREADS + quad + k * quads];
        }
      __syncthreads();
    }
  }
  if (slice != 0) total = u32x4{0, 0, 0, 0};
  for (int k = t; k < SORT_WAVES * MAX_BINS / 8; k += SORT_THREADS) reinterpret_cast<u32x4*>(&part[0][0])[k] = u32x4{0, 0, 0, 0};
  __syncthreads();
  uint32_t rank[ITEMS];
#pragma unroll
  for (int u = 0; u < ITEMS; ++u) {
    const bool in = base + 64 * u + lane < src.n;
    const uint32_t d = (p[u].key >> shift) & (uint32_t)(bins - 1);
    const uint64_t peers = same_digit(d, digit_bits, in);
    const int leader = in ? __ffsll((unsigned long long)peers) - 1 : lane;
    uint32_t seen = 0;
    if (in && lane == leader) {          // (one lane per digit, and the counts are the wave's own)
      seen = part[wave][d];
      part[wave][d] = (uint16_t)(seen + (uint32_t)__popcll(peers));
    }
    rank[u] = __shfl(seen, leader) + (uint32_t)__popcll(peers & ((1ULL << lane) - 1));
  }
  // exclusive prefix of the totals over the bins
  const uint32_t mine = total[0] + total[1] + total[2] + total[3];
  const uint32_t inc = wave_inclusive(mine);
  if (lane == 63) wave_sum[wave] = inc;
  __syncthreads();
  uint32_t run = inc - mine;
#pragma unroll
  for (int w = 0; w < SORT_WAVES; ++w) run += w < wave ? wave_sum[w] : 0u;
  if (slice == 0) {             // (t == quad)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int b = 4 * t + k;
      place[b] = run + before[k];
      run += total[k];
    }
    uint64_t* four = reinterpret_cast<uint64_t*>(&part[0][0]) + t;      // four 16-bit counts, added up without a carry
    uint64_t c[SORT_WAVES], sum = 0;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) c[w] = four[w * (MAX_BINS / 4)];
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) {
      four[w * (MAX_BINS / 4)] = sum;
      sum += c[w];
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < ITEMS; ++u) {
    if (base + 64 * u + lane < src.n) {
      const uint32_t d = (p[u].key >> shift) & (uint32_t)(bins - 1);
      out[place[d] + part[wave][d] + rank[u]] = p[u];
    }
  }
}

// ---- the rows' numbers (row-sparse form) -----------------------------------------------------------------------------
// rank[i] = the number of the distinct id that sorted pair i belongs to; ids[rank] = that id; *count = how many there are.  Two launches,
// as the sort's: heads per tile, then every tile adds up those before it (85,995 pairs: 2.1 and 3.4 us, latency).
__device__ __forceinline__ bool is_head(const pair32* s, int64_t i, uint32_t none) {
  const uint32_t k = s[i].key;
  return k != none && (i == 0 || s[i - 1].key != k);
}
template <int ITEMS>
__global__ __launch_bounds__(SORT_THREADS) void k_rank_count(const pair32* __restrict__ s, int64_t n, uint32_t none, uint32_t* __restrict__ tile_heads) {
  __shared__ int total;
  if (threadIdx.x == 0) total = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * (SORT_THREADS * ITEMS);
  int c = 0;
#pragma unroll
  for (int u = 0; u < ITEMS; ++u) {
    const int64_t i = base + threadIdx.x + SORT_THREADS * u;
    const uint64_t m = __ballot(i < n && is_head(s, i, none));
    c += __popcll(m);
  }
  if ((threadIdx.x & 63) == 0) atomicAdd(&total, c);
  __syncthreads();
  if (threadIdx.x == 0) tile_heads[blockIdx.x] = (uint32_t)total;
}
template <int ITEMS>
__global__ __launch_bounds__(SORT_THREADS) void k_rank(const pair32* __restrict__ s, int64_t n, uint32_t none, const uint32_t* __restrict__ tile_heads,
                                                       uint32_t* __restrict__ rank, int64_t* __restrict__ ids, int32_t* __restrict__ count) {
  __shared__ uint32_t before, wave_heads[SORT_WAVES];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  if (t == 0) before = 0;
  __syncthreads();
  uint32_t sum = 0;
  for (int64_t k = t; k < (int64_t)blockIdx.x; k += SORT_THREADS) sum += tile_heads[k];
#pragma unroll
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  if (lane == 0) atomicAdd(&before, sum);
  const int64_t base = (int64_t)blockIdx.x * (SORT_THREADS * ITEMS) + wave * (64 * ITEMS);
  uint64_t heads[ITEMS];
  uint32_t mine = 0;
#pragma unroll
  for (int u = 0; u < ITEMS; ++u) {
    const int64_t i = base + 64 * u + lane;
    heads[u] = __ballot(i < n && is_head(s, i, none));
    mine += (uint32_t)__popcll(heads[u]);
  }
  if (lane == 0) wave_heads[wave] = mine;
  __syncthreads();
  uint32_t run = before;
  for (int w = 0; w < wave; ++w) run += wave_heads[w];
#pragma unroll
  for (int u = 0; u < ITEMS; ++u) {
    const int64_t i = base + 64 * u + lane;
    const uint32_t upto = run + (uint32_t)__popcll(heads[u] & (~0ULL >> (63 - lane)));      // heads at or before this lane
    if (i < n && s[i].key != none) {
      rank[i] = upto - 1;
      if ((heads[u] >> lane) & 1) ids[upto - 1] = (int64_t)s[i].key;
    }
    run += (uint32_t)__popcll(heads[u]);
  }
  if ((int64_t)blockIdx.x == (int64_t)gridDim.x - 1 && t == SORT_THREADS - 1) *count = (int32_t)run;
}

// ---- sums over the windows of the sorted list ------------------------------------------------------------------------
// The sorted list is cut into windows of `window` pairs.  A team of 2^log_l lanes (a lane holds one 16-byte chunk of the columns; a
// whole workgroup for rows of 4 KB, so that the pieces of a row are requested together: in column blocks far apart in the grid the
// rows' first KBs met a quarter of the HBM channels at a time) walks one window in order.  A run of equal ids that lies inside the
// window is written out; one that crosses a border leaves its sum in `part` for k_segment_join.
// 45,045 ids of 100 fp32 8.8 us (latency: pairs, then rows); 65,536 of 2048 bf16 63 us: 268 MB read and 77 MB written at 5.5 TB/s.
constexpr int SEG_PAIRS = 2048;   // pairs of one workgroup's windows, at most
constexpr int SEG_U = 8;          // rows requested together; the next ones are on their way while these are added
struct seg_args {
  const void* g;                  // [n, width], row stride ld_g (0: every row is the same one)
  int64_t ld_g, n, ld_out;
  const pair32* s;
  const uint32_t* rank;           // or null: a row's place in the output is its id
  void* out;
  float* part;                    // [2 * windows, width]: what a window adds to a run that began before it / that it begins and does not end
  int width, chunks, log_l, window, col_blocks;
  uint32_t none;
  float scale;
};

template <int VEC, class T> struct raw_chunk {        // a chunk as it was loaded
  u32x4 r;
  template <bool PAST = false> __device__ __forceinline__ void load(const T* p) {
    if constexpr (PAST) r = load16_past(p);
    else r = load16(p);
  }
  __device__ __forceinline__ void add_to(float (&acc)[VEC]) const {
    float f[VEC];
    unpack16<T>(r, f);
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] += f[j];
  }
};
template <class T> struct raw_chunk<1, T> {
  T r;
  template <bool PAST = false> __device__ __forceinline__ void load(const T* p) { r = *p; }
  __device__ __forceinline__ void add_to(float (&acc)[1]) const { acc[0] += (float)r; }
};

template <class TI, class TO, int VEC, bool ACCUMULATE, bool PAST>
__global__ __launch_bounds__(256) void k_segment_sum(seg_args a) {
  __shared__ pair32 list[SEG_PAIRS + 2];        // [k + 1] = pair k of the workgroup's windows; its neighbours at both ends
  __shared__ uint32_t row[SEG_PAIRS];           // [k] = the output row of pair k (row-sparse form)
  const int teams = 256 >> a.log_l, team = threadIdx.x >> a.log_l, tl = threadIdx.x & ((1 << a.log_l) - 1);
  const int64_t w0 = (int64_t)(blockIdx.x / (uint32_t)a.col_blocks) * teams;
  const int c = ((int)(blockIdx.x % (uint32_t)a.col_blocks) << a.log_l) + tl;
  const int64_t base = w0 * a.window;
  const int count = (int)(a.n - base < teams * a.window ? a.n - base : teams * a.window);
  for (int k = threadIdx.x; k < count + 2; k += 256) {
    const int64_t i = base - 1 + k;
    const pair32 p = i >= 0 && i < a.n ? a.s[i] : pair32{0u, ~0u};          // (~0u: no key)
    const uint32_t r = a.rank && k < count ? a.rank[base + k] : 0u;          // (here: in the loop below it would wait for the rows on their way)
    list[k] = p;
    if (k < count) row[k] = r;
  }
  __syncthreads();
  const int first = team * a.window, last = min(first + a.window, count);
  if (first >= count || c >= a.chunks || list[first + 1].key == a.none) return;
  const int64_t w = w0 + team;
  const int col = VEC == 1 ? c : min(c * VEC, a.width - VEC), own = c * VEC - col;      // (elements before `own` are the neighbour's)
  const TI* g = (const TI*)a.g + col;
  uint32_t cur = list[first + 1].key;
  bool head = list[first].key == cur;
  int begin = first;              // first pair of the current run in this window
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
  auto flush = [&](bool goes_on) {
    if (cur == a.none) return;
    if (head || goes_on) {
      store_chunk<VEC, float>(a.part + (2 * w + (head ? 0 : 1)) * a.width + col, acc);
      return;
    }
    const int64_t r = a.rank ? row[begin] : cur;
    TO* o = (TO*)a.out + r * a.ld_out + col;
    float f[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = acc[j] * a.scale;
    if constexpr (ACCUMULATE) {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (j >= own) o[j] = (TO)((float)o[j] + f[j]);
    } else {
      store_chunk<VEC, TO>(o, f);
    }
  };
  typedef raw_chunk<VEC, TI> raw;
  auto request = [&](raw (&v)[SEG_U], int k) {
#pragma unroll
    for (int u = 0; u < SEG_U; ++u) v[u].template load<PAST>(g + (int64_t)list[min(k + u, last - 1) + 1].pos * a.ld_g);
  };
  auto add = [&](const raw (&v)[SEG_U], int k) {
#pragma unroll
    for (int u = 0; u < SEG_U; ++u) {
      if (k + u >= last) break;
      const uint32_t key = list[k + u + 1].key;
      if (key != cur) {
        flush(false);
        cur = key;
        head = false;
        begin = k + u;
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
      }
      v[u].add_to(acc);
    }
  };
  raw va[SEG_U], vb[SEG_U];
  request(va, first);
  for (int k = first; k < last; k += 2 * SEG_U) {
    if (k + SEG_U < last) request(vb, k + SEG_U);
    add(va, k);
    if (k + SEG_U >= last) break;
    if (k + 2 * SEG_U < last) request(va, k + 2 * SEG_U);
    add(vb, k + SEG_U);
  }
  flush(list[last + 1].key == cur);
}

// The runs that cross window borders, each taken by the window that begins it: sum of what that window and the following ones left in
// `part`, in their order.  A team takes one window; a run over more than JOIN_SHORT windows is left to the whole workgroup, whose teams
// take a consecutive share of the terms each, JOIN_TEAMS of them at most (narrow rows have up to 1024 teams, whose shares one team then
// adds: 30,391 ids of 5 bf16 52 us, 110 without the limit).  45,045 ids of 100 fp32 7.9 us: latency of heads, lengths and rows in turn.
constexpr int JOIN_SHORT = 16, JOIN_THREADS = 1024, JOIN_TEAMS = 32;
template <class TO, bool ACCUMULATE>
__global__ __launch_bounds__(JOIN_THREADS) void k_segment_join(seg_args a) {
  __shared__ float4 share[JOIN_THREADS];
  struct waiting { int64_t w, r; uint32_t key; };
  __shared__ waiting queue[JOIN_THREADS];
  __shared__ int queued;
  const int lanes = 1 << a.log_l, teams = JOIN_THREADS >> a.log_l, team = threadIdx.x >> a.log_l, tl = threadIdx.x & (lanes - 1);
  const int64_t w = (int64_t)(blockIdx.x / (uint32_t)a.col_blocks) * teams + team;
  const int col = (((int)(blockIdx.x % (uint32_t)a.col_blocks) << a.log_l) + tl) * 4;
  const int have = col >= a.width ? 0 : min(4, a.width - col);
  if (threadIdx.x == 0) queued = 0;
  __syncthreads();
  auto term = [&](int64_t w, int64_t k) {         // k = 0: the beginning window's own sum
    const float* q = a.part + (k == 0 ? 2 * w + 1 : 2 * (w + k)) * a.width + col;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (have == 4) {
      const u32x4 r = load16(q);
      __builtin_memcpy(&v, &r, 16);
    } else {
      if (have > 0) v.x = q[0];
      if (have > 1) v.y = q[1];
      if (have > 2) v.z = q[2];
    }
    return v;
  };
  auto sum = [&](int64_t w, int64_t b, int64_t e) {
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int64_t k = b; k < e; k += 8) {
      float4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = k + u < e ? term(w, k + u) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int u = 0; u < 8; ++u) { acc.x += v[u].x; acc.y += v[u].y; acc.z += v[u].z; acc.w += v[u].w; }
    }
    return acc;
  };
  auto write = [&](int64_t r, float4 acc) {
    TO* o = (TO*)a.out + r * a.ld_out + col;
    const float f[4] = {acc.x * a.scale, acc.y * a.scale, acc.z * a.scale, acc.w * a.scale};
    for (int j = 0; j < have; ++j) o[j] = (TO)(ACCUMULATE ? (float)o[j] + f[j] : f[j]);
  };
  // what decides about the window, requested together: a run costs two round trips (this one, its terms), not one per question
  const int64_t i0 = w * a.window, i1 = i0 + a.window, end = a.n - 1;
  const uint32_t key = a.s[i1 - 1 < end ? i1 - 1 : end].key, next = a.s[i1 < end ? i1 : end].key, prev = a.s[i0 > 0 && i0 <= end ? i0 - 1 : 0].key;
  const int64_t f0 = (w + 1 + tl) * a.window;
  const uint32_t later = a.s[f0 < end ? f0 : end].key;         // of the windows that follow, one per lane
  const int64_t r = a.rank ? (int64_t)a.rank[i1 - 1 < end ? i1 - 1 : end] : (int64_t)key;
  if (i1 < a.n && key != a.none && next == key && !(i0 > 0 && prev == key)) {       // (the same in the team's lanes)
    int terms = 1;              // the window's own sum, and one of each window that begins inside the run
    for (int t0 = 1; t0 <= JOIN_SHORT; t0 += lanes) {
      const int64_t f = (w + t0 + tl) * a.window;
      const uint64_t m = __ballot(f < a.n && (t0 == 1 ? later : a.s[f < end ? f : end].key) == key);
      const uint64_t of_team = lanes == 64 ? m : (m >> (threadIdx.x & 63 & ~(lanes - 1))) & ((1ULL << lanes) - 1);
      const int in = __popcll(of_team);
      terms += in;
      if (in < lanes) break;
    }
    if (terms <= JOIN_SHORT) {
      write(r, sum(w, 0, terms));
    } else if (tl == 0) {
      const int q = atomicAdd(&queued, 1);
      queue[q].w = w;
      queue[q].r = r;
      queue[q].key = key;
    }
  }
  __syncthreads();
  const int todo = queued;
  for (int q = 0; q < todo; ++q) {                // (the order of the queue does not matter: its runs are independent)
    const int64_t w = queue[q].w;
    int64_t terms = 1;
    for (;;) {
      const int64_t f = (w + terms + threadIdx.x) * a.window;
      const int m = __syncthreads_count(f < a.n && a.s[f].key == queue[q].key);
      terms += m;
      if (m < JOIN_THREADS) break;
    }
    const int most = min(teams, JOIN_TEAMS);
    const int64_t each = ceil_div64(terms, most), b = team * each, e = b + each < terms ? b + each : terms;
    if (team < most) share[threadIdx.x] = sum(w, b, e);
    __syncthreads();
    if (team == 0 && have) {
      float4 acc = share[tl];
#pragma unroll 4
      for (int t = 1; t < most; ++t) {
        const float4 v = share[(t << a.log_l) + tl];
        acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
      }
      write(queue[q].r, acc);
    }
    __syncthreads();
  }
}

// ---- short lists -----------------------------------------------------------------------------------------------------
// Up to SMALL_N ids and SMALL_VALUES values there is no order of the whole list to build: every workgroup reads all the ids (26 KB
// for 6600 of them, out of L2), keeps its share in the order of their positions and sorts those few in LDS.
//   dense, one launch (k_small): a hash of the id gives it to a workgroup, which adds its ids' rows.  It also has a share of the
//          table's rows; it marks those with an occurrence and zeroes the others, so that every row is written once.
//   rows, two launches: k_range_sort gives a workgroup the ids of an equal share of [0, num_rows), so that its sorted ids follow
//          those of the workgroup before; it leaves their positions and the number of distinct ones.  k_range_sums adds those numbers
//          up, which tells where every distinct id's row lies, and takes an even share of the runs.
// 600 ids, 9228 rows of 100 fp32: 8.6 us; 6600 row-sparse ids of 1.1 million: 19.4 (sort of the fullest range 12).  Bound by latency.
// Against it: the general path's launches wait for one another (600 ids 28 us, 6600 row-sparse 38 us); the whole list sorted by
// every workgroup took 9 us per radix pass at 6600 ids; the rows' places counted within one launch, over a hash set of all ids,
// took 24 us.
constexpr int SMALL_THREADS = 1024, SMALL_ITEMS = 8, SMALL_N = SMALL_THREADS * SMALL_ITEMS;
constexpr int TINY_THREADS = 256, TINY_N = TINY_THREADS * SMALL_ITEMS;         // workgroups of four waves: cheaper barriers
// Most values, us here and on the general path (row-sparse, dense; 1/rank ids): 2^21 (1000 ids of 2048 fp32) 19 and 29, 17 and 34; 2^23
// (2000 of 4096) 27 and 39, 27 and 48; 2^24 (8000 of 2048) 45 and 50, 35 and 50.  The small workgroups are the faster ones for the rows of
// 2^20 (250 of 4096: 12.6 and 14.3), not for 2^21.
constexpr int64_t SMALL_VALUES = 1 << 24, TINY_VALUES = 1 << 20;
constexpr int SMALL_MAP = 65536;               // table rows of a workgroup's share, at most (bits in LDS)
constexpr int SMALL_RUN = 32;                  // a longer run of equal ids is added by the whole workgroup ...
constexpr int SMALL_TEAMS = 32;                // ... in at most this many consecutive parts
constexpr int SMALL_PAIRS = 512;               // up to this many pairs (and a thread each) are sorted by counting the smaller ones
constexpr int SMALL_DIGIT = 8;                 // digit bits of the sort of longer lists
constexpr int MAX_RANGES = 256;
struct small_args {
  const int64_t* idx64;
  const int32_t* idx32;
  int64_t num_rows, padding;
  const void* g;
  int64_t ld_g, ld_out;
  void* out;
  int n, width, chunks, log_l, col_blocks, zero_rows;
  float scale;
};
// LDS: the list (room for all n: they may be equal, or meet in one hash), and one region in turn for the bit map, the sort's counts,
// and the sums: the parts of a long run and the starts of the runs
struct small_lds { int region, heads, bytes; };
__host__ __device__ inline small_lds small_layout(int threads, int n) {
  small_lds l;
  l.region = (n + 63) / 64 * 64 * 8;
  l.heads = l.region + threads * 8 * 4;
  l.bytes = l.heads + 2 * (n + 1);
  return l;
}
static_assert(((TINY_THREADS / 64 * 2 + 4) << SMALL_DIGIT) <= TINY_THREADS * 32 && ((SMALL_THREADS / 64 * 2 + 4) << SMALL_DIGIT) <= SMALL_THREADS * 32 &&
                  SMALL_MAP / 8 <= TINY_THREADS * 32,
              "the sort's counts and the bit map fit where the parts of a run lie");
// MurmurHash3's finaliser: ids in arithmetic progression (a multiplicative hash keeps them in one) land all over the range
__device__ __forceinline__ uint32_t small_hash(uint32_t key) {
  key ^= key >> 16;
  key *= 0x85ebca6bu;
  key ^= key >> 13;
  key *= 0xc2b2ae35u;
  return key ^ key >> 16;
}

// this thread's ids: pair i = base + 64 * u, `none` for what has no row
template <int THREADS>
__device__ __forceinline__ void small_keys(const small_args& a, int base, int items, uint32_t (&key)[SMALL_ITEMS]) {
#pragma unroll
  for (int u = 0; u < SMALL_ITEMS; ++u) {
    key[u] = (uint32_t)a.num_rows;
    if (u < items && base + 64 * u < a.n) {
      const int64_t id = a.idx64 ? a.idx64[base + 64 * u] : (int64_t)a.idx32[base + 64 * u];
      if (id >= 0 && id < a.num_rows && id != a.padding) key[u] = (uint32_t)id;
    }
  }
}
// numbers 0, 1, .. for the set flags of a wave-by-wave list; returns this wave's first number, *all = how many there are.  Two barriers.
template <int THREADS>
__device__ __forceinline__ uint32_t small_offsets(uint32_t mine, uint32_t* wave_sum, uint32_t* all) {
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) wave_sum[wave] = mine;
  __syncthreads();
  uint32_t run = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    const uint32_t c = wave_sum[w];
    run += w < wave ? c : 0u;
    sum += c;
  }
  __syncthreads();
  *all = sum;
  return run;
}

// sorts the first `m` pairs of `list` by key - least < 2^bits, equal keys in the order they had; all threads of the workgroup call it
template <int THREADS>
__device__ __forceinline__ void small_sort(pair32* list, int m, uint32_t least, int bits, char* region, uint32_t* wave_sum) {
  constexpr int WAVES = THREADS / 64;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  if (m <= min(SMALL_PAIRS, THREADS)) {
    // the keys come four at a time out of LDS, the same for all lanes; a block of 64 pairs before this wave's also counts its equals
    const pair32 p = t < m ? list[t] : pair32{0u, ~0u};
    if (t >= m && t < (m + 63) / 64 * 64) list[t].key = ~0u;
    __syncthreads();
    uint32_t rank = 0;
    if (wave * 64 < m) {
      for (int b = 0; b * 64 < m; ++b) {
        const u32x4* two = reinterpret_cast<const u32x4*>(list + 64 * b);
        const int half = (min(64, m - 64 * b) + 1) / 2;
        if (b < wave) {
#pragma unroll 8
          for (int j = 0; j < 32; ++j) {
            const u32x4 v = two[j];
            rank += (uint32_t)(v[1] <= p.key) + (uint32_t)(v[3] <= p.key);
          }
        } else if (b > wave) {
#pragma unroll 4
          for (int j = 0; j < half; ++j) {
            const u32x4 v = two[j];
            rank += (uint32_t)(v[1] < p.key) + (uint32_t)(v[3] < p.key);
          }
        } else {
#pragma unroll 4
          for (int j = 0; j < half; ++j) {
            const u32x4 v = two[j];
            rank += (uint32_t)(v[1] < p.key || (v[1] == p.key && 2 * j < lane)) + (uint32_t)(v[3] < p.key || (v[3] == p.key && 2 * j + 1 < lane));
          }
        }
      }
    }
    __syncthreads();
    if (t < m) list[rank] = p;
    __syncthreads();
    return;
  }
  const int items = (m + THREADS - 1) / THREADS, base = wave * 64 * items + lane;
  const int passes = (bits + SMALL_DIGIT - 1) / SMALL_DIGIT, digit = max(MIN_DIGIT, (bits + passes - 1) / passes), bins = 1 << digit;
  uint16_t* part = (uint16_t*)region;                    // [wave][bin], as in k_sort_scatter
  uint32_t* place = (uint32_t*)(region + WAVES * 2 * bins);
  pair32 p[SMALL_ITEMS];
#pragma unroll
  for (int u = 0; u < SMALL_ITEMS; ++u) p[u] = u < items && base + 64 * u < m ? list[base + 64 * u] : pair32{0u, least};
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * digit;
    for (int k = t; k < WAVES * bins / 8; k += THREADS) reinterpret_cast<u32x4*>(part)[k] = u32x4{0, 0, 0, 0};
    __syncthreads();
    uint32_t rank[SMALL_ITEMS];
#pragma unroll
    for (int u = 0; u < SMALL_ITEMS; ++u) {
      if (u >= items) break;
      const bool in = base + 64 * u < m;
      const uint32_t d = ((p[u].key - least) >> shift) & (uint32_t)(bins - 1);
      const uint64_t peers = same_digit(d, digit, in);
      const int leader = in ? __ffsll((unsigned long long)peers) - 1 : lane;
      uint32_t seen = 0;
      if (in && lane == leader) {
        seen = part[wave * bins + d];
        part[wave * bins + d] = (uint16_t)(seen + (uint32_t)__popcll(peers));
      }
      rank[u] = __shfl(seen, leader) + (uint32_t)__popcll(peers & ((1ULL << lane) - 1));
    }
    __syncthreads();
    // a thread's two neighbouring bins lie in one word, and their counts (at most SMALL_N) add up without a carry
    uint32_t total = 0;
    if (2 * t < bins) {
      uint32_t* two = reinterpret_cast<uint32_t*>(part) + t;
      uint32_t c[WAVES];
#pragma unroll
      for (int w = 0; w < WAVES; ++w) c[w] = two[w * (bins >> 1)];
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        two[w * (bins >> 1)] = total;
        total += c[w];
      }
    }
    const uint32_t mine = (total & 0xffff) + (total >> 16), inc = wave_inclusive(mine);
    uint32_t all;
    const uint32_t run = small_offsets<THREADS>((uint32_t)__builtin_amdgcn_readlane((int)inc, 63), wave_sum, &all) + inc - mine;
    if (2 * t < bins) {
      place[2 * t] = run;
      place[2 * t + 1] = run + (total & 0xffff);
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < SMALL_ITEMS; ++u) {
      if (u >= items) break;
      if (base + 64 * u < m) {
        const uint32_t d = ((p[u].key - least) >> shift) & (uint32_t)(bins - 1);
        list[place[d] + part[wave * bins + d] + rank[u]] = p[u];
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < SMALL_ITEMS; ++u) {
      if (u >= items) break;
      if (base + 64 * u < m) p[u] = list[base + 64 * u];
    }
  }
}

// heads[r] = where the r-th run of equal keys begins, heads[distinct] = m; returns distinct
template <int THREADS>
__device__ __forceinline__ uint32_t small_heads(const pair32* list, int m, uint16_t* heads, uint32_t* wave_sum) {
  const int lane = threadIdx.x & 63, items = (m + THREADS - 1) / THREADS, base = (threadIdx.x >> 6) * 64 * items + lane;
  uint64_t take[SMALL_ITEMS];
  uint32_t mine = 0, distinct;
#pragma unroll
  for (int u = 0; u < SMALL_ITEMS; ++u) {
    if (u >= items) break;
    const int i = base + 64 * u;
    take[u] = __ballot(i < m && (i == 0 || list[i - 1].key != list[i].key));
    mine += (uint32_t)__popcll(take[u]);
  }
  uint32_t run = small_offsets<THREADS>(mine, wave_sum, &distinct);
#pragma unroll
  for (int u = 0; u < SMALL_ITEMS; ++u) {
    if (u >= items) break;
    if ((take[u] >> lane) & 1) heads[run + (uint32_t)__popcll(take[u] & ((1ULL << lane) - 1))] = (uint16_t)(base + 64 * u);
    run += (uint32_t)__popcll(take[u]);
  }
  if (threadIdx.x == 0) heads[distinct] = (uint16_t)m;
  __syncthreads();
  return distinct;
}

// Adds the rows of `runs` runs and hands each sum to put(run, acc, col, own).  begin(r), end(r): the run's pairs; pos(k): the position of
// pair k.  A team of 2^log_l lanes takes a run; what is longer than SMALL_RUN waits for the whole workgroup, whose teams take a
// consecutive part each.  All threads call it.
template <int THREADS, class TI, int VEC, class B, class E, class P, class W>
__device__ __forceinline__ void small_sums(const small_args& a, int runs, B begin, E end, P pos, W put, float* parts, uint32_t* queue, int* queued) {
  const int t = threadIdx.x, teams = THREADS >> a.log_l, team = t >> a.log_l, tl = t & ((1 << a.log_l) - 1);
  const int c = ((int)(blockIdx.x % (uint32_t)a.col_blocks) << a.log_l) + tl;
  const int col = VEC == 1 ? c : min(c * VEC, a.width - VEC), own = c * VEC - col;
  const bool live = c < a.chunks;
  const TI* g = (const TI*)a.g + (live ? col : 0);
  auto sum = [&](float (&acc)[VEC], int b, int e) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    for (int k = b; k < e; k += SEG_U) {
      raw_chunk<VEC, TI> v[SEG_U];
#pragma unroll
      for (int u = 0; u < SEG_U; ++u) v[u].load(g + (int64_t)pos(min(k + u, e - 1)) * a.ld_g);
#pragma unroll
      for (int u = 0; u < SEG_U; ++u)
        if (k + u < e) v[u].add_to(acc);
    }
  };
  float acc[VEC];
  for (int q0 = 0; q0 < runs; q0 += 64) {          // 64 runs at a time: the queue's room
    for (int r = q0 + team; r < min(runs, q0 + 64); r += teams) {
      const int b = begin(r), e = end(r);
      if (e - b > SMALL_RUN) {
        if (tl == 0) queue[atomicAdd(queued, 1)] = (uint32_t)r;
      } else if (live) {
        sum(acc, b, e);
        put(r, acc, col, own);
      }
    }
    __syncthreads();
    const int todo = *queued, most = min(teams, SMALL_TEAMS);
    for (int q = 0; q < todo; ++q) {
      const int r = (int)queue[q], b = begin(r), e = end(r), each = (e - b + most - 1) / most;
      if (team < most && live) {
        sum(acc, min(e, b + team * each), min(e, b + (team + 1) * each));
#pragma unroll
        for (int j = 0; j < VEC; ++j) parts[t * VEC + j] = acc[j];
      }
      __syncthreads();
      if (team == 0 && live) {
#pragma unroll 4
        for (int k = 1; k < most; ++k)
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] += parts[((k << a.log_l) + tl) * VEC + j];
        put(r, acc, col, own);
      }
      __syncthreads();
    }
    if (q0 + 64 < runs) {
      if (t == 0) *queued = 0;
      __syncthreads();
    }
  }
}

template <int THREADS, class TI, class TO, int VEC, bool ACCUMULATE>
__global__ __launch_bounds__(THREADS) void k_small(small_args a, int bits) {
  extern __shared__ __align__(16) char lds[];
  __shared__ uint32_t wave_sum[THREADS / 64], queue[64];
  __shared__ int queued;
  const small_lds at = small_layout(THREADS, a.n);
  pair32* list = (pair32*)lds;
  uint16_t* heads = (uint16_t*)(lds + at.heads);
  char* region = lds + at.region;
  const int t = threadIdx.x, lane = t & 63, items = (a.n + THREADS - 1) / THREADS, base = (t >> 6) * 64 * items + lane;
  const uint32_t none = (uint32_t)a.num_rows, share = gridDim.x / (uint32_t)a.col_blocks, sh = blockIdx.x / (uint32_t)a.col_blocks;
  uint32_t key[SMALL_ITEMS];
  small_keys<THREADS>(a, base, items, key);
  // this workgroup's rows of the table, for the zeros
  const int64_t row0 = a.zero_rows ? a.num_rows * (int64_t)blockIdx.x / gridDim.x : 0;
  const int zeros = a.zero_rows ? (int)(a.num_rows * (int64_t)(blockIdx.x + 1) / gridDim.x - row0) : 0;
  uint32_t* map = (uint32_t*)region;
  for (int k = t; k < (zeros + 31) / 32; k += THREADS) map[k] = 0;
  if (t == 0) queued = 0;
  // the pairs that a hash gives this workgroup, in the order of their positions
  uint64_t take[SMALL_ITEMS];
  uint32_t mine = 0, m;
#pragma unroll
  for (int u = 0; u < SMALL_ITEMS; ++u) {
    if (u >= items) break;
    take[u] = __ballot(key[u] != none && __umulhi(small_hash(key[u]), share) == sh);
    mine += (uint32_t)__popcll(take[u]);
  }
  uint32_t run = small_offsets<THREADS>(mine, wave_sum, &m);
#pragma unroll
  for (int u = 0; u < SMALL_ITEMS; ++u) {
    if (u >= items) break;
    if ((take[u] >> lane) & 1) list[run + (uint32_t)__popcll(take[u] & ((1ULL << lane) - 1))] = pair32{(uint32_t)(base + 64 * u), key[u]};
    run += (uint32_t)__popcll(take[u]);
    const int64_t r = (int64_t)key[u] - row0;
    if (key[u] != none && r >= 0 && r < zeros) atomicOr(&map[r >> 5], 1u << (r & 31));
  }
  __syncthreads();
  // zeros: a team of lanes takes a row, or a lane does where a row is shorter than 16 bytes
  if (zeros > 0) {
    const int bytes = a.width * (int)sizeof(TO), pieces = bytes < 16 ? 1 : (bytes + 15) / 16;
    int lz = 0;
    while (lz < 6 && (1 << lz) < pieces) ++lz;
    for (int r = t >> lz; r < zeros; r += THREADS >> lz) {
      if ((map[r >> 5] >> (r & 31)) & 1) continue;
      TO* o = (TO*)a.out + (row0 + r) * a.ld_out;
      if (bytes < 16) {
        for (int j = 0; j < a.width; ++j) o[j] = (TO)0.f;
      } else {
        for (int k = t & ((1 << lz) - 1); k < pieces; k += 1 << lz) store16((char*)o + min(16 * k, bytes - 16), u32x4{0, 0, 0, 0});
      }
    }
    __syncthreads();
  }
  small_sort<THREADS>(list, (int)m, 0u, bits, region, wave_sum);
  const int distinct = (int)small_heads<THREADS>(list, (int)m, heads, wave_sum);
  small_sums<THREADS, TI, VEC>(
      a, distinct, [&](int r) { return (int)heads[r]; }, [&](int r) { return (int)heads[r + 1]; }, [&](int k) { return list[k].pos; },
      [&](int r, const float (&acc)[VEC], int col, int own) {
        TO* o = (TO*)a.out + (int64_t)list[heads[r]].key * a.ld_out + col;
        float f[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[j] = acc[j] * a.scale;
        if constexpr (ACCUMULATE) {
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            if (j >= own) o[j] = (TO)((float)o[j] + f[j]);
        } else {
          store_chunk<VEC, TO>(o, f);
        }
      },
      (float*)region, queue, &queued);
}

// what k_range_sort leaves for k_range_sums
struct range_work {
  uint16_t* pos;                // [n] positions in the order of (id, position)
  uint16_t* heads;              // [n] per range, at its first pair's place: where its runs begin, from there
  uint32_t* key;                // [n] the runs' ids, beside heads
  uint32_t* first;              // [ranges + 1] a range's first pair; how many there are
  uint32_t* distinct;           // [ranges]
};
template <int THREADS>
__global__ __launch_bounds__(THREADS) void k_range_sort(small_args a, range_work w) {
  extern __shared__ __align__(16) char lds[];
  __shared__ uint32_t wave_sum[THREADS / 64];
  const small_lds at = small_layout(THREADS, a.n);
  pair32* list = (pair32*)lds;
  uint16_t* heads = (uint16_t*)(lds + at.heads);
  const int t = threadIdx.x, lane = t & 63, items = (a.n + THREADS - 1) / THREADS, base = (t >> 6) * 64 * items + lane;
  uint32_t key[SMALL_ITEMS];
  small_keys<THREADS>(a, base, items, key);
  const uint32_t lo = (uint32_t)(a.num_rows * (int64_t)blockIdx.x / gridDim.x), hi = (uint32_t)(a.num_rows * (int64_t)(blockIdx.x + 1) / gridDim.x);
  uint64_t take[SMALL_ITEMS];
  uint32_t mine = 0, both;            // what is below the range is counted in the upper half (at most SMALL_N in each)
#pragma unroll
  for (int u = 0; u < SMALL_ITEMS; ++u) {
    if (u >= items) break;
    take[u] = __ballot(key[u] >= lo && key[u] < hi);
    mine += (uint32_t)__popcll(take[u]) + ((uint32_t)__popcll(__ballot(key[u] < lo)) << 16);
  }
  uint32_t run = small_offsets<THREADS>(mine, wave_sum, &both) & 0xffff;
  const uint32_t m = both & 0xffff, before = both >> 16;
#pragma unroll
  for (int u = 0; u < SMALL_ITEMS; ++u) {
    if (u >= items) break;
    if ((take[u] >> lane) & 1) list[run + (uint32_t)__popcll(take[u] & ((1ULL << lane) - 1))] = pair32{(uint32_t)(base + 64 * u), key[u]};
    run += (uint32_t)__popcll(take[u]);
  }
  __syncthreads();
  int bits = 1;
  while (((hi - lo) >> bits) != 0) ++bits;
  small_sort<THREADS>(list, (int)m, lo, bits, lds + at.region, wave_sum);
  const uint32_t distinct = small_heads<THREADS>(list, (int)m, heads, wave_sum);
  for (int i = t; i < (int)m; i += THREADS) w.pos[before + i] = (uint16_t)list[i].pos;
  for (int r = t; r < (int)distinct; r += THREADS) {
    w.heads[before + r] = heads[r];
    w.key[before + r] = list[heads[r]].key;
  }
  if (t == 0) {
    w.first[blockIdx.x] = before;
    w.distinct[blockIdx.x] = distinct;
    if (blockIdx.x == gridDim.x - 1) w.first[gridDim.x] = before + m;
  }
}

constexpr int RANGE_RUNS = 64;        // runs whose places are looked up together
template <int THREADS, class TI, class TO, int VEC>
__global__ __launch_bounds__(THREADS) void k_range_sums(small_args a, range_work w, int ranges, int64_t* __restrict__ ids, int32_t* __restrict__ count) {
  __shared__ uint32_t wave_sum[THREADS / 64], queue[64], row[MAX_RANGES + 1], first[MAX_RANGES + 1], begin[2 * RANGE_RUNS], key[RANGE_RUNS];
  __shared__ int queued;
  __shared__ float parts[THREADS * 8];
  static_assert(MAX_RANGES <= THREADS && 2 * RANGE_RUNS <= THREADS, "a thread per range, and per end of a run");
  const int t = threadIdx.x, lane = t & 63;
  const uint32_t mine = t < ranges ? w.distinct[t] : 0u, inc = wave_inclusive(mine);
  if (t <= MAX_RANGES) first[t] = t <= ranges ? w.first[t] : 0u;
  if (THREADS == MAX_RANGES && t == 0 && ranges == MAX_RANGES) first[MAX_RANGES] = w.first[MAX_RANGES];
  if (t == 0) queued = 0;
  uint32_t all;
  const uint32_t run = small_offsets<THREADS>((uint32_t)__builtin_amdgcn_readlane((int)inc, 63), wave_sum, &all) + inc - mine;
  if (t < MAX_RANGES) row[t] = run;                 // rows of the ranges before
  if (t == 0) row[MAX_RANGES] = all;
  __syncthreads();
  if (blockIdx.x == 0 && t == 0) *count = (int32_t)all;
  const int share = (int)(gridDim.x / (uint32_t)a.col_blocks), sh = (int)(blockIdx.x / (uint32_t)a.col_blocks);
  // runs sh, sh + share, ..: frequent ids are often neighbours
  const int mine_all = ((int)all - sh + share - 1) / share;
  for (int r0 = 0; r0 < mine_all; r0 += RANGE_RUNS) {
    const int runs = min(RANGE_RUNS, mine_all - r0);
    if (t < 2 * runs) {         // where a run begins, and the one after it, which is its end
      const int r = sh + (r0 + (t >> 1)) * share + (t & 1);
      int k = 0;                // its range: row[k] <= r < row[k + 1]
#pragma unroll
      for (int step = MAX_RANGES / 2; step; step >>= 1) k += (int)row[k + step] <= r ? step : 0;
      const bool none = (uint32_t)r >= all;
      const uint32_t at = first[k] + (uint32_t)r - row[k];
      begin[t] = none ? first[ranges] : first[k] + w.heads[at];
      if (!(t & 1)) key[t >> 1] = w.key[at];
    }
    __syncthreads();
    small_sums<THREADS, TI, VEC>(
        a, runs, [&](int r) { return (int)begin[2 * r]; }, [&](int r) { return (int)begin[2 * r + 1]; }, [&](int k) { return w.pos[k]; },
        [&](int r, const float (&acc)[VEC], int col, int own) {
          const int64_t to = sh + (int64_t)(r0 + r) * share;
          if (col == 0) ids[to] = (int64_t)key[r];
          float f[VEC];
#pragma unroll
          for (int j = 0; j < VEC; ++j) f[j] = acc[j] * a.scale;
          store_chunk<VEC, TO>((TO*)a.out + to * a.ld_out + col, f);
        },
        parts, queue, &queued);
    __syncthreads();
    if (t == 0) queued = 0;
    __syncthreads();
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------
struct sort_plan { int passes, digit, items; int64_t tiles; };
sort_plan plan_sort(int64_t n, int64_t num_rows) {
  int bits = 1;
  while (bits < 32 && (num_rows >> bits) != 0) ++bits;        // keys 0 .. num_rows
  sort_plan s;
  s.passes = (bits + MAX_DIGIT - 1) / MAX_DIGIT;
  s.digit = std::max(MIN_DIGIT, (bits + s.passes - 1) / s.passes);
  for (s.items = 1;; s.items *= 2) {
    s.tiles = ceil_div64(n, SORT_THREADS * s.items);
    if (s.items == 4 || (s.tiles * 4 << s.digit) <= (s.items == 1 ? ONE_BYTES : TWO_BYTES)) break;
  }
  return s;
}
int log_lanes(int64_t chunks, int most) {       // the smallest team that holds a row's chunks, at most 2^most lanes
  int l = 0;
  while (l < most && (1 << l) < chunks) ++l;
  return l;
}
// Pairs per window: long windows leave fewer sums to join, short ones make more teams; the longest of 8 .. 64 that still gives the
// chip 4096 waves (16 per CU) of 16-bit columns.
int window_of(int64_t n, int64_t width) {
  const int64_t chunks = ceil_div64(width, 8);
  const int l = log_lanes(chunks, 8);
  const int64_t lanes = ceil_div64(chunks, 1 << l) << l;
  int w = 64;
  while (w > 8 && (ceil_div64(n, w) * lanes < 4096 * 64 || (256 >> l) * w > SEG_PAIRS)) w >>= 1;
  return w;
}
struct work_layout { int64_t a, b, counts, totals, heads, rank, part, bytes; };
work_layout layout(int64_t n, int64_t width, int64_t num_rows) {
  const sort_plan s = plan_sort(n, num_rows);
  work_layout l{};
  int64_t o = 0;
  auto take = [&](int64_t bytes) { const int64_t at = o; o += (bytes + 255) / 256 * 256; return at; };
  l.a = take(n * 8);
  l.b = take(n * 8);
  l.counts = take(s.tiles * 4 << s.digit);
  l.totals = take(4LL << s.digit);
  l.heads = take(s.tiles * 4);
  l.rank = take(n * 4);
  l.part = take(2 * ceil_div64(n, window_of(n, width)) * width * 4);
  l.bytes = o;
  return l;
}
// teams of lanes over the columns, and the workgroups of the windows' sums and of their joins
struct sums_grid { int chunks, log_l, col_blocks; int64_t blocks; };
sums_grid segment_grid(int64_t n, int64_t width, int vec) {
  sums_grid g;
  g.chunks = (int)(width < vec ? width : ceil_div64(width, vec));
  g.log_l = log_lanes(g.chunks, 8);
  g.col_blocks = (int)ceil_div64(g.chunks, 1 << g.log_l);
  g.blocks = ceil_div64(ceil_div64(n, window_of(n, width)), 256 >> g.log_l) * g.col_blocks;
  return g;
}
sums_grid join_grid(int64_t n, int64_t width) {
  sums_grid g;
  g.chunks = (int)ceil_div64(width, 4);
  g.log_l = log_lanes(g.chunks, 6);
  g.col_blocks = (int)ceil_div64(g.chunks, 1 << g.log_l);
  g.blocks = ceil_div64(ceil_div64(n, window_of(n, width)) - 1, JOIN_THREADS >> g.log_l) * g.col_blocks;
  return g;
}
template <class TI, class TO, int VEC>
int launch_sums_vec(seg_args a, bool accumulate, hipStream_t stream) {
  const sums_grid grid = segment_grid(a.n, a.width, elems16<TI>);
  a.chunks = grid.chunks;
  a.log_l = grid.log_l;
  a.col_blocks = grid.col_blocks;
  const bool past = VEC > 1 && past_gradient(a.n * a.width * (int64_t)sizeof(TI));
  auto* kernel = accumulate ? (past ? k_segment_sum<TI, TO, VEC, true, VEC != 1> : k_segment_sum<TI, TO, VEC, true, false>)
                            : (past ? k_segment_sum<TI, TO, VEC, false, VEC != 1> : k_segment_sum<TI, TO, VEC, false, false>);
  kernel<<<(unsigned)grid.blocks, 256, 0, stream>>>(a);
  ORCA_LAUNCH_CHECK();
  return ORCA_OK;
}
template <class TI, class TO>
int launch_sums(seg_args a, bool accumulate, hipStream_t stream) {
  constexpr int VEC = elems16<TI>;
  if (int rc = a.width >= VEC ? launch_sums_vec<TI, TO, VEC>(a, accumulate, stream) : launch_sums_vec<TI, TO, 1>(a, accumulate, stream)) return rc;
  const sums_grid grid = join_grid(a.n, a.width);
  if (grid.blocks == 0) return ORCA_OK;          // (one window)
  a.chunks = grid.chunks;
  a.log_l = grid.log_l;
  a.col_blocks = grid.col_blocks;
  if (accumulate) k_segment_join<TO, true><<<(unsigned)grid.blocks, JOIN_THREADS, 0, stream>>>(a);
  else k_segment_join<TO, false><<<(unsigned)grid.blocks, JOIN_THREADS, 0, stream>>>(a);
  ORCA_LAUNCH_CHECK();
  return ORCA_OK;
}

bool is_tiny(int64_t n, int64_t width) { return n <= TINY_N && n * width <= TINY_VALUES; }        // for the small workgroups
bool is_small(int64_t n, int64_t width) { return n <= SMALL_N && n * width <= SMALL_VALUES; }
// Whether k_small's workgroups mark the rows and zero the others: as many rows as they can mark, and no more bytes than pay a launch of
// its own, whose stores run at the full rate.  Marked and filled ahead, us, workgroups of 256 threads (20 ids in rows of 49 fp32): 16 MB 9.0
// and 8.5, 24 MB 10.9 and 9.3, 64 MB 19.6 and 14.3 (rows of 256 bf16: 8.2 and 8.7, 9.6 and 9.8, 15.9 and 14.3); of 1024 threads (2500 ids in
// rows of 8 fp32): 24 MB 15.0 and 16.7, 64 MB 20.4 and 22.4, 128 MB 27.6 and 30.1, 160 MB 33.4 and 33.8.
bool maps(bool tiny, int64_t num_rows, int64_t bytes) { return num_rows <= 256LL * SMALL_MAP && bytes <= (tiny ? 20 : 160) * MB; }
template <class T> void columns(small_args* a) {
  constexpr int VEC = elems16<T>;
  a->chunks = a->width < VEC ? a->width : (a->width + VEC - 1) / VEC;
  // half a wave per row and column block, so that a hub's rows meet more teams (8000 rows of one id, 256 and 2048 fp32: 83 and 86 us, 136
  // and 140 with whole waves; of uniform ids 16 and 38, 16 and 34), while that leaves 16 shares of the ids (2000 ids of 8000 fp32 40, halves 49)
  a->log_l = log_lanes(a->chunks, a->chunks <= 512 ? 5 : 6);
  a->col_blocks = (int)ceil_div64(a->chunks, 1 << a->log_l);
}
int key_bits(int64_t num_rows) {
  int bits = 1;
  while ((num_rows >> bits) != 0) ++bits;
  return bits;
}
// A kernel's dynamic LDS is allowed once per device, and noted when that has happened: another thread's call (autograd runs a backward
// pass on its own) does it again rather than launch ahead of it.
int allow_lds(std::atomic<bool> (&done)[64], const void* kernel, int bytes) {
  int dev = 0;
  ORCA_HIP_TRY(hipGetDevice(&dev));
  const bool known = dev >= 0 && dev < 64;
  if (known && done[dev].load(std::memory_order_acquire)) return ORCA_OK;
  ORCA_HIP_TRY(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (known) done[dev].store(true, std::memory_order_release);
  return ORCA_OK;
}
template <int THREADS, class TI, class TO, int VEC, bool ACCUMULATE>
int launch_small(small_args a, hipStream_t stream) {
  static std::atomic<bool> done[64];
  if (int rc = allow_lds(done, (const void*)k_small<THREADS, TI, TO, VEC, ACCUMULATE>, small_layout(THREADS, THREADS * SMALL_ITEMS).bytes)) return rc;
  columns<TI>(&a);
  // workgroups: four ids, 16 KB of zeros or 65,536 rows each, at most one per CU (and one for each column block)
  int64_t want = ceil_div64(a.n, 4) * a.col_blocks;
  if (a.zero_rows) want = std::max({want, ceil_div64(a.num_rows * a.width * (int64_t)sizeof(TO), 16384), ceil_div64(a.num_rows, SMALL_MAP)});
  const int64_t shares = std::max<int64_t>(1, ceil_div64(std::min<int64_t>(want, 256), a.col_blocks));
  k_small<THREADS, TI, TO, VEC, ACCUMULATE>
      <<<(unsigned)(shares * a.col_blocks), THREADS, small_layout(THREADS, a.n).bytes, stream>>>(a, key_bits(a.num_rows));
  ORCA_LAUNCH_CHECK();
  return ORCA_OK;
}
template <int THREADS, class TI, class TO>
int small_dense(const small_args& a, bool accumulate, hipStream_t stream) {
  constexpr int VEC = elems16<TI>;
  if (a.width >= VEC) return accumulate ? launch_small<THREADS, TI, TO, VEC, true>(a, stream) : launch_small<THREADS, TI, TO, VEC, false>(a, stream);
  return accumulate ? launch_small<THREADS, TI, TO, 1, true>(a, stream) : launch_small<THREADS, TI, TO, 1, false>(a, stream);
}

range_work range_layout(char* ws, int64_t n, int64_t* bytes) {
  range_work w;
  int64_t o = 0;
  auto take = [&](int64_t b) { char* p = ws + o; o += (b + 255) / 256 * 256; return p; };
  w.pos = (uint16_t*)take(2 * n);
  w.heads = (uint16_t*)take(2 * n);
  w.key = (uint32_t*)take(4 * n);
  w.first = (uint32_t*)take(4 * (MAX_RANGES + 1));
  w.distinct = (uint32_t*)take(4 * MAX_RANGES);
  *bytes = o;
  return w;
}
template <int THREADS> int launch_range_sort(const small_args& a, const range_work& w, int ranges, hipStream_t stream) {
  static std::atomic<bool> done[64];
  if (int rc = allow_lds(done, (const void*)k_range_sort<THREADS>, small_layout(THREADS, THREADS * SMALL_ITEMS).bytes)) return rc;
  k_range_sort<THREADS><<<(unsigned)ranges, THREADS, small_layout(THREADS, a.n).bytes, stream>>>(a, w);
  ORCA_LAUNCH_CHECK();
  return ORCA_OK;
}
template <class TI, class TO>
int small_rows(small_args a, char* ws, int64_t* ids, int32_t* count, hipStream_t stream) {
  constexpr int VEC = elems16<TI>;
  columns<TI>(&a);
  int64_t bytes;
  const range_work w = range_layout(ws, a.n, &bytes);
  const int ranges = (int)std::min<int64_t>(MAX_RANGES, ceil_div64(a.n, 4));
  if (int rc = is_tiny(a.n, a.width) ? launch_range_sort<TINY_THREADS>(a, w, ranges, stream) : launch_range_sort<SMALL_THREADS>(a, w, ranges, stream)) return rc;
  // a run per team, no more than are looked up at once, and at most a workgroup per CU (two small ones; one for each column block)
  const int threads = is_tiny(a.n, a.width) ? TINY_THREADS : SMALL_THREADS;
  const int64_t runs = std::min(RANGE_RUNS, threads >> a.log_l);
  const int64_t shares = std::max<int64_t>(1, std::min(ceil_div64(a.n, runs), ceil_div64(is_tiny(a.n, a.width) ? 512 : 256, a.col_blocks)));
  const unsigned grid = (unsigned)(shares * a.col_blocks);
  auto* kernel = is_tiny(a.n, a.width) ? (a.width >= VEC ? k_range_sums<TINY_THREADS, TI, TO, VEC> : k_range_sums<TINY_THREADS, TI, TO, 1>)
                               : (a.width >= VEC ? k_range_sums<SMALL_THREADS, TI, TO, VEC> : k_range_sums<SMALL_THREADS, TI, TO, 1>);
  kernel<<<grid, (unsigned)threads, 0, stream>>>(a, w, ranges, ids, count);
  ORCA_LAUNCH_CHECK();
  return ORCA_OK;
}

// f(gradient element, output element) for the pairs of types that check_gradient lets through
template <class F> int by_types(int g_dtype, int out_dtype, F f) {
  if (g_dtype == ORCA_F32) return f(float{}, float{});
  if (g_dtype == ORCA_BF16) return out_dtype == ORCA_F32 ? f(__bf16{}, float{}) : f(__bf16{}, __bf16{});
  return out_dtype == ORCA_F32 ? f(_Float16{}, float{}) : f(_Float16{}, _Float16{});
}

int64_t workspace_bytes_of(int64_t n, int64_t width, int64_t num_rows) {
  if (!is_small(n, width)) return layout(n, width, num_rows).bytes;
  int64_t bytes;
  range_layout(nullptr, n, &bytes);
  return bytes;
}

int check_gradient(const char* who, const void* g, int g_dtype, int64_t ld_g, const int64_t* idx64, const int32_t* idx32, int64_t n, int64_t width,
                   int64_t num_rows, int out_dtype, const void* workspace, int64_t workspace_bytes) {
  ORCA_REQUIRE(n >= 0 && n < (1LL << 31) && num_rows >= 0 && num_rows < (1LL << 31) - 1, "%s: %lld ids, %lld rows (both under 2^31 - 1)", who,
               (long long)n, (long long)num_rows);
  ORCA_REQUIRE(width >= 1 && width <= MAX_WIDTH, "%s: width %lld (1 to %lld)", who, (long long)width, (long long)MAX_WIDTH);
  ORCA_REQUIRE(g_dtype >= ORCA_F32 && g_dtype <= ORCA_F16 && (out_dtype == g_dtype || out_dtype == ORCA_F32),
               "%s: gradient of type %d into type %d (the same, or fp32)", who, g_dtype, out_dtype);
  if (n == 0) return ORCA_OK;
  ORCA_REQUIRE(g && (idx64 != nullptr) != (idx32 != nullptr), "%s: null gradient, or not exactly one list of ids", who);
  ORCA_REQUIRE(ld_g >= 0, "%s: negative row stride", who);
  ORCA_REQUIRE(is_small(n, width) || (fits_launch(segment_grid(n, width, g_dtype == ORCA_F32 ? elems16<float> : elems16<__bf16>).blocks, 256) &&
                                      fits_launch(join_grid(n, width).blocks, JOIN_THREADS)),
               "%s: %lld ids of width %lld are too many for one call", who, (long long)n, (long long)width);
  ORCA_REQUIRE(((uintptr_t)workspace & 15) == 0, "%s: the workspace is not 16-byte aligned", who);
  ORCA_REQUIRE(workspace && workspace_bytes >= workspace_bytes_of(n, width, num_rows), "%s: the workspace holds %lld of %lld bytes", who,
               (long long)workspace_bytes, (long long)workspace_bytes_of(n, width, num_rows));
  return ORCA_OK;
}

// the pieces of a fill that launch `i` of `launches` takes, and the workgroups for them.  (Even shares: a million rows of 400 bytes 81 us;
// 80 MB in the sort's launches and the rest ahead of the sums: 92; everything ahead of the sort: 100.)  At most FILL_BLOCKS of them, which
// then go round: with the sort's tiles that stays within a launch (in a table with gaps every row is a piece).
constexpr int64_t FILL_BLOCKS = 1 << 22;
static_assert((FILL_BLOCKS + (1LL << 31) / (4 * SORT_THREADS)) * SORT_THREADS < (1LL << 32), "threads of a launch");
unsigned fill_share(fill_job* f, int64_t pieces, int threads, int i, int launches) {
  f->from = pieces * i / launches;
  f->to = pieces * (i + 1) / launches;
  return (unsigned)std::min<int64_t>(ceil_div64(f->to - f->from, threads / 256), FILL_BLOCKS);
}
int launch_fill(fill_job f, int64_t pieces, hipStream_t stream) {
  const unsigned blocks = fill_share(&f, pieces, 256, 0, 1);
  if (blocks) k_fill<<<blocks, 256, 0, stream>>>(f);
  ORCA_LAUNCH_CHECK();
  return ORCA_OK;
}

template <class F> void by_items(int items, F f) {
  if (items == 1) f(std::integral_constant<int, 1>{});
  else if (items == 2) f(std::integral_constant<int, 2>{});
  else f(std::integral_constant<int, 4>{});
}

// sorts (id, position), zeroes the fill's pieces on the way; *sorted = where the result lies
int sort_positions(const int64_t* idx64, const int32_t* idx32, int64_t n, int64_t num_rows, int64_t padding, char* ws, const work_layout& l,
                   fill_job fill, int64_t pieces, const pair32** sorted, hipStream_t stream) {
  const sort_plan s = plan_sort(n, num_rows);
  sort_src src{idx64, idx32, nullptr, n, num_rows, padding};
  uint32_t* counts = (uint32_t*)(ws + l.counts);
  uint32_t* totals = s.items == 4 && s.tiles > DIRECT_TILES ? (uint32_t*)(ws + l.totals) : nullptr;
  pair32* buf[2] = {(pair32*)(ws + l.a), (pair32*)(ws + l.b)};
  for (int p = 0; p < s.passes; ++p) {
    unsigned extra = fill_share(&fill, pieces, SORT_THREADS, 2 * p, 2 * s.passes);
    by_items(s.items, [&](auto items) {
      k_sort_count<items><<<(unsigned)s.tiles + extra, SORT_THREADS, 0, stream>>>(src, p * s.digit, 1 << s.digit, counts, (int)s.tiles, fill);
    });
    ORCA_LAUNCH_CHECK();
    if (totals) {
      k_sort_columns<<<((1 << s.digit) + 63) / 64, 64, 0, stream>>>(counts, s.tiles, 1 << s.digit, totals);
      ORCA_LAUNCH_CHECK();
    }
    extra = fill_share(&fill, pieces, SORT_THREADS, 2 * p + 1, 2 * s.passes);
    by_items(s.items, [&](auto items) {
      k_sort_scatter<items><<<(unsigned)s.tiles + extra, SORT_THREADS, 0, stream>>>(src, p * s.digit, s.digit, counts, totals, buf[p & 1], (int)s.tiles,
                                                                                    fill);
    });
    ORCA_LAUNCH_CHECK();
    src.pairs = buf[p & 1];
  }
  *sorted = src.pairs;
  return ORCA_OK;
}
}  // namespace

ORCA_API int orca_embedding_forward(const void* table, int dtype, int64_t n_rows, int64_t width, int64_t ld, const int64_t* idx64,
                                    const int32_t* idx32, int64_t n, float scale, void* out, void* stream_) {
  ORCA_REQUIRE(dtype >= ORCA_F32 && dtype <= ORCA_F16, "orca_embedding_forward: unknown type %d", dtype);
  ORCA_REQUIRE(n >= 0 && n_rows >= 0 && ld >= 0, "orca_embedding_forward: negative size");
  ORCA_REQUIRE(width >= 1 && width <= MAX_WIDTH, "orca_embedding_forward: width %lld (1 to %lld)", (long long)width, (long long)MAX_WIDTH);
  if (n == 0) return ORCA_OK;
  ORCA_REQUIRE(n < (1LL << 40) && (table || n_rows == 0) && out && (idx64 != nullptr) != (idx32 != nullptr),
               "orca_embedding_forward: null table or output, or not exactly one list of ids");
  hipStream_t stream = (hipStream_t)stream_;
  if (dtype == ORCA_F32) return embedding_typed<float>(table, n_rows, width, ld, idx64, idx32, n, scale, out, stream);
  if (dtype == ORCA_BF16) return embedding_typed<__bf16>(table, n_rows, width, ld, idx64, idx32, n, scale, out, stream);
  return embedding_typed<_Float16>(table, n_rows, width, ld, idx64, idx32, n, scale, out, stream);
}

ORCA_API int64_t orca_embedding_backward_workspace_bytes(int64_t n, int64_t width, int64_t num_rows) {
  if (n < 0 || n >= (1LL << 31) || width < 1 || width > MAX_WIDTH || num_rows < 0 || num_rows >= (1LL << 31) - 1) return -1;
  return workspace_bytes_of(n, width, num_rows);
}

ORCA_API int orca_embedding_backward(const void* grad_out, int grad_dtype, int64_t ld_grad, const int64_t* idx64, const int32_t* idx32, int64_t n,
                                     int64_t width, int64_t num_rows, int64_t padding_idx, float scale, int accumulate, void* grad_table,
                                     int table_dtype, int64_t ld_table, void* workspace, int64_t workspace_bytes, void* stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  if (int rc = check_gradient("orca_embedding_backward", grad_out, grad_dtype, ld_grad, idx64, idx32, n, width, num_rows, table_dtype, workspace,
                              workspace_bytes))
    return rc;
  if (num_rows == 0) return ORCA_OK;
  ORCA_REQUIRE(grad_table && (ld_table >= width || num_rows == 1), "orca_embedding_backward: null table, or rows that overlap");
  fill_job fill{};
  int64_t pieces = 0;
  if (!accumulate) {
    const int64_t e = table_dtype == ORCA_F32 ? 4 : 2;
    const bool gaps = ld_table != width && num_rows > 1;
    fill.p = (char*)grad_table;
    fill.bytes = (gaps ? width : num_rows * width) * e;
    fill.pitch = gaps ? ld_table * e : 0;
    fill.per_row = ceil_div64(fill.bytes, FILL_PIECE);
    pieces = (gaps ? num_rows : 1) * fill.per_row;
    fill.past = past_zeros(num_rows * width * e);
  }
  if (n == 0) return launch_fill(fill, pieces, stream);
  const bool marks = !accumulate && maps(is_tiny(n, width), num_rows, num_rows * width * (table_dtype == ORCA_F32 ? 4 : 2));
  if (is_small(n, width)) {
    if (!accumulate && !marks) {
      if (int rc = launch_fill(fill, pieces, stream)) return rc;
    }
    const small_args a{idx64, idx32, num_rows, padding_idx, grad_out, ld_grad, ld_table, grad_table, (int)n, (int)width, 0, 0, 0, marks, scale};
    return by_types(grad_dtype, table_dtype, [&](auto gi, auto go) {
      return is_tiny(n, width) ? small_dense<TINY_THREADS, decltype(gi), decltype(go)>(a, accumulate != 0, stream)
                         : small_dense<SMALL_THREADS, decltype(gi), decltype(go)>(a, accumulate != 0, stream);
    });
  }
  const work_layout l = layout(n, width, num_rows);
  char* ws = (char*)workspace;
  const pair32* s = nullptr;
  if (int rc = sort_positions(idx64, idx32, n, num_rows, padding_idx, ws, l, fill, pieces, &s, stream)) return rc;
  seg_args a{grad_out, ld_grad, n, ld_table, s, nullptr, grad_table, (float*)(ws + l.part), (int)width, 0, 0, window_of(n, width), 0,
             (uint32_t)num_rows, scale};
  return by_types(grad_dtype, table_dtype,
                  [&](auto gi, auto go) { return launch_sums<decltype(gi), decltype(go)>(a, accumulate != 0, stream); });
}

ORCA_API int orca_embedding_backward_rows(const void* grad_out, int grad_dtype, int64_t ld_grad, const int64_t* idx64, const int32_t* idx32, int64_t n,
                                          int64_t width, int64_t num_rows, int64_t padding_idx, float scale, int64_t* ids, void* rows, int rows_dtype,
                                          int32_t* count, void* workspace, int64_t workspace_bytes, void* stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  if (int rc = check_gradient("orca_embedding_backward_rows", grad_out, grad_dtype, ld_grad, idx64, idx32, n, width, num_rows, rows_dtype, workspace,
                              workspace_bytes))
    return rc;
  ORCA_REQUIRE(count && (n == 0 || (ids && rows)), "orca_embedding_backward_rows: null output");
  if (n == 0) return orca_fill_i32(count, 1, 0, stream_);
  if (is_small(n, width)) {
    const small_args a{idx64, idx32, num_rows, padding_idx, grad_out, ld_grad, width, rows, (int)n, (int)width, 0, 0, 0, 0, scale};
    return by_types(grad_dtype, rows_dtype,
                    [&](auto gi, auto go) { return small_rows<decltype(gi), decltype(go)>(a, (char*)workspace, ids, count, stream); });
  }
  const work_layout l = layout(n, width, num_rows);
  char* ws = (char*)workspace;
  const pair32* s = nullptr;
  if (int rc = sort_positions(idx64, idx32, n, num_rows, padding_idx, ws, l, fill_job{}, 0, &s, stream)) return rc;
  const sort_plan plan = plan_sort(n, num_rows);
  const unsigned tiles = (unsigned)plan.tiles;
  uint32_t *rank = (uint32_t*)(ws + l.rank), *heads = (uint32_t*)(ws + l.heads);
  by_items(plan.items, [&](auto items) { k_rank_count<items><<<tiles, SORT_THREADS, 0, stream>>>(s, n, (uint32_t)num_rows, heads); });
  ORCA_LAUNCH_CHECK();
  by_items(plan.items, [&](auto items) { k_rank<items><<<tiles, SORT_THREADS, 0, stream>>>(s, n, (uint32_t)num_rows, heads, rank, ids, count); });
  ORCA_LAUNCH_CHECK();
  seg_args a{grad_out, ld_grad, n, width, s, rank, rows, (float*)(ws + l.part), (int)width, 0, 0, window_of(n, width), 0, (uint32_t)num_rows, scale};
  return by_types(grad_dtype, rows_dtype, [&](auto gi, auto go) { return launch_sums<decltype(gi), decltype(go)>(a, false, stream); });
}
