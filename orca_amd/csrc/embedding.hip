// Embedding rows and their gradient: out[p] = scale * table[ids[p]], and for the table
//   G[v] = round(scale * sum over {p : ids[p] = v} of g[p])
// as a dense table or as (ascending distinct ids, their rows, their number).  The sums are fp32 (each g is 16 or 32 bits wide; the
// one rounding to the output's type is the last step) and their order is fixed by (id, position) alone: the positions are sorted
// by id with a stable radix sort and the sorted list is cut into windows of equal length, so that a hub id with thousands of
// occurrences is spread over as many windows as it needs and two runs give the same bits.  (orca_scatter_add_flagged adds with
// fp32 atomics in whatever order they arrive.)
#include <algorithm>
#include "elem.h"

namespace {
// VEC consecutive elements of a row as floats: one 16-byte access, or single elements (VEC = 1) where a row is shorter than that
template <int VEC, class T> __device__ __forceinline__ void load_chunk(const T* p, float (&f)[VEC]) {
  if constexpr (VEC == 1) f[0] = (float)p[0];
  else unpack16<T>(load16(p), f);
}
template <int VEC, class T> __device__ __forceinline__ void store_chunk(T* p, const float (&f)[VEC]) {
  if constexpr (VEC * sizeof(T) < 16) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) p[j] = (T)f[j];
  } else {
#pragma unroll
    for (int k = 0; k < VEC; k += elems16<T>) store16(p + k, pack16<T>(f + k));
  }
}

constexpr int64_t MAX_WIDTH = 65536;      // x * C of the division below stays under 2^32

// ---- lookup ----------------------------------------------------------------------------------------------------------
// The output is a list of n * C chunks of 16 bytes; the last chunk of a row starts at width - VEC, so that every access is
// whole (it overlaps the one before it: both write the same values).  Rows narrower than a chunk go element by element.
constexpr int LOOK_U = 4;                 // chunks per thread: that many independent id -> row chains
template <class T, int VEC, class I>
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
    store_chunk<VEC, T>(out + at[u], v[u]);
  }
}

template <class T, int VEC, class I>
int launch_embedding(const void* table, int64_t n_rows, int64_t width, int64_t ld, const I* ids, int64_t n, float scale, void* out,
                     hipStream_t stream) {
  const int64_t C = ceil_div64(width, VEC), total = n * C, blocks = ceil_div64(total, 256 * LOOK_U);
  ORCA_REQUIRE(blocks < (1LL << 31), "orca_embedding_forward: %lld rows of %lld values are too many for one call", (long long)n, (long long)width);
  const uint32_t magic = C == 1 ? 0 : (uint32_t)(((1ULL << 32) + C - 1) / C);
  k_embedding<T, VEC, I><<<(unsigned)blocks, 256, 0, stream>>>((const T*)table, n_rows, ld, ids, total, (int)width, (uint32_t)C, magic, scale,
                                                               (T*)out);
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

// ---- sort of the positions by id -------------------------------------------------------------------------------------
// Stable least-significant-digit radix sort of (key, position) pairs; key = the id, or num_rows for what has no row (the padding
// id, ids outside the table): those end up last and are dropped.  A tile is SORT_TILE consecutive pairs of one workgroup; within it
// a wave owns 64 * SORT_ITEMS consecutive pairs and ranks them 64 at a time: the lanes with the same digit find each other with one
// ballot per digit bit.
constexpr int SORT_THREADS = 512, SORT_WAVES = SORT_THREADS / 64, SORT_ITEMS = 4, SORT_TILE = SORT_THREADS * SORT_ITEMS;
constexpr int MAX_DIGIT = 11, MAX_BINS = 1 << MAX_DIGIT;
static_assert(SORT_TILE <= 65536, "16-bit counts within a tile");
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
__global__ __launch_bounds__(SORT_THREADS) void k_sort_count(sort_src src, int shift, int bins, uint32_t* __restrict__ counts) {
  __shared__ uint32_t h[MAX_BINS];
  for (int b = threadIdx.x; b < bins; b += SORT_THREADS) h[b] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * SORT_TILE;
#pragma unroll
  for (int u = 0; u < SORT_ITEMS; ++u) {
    const int64_t i = base + threadIdx.x + SORT_THREADS * u;
    if (i < src.n) atomicAdd(&h[(sort_read(src, i).key >> shift) & (bins - 1)], 1u);
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += SORT_THREADS) counts[(int64_t)blockIdx.x * bins + b] = h[b];
}

// counts[tile][bin] -> the number in the tiles before; totals[bin]
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

__device__ __forceinline__ uint32_t wave_inclusive(uint32_t v, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  return v;
}

__global__ __launch_bounds__(SORT_THREADS) void k_sort_scatter(sort_src src, int shift, int digit_bits, const uint32_t* __restrict__ counts,
                                                               const uint32_t* __restrict__ totals, pair32* __restrict__ out) {
  __shared__ uint32_t place[MAX_BINS];                   // where the tile's first pair of a digit goes
  __shared__ uint16_t part[SORT_WAVES][MAX_BINS];        // the wave's counts of a digit, then those of the waves before it
  __shared__ uint32_t wave_sum[SORT_WAVES];
  const int bins = 1 << digit_bits, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  for (int b = t; b < bins; b += SORT_THREADS)
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) part[w][b] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * SORT_TILE + wave * (64 * SORT_ITEMS);
  pair32 p[SORT_ITEMS];
  uint32_t rank[SORT_ITEMS];
#pragma unroll
  for (int u = 0; u < SORT_ITEMS; ++u) {
    const int64_t i = base + 64 * u + lane;
    p[u] = i < src.n ? sort_read(src, i) : pair32{0u, 0u};
  }
#pragma unroll
  for (int u = 0; u < SORT_ITEMS; ++u) {
    const bool in = base + 64 * u + lane < src.n;
    const uint32_t d = (p[u].key >> shift) & (uint32_t)(bins - 1);
    uint64_t peers = __ballot(in);
    for (int k = 0; k < digit_bits; ++k) {
      const uint64_t m = __ballot((d >> k) & 1);
      peers &= (d >> k) & 1 ? m : ~m;
    }
    const int leader = in ? __ffsll((unsigned long long)peers) - 1 : lane;
    uint32_t before = 0;
    if (in && lane == leader) {          // (one lane per digit, and the counts are the wave's own)
      before = part[wave][d];
      part[wave][d] = (uint16_t)(before + (uint32_t)__popcll(peers));
    }
    before = __shfl(before, leader);
    rank[u] = before + (uint32_t)__popcll(peers & ((1ULL << lane) - 1));
  }
  // exclusive prefix of totals over the bins: a thread takes MAX_BINS / SORT_THREADS neighbouring bins
  constexpr int PER = MAX_BINS / SORT_THREADS;
  uint32_t tot[PER], mine = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int b = t * PER + k;
    tot[k] = b < bins ? totals[b] : 0u;
    mine += tot[k];
  }
  const uint32_t inc = wave_inclusive(mine, lane);
  if (lane == 63) wave_sum[wave] = inc;
  __syncthreads();
  uint32_t run = inc - mine;
  for (int w = 0; w < wave; ++w) run += wave_sum[w];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int b = t * PER + k;
    if (b < bins) {
      place[b] = run + counts[(int64_t)blockIdx.x * bins + b];
      uint32_t sum = 0;
#pragma unroll
      for (int w = 0; w < SORT_WAVES; ++w) {
        const uint32_t c = part[w][b];
        part[w][b] = (uint16_t)sum;
        sum += c;
      }
    }
    run += tot[k];
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < SORT_ITEMS; ++u)
    if (base + 64 * u + lane < src.n) {
      const uint32_t d = (p[u].key >> shift) & (uint32_t)(bins - 1);
      out[place[d] + part[wave][d] + rank[u]] = p[u];
    }
}

// ---- the rows' numbers (row-sparse form) -----------------------------------------------------------------------------
// rank[i] = the number of the distinct id that sorted pair i belongs to; ids[rank] = that id; *count = how many there are.
__device__ __forceinline__ bool is_head(const pair32* s, int64_t i, uint32_t none) {
  const uint32_t k = s[i].key;
  return k != none && (i == 0 || s[i - 1].key != k);
}
__global__ __launch_bounds__(SORT_THREADS) void k_rank_count(const pair32* __restrict__ s, int64_t n, uint32_t none, uint32_t* __restrict__ tile_heads) {
  __shared__ int total;
  if (threadIdx.x == 0) total = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * SORT_TILE;
  int c = 0;
#pragma unroll
  for (int u = 0; u < SORT_ITEMS; ++u) {
    const int64_t i = base + threadIdx.x + SORT_THREADS * u;
    const uint64_t m = __ballot(i < n && is_head(s, i, none));
    c += __popcll(m);
  }
  if ((threadIdx.x & 63) == 0) atomicAdd(&total, c);
  __syncthreads();
  if (threadIdx.x == 0) tile_heads[blockIdx.x] = (uint32_t)total;
}
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
  const int64_t base = (int64_t)blockIdx.x * SORT_TILE + wave * (64 * SORT_ITEMS);
  uint64_t heads[SORT_ITEMS];
  uint32_t mine = 0;
#pragma unroll
  for (int u = 0; u < SORT_ITEMS; ++u) {
    const int64_t i = base + 64 * u + lane;
    heads[u] = __ballot(i < n && is_head(s, i, none));
    mine += (uint32_t)__popcll(heads[u]);
  }
  if (lane == 0) wave_heads[wave] = mine;
  __syncthreads();
  uint32_t run = before;
  for (int w = 0; w < wave; ++w) run += wave_heads[w];
#pragma unroll
  for (int u = 0; u < SORT_ITEMS; ++u) {
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
constexpr int WINDOW = 32;        // sorted pairs per team
struct seg_args {
  const void* g;                  // [n, width], row stride ld_g (0: every row is the same one)
  int64_t ld_g, n, ld_out;
  const pair32* s;
  const uint32_t* rank;           // or null: a row's place in the output is its id
  void* out;
  float* part;                    // [2 * windows, width]: what a window adds to a run that began before it / that it begins and does not end
  int width, chunks, log_l, accumulate;
  uint32_t none;
  float scale;
};

// A team of 2^log_l lanes walks one window of the sorted list in order, a lane holding one 16-byte chunk of the columns.  A run of
// equal ids that lies inside the window is written out; one that crosses a border leaves its sum in `part` for k_segment_join.
template <class TI, class TO, int VEC>
__global__ __launch_bounds__(256) void k_segment_sum(seg_args a) {
  const int team = threadIdx.x >> a.log_l, tl = threadIdx.x & ((1 << a.log_l) - 1);
  const int64_t w = (int64_t)blockIdx.x * (256 >> a.log_l) + team;
  const int c = ((int)blockIdx.y << a.log_l) + tl;
  const int64_t i0 = w * WINDOW;
  if (i0 >= a.n || c >= a.chunks) return;
  const int64_t i1 = i0 + WINDOW < a.n ? i0 + WINDOW : a.n;
  const int col = VEC == 1 ? c : min(c * VEC, a.width - VEC), own = c * VEC - col;      // (elements before `own` are the neighbour's)
  const TI* g = (const TI*)a.g + col;
  uint32_t cur = a.s[i0].key;
  bool head = i0 > 0 && a.s[i0 - 1].key == cur;
  int64_t first = i0;             // first pair of the current run in this window
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
  auto flush = [&](bool goes_on) {
    if (cur == a.none) return;
    if (head || goes_on) {
      store_chunk<VEC, float>(a.part + (2 * w + (head ? 0 : 1)) * a.width + col, acc);
      return;
    }
    const int64_t r = a.rank ? (int64_t)a.rank[first] : (int64_t)cur;
    TO* o = (TO*)a.out + r * a.ld_out + col;
    float f[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = acc[j] * a.scale;
    if (a.accumulate) {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (j >= own) o[j] = (TO)((float)o[j] + f[j]);
    } else {
      store_chunk<VEC, TO>(o, f);
    }
  };
  constexpr int U = 8;
  for (int64_t i = i0; i < i1 && cur != a.none; i += U) {
    pair32 p[U];
    float v[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) p[u] = a.s[i + u < i1 ? i + u : i1 - 1];
#pragma unroll
    for (int u = 0; u < U; ++u) load_chunk<VEC, TI>(g + (int64_t)p[u].pos * a.ld_g, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u >= i1) break;
      if (p[u].key != cur) {
        flush(false);
        cur = p[u].key;
        head = false;
        first = i + u;
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] += v[u][j];
    }
  }
  flush(i1 < a.n && a.s[i1].key == cur);
}

// The runs that cross window borders: a workgroup takes the run that window blockIdx.x begins and does not end, its teams each a
// consecutive share of the windows' sums; the shares are added in the windows' order.
template <class TO>
__global__ __launch_bounds__(256) void k_segment_join(seg_args a) {
  __shared__ float4 share[256];
  const int64_t w = blockIdx.x, i0 = w * WINDOW, i1 = i0 + WINDOW;
  if (i1 >= a.n) return;
  const uint32_t key = a.s[i1 - 1].key;
  if (key == a.none || a.s[i1].key != key || (i0 > 0 && a.s[i0 - 1].key == key)) return;      // (workgroup-uniform)
  int64_t terms = 1;              // the window's own sum, and one of each window that begins inside the run
  for (;;) {
    const int64_t f = (w + terms + threadIdx.x) * WINDOW;
    const int m = __syncthreads_count(f < a.n && a.s[f].key == key);
    terms += m;
    if (m < 256) break;
  }
  const int lanes = 1 << a.log_l, teams = 256 >> a.log_l, team = threadIdx.x >> a.log_l, tl = threadIdx.x & (lanes - 1);
  const int col = (((int)blockIdx.y << a.log_l) + tl) * 4;
  const int have = col >= a.width ? 0 : min(4, a.width - col);
  const int64_t each = ceil_div64(terms, teams), b = team * each, e = b + each < terms ? b + each : terms;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto term = [&](int64_t k) {
    const float* q = a.part + (k == 0 ? 2 * w + 1 : 2 * (w + k)) * a.width + col;
    float4 v;
    v.x = have > 0 ? q[0] : 0.f;
    v.y = have > 1 ? q[1] : 0.f;
    v.z = have > 2 ? q[2] : 0.f;
    v.w = have > 3 ? q[3] : 0.f;
    return v;
  };
  for (int64_t k = b; k < e; k += 8) {
    float4 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = k + u < e ? term(k + u) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int u = 0; u < 8; ++u) { acc.x += v[u].x; acc.y += v[u].y; acc.z += v[u].z; acc.w += v[u].w; }
  }
  share[threadIdx.x] = acc;
  __syncthreads();
  if (team != 0 || have == 0) return;
  for (int q = 1; q < teams; ++q) {
    const float4 v = share[(q << a.log_l) + tl];
    acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
  }
  const int64_t r = a.rank ? (int64_t)a.rank[i1 - 1] : (int64_t)key;
  TO* o = (TO*)a.out + r * a.ld_out + col;
  const float f[4] = {acc.x * a.scale, acc.y * a.scale, acc.z * a.scale, acc.w * a.scale};
  for (int j = 0; j < have; ++j) o[j] = (TO)(a.accumulate ? (float)o[j] + f[j] : f[j]);
}

// zeros over the rows of a table (rows of `bytes` bytes, `pitch` bytes apart; a table without gaps is one row)
__global__ __launch_bounds__(256) void k_zero_rows(char* __restrict__ out, int64_t rows, int64_t bytes, int64_t pitch) {
  const int64_t per = ceil_div64(bytes, 16), total = rows * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = rows == 1 ? 0 : i / per, b = (i - r * per) * 16;
    char* p = out + r * pitch + b;
    if (b + 16 <= bytes) {
      store16(p, u32x4{0, 0, 0, 0});
    } else {
      for (int64_t k = b; k < bytes; k += 2) *reinterpret_cast<uint16_t*>(out + r * pitch + k) = 0;
    }
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------
struct sort_plan { int passes, digit; int64_t tiles; };
sort_plan plan_sort(int64_t n, int64_t num_rows) {
  int bits = 1;
  while (bits < 32 && (num_rows >> bits) != 0) ++bits;        // keys 0 .. num_rows
  sort_plan s;
  s.passes = (bits + MAX_DIGIT - 1) / MAX_DIGIT;
  s.digit = (bits + s.passes - 1) / s.passes;
  s.tiles = ceil_div64(n, SORT_TILE);
  return s;
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
  l.part = take(2 * ceil_div64(n, WINDOW) * width * 4);
  l.bytes = o;
  return l;
}
int log_lanes(int64_t chunks) {       // the smallest team that holds a row's chunks, at most a wave
  int l = 0;
  while (l < 6 && (1 << l) < chunks) ++l;
  return l;
}

template <class TI, class TO>
int launch_sums(seg_args a, hipStream_t stream) {
  constexpr int VEC = elems16<TI>;
  const bool wide = a.width >= VEC;
  a.chunks = wide ? (a.width + VEC - 1) / VEC : a.width;
  a.log_l = log_lanes(a.chunks);
  const int64_t windows = ceil_div64(a.n, WINDOW);
  dim3 grid((unsigned)ceil_div64(windows, 256 >> a.log_l), (unsigned)ceil_div64(a.chunks, 1 << a.log_l));
  if (wide) k_segment_sum<TI, TO, VEC><<<grid, 256, 0, stream>>>(a);
  else k_segment_sum<TI, TO, 1><<<grid, 256, 0, stream>>>(a);
  ORCA_LAUNCH_CHECK();
  if (windows < 2) return ORCA_OK;
  a.chunks = (a.width + 3) / 4;
  a.log_l = log_lanes(a.chunks);
  k_segment_join<TO><<<dim3((unsigned)(windows - 1), (unsigned)ceil_div64(a.chunks, 1 << a.log_l)), 256, 0, stream>>>(a);
  ORCA_LAUNCH_CHECK();
  return ORCA_OK;
}

int sum_by_type(int g_dtype, int out_dtype, const seg_args& a, hipStream_t stream) {
  if (out_dtype == ORCA_F32) {
    if (g_dtype == ORCA_F32) return launch_sums<float, float>(a, stream);
    return g_dtype == ORCA_BF16 ? launch_sums<__bf16, float>(a, stream) : launch_sums<_Float16, float>(a, stream);
  }
  return g_dtype == ORCA_BF16 ? launch_sums<__bf16, __bf16>(a, stream) : launch_sums<_Float16, _Float16>(a, stream);
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
  ORCA_REQUIRE(workspace && workspace_bytes >= layout(n, width, num_rows).bytes, "%s: the workspace holds %lld of %lld bytes", who,
               (long long)workspace_bytes, (long long)layout(n, width, num_rows).bytes);
  return ORCA_OK;
}

// sorts (id, position); *sorted = where the result lies
int sort_positions(const int64_t* idx64, const int32_t* idx32, int64_t n, int64_t num_rows, int64_t padding, char* ws, const work_layout& l,
                   const pair32** sorted, hipStream_t stream) {
  const sort_plan s = plan_sort(n, num_rows);
  sort_src src{idx64, idx32, nullptr, n, num_rows, padding};
  uint32_t* counts = (uint32_t*)(ws + l.counts);
  uint32_t* totals = (uint32_t*)(ws + l.totals);
  pair32* buf[2] = {(pair32*)(ws + l.a), (pair32*)(ws + l.b)};
  for (int p = 0; p < s.passes; ++p) {
    k_sort_count<<<(unsigned)s.tiles, SORT_THREADS, 0, stream>>>(src, p * s.digit, 1 << s.digit, counts);
    ORCA_LAUNCH_CHECK();
    k_sort_columns<<<((1 << s.digit) + 63) / 64, 64, 0, stream>>>(counts, s.tiles, 1 << s.digit, totals);
    ORCA_LAUNCH_CHECK();
    k_sort_scatter<<<(unsigned)s.tiles, SORT_THREADS, 0, stream>>>(src, p * s.digit, s.digit, counts, totals, buf[p & 1]);
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
  return layout(n, width, num_rows).bytes;
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
  if (!accumulate) {
    const int64_t e = table_dtype == ORCA_F32 ? 4 : 2;
    const bool gaps = ld_table != width && num_rows > 1;
    const int64_t rows = gaps ? num_rows : 1, bytes = (gaps ? width : num_rows * width) * e;
    k_zero_rows<<<(unsigned)std::min<int64_t>(2048, ceil_div64(rows * ceil_div64(bytes, 16), 256)), 256, 0, stream>>>((char*)grad_table, rows, bytes,
                                                                                                                  ld_table * e);
    ORCA_LAUNCH_CHECK();
  }
  if (n == 0) return ORCA_OK;
  const work_layout l = layout(n, width, num_rows);
  char* ws = (char*)workspace;
  const pair32* s = nullptr;
  if (int rc = sort_positions(idx64, idx32, n, num_rows, padding_idx, ws, l, &s, stream)) return rc;
  seg_args a{grad_out, ld_grad, n, ld_table, s, nullptr, grad_table, (float*)(ws + l.part), (int)width, 0, 0, accumulate != 0, (uint32_t)num_rows, scale};
  return sum_by_type(grad_dtype, table_dtype, a, stream);
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
  const work_layout l = layout(n, width, num_rows);
  char* ws = (char*)workspace;
  const pair32* s = nullptr;
  if (int rc = sort_positions(idx64, idx32, n, num_rows, padding_idx, ws, l, &s, stream)) return rc;
  const unsigned tiles = (unsigned)plan_sort(n, num_rows).tiles;
  uint32_t* rank = (uint32_t*)(ws + l.rank);
  k_rank_count<<<tiles, SORT_THREADS, 0, stream>>>(s, n, (uint32_t)num_rows, (uint32_t*)(ws + l.heads));
  ORCA_LAUNCH_CHECK();
  k_rank<<<tiles, SORT_THREADS, 0, stream>>>(s, n, (uint32_t)num_rows, (const uint32_t*)(ws + l.heads), rank, ids, count);
  ORCA_LAUNCH_CHECK();
  seg_args a{grad_out, ld_grad, n, width, s, rank, rows, (float*)(ws + l.part), (int)width, 0, 0, 0, (uint32_t)num_rows, scale};
  return sum_by_type(grad_dtype, rows_dtype, a, stream);
}
