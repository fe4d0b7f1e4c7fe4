// Embedding lookup with scaling and its gradient by sorted ids:
//   out[i, :]    = scale * table[ids[i], :]                     (ids outside [0, rows): padding, a row of zeros)
//   d table[r,:] = scale * sum over {i : ids[i] = r} of d out[i, :]   (zeros for rows nobody read)
// What tf.gather / tf.nn.embedding_lookup do inside a likelihood or a surrogate's network; with the chains (or ELBO
// samples) of a run as the columns it is the group-level effect of a regression, table[group, chain].
//
// The gradient sums each row's positions in the order of a stable sort of the ids, so it has no atomics and the same
// bits every time.  `plan` = what depends on the ids alone (the sort), so that a fixed dataset sorts once:
//   int32 order[n]    positions, sorted by id, equal ids in ascending position; padding last
//   int32 key[n]      the ids in that order (padding: `rows`)
//   int32 start[rows + 1]   first entry of each row; start[rows] = number of positions that are not padding
#include "bvi_common.h"

namespace {

template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T e[V];
};

// ---- forward -------------------------------------------------------------------------------------------------------
// One thread moves one vector of V elements; tc threads side by side hold one row's columns (all of them up to 256,
// else equal parts), 256 / tc rows per step, four steps' ids and vectors in flight.  Nothing but bytes: 65537 rows of 640
// bf16 out of 100003 take 32 us from memory, 5.2 TB/s of reads and writes (26 where a cache holds some of the table);
// 919 x 4 are the launch, 3 us.
constexpr int LK_UNROLL = 4;

template <typename T, int V, typename I>
__global__ __launch_bounds__(256) void lookup_kernel(const T* __restrict__ table, int64_t stride, int64_t rows,
                                                     const I* __restrict__ ids, int64_t n, int64_t width, int W, int tc,
                                                     float scale, T* __restrict__ out) {
  const int per_step = 256 / tc;
  const int sub = threadIdx.x / tc, col0 = threadIdx.x - sub * tc;
  if (sub >= per_step) return;
  const int64_t per_block = (int64_t)per_step * LK_UNROLL;
  for (int64_t base = blockIdx.x * per_block; base < n; base += gridDim.x * per_block) {
    int64_t id[LK_UNROLL];
#pragma unroll
    for (int u = 0; u < LK_UNROLL; ++u) {
      const int64_t i = base + u * per_step + sub;
      id[u] = i < n ? (int64_t)ids[i] : -1;
      if (id[u] >= rows) id[u] = -1;
    }
    for (int col = col0; col < W; col += tc) {
      Pack<T, V> p[LK_UNROLL];
#pragma unroll
      for (int u = 0; u < LK_UNROLL; ++u) {
        if (id[u] >= 0) {
          p[u] = *reinterpret_cast<const Pack<T, V>*>(table + id[u] * stride + (int64_t)col * V);
        } else {
#pragma unroll
          for (int k = 0; k < V; ++k) p[u].e[k] = (T)0.f;
        }
      }
#pragma unroll
      for (int u = 0; u < LK_UNROLL; ++u) {
        const int64_t i = base + u * per_step + sub;
        // the product in float, rounded once; 0 * scale would turn padding into NaN for an infinite scale
#pragma unroll
        for (int k = 0; k < V; ++k) p[u].e[k] = id[u] >= 0 ? (T)((float)p[u].e[k] * scale) : (T)0.f;
        if (i < n) *reinterpret_cast<Pack<T, V>*>(out + i * width + (int64_t)col * V) = p[u];
      }
    }
  }
}

// ---- the sort: least significant digit first, at most 11 bits per pass, stable ---------------------------------------
// Few launches count more than bytes here: two passes cover four million rows.  A workgroup's tile is ROUNDS x 256
// positions; up to SORT_FUSED workgroups the scatter launch adds up the counts of the others by itself, beyond that a
// launch between the two does.  65537 ids below 100003: two passes of 5 + 9 us, all of it latency; 2M ids below 5000, two
// passes of 11 + 5 + 25 to 39 us, whose scattered 8 bytes are the cost.
constexpr int SORT_MAX_BITS = 11, SORT_MAX_DIGITS = 1 << SORT_MAX_BITS, SORT_FUSED = 128;

// the sort key of position i: the id, or `rows` for padding; later passes read the keys of the pass before
template <typename I>
__device__ __forceinline__ uint32_t sort_key(const I* __restrict__ ids, const uint32_t* __restrict__ keys, int64_t rows,
                                             int64_t i) {
  if (keys) return keys[i];
  const int64_t id = (int64_t)ids[i];
  return (uint32_t)(id >= 0 && id < rows ? id : rows);
}

// count[d digit_stride + block block_stride] = the block's positions with digit d
template <typename I, int ROUNDS>
__global__ __launch_bounds__(256) void sort_count_kernel(const I* __restrict__ ids, const uint32_t* __restrict__ keys,
                                                         int64_t n, int64_t rows, int shift, int digits,
                                                         int64_t digit_stride, int64_t block_stride,
                                                         uint32_t* __restrict__ count) {
  __shared__ uint32_t hist[SORT_MAX_DIGITS];
  for (int d = threadIdx.x; d < digits; d += 256) hist[d] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * (256 * ROUNDS) + threadIdx.x;
#pragma unroll
  for (int j = 0; j < ROUNDS; ++j) {
    const int64_t i = base + j * 256;
    if (i < n) atomicAdd(&hist[(sort_key(ids, keys, rows, i) >> shift) & (digits - 1)], 1u);   // integers: order-free
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += 256) count[d * digit_stride + blockIdx.x * block_stride] = hist[d];
}

__device__ __forceinline__ uint32_t inclusive_wave_sum(uint32_t v) {
  const int lane = threadIdx.x & 63;
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t t = __shfl_up(v, off, 64);
    if (lane >= off) v += t;
  }
  return v;
}

// workgroup d: exclusive sums of digit d's counts over the blocks, in place, and the digit's total
__global__ __launch_bounds__(256) void sort_scan_kernel(int n_blocks, uint32_t* __restrict__ count,
                                                        uint32_t* __restrict__ total) {
  __shared__ uint32_t wave_sum[4];
  uint32_t* c = count + (int64_t)blockIdx.x * n_blocks;
  const int wave = threadIdx.x >> 6;
  uint32_t carry = 0;
  for (int b0 = 0; b0 < n_blocks; b0 += 256) {
    const int b = b0 + threadIdx.x;
    const uint32_t own = b < n_blocks ? c[b] : 0u;
    const uint32_t v = inclusive_wave_sum(own);
    if ((threadIdx.x & 63) == 63) wave_sum[wave] = v;
    __syncthreads();
    uint32_t before = carry, all = 0;
    for (int w = 0; w < 4; ++w) {
      if (w < wave) before += wave_sum[w];
      all += wave_sum[w];
    }
    if (b < n_blocks) c[b] = before + v - own;
    carry += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) total[blockIdx.x] = carry;
}

// Each wave owns ROUNDS x 64 consecutive positions and ranks them 64 at a time: one ballot per bit gives the lanes with
// the same digit, a counter per wave and digit the earlier rounds'.  Positions are visited in ascending order: stable.
template <typename I, int ROUNDS, bool FUSED, int EACH>
__global__ __launch_bounds__(256) void sort_scatter_kernel(const I* __restrict__ ids, const uint32_t* __restrict__ keys,
                                                           const uint32_t* __restrict__ vals, int64_t n, int64_t rows,
                                                           int shift, int bits, int n_blocks,
                                                           const uint32_t* __restrict__ count,
                                                           const uint32_t* __restrict__ total,
                                                           uint32_t* __restrict__ keys_out,
                                                           uint32_t* __restrict__ vals_out) {
  __shared__ uint32_t seen[4][SORT_MAX_DIGITS];
  __shared__ uint32_t wave_sum[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, digits = 1 << bits;
  for (int d = threadIdx.x; d < digits; d += 256)
#pragma unroll
    for (int w = 0; w < 4; ++w) seen[w][d] = 0;
  const int64_t base = (int64_t)blockIdx.x * (256 * ROUNDS) + wave * (64 * ROUNDS) + lane;
  uint32_t key[ROUNDS], rank[ROUNDS];
#pragma unroll
  for (int j = 0; j < ROUNDS; ++j) {
    const int64_t i = base + j * 64;
    key[j] = i < n ? sort_key(ids, keys, rows, i) : 0u;
  }
  // where each wave's entries of digit d go: digits before d, d's entries of earlier blocks, of earlier waves.  Thread t
  // takes EACH neighbouring digits.
  uint32_t at[EACH], all[EACH] = {}, own = 0;
  const int d0 = threadIdx.x * EACH;
  if (d0 < digits) {
    if (FUSED) {
      uint32_t before[EACH] = {};
      for (int b0 = 0; b0 < n_blocks; b0 += 16) {
        Pack<uint32_t, EACH> c[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) {
          const int b = b0 + u < n_blocks ? b0 + u : n_blocks - 1;
          c[u] = *reinterpret_cast<const Pack<uint32_t, EACH>*>(count + (int64_t)b * digits + d0);
        }
#pragma unroll
        for (int u = 0; u < 16; ++u)
#pragma unroll
          for (int k = 0; k < EACH; ++k) {
            all[k] += b0 + u < n_blocks ? c[u].e[k] : 0u;
            before[k] += b0 + u < (int)blockIdx.x ? c[u].e[k] : 0u;
          }
      }
#pragma unroll
      for (int k = 0; k < EACH; ++k) at[k] = before[k];
    } else {
#pragma unroll
      for (int k = 0; k < EACH; ++k) {
        all[k] = total[d0 + k];
        at[k] = count[(int64_t)(d0 + k) * n_blocks + blockIdx.x];
      }
    }
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      at[k] += own;
      own += all[k];
    }
  }
  __syncthreads();
  volatile uint32_t* mine = seen[wave];
#pragma unroll
  for (int j = 0; j < ROUNDS; ++j) {
    const bool in = base + j * 64 < n;
    const uint32_t d = (key[j] >> shift) & (digits - 1);
    uint64_t same = __ballot(in);
#pragma unroll
    for (int b = 0; b < SORT_MAX_BITS; ++b) {
      const uint64_t bit = __ballot((d >> b) & 1u);
      same &= ((d >> b) & 1u) ? bit : ~bit;
    }
    const uint32_t before = __popcll(same & ((1ull << lane) - 1ull));
    const uint32_t prior = mine[d];
    rank[j] = prior + before;
    __builtin_amdgcn_wave_barrier();
    if (in && before == 0) mine[d] = prior + (uint32_t)__popcll(same);     // the group's first lane
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  const uint32_t v = inclusive_wave_sum(own);
  if (lane == 63) wave_sum[wave] = v;
  __syncthreads();
  uint32_t first = v - own;
  for (int w = 0; w < wave; ++w) first += wave_sum[w];
  if (d0 < digits) {
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      uint32_t to = first + at[k];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t c = seen[w][d0 + k];
        seen[w][d0 + k] = to;
        to += c;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < ROUNDS; ++j) {
    const int64_t i = base + j * 64;
    if (i < n) {
      const uint32_t to = seen[wave][(key[j] >> shift) & (digits - 1)] + rank[j];
      keys_out[to] = key[j];
      vals_out[to] = vals ? vals[i] : (uint32_t)i;
    }
  }
}

// ---- few positions: each one's place is the number of positions sorted before it, counted against all of them --------
// n^2 comparisons, two instructions each, over the whole chip and in one launch.  Eight neighbouring lanes share a
// position and take every eighth vector of four keys.  919 positions 5.5 us, start to end; one pass of the sort is as long.
constexpr int RANK_MAX = 4096;
template <typename I>
__global__ __launch_bounds__(256) void sort_rank_kernel(const I* __restrict__ ids, int n, int64_t rows,
                                                        uint32_t* __restrict__ order, uint32_t* __restrict__ key_out) {
  __shared__ uint4 keys4[RANK_MAX / 4];
  uint32_t* keys = reinterpret_cast<uint32_t*>(keys4);
  const int vectors = (n + 31) / 32 * 8;
  for (int j0 = threadIdx.x; j0 < vectors * 4; j0 += 256 * 8) {       // eight loads in flight
    uint32_t k[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int j = j0 + u * 256;
      k[u] = sort_key(ids, (const uint32_t*)nullptr, rows, j < n ? j : 0);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int j = j0 + u * 256;
      if (j < vectors * 4) keys[j] = j < n ? k[u] : 0xffffffffu;
    }
  }
  __syncthreads();
  const int i = blockIdx.x * 32 + (threadIdx.x >> 3), part = threadIdx.x & 7;
  const uint32_t k = i < n ? keys[i] : 0u;
  uint32_t place = 0;
#pragma unroll 4
  for (int v = part; v < vectors; v += 8) {
    const uint4 x = keys4[v];
    const uint32_t below = v < (i >> 2) ? k + 1u : k;          // equal keys in front of i count too
    place += (x.x < below ? 1u : 0u) + (x.y < below ? 1u : 0u) + (x.z < below ? 1u : 0u) + (x.w < below ? 1u : 0u);
  }
  if (part == 0 && i < n)
    for (int j = i & ~3; j < i; ++j) place += keys[j] == k ? 1u : 0u;     // and those in i's own vector
  place += __shfl_xor(place, 1, 64);
  place += __shfl_xor(place, 2, 64);
  place += __shfl_xor(place, 4, 64);
  if (part == 0 && i < n) {
    order[place] = (uint32_t)i;
    key_out[place] = k;
  }
}

// start[r] = number of sorted keys below r.  With at least as many positions as rows: position p fills in the rows between
// its neighbour's and its own, a wave together where those are many.
__device__ __forceinline__ void fill_start(int64_t p, const uint32_t* __restrict__ key, int64_t n, uint32_t rows,
                                           int32_t* __restrict__ start) {
  const int lane = threadIdx.x & 63;
  const uint32_t from = p == 0 || p > n ? 0u : key[p - 1] + 1u;      // rows [from, to] start at p
  const uint32_t to = p < n ? key[p] : rows;
  const uint32_t gap = p <= n && to + 1u > from ? to + 1u - from : 0u;
  if (gap <= 8)
    for (uint32_t r = 0; r < gap; ++r) start[from + r] = (int32_t)p;
  for (uint64_t wide = __ballot(gap > 8); wide; wide &= wide - 1ull) {
    const int src = __ffsll((unsigned long long)wide) - 1;
    const uint32_t f = __shfl(from, src, 64), m = __shfl(gap, src, 64);
    const int32_t at = (int32_t)(p - lane + src);
    for (uint32_t r = lane; r < m; r += 64) start[f + r] = at;
  }
}

// With fewer: a search per row.  Sixteen probes at a time: the search waits for loads, not for their number.
__device__ __forceinline__ void search_start(int64_t r, const uint32_t* __restrict__ key, int n, int64_t rows,
                                             int32_t* __restrict__ start) {
  if (r > rows) return;
  int lo = 0, hi = n;                              // the answer lies in [lo, hi]
  while (lo < hi) {
    const int step = (hi - lo + 15) >> 4;
    uint32_t k[16];
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      const int at = lo + (u + 1) * step - 1;      // below 2^31: n has room for a step more
      k[u] = key[at < hi ? at : hi - 1];
    }
    int below = 0;
#pragma unroll
    for (int u = 0; u < 16; ++u) below += lo + (u + 1) * step - 1 < hi && (int64_t)k[u] < r ? 1 : 0;
    lo += below * step;
    hi = below == 16 ? lo : min(hi, lo + step - 1);
  }
  start[r] = lo;
}

struct StartJob {
  const uint32_t* key;
  int32_t* start;
  int64_t n, rows;
  int blocks;                                      // of 256 threads; 0: nothing to do
};
__device__ __forceinline__ void start_part(const StartJob& j) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (j.n >= j.rows) fill_start(i, j.key, j.n, (uint32_t)j.rows, j.start);
  else search_start(i, j.key, (int)j.n, j.rows, j.start);
}
__global__ __launch_bounds__(256) void sort_start_kernel(StartJob j) { start_part(j); }

// ---- gradient ------------------------------------------------------------------------------------------------------
// So that no thread has many positions of one row to add: blocks of 2^chunk_bits sorted positions that belong to one row
// are summed beforehand (level 1), blocks of 2^fan_bits of those again (level 2), and so on; a row adds the entries at
// its ends one by one and whole blocks in between.  Two forms of the three kernels:
//   wide rows, or few positions per row: a thread per vector of V columns, three positions in flight
//   (65537 x 640 bf16 into 100003 rows, 212 MB that no cache holds: 62 us, 3.4 TB/s; a row's start, its position and its
//   vector wait for one another, yet neither positions fetched a row ahead, 62, nor four rows at a time, 82, nor three rows
//   carried along in registers, 79, hid more than a wave more per SIMD does);
//   narrow rows: a wave per row, LE lanes across the columns times Q = 64 / LE over the positions (2M x 16 into 5000 rows
//   14 us after 29 us for the blocks of 128; a thread per vector took 43 after 42; waves that walk the sorted positions and
//   read everything once 41 - 51, since a gathered row of 64 bytes costs the 128 of its line whoever reads it).
constexpr int GRAD_LEVELS = 8;
struct GradLevels {
  int count, chunk_bits, fan_bits;
  int64_t n[GRAD_LEVELS];             // blocks of the level
  int64_t at[GRAD_LEVELS];            // where its sums start in the workspace (floats)
};

__host__ __device__ __forceinline__ int64_t level_space(int64_t floats) { return (floats + 63) / 64 * 64; }

// acc += columns [col, col + V) of the rows src[order[p]] (or src[p] without an order), p = a, a + Q, ... below b
template <typename S, int V, bool PERM, int Q, int DEEP>
__device__ __forceinline__ void grad_sum(float (&acc)[V], const S* __restrict__ src, int64_t stride, int64_t col,
                                         const int32_t* __restrict__ order, int a, int b) {
  for (int p = a; p < b; p += DEEP * Q) {
    Pack<S, V> x[DEEP];
    int32_t i[DEEP];
#pragma unroll
    for (int u = 0; u < DEEP; ++u) {                      // beyond the end: the first one again, not added
      i[u] = p + u * Q < b ? p + u * Q : p;
      if (PERM) i[u] = order[i[u]];
    }
#pragma unroll
    for (int u = 0; u < DEEP; ++u) x[u] = *reinterpret_cast<const Pack<S, V>*>(src + (int64_t)i[u] * stride + col);
#pragma unroll
    for (int u = 0; u < DEEP; ++u)
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] += p + u * Q < b ? (float)x[u].e[k] : 0.f;
  }
}

// acc += one row's positions [a, b), by way of the levels; lane q of Q takes every Q-th entry of each stretch
template <typename T, int V, int Q, int DEEP>
__device__ __forceinline__ void grad_row_sum(float (&acc)[V], const T* __restrict__ g, int64_t stride, int64_t at,
                                             const int32_t* __restrict__ order, int a, int b, int q, int64_t width,
                                             const GradLevels& lv, const float* __restrict__ sums) {
  int bits = lv.chunk_bits, level = 0;                       // a, b below 2^31 with room for a block
  const float* below = sums;                                 // the level's sums, found step by step: an array indexed by
  int64_t blocks = lv.n[0];                                  // a lane's own level would be copied into registers
  while (true) {
    const int up = (a + (1 << bits) - 1) >> bits, down = b >> bits;
    const bool split = level < lv.count && up < down;        // whole blocks of the next level in the middle
#pragma unroll 1
    for (int side = 0; side < (split ? 2 : 1); ++side) {     // one copy of the code: registers decide the speed
      const int from = side ? down << bits : a, to = split && !side ? up << bits : b;
      if (level == 0)
        grad_sum<T, V, true, Q, DEEP>(acc, g, stride, at, order, from + q, to);
      else
        grad_sum<float, V, false, Q, DEEP>(acc, below, width, at, nullptr, from + q, to);
    }
    if (!split) break;
    a = up;
    b = down;
    bits = lv.fan_bits;
    if (level) {
      below += level_space(blocks * width);
      blocks >>= bits;
    }
    ++level;
  }
}

template <int V, int LE>
__device__ __forceinline__ void grad_join(float (&acc)[V]) {
#pragma unroll
  for (int off = LE; off < 64; off <<= 1)
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] += __shfl_xor(acc[k], off, 64);
}
template <typename O, int V>
__device__ __forceinline__ void grad_store(O* __restrict__ to, const float (&acc)[V]) {
  Pack<O, V> o;
#pragma unroll
  for (int k = 0; k < V; ++k) o.e[k] = (O)acc[k];
  *reinterpret_cast<Pack<O, V>*>(to) = o;
}

// One level: block b adds entries [b << bits, (b + 1) << bits) of the level below (the positions themselves for level 1,
// PERM) if the 1 << span_bits positions that they cover belong to one row.  LE = 0: tc threads per block; else a wave.
// Level 1 may take the search for the rows' starts along, in workgroups of its own: neither needs the other, and a launch
// less saves some 8 us.
template <typename S, int V, int LE, bool PERM>
__global__ __launch_bounds__(256) void grad_level_kernel(const S* __restrict__ src, int64_t stride, int W, int tc,
                                                         const int32_t* __restrict__ order,
                                                         const uint32_t* __restrict__ key, int64_t rows, int64_t n_blocks,
                                                         int bits, int span_bits, StartJob job,
                                                         float* __restrict__ sums) {
  if (PERM && (int)blockIdx.x < job.blocks) {
    if (blockIdx.y == 0) start_part(job);
    return;
  }
  constexpr int Q = LE ? 64 / (LE ? LE : 1) : 1;
  const int per = LE ? 4 : 256 / tc, sub = LE ? threadIdx.x >> 6 : threadIdx.x / tc;
  const int t = LE ? threadIdx.x & 63 : threadIdx.x - sub * tc, step = LE ? LE : tc;
  const int q = LE ? t / step : 0, col0 = blockIdx.y * step + (LE ? t % step : t), col_step = gridDim.y * step;
  if (sub >= per) return;
  const int64_t first = (int64_t)blockIdx.x - (PERM ? job.blocks : 0), step_blocks = (int64_t)gridDim.x - (PERM ? job.blocks : 0);
  for (int64_t b = first * per + sub; b < n_blocks; b += step_blocks * per) {
    const uint32_t k0 = key[b << span_bits];
    if (k0 != key[((b + 1) << span_bits) - 1] || k0 >= rows) continue;
    for (int col = col0; col - (LE ? t % step : 0) < W; col += col_step) {     // by waves: all lanes as long as one has a column
      float acc[V] = {};
      if (col < W)
        grad_sum<S, V, PERM, Q, LE ? 8 : 4>(acc, src, stride, (int64_t)col * V, order, (int)(b << bits) + q,
                                            (int)((b + 1) << bits));
      if (LE) grad_join<V, LE ? LE : 64>(acc);
      if (q == 0 && col < W) grad_store<float, V>(sums + (b * W + col) * V, acc);
    }
  }
}

// blockIdx.y: columns beyond the first 256 vectors, where rows (or, above, blocks) are too few to fill the chip (2100
// positions x 1999 columns into three rows: 114 -> 29 us).
// A thread per vector; the next row's place in the order is on its way while this one's positions are added.  Vectors of
// eight are added up in halves where a row has several positions: 64 registers instead of 86, eight waves instead of five
// (65537 x 640 bf16 into 100003 rows 71 -> 62 us; where rows have six positions each, 300000 x 256 f16 into 50000, 53 -> 57).
template <typename T, int V>
__global__ __launch_bounds__(256) void grad_row_kernel(const T* __restrict__ g, int64_t stride, int W, int tc,
                                                       const int32_t* __restrict__ order,
                                                       const int32_t* __restrict__ start, int64_t rows, GradLevels lv,
                                                       const float* __restrict__ sums, float scale, T* __restrict__ out) {
  const int per_step = 256 / tc, sub = threadIdx.x / tc, col0 = blockIdx.y * tc + threadIdx.x - sub * tc;
  const int col_step = gridDim.y * tc;
  int64_t r = (int64_t)blockIdx.x * per_step + sub;
  if (sub >= per_step || r >= rows) return;
  const int64_t width = (int64_t)W * V, step = (int64_t)gridDim.x * per_step;
  int s = start[r], e = start[r + 1];
  while (true) {
    const int64_t next = r + step < rows ? r + step : r;
    const int sn = start[next], en = start[next + 1];
    if (e - s <= 1) {                                    // most rows of a large table: one position or none
      const T* from = g + (e > s ? order[s] * stride : 0);
      for (int col = col0; col < W; col += col_step) {
        float acc[V] = {};
        if (e > s) {
          const Pack<T, V> x = *reinterpret_cast<const Pack<T, V>*>(from + (int64_t)col * V);
#pragma unroll
          for (int k = 0; k < V; ++k) acc[k] = (float)x.e[k] * scale;
        }
        grad_store<T, V>(out + r * width + (int64_t)col * V, acc);
      }
    } else {
      constexpr int H = V == 8 ? 4 : V, PARTS = V / H;
#pragma unroll 1
      for (int part = col0 * PARTS; part < W * PARTS; part += (part + 1) % PARTS ? 1 : (col_step - 1) * PARTS + 1) {
        const int64_t at = (int64_t)part * H;
        float acc[H] = {};
        grad_row_sum<T, H, 1, 3>(acc, g, stride, at, order, s, e, 0, width, lv, sums);
#pragma unroll
        for (int k = 0; k < H; ++k) acc[k] *= scale;
        grad_store<T, H>(out + r * width + at, acc);
      }
    }
    if (next == r) return;
    r = next;
    s = sn;
    e = en;
  }
}

// A wave per row.
template <typename T, int V, int LE>
__global__ __launch_bounds__(256) void grad_row_wave_kernel(const T* __restrict__ g, int64_t stride, int W,
                                                            const int32_t* __restrict__ order,
                                                            const int32_t* __restrict__ start, int64_t rows, GradLevels lv,
                                                            const float* __restrict__ sums, float scale,
                                                            T* __restrict__ out) {
  const int lane = threadIdx.x & 63, q = lane / LE, le = lane % LE;
  const int64_t width = (int64_t)W * V;
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += (int64_t)gridDim.x * 4) {
    const int s = start[r], e = start[r + 1];
    for (int col = le; col - le < W; col += LE) {
      float acc[V] = {};
      if (col < W)
        grad_row_sum<T, V, 64 / LE, 4>(acc, g, stride, (int64_t)col * V, order, s, e, q, width, lv, sums);
      grad_join<V, LE>(acc);
      if (q == 0 && col < W) {
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] = e > s ? acc[k] * scale : 0.f;
        grad_store<T, V>(out + r * width + (int64_t)col * V, acc);
      }
    }
  }
}

// Few positions and rows: no sort at all.  A wave per row looks through the ids, 64 at a time, lists the positions it
// finds in ascending order, and sums them, LE lanes across the columns times Q = 64 / LE over the list.  919 x 4 into 85
// rows: 5.5 us, one launch; ranking, the start of each row and the sums are three.  A list of more than SCAN_ALONE rounds
// is shared by the workgroup's four waves, and where rows are few their columns go to workgroups of their own (each looks
// through the ids again, 4 us): 2048 positions x 1999 columns into one row 45 us, x 2000 32; by one wave alone 11 ms and 2.1.
constexpr int SCAN_MAX = 2048, SCAN_DEEP = 4, SCAN_ALONE = 4;
template <typename T, int V, int LE, typename I>
__global__ __launch_bounds__(256) void grad_scan_kernel(const T* __restrict__ g, int64_t stride, int W,
                                                        const I* __restrict__ ids, int n, int64_t rows, float scale,
                                                        T* __restrict__ out) {
  constexpr int Q = 64 / LE, LONG = SCAN_ALONE * SCAN_DEEP * Q;
  __shared__ uint16_t lists[4][SCAN_MAX];
  __shared__ int counts[4];
  __shared__ float parts[3][LE * V];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane / LE, le = lane % LE;
  const int64_t r0 = (int64_t)blockIdx.x * 4, r = r0 + wave;
  uint16_t* list = lists[wave];
  int found = 0;
  if (r < rows) {
    for (int i0 = 0; i0 < n; i0 += 256) {
      bool hit[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * 64 + lane;
        hit[u] = i < n && (int64_t)ids[i < n ? i : 0] == r;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint64_t m = __ballot(hit[u]);
        if (hit[u]) list[found + __popcll(m & ((1ull << lane) - 1ull))] = (uint16_t)(i0 + u * 64 + lane);
        found += __popcll(m);
      }
    }
  }
  if (lane == 0) counts[wave] = found;
  __syncthreads();
  // acc += the row's positions first, first + step, ... at one vector of columns
  auto add = [&](float (&acc)[V], const uint16_t* of, int count, int first, int step, int col) {
    const T* at = g + (int64_t)col * V;
    for (int p = first; p < count; p += SCAN_DEEP * step) {
      Pack<T, V> x[SCAN_DEEP];
#pragma unroll
      for (int u = 0; u < SCAN_DEEP; ++u)
        if (p + u * step < count) x[u] = *reinterpret_cast<const Pack<T, V>*>(at + (int64_t)of[p + u * step] * stride);
#pragma unroll
      for (int u = 0; u < SCAN_DEEP; ++u)
        if (p + u * step < count)
#pragma unroll
          for (int k = 0; k < V; ++k) acc[k] += (float)x[u].e[k];
    }
  };
  auto put = [&](int64_t row, float (&acc)[V], int count, int col) {
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = count ? acc[k] * scale : 0.f;
    grad_store<T, V>(out + (row * W + col) * V, acc);
  };
  const int col0 = blockIdx.y * LE, col_step = gridDim.y * LE;
  if (r < rows && found <= LONG) {
    for (int c = col0; c < W; c += col_step) {
      const int col = c + le;
      float acc[V] = {};
      if (col < W) add(acc, list, found, q, Q, col);
      grad_join<V, LE>(acc);
      if (q == 0 && col < W) put(r, acc, found, col);
    }
  }
  for (int k = 0; k < 4; ++k) {                          // the same for every thread: a row that does not exist has no list
    const int count = counts[k];
    if (count <= LONG) continue;
    for (int c = col0; c < W; c += col_step) {
      const int col = c + le;
      float acc[V] = {};
      if (col < W) add(acc, lists[k], count, wave * Q + q, 4 * Q, col);
      grad_join<V, LE>(acc);
      if (wave > 0 && q == 0)
#pragma unroll
        for (int j = 0; j < V; ++j) parts[wave - 1][le * V + j] = acc[j];
      __syncthreads();
      if (wave == 0 && q == 0 && col < W) {
#pragma unroll
        for (int w = 0; w < 3; ++w)
#pragma unroll
          for (int j = 0; j < V; ++j) acc[j] += parts[w][le * V + j];
        put(r0 + k, acc, count, col);
      }
      __syncthreads();
    }
  }
}

// ---- launch policy ---------------------------------------------------------------------------------------------------
int type_size(int dtype) { return dtype == BVI_TYPE_F32 ? 4 : dtype == BVI_TYPE_BF16 || dtype == BVI_TYPE_F16 ? 2 : 0; }

// elements per access: the widest power of two up to 16 bytes that the width, the row stride and the addresses allow
int vector_elements(int64_t width, int64_t stride, int size, const void* a, const void* b) {
  int v = 16 / size;
  while (v > 1 && (width % v || stride % v || (uintptr_t)a % ((size_t)v * size) || (uintptr_t)b % ((size_t)v * size))) v >>= 1;
  return v;
}

template <typename T, int V, typename I>
int launch_lookup(const void* table, int64_t rows, int64_t width, int64_t stride, const void* ids, int64_t n, float scale,
                  void* out, hipStream_t s) {
  const int W = (int)(width / V);
  const int parts = bvi_ceil_div(W, 256), tc = bvi_ceil_div(W, parts);
  const int64_t per_block = (int64_t)(256 / tc) * LK_UNROLL;
  const int64_t blocks = (n + per_block - 1) / per_block;
  hipLaunchKernelGGL((lookup_kernel<T, V, I>), dim3((unsigned)(blocks < (1 << 22) ? blocks : (1 << 22))), dim3(256), 0, s,
                     (const T*)table, stride, rows, (const I*)ids, n, width, W, tc, scale, (T*)out);
  BVI_HIP_CHECK_LAUNCH();
  return BVI_OK;
}

template <typename T, typename I>
int launch_lookup_v(int v, const void* table, int64_t rows, int64_t width, int64_t stride, const void* ids, int64_t n,
                    float scale, void* out, hipStream_t s) {
  switch (v) {
    case 8: if constexpr (sizeof(T) == 2) return launch_lookup<T, 8, I>(table, rows, width, stride, ids, n, scale, out, s);
    case 4: return launch_lookup<T, 4, I>(table, rows, width, stride, ids, n, scale, out, s);
    case 2: return launch_lookup<T, 2, I>(table, rows, width, stride, ids, n, scale, out, s);
    default: return launch_lookup<T, 1, I>(table, rows, width, stride, ids, n, scale, out, s);
  }
}

// ---- the plan's and the scratch's layout, in 4-byte words, 64 words aligned ----
int64_t words(int64_t n) { return (n + 63) / 64 * 64; }

struct SortShape {
  int rounds, n_blocks, passes, bits;
};
SortShape sort_shape(int64_t rows, int64_t n) {
  SortShape t;
  t.rounds = n <= 131072 ? 4 : 16;
  t.n_blocks = bvi_ceil_div(n, 256 * t.rounds);
  int bits = 1;
  while (bits < 32 && ((uint64_t)rows >> bits)) ++bits;                // keys go up to `rows` (padding)
  t.passes = (bits + SORT_MAX_BITS - 1) / SORT_MAX_BITS;
  t.bits = (bits + t.passes - 1) / t.passes;
  return t;
}
struct SortScratch {
  int64_t key, val, count, total, all;
};
SortScratch sort_scratch(int64_t rows, int64_t n) {
  SortScratch t = {};
  if (n <= RANK_MAX) return t;
  const SortShape h = sort_shape(rows, n);
  t.val = words(n);
  t.count = 2 * words(n);
  t.total = t.count + words((int64_t)h.n_blocks << h.bits);
  t.all = t.total + words((int64_t)1 << h.bits);
  return t;
}

template <typename I, int ROUNDS, bool FUSED>
void launch_scatter(const SortShape& h, const I* ids, const uint32_t* k_in, const uint32_t* v_in, int64_t n, int64_t rows,
                    int shift, const uint32_t* count, const uint32_t* total, uint32_t* k_out, uint32_t* v_out,
                    hipStream_t s) {
#define BVI_SCATTER(E)                                                                                                   \
  hipLaunchKernelGGL((sort_scatter_kernel<I, ROUNDS, FUSED, E>), dim3(h.n_blocks), dim3(256), 0, s, ids, k_in, v_in, n, \
                     rows, shift, h.bits, h.n_blocks, count, total, k_out, v_out)
  if (h.bits == 11) BVI_SCATTER(8);
  else if (h.bits == 10) BVI_SCATTER(4);
  else if (h.bits == 9) BVI_SCATTER(2);
  else BVI_SCATTER(1);
#undef BVI_SCATTER
}

template <typename I, int ROUNDS>
void launch_sort(const I* ids, int64_t n, int64_t rows, uint32_t* order, uint32_t* key, uint32_t* ws, hipStream_t s) {
  const SortScratch t = sort_scratch(rows, n);
  const SortShape h = sort_shape(rows, n);
  const uint32_t* k_in = nullptr;
  const uint32_t* v_in = nullptr;
  const int digits = 1 << h.bits;
  uint32_t *count = ws + t.count, *total = ws + t.total;
  for (int p = 0; p < h.passes; ++p) {
    const bool to_plan = ((h.passes - 1 - p) & 1) == 0;                 // the last pass writes the plan
    uint32_t* k_out = to_plan ? key : ws + t.key;
    uint32_t* v_out = to_plan ? order : ws + t.val;
    const int shift = p * h.bits;
    if (h.n_blocks <= SORT_FUSED) {
      hipLaunchKernelGGL((sort_count_kernel<I, ROUNDS>), dim3(h.n_blocks), dim3(256), 0, s, ids, k_in, n, rows, shift,
                         digits, (int64_t)1, (int64_t)digits, count);
      launch_scatter<I, ROUNDS, true>(h, ids, k_in, v_in, n, rows, shift, count, total, k_out, v_out, s);
    } else {
      hipLaunchKernelGGL((sort_count_kernel<I, ROUNDS>), dim3(h.n_blocks), dim3(256), 0, s, ids, k_in, n, rows, shift,
                         digits, (int64_t)h.n_blocks, (int64_t)1, count);
      hipLaunchKernelGGL(sort_scan_kernel, dim3(digits), dim3(256), 0, s, h.n_blocks, count, total);
      launch_scatter<I, ROUNDS, false>(h, ids, k_in, v_in, n, rows, shift, count, total, k_out, v_out, s);
    }
    k_in = k_out;
    v_in = v_out;
  }
}

StartJob start_job(const uint32_t* plan, int64_t n, int64_t rows) {
  StartJob j;
  j.key = plan + words(n);
  j.start = (int32_t*)(plan + 2 * words(n));
  j.n = n;
  j.rows = rows;
  j.blocks = (int)(((n >= rows ? n : rows) + 256) / 256);
  return j;
}

template <typename I>
int launch_plan(const I* ids, int64_t n, int64_t rows, uint32_t* plan, uint32_t* ws, bool with_start, hipStream_t s) {
  uint32_t* order = plan;
  uint32_t* key = plan + words(n);
  if (n > 0 && n <= RANK_MAX)
    hipLaunchKernelGGL((sort_rank_kernel<I>), dim3(bvi_ceil_div(n, 32)), dim3(256), 0, s, ids, (int)n, rows, order, key);
  else if (n > 0 && sort_shape(rows, n).rounds == 4)
    launch_sort<I, 4>(ids, n, rows, order, key, ws, s);
  else if (n > 0)
    launch_sort<I, 16>(ids, n, rows, order, key, ws, s);
  if (with_start) {
    const StartJob j = start_job(plan, n, rows);
    hipLaunchKernelGGL(sort_start_kernel, dim3(j.blocks), dim3(256), 0, s, j);
  }
  BVI_HIP_CHECK_LAUNCH();
  return BVI_OK;
}
int launch_plan_of(const void* ids, int ids_type, int64_t n, int64_t rows, void* plan, void* ws, bool with_start,
                   hipStream_t s) {
  if (ids_type == BVI_IDS_I32)
    return launch_plan((const int32_t*)ids, n, rows, (uint32_t*)plan, (uint32_t*)ws, with_start, s);
  return launch_plan((const int64_t*)ids, n, rows, (uint32_t*)plan, (uint32_t*)ws, with_start, s);
}
int64_t plan_words(int64_t rows, int64_t n) { return 2 * words(n) + words(rows + 1); }

// whether a wave sums a row (else threads do): rows of few vectors that have several positions each.  The vectors of a
// row are counted at their widest: the type is not known where the workspace is sized, an address even less.
bool grad_by_wave(int64_t rows, int64_t width, int64_t n, int size) {
  int v = 16 / size;
  while (v > 1 && width % v) v >>= 1;
  return width / v <= 16 && n >= 4 * rows;
}
// the levels of block sums: another one wherever a row could be left with many entries of the one below
GradLevels grad_levels(int64_t n, int64_t width, bool wave) {
  GradLevels t;
  t.count = 0;
  t.n[0] = 0;
  t.chunk_bits = wave ? 7 : 4;
  t.fan_bits = wave ? 6 : 5;
  int64_t at = 0, m = n >> t.chunk_bits;
  while (t.count < GRAD_LEVELS && m >= 4) {
    t.n[t.count] = m;
    t.at[t.count] = at;
    at += level_space(m * width);
    ++t.count;
    if (m <= 128) break;                          // a launch costs as much as the longest row's 128 vectors
    m >>= t.fan_bits;
  }
  return t;
}
int64_t level_words(int64_t n, int64_t width, bool wave) {
  const GradLevels t = grad_levels(n, width, wave);
  return t.count ? t.at[t.count - 1] + level_space(t.n[t.count - 1] * width) : 0;
}
// whether looking through all ids for every row is the quickest way
bool grad_by_scan(int64_t rows, int64_t n) { return n <= SCAN_MAX && rows * (n > 0 ? n : 1) <= (1 << 22); }

// workgroups side by side for the columns of what `blocks` workgroups would take in `steps` steps: as long as the chip is
// not full (two for each CU)
constexpr int64_t FILL_BLOCKS = 512;
unsigned column_blocks(int64_t blocks, int64_t steps) {
  const int64_t wanted = FILL_BLOCKS / (blocks < 1 ? 1 : blocks);
  return (unsigned)(wanted < 1 ? 1 : wanted < steps ? wanted : steps);
}

struct GradCall {
  const void* g;
  int64_t stride, n, width;
  const void* ids;
  int ids_type;
  bool scan, start_missing;
  const uint32_t* plan;
  int64_t rows;
  float scale;
  void* out;
  float* ws;
  hipStream_t s;
};

// LE = 0: threads
template <typename T, int V, int LE>
int launch_grad(const GradCall& c) {
  const int32_t* order = (const int32_t*)c.plan;
  const uint32_t* key = c.plan + words(c.n);
  const int32_t* start = (const int32_t*)(c.plan + 2 * words(c.n));
  const int W = (int)(c.width / V), parts = bvi_ceil_div(W, 256), tc = bvi_ceil_div(W, parts), per = LE ? 4 : 256 / tc;
  const GradLevels lv = grad_levels(c.n, c.width, LE != 0);
  StartJob job = start_job(c.plan, c.n, c.rows), none = job;
  none.blocks = 0;
  if (!c.start_missing) job = none;
  if (job.blocks && lv.count == 0) hipLaunchKernelGGL(sort_start_kernel, dim3(job.blocks), dim3(256), 0, c.s, job);
  int span_bits = 0;
  for (int l = 0; l < lv.count; ++l) {
    const int bits = l == 0 ? lv.chunk_bits : lv.fan_bits;
    const int64_t wanted = (lv.n[l] + per - 1) / per;
    const unsigned blocks = (unsigned)(wanted < (1 << 22) ? wanted : (1 << 22));
    const unsigned columns = column_blocks(blocks, LE ? 1 : parts);
    span_bits += bits;
    if (l == 0)
      hipLaunchKernelGGL((grad_level_kernel<T, V, LE, true>), dim3(blocks + job.blocks, columns), dim3(256), 0, c.s, (const T*)c.g,
                         c.stride, W, tc, order, key, c.rows, lv.n[0], bits, span_bits, job, c.ws);
    else
      hipLaunchKernelGGL((grad_level_kernel<float, V, LE, false>), dim3(blocks, columns), dim3(256), 0, c.s, c.ws + lv.at[l - 1],
                         c.width, W, tc, order, key, c.rows, lv.n[l], bits, span_bits, none, c.ws + lv.at[l]);
  }
  if (LE) {
    const int64_t blocks = (c.rows + 3) / 4;
    hipLaunchKernelGGL((grad_row_wave_kernel<T, V, LE ? LE : 1>), dim3((unsigned)(blocks < (1 << 22) ? blocks : (1 << 22))),
                       dim3(256), 0, c.s, (const T*)c.g, c.stride, W, order, start, c.rows, lv, c.ws, c.scale, (T*)c.out);
  } else {
    const int64_t blocks = (c.rows + per - 1) / per;
    hipLaunchKernelGGL((grad_row_kernel<T, V>), dim3((unsigned)(blocks < 4096 ? blocks : 4096), column_blocks(blocks, parts)),
                       dim3(256), 0, c.s,
                       (const T*)c.g, c.stride, W, tc, order, start, c.rows, lv, c.ws, c.scale, (T*)c.out);
  }
  BVI_HIP_CHECK_LAUNCH();
  return BVI_OK;
}
template <typename T, int V>
int launch_grad_le(const GradCall& c) {
  if (!grad_by_wave(c.rows, c.width, c.n, (int)sizeof(T))) return launch_grad<T, V, 0>(c);
  const int64_t W = c.width / V;
  if (W > 8) return launch_grad<T, V, 16>(c);
  if (W > 4) return launch_grad<T, V, 8>(c);
  if (W > 2) return launch_grad<T, V, 4>(c);
  if (W > 1) return launch_grad<T, V, 2>(c);
  return launch_grad<T, V, 1>(c);
}

template <typename T, int V, int LE>
int launch_scan_le(const GradCall& c) {
  const int W = (int)(c.width / V);
  const int64_t row_blocks = (c.rows + 3) / 4;
  const dim3 grid((unsigned)row_blocks, column_blocks(row_blocks, (W + (int64_t)LE - 1) / LE));
  if (c.ids_type == BVI_IDS_I32)
    hipLaunchKernelGGL((grad_scan_kernel<T, V, LE, int32_t>), grid, dim3(256), 0, c.s, (const T*)c.g, c.stride, W,
                       (const int32_t*)c.ids, (int)c.n, c.rows, c.scale, (T*)c.out);
  else
    hipLaunchKernelGGL((grad_scan_kernel<T, V, LE, int64_t>), grid, dim3(256), 0, c.s, (const T*)c.g, c.stride, W,
                       (const int64_t*)c.ids, (int)c.n, c.rows, c.scale, (T*)c.out);
  BVI_HIP_CHECK_LAUNCH();
  return BVI_OK;
}
template <typename T, int V>
int launch_scan(const GradCall& c) {
  const int64_t W = c.width / V;
  // 64 lanes across the columns where that leaves workgroups enough, else 16 with four positions at a time
  if (W >= 48 && (c.rows + 3) / 4 * ((W + 63) / 64) >= FILL_BLOCKS / 2) return launch_scan_le<T, V, 64>(c);
  if (W >= 6) return launch_scan_le<T, V, 16>(c);
  if (W >= 2) return launch_scan_le<T, V, 4>(c);
  return launch_scan_le<T, V, 1>(c);
}

template <typename T>
int launch_grad_v(const GradCall& c) {
  const int v = vector_elements(c.width, c.stride, (int)sizeof(T), c.g, c.out);
#define BVI_GRAD_CALL(X) return c.scan ? launch_scan<T, X>(c) : launch_grad_le<T, X>(c)
  switch (v) {
    case 8: if constexpr (sizeof(T) == 2) BVI_GRAD_CALL(8);
    case 4: BVI_GRAD_CALL(4);
    case 2: BVI_GRAD_CALL(2);
    default: BVI_GRAD_CALL(1);
  }
#undef BVI_GRAD_CALL
}

// addresses between two elements, and scratch that the kernels' 16-byte accesses would straddle, are refused
bool off_type(const void* p, int size) { return (uintptr_t)p % (size_t)size != 0; }
int ids_size(int ids_type) { return ids_type == BVI_IDS_I32 ? 4 : 8; }

bool sizes_ok(int64_t rows, int64_t n) {
  return rows >= 1 && rows <= BVI_LOOKUP_MAX && n >= 0 && n <= BVI_LOOKUP_MAX;
}

}  // namespace

extern "C" {

int bvi_lookup(const void* table, int dtype, int64_t rows, int64_t width, int64_t row_stride, const void* ids,
               int ids_type, int64_t n, float scale, void* out, void* stream) {
  const int size = type_size(dtype);
  if (!table || !size || width < 1 || row_stride < width || n < 0 || rows < 1 || (n > 0 && (!ids || !out)))
    return BVI_ERR_ARG;
  if (ids_type != BVI_IDS_I32 && ids_type != BVI_IDS_I64) return BVI_ERR_ARG;
  if (off_type(table, size) || off_type(out, size) || off_type(ids, ids_size(ids_type))) return BVI_ERR_ARG;
  if (width > BVI_LOOKUP_MAX || rows > BVI_LOOKUP_MAX || n > BVI_LOOKUP_MAX) return BVI_ERR_UNSUPPORTED;
  if (n == 0) return BVI_OK;
  const hipStream_t s = (hipStream_t)stream;
  const int v = vector_elements(width, row_stride, size, table, out);
#define BVI_LOOKUP_CALL(T)                                                                                       \
  return ids_type == BVI_IDS_I32 ? launch_lookup_v<T, int32_t>(v, table, rows, width, row_stride, ids, n, scale, out, s) \
                                 : launch_lookup_v<T, int64_t>(v, table, rows, width, row_stride, ids, n, scale, out, s)
  if (dtype == BVI_TYPE_F32) BVI_LOOKUP_CALL(float);
  if (dtype == BVI_TYPE_BF16) BVI_LOOKUP_CALL(__bf16);
  BVI_LOOKUP_CALL(_Float16);
#undef BVI_LOOKUP_CALL
}

int bvi_lookup_plan_bytes(int64_t rows, int64_t n, size_t* plan_bytes, size_t* ws_bytes) {
  if (!plan_bytes || !ws_bytes || rows < 1 || n < 0) return BVI_ERR_ARG;
  if (!sizes_ok(rows, n)) return BVI_ERR_UNSUPPORTED;
  *plan_bytes = 4 * (size_t)plan_words(rows, n);
  *ws_bytes = 4 * (size_t)sort_scratch(rows, n).all;
  return BVI_OK;
}

int bvi_lookup_plan(const void* ids, int ids_type, int64_t n, int64_t rows, void* plan, size_t plan_bytes, void* ws,
                    size_t ws_bytes, void* stream) {
  if ((!ids && n > 0) || n < 0 || rows < 1 || (ids_type != BVI_IDS_I32 && ids_type != BVI_IDS_I64)) return BVI_ERR_ARG;
  if (off_type(ids, ids_size(ids_type)) || off_type(plan, 16) || off_type(ws, 16)) return BVI_ERR_ARG;
  if (!sizes_ok(rows, n)) return BVI_ERR_UNSUPPORTED;
  size_t need, scratch;
  bvi_lookup_plan_bytes(rows, n, &need, &scratch);
  if (!plan || plan_bytes < need || (scratch && (!ws || ws_bytes < scratch))) return BVI_ERR_WORKSPACE;
  return launch_plan_of(ids, ids_type, n, rows, plan, ws, true, (hipStream_t)stream);
}

// workspace: the level sums, and without a plan the call's own plan and its sort's scratch
int bvi_lookup_grad_ws_bytes(int64_t rows, int64_t width, int64_t n, int has_plan, size_t* ws_bytes) {
  if (!ws_bytes || rows < 1 || width < 1 || n < 0) return BVI_ERR_ARG;
  if (!sizes_ok(rows, n) || width > BVI_LOOKUP_MAX) return BVI_ERR_UNSUPPORTED;
  *ws_bytes = 0;
  if (!has_plan && grad_by_scan(rows, n)) return BVI_OK;
  // the type is not known here: the larger of the two forms' levels
  const int64_t a = level_words(n, width, false), b = level_words(n, width, true);
  *ws_bytes = 4 * (size_t)((a > b ? a : b) + (has_plan ? 0 : plan_words(rows, n) + sort_scratch(rows, n).all));
  return BVI_OK;
}

int bvi_lookup_grad(const void* grad_out, int dtype, int64_t n, int64_t width, int64_t row_stride, const void* ids,
                    int ids_type, const void* plan, int64_t rows, float scale, void* grad_table, void* ws,
                    size_t ws_bytes, void* stream) {
  if ((!grad_out && n > 0) || !type_size(dtype) || n < 0 || width < 1 || row_stride < width || rows < 1 || !grad_table)
    return BVI_ERR_ARG;
  if ((!plan && !ids && n > 0) || (ids && (ids_type != BVI_IDS_I32 && ids_type != BVI_IDS_I64))) return BVI_ERR_ARG;
  if (off_type(grad_out, type_size(dtype)) || off_type(grad_table, type_size(dtype)) ||
      (ids && off_type(ids, ids_size(ids_type))) || off_type(plan, 16) || off_type(ws, 16))
    return BVI_ERR_ARG;
  if (!sizes_ok(rows, n) || width > BVI_LOOKUP_MAX) return BVI_ERR_UNSUPPORTED;
  size_t need;
  bvi_lookup_grad_ws_bytes(rows, width, n, plan != nullptr, &need);
  if (need && (!ws || ws_bytes < need)) return BVI_ERR_WORKSPACE;
  // the same way with and without a plan, so that both give the same bits
  const bool scan = (ids || n == 0) && grad_by_scan(rows, n);
  GradCall c{grad_out, row_stride, n, width, ids, ids_type, scan, false, (const uint32_t*)plan, rows, scale, grad_table,
             (float*)ws, (hipStream_t)stream};
  if (!plan && !scan) {
    uint32_t* own = (uint32_t*)((char*)ws + need) - plan_words(rows, n) - sort_scratch(rows, n).all;
    const int st = launch_plan_of(ids, ids_type, n, rows, own, own + plan_words(rows, n), false, c.s);
    if (st) return st;
    c.plan = own;
    c.start_missing = true;
  }
  if (dtype == BVI_TYPE_F32) return launch_grad_v<float>(c);
  if (dtype == BVI_TYPE_BF16) return launch_grad_v<__bf16>(c);
  return launch_grad_v<_Float16>(c);
}

}  // extern "C"
