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
// else equal parts), 256 / tc rows per step, four steps' ids and vectors in flight.
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

// ---- the sort: least significant digit first, at most 8 bits per pass, stable ----------------------------------------
constexpr int RS_THREADS = 256, RS_ITEMS = 16, RS_TILE = RS_THREADS * RS_ITEMS, RS_DIGITS = 256;

// the sort key of position i: the id, or `rows` for padding; later passes read the keys of the pass before
template <typename I>
__device__ __forceinline__ uint32_t rs_key(const I* __restrict__ ids, const uint32_t* __restrict__ keys, int64_t rows,
                                           int64_t i) {
  if (keys) return keys[i];
  const int64_t id = (int64_t)ids[i];
  return (uint32_t)(id >= 0 && id < rows ? id : rows);
}

template <typename I>
__global__ __launch_bounds__(RS_THREADS) void sort_count_kernel(const I* __restrict__ ids,
                                                                const uint32_t* __restrict__ keys, int64_t n,
                                                                int64_t rows, int shift, uint32_t mask, int n_blocks,
                                                                uint32_t* __restrict__ count) {
  __shared__ uint32_t hist[RS_DIGITS];
  hist[threadIdx.x] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * RS_TILE;
#pragma unroll
  for (int j = 0; j < RS_ITEMS; ++j) {
    const int64_t i = base + j * RS_THREADS + threadIdx.x;
    if (i < n) atomicAdd(&hist[(rs_key(ids, keys, rows, i) >> shift) & mask], 1u);   // integer counts: order-free
  }
  __syncthreads();
  count[(int64_t)threadIdx.x * n_blocks + blockIdx.x] = hist[threadIdx.x];
}

// workgroup d: exclusive sums of digit d's counts over the blocks, in place, and the digit's total
__global__ __launch_bounds__(256) void sort_scan_kernel(int n_blocks, uint32_t* __restrict__ count,
                                                        uint32_t* __restrict__ total) {
  __shared__ uint32_t wave_sum[4];
  uint32_t* c = count + (int64_t)blockIdx.x * n_blocks;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t carry = 0;
  for (int b0 = 0; b0 < n_blocks; b0 += 256) {
    const int b = b0 + threadIdx.x;
    const uint32_t own = b < n_blocks ? c[b] : 0u;
    uint32_t v = own;
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t t = __shfl_up(v, off, 64);
      if (lane >= off) v += t;
    }
    if (lane == 63) wave_sum[wave] = v;
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

// Each wave owns RS_TILE / 4 consecutive positions and ranks them 64 at a time: eight ballots give the lanes with the
// same digit, a counter per wave and digit the earlier rounds'.  Positions are visited in ascending order: stable.
template <typename I>
__global__ __launch_bounds__(RS_THREADS) void sort_scatter_kernel(
    const I* __restrict__ ids, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ vals, int64_t n,
    int64_t rows, int shift, uint32_t mask, int n_blocks, const uint32_t* __restrict__ count,
    const uint32_t* __restrict__ total, uint32_t* __restrict__ keys_out, uint32_t* __restrict__ vals_out) {
  __shared__ uint32_t seen[4][RS_DIGITS];
  __shared__ uint32_t wave_sum[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int w = 0; w < 4; ++w) seen[w][threadIdx.x] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * RS_TILE + wave * (RS_TILE / 4) + lane;
  uint32_t key[RS_ITEMS], rank[RS_ITEMS];
#pragma unroll
  for (int j = 0; j < RS_ITEMS; ++j) {
    const int64_t i = base + j * 64;
    key[j] = i < n ? rs_key(ids, keys, rows, i) : 0u;
  }
  volatile uint32_t* mine = seen[wave];
#pragma unroll
  for (int j = 0; j < RS_ITEMS; ++j) {
    const bool in = base + j * 64 < n;
    const uint32_t d = (key[j] >> shift) & mask;
    uint64_t same = __ballot(in);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
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
  // where each wave's entries of digit d go: digits before d, d's entries of earlier blocks, of earlier waves
  const int d = threadIdx.x;
  const uint32_t own = total[d];
  uint32_t v = own;
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t t = __shfl_up(v, off, 64);
    if (lane >= off) v += t;
  }
  if (lane == 63) wave_sum[wave] = v;
  __syncthreads();
  uint32_t at = v - own + count[(int64_t)d * n_blocks + blockIdx.x];
  for (int w = 0; w < wave; ++w) at += wave_sum[w];
  for (int w = 0; w < 4; ++w) {
    const uint32_t c = seen[w][d];
    seen[w][d] = at;
    at += c;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < RS_ITEMS; ++j) {
    const int64_t i = base + j * 64;
    if (i < n) {
      const uint32_t to = seen[wave][(key[j] >> shift) & mask] + rank[j];
      keys_out[to] = key[j];
      vals_out[to] = vals ? vals[i] : (uint32_t)i;
    }
  }
}

// start[r] = number of sorted keys below r
__global__ __launch_bounds__(256) void sort_start_kernel(const uint32_t* __restrict__ key, int64_t n, int64_t rows,
                                                         int32_t* __restrict__ start) {
  const int64_t r = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (r > rows) return;
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if ((int64_t)key[mid] < r) lo = mid + 1;
    else hi = mid;
  }
  start[r] = (int32_t)lo;
}

// ---- gradient ------------------------------------------------------------------------------------------------------
// A wave is LE lanes across the columns times 64 / LE lanes over positions.  A row read at most a few hundred times is
// one wave's work; where a row has more, whole blocks of `chunk` sorted positions that belong to it ("pure" blocks) are
// summed beforehand by a wave each, and blocks of 64 pure blocks once more.
constexpr int LG_FAN = 64;

// acc += rows src[order[p]] for p in [s, e); lane q takes p = s + q, s + q + Q, ...; four loads in flight
template <typename S, int V, int LE, bool PERM>
__device__ __forceinline__ void lg_sum(float (&acc)[V], const S* __restrict__ src, int64_t stride, int64_t col,
                                       const int32_t* __restrict__ order, int64_t s, int64_t e, int q, bool active) {
  constexpr int Q = 64 / LE;
  if (!active) return;
  int64_t p = s + q;
  for (; p + 3 * Q < e; p += 4 * Q) {
    Pack<S, V> x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t i = PERM ? (int64_t)order[p + u * Q] : p + u * Q;
      x[u] = *reinterpret_cast<const Pack<S, V>*>(src + i * stride + col);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] += (float)x[u].e[k];
  }
  for (; p < e; p += Q) {
    const int64_t i = PERM ? (int64_t)order[p] : p;
    const Pack<S, V> x = *reinterpret_cast<const Pack<S, V>*>(src + i * stride + col);
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] += (float)x.e[k];
  }
}

template <int V, int LE>
__device__ __forceinline__ void lg_reduce(float (&acc)[V]) {
#pragma unroll
  for (int off = LE; off < 64; off <<= 1)
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] += __shfl_xor(acc[k], off, 64);
}

// wave b: the sum of sorted positions [b chunk, (b + 1) chunk) if they belong to one row
template <typename T, int V, int LE>
__global__ __launch_bounds__(256) void grad_chunk_kernel(const T* __restrict__ g, int64_t stride, int W,
                                                         const int32_t* __restrict__ order,
                                                         const uint32_t* __restrict__ key, int64_t rows, int64_t n_chunks,
                                                         int chunk, float* __restrict__ part) {
  const int64_t b = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (b >= n_chunks) return;
  const uint32_t k0 = key[b * chunk];
  if (k0 != key[b * chunk + chunk - 1] || k0 >= rows) return;
  const int lane = threadIdx.x & 63, q = lane / LE, le = lane % LE;
  for (int col = le; col - le < W; col += LE) {
    float acc[V] = {};
    lg_sum<T, V, LE, true>(acc, g, stride, (int64_t)col * V, order, b * chunk, (b + 1) * chunk, q, col < W);
    lg_reduce<V, LE>(acc);
    if (q == 0 && col < W)
#pragma unroll
      for (int k = 0; k < V; ++k) part[(b * W + col) * V + k] = acc[k];
  }
}

// wave b: the sum of LG_FAN pure blocks if they belong to one row
template <int V, int LE>
__global__ __launch_bounds__(256) void grad_fan_kernel(const float* __restrict__ part, int W,
                                                       const uint32_t* __restrict__ key, int64_t rows, int64_t n_fans,
                                                       int chunk, float* __restrict__ part2) {
  const int64_t b = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (b >= n_fans) return;
  const int64_t span = (int64_t)chunk * LG_FAN;
  const uint32_t k0 = key[b * span];
  if (k0 != key[(b + 1) * span - 1] || k0 >= rows) return;
  const int lane = threadIdx.x & 63, q = lane / LE, le = lane % LE;
  for (int col = le; col - le < W; col += LE) {
    float acc[V] = {};
    lg_sum<float, V, LE, false>(acc, part, (int64_t)W * V, (int64_t)col * V, nullptr, b * LG_FAN, (b + 1) * LG_FAN, q,
                                col < W);
    lg_reduce<V, LE>(acc);
    if (q == 0 && col < W)
#pragma unroll
      for (int k = 0; k < V; ++k) part2[(b * W + col) * V + k] = acc[k];
  }
}

template <typename T, int V, int LE, typename O>
__global__ __launch_bounds__(256) void grad_row_kernel(const T* __restrict__ g, int64_t stride, int W,
                                                       const int32_t* __restrict__ order,
                                                       const int32_t* __restrict__ start, int64_t rows, int64_t n_chunks,
                                                       int64_t n_fans, int chunk, const float* __restrict__ part,
                                                       const float* __restrict__ part2, float scale,
                                                       O* __restrict__ out) {
  const int lane = threadIdx.x & 63, q = lane / LE, le = lane % LE;
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += (int64_t)gridDim.x * 4) {
    const int64_t s = start[r], e = start[r + 1];
    // positions: [s, c0 chunk) and [c1 chunk, e) one by one; pure blocks: [c0, f0 FAN) and [f1 FAN, c1); fans [f0, f1)
    int64_t c0 = (s + chunk - 1) / chunk, c1 = e / chunk;
    if (c1 > n_chunks) c1 = n_chunks;
    const bool split = c0 < c1;
    int64_t f0 = (c0 + LG_FAN - 1) / LG_FAN, f1 = c1 / LG_FAN;
    if (f1 > n_fans) f1 = n_fans;
    const bool fans = split && f0 < f1;
    for (int col = le; col - le < W; col += LE) {
      const bool on = col < W;
      const int64_t at = (int64_t)col * V, ps = (int64_t)W * V;
      float acc[V] = {};
      lg_sum<T, V, LE, true>(acc, g, stride, at, order, s, split ? c0 * chunk : e, q, on);
      if (split) {
        lg_sum<float, V, LE, false>(acc, part, ps, at, nullptr, c0, fans ? f0 * LG_FAN : c1, q, on);
        if (fans) {
          lg_sum<float, V, LE, false>(acc, part2, ps, at, nullptr, f0, f1, q, on);
          lg_sum<float, V, LE, false>(acc, part, ps, at, nullptr, f1 * LG_FAN, c1, q, on);
        }
        lg_sum<T, V, LE, true>(acc, g, stride, at, order, c1 * chunk, e, q, on);
      }
      lg_reduce<V, LE>(acc);
      if (q == 0 && on) {
        Pack<O, V> o;
  #pragma unroll
        for (int k = 0; k < V; ++k) o.e[k] = (O)(e > s ? acc[k] * scale : 0.f);
        *reinterpret_cast<Pack<O, V>*>(out + r * ps + at) = o;
      }
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
struct SortScratch {
  int64_t key, val, count, total, all;
};
SortScratch sort_scratch(int64_t n) {
  SortScratch t;
  t.key = 0;
  t.val = words(n);
  t.count = 2 * words(n);
  t.total = t.count + words((int64_t)RS_DIGITS * bvi_ceil_div(n, RS_TILE));
  t.all = t.total + RS_DIGITS;
  return t;
}

template <typename I>
int launch_plan(const I* ids, int64_t n, int64_t rows, uint32_t* plan, uint32_t* ws, hipStream_t s) {
  uint32_t* order = plan;
  uint32_t* key = plan + words(n);
  int32_t* start = (int32_t*)(plan + 2 * words(n));
  if (n > 0) {
    const SortScratch t = sort_scratch(n);
    const int n_blocks = bvi_ceil_div(n, RS_TILE);
    int bits = 1;
    while (bits < 32 && ((uint64_t)rows >> bits)) ++bits;              // keys go up to `rows` (padding)
    const int passes = (bits + 7) / 8, per = (bits + passes - 1) / passes;
    const uint32_t* k_in = nullptr;
    const uint32_t* v_in = nullptr;
    for (int p = 0; p < passes; ++p) {
      const bool to_plan = ((passes - 1 - p) & 1) == 0;                 // the last pass writes the plan
      uint32_t* k_out = to_plan ? key : ws + t.key;
      uint32_t* v_out = to_plan ? order : ws + t.val;
      const uint32_t mask = (1u << per) - 1u;
      hipLaunchKernelGGL((sort_count_kernel<I>), dim3(n_blocks), dim3(RS_THREADS), 0, s, ids, k_in, n, rows, p * per,
                         mask, n_blocks, ws + t.count);
      hipLaunchKernelGGL(sort_scan_kernel, dim3(RS_DIGITS), dim3(256), 0, s, n_blocks, ws + t.count, ws + t.total);
      hipLaunchKernelGGL((sort_scatter_kernel<I>), dim3(n_blocks), dim3(RS_THREADS), 0, s, ids, k_in, v_in, n, rows,
                         p * per, mask, n_blocks, ws + t.count, ws + t.total, k_out, v_out);
      k_in = k_out;
      v_in = v_out;
    }
  }
  hipLaunchKernelGGL(sort_start_kernel, dim3((unsigned)((rows + 256) / 256)), dim3(256), 0, s, key, n, rows, start);
  BVI_HIP_CHECK_LAUNCH();
  return BVI_OK;
}

// positions per pure block: a few vectors per lane, more where that would make very many blocks
int64_t grad_chunk(int64_t n) { return n >= (1 << 22) ? 512 : 128; }
int64_t grad_chunks(int64_t n) { return n / grad_chunk(n); }
int64_t grad_fans(int64_t n) { return grad_chunks(n) >= 4 * LG_FAN ? grad_chunks(n) / LG_FAN : 0; }

template <typename T, int V, int LE, typename O>
int launch_grad(const void* grad_out, int64_t stride, int64_t n, int64_t width, const uint32_t* plan, int64_t rows,
                float scale, void* grad_table, float* ws, hipStream_t s) {
  const int32_t* order = (const int32_t*)plan;
  const uint32_t* key = plan + words(n);
  const int32_t* start = (const int32_t*)(plan + 2 * words(n));
  const int W = (int)(width / V), chunk = (int)grad_chunk(n);
  const int64_t n_chunks = grad_chunks(n), n_fans = grad_fans(n);
  float* part = ws;
  float* part2 = ws + words(n_chunks * width);
  if (n_chunks > 0) {
    hipLaunchKernelGGL((grad_chunk_kernel<T, V, LE>), dim3(bvi_ceil_div(n_chunks, 4)), dim3(256), 0, s,
                       (const T*)grad_out, stride, W, order, key, rows, n_chunks, chunk, part);
    if (n_fans > 0)
      hipLaunchKernelGGL((grad_fan_kernel<V, LE>), dim3(bvi_ceil_div(n_fans, 4)), dim3(256), 0, s, part, W, key, rows,
                         n_fans, chunk, part2);
  }
  hipLaunchKernelGGL((grad_row_kernel<T, V, LE, O>), dim3((unsigned)((rows + 3) / 4 < (1 << 23) ? (rows + 3) / 4 : (1 << 23))),
                     dim3(256), 0, s, (const T*)grad_out, stride, W, order, start, rows, n_chunks, n_fans, chunk, part, part2, scale,
                     (O*)grad_table);
  BVI_HIP_CHECK_LAUNCH();
  return BVI_OK;
}

template <typename T, int V, typename O>
int launch_grad_le(const void* g, int64_t stride, int64_t n, int64_t width, const uint32_t* plan, int64_t rows,
                   float scale, void* out, float* ws, hipStream_t s) {
  // lanes across the columns: the most that leave at most an eighth of the lanes without a column
  const int W = (int)(width / V);
  int le = 64;
  while (le > 1 && (int64_t)bvi_ceil_div(W, le) * le * 7 > (int64_t)W * 8) le >>= 1;
  switch (le) {
    case 64: return launch_grad<T, V, 64, O>(g, stride, n, width, plan, rows, scale, out, ws, s);
    case 32: return launch_grad<T, V, 32, O>(g, stride, n, width, plan, rows, scale, out, ws, s);
    case 16: return launch_grad<T, V, 16, O>(g, stride, n, width, plan, rows, scale, out, ws, s);
    case 8: return launch_grad<T, V, 8, O>(g, stride, n, width, plan, rows, scale, out, ws, s);
    case 4: return launch_grad<T, V, 4, O>(g, stride, n, width, plan, rows, scale, out, ws, s);
    case 2: return launch_grad<T, V, 2, O>(g, stride, n, width, plan, rows, scale, out, ws, s);
    default: return launch_grad<T, V, 1, O>(g, stride, n, width, plan, rows, scale, out, ws, s);
  }
}

template <typename T>
int launch_grad_v(const void* g, int64_t stride, int64_t n, int64_t width, const uint32_t* plan, int64_t rows,
                  float scale, void* out, float* ws, hipStream_t s) {
  switch (vector_elements(width, stride, (int)sizeof(T), g, out)) {
    case 8: if constexpr (sizeof(T) == 2) return launch_grad_le<T, 8, T>(g, stride, n, width, plan, rows, scale, out, ws, s);
    case 4: return launch_grad_le<T, 4, T>(g, stride, n, width, plan, rows, scale, out, ws, s);
    case 2: return launch_grad_le<T, 2, T>(g, stride, n, width, plan, rows, scale, out, ws, s);
    default: return launch_grad_le<T, 1, T>(g, stride, n, width, plan, rows, scale, out, ws, s);
  }
}

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
  if (width > BVI_LOOKUP_MAX) return BVI_ERR_UNSUPPORTED;
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
  *plan_bytes = 4 * (size_t)(2 * words(n) + words(rows + 1));
  *ws_bytes = 4 * (size_t)sort_scratch(n).all;
  return BVI_OK;
}

int bvi_lookup_plan(const void* ids, int ids_type, int64_t n, int64_t rows, void* plan, size_t plan_bytes, void* ws,
                    size_t ws_bytes, void* stream) {
  if ((!ids && n > 0) || n < 0 || rows < 1 || (ids_type != BVI_IDS_I32 && ids_type != BVI_IDS_I64)) return BVI_ERR_ARG;
  if (!sizes_ok(rows, n)) return BVI_ERR_UNSUPPORTED;
  size_t need, scratch;
  bvi_lookup_plan_bytes(rows, n, &need, &scratch);
  if (!plan || plan_bytes < need || (n > 0 && (!ws || ws_bytes < scratch))) return BVI_ERR_WORKSPACE;
  if (ids_type == BVI_IDS_I32)
    return launch_plan((const int32_t*)ids, n, rows, (uint32_t*)plan, (uint32_t*)ws, (hipStream_t)stream);
  return launch_plan((const int64_t*)ids, n, rows, (uint32_t*)plan, (uint32_t*)ws, (hipStream_t)stream);
}

int bvi_lookup_grad_ws_bytes(int64_t rows, int64_t width, int64_t n, size_t* ws_bytes) {
  if (!ws_bytes || rows < 1 || width < 1 || n < 0) return BVI_ERR_ARG;
  if (!sizes_ok(rows, n) || width > BVI_LOOKUP_MAX) return BVI_ERR_UNSUPPORTED;
  *ws_bytes = 4 * (size_t)(words(grad_chunks(n) * width) + words(grad_fans(n) * width));
  return BVI_OK;
}

int bvi_lookup_grad(const void* grad_out, int dtype, int64_t n, int64_t width, int64_t row_stride, const void* plan,
                    int64_t rows, float scale, void* grad_table, void* ws, size_t ws_bytes, void* stream) {
  if ((!grad_out && n > 0) || !type_size(dtype) || n < 0 || width < 1 || row_stride < width || rows < 1 || !plan ||
      !grad_table)
    return BVI_ERR_ARG;
  if (!sizes_ok(rows, n) || width > BVI_LOOKUP_MAX) return BVI_ERR_UNSUPPORTED;
  size_t need;
  bvi_lookup_grad_ws_bytes(rows, width, n, &need);
  if (need && (!ws || ws_bytes < need)) return BVI_ERR_WORKSPACE;
  const hipStream_t s = (hipStream_t)stream;
  const uint32_t* p = (const uint32_t*)plan;
  if (dtype == BVI_TYPE_F32)
    return launch_grad_v<float>(grad_out, row_stride, n, width, p, rows, scale, grad_table, (float*)ws, s);
  if (dtype == BVI_TYPE_BF16)
    return launch_grad_v<__bf16>(grad_out, row_stride, n, width, p, rows, scale, grad_table, (float*)ws, s);
  return launch_grad_v<_Float16>(grad_out, row_stride, n, width, p, rows, scale, grad_table, (float*)ws, s);
}

}  // extern "C"
