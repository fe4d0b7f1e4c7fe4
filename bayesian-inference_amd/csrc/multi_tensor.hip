// Operators over a list of tensors (the gradients or variables of a model), each in a few launches whatever the list:
//   global norm           s = sqrt(sum_t sum_i g_t[i]^2)                                    (tf.linalg.global_norm)
//   clip by global norm   out_t = g_t * min(1, clip / s); every entry NaN if s is not finite (tf.clip_by_global_norm)
//   Adam step             per variable g <- g min(1, clip / |g|) (the reference's tf.clip_by_norm, vi.py:70), then
//                         jointly g <- g min(1, global_clip / s) (tf.optimizers.Adam(global_clipnorm=)), then
//                         m <- b1 m + (1 - b1) g;  v <- b2 v + (1 - b2) g^2;  x -= lr_t m / (sqrt(v) + eps)
// The pointers travel in the kernel arguments (MT_MAX tensors per launch), so a call copies nothing to the device and
// can be recorded into a graph.  A tensor is cut into items of MT_ITEM elements; a workgroup takes items in turn.
// Squares are summed in double: no overflow for any float, and the order of the sum is fixed by the sizes alone.
#include "bvi_common.h"

#include <algorithm>
#include <new>
#include <utility>
#include <vector>

namespace {

constexpr int MT_MAX = 80;            // tensors per launch: the arguments stay below 4 KB
constexpr int MT_ITEM = 4096;         // elements per item: 16 per thread
constexpr int MT_NORM_ITEM = 4 * MT_ITEM;   // of Adam's norm pass, whose partial sums one workgroup adds up
constexpr int MT_BLOCKS = 1024;       // workgroups of a norm pass: 4 per CU, and as many partial sums at most
// A list of at most MT_SMALL items of MT_SMALL_ITEM elements and MT_SMALL_ALL elements in all is one workgroup's work, in
// one launch (Adam over one variable: 6.9 us at 4096 elements, 10.5 at 16384, 17.0 at 32768, where the three launches of a
// longer list take 11.7).
constexpr int MT_SMALL_ITEM = 1024, MT_SMALL = 32, MT_SMALL_ALL = 16384;

struct NormArgs {
  const void* src[MT_MAX];
  int64_t n[MT_MAX];
  int32_t first[MT_MAX + 1];          // first item of each tensor
  uint8_t type[MT_MAX];
  int count;
};
struct ClipArgs {
  NormArgs in;
  void* dst[MT_MAX];
};
struct AdamArgs {
  float* x[MT_MAX];
  float* g[MT_MAX];
  float* m[MT_MAX];
  float* v[MT_MAX];
  int64_t n[MT_MAX];
  int32_t first[MT_MAX + 1];
  int count;
};

// the tensor that item `it` belongs to (first[] ascends; tensors without elements have no item)
__device__ __forceinline__ int mt_find(const int32_t* first, int count, int it) {
  int lo = 0, hi = count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= it) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <typename T>
struct alignas(16) Vec16 {
  T e[16 / sizeof(T)];
};

// PAST_CACHE: results that no cache will hold until they are read need not push the operands out of it (fixed at compile
// time: a branch between the two stores is folded into one plain store)
template <bool PAST_CACHE, typename T>
__device__ __forceinline__ void store16(T* to, const Vec16<T>& x) {
  if (PAST_CACHE) {
    f32x4 y;
    __builtin_memcpy(&y, &x, 16);
    __builtin_nontemporal_store(y, reinterpret_cast<f32x4*>(to));
  } else {
    *reinterpret_cast<Vec16<T>*>(to) = x;
  }
}

// sum of squares of p[0, len), `lanes` threads side by side
template <typename T>
__device__ __forceinline__ double mt_square_sum(const T* __restrict__ p, int len, int id, int lanes) {
  constexpr int V = 16 / sizeof(T);
  double s = 0.0;
  int done = 0;
  if ((uintptr_t)p % 16 == 0 && len == MT_ITEM && lanes == 256) {      // all of a thread's vectors in flight
    Vec16<T> x[MT_ITEM / 256 / V];
#pragma unroll
    for (int u = 0; u < MT_ITEM / 256 / V; ++u) x[u] = *reinterpret_cast<const Vec16<T>*>(p + (u * 256 + id) * V);
#pragma unroll
    for (int u = 0; u < MT_ITEM / 256 / V; ++u)
#pragma unroll
      for (int k = 0; k < V; ++k) s = fma((double)(float)x[u].e[k], (double)(float)x[u].e[k], s);
    return s;
  }
  if ((uintptr_t)p % 16 == 0) {
    done = len / V * V;
    for (int i = id * V; i < done; i += lanes * V) {
      const Vec16<T> x = *reinterpret_cast<const Vec16<T>*>(p + i);
#pragma unroll
      for (int k = 0; k < V; ++k) s = fma((double)(float)x.e[k], (double)(float)x.e[k], s);
    }
  }
  for (int i = done + id; i < len; i += lanes) s = fma((double)(float)p[i], (double)(float)p[i], s);
  return s;
}

__device__ __forceinline__ double mt_item_square_sum(const NormArgs& a, int t, int64_t at, int len, int id, int lanes) {
  if (a.type[t] == BVI_TYPE_F32) return mt_square_sum((const float*)a.src[t] + at, len, id, lanes);
  if (a.type[t] == BVI_TYPE_BF16) return mt_square_sum((const __bf16*)a.src[t] + at, len, id, lanes);
  return mt_square_sum((const _Float16*)a.src[t] + at, len, id, lanes);
}

template <bool PAST_CACHE, typename T>
__device__ __forceinline__ void mt_scale(const T* p, T* o, int len, float factor, int id, int lanes) {   // o may be p
  constexpr int V = 16 / sizeof(T);
  int done = 0;
  if (((uintptr_t)p | (uintptr_t)o) % 16 == 0 && len == MT_ITEM && lanes == 256) {
    Vec16<T> x[MT_ITEM / 256 / V];
#pragma unroll
    for (int u = 0; u < MT_ITEM / 256 / V; ++u) x[u] = *reinterpret_cast<const Vec16<T>*>(p + (u * 256 + id) * V);
#pragma unroll
    for (int u = 0; u < MT_ITEM / 256 / V; ++u) {
#pragma unroll
      for (int k = 0; k < V; ++k) x[u].e[k] = (T)((float)x[u].e[k] * factor);
      store16<PAST_CACHE>(o + (u * 256 + id) * V, x[u]);
    }
    return;
  }
  if (((uintptr_t)p | (uintptr_t)o) % 16 == 0) {
    done = len / V * V;
    for (int i = id * V; i < done; i += lanes * V) {
      Vec16<T> x = *reinterpret_cast<const Vec16<T>*>(p + i);
#pragma unroll
      for (int k = 0; k < V; ++k) x.e[k] = (T)((float)x.e[k] * factor);     // the product in float, rounded once
      *reinterpret_cast<Vec16<T>*>(o + i) = x;
    }
  }
  for (int i = done + id; i < len; i += lanes) o[i] = (T)((float)p[i] * factor);
}

template <bool PAST_CACHE>
__device__ __forceinline__ void mt_item_scale(const ClipArgs& a, int t, int64_t at, int len, float factor, int id,
                                              int lanes) {
  if (a.in.type[t] == BVI_TYPE_F32)
    mt_scale<PAST_CACHE>((const float*)a.in.src[t] + at, (float*)a.dst[t] + at, len, factor, id, lanes);
  else if (a.in.type[t] == BVI_TYPE_BF16)
    mt_scale<PAST_CACHE>((const __bf16*)a.in.src[t] + at, (__bf16*)a.dst[t] + at, len, factor, id, lanes);
  else
    mt_scale<PAST_CACHE>((const _Float16*)a.in.src[t] + at, (_Float16*)a.dst[t] + at, len, factor, id, lanes);
}

__device__ __forceinline__ double mt_wave_sum(double v) {
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}
__device__ __forceinline__ double mt_block_sum(double v, double* red) {
  v = mt_wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double t = 0.0;
  for (int w = 0; w < (int)(blockDim.x >> 6); ++w) t += red[w];
  return t;
}

// what the gradients are multiplied with; NaN where the norm says that one of them is not finite, as tf does
__device__ __forceinline__ double mt_factor(double norm, double clip) {
  if (!(norm <= 3.4028234663852886e38)) return (double)NAN;      // also beyond float: the norm is reported as infinite
  return norm > clip ? clip / norm : 1.0;
}

// One read: 58M values, bf16 and float (216 MB), 38 us = 5.6 TB/s (33 where the caches hold some of it).
__global__ __launch_bounds__(256) void norm_kernel(NormArgs a, double* __restrict__ part) {
  __shared__ double red[4];
  double s = 0.0;
  const int items = a.first[a.count];
  for (int it = blockIdx.x; it < items; it += gridDim.x) {
    const int t = mt_find(a.first, a.count, it);
    const int64_t at = (int64_t)(it - a.first[t]) * MT_ITEM;
    const int64_t left = a.n[t] - at;
    s += mt_item_square_sum(a, t, at, (int)(left < MT_ITEM ? left : MT_ITEM), threadIdx.x, 256);
  }
  s = mt_block_sum(s, red);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__global__ __launch_bounds__(256) void norm_finish_kernel(const double* __restrict__ part, int n_part,
                                                          float* __restrict__ norm) {
  __shared__ double red[4];
  double s = 0.0;
  for (int i = threadIdx.x; i < n_part; i += 256) s += part[i];
  s = mt_block_sum(s, red);
  if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

// The partial sums of a list of several launches, added up once (in the order in which clip_kernel adds those of one): every
// workgroup of every launch would read all of them (1600 tensors of 40000 elements: 160 KB each, the 20 clipping launches
// 334 us, with one sum beforehand 200 + 6).
__global__ __launch_bounds__(256) void norm_join_kernel(const double* __restrict__ part, int n_part,
                                                        double* __restrict__ total) {
  __shared__ double red[4];
  double s = 0.0;
#pragma unroll 8
  for (int i = threadIdx.x; i < n_part; i += 256) s += part[i];
  s = mt_block_sum(s, red);
  if (threadIdx.x == 0) *total = s;
}

// every workgroup adds up the same partial sums (at most 8 KB from L2) instead of waiting for a launch that does.
// One read and one write: the same 58M values 68 us = 6.4 TB/s.
template <bool PAST_CACHE>
__global__ __launch_bounds__(256) void clip_kernel(ClipArgs a, const double* __restrict__ part, int n_part,
                                                   const float* __restrict__ use_norm, double clip,
                                                   float* __restrict__ norm_out) {
  __shared__ double red[4];
  double norm;
  if (use_norm) {
    norm = (double)*use_norm;
  } else {
    double s = 0.0;
    for (int i = threadIdx.x; i < n_part; i += 256) s += part[i];
    norm = sqrt(mt_block_sum(s, red));
  }
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  const float factor = (float)mt_factor(norm, clip);
  const int items = a.in.first[a.in.count];
  for (int it = blockIdx.x; it < items; it += gridDim.x) {
    const int t = mt_find(a.in.first, a.in.count, it);
    if (factor == 1.f && a.dst[t] == a.in.src[t]) continue;      // in place and nothing to change
    const int64_t at = (int64_t)(it - a.in.first[t]) * MT_ITEM;
    const int64_t left = a.in.n[t] - at;
    mt_item_scale<PAST_CACHE>(a, t, at, (int)(left < MT_ITEM ? left : MT_ITEM), factor, threadIdx.x, 256);
  }
}

// A short list: one workgroup of 16 waves, an item per wave.
__global__ __launch_bounds__(1024) void clip_small_kernel(ClipArgs a, const float* __restrict__ use_norm, double clip,
                                                          int norm_only, float* __restrict__ norm_out) {
  __shared__ double red[16];
  const int items = a.in.first[a.in.count], lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double norm;
  if (use_norm) {
    norm = (double)*use_norm;
  } else {
    double s = 0.0;
    for (int it = wave; it < items; it += 16) {
      const int t = mt_find(a.in.first, a.in.count, it);
      const int64_t at = (int64_t)(it - a.in.first[t]) * MT_SMALL_ITEM, left = a.in.n[t] - at;
      s += mt_item_square_sum(a.in, t, at, (int)(left < MT_SMALL_ITEM ? left : MT_SMALL_ITEM), lane, 64);
    }
    norm = sqrt(mt_block_sum(s, red));
  }
  if (norm_out && threadIdx.x == 0) *norm_out = (float)norm;
  if (norm_only) return;
  const float factor = (float)mt_factor(norm, clip);
  for (int it = wave; it < items; it += 16) {
    const int t = mt_find(a.in.first, a.in.count, it);
    if (factor == 1.f && a.dst[t] == a.in.src[t]) continue;
    const int64_t at = (int64_t)(it - a.in.first[t]) * MT_SMALL_ITEM, left = a.in.n[t] - at;
    mt_item_scale<false>(a, t, at, (int)(left < MT_SMALL_ITEM ? left : MT_SMALL_ITEM), factor, lane, 64);
  }
}

// ---- Adam ----
// part[item] = the item's sum of squares
__global__ __launch_bounds__(256) void adam_norm_kernel(AdamArgs a, double* __restrict__ part) {
  __shared__ double red[4];
  const int items = a.first[a.count];
  for (int it = blockIdx.x; it < items; it += gridDim.x) {
    const int t = mt_find(a.first, a.count, it);
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < MT_NORM_ITEM / MT_ITEM; ++k) {
      const int64_t at = (int64_t)(it - a.first[t]) * MT_NORM_ITEM + k * MT_ITEM, left = a.n[t] - at;
      if (left > 0) s += mt_square_sum(a.g[t] + at, (int)(left < MT_ITEM ? left : MT_ITEM), threadIdx.x, 256);
    }
    s = mt_block_sum(s, red);
    if (threadIdx.x == 0) part[it] = s;
  }
}

// per-variable factor for a sum of squares (clip <= 0: none); a NaN norm leaves the variable's gradient as it is, as
// bvi_clip_adam_step does
__device__ __forceinline__ float adam_variable_factor(double s2, float clip) {
  const double norm = sqrt(s2);
  return clip > 0.f && norm > (double)clip ? (float)((double)clip / norm) : 1.f;
}

struct AdamHyper {
  double lr, b1d, b2d;               // lr_t in double
  float b1, b2, c1, c2;              // the moments' weights; c = 1 - b taken in double: 1.f - 0.999f is 1.3e-5 off
  float eps, clip, global_clip;
};
// what the update needs of the whole list, on the device: state[0] = sum over the variables so far of the squared norm
// after their own clipping, state[1] = joint factor, state[2] = lr_t
__device__ __forceinline__ void adam_joint(double sum, const AdamHyper& h, double* __restrict__ t,
                                           double* __restrict__ state) {
  const double tt = *t + 1.0;
  *t = tt;
  state[1] = h.global_clip > 0.f ? mt_factor(sqrt(sum), (double)h.global_clip) : 1.0;
  state[2] = h.lr * sqrt(1.0 - pow(h.b2d, tt)) / (1.0 - pow(h.b1d, tt));
}

__global__ __launch_bounds__(1024) void adam_factor_kernel(AdamArgs a, AdamHyper h, const double* __restrict__ part,
                                                           int first_batch, int last_batch, float* __restrict__ factor,
                                                           double* __restrict__ state, double* __restrict__ step) {
  __shared__ double sq[MT_MAX];
  __shared__ double red[16];
  const int lane = threadIdx.x & 63;
  auto keep = [&](int t, double sum) {
    const float f = adam_variable_factor(sum, h.clip);
    factor[t] = f;
    sq[t] = (double)f * (double)f * sum;
  };
  // a wave per variable, the workgroup together for a large one
  for (int t = threadIdx.x >> 6; t < a.count; t += 16) {
    if (a.first[t + 1] - a.first[t] > 256) continue;
    double s = 0.0;
    for (int i = a.first[t] + lane; i < a.first[t + 1]; i += 64) s += part[i];
    s = mt_wave_sum(s);
    if (lane == 0) keep(t, s);
  }
  for (int t = 0; t < a.count; ++t) {
    if (a.first[t + 1] - a.first[t] <= 256) continue;
    double s = 0.0;
#pragma unroll 4
    for (int i = a.first[t] + threadIdx.x; i < a.first[t + 1]; i += 1024) s += part[i];
    s = mt_block_sum(s, red);
    if (threadIdx.x == 0) keep(t, s);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double sum = first_batch ? 0.0 : state[0];
    for (int t = 0; t < a.count; ++t) sum += sq[t];
    state[0] = sum;
    if (last_batch) adam_joint(sum, h, step, state);
  }
}

__device__ __forceinline__ void adam_element(float& x, float& g, float& m, float& v, float factor, float lr_t,
                                             const AdamHyper& h) {
  g *= factor;
  m = h.b1 * m + h.c1 * g;
  v = h.b2 * v + h.c2 * g * g;
  x -= lr_t * m / (sqrtf(v) + h.eps);
}

__device__ __forceinline__ void adam_update(float* __restrict__ x, float* __restrict__ g, float* __restrict__ m,
                                            float* __restrict__ v, int len, float factor, float lr_t,
                                            const AdamHyper& h, int id, int lanes) {
  int done = 0;
  if (((uintptr_t)x | (uintptr_t)g | (uintptr_t)m | (uintptr_t)v) % 16 == 0) {
    done = len / 4 * 4;
    for (int i = id * 4; i < done; i += lanes * 4) {
      Vec16<float> xi = *reinterpret_cast<Vec16<float>*>(x + i), gi = *reinterpret_cast<Vec16<float>*>(g + i),
                   mi = *reinterpret_cast<Vec16<float>*>(m + i), vi = *reinterpret_cast<Vec16<float>*>(v + i);
#pragma unroll
      for (int k = 0; k < 4; ++k) adam_element(xi.e[k], gi.e[k], mi.e[k], vi.e[k], factor, lr_t, h);
      if (factor != 1.f) *reinterpret_cast<Vec16<float>*>(g + i) = gi;     // the clipped gradient stays readable
      *reinterpret_cast<Vec16<float>*>(m + i) = mi;
      *reinterpret_cast<Vec16<float>*>(v + i) = vi;
      *reinterpret_cast<Vec16<float>*>(x + i) = xi;
    }
  }
  for (int i = done + id; i < len; i += lanes) {
    float xi = x[i], gi = g[i], mi = m[i], vi = v[i];
    adam_element(xi, gi, mi, vi, factor, lr_t, h);
    if (factor != 1.f) g[i] = gi;
    m[i] = mi;
    v[i] = vi;
    x[i] = xi;
  }
}

// Four arrays read, three or (where a factor is not one) four written: 29M elements 146 us for 820 MB = 5.6 TB/s, or 160 us
// for 937 MB = 5.9 TB/s.  Only bytes count; the norm pass before it is the fifth read, since every variable's norm is needed
// before its first step.
__global__ __launch_bounds__(256) void adam_update_kernel(AdamArgs a, AdamHyper h, const float* __restrict__ factor,
                                                          const double* __restrict__ state) {
  const float joint = (float)state[1], lr_t = (float)state[2];
  const int items = a.first[a.count];
  for (int it = blockIdx.x; it < items; it += gridDim.x) {
    const int t = mt_find(a.first, a.count, it);
    const int64_t at = (int64_t)(it - a.first[t]) * MT_ITEM;
    const int64_t left = a.n[t] - at;
    adam_update(a.x[t] + at, a.g[t] + at, a.m[t] + at, a.v[t] + at, (int)(left < MT_ITEM ? left : MT_ITEM),
                factor[t] * joint, lr_t, h, threadIdx.x, 256);
  }
}

// the whole step of a short list in one launch
__global__ __launch_bounds__(1024) void adam_small_kernel(AdamArgs a, AdamHyper h, double* __restrict__ step) {
  __shared__ double part[MT_SMALL], sq[MT_MAX], state[3];
  __shared__ float factor[MT_MAX];
  const int items = a.first[a.count], lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int it = wave; it < items; it += 16) {
    const int t = mt_find(a.first, a.count, it);
    const int64_t at = (int64_t)(it - a.first[t]) * MT_SMALL_ITEM, left = a.n[t] - at;
    const double s = mt_wave_sum(
        mt_square_sum(a.g[t] + at, (int)(left < MT_SMALL_ITEM ? left : MT_SMALL_ITEM), lane, 64));
    if (lane == 0) part[it] = s;
  }
  __syncthreads();
  for (int t = threadIdx.x; t < a.count; t += 1024) {
    double s = 0.0;
    for (int i = a.first[t]; i < a.first[t + 1]; ++i) s += part[i];
    const float f = adam_variable_factor(s, h.clip);
    factor[t] = f;
    sq[t] = (double)f * (double)f * s;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double sum = 0.0;
    for (int t = 0; t < a.count; ++t) sum += sq[t];
    adam_joint(sum, h, step, state);
  }
  __syncthreads();
  const float joint = (float)state[1], lr_t = (float)state[2];
  for (int it = wave; it < items; it += 16) {
    const int t = mt_find(a.first, a.count, it);
    const int64_t at = (int64_t)(it - a.first[t]) * MT_SMALL_ITEM, left = a.n[t] - at;
    adam_update(a.x[t] + at, a.g[t] + at, a.m[t] + at, a.v[t] + at, (int)(left < MT_SMALL_ITEM ? left : MT_SMALL_ITEM),
                factor[t] * joint, lr_t, h, lane, 64);
  }
}

// ---- host ----
int type_size(int dtype) { return dtype == BVI_TYPE_F32 ? 4 : dtype == BVI_TYPE_BF16 || dtype == BVI_TYPE_F16 ? 2 : 0; }

bool list_ok(int count, const int64_t* sizes) {
  if (count < 1 || !sizes) return false;
  for (int t = 0; t < count; ++t)
    if (sizes[t] < 0) return false;
  return true;
}
int64_t items_of(int64_t n, int item = MT_ITEM) { return (n + item - 1) / item; }
bool is_small(int count, const int64_t* sizes) {
  if (count > MT_MAX) return false;
  int64_t items = 0, all = 0;
  for (int t = 0; t < count && items <= MT_SMALL; ++t) {
    items += items_of(sizes[t], MT_SMALL_ITEM);
    all += sizes[t];
  }
  return items <= MT_SMALL && all <= MT_SMALL_ALL;
}
// every batch of MT_MAX tensors has fewer than 2^31 items
bool items_fit(int count, const int64_t* sizes) {
  for (int t0 = 0; t0 < count; t0 += MT_MAX) {
    int64_t items = 0;
    for (int t = t0; t < count && t < t0 + MT_MAX; ++t) {
      if (sizes[t] > (int64_t)1 << 40) return false;
      items += items_of(sizes[t]);
    }
    if (items > 0x7fffffff) return false;
  }
  return true;
}
int batches_of(int count) { return (count + MT_MAX - 1) / MT_MAX; }

void fill(NormArgs& a, int t0, int count, const void* const* src, const int64_t* sizes, const int* types,
          int item = MT_ITEM) {
  a.count = count - t0 < MT_MAX ? count - t0 : MT_MAX;
  a.first[0] = 0;
  for (int k = 0; k < a.count; ++k) {
    a.src[k] = src[t0 + k];
    a.n[k] = sizes[t0 + k];
    a.type[k] = (uint8_t)types[t0 + k];
    a.first[k + 1] = a.first[k] + (int32_t)items_of(a.n[k], item);
  }
}
unsigned blocks_for(int items, int most) { return (unsigned)(items < 1 ? 1 : items < most ? items : most); }

int check_list(int count, const void* const* src, const int64_t* sizes, const int* types) {
  if (!list_ok(count, sizes) || !src || !types) return BVI_ERR_ARG;
  for (int t = 0; t < count; ++t)
    if (!type_size(types[t]) || (!src[t] && sizes[t] > 0) || (uintptr_t)src[t] % (size_t)type_size(types[t]))
      return BVI_ERR_ARG;
  return items_fit(count, sizes) ? BVI_OK : BVI_ERR_UNSUPPORTED;
}

// whether any two of the lists' ranges share memory: the kernels write them in no particular order
bool shares_memory(int count, const int64_t* sizes, float* const* const (&lists)[4]) {
  std::vector<std::pair<uintptr_t, uintptr_t>> span;
  span.reserve((size_t)count * 4);
  for (float* const* list : lists)
    for (int t = 0; t < count; ++t)
      if (sizes[t] > 0) span.emplace_back((uintptr_t)list[t], (uintptr_t)(list[t] + sizes[t]));
  std::sort(span.begin(), span.end());
  for (size_t k = 1; k < span.size(); ++k)
    if (span[k].first < span[k - 1].second) return true;
  return false;
}

int launch_norm(int count, const void* const* src, const int64_t* sizes, const int* types, double* part, int* n_part,
                hipStream_t s) {
  *n_part = 0;
  for (int t0 = 0; t0 < count; t0 += MT_MAX) {
    NormArgs a;
    fill(a, t0, count, src, sizes, types);
    const unsigned blocks = blocks_for(a.first[a.count], MT_BLOCKS);
    hipLaunchKernelGGL(norm_kernel, dim3(blocks), dim3(256), 0, s, a, part + *n_part);
    *n_part += (int)blocks;
  }
  BVI_HIP_CHECK_LAUNCH();
  return BVI_OK;
}

}  // namespace

extern "C" {

int bvi_global_norm_ws_bytes(int n_tensors, size_t* ws_bytes) {
  if (!ws_bytes || n_tensors < 1) return BVI_ERR_ARG;
  *ws_bytes = ((size_t)batches_of(n_tensors) * MT_BLOCKS + 1) * sizeof(double);
  return BVI_OK;
}

int bvi_global_norm(int n_tensors, const void* const* tensors, const int64_t* sizes, const int* dtypes, float* norm,
                    void* ws, size_t ws_bytes, void* stream) {
  const int bad = check_list(n_tensors, tensors, sizes, dtypes);
  if (bad || !norm) return bad ? bad : BVI_ERR_ARG;
  size_t need;
  bvi_global_norm_ws_bytes(n_tensors, &need);
  if (!ws || ws_bytes < need) return BVI_ERR_WORKSPACE;
  if ((uintptr_t)ws % sizeof(double)) return BVI_ERR_ARG;
  if (is_small(n_tensors, sizes)) {
    ClipArgs a;
    fill(a.in, 0, n_tensors, tensors, sizes, dtypes, MT_SMALL_ITEM);
    hipLaunchKernelGGL(clip_small_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, a, (const float*)nullptr, 1.0,
                       1, norm);
    BVI_HIP_CHECK_LAUNCH();
    return BVI_OK;
  }
  int n_part;
  const int st = launch_norm(n_tensors, tensors, sizes, dtypes, (double*)ws, &n_part, (hipStream_t)stream);
  if (st) return st;
  hipLaunchKernelGGL(norm_finish_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream, (const double*)ws, n_part, norm);
  BVI_HIP_CHECK_LAUNCH();
  return BVI_OK;
}

int bvi_clip_by_global_norm(int n_tensors, const void* const* tensors, void* const* outputs, const int64_t* sizes,
                            const int* dtypes, float clip_norm, const float* use_norm, float* norm, void* ws,
                            size_t ws_bytes, void* stream) {
  const int bad = check_list(n_tensors, tensors, sizes, dtypes);
  if (bad) return bad;
  if (!outputs || !(clip_norm > 0.f)) return BVI_ERR_ARG;
  for (int t = 0; t < n_tensors; ++t)
    if ((!outputs[t] && sizes[t] > 0) || (uintptr_t)outputs[t] % (size_t)type_size(dtypes[t])) return BVI_ERR_ARG;
  size_t need;
  bvi_global_norm_ws_bytes(n_tensors, &need);
  if (!use_norm && (!ws || ws_bytes < need)) return BVI_ERR_WORKSPACE;
  if ((uintptr_t)ws % sizeof(double)) return BVI_ERR_ARG;
  const hipStream_t s = (hipStream_t)stream;
  if (is_small(n_tensors, sizes)) {
    ClipArgs a;
    fill(a.in, 0, n_tensors, tensors, sizes, dtypes, MT_SMALL_ITEM);
    for (int k = 0; k < n_tensors; ++k) a.dst[k] = outputs[k];
    hipLaunchKernelGGL(clip_small_kernel, dim3(1), dim3(1024), 0, s, a, use_norm, (double)clip_norm,
                       0, norm);
    BVI_HIP_CHECK_LAUNCH();
    return BVI_OK;
  }
  int n_part = 0;
  if (!use_norm) {
    const int st = launch_norm(n_tensors, tensors, sizes, dtypes, (double*)ws, &n_part, s);
    if (st) return st;
  }
  const double* part = (const double*)ws;
  if (n_part > MT_BLOCKS) {
    double* total = (double*)((char*)ws + need) - 1;
    hipLaunchKernelGGL(norm_join_kernel, dim3(1), dim3(256), 0, s, part, n_part, total);
    part = total;
    n_part = 1;
  }
  // results beyond the 32 MB of L2 go past the caches: 58M values 70 -> 66 us here, and 42 -> 33 us in the next norm pass
  // over the same gradients
  int64_t bytes = 0;
  for (int t = 0; t < n_tensors; ++t) bytes += sizes[t] * type_size(dtypes[t]);
  const bool past_cache = bytes > (32 << 20);
  for (int t0 = 0; t0 < n_tensors; t0 += MT_MAX) {
    ClipArgs a;
    fill(a.in, t0, n_tensors, tensors, sizes, dtypes);
    for (int k = 0; k < a.in.count; ++k) a.dst[k] = outputs[t0 + k];
    const dim3 grid(blocks_for(a.in.first[a.in.count], 2 * MT_BLOCKS));
    float* norm_out = t0 == 0 ? norm : nullptr;
    if (past_cache)
      hipLaunchKernelGGL(clip_kernel<true>, grid, dim3(256), 0, s, a, part, n_part, use_norm,
                         (double)clip_norm, norm_out);
    else
      hipLaunchKernelGGL(clip_kernel<false>, grid, dim3(256), 0, s, a, part, n_part, use_norm,
                         (double)clip_norm, norm_out);
  }
  BVI_HIP_CHECK_LAUNCH();
  return BVI_OK;
}

int bvi_adam_step_ws_bytes(int n_tensors, const int64_t* sizes, size_t* ws_bytes) {
  if (!ws_bytes || !list_ok(n_tensors, sizes)) return BVI_ERR_ARG;
  if (!items_fit(n_tensors, sizes)) return BVI_ERR_UNSUPPORTED;
  int64_t most = 0;                                    // the partial sums are used batch by batch
  for (int t0 = 0; t0 < n_tensors; t0 += MT_MAX) {
    int64_t items = 0;
    for (int t = t0; t < n_tensors && t < t0 + MT_MAX; ++t) items += items_of(sizes[t], MT_NORM_ITEM);
    most = items > most ? items : most;
  }
  *ws_bytes = (size_t)(4 + most) * sizeof(double) + (size_t)n_tensors * sizeof(float);
  return BVI_OK;
}

int bvi_adam_step(int n_tensors, float* const* x, float* const* grad, float* const* m, float* const* v,
                  const int64_t* sizes, double* step_count, double learning_rate, double beta_1, double beta_2,
                  double epsilon, float clip_norm, float global_clip_norm, void* ws, size_t ws_bytes, void* stream) {
  if (!list_ok(n_tensors, sizes) || !x || !grad || !m || !v || !step_count) return BVI_ERR_ARG;
  for (int t = 0; t < n_tensors; ++t)
    if ((sizes[t] > 0 && (!x[t] || !grad[t] || !m[t] || !v[t])) ||
        ((uintptr_t)x[t] | (uintptr_t)grad[t] | (uintptr_t)m[t] | (uintptr_t)v[t]) % sizeof(float))
      return BVI_ERR_ARG;
  if ((uintptr_t)ws % sizeof(double) || (uintptr_t)step_count % sizeof(double)) return BVI_ERR_ARG;
  size_t need;
  const int st = bvi_adam_step_ws_bytes(n_tensors, sizes, &need);
  if (st) return st;
  if (!ws || ws_bytes < need) return BVI_ERR_WORKSPACE;
  try {
    if (shares_memory(n_tensors, sizes, {x, grad, m, v})) return BVI_ERR_ARG;
  } catch (const std::bad_alloc&) {
    return BVI_ERR_WORKSPACE;
  }
  const hipStream_t s = (hipStream_t)stream;
  double* state = (double*)ws;
  float* factor = (float*)((char*)ws + need) - n_tensors;
  double* part = state + 4;
  const AdamHyper h{learning_rate, beta_1, beta_2, (float)beta_1, (float)beta_2, (float)(1.0 - beta_1),
                    (float)(1.0 - beta_2), (float)epsilon, clip_norm, global_clip_norm};
  const bool small = is_small(n_tensors, sizes);
  for (int pass = small ? 1 : 0; pass < 2; ++pass)
    for (int t0 = 0; t0 < n_tensors; t0 += MT_MAX) {
      AdamArgs a;
      a.count = n_tensors - t0 < MT_MAX ? n_tensors - t0 : MT_MAX;
      a.first[0] = 0;
      for (int k = 0; k < a.count; ++k) {
        a.x[k] = x[t0 + k];
        a.g[k] = grad[t0 + k];
        a.m[k] = m[t0 + k];
        a.v[k] = v[t0 + k];
        a.n[k] = sizes[t0 + k];
        a.first[k + 1] = a.first[k] + (int32_t)items_of(a.n[k], small ? MT_SMALL_ITEM : pass == 0 ? MT_NORM_ITEM : MT_ITEM);
      }
      if (small) {
        hipLaunchKernelGGL(adam_small_kernel, dim3(1), dim3(1024), 0, s, a, h, step_count);
        break;
      }
      const int items = a.first[a.count];
      if (pass == 0) {
        hipLaunchKernelGGL(adam_norm_kernel, dim3(blocks_for(items, 4 * MT_BLOCKS)), dim3(256), 0, s, a, part);
        hipLaunchKernelGGL(adam_factor_kernel, dim3(1), dim3(1024), 0, s, a, h, (const double*)part, t0 == 0,
                           t0 + MT_MAX >= n_tensors, factor + t0, state, step_count);
      } else {
        hipLaunchKernelGGL(adam_update_kernel, dim3(blocks_for(items, 4 * MT_BLOCKS)), dim3(256), 0, s, a, h,
                           (const float*)(factor + t0), (const double*)state);
      }
    }
  BVI_HIP_CHECK_LAUNCH();
  return BVI_OK;
}

}  // extern "C"
