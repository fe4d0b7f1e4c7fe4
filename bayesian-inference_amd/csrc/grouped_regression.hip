// Gaussian linear regression with group-level effects, for all chains at once:
//   eta_ci = b_c + sum_j w_cj x_ij + sum_l z_il u_l,c[group_l(i)],   y_i ~ Normal(eta_ci, s_c)
//   logp_c      = -n log s - n/2 log(2 pi) - sum_i e_ci^2 / (2 s^2),   e = y - eta
//   d b = sum_i e / s^2;  d w_j = sum_i e x_ij / s^2;  d s = -n / s + sum_i e^2 / s^3
//   d u_l[v]    = sum over {i : group_l(i) = v} of z_il e / s^2        (the gradient of a table lookup by sorted ids)
// theta_c = (b, w[d], s, u_1[rows_1], u_2[rows_2], ...).  z_l may be absent (ones: a varying intercept) or a column
// (a varying slope).  A row whose group is outside [0, rows_l) has no effect of lookup l.
//
// The dataset is fixed, so its rows are laid out once per lookup in that lookup's sorted order (`packed`).  A pass over
// the l-th copy walks the rows in that order, a wave per stretch of `span` rows, and ends a running sum wherever the
// group changes: each group's sum is complete within a wave or split over neighbouring ones.  Walking along the rows,
// every new stretch raises (group + wave), so that sum is a slot number of its own without any list, and group v's
// slots are v + first wave .. v + last wave.  The lookups of the other tables are gathers in the same pass; nothing of
// size rows x chains is ever written.  A second launch adds up the slots and the dense sums in a fixed order.
#include "bvi_common.h"

#include <math.h>

namespace {

constexpr int GR_WAVES = 4;             // waves per workgroup
constexpr int GR_PAD = 32;              // rows behind the last one that may be read (and are not used)
constexpr int GR_MAX_WAVES = 4096;      // stretches per pass: 16 waves per CU, or more of them:
constexpr int GR_MAX_SPAN = 2048;       // rows of a stretch, beyond 8.4M rows; a float holds the sums that a wave writes
                                        // (a group's, a feature's) to 2^-24 of so many terms, however many rows there are

struct GrPass {                         // one lookup's copy of the rows
  const float* y;
  const float* X;                       // [n, D], columns beyond d are zero
  const int32_t* id[BVI_MAX_LOOKUPS];   // group of every lookup in this order; id[own] ascends
  const float* z[BVI_MAX_LOOKUPS];      // or NULL
  const int32_t* start;                 // of the own lookup
  int64_t rows[BVI_MAX_LOOKUPS];
  const float* tab[BVI_MAX_LOOKUPS];    // u_l of group g and chain c: tab[l][g group_stride + c chain_stride], in theta or
  int64_t group_stride, chain_stride;   // in its transposed copy
  float* slots;                         // of the own lookup
  int own, lookups;
};
struct GrPasses {
  GrPass pass[BVI_MAX_LOOKUPS];
};

// the workgroup's dense sums: [0] e^2, [1] e, [2 + j] e x_j; eight at a time through LDS
template <int CP, int D, bool GRAD, int DD>
__device__ __forceinline__ void grouped_dense(double sum_sq, double sum_e, const float (&gw)[DD], int d, int C,
                                              int chain0, double* __restrict__ dense) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, cl = lane % CP, q = lane / CP;
  constexpr int COUNT = GRAD ? 2 + D : 1;
  const int count = GRAD ? 2 + d : 1;
  __shared__ double red[GR_WAVES][8][CP];
#pragma unroll
  for (int k0 = 0; k0 < COUNT; k0 += 8) {
    __syncthreads();
#pragma unroll
    for (int k = k0; k < k0 + 8 && k < COUNT; ++k) {
      double v = k == 0 ? sum_sq : k == 1 ? sum_e : (double)gw[k >= 2 ? k - 2 : 0];
#pragma unroll
      for (int off = CP; off < 64; off <<= 1) v += __shfl_xor(v, off, 64);
      if (q == 0) red[wave][k - k0][cl] = v;
    }
    __syncthreads();
    for (int t = threadIdx.x; t < 8 * CP; t += 64 * GR_WAVES) {
      const int k = k0 + t / CP, ch = chain0 + t % CP;
      if (k < count && ch < C) {
        double v = 0.0;
#pragma unroll
        for (int x = 0; x < GR_WAVES; ++x) v += red[x][t / CP][t % CP];
        dense[((int64_t)blockIdx.x * count + k) * C + ch] = v;
      }
    }
  }
}

// Up to 16 chains: CP chains x Q = 64 / CP rows per wave, every lane its own row with its own group's effect, so that
// groups of a few rows keep all lanes busy.  Rows are sorted by group: Q rows of one group are added lane by lane; where
// they are of several, log2 Q shuffles leave each one's sum in its first lane (300k rows of one chain in 100k groups 10 us
// of 5 MB; a wave that took the groups one by one 32).  300001 rows, 3 features, 4 chains, two lookups: 24 us, shuffles and
// gathers, not bytes.  blockIdx.z: the lookup whose pass this is; the first also takes the sums that need every row once.
template <int CP, int D, bool GRAD>
__global__ __launch_bounds__(64 * GR_WAVES) void grouped_kernel(GrPasses passes, int64_t n, int d, int64_t span, int C,
                                                                int64_t P, const float* __restrict__ theta,
                                                                double* __restrict__ dense) {
  const GrPass& a = passes.pass[blockIdx.z];
  const bool FIRST = blockIdx.z == 0;
  const float* __restrict__ y = a.y;
  const float* __restrict__ X = a.X;
  const int32_t* __restrict__ key = a.id[a.own];
  const float* __restrict__ zown = a.z[a.own];
  float* __restrict__ slots = a.slots;
  constexpr int Q = 64 / CP;
  constexpr int DD = D ? D : 1;
  constexpr int U = D <= 16 ? 4 : 1;                       // rows per lane in flight
  constexpr int NONE = -2147483647 - 1;
  const int lane = threadIdx.x & 63, cl = lane % CP, q = lane / CP;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int chain = blockIdx.y * CP + cl;
  const bool live = chain < C;
  const int c = live ? chain : C - 1;
  const float* th = theta + (int64_t)c * P;
  const float b = th[0];
  float w[DD], gw[DD];
#pragma unroll
  for (int j = 0; j < DD; ++j) {
    w[j] = j < d ? th[1 + j] : 0.f;
    gw[j] = 0.f;
  }
  double sum_e = 0.0, sum_sq = 0.0;
  const int own = a.own, rows = (int)a.rows[own];
  const int64_t wid = (int64_t)blockIdx.x * GR_WAVES + wave;
  const int64_t begin = wid * span, end = begin + span < n ? begin + span : n;
  int run_key = NONE;                                      // the group whose sum is not over yet, and every lane's part
  float run = 0.f;
  int kept_key = NONE;
  float kept = 0.f;
  auto total = [&](float v) {
#pragma unroll
    for (int off = CP; off < 64; off <<= 1) v += __shfl_xor(v, off, 64);
    return v;
  };
  auto put = [&](int g, float v) {
    if (g >= 0 && g < rows && live) slots[(g + wid) * C + c] = v;
  };
  for (int64_t i0 = begin; i0 < end; i0 += U * Q) {
    float e[U], zo[U], u[U];
    int k[U];
    float se = 0.f, sq = 0.f;
    auto at = [&](int t) { return i0 + t * Q + q < end ? i0 + t * Q + q : end - 1; };
    auto effect = [&](int g) {
      if (g < 0 || g >= rows) g = 0;                       // not used
      return a.tab[own][g * a.group_stride + c * a.chain_stride];
    };
    float x[U][DD], yt[U];                                 // every row's loads leave before the first is waited for
#pragma unroll
    for (int t = 0; t < U; ++t) {
      const int64_t i = at(t);
      k[t] = key[i];
      yt[t] = y[i];
      zo[t] = zown ? zown[i] : 1.f;
#pragma unroll
      for (int j = 0; j < D; ++j) x[t][j] = X[i * D + j];
    }
    // one entry per chain while a group lasts: a gather for every row touches a line per lane
    if (__builtin_amdgcn_readfirstlane(k[0]) == __builtin_amdgcn_readlane(k[U - 1], 63)) {
      if (k[0] != kept_key) kept = effect(k[0]);
      kept_key = k[0];
#pragma unroll
      for (int t = 0; t < U; ++t) u[t] = kept;
    } else {
#pragma unroll
      for (int t = 0; t < U; ++t) u[t] = effect(k[t]);
    }
#pragma unroll
    for (int t = 0; t < U; ++t) {
      const bool in = i0 + t * Q + q < end;
      const int64_t i = at(t);
      float r = yt[t] - b;
      r = k[t] >= 0 && k[t] < rows ? fmaf(-u[t], zo[t], r) : r;
      for (int l = 0; l < a.lookups; ++l) {
        if (l == own) continue;
        const int64_t m = a.id[l][i];
        if (m >= 0 && m < a.rows[l])
          r -= a.tab[l][m * a.group_stride + c * a.chain_stride] * (a.z[l] ? a.z[l][i] : 1.f);
      }
#pragma unroll
      for (int j = 0; j < D; ++j) r = fmaf(-w[j], x[t][j], r);
      r = in ? r : 0.f;
      k[t] = in ? k[t] : NONE;
      e[t] = r;
      if (FIRST) sq = fmaf(r, r, sq);
      if (FIRST && GRAD) {
        se += r;
#pragma unroll
        for (int j = 0; j < D; ++j) gw[j] = fmaf(r, x[t][j], gw[j]);
      }
    }
    if (FIRST) {
      sum_sq += (double)sq;
      sum_e += (double)se;
    }
    if (GRAD) {
#pragma unroll
      for (int t = 0; t < U; ++t) {
        float v = e[t] * zo[t];
        const int first = __builtin_amdgcn_readfirstlane(k[t]), last = __builtin_amdgcn_readlane(k[t], 63);
        if (first == last) {                               // all of one group: no shuffles while it lasts
          if (first == run_key) {
            run += v;
          } else {
            run = total(run);
            if (q == 0) put(run_key, run);
            run_key = first;
            run = v;
          }
          continue;
        }
        const float carry = total(run);
#pragma unroll
        for (int off = 1; off < Q; off <<= 1) {            // the sum from here to the group's end within these rows
          const float more = __shfl_down(v, off * CP, 64);
          const int there = __shfl_down(k[t], off * CP, 64);
          v += q + off < Q && there == k[t] ? more : 0.f;
        }
        const int left = __shfl_up(k[t], CP, 64);
        const bool head = q == 0 || left != k[t];
        if (q == 0) {
          if (first == run_key) v += carry;
          else put(run_key, carry);
        }
        if (head && k[t] != last) put(k[t], v);
        // the last group goes on: its first lane here keeps its sum
        run = head && k[t] == last ? v : 0.f;
        run_key = last;
      }
    }
  }
  if (GRAD) {
    run = total(run);
    if (q == 0) put(run_key, run);
  }
  if (FIRST) grouped_dense<CP, D, GRAD>(sum_sq, sum_e, gw, d, C, blockIdx.y * CP, dense);
}

// 64 chains per wave: 32 lanes of two chains each times two rows.  A wave keeps 32 rows in LDS (its own part: no
// barriers) and has the next ones on their way in registers, long enough to hide their latency; a row's features are then
// read by broadcast, once for two chains.  What remains is 2 D + 3 vector instructions per row and chain, 35 us of the 54
// that 1M rows, D = 8, 64 chains take.  Read straight from memory through scalar loads, rows cost 81 us there; with the
// next block of scalars on its way too many registers (93 us).  OTHERS: tables beside the own one (2: any number beyond
// one).  Beyond 16 features a lane has registers for one chain, and the tile is 16 rows.
template <int D, bool GRAD, bool FIRST, int OTHERS>
__global__ __launch_bounds__(64 * GR_WAVES) void grouped_wide_kernel(
    GrPass a, const float* __restrict__ y, const float* __restrict__ X, const int32_t* __restrict__ key,
    const float* __restrict__ zown, const int32_t* __restrict__ start, int64_t n, int d, int64_t span, int C, int64_t P,
    const float* __restrict__ theta, float* __restrict__ slots, double* __restrict__ dense) {
  constexpr int K = D <= 16 ? 2 : 1, CL = 64 / K, DD = D ? D : 1;
  constexpr int GR_TILE = D <= 16 ? 32 : 16;
  constexpr int XV = D ? (GR_TILE * D + 255) / 256 : 1;           // 16-byte loads per lane and tile
  constexpr int IDS = OTHERS ? BVI_MAX_LOOKUPS : 1;
  __shared__ f32x4 lds_x[GR_WAVES][D ? GR_TILE * D / 4 + 1 : 1];
  __shared__ float lds_y[GR_WAVES][GR_TILE], lds_z[GR_WAVES][GR_TILE];
  __shared__ int lds_id[GR_WAVES][IDS][GR_TILE];
  const int lane = threadIdx.x & 63, cl = lane % CL, q = lane / CL;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int c[K];
  bool live[K];
  float b[K], w[K][DD], gw[K][DD];
  double sum_e[K] = {}, sum_sq[K] = {};
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int chain = blockIdx.y * 64 + k * CL + cl;
    live[k] = chain < C;
    c[k] = live[k] ? chain : C - 1;
    const float* th = theta + (int64_t)c[k] * P;
    b[k] = th[0];
#pragma unroll
    for (int j = 0; j < DD; ++j) {
      w[k][j] = j < d ? th[1 + j] : 0.f;
      gw[k][j] = 0.f;
    }
  }
  const int own = a.own, rows = (int)a.rows[own];
  const int64_t wid = (int64_t)blockIdx.x * GR_WAVES + wave;
  const int64_t begin = wid * span, end = begin + span < n ? begin + span : n;
  if (begin < end) {
    // group g's end and the own table's entries, and those of group g + 1 (end -1: there is none); rows without a group
    // come last, as one group whose number is `rows`
    int g;
    int64_t e0, next_end;
    float u[K], next_u[K], run[K] = {};               // run: of group g, without this tile's part in se or su
    float se[K] = {}, sq[K] = {}, su[K] = {};         // this tile's, at most GR_TILE / K rows in a lane
    auto effect = [&](int v, float (&to)[K]) {
#pragma unroll
      for (int k = 0; k < K; ++k)
        to[k] = a.tab[own][v * a.group_stride + c[k] * a.chain_stride];
    };
    auto look_ahead = [&]() {
      next_end = g + 1 < rows ? (int64_t)start[g + 2] : -1;
      if (g + 1 < rows) effect(g + 1, next_u);
    };
    auto look_up = [&](int64_t i) {
      g = __builtin_amdgcn_readfirstlane(key[i]);
      const bool inside = g >= 0 && g < rows;
      g = inside ? g : rows;
      e0 = inside ? (int64_t)start[g + 1] : end;
#pragma unroll
      for (int k = 0; k < K; ++k) u[k] = 0.f;
      if (inside) effect(g, u);
      look_ahead();
    };
    // a tile's rows, one part per lane
    f32x4 px[XV];
    float py, pz = 1.f;
    int pid[IDS];
    auto fetch = [&](int64_t i) {
      if (D > 0) {
#pragma unroll
        for (int v = 0; v < XV; ++v)
          if ((v * 64 + lane) * 4 < GR_TILE * D) px[v] = *reinterpret_cast<const f32x4*>(X + i * D + (v * 64 + lane) * 4);
      }
      if (lane < GR_TILE) {
        py = y[i + lane];
        if (zown) pz = zown[i + lane];
        if (OTHERS)
#pragma unroll
          for (int l = 0; l < IDS; ++l)
            if (l < a.lookups) pid[l] = a.id[l][i + lane];
      }
    };
    auto keep = [&]() {
      __builtin_amdgcn_wave_barrier();
      if (D > 0) {
#pragma unroll
        for (int v = 0; v < XV; ++v)
          if ((v * 64 + lane) * 4 < GR_TILE * D) lds_x[wave][v * 64 + lane] = px[v];
      }
      if (lane < GR_TILE) {
        lds_y[wave][lane] = py;
        lds_z[wave][lane] = pz;
        if (OTHERS)
#pragma unroll
          for (int l = 0; l < IDS; ++l)
            if (l < a.lookups) lds_id[wave][l][lane] = pid[l];
      }
      __builtin_amdgcn_wave_barrier();
    };
    // what leaves a tile is added up in double: log-densities of 10^7 and more rows are compared across chains to 0.01.  A
    // float that ran on as long as a group lasts lost 23 to 28 nats of 1.3e7 at 9M rows in two groups whose values lie on a
    // grid of 2^-8 (ties always rounded the same way).  Cost: within 1 % (1M rows, D = 8, 64 chains 63 us before and after)
    auto settle = [&]() {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (FIRST) {
          sum_sq[k] += (double)sq[k];
          sum_e[k] += (double)se[k];
          sq[k] = 0.f;
        }
        if (GRAD) {
          run[k] += zown ? su[k] : se[k];
          se[k] = su[k] = 0.f;
        }
      }
    };
    auto close = [&]() {                              // the running sums of group g end here
      settle();
      if (!GRAD) return;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float v = run[k];
        if (K == 2) v += __shfl_xor(v, 32, 64);
        if (g < rows && live[k] && q == 0) slots[(g + wid) * C + c[k]] = v;
        run[k] = 0.f;
      }
    };
    const float* tx = reinterpret_cast<const float*>(lds_x[wave]);
    fetch(begin);
    look_up(begin);
    for (int64_t i0 = begin; i0 < end; i0 += GR_TILE) {
      keep();
      if (i0 + GR_TILE < end) fetch(i0 + GR_TILE);
      const int count = (int)(end - i0 < GR_TILE ? end - i0 : GR_TILE);
      int p = 0;
      while (true) {
        const int64_t left = e0 - i0;
        const int to = left < count ? (int)left : count;
#pragma unroll 2
        for (; p < to; p += K) {
          const bool in = p + q < to;
          const int r = in ? p + q : p;
          const float yr = lds_y[wave][r];
          const float zr = zown ? lds_z[wave][r] : 1.f;
          float x[DD];
          if (D >= 4) {
#pragma unroll
            for (int j = 0; j < D; j += 4) {
              const f32x4 t = lds_x[wave][(r * D + j) / 4];
#pragma unroll
              for (int m = 0; m < 4; ++m) x[j + m < DD ? j + m : 0] = t[m];
            }
          } else {
#pragma unroll
            for (int j = 0; j < D; ++j) x[j] = tx[r * D + j];
          }
          float e[K];
#pragma unroll
          for (int k = 0; k < K; ++k) {
            e[k] = yr - b[k];
            e[k] = zown ? fmaf(-u[k], zr, e[k]) : e[k] - u[k];
          }
          if (OTHERS) {
#pragma unroll
            for (int l = 0; l < (OTHERS == 1 ? 2 : IDS); ++l) {
              if (l == own || l >= a.lookups) continue;
              const int m = lds_id[wave][l][r];
              const bool has = m >= 0 && m < (int)a.rows[l];
              const float zl = a.z[l] ? a.z[l][i0 + r] : 1.f;
#pragma unroll
              for (int k = 0; k < K; ++k) {
                const float t = a.tab[l][(has ? m : 0) * a.group_stride + c[k] * a.chain_stride];
                e[k] = has ? fmaf(-t, zl, e[k]) : e[k];
              }
            }
          }
#pragma unroll
          for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int j = 0; j < D; ++j) e[k] = fmaf(-w[k][j], x[j], e[k]);
            e[k] = in ? e[k] : 0.f;
            if (FIRST) sq[k] = fmaf(e[k], e[k], sq[k]);
            if (GRAD) se[k] += e[k];
            if (GRAD && zown) su[k] = fmaf(e[k], zr, su[k]);
            if (FIRST && GRAD) {
#pragma unroll
              for (int j = 0; j < D; ++j) gw[k][j] = fmaf(e[k], x[j], gw[k][j]);
            }
          }
        }
        p = to;
        if (p == count) break;
        close();
        if (next_end > e0) {                          // group g + 1 has rows, as most have
          ++g;
          e0 = next_end;
#pragma unroll
          for (int k = 0; k < K; ++k) u[k] = next_u[k];
          look_ahead();
        } else {
          look_up(i0 + p);
        }
      }
      if (e0 == i0 + count && e0 < end) {             // a group that ends with the tile
        close();
        look_up(e0);
      } else {
        settle();
      }
    }
    close();
  }
  if (FIRST)
#pragma unroll
    for (int k = 0; k < K; ++k) grouped_dense<CL, D, GRAD>(sum_sq[k], sum_e[k], gw[k], d, C, blockIdx.y * 64 + k * CL, dense);
}

// theta's tables [C, rows] -> [rows, C], 64 x 64 through LDS
__global__ __launch_bounds__(256) void grouped_transpose_kernel(const float* __restrict__ theta, int64_t P, int64_t first,
                                                                int64_t rows, int C, float* __restrict__ tables) {
  __shared__ float tile[64][65];
  const int64_t r0 = (int64_t)blockIdx.x * 64;
  const int c0 = blockIdx.y * 64, lane = threadIdx.x & 63;
  for (int k = threadIdx.x >> 6; k < 64; k += 4)
    if (c0 + k < C && r0 + lane < rows) tile[k][lane] = theta[(int64_t)(c0 + k) * P + first + r0 + lane];
  __syncthreads();
  for (int k = threadIdx.x >> 6; k < 64; k += 4)
    if (r0 + k < rows && c0 + lane < C) tables[(r0 + k) * C + c0 + lane] = tile[lane][k];
}

struct GrFinish {
  const int32_t* start[BVI_MAX_LOOKUPS];
  const float* slots[BVI_MAX_LOOKUPS];
  int64_t rows[BVI_MAX_LOOKUPS];
  int64_t offset[BVI_MAX_LOOKUPS];
  int64_t tile_end[BVI_MAX_LOOKUPS];    // workgroups of the lookups up to this one, behind the dense ones
  int lookups;
};

// Workgroup x < count: dense sum x.  Others: 1024 / CP groups of a table.  A thread adds up a group's slots for one chain
// where they are few, a wave where they are not, the workgroup together where the wave's lanes would be too few.
constexpr int GR_MANY = 16, GR_VERY_MANY = 512;
template <int CP>
__global__ __launch_bounds__(1024) void grouped_finish_kernel(GrFinish f, int64_t n, int d, int count, int64_t span,
                                                              int n_blocks, int C, int64_t P,
                                                              const float* __restrict__ theta,
                                                              const double* __restrict__ dense,
                                                              const double* __restrict__ logp_ref,
                                                              float* __restrict__ logp, float* __restrict__ grad) {
  constexpr int GT = 1024 / CP, Q = 64 / CP;
  __shared__ double red[1024], val[1024];
  const int cl = threadIdx.x % CP, q = threadIdx.x / CP;
  const int chain = blockIdx.y * CP + cl;
  const int c = chain < C ? chain : C - 1;
  const double s = (double)theta[(int64_t)c * P + 1 + d];
  // entries first, first + step, ... below `past` of one chain's column; eight loads in flight
  auto column = [&](auto* __restrict__ p, int64_t first, int64_t past, int step, int64_t stride) {
    double v = 0.0;
    for (int64_t k = first; k < past; k += 8 * step) {
      double x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int64_t at = k + u * step;
        x[u] = (double)p[(at < past ? at : k) * stride];
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) v += k + u * step < past ? x[u] : 0.0;
    }
    return v;
  };
  auto block_total = [&](double v) {                             // over q, for every cl
    red[threadIdx.x] = v;
    __syncthreads();
    for (int h = GT / 2; h >= 1; h >>= 1) {
      if (q < h) red[threadIdx.x] += red[threadIdx.x + h * CP];
      __syncthreads();
    }
    v = red[cl];
    __syncthreads();
    return v;
  };
  if ((int)blockIdx.x < count) {
    const int k = blockIdx.x;
    const double v = block_total(column(dense + (int64_t)k * C + c, q, n_blocks, GT, (int64_t)count * C));
    if (q == 0 && chain < C) {
      if (k == 0) {
        const double level = logp_ref ? *logp_ref : 0.0;
        logp[c] = (float)(-(double)n * log(s) - 0.5 * (double)n * BVI_LN2PI_D - 0.5 * v / (s * s) - level);
        if (grad) grad[(int64_t)c * P + 1 + d] = (float)(v / (s * s * s) - (double)n / s);
      } else {
        grad[(int64_t)c * P + (k == 1 ? 0 : k - 1)] = (float)(v / (s * s));
      }
    }
    return;
  }
  const int64_t tile = blockIdx.x - count;
  int l = 0;
  while (l + 1 < f.lookups && tile >= f.tile_end[l]) ++l;
  const int64_t g0 = (tile - (l ? f.tile_end[l - 1] : 0)) * GT, rows = f.rows[l];
  const float* slots = f.slots[l];
  const int32_t* start = f.start[l];
  // slots [first, past) of the tile's group k
  auto slots_of = [&](int k, int64_t* first, int64_t* past) {
    *first = *past = 0;
    if (g0 + k >= rows) return;
    const int64_t b = start[g0 + k], e = start[g0 + k + 1];
    if (e > b) {
      *first = g0 + k + b / span;
      *past = g0 + k + (e - 1) / span + 1;
    }
  };
  __shared__ int some[GT], very[GT], n_some, n_very;             // groups left to the waves, to the workgroup
  if (threadIdx.x == 0) n_some = n_very = 0;
  __syncthreads();
  int64_t first, past;
  slots_of(q, &first, &past);
  if (past - first <= GR_MANY) {
    val[threadIdx.x] = column(slots + c, first, past, 1, C);
  } else if (cl == 0) {
    // the order of the lists only says who does which group
    if (past - first <= GR_VERY_MANY) some[atomicAdd(&n_some, 1)] = q;
    else very[atomicAdd(&n_very, 1)] = q;
  }
  __syncthreads();
  const int lane = threadIdx.x & 63, wq = lane / CP;             // cl is also the lane's chain: CP divides 64
  for (int x = threadIdx.x >> 6; x < n_some; x += 16) {
    slots_of(some[x], &first, &past);
    double v = column(slots + c, first + wq, past, Q, C);
#pragma unroll
    for (int off = CP; off < 64; off <<= 1) v += __shfl_xor(v, off, 64);
    if (wq == 0) val[some[x] * CP + cl] = v;
  }
  const int waiting = n_very;
  for (int x = 0; x < waiting; ++x) {
    slots_of(very[x], &first, &past);
    const double v = block_total(column(slots + c, first + q, past, GT, C));
    if (q == 0) val[very[x] * CP + cl] = v;
  }
  __syncthreads();
  // neighbouring threads write neighbouring groups of one chain
  float* out = reinterpret_cast<float*>(red);
  out[threadIdx.x] = (float)(val[threadIdx.x] / (s * s));
  __syncthreads();
  const int wc = threadIdx.x / GT, wg = threadIdx.x % GT;
  if (blockIdx.y * CP + wc < (unsigned)C && g0 + wg < rows)
    grad[(int64_t)(blockIdx.y * CP + wc) * P + f.offset[l] + g0 + wg] = out[wg * CP + wc];
}

// ---- packing: copy l of the rows, in the order of its plan ----
__global__ __launch_bounds__(256) void grouped_pack_kernel(const float* __restrict__ X, const float* __restrict__ y,
                                                           int64_t n, int d, int D, const int32_t* __restrict__ order,
                                                           float* __restrict__ Xo, float* __restrict__ yo) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int64_t k = order[i];
  yo[i] = y[k];
  for (int j = 0; j < D; ++j) Xo[i * D + j] = j < d ? X[k * d + j] : 0.f;
}
__global__ __launch_bounds__(256) void grouped_pack_column_kernel(const int32_t* __restrict__ id,
                                                                  const float* __restrict__ z, int64_t rows, int64_t n,
                                                                  const int32_t* __restrict__ order,
                                                                  int32_t* __restrict__ ido, float* __restrict__ zo) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int64_t k = order[i];
  const int32_t g = id[k];
  ido[i] = g;
  if (zo) zo[i] = g >= 0 && g < rows ? z[k] : 0.f;       // what stands beside no group is not a number to multiply with
}
__global__ __launch_bounds__(256) void grouped_pack_start_kernel(const int32_t* __restrict__ start, int64_t m,
                                                                 int32_t* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i < m) out[i] = start[i];
}

// ---- host ----
int64_t words(int64_t n) { return (n + 63) / 64 * 64; }
int padded_d(int d) { return d == 0 ? 0 : d <= 1 ? 1 : d <= 2 ? 2 : d <= 4 ? 4 : d <= 8 ? 8 : d <= 16 ? 16 : d <= 32 ? 32 : 64; }

bool shape_ok(int64_t n, int d, int lookups, const int64_t* rows) {
  if (n < 0 || d < 0 || lookups < 1 || !rows) return false;
  for (int l = 0; l < lookups && l < BVI_MAX_LOOKUPS; ++l)
    if (rows[l] < 1) return false;
  return true;
}
bool shape_supported(int64_t n, int d, int lookups, const int64_t* rows) {
  if (d > 64 || lookups > BVI_MAX_LOOKUPS || n > BVI_LOOKUP_MAX) return false;
  int64_t all = 0;
  for (int l = 0; l < lookups; ++l) {
    if (rows[l] > (1 << 25)) return false;
    all += rows[l];
  }
  return all <= (1 << 25);                          // the finishing launch has up to 64 threads for each
}

// 4-byte words of one copy: start, y, X, and per lookup the groups and, where there is one, the column
struct Layout {
  int64_t start, y, X, id[BVI_MAX_LOOKUPS], z[BVI_MAX_LOOKUPS], all;
};
Layout layout(int64_t n, int d, int lookups, int64_t rows, unsigned columns) {
  Layout t;
  int64_t at = 0;
  t.start = at; at += words(rows + 1);
  t.y = at; at += words(n + GR_PAD);
  t.X = at; at += words((n + GR_PAD) * padded_d(d));
  for (int l = 0; l < lookups; ++l) {
    t.id[l] = at; at += words(n + GR_PAD);
    t.z[l] = -1;
    if (columns >> l & 1u) { t.z[l] = at; at += words(n + GR_PAD); }
  }
  t.all = at;
  return t;
}
int64_t packed_words(int64_t n, int d, int lookups, const int64_t* rows, unsigned columns) {
  int64_t all = 0;
  for (int l = 0; l < lookups; ++l) all += layout(n, d, lookups, rows[l], columns).all;
  return all;
}

int chain_lanes(int C) { return bvi_chain_pack(C); }
// rows per wave: 16, or as many as leave GR_MAX_WAVES waves busy, but at most GR_MAX_SPAN
int64_t span_of(int64_t n) {
  const int64_t even = (n + GR_MAX_WAVES - 1) / GR_MAX_WAVES;
  const int64_t span = even < 16 ? 16 : even < GR_MAX_SPAN ? even : GR_MAX_SPAN;
  return (span + 3) / 4 * 4;                                 // a stretch starts on a 16-byte boundary
}
int64_t waves_of(int64_t n) { const int64_t s = span_of(n); return n > 0 ? (n + s - 1) / s : 1; }
int64_t blocks_of(int64_t n) { return (waves_of(n) + GR_WAVES - 1) / GR_WAVES; }

bool transposes(int lookups, int C);

// 4-byte words of the workspace: the dense sums, the transposed tables, the slots of every lookup
struct Space {
  int64_t dense, tables, slots[BVI_MAX_LOOKUPS], all;
};
Space space(int64_t n, int d, int lookups, const int64_t* rows, int C) {
  Space t;
  int64_t at = 0;
  t.dense = at; at += words(2 * blocks_of(n) * (2 + d) * C);
  int64_t sum = 0;
  for (int l = 0; l < lookups; ++l) sum += rows[l];
  t.tables = at; at += transposes(lookups, C) ? words(sum * C) : 0;
  for (int l = 0; l < lookups; ++l) {
    t.slots[l] = at;
    at += words((rows[l] + GR_WAVES * blocks_of(n)) * C);
  }
  t.all = at;
  return t;
}

struct GrCall {
  GrPasses passes;
  int64_t n, span, P;
  int d, lookups, C, blocks;
  const float* theta;
  double* dense;
  hipStream_t s;
};

// up to 16 chains: every lookup's pass in one launch
template <int CP, int D>
void launch_narrow(const GrCall& c, bool grad) {
  const dim3 grid(c.blocks, bvi_ceil_div(c.C, CP), grad ? c.lookups : 1);
  if (grad)
    hipLaunchKernelGGL((grouped_kernel<CP, D, true>), grid, dim3(64 * GR_WAVES), 0, c.s, c.passes, c.n, c.d, c.span, c.C, c.P,
                       c.theta, c.dense);
  else
    hipLaunchKernelGGL((grouped_kernel<CP, D, false>), grid, dim3(64 * GR_WAVES), 0, c.s, c.passes, c.n, c.d, c.span, c.C,
                       c.P, c.theta, c.dense);
}

// more: their passes are long enough, and those after the first do less
template <int D, bool GRAD, bool FIRST>
void launch_wide_pass(const GrCall& c, const GrPass& a) {
  const dim3 grid(c.blocks, bvi_ceil_div(c.C, 64));
#define GR_WIDE(N)                                                                                                    \
  hipLaunchKernelGGL((grouped_wide_kernel<D, GRAD, FIRST, N>), grid, dim3(64 * GR_WAVES), 0, c.s, a, a.y, a.X,          \
                     a.id[a.own], a.z[a.own], a.start, c.n, c.d, c.span, c.C, c.P, c.theta, a.slots, c.dense)
  if (a.lookups == 1) GR_WIDE(0);
  else if (a.lookups == 2) GR_WIDE(1);
  else GR_WIDE(2);
#undef GR_WIDE
}
template <int D>
void launch_wide(const GrCall& c, bool grad) {
  if (!grad) return launch_wide_pass<D, false, true>(c, c.passes.pass[0]);
  launch_wide_pass<D, true, true>(c, c.passes.pass[0]);
  for (int l = 1; l < c.lookups; ++l) launch_wide_pass<D, true, false>(c, c.passes.pass[l]);
}

template <int D>
void launch_passes(const GrCall& c, bool grad) {
  switch (chain_lanes(c.C)) {
    case 1: return launch_narrow<1, D>(c, grad);
    case 4: return launch_narrow<4, D>(c, grad);
    case 16: return launch_narrow<16, D>(c, grad);
    default: return launch_wide<D>(c, grad);
  }
}
// whether the tables are copied to [group, chain] first: a row's own entry comes once per group, those of other lookups
// by gathers of a line per chain.  us a call without / with the copy, 300001 rows:
//   20000 and 60 groups, D = 3     4 chains 36.0 / 37.5,  8 chains 76.9 / 78.5,  16 chains 87.6 / 84.7,  64 chains 187 / 125
//   2000 and 2000 groups           26.2 / 29.4,           41.6 / 45.0,           53.4 / 46.8,            183 / 96
//   200000 and 50000, D = 2        47.0 / 53.2,           110 / 115,             166 / 122,              988 / 293
// (2000 rows, where nothing but launches counts, 16 chains 19 / 22, 64 chains 23 / 30)
bool transposes(int lookups, int C) { return lookups > 1 && C > 8; }

}  // namespace

extern "C" {

int bvi_grouped_packed_bytes(int64_t n, int d, int n_lookups, const int64_t* rows, unsigned columns, size_t* packed_bytes,
                             size_t* ws_bytes) {
  if (!packed_bytes || !ws_bytes || !shape_ok(n, d, n_lookups, rows)) return BVI_ERR_ARG;
  if (!shape_supported(n, d, n_lookups, rows)) return BVI_ERR_UNSUPPORTED;
  *packed_bytes = 4 * (size_t)packed_words(n, d, n_lookups, rows, columns);
  size_t most = 0;
  for (int l = 0; l < n_lookups; ++l) {
    size_t plan, scratch;
    bvi_lookup_plan_bytes(rows[l], n, &plan, &scratch);
    most = plan + scratch > most ? plan + scratch : most;
  }
  *ws_bytes = most;
  return BVI_OK;
}

int bvi_grouped_pack(const float* X, const float* y, int64_t n, int d, int n_lookups, const int64_t* rows,
                     const int32_t* const* ids, const float* const* columns, void* packed, size_t packed_bytes, void* ws,
                     size_t ws_bytes, void* stream) {
  if (!shape_ok(n, d, n_lookups, rows) || (n > 0 && (!y || (d > 0 && !X) || !ids))) return BVI_ERR_ARG;
  if (!shape_supported(n, d, n_lookups, rows)) return BVI_ERR_UNSUPPORTED;
  unsigned mask = 0;
  for (int l = 0; l < n_lookups; ++l) {
    if (n > 0 && !ids[l]) return BVI_ERR_ARG;
    if (columns && columns[l]) mask |= 1u << l;
  }
  size_t need, scratch;
  bvi_grouped_packed_bytes(n, d, n_lookups, rows, mask, &need, &scratch);
  if (!packed || packed_bytes < need || !ws || ws_bytes < scratch) return BVI_ERR_WORKSPACE;
  if (((uintptr_t)packed | (uintptr_t)ws) % 16) return BVI_ERR_ARG;
  const hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)((n + 255) / 256));
  float* base = (float*)packed;
  for (int l = 0; l < n_lookups; ++l) {
    const Layout t = layout(n, d, n_lookups, rows[l], mask);
    size_t plan_bytes, sort_bytes;
    bvi_lookup_plan_bytes(rows[l], n, &plan_bytes, &sort_bytes);
    const int st = bvi_lookup_plan(n > 0 ? ids[l] : nullptr, BVI_IDS_I32, n, rows[l], ws, plan_bytes,
                                   (char*)ws + plan_bytes, sort_bytes, stream);
    if (st) return st;
    const int32_t* order = (const int32_t*)ws;
    const int32_t* start = (const int32_t*)ws + 2 * words(n);
    hipLaunchKernelGGL(grouped_pack_start_kernel, dim3((unsigned)((rows[l] + 256) / 256)), dim3(256), 0, s, start,
                       rows[l] + 1, (int32_t*)(base + t.start));
    if (n > 0) {
      hipLaunchKernelGGL(grouped_pack_kernel, grid, dim3(256), 0, s, X, y, n, d, padded_d(d), order, base + t.X,
                         base + t.y);
      for (int k = 0; k < n_lookups; ++k)
        hipLaunchKernelGGL(grouped_pack_column_kernel, grid, dim3(256), 0, s, ids[k],
                           t.z[k] >= 0 ? columns[k] : nullptr, rows[k], n, order, (int32_t*)(base + t.id[k]),
                           t.z[k] >= 0 ? base + t.z[k] : nullptr);
    }
    base += t.all;
  }
  BVI_HIP_CHECK_LAUNCH();
  return BVI_OK;
}

int bvi_grouped_ws_bytes(int64_t n, int d, int n_lookups, const int64_t* rows, int n_chains, size_t* ws_bytes) {
  if (!ws_bytes || !shape_ok(n, d, n_lookups, rows) || n_chains < 1) return BVI_ERR_ARG;
  if (!shape_supported(n, d, n_lookups, rows)) return BVI_ERR_UNSUPPORTED;
  if (n_chains > BVI_GROUPED_MAX_CHAINS) return BVI_ERR_UNSUPPORTED;
  *ws_bytes = 4 * (size_t)space(n, d, n_lookups, rows, n_chains).all;
  return BVI_OK;
}

int bvi_grouped_logp_grad(const void* packed, int64_t n, int d, int n_lookups, const int64_t* rows, unsigned columns,
                          const float* theta, int n_chains, float* logp, float* grad, const double* logp_ref, void* ws,
                          size_t ws_bytes, void* stream) {
  if (!packed || (uintptr_t)packed % 16 || !shape_ok(n, d, n_lookups, rows) || !theta || n_chains < 1 || !logp) return BVI_ERR_ARG;
  if (!shape_supported(n, d, n_lookups, rows)) return BVI_ERR_UNSUPPORTED;
  if (n_chains > BVI_GROUPED_MAX_CHAINS) return BVI_ERR_UNSUPPORTED;
  const int C = n_chains;
  const Space t = space(n, d, n_lookups, rows, C);
  if (!ws || ws_bytes < 4 * (size_t)t.all) return BVI_ERR_WORKSPACE;
  if ((uintptr_t)ws % 16) return BVI_ERR_ARG;
  const hipStream_t s = (hipStream_t)stream;
  const int64_t span = span_of(n);
  const int blocks = (int)blocks_of(n), cp = chain_lanes(C), count = grad ? 2 + d : 1;
  int64_t P = d + 2, sum = 0;
  for (int l = 0; l < n_lookups; ++l) P += rows[l];
  float* w = (float*)ws;
  double* dense = (double*)(w + t.dense);
  const bool copy = transposes(n_lookups, C);
  if (copy)
    hipLaunchKernelGGL(grouped_transpose_kernel, dim3((unsigned)((P - d - 2 + 63) / 64), bvi_ceil_div(C, 64)), dim3(256), 0,
                       s, theta, P, (int64_t)(d + 2), P - d - 2, C, w + t.tables);
  GrCall call;
  call.n = n;
  call.span = span;
  call.P = P;
  call.d = d;
  call.lookups = n_lookups;
  call.C = C;
  call.blocks = blocks;
  call.theta = theta;
  call.dense = dense;
  call.s = s;
  GrFinish f;
  f.lookups = n_lookups;
  const float* base = (const float*)packed;
  int64_t tiles = 0;
  for (int l = 0; l < n_lookups; ++l) {
    const Layout p = layout(n, d, n_lookups, rows[l], columns);
    GrPass& a = call.passes.pass[l];
    a.y = base + p.y;
    a.X = base + p.X;
    a.start = (const int32_t*)(base + p.start);
    a.slots = w + t.slots[l];
    a.own = l;
    a.lookups = n_lookups;
    a.group_stride = copy ? C : 1;
    a.chain_stride = copy ? 1 : P;
    int64_t at = 0;
    for (int k = 0; k < n_lookups; ++k) {
      a.id[k] = (const int32_t*)(base + p.id[k]);
      a.z[k] = p.z[k] >= 0 ? base + p.z[k] : nullptr;
      a.rows[k] = rows[k];
      a.tab[k] = copy ? w + t.tables + at * C : theta + d + 2 + at;
      at += rows[k];
    }
    f.start[l] = a.start;
    f.slots[l] = a.slots;
    f.rows[l] = rows[l];
    f.offset[l] = d + 2 + sum;
    sum += rows[l];
    tiles += (rows[l] + 1024 / cp - 1) / (1024 / cp);
    f.tile_end[l] = tiles;
    base += p.all;
  }
#define GR_D(X) \
  case X: launch_passes<X>(call, grad != nullptr); break
  switch (padded_d(d)) {
    GR_D(0); GR_D(1); GR_D(2); GR_D(4); GR_D(8); GR_D(16); GR_D(32); GR_D(64);
  }
#undef GR_D
  const dim3 grid((unsigned)(count + (grad ? tiles : 0)), bvi_ceil_div(C, cp));
#define GR_CP(X)                                                                                                   \
  case X:                                                                                                          \
    hipLaunchKernelGGL(grouped_finish_kernel<X>, grid, dim3(1024), 0, s, f, n, d, count, span, blocks, C, P, theta, \
                       (const double*)dense, logp_ref, logp, grad);                                                \
    break
  switch (cp) { GR_CP(1); GR_CP(4); GR_CP(16); GR_CP(64); }
#undef GR_CP
  BVI_HIP_CHECK_LAUNCH();
  return BVI_OK;
}

}  // extern "C"
