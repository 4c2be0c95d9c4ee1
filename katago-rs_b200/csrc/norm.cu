// Masked group norm with an activation on channels-last board tokens, forward and backward (kc_group_norm_act,
// kc_group_norm_act_backward).
//
//   on = mask != 0, M = (points on) * channels / groups, mean = sum_on x / M, var = sum_on (x - mean)^2 / M,
//   rstd = 1 / sqrt(var + eps), xh = (x - mean) rstd, z = xh w + b, y = act(z) where on, 0 elsewhere
//   gz = dy act'(z) where on, S1[c] = sum gz, S2[c] = sum gz xh (over a board's points),
//   c1 = sum_{c of the group} w S1 / M, c2 = sum w S2 / M, dx = rstd (gz w - c1 - xh c2) where on,
//   dbias = sum over boards of S1, dweight = of S2
//
// Statistics and sums are float32 (means are merged in float64). A thread's share of a mean and of a sum of squares
// is taken around its own mean and shares are merged by count, so that a large mean costs no digits of the variance.

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "../../include/katago_cuda.h"
#include "gemm.cuh"
#include "ops_common.h"

namespace kc {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTiles = 64;

struct NormParams {
  const void* x;
  const float* mask;
  const float* weight;
  const float* bias;
  void* y;               // forward: y; backward: dx
  const void* dy;
  float2* stats;         // [n][groups] (mean, rstd): written by the forward pass (may be null), read by the backward
  float2* part;          // [n][tiles][channels]: forward (mean, M2), backward (S1, S2)
  int* part_n;           // [n][tiles] points on
  float2* coef;          // [n][groups]: forward (mean, rstd), backward (c1, c2)
  float2* sums;          // [n][channels] backward (S1, S2) of a board
  int64_t xb, xr, yb, yr, mb;
  int n, points, C, G, cg, act;
  float eps;
  int tiles, tile_rows;
};

__device__ __forceinline__ bool point_on(const NormParams& p, int b, int r) {
  return p.mask == nullptr || __ldg(p.mask + (int64_t)b * p.mb + r) != 0.0f;
}

// relu keeps a NaN, as the other activations do
__device__ __forceinline__ float norm_act(float z, int act) {
  if (act == KC_ACT_RELU) return z < 0.0f ? 0.0f : z;
  if (act == KC_ACT_MISH) return act_fn<2>(z);
  if (act == KC_ACT_SILU) return act_fn<3>(z);
  return z;
}

// act'(z). relu's side of 0 is decided by the caller (relu_on).
// mish = z n / d with e = exp(z), n = e^2 + 2 e, d = n + 2: mish' = n / d + z 4 e (e + 1) / d^2 (1 above 20, where
// the rest is below 2^-24). silu' = s (1 + z (1 - s)), s = 1 / (1 + exp(-z)).
__device__ __forceinline__ float norm_act_slope(float z, int act) {
  if (act == KC_ACT_MISH) {
    const float e = __expf(fminf(z, 20.0f));
    const float n = e * (e + 2.0f);
    const float r = __fdividef(1.0f, n + 2.0f);
    const float g = n * r;
    const float s = g + z * (4.0f * e) * ((e + 1.0f) * r) * r;
    return z > 20.0f ? 1.0f : s;
  }
  if (act == KC_ACT_SILU) {
    const float s = __fdividef(1.0f, 1.0f + __expf(-z));
    const float v = s * (1.0f + z * (1.0f - s));
    return z < -80.0f ? 0.0f : v;  // exp(-z) leaves the fast divide's range
  }
  return 1.0f;
}

// Whether relu passes z = (x - mean) rstd w + b: in 64 bits where 32 cannot tell (the float32 z is off by less than
// 3 * 2^-24 |b|, since both factors' errors are relative to their product, which is near -b there).
__device__ __forceinline__ bool relu_on(float z, float x, float mean, float rstd, float w, float b) {
  if (fabsf(z) > 1e-6f * fabsf(b)) return z > 0.0f;
  return ((double)x - (double)mean) * (double)rstd * (double)w + (double)b > 0.0;
}

template <typename T, int VEC>
struct alignas(VEC * sizeof(T)) Pack {
  T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ void load_pack(const T* p, float (&v)[VEC]) {
  const Pack<T, VEC> u = *reinterpret_cast<const Pack<T, VEC>*>(p);
#pragma unroll
  for (int j = 0; j < VEC; j++) v[j] = to_f<T>(u.v[j]);
}

template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T* p, const float (&v)[VEC]) {
  Pack<T, VEC> u;
#pragma unroll
  for (int j = 0; j < VEC; j++) u.v[j] = from_f<T>(v[j]);
  *reinterpret_cast<Pack<T, VEC>*>(p) = u;
}

// ---------------------------------------------------------------------------------------------------------------
// The split path, for boards too large for one cluster of blocks: column vectors of VEC channels (lanes tx) by rows
// (ty), a tile of rows per block. grid (tiles * column blocks, boards modulo grid.y).
// ---------------------------------------------------------------------------------------------------------------
struct TileIds {
  int tile, col0, tx, ty, rows_at_once;
  bool active;
};

template <int VEC>
__device__ __forceinline__ TileIds tile_ids(const NormParams& p) {
  const int V = p.C / VEC, vc = V < 64 ? V : 64;  // column vectors of a block
  TileIds t;
  t.tile = blockIdx.x % p.tiles;
  t.tx = threadIdx.x % vc;
  t.ty = threadIdx.x / vc;
  t.rows_at_once = kThreads / vc;
  const int cv = (blockIdx.x / p.tiles) * vc + t.tx;
  t.col0 = cv * VEC;
  t.active = t.ty < t.rows_at_once && cv < V;
  return t;
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) norm_tile_stats_kernel(const __grid_constant__ NormParams p) {
  __shared__ float2 red[kThreads * VEC];
  __shared__ int red_n[kThreads];
  const TileIds t = tile_ids<VEC>(p);
  const int r1 = min(p.points, (t.tile + 1) * p.tile_rows);
  for (int b = blockIdx.y; b < p.n; b += gridDim.y) {
    const T* x = static_cast<const T*>(p.x) + (int64_t)b * p.xb + t.col0;
    float mean[VEC] = {}, m2[VEC] = {};
    int cnt = 0;
    if (t.active) {
      for (int r = t.tile * p.tile_rows + t.ty; r < r1; r += 4 * t.rows_at_once) {
        float v[4][VEC];
        bool on[4];
        int k = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int ri = r + i * t.rows_at_once;
          on[i] = ri < r1 && point_on(p, b, ri);
          if (on[i]) {
            load_pack<T, VEC>(x + (int64_t)ri * p.xr, v[i]);
            k++;
          }
        }
        if (!k) continue;
        const float ik = 1.0f / (float)k, share = (float)k / (float)(cnt + k);
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          float s = 0.0f, q = 0.0f;
#pragma unroll
          for (int i = 0; i < 4; i++) s += on[i] ? v[i][j] : 0.0f;
          s *= ik;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float d = on[i] ? v[i][j] - s : 0.0f;
            q += d * d;
          }
          const float d = s - mean[j];
          mean[j] += d * share;
          m2[j] += cnt ? q + d * d * ((float)cnt * share) : q;  // the first share has no distance to square
        }
        cnt += k;
      }
    }
    if (t.active) {
#pragma unroll
      for (int j = 0; j < VEC; j++) red[(t.ty * VEC + j) * (kThreads / t.rows_at_once) + t.tx] = make_float2(mean[j], m2[j]);
      if (t.tx == 0) red_n[t.ty] = cnt;
    }
    __syncthreads();
    if (t.active && t.ty == 0) {
      int N = 0;
      for (int i = 0; i < t.rows_at_once; i++) N += red_n[i];
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        double s = 0.0;
        for (int i = 0; i < t.rows_at_once; i++)
          s += (double)red_n[i] * red[(i * VEC + j) * (kThreads / t.rows_at_once) + t.tx].x;
        const double mu = N ? s / N : 0.0;
        float q = 0.0f;
        for (int i = 0; i < t.rows_at_once; i++) {
          const float2 u = red[(i * VEC + j) * (kThreads / t.rows_at_once) + t.tx];
          const float d = (float)(u.x - mu);
          q += red_n[i] ? u.y + d * d * (float)red_n[i] : 0.0f;
        }
        p.part[((int64_t)b * p.tiles + t.tile) * p.C + t.col0 + j] = make_float2((float)mu, q);
      }
      if (t.col0 == 0) p.part_n[(int64_t)b * p.tiles + t.tile] = N;
    }
    __syncthreads();
  }
}

// Merges the tiles and channels of one group: a warp per (board, group).
__global__ void __launch_bounds__(kThreads) norm_merge_stats_kernel(const __grid_constant__ NormParams p) {
  const int64_t id = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / 32;
  const int lane = threadIdx.x & 31;
  if (id >= (int64_t)p.n * p.G) return;
  const int b = (int)(id / p.G), g = (int)(id % p.G);
  const float2* part = p.part + (int64_t)b * p.tiles * p.C + (int64_t)g * p.cg;
  const int* pn = p.part_n + (int64_t)b * p.tiles;
  const int64_t items = (int64_t)p.tiles * p.cg;
  double s = 0.0, N = 0.0;
  for (int64_t i = lane; i < items; i += 32) {
    const int t = (int)(i / p.cg);
    const int k = pn[t];
    N += k;
    s += (double)k * part[(int64_t)t * p.C + i % p.cg].x;
  }
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    N += __shfl_xor_sync(0xffffffffu, N, o);
  }
  const double mu = N > 0.0 ? s / N : 0.0;
  double q = 0.0;
  for (int64_t i = lane; i < items; i += 32) {
    const int t = (int)(i / p.cg);
    const int k = pn[t];
    const float2 u = part[(int64_t)t * p.C + i % p.cg];
    const float d = (float)(u.x - mu);
    if (k) q += u.y + d * d * (float)k;
  }
  for (int o = 16; o > 0; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
  if (lane == 0) {
    const float2 st = N > 0.0 ? make_float2((float)mu, 1.0f / sqrtf((float)(q / N) + p.eps)) : make_float2(0.0f, 0.0f);
    p.coef[id] = st;
    if (p.stats) p.stats[id] = st;
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) norm_tile_apply_kernel(const __grid_constant__ NormParams p) {
  const TileIds t = tile_ids<VEC>(p);
  if (!t.active) return;
  const int r1 = min(p.points, (t.tile + 1) * p.tile_rows);
  for (int b = blockIdx.y; b < p.n; b += gridDim.y) {
    const T* x = static_cast<const T*>(p.x) + (int64_t)b * p.xb + t.col0;
    T* y = static_cast<T*>(p.y) + (int64_t)b * p.yb + t.col0;
    float mean[VEC], a[VEC], bias[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) {
      const float2 st = p.coef[(int64_t)b * p.G + (t.col0 + j) / p.cg];
      mean[j] = st.x;
      a[j] = st.y * (p.weight ? __ldg(p.weight + t.col0 + j) : 1.0f);
      bias[j] = p.bias ? __ldg(p.bias + t.col0 + j) : 0.0f;
    }
    for (int r = t.tile * p.tile_rows + t.ty; r < r1; r += t.rows_at_once) {
      float v[VEC] = {};
      if (point_on(p, b, r)) {
        load_pack<T, VEC>(x + (int64_t)r * p.xr, v);
#pragma unroll
        for (int j = 0; j < VEC; j++) v[j] = norm_act((v[j] - mean[j]) * a[j] + bias[j], p.act);
      }
      store_pack<T, VEC>(y + (int64_t)r * p.yr, v);
    }
  }
}

// Backward, per-channel constants of a thread's column vector.
template <int VEC>
struct Channel {
  float mean[VEC], rstd[VEC], w[VEC], b[VEC];
};

template <int VEC>
__device__ __forceinline__ Channel<VEC> load_channel(const NormParams& p, int b, int col0) {
  Channel<VEC> c;
#pragma unroll
  for (int j = 0; j < VEC; j++) {
    const float2 st = p.stats[(int64_t)b * p.G + (col0 + j) / p.cg];
    c.mean[j] = st.x;
    c.rstd[j] = st.y;
    c.w[j] = p.weight ? __ldg(p.weight + col0 + j) : 1.0f;
    c.b[j] = p.bias ? __ldg(p.bias + col0 + j) : 0.0f;
  }
  return c;
}

// xh and gz of one vector (x, dy in; xh, gz out).
template <int VEC>
__device__ __forceinline__ void back_vec(const Channel<VEC>& c, int act, float (&x)[VEC], float (&g)[VEC]) {
#pragma unroll
  for (int j = 0; j < VEC; j++) {
    const float xh = (x[j] - c.mean[j]) * c.rstd[j];
    const float z = xh * c.w[j] + c.b[j];
    if (act == KC_ACT_RELU)
      g[j] = relu_on(z, x[j], c.mean[j], c.rstd[j], c.w[j], c.b[j]) ? g[j] : 0.0f;
    else
      g[j] *= norm_act_slope(z, act);
    x[j] = xh;
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) norm_tile_back_kernel(const __grid_constant__ NormParams p) {
  __shared__ float2 red[kThreads * VEC];
  __shared__ int red_n[kThreads];
  const TileIds t = tile_ids<VEC>(p);
  const int r1 = min(p.points, (t.tile + 1) * p.tile_rows);
  for (int b = blockIdx.y; b < p.n; b += gridDim.y) {
    float s1[VEC] = {}, s2[VEC] = {};
    int cnt = 0;
    if (t.active) {
      const T* x = static_cast<const T*>(p.x) + (int64_t)b * p.xb + t.col0;
      const T* dy = static_cast<const T*>(p.dy) + (int64_t)b * p.yb + t.col0;
      const Channel<VEC> c = load_channel<VEC>(p, b, t.col0);
      for (int r = t.tile * p.tile_rows + t.ty; r < r1; r += t.rows_at_once) {
        if (!point_on(p, b, r)) continue;
        float v[VEC], g[VEC];
        load_pack<T, VEC>(x + (int64_t)r * p.xr, v);
        load_pack<T, VEC>(dy + (int64_t)r * p.yr, g);
        back_vec<VEC>(c, p.act, v, g);
        cnt++;
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          s1[j] += g[j];
          s2[j] += g[j] * v[j];
        }
      }
    }
    if (t.active) {
#pragma unroll
      for (int j = 0; j < VEC; j++) red[(t.ty * VEC + j) * (kThreads / t.rows_at_once) + t.tx] = make_float2(s1[j], s2[j]);
      if (t.tx == 0) red_n[t.ty] = cnt;
    }
    __syncthreads();
    if (t.active && t.ty == 0) {
      int N = 0;
      for (int i = 0; i < t.rows_at_once; i++) N += red_n[i];
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        float2 s = make_float2(0.0f, 0.0f);
        for (int i = 0; i < t.rows_at_once; i++) {
          const float2 u = red[(i * VEC + j) * (kThreads / t.rows_at_once) + t.tx];
          s.x += u.x;
          s.y += u.y;
        }
        p.part[((int64_t)b * p.tiles + t.tile) * p.C + t.col0 + j] = s;
      }
      if (t.col0 == 0) p.part_n[(int64_t)b * p.tiles + t.tile] = N;
    }
    __syncthreads();
  }
}

// Adds the tiles of one group's channels and makes its c1, c2: a warp per (board, group).
__global__ void __launch_bounds__(kThreads) norm_merge_back_kernel(const __grid_constant__ NormParams p) {
  const int64_t id = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / 32;
  const int lane = threadIdx.x & 31;
  if (id >= (int64_t)p.n * p.G) return;
  const int b = (int)(id / p.G), g = (int)(id % p.G);
  const int* pn = p.part_n + (int64_t)b * p.tiles;
  double N = 0.0;
  for (int t = 0; t < p.tiles; t++) N += pn[t];
  N *= p.cg;
  double c1 = 0.0, c2 = 0.0;
  for (int i = lane; i < p.cg; i += 32) {
    const int c = g * p.cg + i;
    float2 s = make_float2(0.0f, 0.0f);
    for (int t = 0; t < p.tiles; t++) {
      const float2 u = p.part[((int64_t)b * p.tiles + t) * p.C + c];
      s.x += u.x;
      s.y += u.y;
    }
    p.sums[(int64_t)b * p.C + c] = s;
    const float w = p.weight ? __ldg(p.weight + c) : 1.0f;
    c1 += (double)w * s.x;
    c2 += (double)w * s.y;
  }
  for (int o = 16; o > 0; o >>= 1) {
    c1 += __shfl_xor_sync(0xffffffffu, c1, o);
    c2 += __shfl_xor_sync(0xffffffffu, c2, o);
  }
  if (lane == 0) p.coef[id] = N > 0.0 ? make_float2((float)(c1 / N), (float)(c2 / N)) : make_float2(0.0f, 0.0f);
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) norm_tile_dx_kernel(const __grid_constant__ NormParams p) {
  const TileIds t = tile_ids<VEC>(p);
  if (!t.active) return;
  const int r1 = min(p.points, (t.tile + 1) * p.tile_rows);
  for (int b = blockIdx.y; b < p.n; b += gridDim.y) {
    const T* x = static_cast<const T*>(p.x) + (int64_t)b * p.xb + t.col0;
    const T* dy = static_cast<const T*>(p.dy) + (int64_t)b * p.yb + t.col0;
    T* dx = static_cast<T*>(p.y) + (int64_t)b * p.xb + t.col0;
    const Channel<VEC> c = load_channel<VEC>(p, b, t.col0);
    float2 k[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) k[j] = p.coef[(int64_t)b * p.G + (t.col0 + j) / p.cg];
    for (int r = t.tile * p.tile_rows + t.ty; r < r1; r += t.rows_at_once) {
      float v[VEC], g[VEC], o[VEC] = {};
      if (point_on(p, b, r)) {
        load_pack<T, VEC>(x + (int64_t)r * p.xr, v);
        load_pack<T, VEC>(dy + (int64_t)r * p.yr, g);
        back_vec<VEC>(c, p.act, v, g);
#pragma unroll
        for (int j = 0; j < VEC; j++) o[j] = (g[j] * c.w[j] - k[j].x - v[j] * k[j].y) * c.rstd[j];
      }
      store_pack<T, VEC>(dx + (int64_t)r * p.xr, o);
    }
  }
}

// dbias, dweight [c] = the boards' sums in a fixed order: 32 channels a block, 8 board lanes each.
__global__ void __launch_bounds__(kThreads) norm_boards_kernel(const float2* __restrict__ sums, int n, int C,
                                                               float* __restrict__ dweight,
                                                               float* __restrict__ dbias) {
  __shared__ double2 red[8][32];
  const int tx = threadIdx.x & 31, ty = threadIdx.x / 32;
  const int c = blockIdx.x * 32 + tx;
  double2 s = make_double2(0.0, 0.0);
  if (c < C)
    for (int b = ty; b < n; b += 8) {
      const float2 u = sums[(int64_t)b * C + c];
      s.x += u.x;
      s.y += u.y;
    }
  red[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && c < C) {
    for (int i = 1; i < 8; i++) {
      s.x += red[i][tx].x;
      s.y += red[i][tx].y;
    }
    if (dbias) dbias[c] = (float)s.x;
    if (dweight) dweight[c] = (float)s.y;
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------------------------
[[noreturn]] void bad(const std::string& m) { fail(KC_ERR_INVALID, "CUDA backend: group norm: " + m); }

void check_desc(const kc_group_norm_desc* d) {
  if (!d) bad("null descriptor");
  if (d->dtype != KC_PRECISION_F32 && d->dtype != KC_PRECISION_F16 && d->dtype != KC_PRECISION_BF16)
    bad("dtype must be KC_PRECISION_F32, F16 or BF16");
  if (d->act < KC_ACT_IDENTITY || d->act > KC_ACT_SILU) bad("unknown activation");
  if (d->n < 0 || d->points < 0) bad("n and points must not be negative");
  if (d->channels < 1 || d->groups < 1) bad("channels and groups must be positive");
  if (d->channels % d->groups != 0) bad("channels must be a multiple of groups");
  if (!(d->eps >= 0.0f) || !std::isfinite(d->eps)) bad("eps must be finite and not negative");
  if (d->reserved != 0) bad("reserved must be 0");
}

Rows x_rows(const kc_group_norm_desc& d, const void* p) {
  return {p, d.n, d.points, d.channels, d.x_board_stride, d.x_row_stride, dtype_bytes(d.dtype)};
}
Rows y_rows(const kc_group_norm_desc& d, const void* p) {
  return {p, d.n, d.points, d.channels, d.y_board_stride, d.y_row_stride, dtype_bytes(d.dtype)};
}

// Tiles of rows of the split path: enough blocks for every SM several times over, of at least 32 rows.
void split_shape(const kc_group_norm_desc& d, int& tiles, int& tile_rows) {
  const int64_t per_board = std::max<int64_t>(1, 2048 / ((int64_t)std::max(1, d.n) * ((d.channels + 511) / 512)));
  const int64_t t = std::min<int64_t>({(int64_t)kMaxTiles, per_board, (d.points + 31) / 32});
  tile_rows = (int)((d.points + std::max<int64_t>(1, t) - 1) / std::max<int64_t>(1, t));
  tiles = (d.points + tile_rows - 1) / std::max(1, tile_rows);
}

struct Layout {
  size_t part = 0, part_n = 0, coef = 0, sums = 0, total = 0;
};
size_t round256(size_t v) { return (v + 255) / 256 * 256; }

Layout workspace_layout(const kc_group_norm_desc& d, bool backward) {
  Layout l;
  if (d.n == 0 || d.points == 0) return l;
  int tiles, tile_rows;
  split_shape(d, tiles, tile_rows);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += round256(bytes);
    return here;
  };
  l.part = take((size_t)d.n * tiles * d.channels * sizeof(float2));
  l.part_n = take((size_t)d.n * tiles * sizeof(int));
  l.coef = take((size_t)d.n * d.groups * sizeof(float2));
  if (backward) l.sums = take((size_t)d.n * d.channels * sizeof(float2));
  l.total = at;
  return l;
}

// The widest vector that channels, strides and addresses allow.
int vec_of(const kc_group_norm_desc& d, std::initializer_list<const void*> ptrs) {
  const int es = dtype_bytes(d.dtype);
  for (int v = 16 / es; v > 1; v /= 2) {
    const bool board = d.n == 1 || (d.x_board_stride % v == 0 && d.y_board_stride % v == 0);
    const bool row = d.points == 1 || (d.x_row_stride % v == 0 && d.y_row_stride % v == 0);
    bool ok = d.channels % v == 0 && board && row;
    for (const void* p : ptrs) ok = ok && aligned_to(p, (size_t)v * es);
    if (ok) return v;
  }
  return 1;
}

template <typename T, int VEC>
void split_forward(const NormParams& p, cudaStream_t st) {
  const int V = p.C / VEC, vc = std::min(V, 64);
  const dim3 grid((unsigned)(p.tiles * ((V + vc - 1) / vc)), (unsigned)std::min(p.n, 65535));
  const unsigned warps = (unsigned)(((int64_t)p.n * p.G + kThreads / 32 - 1) / (kThreads / 32));
  norm_tile_stats_kernel<T, VEC><<<grid, kThreads, 0, st>>>(p);
  KC_CUDA(cudaGetLastError());
  norm_merge_stats_kernel<<<warps, kThreads, 0, st>>>(p);
  KC_CUDA(cudaGetLastError());
  norm_tile_apply_kernel<T, VEC><<<grid, kThreads, 0, st>>>(p);
  KC_CUDA(cudaGetLastError());
}

template <typename T, int VEC>
void split_backward(const NormParams& p, cudaStream_t st) {
  const int V = p.C / VEC, vc = std::min(V, 64);
  const dim3 grid((unsigned)(p.tiles * ((V + vc - 1) / vc)), (unsigned)std::min(p.n, 65535));
  const unsigned warps = (unsigned)(((int64_t)p.n * p.G + kThreads / 32 - 1) / (kThreads / 32));
  norm_tile_back_kernel<T, VEC><<<grid, kThreads, 0, st>>>(p);
  KC_CUDA(cudaGetLastError());
  norm_merge_back_kernel<<<warps, kThreads, 0, st>>>(p);
  KC_CUDA(cudaGetLastError());
  norm_tile_dx_kernel<T, VEC><<<grid, kThreads, 0, st>>>(p);
  KC_CUDA(cudaGetLastError());
}

template <typename T, int VEC>
void run_vec(const NormParams& p, bool backward, cudaStream_t st) {
  backward ? split_backward<T, VEC>(p, st) : split_forward<T, VEC>(p, st);
}

template <typename T>
void run_type(const NormParams& p, int vec, bool backward, cudaStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (vec == 8) return run_vec<T, 8>(p, backward, st);
  if (vec == 4) return run_vec<T, 4>(p, backward, st);
  if (vec == 2) return run_vec<T, 2>(p, backward, st);
  run_vec<T, 1>(p, backward, st);
}

void run(const kc_group_norm_desc& d, NormParams p, int vec, bool backward, void* workspace, cudaStream_t st) {
  p.n = d.n;
  p.points = d.points;
  p.C = d.channels;
  p.G = d.groups;
  p.cg = d.channels / d.groups;
  p.act = d.act;
  p.eps = d.eps;
  p.xb = d.x_board_stride;
  p.xr = d.x_row_stride;
  p.yb = d.y_board_stride;
  p.yr = d.y_row_stride;
  p.mb = d.mask_board_stride;
  split_shape(d, p.tiles, p.tile_rows);
  const Layout l = workspace_layout(d, backward);
  char* ws = static_cast<char*>(workspace);
  p.part = reinterpret_cast<float2*>(ws + l.part);
  p.part_n = reinterpret_cast<int*>(ws + l.part_n);
  p.coef = reinterpret_cast<float2*>(ws + l.coef);
  p.sums = reinterpret_cast<float2*>(ws + l.sums);
  if (d.dtype == KC_PRECISION_F32) run_type<float>(p, vec, backward, st);
  else if (d.dtype == KC_PRECISION_F16) run_type<__half>(p, vec, backward, st);
  else run_type<__nv_bfloat16>(p, vec, backward, st);
}

void check_tensors(const kc_group_norm_desc& d, std::initializer_list<Rows> rows, const float* mask,
                   std::initializer_list<const void*> small) {
  const Rows m{mask, d.n, 1, d.points, d.mask_board_stride, 0, 4};
  if (mask && !rows_in_range(m)) bad("mask stride out of range");
  for (const Rows& r : rows) {
    if (!rows_in_range(r)) bad("strides must not be negative, nor reach past 2^46 elements");
    if (!aligned_to(r.p, r.bytes)) bad("a tensor is not aligned to its element");
  }
  for (const void* s : small)
    if (!aligned_to(s, 4)) bad("a float32 tensor is not aligned to its element");
}

// Outputs share no memory with each other or with an input; only a tensor may be its own output.
struct Range {
  const void* p;
  int64_t bytes;
};

void check_outputs(const kc_group_norm_desc& d, const Rows& out, std::initializer_list<Rows> ins, const float* mask,
                   std::initializer_list<Range> small_in, std::initializer_list<Range> small_out) {
  if (!rows_distinct(out)) bad("rows of the output share memory");
  for (const Rows& i : ins)
    if (rows_overlap(out, i) && !out.same(i)) bad("the output overlaps an input it does not match");
  const Rows m{mask, d.n, 1, d.points, d.mask_board_stride, 0, 4};
  if (rows_overlap(out, m)) bad("the output overlaps the mask");
  for (const Range& s : small_in)
    if (ranges_meet(s.p, s.bytes, out)) bad("the output overlaps another tensor of the call");
  for (const Range* o = small_out.begin(); o != small_out.end(); o++) {
    bool meets = ranges_meet(o->p, o->bytes, out) || ranges_meet(o->p, o->bytes, m);
    for (const Rows& i : ins) meets = meets || ranges_meet(o->p, o->bytes, i);
    for (const Range& s : small_in) meets = meets || ranges_meet(o->p, o->bytes, {s.p, 1, 1, s.bytes, 0, 0, s.p ? 1 : 0});
    for (const Range* q = o + 1; q != small_out.end(); q++)
      meets = meets || ranges_meet(o->p, o->bytes, {q->p, 1, 1, q->bytes, 0, 0, q->p ? 1 : 0});
    if (meets) bad("the statistics, parameter gradients or workspace overlap another tensor of the call");
  }
}

void check_workspace(const void* ws, size_t have, size_t need) {
  if (need == 0) return;
  if (!ws || have < need) bad("workspace of " + std::to_string(need) + " bytes needed");
  if (!aligned_to(ws, 16)) bad("the workspace must be 16-byte aligned");
}

}  // namespace
}  // namespace kc

extern "C" int kc_group_norm_act_workspace(const kc_group_norm_desc* desc, int backward, size_t* bytes) {
  return kc::guard_entry([&] {
    kc::check_desc(desc);
    if (!bytes) kc::bad("null result");
    *bytes = kc::workspace_layout(*desc, backward != 0).total;
  });
}

extern "C" int kc_group_norm_act(const kc_group_norm_desc* desc, const void* d_x, const float* d_mask,
                                 const float* d_weight, const float* d_bias, void* d_y, float* d_stats,
                                 void* d_workspace, size_t workspace_bytes, void* stream) {
  return kc::guard_entry([&] {
    using namespace kc;
    check_desc(desc);
    const kc_group_norm_desc d = *desc;
    const bool none = d.n == 0 || d.points == 0;
    if (!none && (!d_x || !d_y)) bad("null tensor");
    const Rows x = x_rows(d, d_x), y = y_rows(d, d_y);
    const int64_t ch = 4 * (int64_t)d.channels, sb = 8 * (int64_t)d.n * d.groups;
    check_tensors(d, {x, y}, d_mask, {d_mask, d_weight, d_bias, d_stats});
    if (!aligned_to(d_stats, 8)) bad("the statistics must be 8-byte aligned");
    const size_t need = workspace_layout(d, false).total;
    check_outputs(d, y, {x}, d_mask, {{d_weight, ch}, {d_bias, ch}}, {{d_stats, sb}, {d_workspace, (int64_t)need}});
    check_workspace(d_workspace, workspace_bytes, need);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (none && (d.n == 0 || !d_stats)) return;
    TensorDevice dev("group norm", {d_x, d_mask, d_weight, d_bias, d_y, d_stats, need ? d_workspace : nullptr});
    if (none) {
      KC_CUDA(cudaMemsetAsync(d_stats, 0, (size_t)sb, st));
      return;
    }
    NormParams p{};
    p.x = d_x;
    p.mask = d_mask;
    p.weight = d_weight;
    p.bias = d_bias;
    p.y = d_y;
    p.stats = reinterpret_cast<float2*>(d_stats);
    run(d, p, vec_of(d, {d_x, d_y}), false, d_workspace, st);
  });
}

extern "C" int kc_group_norm_act_backward(const kc_group_norm_desc* desc, const void* d_x, const float* d_mask,
                                          const float* d_weight, const float* d_bias, const float* d_stats,
                                          const void* d_dy, void* d_dx, float* d_dweight, float* d_dbias,
                                          void* d_workspace, size_t workspace_bytes, void* stream) {
  return kc::guard_entry([&] {
    using namespace kc;
    check_desc(desc);
    const kc_group_norm_desc d = *desc;
    const bool none = d.n == 0 || d.points == 0;
    if (!none && (!d_x || !d_dy || !d_dx || !d_stats)) bad("null tensor");
    const Rows x = x_rows(d, d_x), dy = y_rows(d, d_dy), dx = x_rows(d, d_dx);
    const int64_t ch = 4 * (int64_t)d.channels, sb = 8 * (int64_t)d.n * d.groups;
    check_tensors(d, {x, dy, dx}, d_mask, {d_mask, d_weight, d_bias, d_stats, d_dweight, d_dbias});
    if (!aligned_to(d_stats, 8)) bad("the statistics must be 8-byte aligned");
    const size_t need = workspace_layout(d, true).total;
    check_outputs(d, dx, {x, dy}, d_mask, {{d_weight, ch}, {d_bias, ch}, {d_stats, sb}},
                  {{d_dweight, ch}, {d_dbias, ch}, {d_workspace, (int64_t)need}});
    check_workspace(d_workspace, workspace_bytes, need);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (none && !d_dweight && !d_dbias) return;
    TensorDevice dev("group norm", {d_x, d_mask, d_weight, d_bias, d_stats, d_dy, d_dx, d_dweight, d_dbias,
                                    need ? d_workspace : nullptr});
    if (none) {
      if (d_dweight) KC_CUDA(cudaMemsetAsync(d_dweight, 0, (size_t)ch, st));
      if (d_dbias) KC_CUDA(cudaMemsetAsync(d_dbias, 0, (size_t)ch, st));
      return;
    }
    NormParams p{};
    p.x = d_x;
    p.mask = d_mask;
    p.weight = d_weight;
    p.bias = d_bias;
    p.y = d_dx;
    p.dy = d_dy;
    p.stats = const_cast<float2*>(reinterpret_cast<const float2*>(d_stats));
    run(d, p, vec_of(d, {d_x, d_dy, d_dx}), true, d_workspace, st);
    if (d_dweight || d_dbias) {
      const Layout l = workspace_layout(d, true);
      norm_boards_kernel<<<(d.channels + 31) / 32, kThreads, 0, st>>>(
          reinterpret_cast<const float2*>(static_cast<char*>(d_workspace) + l.sums), d.n, d.channels, d_dweight, d_dbias);
      KC_CUDA(cudaGetLastError());
    }
  });
}
