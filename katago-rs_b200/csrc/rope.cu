// Rotary positions with several axes on Q and K heads, forward and backward (kc_rope_axes, kc_rope_axes_backward).
//
//   angle[t][tb][j] = sum_a pos[t][a] freqs[tb][j][a], (y1, y2) = (x1 cos - x2 sin, x1 sin + x2 cos)
//   backward: dx = the gradient turned by -angle; d angle = dx2 x1 - dx1 x2;
//   dfreqs[tb][j][a] = sum_t pos[t][a] sum over the table's heads of d angle
//
// Angles are held in turns, as 64-bit fractions: a frequency is freq / (2 pi) mod 1 scaled by 2^64 (from float64, so
// 53 bits of freq / (2 pi)), and whole turns of pos * frequency drop out of the 64-bit product by themselves. The
// error is that of freq / (2 pi), 2^-53 of the angle; far positions keep their digits, at three integer
// multiply-adds an axis.
//
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <string>

#include "../../include/katago_cuda.h"
#include "gemm.cuh"
#include "ops_common.h"

namespace kc {
namespace {

constexpr int kThreads = 256;

struct Heads {
  const void* in;
  void* out;
  const void* x;  // backward: the forward pass's input
  int64_t in_t, in_h, out_t, out_h, x_t, x_h;
  int per_table;
};

struct RopeParams {
  Heads q, k;
  const int* pos;
  const float* freqs;
  int64_t tokens;
  int axes, pairs, rest, tables;  // rest: head dimensions behind the rotated ones
  int sign;                       // +1 forward, -1 backward
  // kernels that go over tiles of tokens
  int tile, rounds;               // tokens of a tile, threads that share a table's heads (head i of one: i mod rounds)
  uint32_t by_token, by_table, by_head;  // magic() of a token's items, a table's, a head's
  // backward with the frequencies' gradient
  int head_lanes;                 // threads that share a table's heads: lane l takes heads l, l + head_lanes, ...
  int width, lanes;               // a block's columns (table, head lane, vector of a head) and tokens at once
  int columns;                    // of all blocks y
  int shared;                     // the frequencies' fractions are staged in shared memory
  float* partial;                 // [blocks][tables][pairs][axes]
  float* dfreqs;
  int blocks;
};

template <typename T, int N>
struct alignas(N * sizeof(T)) Pack {
  T v[N];
};

// freq / (2 pi) mod 1, times 2^64. A frequency that is not finite gives 0 here; its angle is made NaN apart.
__device__ __forceinline__ unsigned long long turn_fraction(float freq) {
  const double t = (double)freq * 0.15915494309189533577;  // 1 / (2 pi)
  const double f = t - floor(t);
  return f >= 0.0 && f < 1.0 ? (unsigned long long)(f * 18446744073709551616.0) : 0ull;
}

__device__ __forceinline__ float sin_fast(float x) {
  float y;
  asm("sin.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float cos_fast(float x) {
  float y;
  asm("cos.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// n / d by magic(d).
__device__ __forceinline__ int quotient(int n, uint32_t magic) { return magic ? (int)__umulhi((uint32_t)n, magic) : n; }

struct Position {
  int at[KC_ROPE_MAX_AXES];
  __device__ __forceinline__ void load(const RopeParams& p, int64_t t) {
#pragma unroll
    for (int a = 0; a < KC_ROPE_MAX_AXES; a++) at[a] = a < p.axes ? __ldg(p.pos + t * p.axes + a) : 0;
  }
};

// (cos, sin) of an angle of turns * 2^-64. float32 takes the accurate functions; for 2-byte results the fast ones on
// half a turn either way (off by 2^-21) are far below the rounding.
template <typename T>
__device__ __forceinline__ float2 turned(unsigned long long turns) {
  const float part = (float)(int)(turns >> 32);  // in 2^-32 turns, [-2^31, 2^31)
  float2 r;
  if constexpr (sizeof(T) == 4) {
    sincospif(part * 4.656612873077393e-10f, &r.y, &r.x);  // 2^-31
  } else {
    const float x = part * 1.4629180792671596e-09f;  // 2 pi 2^-32
    r.x = cos_fast(x);
    r.y = sin_fast(x);
  }
  return r;
}

// sin and cos of VP pairs' angles at one token, from the fractions in shared memory ([pair of the vector][axis] rows
// of `stride` columns, so that neighbouring threads read neighbouring words) or from the frequencies `f`.
template <typename T, int VP, bool STAGED>
__device__ __forceinline__ void angles(const RopeParams& p, const Position& at, const unsigned long long* g, int stride,
                                       const float* f, float (&c)[VP], float (&s)[VP]) {
#pragma unroll
  for (int j = 0; j < VP; j++) {
    unsigned long long turns = 0;
    float bad = 0.0f;  // NaN where a frequency is not finite
#pragma unroll
    for (int a = 0; a < KC_ROPE_MAX_AXES; a++)
      if (a < p.axes) {
        const unsigned long long n = (unsigned long long)((long long)at.at[a] * p.sign);
        if constexpr (STAGED) {
          turns += n * g[(j * p.axes + a) * stride];
        } else {
          const float fr = __ldg(f + j * p.axes + a);
          bad += fr - fr;
          turns += n * turn_fraction(fr);
        }
      }
    const float2 cs = turned<T>(turns);
    c[j] = cs.x;
    s[j] = cs.y;
    if constexpr (!STAGED) {
      s[j] += bad;
      c[j] += bad;
    }
  }
}

// The two halves of VP pairs of a head that starts at h: pair j of [j0, j0 + VP).
template <typename T, int VP, int LAYOUT>
struct Pairs {
  Pack<T, VP> u, v;
  __device__ __forceinline__ void load(const T* h, int j0, int pairs) {
    if constexpr (LAYOUT == KC_ROPE_HALVES) {
      u = *reinterpret_cast<const Pack<T, VP>*>(h + j0);
      v = *reinterpret_cast<const Pack<T, VP>*>(h + pairs + j0);
    } else {
      u = reinterpret_cast<const Pack<T, VP>*>(h + 2 * j0)[0];
      v = reinterpret_cast<const Pack<T, VP>*>(h + 2 * j0)[1];
    }
  }
  __device__ __forceinline__ void store(T* h, int j0, int pairs) const {
    if constexpr (LAYOUT == KC_ROPE_HALVES) {
      *reinterpret_cast<Pack<T, VP>*>(h + j0) = u;
      *reinterpret_cast<Pack<T, VP>*>(h + pairs + j0) = v;
    } else {
      reinterpret_cast<Pack<T, VP>*>(h + 2 * j0)[0] = u;
      reinterpret_cast<Pack<T, VP>*>(h + 2 * j0)[1] = v;
    }
  }
  // element k of the 2 VP as they lie: halves: first halves then second ones; pairs: alternating
  __device__ __forceinline__ T& at(int k) { return k < VP ? u.v[k] : v.v[k - VP]; }
  __device__ __forceinline__ void get(int j, float& a, float& b) {
    a = to_f<T>(LAYOUT == KC_ROPE_HALVES ? u.v[j] : at(2 * j));
    b = to_f<T>(LAYOUT == KC_ROPE_HALVES ? v.v[j] : at(2 * j + 1));
  }
  __device__ __forceinline__ void set(int j, float a, float b) {
    if constexpr (LAYOUT == KC_ROPE_HALVES) {
      u.v[j] = from_f<T>(a);
      v.v[j] = from_f<T>(b);
    } else {
      at(2 * j) = from_f<T>(a);
      at(2 * j + 1) = from_f<T>(b);
    }
  }
};

// A thread's place: columns are (table, head lane, vector of a head: first the pairs', then the unrotated rest's),
// so that neighbouring threads read neighbouring memory of a token; the block's other threads take other tokens.
struct Place {
  int lane, table, head, col, pv;
  bool here;
};

template <int VP>
__device__ __forceinline__ Place place(const RopeParams& p) {
  Place w;
  w.pv = p.pairs / VP;
  const int cols = w.pv + p.rest / VP, column = blockIdx.y * p.width + threadIdx.x % p.width;
  w.lane = threadIdx.x / p.width;
  w.here = w.lane < p.lanes && column < p.columns;
  w.col = column % cols;
  w.head = column / cols % p.head_lanes;
  w.table = column / cols / p.head_lanes;
  return w;
}

extern __shared__ __align__(16) unsigned long long rope_smem[];

// The fractions of all frequencies into shared memory, as angles() reads them; false where they are not wanted there
// or one is not finite.
template <int VP>
__device__ __forceinline__ bool stage_freqs(const RopeParams& p) {
  if (!p.shared) return false;
  const int row = VP * p.axes, vectors = p.tables * p.pairs / VP;
  bool bad = false;
  for (int i = threadIdx.x; i < row * vectors; i += kThreads) {
    const float f = __ldg(p.freqs + i);
    rope_smem[i % row * vectors + i / row] = turn_fraction(f);
    bad = bad || !isfinite(f);
  }
  return !__syncthreads_or(bad);
}

// A thread's N heads: the addresses of its vector in each, moved from token to token. Head i of a table is one of its
// Q heads or, behind them, K heads.
template <typename T, int N, bool X>
struct HeadPtrs {
  const T* in[N];
  T* out[N];
  const T* x[X ? N : 1];
  bool is_q[N];
  int count;
  // heads first, first + head_lanes, ..; first < heads
  __device__ __forceinline__ HeadPtrs(const RopeParams& p, const Place& w, int first, int64_t t, int d) {
    const int heads = p.q.per_table + p.k.per_table;
    count = min(N, (heads - first + p.head_lanes - 1) / p.head_lanes);
#pragma unroll
    for (int k = 0; k < N; k++) {
      const int i = min(first + k * p.head_lanes, heads - 1);
      is_q[k] = i < p.q.per_table;
      const Heads& h = is_q[k] ? p.q : p.k;
      const int64_t n = (int64_t)w.table * h.per_table + (is_q[k] ? i : i - p.q.per_table);
      in[k] = static_cast<const T*>(h.in) + t * h.in_t + n * h.in_h + d;
      out[k] = static_cast<T*>(h.out) + t * h.out_t + n * h.out_h + d;
      if constexpr (X) x[k] = static_cast<const T*>(h.x) + t * h.x_t + n * h.x_h + d;
    }
  }
  __device__ __forceinline__ void next_in(const RopeParams& p, int64_t tokens) {
    const int64_t sq = p.q.in_t * tokens, sk = p.k.in_t * tokens, xq = p.q.x_t * tokens, xk = p.k.x_t * tokens;
#pragma unroll
    for (int k = 0; k < N; k++) {
      in[k] += is_q[k] ? sq : sk;
      if constexpr (X) x[k] += is_q[k] ? xq : xk;
    }
  }
  __device__ __forceinline__ void next_out(const RopeParams& p, int64_t tokens) {
    const int64_t sq = p.q.out_t * tokens, sk = p.k.out_t * tokens;
#pragma unroll
    for (int k = 0; k < N; k++) out[k] += is_q[k] ? sq : sk;
  }
};

// The unrotated rest of a thread's heads.
template <typename T, int VP, int N>
__device__ __forceinline__ void copy_rest(const RopeParams& p, const Place& w, int first, int64_t t0, int64_t step) {
  HeadPtrs<T, N, false> h(p, w, first, t0, 2 * p.pairs + (w.col - w.pv) * VP);
  for (int64_t t = t0; t < p.tokens; t += step) {
    Pack<T, VP> v[N];
#pragma unroll
    for (int k = 0; k < N; k++)
      if (k < h.count) v[k] = *reinterpret_cast<const Pack<T, VP>*>(h.in[k]);
#pragma unroll
    for (int k = 0; k < N; k++)
      if (k < h.count && h.in[k] != h.out[k]) *reinterpret_cast<Pack<T, VP>*>(h.out[k]) = v[k];
    h.next_in(p, step);
    h.next_out(p, step);
  }
}

// One vector of one head of one token to a thread, which makes its own angles: for few tokens, where a launch is
// latency, and for tables too large for shared memory. grid.x threads over (token, table, head, vector).
template <typename T, int VP, int LAYOUT>
__global__ void __launch_bounds__(kThreads) rope_axes_kernel(const __grid_constant__ RopeParams p) {
  const int heads = p.q.per_table + p.k.per_table, pv = p.pairs / VP, cols = pv + p.rest / VP;
  const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x, per_token = (int64_t)p.tables * heads * cols;
  const int64_t t = id / per_token;
  if (t >= p.tokens) return;
  const int r = (int)(id - t * per_token), col = r % cols, i = r / cols % heads, table = r / cols / heads;
  const bool is_q = i < p.q.per_table;
  const Heads& h = is_q ? p.q : p.k;
  const int64_t n = (int64_t)table * h.per_table + (is_q ? i : i - p.q.per_table);
  const T* in = static_cast<const T*>(h.in) + t * h.in_t + n * h.in_h;
  T* out = static_cast<T*>(h.out) + t * h.out_t + n * h.out_h;
  if (col >= pv) {
    const int d = 2 * p.pairs + (col - pv) * VP;
    if (in != out) *reinterpret_cast<Pack<T, VP>*>(out + d) = *reinterpret_cast<const Pack<T, VP>*>(in + d);
    return;
  }
  Pairs<T, VP, LAYOUT> x;
  x.load(in, col * VP, p.pairs);
  Position at;
  at.load(p, t);
  float c[VP], s[VP];
  angles<T, VP, false>(p, at, nullptr, 0, p.freqs + ((int64_t)table * p.pairs + col * VP) * p.axes, c, s);
#pragma unroll
  for (int j = 0; j < VP; j++) {
    float a, b;
    x.get(j, a, b);
    x.set(j, a * c[j] - b * s[j], a * s[j] + b * c[j]);
  }
  x.store(out, col * VP, p.pairs);
}

// Sine and cosine of a tile's angles into shared memory: a thread keeps an entry's (table, pair) fractions and goes
// over the tile's tokens. An entry's place: [chunk of two pairs of a vector][vector of the tile], (cos, sin) pairs, so
// that neighbouring threads read neighbouring 16-byte chunks.
template <typename T, int VP, int AXES>
__device__ __forceinline__ void tile_angles(const RopeParams& p, int64_t t0, int tokens, const unsigned long long* g,
                                            int entries, int vectors, float2* table) {
  constexpr int CH = VP < 2 ? 1 : 2;
  const int width = min(entries, kThreads), groups = kThreads / width;
  const int first = threadIdx.x % width, group = threadIdx.x / width;
  if (group >= groups) return;
  for (int e = first; e < entries; e += width) {
    unsigned long long fr[AXES];
#pragma unroll
    for (int a = 0; a < AXES; a++) fr[a] = g[a * entries + e];
    const int j = e % VP;
    float2* o = table + (j / CH * vectors + e / VP) * CH + j % CH;
    const int* pos = p.pos + t0 * AXES;
#pragma unroll 2
    for (int tt = group; tt < tokens; tt += groups) {
      unsigned long long turns = 0;
#pragma unroll
      for (int a = 0; a < AXES; a++) turns += (unsigned long long)(long long)__ldg(pos + tt * AXES + a) * fr[a];
      o[tt * (entries / VP) * CH] = turned<T>(turns);
    }
  }
}

// Tiles of tokens: the block makes the sines and cosines of a tile once, in shared memory, and then streams the
// heads through them, N heads of a table to a thread (so that a vector's sines serve N loads). Few registers and many
// blocks to an SM: one block's trigonometry runs under the others' loads and stores.
template <typename T, int VP, int LAYOUT, int N>
__global__ void __launch_bounds__(kThreads, 4) rope_axes_tile_kernel(const __grid_constant__ RopeParams p) {
  constexpr int CH = VP < 2 ? 1 : 2, CHUNKS = VP / CH;
  const int entries = p.tables * p.pairs, vectors = (entries / VP * p.tile) | 1;
  unsigned long long* g = rope_smem;  // [axes][entries]
  float2* table = reinterpret_cast<float2*>(g + entries * p.axes + (entries * p.axes & 1));
  bool bad = false;
  for (int i = threadIdx.x; i < entries * p.axes; i += kThreads) {
    const float f = __ldg(p.freqs + i);
    const unsigned long long turn = turn_fraction(f);
    g[i % p.axes * entries + i / p.axes] = p.sign < 0 ? 0 - turn : turn;
    bad = bad || !isfinite(f);
  }
  bad = __syncthreads_or(bad);
  const int heads = p.q.per_table + p.k.per_table, pv = p.pairs / VP, cols = pv + p.rest / VP;
  const int per_token = p.tables * p.rounds * cols;
  for (int64_t t0 = (int64_t)blockIdx.x * p.tile; t0 < p.tokens; t0 += (int64_t)gridDim.x * p.tile) {
    const int tokens = (int)min((int64_t)p.tile, p.tokens - t0);
    if (p.axes == 1) tile_angles<T, VP, 1>(p, t0, tokens, g, entries, vectors, table);
    else if (p.axes == 2) tile_angles<T, VP, 2>(p, t0, tokens, g, entries, vectors, table);
    else if (p.axes == 3) tile_angles<T, VP, 3>(p, t0, tokens, g, entries, vectors, table);
    else tile_angles<T, VP, 4>(p, t0, tokens, g, entries, vectors, table);
    __syncthreads();
    if (bad) {  // NaN where a frequency is not finite
      for (int i = threadIdx.x; i < tokens * entries; i += kThreads) {
        const int tt = i / entries, e = i - tt * entries, j = e % VP;
        float2* o = table + (j / CH * vectors + tt * (entries / VP) + e / VP) * CH + j % CH;
        for (int a = 0; a < p.axes; a++) {
          const float f = __ldg(p.freqs + (int64_t)e * p.axes + a);
          o->x += f - f;
          o->y += f - f;
        }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < tokens * per_token; i += kThreads) {
      const int tt = quotient(i, p.by_token), r = i - tt * per_token;
      const int tb = quotient(r, p.by_table), r2 = r - tb * (p.rounds * cols);
      const int first = quotient(r2, p.by_head), col = r2 - first * cols;
      const int64_t t = t0 + tt;
      const T* in[N];
      T* out[N];
#pragma unroll
      for (int k = 0; k < N; k++) {
        const int h = min(first + k * p.rounds, heads - 1);
        const bool is_q = h < p.q.per_table;
        const Heads& hd = is_q ? p.q : p.k;
        const int n = tb * hd.per_table + (is_q ? h : h - p.q.per_table);
        in[k] = static_cast<const T*>(hd.in) + t * hd.in_t + n * hd.in_h;
        out[k] = static_cast<T*>(hd.out) + t * hd.out_t + n * hd.out_h;
      }
      if (col >= pv) {
        const int d = 2 * p.pairs + (col - pv) * VP;
#pragma unroll
        for (int k = 0; k < N; k++)
          if (first + k * p.rounds < heads && in[k] != out[k])
            *reinterpret_cast<Pack<T, VP>*>(out[k] + d) = *reinterpret_cast<const Pack<T, VP>*>(in[k] + d);
        continue;
      }
      Pairs<T, VP, LAYOUT> x[N];
#pragma unroll
      for (int k = 0; k < N; k++)
        if (first + k * p.rounds < heads) x[k].load(in[k], col * VP, p.pairs);
      Pack<float2, CH> cs[CHUNKS];
      const int v = tt * (entries / VP) + tb * pv + col;
#pragma unroll
      for (int q = 0; q < CHUNKS; q++) cs[q] = *reinterpret_cast<const Pack<float2, CH>*>(table + (q * vectors + v) * CH);
#pragma unroll
      for (int k = 0; k < N; k++)
        if (first + k * p.rounds < heads) {
#pragma unroll
          for (int j = 0; j < VP; j++) {
            float a, b;
            x[k].get(j, a, b);
            const float2 w = cs[j / CH].v[j % CH];
            x[k].set(j, a * w.x - b * w.y, a * w.y + b * w.x);
          }
          x[k].store(out[k], col * VP, p.pairs);
        }
    }
    __syncthreads();
  }
}

// Backward with the frequencies' gradient: a thread also adds pos * d angle over its tokens in float32; the block's
// threads of one (table, pair vector) are added in order into the block's partial sums.
template <typename T, int VP, int LAYOUT, int N>
__global__ void __launch_bounds__(kThreads) rope_axes_back_kernel(const __grid_constant__ RopeParams p) {
  __shared__ float red[kThreads * VP];
  const bool staged = stage_freqs<VP>(p);
  const Place w = place<VP>(p);
  const int64_t t0 = (int64_t)blockIdx.x * p.lanes + w.lane, step = (int64_t)gridDim.x * p.lanes;
  const int j0 = w.col * VP, vectors = p.tables * w.pv;
  float acc[KC_ROPE_MAX_AXES][VP] = {};
  // a block holds all head lanes of a table (its sums are the block's), so that many heads take several rounds
  const int heads = w.here ? p.q.per_table + p.k.per_table : 0;
  for (int first = w.head; first < heads; first += N * p.head_lanes) {
    if (w.col >= w.pv) {
      copy_rest<T, VP, N>(p, w, first, t0, step);
      continue;
    }
    const unsigned long long* g = rope_smem + w.table * w.pv + w.col;
    const float* f = p.freqs + ((int64_t)w.table * p.pairs + j0) * p.axes;
    HeadPtrs<T, N, true> h(p, w, first, t0, 0);
    for (int64_t t = t0; t < p.tokens; t += step) {
      Pairs<T, VP, LAYOUT> dy[N], x[N];
#pragma unroll
      for (int k = 0; k < N; k++)
        if (k < h.count) {
          dy[k].load(h.in[k], j0, p.pairs);
          x[k].load(h.x[k], j0, p.pairs);
        }
      Position at;
      at.load(p, t);
      float c[VP], s[VP], turn[VP] = {};
      if (staged) angles<T, VP, true>(p, at, g, vectors, f, c, s);
      else angles<T, VP, false>(p, at, g, vectors, f, c, s);
#pragma unroll
      for (int k = 0; k < N; k++) {
        if (k < h.count) {
#pragma unroll
          for (int j = 0; j < VP; j++) {
            float a, b, xa, xb;
            dy[k].get(j, a, b);
            x[k].get(j, xa, xb);
            const float da = a * c[j] - b * s[j], db = a * s[j] + b * c[j];
            turn[j] += db * xa - da * xb;
            dy[k].set(j, da, db);
          }
          dy[k].store(h.out[k], j0, p.pairs);
        }
      }
#pragma unroll
      for (int a = 0; a < KC_ROPE_MAX_AXES; a++) {
        if (a >= p.axes) break;
        const float pos = (float)at.at[a];
#pragma unroll
        for (int j = 0; j < VP; j++) acc[a][j] += pos * turn[j];
      }
      h.next_in(p, step);
      h.next_out(p, step);
    }
  }
  const int cols = w.pv + p.rest / VP;
#pragma unroll
  for (int a = 0; a < KC_ROPE_MAX_AXES; a++) {
    if (a >= p.axes) break;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < VP; j++) red[j * kThreads + threadIdx.x] = acc[a][j];
    __syncthreads();
    if (w.here && w.lane == 0 && w.head == 0 && w.col < w.pv) {
      float* o = p.partial + (((int64_t)blockIdx.x * p.tables + w.table) * p.pairs + j0) * p.axes + a;
#pragma unroll
      for (int j = 0; j < VP; j++) {
        float v = 0.0f;
        for (int l = 0; l < p.lanes; l++)
          for (int h = 0; h < p.head_lanes; h++) v += red[j * kThreads + l * p.width + threadIdx.x + h * cols];
        o[(int64_t)j * p.axes] = v;
      }
    }
  }
}

// dfreqs = the blocks' partial sums, in order and in 64 bits: 8 frequencies a block, 32 lanes of blocks each.
__global__ void __launch_bounds__(kThreads) rope_freqs_kernel(const float* __restrict__ partial, int blocks, int count,
                                                              float* __restrict__ dfreqs) {
  __shared__ double red[32][8];
  const int tx = threadIdx.x & 7, ty = threadIdx.x / 8;
  const int i = blockIdx.x * 8 + tx;
  double s = 0.0;
  if (i < count)
#pragma unroll 4
    for (int b = ty; b < blocks; b += 32) s += partial[(int64_t)b * count + i];
  red[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && i < count) {
    for (int k = 1; k < 32; k++) s += red[k][tx];
    dfreqs[i] = (float)s;
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------------------------
[[noreturn]] void bad(const std::string& m) { fail(KC_ERR_INVALID, "CUDA backend: rotary positions: " + m); }

void check_desc(const kc_rope_desc* d) {
  if (!d) bad("null descriptor");
  if (d->dtype != KC_PRECISION_F32 && d->dtype != KC_PRECISION_F16 && d->dtype != KC_PRECISION_BF16)
    bad("dtype must be KC_PRECISION_F32, F16 or BF16");
  if (d->layout != KC_ROPE_HALVES && d->layout != KC_ROPE_PAIRS) bad("unknown layout");
  if (d->axes < 1 || d->axes > KC_ROPE_MAX_AXES) bad("1 to " + std::to_string(KC_ROPE_MAX_AXES) + " axes");
  if (d->tokens < 0) bad("tokens must not be negative");
  if (d->q_heads < 1 || d->k_heads < 0 || d->q_heads > 4096 || d->k_heads > 4096)
    bad("1 to 4096 q heads, 0 to 4096 k heads");
  if (d->head_dim < 2 || d->head_dim > 1024) bad("head_dim must be 2 to 1024");
  if (d->rotary_dim < 2 || d->rotary_dim % 2 != 0 || d->rotary_dim > d->head_dim)
    bad("rotary_dim must be even, 2 to head_dim");
  if (d->tables < 1 || d->q_heads % d->tables != 0 || d->k_heads % d->tables != 0)
    bad("tables must divide q_heads and k_heads");
}

Rows rows(const kc_rope_desc& d, const void* p, int heads, int64_t ts, int64_t hs) {
  return {heads ? p : nullptr, d.tokens, heads, d.head_dim, ts, hs, dtype_bytes(d.dtype)};
}
Rows q_in(const kc_rope_desc& d, const void* p) { return rows(d, p, d.q_heads, d.q_token_stride, d.q_head_stride); }
Rows k_in(const kc_rope_desc& d, const void* p) { return rows(d, p, d.k_heads, d.k_token_stride, d.k_head_stride); }
Rows q_out(const kc_rope_desc& d, const void* p) {
  return rows(d, p, d.q_heads, d.q_out_token_stride, d.q_out_head_stride);
}
Rows k_out(const kc_rope_desc& d, const void* p) {
  return rows(d, p, d.k_heads, d.k_out_token_stride, d.k_out_head_stride);
}

struct Range {
  const void* p;
  int64_t bytes;
};

// The outputs' own memory, and what each of them may meet: only its own input, in place.
void check_tensors(const kc_rope_desc& d, const Rows (&in)[2], const Rows (&out)[2], std::initializer_list<Rows> more,
                   std::initializer_list<Range> small_in, std::initializer_list<Range> small_out) {
  auto each = [&](const Rows& r) {
    if (!rows_in_range(r)) bad("strides must not be negative, nor reach past 2^46 elements");
    if (!aligned_to(r.p, r.bytes)) bad("a tensor is not aligned to its element");
  };
  for (int i = 0; i < 2; i++) {
    each(in[i]);
    each(out[i]);
    if (!rows_distinct(out[i])) bad("heads of an output share memory");
  }
  for (const Rows& r : more) each(r);
  for (const Range& r : small_in)
    if (!aligned_to(r.p, 4)) bad("positions or frequencies are not aligned to their element");
  for (int i = 0; i < 2; i++) {
    if (rows_overlap(out[i], in[i]) && !out[i].same(in[i])) bad("an output overlaps an input it does not match");
    if (rows_overlap(out[i], in[1 - i])) bad("an output overlaps the other input");
    for (const Rows& r : more)
      if (rows_overlap(out[i], r)) bad("an output overlaps an input");
    for (const Range& r : small_in)
      if (ranges_meet(r.p, r.bytes, out[i])) bad("an output overlaps the positions or frequencies");
    for (const Range& r : small_out)
      if (ranges_meet(r.p, r.bytes, out[i])) bad("an output overlaps the frequencies' gradient or the workspace");
  }
  if (rows_overlap(out[0], out[1])) bad("the outputs overlap");
  for (const Range* o = small_out.begin(); o != small_out.end(); o++) {
    bool meets = ranges_meet(o->p, o->bytes, in[0]) || ranges_meet(o->p, o->bytes, in[1]);
    for (const Rows& r : more) meets = meets || ranges_meet(o->p, o->bytes, r);
    for (const Range& r : small_in) meets = meets || ranges_meet(o->p, o->bytes, {r.p, 1, 1, r.bytes, 0, 0, r.p ? 1 : 0});
    for (const Range* q = o + 1; q != small_out.end(); q++)
      meets = meets || ranges_meet(o->p, o->bytes, {q->p, 1, 1, q->bytes, 0, 0, q->p ? 1 : 0});
    if (meets) bad("the frequencies' gradient or the workspace overlaps another tensor of the call");
  }
}

// The most neighbouring pairs a vector access can take, for every tensor of the call.
int vec_of(const kc_rope_desc& d, std::initializer_list<Rows> all) {
  const int es = dtype_bytes(d.dtype), rest = d.head_dim - d.rotary_dim;
  for (int v = 16 / es; v > 1; v /= 2) {
    bool ok = d.rotary_dim / 2 % v == 0 && rest % v == 0;
    for (const Rows& r : all) {
      if (!r.p) continue;
      ok = ok && aligned_to(r.p, (size_t)v * es) && (r.outer == 1 || r.outer_stride % v == 0) &&
           (r.inner == 1 || r.inner_stride % v == 0);
    }
    if (ok) return v;
  }
  return 1;
}

constexpr int kSms = 148;
constexpr int kMaxFreqBytes = 64 * 1024;  // of shared memory for the frequencies' fractions

// Blocks of a backward pass with the frequencies' gradient: two to an SM (registers), each with its partial sums.
int64_t back_blocks(const kc_rope_desc& d) {
  return std::min<int64_t>(kSms * 2, std::max<int64_t>(1, d.tokens));
}
size_t back_bytes(const kc_rope_desc& d) {
  if (d.tokens == 0) return 0;
  return (size_t)back_blocks(d) * d.tables * (d.rotary_dim / 2) * d.axes * sizeof(float);
}

RopeParams params(const kc_rope_desc& d, const int32_t* pos, const float* freqs, int sign) {
  RopeParams p{};
  p.pos = pos;
  p.freqs = freqs;
  p.tokens = d.tokens;
  p.axes = d.axes;
  p.pairs = d.rotary_dim / 2;
  p.rest = d.head_dim - d.rotary_dim;
  p.tables = d.tables;
  p.sign = sign;
  return p;
}

Heads heads(const Rows& in, const Rows& out, const Rows& x, int tables) {
  return {in.p, const_cast<void*>(out.p), x.p, in.outer_stride, in.inner_stride, out.outer_stride, out.inner_stride,
          x.outer_stride, x.inner_stride, (int)(in.inner / tables)};
}

unsigned grid_of(int64_t threads) {
  const int64_t b = (threads + kThreads - 1) / kThreads;
  if (b > 0x7fffffff) bad("more work than one launch takes");
  return (unsigned)b;
}

template <auto kernel>
void launch_kernel(const RopeParams& p, dim3 grid, size_t smem, cudaStream_t st) {
  if (smem > 48 * 1024) {
    static std::atomic<uint64_t> allowed[2];  // devices on which this kernel may take more than 48 KB
    int dev = 0;
    KC_CUDA(cudaGetDevice(&dev));
    if (dev >= 128) bad("device index above 127");
    if (!(allowed[dev / 64].load(std::memory_order_acquire) >> (dev % 64) & 1)) {
      KC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxFreqBytes));
      allowed[dev / 64].fetch_or(1ull << (dev % 64), std::memory_order_release);
    }
  }
  kernel<<<grid, kThreads, smem, st>>>(p);
  KC_CUDA(cudaGetLastError());
}

// n * magic >> 32 = n / d for n d < 2^32 (0 stands for d = 1)
uint32_t magic(int64_t d) { return d == 1 ? 0 : (uint32_t)(0xffffffffu / d + 1); }

template <typename T, int VP, int LAYOUT>
void launch_back(RopeParams p, cudaStream_t st) {
  const int heads = p.q.per_table + p.k.per_table, cols = p.pairs / VP + p.rest / VP;
  // a thread takes two heads of a table to its angles, one where there are too few tokens for that; the sums over a
  // table's head lanes are a block's: it holds whole tables
  const int per = p.tokens * p.tables * cols * ((heads + 1) / 2) >= kSms * 512 ? 2 : 1;
  p.head_lanes = std::min((heads + per - 1) / per, std::max(1, kThreads / cols));
  p.columns = p.tables * p.head_lanes * cols;
  p.width = std::min(p.columns, kThreads);
  if (p.head_lanes > 1) p.width = p.width / (p.head_lanes * cols) * (p.head_lanes * cols);
  p.lanes = kThreads / p.width;
  const size_t bytes = (size_t)p.tables * p.pairs * p.axes * sizeof(unsigned long long);
  p.shared = bytes <= (size_t)kMaxFreqBytes && p.tokens >= (int64_t)p.blocks * p.lanes * 4;
  launch_kernel<rope_axes_back_kernel<T, VP, LAYOUT, 2>>(
      p, dim3((unsigned)p.blocks, (unsigned)((p.columns + p.width - 1) / p.width)), p.shared ? bytes : 0, st);
  const int count = p.tables * p.pairs * p.axes;
  rope_freqs_kernel<<<(count + 7) / 8, kThreads, 0, st>>>(p.partial, p.blocks, count, p.dfreqs);
  KC_CUDA(cudaGetLastError());
}

template <typename T, int VP, int LAYOUT>
void launch(RopeParams p, cudaStream_t st) {
  if (p.dfreqs) return launch_back<T, VP, LAYOUT>(p, st);
  const int64_t heads = p.q.per_table + p.k.per_table, cols = p.pairs / VP + p.rest / VP;
  const int64_t entries = (int64_t)p.tables * p.pairs;
  // tiles of at most 32 KB of sines, not more tokens than leave every SM four blocks' work
  const int64_t fit = 32 * 1024 / (entries * 8), spread = p.tokens / (kSms * 4);
  p.tile = (int)std::max<int64_t>(1, std::min<int64_t>({fit, spread, 64}));
  const int64_t n = heads > 1 ? 2 : 1;
  p.rounds = (int)((heads + n - 1) / n);
  const int64_t per_token = (int64_t)p.tables * p.rounds * cols;
  const size_t smem = (size_t)(entries * p.axes + 1) / 2 * 16 + (size_t)((entries / VP * p.tile) | 1) * VP * 8;
  const bool small = p.tokens * p.tables * heads * cols <= kSms * 2048;  // one wave of threads
  if (small || smem > (size_t)kMaxFreqBytes || per_token * per_token * p.tile > 0xffffffffll) {
    launch_kernel<rope_axes_kernel<T, VP, LAYOUT>>(p, dim3(grid_of(p.tokens * p.tables * heads * cols)), 0, st);
    return;
  }
  p.by_token = magic(per_token);
  p.by_table = magic(p.rounds * cols);
  p.by_head = magic(cols);
  const int64_t tiles = (p.tokens + p.tile - 1) / p.tile;
  const dim3 grid((unsigned)std::min<int64_t>(tiles, kSms * 8));
  if (n == 2) launch_kernel<rope_axes_tile_kernel<T, VP, LAYOUT, 2>>(p, grid, smem, st);
  else launch_kernel<rope_axes_tile_kernel<T, VP, LAYOUT, 1>>(p, grid, smem, st);
}

template <typename T, int VP>
void launch_layout(const RopeParams& p, int layout, cudaStream_t st) {
  layout == KC_ROPE_HALVES ? launch<T, VP, KC_ROPE_HALVES>(p, st) : launch<T, VP, KC_ROPE_PAIRS>(p, st);
}

template <typename T>
void launch_type(const RopeParams& p, int layout, int vp, cudaStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (vp == 8) return launch_layout<T, 8>(p, layout, st);
  if (vp == 4) return launch_layout<T, 4>(p, layout, st);
  if (vp == 2) return launch_layout<T, 2>(p, layout, st);
  launch_layout<T, 1>(p, layout, st);
}

void run(const kc_rope_desc& d, const RopeParams& p, int vp, cudaStream_t st) {
  if (d.dtype == KC_PRECISION_F32) launch_type<float>(p, d.layout, vp, st);
  else if (d.dtype == KC_PRECISION_F16) launch_type<__half>(p, d.layout, vp, st);
  else launch_type<__nv_bfloat16>(p, d.layout, vp, st);
}

}  // namespace
}  // namespace kc

extern "C" int kc_rope_axes_freqs(int axes, const int32_t* sections, double theta, int rotary_dim, float* freqs) {
  return kc::guard_entry([&] {
    using namespace kc;
    if (!sections || !freqs) bad("null array");
    if (axes < 1 || axes > KC_ROPE_MAX_AXES) bad("1 to " + std::to_string(KC_ROPE_MAX_AXES) + " axes");
    if (rotary_dim < 2 || rotary_dim % 2 != 0) bad("rotary_dim must be even and positive");
    if (!(theta > 0.0) || !std::isfinite(theta)) bad("theta must be positive and finite");
    int64_t total = 0;
    for (int a = 0; a < axes; a++) {
      if (sections[a] < 0) bad("sections must not be negative");
      total += sections[a];
    }
    if (total != rotary_dim / 2) bad("the sections must add up to rotary_dim / 2");
    std::fill(freqs, freqs + (int64_t)(rotary_dim / 2) * axes, 0.0f);
    int j = 0;
    for (int a = 0; a < axes; a++)
      for (int i = 0; i < sections[a]; i++, j++)
        freqs[(int64_t)j * axes + a] = (float)std::pow(theta, -(double)i / (double)sections[a]);
  });
}

extern "C" int kc_rope_axes(const kc_rope_desc* desc, const void* d_q, const void* d_k, const int32_t* d_pos,
                            const float* d_freqs, void* d_q_out, void* d_k_out, void* stream) {
  return kc::guard_entry([&] {
    using namespace kc;
    check_desc(desc);
    const kc_rope_desc d = *desc;
    const bool with_k = d.k_heads > 0;
    if (d.tokens > 0 && (!d_q || !d_q_out || !d_pos || !d_freqs || (with_k && (!d_k || !d_k_out)))) bad("null tensor");
    const Rows in[2] = {q_in(d, d_q), k_in(d, d_k)}, out[2] = {q_out(d, d_q_out), k_out(d, d_k_out)};
    const Rows none{nullptr, 0, 0, 0, 0, 0, 1};
    check_tensors(d, in, out, {},
                  {{d_pos, 4 * d.tokens * d.axes}, {d_freqs, 2 * (int64_t)d.tables * d.rotary_dim * d.axes}}, {});
    if (d.tokens == 0) return;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    TensorDevice dev("rotary positions", {d_q, in[1].p, d_pos, d_freqs, d_q_out, out[1].p});
    RopeParams p = params(d, d_pos, d_freqs, 1);
    p.q = heads(in[0], out[0], none, d.tables);
    p.k = heads(in[1], out[1], none, d.tables);
    run(d, p, vec_of(d, {in[0], in[1], out[0], out[1]}), st);
  });
}

extern "C" int kc_rope_axes_backward_workspace(const kc_rope_desc* desc, size_t* bytes) {
  return kc::guard_entry([&] {
    kc::check_desc(desc);
    if (!bytes) kc::bad("null result");
    *bytes = kc::back_bytes(*desc);
  });
}

extern "C" int kc_rope_axes_backward(const kc_rope_desc* desc, const void* d_dq_out, const void* d_dk_out,
                                     const void* d_q, const void* d_k, const int32_t* d_pos, const float* d_freqs,
                                     void* d_dq, void* d_dk, float* d_dfreqs, void* d_workspace,
                                     size_t workspace_bytes, void* stream) {
  return kc::guard_entry([&] {
    using namespace kc;
    check_desc(desc);
    const kc_rope_desc d = *desc;
    const bool with_k = d.k_heads > 0;
    if (d.tokens > 0 && (!d_dq_out || !d_dq || !d_pos || !d_freqs || (with_k && (!d_dk_out || !d_dk)) ||
                         (d_dfreqs && (!d_q || (with_k && !d_k)))))
      bad("null tensor");
    const Rows none{nullptr, 0, 0, 0, 0, 0, 1};
    const Rows in[2] = {q_out(d, d_dq_out), k_out(d, d_dk_out)}, out[2] = {q_in(d, d_dq), k_in(d, d_dk)};
    const Rows x[2] = {d_dfreqs ? q_in(d, d_q) : none, d_dfreqs ? k_in(d, d_k) : none};
    const size_t need = d_dfreqs ? back_bytes(d) : 0;
    const int64_t fb = 2 * (int64_t)d.tables * d.rotary_dim * d.axes;
    check_tensors(d, in, out, {x[0], x[1]}, {{d_pos, 4 * d.tokens * d.axes}, {d_freqs, fb}},
                  {{d_dfreqs, d_dfreqs ? fb : 0}, {d_workspace, (int64_t)need}});
    if (!aligned_to(d_dfreqs, 4)) bad("the frequencies' gradient is not aligned to its element");
    if (need && (!d_workspace || workspace_bytes < need)) bad("workspace of " + std::to_string(need) + " bytes needed");
    if (need && !aligned_to(d_workspace, 16)) bad("the workspace must be 16-byte aligned");
    if (d.tokens == 0 && !d_dfreqs) return;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    TensorDevice dev("rotary positions", {in[0].p, in[1].p, out[0].p, out[1].p, x[0].p, x[1].p, d_pos, d_freqs,
                                          d_dfreqs, need ? d_workspace : nullptr});
    if (d.tokens == 0) {
      KC_CUDA(cudaMemsetAsync(d_dfreqs, 0, (size_t)fb, st));
      return;
    }
    RopeParams p = params(d, d_pos, d_freqs, -1);
    p.q = heads(in[0], out[0], x[0], d.tables);
    p.k = heads(in[1], out[1], x[1], d.tables);
    p.dfreqs = d_dfreqs;
    p.partial = static_cast<float*>(d_workspace);
    p.blocks = (int)back_blocks(d);
    run(d, p, vec_of(d, {in[0], in[1], out[0], out[1], x[0], x[1]}), st);
  });
}
