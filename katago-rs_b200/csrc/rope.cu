// Rotary positions with several axes on Q and K heads, forward and backward (kc_rope_axes, kc_rope_axes_backward).
//
//   angle[t][tb][j] = sum_a pos[t][a] freqs[tb][j][a], (y1, y2) = (x1 cos - x2 sin, x1 sin + x2 cos)
//   backward: dx = the gradient turned by -angle; d angle = dx2 x1 - dx1 x2;
//   dfreqs[tb][j][a] = sum_t pos[t][a] sum over the table's heads of d angle
//
// Angles are held in turns, as 64-bit fractions: a frequency is freq / (2 pi) mod 1 scaled by 2^64 (from float64, so
// 53 bits of freq / (2 pi)), and whole turns of pos * frequency drop out of the 64-bit product by themselves. The
// error is that of freq / (2 pi), 2^-53 of the angle; far positions keep their digits, at two integer multiply-adds
// an axis (float64 angles reduced with rint were 3 to 4 times the instructions).
//
// What bounds it: HBM for a table shared by all heads; with a table per key head the angles (17.7 million for 256
// boards, about 28 instructions each) take as long as the transfers. Measured on a B200 (6,554 GB/s copy), bytes that
// have to move / time:
//   256 boards x 361 tokens, 6 + 6 heads of 64, f16: 284 MB in 53.7 us (5,300 GB/s) with one table, in 66.9 us
//     (4,255 GB/s) with a table per key head; a thread per pair vector with its own float64 angles: 86 us
//   57,767 tokens, 16 + 4 heads of 128, 96 of them turned, 3 axes, bf16: 592 MB in 119.5 us, 4,960 GB/s
//   backward with the frequencies' gradient, 34,656 tokens, 12 + 4 heads of 64, 4 tables, bf16: 213 MB in 55.9 us,
//     3,810 GB/s: 24 warps to an SM (80 registers), most of the time waiting for their loads; 1.6 us of it are the
//     sines of a float32 result
//   backward without it, 4,099 tokens, 12 + 12 heads of 64, float32: 50 MB in 11.9 us

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <string>

#include "../../include/katago_cuda.h"
#include "gemm_pair.cuh"
#include "ops_common.h"

namespace kc {
namespace {

constexpr int kThreads = 256;
// Blocks of the tile kernels to an SM, forward and backward with the frequencies' gradient (registers).
constexpr int kTileBlocks = 3, kBackBlocks = 3;

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
  int width, lanes;               // a block's columns (table, head i mod rounds, vector of a head) and tokens at once
  int columns;                    // of all blocks y
  float* partial;                 // [blocks][tables][pairs][axes]
  float* dfreqs;
  int blocks;
};

template <typename T, int N>
struct alignas(N * sizeof(T)) Pack {
  T v[N];
};

// freq / (2 pi) mod 1, times 2^64. The distance from the nearest whole turn, exact in float64, keeps the digits of a
// small frequency of either sign (from the turn below, a negative one's would be 1 less them). Half a turn saturates
// to 2^-64 below it. A frequency that is not finite gives no angle; its sines are made NaN apart.
__device__ __forceinline__ unsigned long long turn_fraction(float freq) {
  const double t = (double)freq * 0.15915494309189533577;  // 1 / (2 pi)
  return (unsigned long long)__double2ll_rz((t - rint(t)) * 18446744073709551616.0);
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

// (cos, sin) of an angle of turns * 2^-64, for results of T. 2-byte results take the fast functions on half a turn
// either way (off by 2^-21, far below the rounding). float32 ones, the frequencies' gradient among them whatever the
// heads' type, take polynomials in an eighth of a turn either way from the nearest quarter, y = 8 angle / turn:
// sin(y pi / 4) = y (pi / 4 + y^2 P(y^2)), cos(y pi / 4) = 1 + y^2 Q(y^2), P and Q with the least largest error (2e-9
// and 5e-11 of the result, by weighted least squares), pi / 4 in two floats. Off by at most 7.5e-8.
template <typename T>
__device__ __forceinline__ float2 turned(unsigned long long turns) {
  const uint32_t part = (uint32_t)(turns >> 32);  // in 2^-32 turns
  float2 r;
  if constexpr (sizeof(T) == 4) {
    const uint32_t q = part + 0x20000000u;  // the nearest quarter in the upper two bits
    const float y = (float)(int)(part - (q & 0xc0000000u)) * 0x1p-29f, z = y * y;
    float u = fmaf(z, -3.59389829e-05f, 2.48998965e-03f);
    u = fmaf(u, z, -8.07454347e-02f);
    u = fmaf(u, z, -2.18556941e-08f);
    float v = fmaf(z, 3.53132860e-06f, -3.25941998e-04f);
    v = fmaf(v, z, 1.58543277e-02f);
    v = fmaf(v, z, -3.08425136e-01f);
    u = fmaf(y, 0.785398185f, y * u);
    v = fmaf(v, z, 1.0f);
    const bool odd = q & 0x40000000u;
    r.x = __uint_as_float(__float_as_uint(odd ? u : v) ^ ((q + 0x40000000u) & 0x80000000u));
    r.y = __uint_as_float(__float_as_uint(odd ? v : u) ^ (q & 0x80000000u));
  } else {
    const float x = (float)(int)part * 1.4629180792671596e-09f;  // 2 pi 2^-32
    r.x = cos_fast(x);
    r.y = sin_fast(x);
  }
  return r;
}

// sin and cos of VP pairs' angles at one token, from the frequencies `f`.
template <typename T, int VP>
__device__ __forceinline__ void angles(const RopeParams& p, int64_t t, const float* f, float (&c)[VP], float (&s)[VP]) {
  long long pos[KC_ROPE_MAX_AXES];
#pragma unroll
  for (int a = 0; a < KC_ROPE_MAX_AXES; a++)
    pos[a] = a < p.axes ? (long long)__ldg(p.pos + t * p.axes + a) * p.sign : 0;
#pragma unroll
  for (int j = 0; j < VP; j++) {
    unsigned long long turns = 0;
    float bad = 0.0f;  // NaN where a frequency is not finite
#pragma unroll
    for (int a = 0; a < KC_ROPE_MAX_AXES; a++)
      if (a < p.axes) {
        const float fr = __ldg(f + j * p.axes + a);
        bad += fr - fr;
        turns += (unsigned long long)pos[a] * turn_fraction(fr);
      }
    const float2 cs = turned<T>(turns);
    c[j] = cs.x + bad;
    s[j] = cs.y + bad;
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
  // pairs j and j + 1 (j even; where a vector has one pair the second is 0)
  __device__ __forceinline__ void get2(int j, f32x2& a, f32x2& b) {
    float a0, b0, a1 = 0.0f, b1 = 0.0f;
    get(j, a0, b0);
    if (VP > 1) get(j + 1, a1, b1);
    a = {a0, a1};
    b = {b0, b1};
  }
  __device__ __forceinline__ void set2(int j, f32x2 a, f32x2 b) {
    set(j, a.x, b.x);
    if (VP > 1) set(j + 1, a.y, b.y);
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

// (a, b) turned: a c - b s, a s + b c, two pairs at once, with the same roundings in every kernel: one token at a
// time gives the bits of the whole sequence.
__device__ __forceinline__ void turn2(f32x2& a, f32x2& b, f32x2 c, f32x2 s) {
  const f32x2 ya = fma2({-b.x, -b.y}, s, mul2(a, c));
  b = fma2(a, s, mul2(b, c));
  a = ya;
}

// One vector of one head of one token to a thread, which makes its own angles: for few tokens, where a launch is
// latency, and for what the tiles cannot take. Threads over (token, table, head, vector). S: the type that the sines
// are good for.
template <typename T, int VP, int LAYOUT, typename S>
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
  float c[VP], s[VP];
  angles<S, VP>(p, t, p.freqs + ((int64_t)table * p.pairs + col * VP) * p.axes, c, s);
#pragma unroll
  for (int j = 0; j < VP; j += 2) {
    f32x2 a, b;
    x.get2(j, a, b);
    if constexpr (VP > 1) turn2(a, b, {c[j], c[j + 1]}, {s[j], s[j + 1]});
    else turn2(a, b, {c[j], 0.0f}, {s[j], 0.0f});
    x.set2(j, a, b);
  }
  x.store(out, col * VP, p.pairs);
}

// ---------------------------------------------------------------------------------------------------------------
// Tiles of tokens. A block makes the sines and cosines of a tile's (token, table, pair) entries once, in shared
// memory, and then streams the heads through them, two heads of a table to a thread, so that a vector's sines serve
// two loads. Several blocks to an SM: one's trigonometry runs under the others' loads and stores.
// ---------------------------------------------------------------------------------------------------------------
extern __shared__ __align__(16) unsigned char rope_smem[];

// A head's first vector at token 0 and the bytes from token to token.
struct alignas(16) HeadAddr {
  const char* in;
  char* out;
  const char* x;
  uint32_t in_step, out_step;
};

// A tile's shared memory: the heads [tables][heads], the frequencies' fractions [axes][entries], the phase of the
// positions' bias [entries], the tile's positions [tokens][axes], and the sines: [chunk of two pairs of a vector]
// [vector of the tile] (cos, cos, sin, sin), so that neighbouring threads read neighbouring 16-byte chunks.
template <int VP>
struct Tile {
  static constexpr int CH = VP < 2 ? 1 : 2, CHUNKS = VP / CH;
  unsigned long long *fraction, *bias;
  HeadAddr* heads;
  uint32_t* pos;
  float* sines;
  int entries, vectors;
  __host__ __device__ static size_t bytes(int64_t entries, int axes, int64_t heads, int64_t tile) {
    return (size_t)heads * sizeof(HeadAddr) + (size_t)((entries * (axes + 1) + 1) / 2 * 16) +
           (size_t)((tile * axes + 3) / 4 * 16) + (size_t)((entries / VP * tile) | 1) * VP * 8;
  }
  __device__ __forceinline__ explicit Tile(const RopeParams& p) {
    entries = p.tables * p.pairs;
    vectors = (entries / VP * p.tile) | 1;
    heads = reinterpret_cast<HeadAddr*>(rope_smem);
    fraction = reinterpret_cast<unsigned long long*>(heads + p.tables * (p.q.per_table + p.k.per_table));
    bias = fraction + entries * p.axes;
    pos = reinterpret_cast<uint32_t*>(fraction + (entries * (p.axes + 1) + 1) / 2 * 2);
    sines = reinterpret_cast<float*>(pos + (p.tile * p.axes + 3) / 4 * 4);
  }
  // an entry's cosine in the tile (its sine is CH floats behind), and what the next token adds
  __device__ __forceinline__ float* at(int e) const {
    return sines + ((size_t)(e % VP / CH) * vectors + e / VP) * (2 * CH) + e % CH;
  }
  __device__ __forceinline__ int per_token() const { return entries / VP * (2 * CH); }
  __device__ __forceinline__ void read(int vector, f32x2 (&c)[(VP + 1) / 2], f32x2 (&s)[(VP + 1) / 2]) const {
#pragma unroll
    for (int q = 0; q < CHUNKS; q++) {
      const float* chunk = sines + ((size_t)q * vectors + vector) * (2 * CH);
      const Pack<float, 2 * CH> v = *reinterpret_cast<const Pack<float, 2 * CH>*>(chunk);
      c[q] = {v.v[0], CH == 2 ? v.v[1] : 0.0f};
      s[q] = {v.v[CH], CH == 2 ? v.v[CH + 1] : 0.0f};
    }
  }
};

// A tile's positions, as unsigned numbers 2^31 higher (fewer steps in the 64-bit product); the bias takes that out.
template <int VP>
__device__ __forceinline__ void tile_positions(const RopeParams& p, const Tile<VP>& tile, int64_t t0) {
  if (t0 >= p.tokens) return;
  const int n = (int)min((int64_t)p.tile, p.tokens - t0) * p.axes;
  for (int i = threadIdx.x; i < n; i += kThreads) tile.pos[i] = (uint32_t)__ldg(p.pos + t0 * p.axes + i) ^ 0x80000000u;
}

// Once per block, with the first tile's positions. False where a frequency is not finite.
template <typename T, int VP>
__device__ __forceinline__ bool tile_setup(const RopeParams& p, const Tile<VP>& tile) {
  tile_positions<VP>(p, tile, (int64_t)blockIdx.x * p.tile);
  bool bad = false;
  for (int e = threadIdx.x; e < tile.entries; e += kThreads) {
    unsigned long long sum = 0;
    for (int a = 0; a < p.axes; a++) {
      const float f = __ldg(p.freqs + (int64_t)e * p.axes + a);
      const unsigned long long turn = turn_fraction(f);
      tile.fraction[a * tile.entries + e] = p.sign < 0 ? 0 - turn : turn;
      sum += tile.fraction[a * tile.entries + e];
      bad = bad || !isfinite(f);
    }
    tile.bias[e] = 0 - (sum << 31);
  }
  const int per = p.q.per_table + p.k.per_table;
  for (int i = threadIdx.x; i < p.tables * per; i += kThreads) {
    const int table = i / per, h = i - table * per;
    const bool is_q = h < p.q.per_table;
    const Heads& hd = is_q ? p.q : p.k;
    const int64_t n = (int64_t)table * hd.per_table + (is_q ? h : h - p.q.per_table);
    HeadAddr& o = tile.heads[i];
    o.in = reinterpret_cast<const char*>(static_cast<const T*>(hd.in) + n * hd.in_h);
    o.out = reinterpret_cast<char*>(static_cast<T*>(hd.out) + n * hd.out_h);
    o.x = reinterpret_cast<const char*>(static_cast<const T*>(hd.x) + n * hd.x_h);
    o.in_step = (uint32_t)(hd.in_t * sizeof(T));
    o.out_step = (uint32_t)(hd.out_t * sizeof(T));
  }
  return !__syncthreads_or(bad);
}

// The tile's sines: a thread keeps an entry's fractions and goes over the tokens.
template <typename T, int VP, int AXES>
__device__ __forceinline__ void tile_angles(const Tile<VP>& tile, int tokens) {
  const int width = min(tile.entries, kThreads), groups = kThreads / width;
  const int first = threadIdx.x % width, group = threadIdx.x / width;
  if (group >= groups) return;
  const int step = tile.per_token() * groups;
  for (int e = first; e < tile.entries; e += width) {
    uint32_t lo[AXES], hi[AXES];
#pragma unroll
    for (int a = 0; a < AXES; a++) {
      const unsigned long long f = tile.fraction[a * tile.entries + e];
      lo[a] = (uint32_t)f;
      hi[a] = (uint32_t)(f >> 32);
    }
    const unsigned long long bias = tile.bias[e];
    float* o = tile.at(e) + tile.per_token() * group;
    const uint32_t* pos = tile.pos + group * AXES;
#pragma unroll 4
    for (int tt = group; tt < tokens; tt += groups, o += step, pos += groups * AXES) {
      unsigned long long turns = bias;
      uint32_t high = 0;
#pragma unroll
      for (int a = 0; a < AXES; a++) {
        turns += (unsigned long long)pos[a] * lo[a];
        high += pos[a] * hi[a];
      }
      const float2 cs = turned<T>(turns + ((unsigned long long)high << 32));
      o[0] = cs.x;
      o[Tile<VP>::CH] = cs.y;
    }
  }
}

template <typename T, int VP>
__device__ __forceinline__ void tile_sines(const RopeParams& p, const Tile<VP>& tile, int64_t t0, int tokens,
                                           bool finite) {
  if (p.axes == 1) tile_angles<T, VP, 1>(tile, tokens);
  else if (p.axes == 2) tile_angles<T, VP, 2>(tile, tokens);
  else if (p.axes == 3) tile_angles<T, VP, 3>(tile, tokens);
  else tile_angles<T, VP, 4>(tile, tokens);
  __syncthreads();
  tile_positions<VP>(p, tile, t0 + (int64_t)gridDim.x * p.tile);  // the next tile's, seen after the tile's last barrier
  if (finite) return;
  for (int i = threadIdx.x; i < tokens * tile.entries; i += kThreads) {  // NaN where a frequency is not finite
    const int tt = i / tile.entries, e = i - tt * tile.entries;
    float* o = tile.at(e) + tile.per_token() * tt;
    for (int a = 0; a < p.axes; a++) {
      const float f = __ldg(p.freqs + (int64_t)e * p.axes + a);
      o[0] += f - f;
      o[Tile<VP>::CH] += f - f;
    }
  }
  __syncthreads();
}

template <typename T, int VP, int LAYOUT>
__global__ void __launch_bounds__(kThreads, kTileBlocks) rope_axes_tile_kernel(const __grid_constant__ RopeParams p) {
  using P = Pairs<T, VP, LAYOUT>;
  constexpr int N = 2, NP = (VP + 1) / 2;
  const Tile<VP> tile(p);
  const bool finite = tile_setup<T, VP>(p, tile);
  const int heads = p.q.per_table + p.k.per_table, pv = p.pairs / VP, cols = pv + p.rest / VP;
  const int per_token = p.tables * p.rounds * cols;
  for (int64_t t0 = (int64_t)blockIdx.x * p.tile; t0 < p.tokens; t0 += (int64_t)gridDim.x * p.tile) {
    const int tokens = (int)min((int64_t)p.tile, p.tokens - t0);
    tile_sines<T, VP>(p, tile, t0, tokens, finite);
    for (int i = threadIdx.x; i < tokens * per_token; i += kThreads) {
      const int tt = quotient(i, p.by_token), r = i - tt * per_token;
      const int table = quotient(r, p.by_table), r2 = r - table * (p.rounds * cols);
      const int first = quotient(r2, p.by_head), col = r2 - first * cols;
      const uint32_t t = (uint32_t)t0 + tt;
      const HeadAddr* h = tile.heads + table * heads + first;
      const bool two = first + p.rounds < heads;
      const char* in[N] = {h->in + (uint64_t)t * h->in_step, nullptr};
      char* out[N] = {h->out + (uint64_t)t * h->out_step, nullptr};
      if (two) {
        h += p.rounds;
        in[1] = h->in + (uint64_t)t * h->in_step;
        out[1] = h->out + (uint64_t)t * h->out_step;
      }
      if (col >= pv) {
        const uint32_t d = (2 * p.pairs + (col - pv) * VP) * sizeof(T);
        Pack<T, VP> v[N];
#pragma unroll
        for (int k = 0; k < N; k++)
          if (k == 0 || two) v[k] = *reinterpret_cast<const Pack<T, VP>*>(in[k] + d);
#pragma unroll
        for (int k = 0; k < N; k++)
          if ((k == 0 || two) && in[k] != out[k]) *reinterpret_cast<Pack<T, VP>*>(out[k] + d) = v[k];
        continue;
      }
      P x[N];
#pragma unroll
      for (int k = 0; k < N; k++)
        if (k == 0 || two) x[k].load(reinterpret_cast<const T*>(in[k]), col * VP, p.pairs);
      f32x2 c[NP], s[NP];
      tile.read(tt * (tile.entries / VP) + table * pv + col, c, s);
#pragma unroll
      for (int k = 0; k < N; k++)
        if (k == 0 || two) {
#pragma unroll
          for (int j = 0; j < NP; j++) {
            f32x2 a, b;
            x[k].get2(2 * j, a, b);
            turn2(a, b, c[j], s[j]);
            x[k].set2(2 * j, a, b);
          }
          x[k].store(reinterpret_cast<T*>(out[k]), col * VP, p.pairs);
        }
    }
    __syncthreads();
  }
}

// Backward with the frequencies' gradient: a thread keeps one column (table, head i mod rounds, pair vector) and goes
// over tokens; it adds pos * d angle in float32, and the block's threads of one (table, pair vector) are added in
// order into the block's partial sums. `rounds` threads share a table's heads: head h, h + rounds, ... to one.
template <typename T, int VP, int LAYOUT, int AXES>  // AXES: at most
__global__ void __launch_bounds__(kThreads, kBackBlocks) rope_axes_back_kernel(const __grid_constant__ RopeParams p) {
  using P = Pairs<T, VP, LAYOUT>;
  constexpr int NP = (VP + 1) / 2;
  __shared__ float red[kThreads * VP];
  const Tile<VP> tile(p);
  const bool finite = tile_setup<T, VP>(p, tile);
  const int heads = p.q.per_table + p.k.per_table, pv = p.pairs / VP, cols = pv + p.rest / VP;
  const int column = blockIdx.y * p.width + threadIdx.x % p.width, lane = threadIdx.x / p.width;
  const bool here = lane < p.lanes && column < p.columns;
  const int col = column % cols, first = column / cols % p.rounds, table = here ? column / cols / p.rounds : 0;
  f32x2 acc[AXES][NP] = {};
  for (int64_t t0 = (int64_t)blockIdx.x * p.tile; t0 < p.tokens; t0 += (int64_t)gridDim.x * p.tile) {
    const int tokens = (int)min((int64_t)p.tile, p.tokens - t0);
    tile_sines<float, VP>(p, tile, t0, tokens, finite);
    for (int tt = lane; here && tt < tokens; tt += p.lanes) {
      const uint32_t t = (uint32_t)t0 + tt;
      if (col >= pv) {
        const uint32_t d = (2 * p.pairs + (col - pv) * VP) * sizeof(T);
        for (int i = first; i < heads; i += p.rounds) {
          const HeadAddr& h = tile.heads[table * heads + i];
          const char* in = h.in + (uint64_t)t * h.in_step;
          char* out = h.out + (uint64_t)t * h.out_step;
          if (in != out) *reinterpret_cast<Pack<T, VP>*>(out + d) = *reinterpret_cast<const Pack<T, VP>*>(in + d);
        }
        continue;
      }
      f32x2 c[NP], s[NP], turn[NP] = {};
      tile.read(tt * (tile.entries / VP) + table * pv + col, c, s);
      constexpr int N = 2;  // heads in flight
      for (int i = first; i < heads; i += N * p.rounds) {
        const HeadAddr* h = tile.heads + table * heads + i;
        const bool two = i + p.rounds < heads;
        P dy[N], x[N];
#pragma unroll
        for (int k = 0; k < N; k++)
          if (k == 0 || two) {
            // x lies at the gradient's strides
            const HeadAddr& hk = h[k * p.rounds];
            dy[k].load(reinterpret_cast<const T*>(hk.in + (uint64_t)t * hk.in_step), col * VP, p.pairs);
            x[k].load(reinterpret_cast<const T*>(hk.x + (uint64_t)t * hk.out_step), col * VP, p.pairs);
          }
#pragma unroll
        for (int k = 0; k < N; k++)
          if (k == 0 || two) {
#pragma unroll
            for (int j = 0; j < NP; j++) {
              f32x2 a, b, xa, xb;
              dy[k].get2(2 * j, a, b);
              x[k].get2(2 * j, xa, xb);
              turn2(a, b, c[j], s[j]);
              turn[j] = fma2(b, xa, fma2({-a.x, -a.y}, xb, turn[j]));
              dy[k].set2(2 * j, a, b);
            }
            const HeadAddr& hk = h[k * p.rounds];
            dy[k].store(reinterpret_cast<T*>(hk.out + (uint64_t)t * hk.out_step), col * VP, p.pairs);
          }
      }
#pragma unroll
      for (int a = 0; a < AXES; a++) {
        if (a >= p.axes) break;
        const float pos = (float)__ldg(p.pos + (int64_t)t * p.axes + a);
#pragma unroll
        for (int j = 0; j < NP; j++) acc[a][j] = fma2(f32x2{pos, pos}, turn[j], acc[a][j]);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int a = 0; a < AXES; a++) {
    if (a >= p.axes) break;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < VP; j++) red[j * kThreads + threadIdx.x] = j % 2 ? acc[a][j / 2].y : acc[a][j / 2].x;
    __syncthreads();
    if (here && lane == 0 && first == 0 && col < pv) {
      float* o = p.partial + (((int64_t)blockIdx.x * p.tables + table) * p.pairs + col * VP) * p.axes + a;
#pragma unroll
      for (int j = 0; j < VP; j++) {
        float v = 0.0f;
        for (int l = 0; l < p.lanes; l++)
          for (int h = 0; h < p.rounds; h++) v += red[j * kThreads + l * p.width + threadIdx.x + h * cols];
        o[(int64_t)j * p.axes] = v;
      }
    }
  }
}

// The frequencies' gradient alone, for what the tiles cannot take (tables too large for shared memory, steps past 32
// bits): a thread per (table, pair) entry, blocks x share the tokens.
template <typename T, int LAYOUT>
__global__ void __launch_bounds__(kThreads) rope_freqs_direct_kernel(const __grid_constant__ RopeParams p) {
  const int e = blockIdx.y * kThreads + threadIdx.x;
  if (e >= p.tables * p.pairs) return;
  const int table = e / p.pairs, j = e - table * p.pairs;
  float acc[KC_ROPE_MAX_AXES] = {};
  for (int64_t t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    float c[1], s[1], turn = 0.0f;
    angles<float, 1>(p, t, p.freqs + (int64_t)e * p.axes, c, s);
    for (int i = 0; i < p.q.per_table + p.k.per_table; i++) {
      const bool is_q = i < p.q.per_table;
      const Heads& h = is_q ? p.q : p.k;
      const int64_t n = (int64_t)table * h.per_table + (is_q ? i : i - p.q.per_table);
      Pairs<T, 1, LAYOUT> dy, x;
      dy.load(static_cast<const T*>(h.in) + t * h.in_t + n * h.in_h, j, p.pairs);
      x.load(static_cast<const T*>(h.x) + t * h.x_t + n * h.x_h, j, p.pairs);
      float a, b, xa, xb;
      dy.get(0, a, b);
      x.get(0, xa, xb);
      turn += (a * s[0] + b * c[0]) * xa - (a * c[0] - b * s[0]) * xb;
    }
#pragma unroll
    for (int a = 0; a < KC_ROPE_MAX_AXES; a++)
      if (a < p.axes) acc[a] += (float)__ldg(p.pos + t * p.axes + a) * turn;
  }
#pragma unroll
  for (int a = 0; a < KC_ROPE_MAX_AXES; a++)
    if (a < p.axes) p.partial[((int64_t)blockIdx.x * p.tables * p.pairs + e) * p.axes + a] = acc[a];
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
  if (d->tokens < 0 || d->tokens > (int64_t)1 << 46) bad("tokens must be 0 to 2^46");
  if (d->q_heads < 1 || d->k_heads < 0 || d->q_heads > 4096 || d->k_heads > 4096)
    bad("1 to 4096 q heads, 0 to 4096 k heads");
  if (d->head_dim < 2 || d->head_dim > 1024) bad("head_dim must be 2 to 1024");
  if (d->rotary_dim < 2 || d->rotary_dim % 2 != 0 || d->rotary_dim > d->head_dim)
    bad("rotary_dim must be even, 2 to head_dim");
  if (d->tables < 1 || d->q_heads % d->tables != 0 || d->k_heads % d->tables != 0)
    bad("tables must divide q_heads and k_heads");
}

Rows rows(const kc_rope_desc& d, const void* p, int heads, int64_t ts, int64_t hs) {
  if (!heads) return {nullptr, d.tokens, 0, d.head_dim, 0, 0, dtype_bytes(d.dtype)};
  return {p, d.tokens, heads, d.head_dim, ts, hs, dtype_bytes(d.dtype)};
}
Rows q_in(const kc_rope_desc& d, const void* p) { return rows(d, p, d.q_heads, d.q_token_stride, d.q_head_stride); }
Rows k_in(const kc_rope_desc& d, const void* p) { return rows(d, p, d.k_heads, d.k_token_stride, d.k_head_stride); }
Rows q_out(const kc_rope_desc& d, const void* p) {
  return rows(d, p, d.q_heads, d.q_out_token_stride, d.q_out_head_stride);
}
Rows k_out(const kc_rope_desc& d, const void* p) {
  return rows(d, p, d.k_heads, d.k_out_token_stride, d.k_out_head_stride);
}

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
      if (ranges_meet(r, out[i])) bad("an output overlaps the positions or frequencies");
    for (const Range& r : small_out)
      if (ranges_meet(r, out[i])) bad("an output overlaps the frequencies' gradient or the workspace");
  }
  if (rows_overlap(out[0], out[1])) bad("the outputs overlap");
  for (const Range* o = small_out.begin(); o != small_out.end(); o++) {
    bool meets = ranges_meet(*o, in[0]) || ranges_meet(*o, in[1]);
    for (const Rows& r : more) meets = meets || ranges_meet(*o, r);
    for (const Range& r : small_in) meets = meets || ranges_meet(*o, r);
    for (const Range* q = o + 1; q != small_out.end(); q++)
      meets = meets || ranges_meet(*o, *q);
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
constexpr int kMaxTileBytes = 100 * 1024;  // of shared memory a block of the tile kernels

// Blocks of a backward pass with the frequencies' gradient, each with its partial sums: as many as the SMs hold.
int64_t back_blocks(const kc_rope_desc& d) {
  return std::min<int64_t>(kSms * kBackBlocks, std::max<int64_t>(1, d.tokens));
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

// The strides of one token and of one head, which no address needs, are 0.
Heads heads(const Rows& in, const Rows& out, const Rows& x, int tables) {
  auto token = [](const Rows& r) { return r.outer > 1 ? r.outer_stride : 0; };
  auto head = [](const Rows& r) { return r.inner > 1 ? r.inner_stride : 0; };
  return {in.p, const_cast<void*>(out.p), x.p, token(in), head(in), token(out), head(out), token(x), head(x),
          (int)(in.inner / tables)};
}

unsigned grid_of(int64_t threads) {
  const int64_t b = (threads + kThreads - 1) / kThreads;
  if (b > 0x7fffffff) bad("more work than one launch takes");
  return (unsigned)b;
}

template <auto kernel>
void launch_kernel(const RopeParams& p, dim3 grid, size_t smem, cudaStream_t st) {
  if (smem > 0) {  // what a block gets unasked, 48 KB, has to hold the kernel's own shared memory too
    static std::atomic<uint64_t> allowed[2];  // devices on which this kernel may take more
    int dev = 0;
    KC_CUDA(cudaGetDevice(&dev));
    if (dev >= 128) bad("device index above 127");
    if (!(allowed[dev / 64].load(std::memory_order_acquire) >> (dev % 64) & 1)) {
      KC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxTileBytes));
      allowed[dev / 64].fetch_or(1ull << (dev % 64), std::memory_order_release);
    }
  }
  kernel<<<grid, kThreads, smem, st>>>(p);
  KC_CUDA(cudaGetLastError());
}

// n * magic >> 32 = n / d for n d < 2^32 (0 stands for d = 1)
uint32_t magic(int64_t d) { return d == 1 ? 0 : (uint32_t)(0xffffffffu / d + 1); }

// Tokens of a tile, at most `most` (32 KB of sines): every block gets the same number of tiles.
int tile_tokens(int64_t tokens, int64_t blocks, int64_t most) {
  const int64_t share = (tokens + blocks - 1) / blocks, cap = std::max<int64_t>(1, most);
  const int64_t tiles = (share + cap - 1) / cap;
  return (int)((share + tiles - 1) / tiles);
}

// Steps the tile kernels can index with: a token's in 32 bits of bytes, tokens in 32 bits.
bool small_steps(const RopeParams& p, int64_t es) {
  const int64_t most = std::max({p.q.in_t, p.q.out_t, p.q.x_t, p.k.in_t, p.k.out_t, p.k.x_t});
  return p.tokens <= 0x7fffffff && most * es <= 0xffffffffll;
}

// Backward with the frequencies' gradient: the columns of a block. A thread takes two heads of a table or more: the
// sums over the threads that share a table's heads are a block's, so that it holds whole tables.
template <typename T, int VP, int LAYOUT>
void launch_back(RopeParams p, cudaStream_t st) {
  const int heads = p.q.per_table + p.k.per_table, cols = p.pairs / VP + p.rest / VP;
  p.rounds = std::min((heads + 1) / 2, std::max(1, kThreads / cols));
  p.columns = p.tables * p.rounds * cols;
  p.width = std::min(p.columns, kThreads);
  if (p.rounds > 1) p.width = p.width / (p.rounds * cols) * (p.rounds * cols);
  p.lanes = kThreads / p.width;
  const int64_t entries = (int64_t)p.tables * p.pairs;
  auto bytes = [&](int64_t tile) { return Tile<VP>::bytes(entries, p.axes, (int64_t)p.tables * heads, tile); };
  p.tile = tile_tokens(p.tokens, p.blocks, std::min<int64_t>(64, 32 * 1024 / (entries * 8)));
  if (bytes(p.tile) <= (size_t)kMaxTileBytes && small_steps(p, sizeof(T))) {
    const dim3 grid((unsigned)p.blocks, (unsigned)((p.columns + p.width - 1) / p.width));
    if (p.axes <= 2) launch_kernel<rope_axes_back_kernel<T, VP, LAYOUT, 2>>(p, grid, bytes(p.tile), st);
    else launch_kernel<rope_axes_back_kernel<T, VP, LAYOUT, KC_ROPE_MAX_AXES>>(p, grid, bytes(p.tile), st);
  } else {  // before the gradients, which may take the place of what it reads
    launch_kernel<rope_freqs_direct_kernel<T, LAYOUT>>(
        p, dim3((unsigned)p.blocks, (unsigned)((entries + kThreads - 1) / kThreads)), 0, st);
    launch_kernel<rope_axes_kernel<T, VP, LAYOUT, float>>(p, dim3(grid_of(p.tokens * p.tables * heads * cols)), 0, st);
  }
  const int count = p.tables * p.pairs * p.axes;
  rope_freqs_kernel<<<(count + 7) / 8, kThreads, 0, st>>>(p.partial, p.blocks, count, p.dfreqs);
  KC_CUDA(cudaGetLastError());
}

template <typename T, int VP, int LAYOUT>
void launch(RopeParams p, cudaStream_t st) {
  // backward 8-byte vectors, whose registers let three blocks run on an SM: 55.4 us against 72.3 us with 16 bytes and
  // two blocks (34,656 tokens, 12 + 4 heads of 64, bf16)
  if (p.dfreqs) return launch_back<T, VP == 8 ? 4 : VP, LAYOUT>(p, st);
  const int64_t heads = p.q.per_table + p.k.per_table, cols = p.pairs / VP + p.rest / VP;
  const int64_t entries = (int64_t)p.tables * p.pairs;
  p.tile = tile_tokens(p.tokens, kSms * kTileBlocks, std::min<int64_t>(32, 32 * 1024 / (entries * 8)));
  p.rounds = (int)((heads + 1) / 2);
  const int64_t per_token = (int64_t)p.tables * p.rounds * cols;
  const size_t smem = Tile<VP>::bytes(entries, p.axes, p.tables * heads, p.tile);
  const bool one_wave = p.tokens * p.tables * heads * cols <= kSms * 2048;  // of threads
  if (one_wave || smem > (size_t)kMaxTileBytes || per_token * per_token * p.tile > 0xffffffffll ||
      !small_steps(p, sizeof(T))) {
    launch_kernel<rope_axes_kernel<T, VP, LAYOUT, T>>(p, dim3(grid_of(p.tokens * p.tables * heads * cols)), 0, st);
    return;
  }
  p.by_token = magic(per_token);
  p.by_table = magic(p.rounds * cols);
  p.by_head = magic(cols);
  const int64_t tiles = (p.tokens + p.tile - 1) / p.tile;
  const dim3 grid((unsigned)std::min<int64_t>(tiles, kSms * kTileBlocks));
  launch_kernel<rope_axes_tile_kernel<T, VP, LAYOUT>>(p, grid, smem, st);
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
