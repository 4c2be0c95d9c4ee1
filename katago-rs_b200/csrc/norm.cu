// Masked group norm with an activation on channels-last board tokens, forward and backward (kc_group_norm_act,
// kc_group_norm_act_backward).
//
//   on = mask != 0, M = (points on) * channels / groups, mean = sum_on x / M, var = sum_on (x - mean)^2 / M,
//   rstd = 1 / sqrt(var + eps), xh = (x - mean) rstd, z = xh w + b, y = act(z) where on, 0 elsewhere
//   gz = dy act'(z) where on, S1[c] = sum gz, S2[c] = sum gz xh (over a board's points),
//   c1 = sum_{c of the group} w S1 / M, c2 = sum w S2 / M, dx = rstd (gz w - c1 - xh c2) where on,
//   dbias = sum over boards of S1, dweight = of S2
//
// Statistics and sums are float32. A thread's share of a mean and of a sum of squares
// is taken around a value of its own and shares are merged by count as distances from one of them, so that a large
// mean costs no digits of the variance.
//
// What bounds it: HBM, once reading and writing the tensor is all the traffic there is; each element that is on also
// costs about 24 instructions forward (mish) and 37 backward, which takes as long. So a board's chunk of channels is
// read once into shared memory and stays there (resident path). Measured on a B200 (6,554 GB/s copy), bytes that have
// to move / time:
//   forward, 256 boards x 361 points x 384 channels, 32 groups, bf16, mish, mixed board sizes: 119 MB in 34.3 us,
//     3,480 GB/s (the split path's three launches with two reads: 178 us). 54% of the issue slots, 18 us of bytes:
//     transfers and arithmetic follow each other. 20 warps to an SM (96 registers, 39 KB of slots a block; 17 active on
//     average), which wait for their own arithmetic and two barriers a chunk
//   1,024 of those boards: 477 MB in 114 us, 4,180 GB/s
//   backward, 512 such boards: 334 MB in 110.6 us, 3,020 GB/s (split path: 426 us), 49% of the issue slots; 128
//     registers and 113 KB of shared memory leave two blocks of 256 to an SM
//   forward, 64 boards x 361 x 768, one group, float32, silu: 119 MB in 52 us, 2,290 GB/s: a board fills a cluster of
//     16 blocks, all boards in four turns of all SMs that load, reduce and store in step
//   forward, 32 x 5,776 x 256, 32 groups, bf16, silu: 189 MB in 56 us, 3,380 GB/s (clusters of 4)

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
constexpr int kMaxTiles = 64;
constexpr int kMaxSmem = 227 * 1024;  // of a block
constexpr int kSms = 148;

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
  float2* sums;          // [rows][channels] backward (S1, S2): split path of a board, resident path of a block's boards
  float* dweight;
  float* dbias;
  int64_t xb, xr, yb, yr, mb;
  int n, points, C, G, cg, act;
  float eps;
  int tiles, tile_rows;
};

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
// The resident path: a chunk of whole groups (V column vectors of VEC channels) of one board is read once and stays
// in the shared memory of a block, or of a cluster of blocks that share the board's points, until it is written. A
// thread owns rows ty, ty + R, ... of its block's points at one column vector, R = threads / V; it copies those that
// are on into `slots` of its own (every threads-th vector of shared memory) itself (cp.async), so that no barrier
// stands between the copy and the statistics.
// U neighbouring channels of a vector lie in one group (VEC, 4 or 1 of them), so that a thread's statistics are
// VEC / U triples of (count, mean, sum of squares around it).
//
// Why this shape: shared memory and not registers, since vectors in registers had to be unrolled and unpacked floats
// stayed live across the passes (206 registers, one block to an SM: 152 us for the 256 boards above). Chunks of at
// least 64 bytes of a row: with 48 bytes the fixed work of a chunk weighs more (42 us), with 128 bytes clusters
// are needed (54 us). Blocks of 128 forward: the fixed work of a chunk (about 500 instructions a warp) is spread over
// more rows a thread than with 256 (36 us). Only rows that are on are read. (Times of the 256 boards with a mish of
// three instructions less, which took 32.6 us in this shape.)
// ---------------------------------------------------------------------------------------------------------------
constexpr int kMaxSlots = 32;  // a thread's rows are bits of one word

struct ResShape {
  int cw;      // channels of a chunk (the last one of a row may have fewer)
  int cs, cs_log2;  // blocks of a cluster
  int rows;    // points per block
  int threads;
  int R;       // rows at once
  int slots;   // vectors a thread has room for
  uint32_t vdiv;  // 2^20 / V + 1: (t * vdiv) >> 20 = t / V for t, V <= 512
  int slot_bytes;  // backward: of all slots, and at least the channel sums'
  int boards;  // backward: blocks that share a chunk's boards
  int chunks;  // of a board
  int blocks, step_boards, step_chunks;  // forward: blocks (clusters), and their distance in boards and chunks
  int wvec;    // weight and bias may be read as 16-byte vectors
};

// A vector as pairs of floats (one channel: the second is 0).
template <typename T, int VEC>
struct Vec {
  static constexpr int NP = (VEC + 1) / 2;
  static constexpr int BYTES = VEC * (int)sizeof(T);
  using Raw = typename std::conditional<BYTES == 16, uint4, typename std::conditional<BYTES == 8, uint2,
              typename std::conditional<BYTES == 4, uint32_t, uint16_t>::type>::type>::type;

  __device__ static __forceinline__ f32x2 word(uint32_t w) {  // two 2-byte values
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      return {__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
      return {f.x, f.y};
    }
  }
  __device__ static __forceinline__ void unpack(Raw r, f32x2 (&v)[NP]) {
    if constexpr (VEC == 1) {
      v[0] = {to_f<T>(*reinterpret_cast<const T*>(&r)), 0.0f};
    } else {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
      for (int i = 0; i < NP; i++) {
        if constexpr (sizeof(T) == 4) v[i] = {__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1])};
        else v[i] = word(w[i]);
      }
    }
  }
  __device__ static __forceinline__ Raw pack(const f32x2 (&v)[NP]) {
    Raw r;
    if constexpr (VEC == 1) {
      *reinterpret_cast<T*>(&r) = from_f<T>(v[0].x);
    } else {
      uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
      for (int i = 0; i < NP; i++) {
        if constexpr (sizeof(T) == 4) {
          w[2 * i] = __float_as_uint(v[i].x);
          w[2 * i + 1] = __float_as_uint(v[i].y);
        } else {
          w[i] = pack2<T>(v[i].x, v[i].y);
        }
      }
    }
    return r;
  }
  // global -> shared; complete for the issuing thread after copies_done()
  __device__ static __forceinline__ void copy_in(Raw* dst, const T* src) {
    if constexpr (BYTES == 16)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
    else if constexpr (BYTES >= 4)
      asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src), "n"(BYTES) : "memory");
    else
      *dst = *reinterpret_cast<const Raw*>(src);
  }
};

__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

__device__ __forceinline__ float2 ld_cluster(const float2* p, uint32_t rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
               : "=f"(v.x), "=f"(v.y) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ int ld_cluster(const int* p, uint32_t rank) {
  int v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
  return v;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f;

// act of two elements.
// mish = z f, f = tanh(log(1 + e)) = n / (n + 2), n = e^2 + 2 e, e = exp(z) (held to 2^60, where f is 1), which keeps
// its digits where f is small. 1 - 2 / ((1 + e)^2 + 1) takes three instructions less (32.6 us where this takes 34.3,
// 256 boards x 361 x 384, bf16), but has lost half an f16 step already where the result is 2^-8, 12 of them at z = -12.
// silu = z / (1 + exp(-z)), 0 where exp(-z) overflows.
template <int ACT>
__device__ __forceinline__ f32x2 act2(f32x2 z) {
  if constexpr (ACT == KC_ACT_RELU) {
    return {z.x < 0.0f ? 0.0f : z.x, z.y < 0.0f ? 0.0f : z.y};
  } else if constexpr (ACT == KC_ACT_MISH) {
    const f32x2 t = mul2(z, {kLog2e, kLog2e});
    const f32x2 e = {ex2(fminf(t.x, 60.0f)), ex2(fminf(t.y, 60.0f))};
    const f32x2 n = mul2(e, add2(e, {2.0f, 2.0f}));
    const f32x2 d = add2(n, {2.0f, 2.0f});
    return mul2(z, mul2(n, {rcp(d.x), rcp(d.y)}));
  } else if constexpr (ACT == KC_ACT_SILU) {
    const f32x2 t = mul2(z, {-kLog2e, -kLog2e});
    const f32x2 d = add2({ex2(t.x), ex2(t.y)}, {1.0f, 1.0f});
    return mul2(z, {rcp(d.x), rcp(d.y)});
  } else {
    return z;
  }
}

// act' of two elements (relu apart: relu_on).
// mish = z n / d with e = exp(z), n = e^2 + 2 e, d = n + 2: mish' = n / d + z 4 e (e + 1) / d^2 (e held to 2^60).
// silu' = s (1 + z (1 - s)), s = 1 / (1 + exp(-z)), exp(-z) held to 2^60.
template <int ACT>
__device__ __forceinline__ f32x2 slope2(f32x2 z) {
  if constexpr (ACT == KC_ACT_MISH) {
    const f32x2 t = mul2(z, {kLog2e, kLog2e});
    const f32x2 e = {ex2(fminf(t.x, 60.0f)), ex2(fminf(t.y, 60.0f))};
    const f32x2 n = mul2(e, add2(e, {2.0f, 2.0f}));
    const f32x2 d = add2(n, {2.0f, 2.0f});
    const f32x2 rd = {rcp(d.x), rcp(d.y)};
    const f32x2 er = mul2(e, rd);                                 // e / d
    const f32x2 k = mul2({4.0f, 4.0f}, mul2(er, add2(er, rd)));   // 4 e (e + 1) / d^2
    return fma2(z, k, mul2(n, rd));
  } else if constexpr (ACT == KC_ACT_SILU) {
    const f32x2 t = mul2(z, {-kLog2e, -kLog2e});
    const f32x2 d = add2({ex2(fminf(t.x, 60.0f)), ex2(fminf(t.y, 60.0f))}, {1.0f, 1.0f});
    const f32x2 s = {rcp(d.x), rcp(d.y)};
    const f32x2 u = fma2({-s.x, -s.y}, z, z);                     // z (1 - s)
    return fma2(s, u, s);
  } else {
    return {1.0f, 1.0f};
  }
}

// a / b of non-negative integers, a < 2^19: (a + 1/2) / b is at least 1 / (2 b) from a whole number, the fast divide
// off by at most 2^-21 of it.
__device__ __forceinline__ int small_div(int a, int b) {
  return (int)__fdividef((float)a + 0.5f, (float)b);
}

__host__ __device__ __forceinline__ size_t round16(size_t v) { return (v + 15) & ~(size_t)15; }

// A thread's place in its block, for every chunk of every board.
struct ResIds {
  int rank, tx, ty;
  int r0, r1;  // the block's points; the thread's are r0 + ty + i R
};

template <int VEC>
__device__ __forceinline__ ResIds res_ids(const NormParams& p, const ResShape& s) {
  ResIds t;
  t.rank = blockIdx.x & (s.cs - 1);
  t.ty = (int)((threadIdx.x * s.vdiv) >> 20);
  t.tx = threadIdx.x - t.ty * (s.cw / VEC);
  t.r0 = min(p.points, t.rank * s.rows);
  t.r1 = min(p.points, t.r0 + s.rows);
  return t;
}

// A chunk of a board.
struct Chunk {
  int b, index, c0;
  int cw;         // its channels (the last one of a row may have fewer)
  int col;        // the thread's first channel
  bool here;      // the thread has a column vector and rows
  uint32_t all;   // the points that there are in its row lane

  template <int VEC>
  __device__ __forceinline__ void set(const NormParams& p, const ResShape& s, const ResIds& t, int board, int chunk) {
    b = board;
    index = chunk;
    c0 = chunk * s.cw;
    cw = min(s.cw, p.C - c0);
    col = c0 + t.tx * VEC;
    here = t.ty < s.R && t.tx * VEC < cw;
    const int left = t.r1 - t.r0 - t.ty;
    const int k = here && left > 0 ? small_div(left + s.R - 1, s.R) : 0;
    all = k >= 32 ? 0xffffffffu : (1u << k) - 1;
  }
};

// on[y]: which points of row lane y are on, bit i being point r0 + y + i R. The mask's values are loaded early (the
// first MASKS a thread), set to bits between two barriers in words that were cleared before the first of them.
constexpr int kMasks = 4;

__device__ __forceinline__ void load_masks(const NormParams& p, const ResShape& s, const ResIds& t, int b,
                                           float (&v)[kMasks]) {
  const float* m = p.mask + (int64_t)b * p.mb + t.r0;
#pragma unroll
  for (int k = 0; k < kMasks; k++) {
    const int r = threadIdx.x + k * s.threads;
    v[k] = r < t.r1 - t.r0 ? __ldg(m + r) : 0.0f;
  }
}

__device__ __forceinline__ void set_bits(const NormParams& p, const ResShape& s, const ResIds& t, int b,
                                         const float (&v)[kMasks], uint32_t* on) {
  auto set = [&](int r) {
    const int i = small_div(r, s.R);
    atomicOr(on + r - i * s.R, 1u << i);
  };
#pragma unroll
  for (int k = 0; k < kMasks; k++)
    if (v[k] != 0.0f) set(threadIdx.x + k * s.threads);
  const float* m = p.mask + (int64_t)b * p.mb + t.r0;
  for (int r = threadIdx.x + kMasks * s.threads; r < t.r1 - t.r0; r += s.threads)
    if (__ldg(m + r) != 0.0f) set(r);
}

// Rows of a tensor as the thread meets them: its i-th point is i * step bytes behind its first one (the host sees to
// it that step fits 32 bits: one wide multiply-add an address).
template <typename P>
__device__ __forceinline__ P* nth_row(P* first, int i, uint32_t step) {
  using B = typename std::conditional<std::is_const<P>::value, const char, char>::type;
  return reinterpret_cast<P*>(reinterpret_cast<B*>(first) + (uint64_t)(uint32_t)i * step);
}

// f(i) of the rows that are on, N of them side by side (independent work hides the latency of a vector's chain).
template <int N, typename F>
__device__ __forceinline__ void each_on(uint32_t on, F&& f) {
  int left = __popc(on);
  for (; left >= N; left -= N) {
    int i[N];
#pragma unroll
    for (int k = 0; k < N; k++) {
      i[k] = __ffs(on) - 1;
      on &= on - 1;
    }
    f(i);
  }
  for (; N > 1 && left > 0; left--) {
    const int i[1] = {__ffs(on) - 1};
    on &= on - 1;
    f(i);
  }
}

// The rows that are on into consecutive slots.
template <typename T, int VEC>
__device__ __forceinline__ void copy_rows(const T* x, uint32_t step, uint32_t on, void* slots, int slot_bytes) {
  char* slot = static_cast<char*>(slots);
  each_on<4>(on, [&](const auto& i) {
#pragma unroll
    for (int k = 0; k < (int)(sizeof(i) / sizeof(int)); k++, slot += slot_bytes)
      Vec<T, VEC>::copy_in(reinterpret_cast<typename Vec<T, VEC>::Raw*>(slot), nth_row(x, i[k], step));
  });
}

template <int VEC>
__device__ __forceinline__ void load_params(const float* w, float other, bool vec, int col,
                                            f32x2 (&o)[(VEC + 1) / 2]) {
  if (!w) {
#pragma unroll
    for (int j = 0; j < (VEC + 1) / 2; j++) o[j] = {other, other};
  } else if (VEC % 4 == 0 && vec) {
#pragma unroll
    for (int j = 0; j < VEC / 4; j++) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(w + col) + j);
      o[2 * j] = {f.x, f.y};
      o[2 * j + 1] = {f.z, f.w};
    }
  } else {
#pragma unroll
    for (int j = 0; j < (VEC + 1) / 2; j++)
      o[j] = {__ldg(w + col + 2 * j), VEC > 1 ? __ldg(w + col + 2 * j + 1) : other};
  }
}

template <typename T, int VEC, int ACT>
__device__ __forceinline__ void apply_rows(uint32_t on, const typename Vec<T, VEC>::Raw* slot, int slot_step, T* y,
                                           uint32_t step,
                                           const f32x2 (&neg_mean)[Vec<T, VEC>::NP], const f32x2 (&a)[Vec<T, VEC>::NP],
                                           const f32x2 (&b)[Vec<T, VEC>::NP]) {
  using V = Vec<T, VEC>;
  each_on<2>(on, [&](const auto& i) {
    constexpr int N = sizeof(i) / sizeof(int);
    f32x2 v[N][V::NP];
#pragma unroll
    for (int k = 0; k < N; k++, slot += slot_step) V::unpack(*slot, v[k]);
#pragma unroll
    for (int k = 0; k < N; k++)
#pragma unroll
      for (int j = 0; j < V::NP; j++) v[k][j] = act2<ACT>(fma2(add2(v[k][j], neg_mean[j]), a[j], b[j]));
#pragma unroll
    for (int k = 0; k < N; k++) *reinterpret_cast<typename V::Raw*>(nth_row(y, i[k], step)) = V::pack(v[k]);
  });
}

// 0 in the rows of the bits.
template <typename T, int VEC>
__device__ __forceinline__ void zero_rows(uint32_t which, T* y, uint32_t step) {
  using V = Vec<T, VEC>;
  const f32x2 v[V::NP] = {};
  each_on<1>(which, [&](const auto& i) { *reinterpret_cast<typename V::Raw*>(nth_row(y, i[0], step)) = V::pack(v); });
}

extern __shared__ __align__(16) unsigned char norm_smem[];

// A group's (mean, rstd), also into the statistics the caller wants. 1 / sqrt by the fast function (2^-22) and one
// Newton step; a variance of 0 with eps 0 gives infinity, one whose squares passed float32's range NaN (1 / sqrt would
// be 0, and the outputs those of a board of equal values).
__device__ __forceinline__ float2 final_stats(float mean, float var, bool any, float eps, float2* stats, int64_t g) {
  const float v = (var < 0.0f ? 0.0f : var) + eps;
  float r = v <= 3.402823466e38f ? rsqrtf(v) : __int_as_float(0x7fc00000);
  if (v > 0.0f && v < 1e38f) r = r * (1.5f - 0.5f * v * r * r);
  const float2 st = any ? make_float2(mean, r) : make_float2(0.0f, 0.0f);
  if (stats) stats[g] = st;
  return st;
}

// A block goes over chunks of boards, gridDim.x / cs apart in the order of memory, with two barriers each: the next
// chunk's rows are copied into the slots as soon as the thread has written this one's, so that the copy runs under the
// other threads' work and the next mask is known by then.
template <typename T, int VEC, int U, int THREADS>  // THREADS: at most; blocks of 128 run five to an SM
__global__ void __launch_bounds__(THREADS, THREADS == 128 ? 5 : 1)
    norm_resident_kernel(const __grid_constant__ NormParams p, const __grid_constant__ ResShape sh) {
  using V = Vec<T, VEC>;
  constexpr int NU = VEC / U, NP = V::NP;
  const ResIds t = res_ids<VEC>(p, sh);
  const int units = sh.cw / U;  // of a row of the chunk
  const int upg = p.cg / U, all_groups = sh.cw / p.cg;
  typename V::Raw* slots = reinterpret_cast<typename V::Raw*>(norm_smem) + threadIdx.x;  // every threads-th
  float2* part = reinterpret_cast<float2*>(norm_smem + round16((size_t)sh.slots * sh.threads * V::BYTES));
  float2* fin = part + sh.R * units;   // the groups' (mean, rstd)
  float2* mine = fin + all_groups;     // [2][groups] the block's (mean, M2), of even and odd turns (cluster)
  uint32_t* bits = reinterpret_cast<uint32_t*>(mine + (sh.cs > 1 ? 2 * all_groups : 0));  // [2][R]
  int* counts = reinterpret_cast<int*>(bits + 2 * sh.R);                // [2]
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, warps = sh.threads / 32;
  const int y0 = small_div(lane, upg), u0 = lane - y0 * upg, dy = small_div(32, upg), du = 32 - dy * upg;
  const uint32_t x_step = (uint32_t)(sh.R * p.xr * sizeof(T)), y_step = (uint32_t)(sh.R * p.yr * sizeof(T));
  const T* x = static_cast<const T*>(p.x) + (int64_t)(t.r0 + t.ty) * p.xr;
  Chunk now = {}, next = {};
  {
    const int first = blockIdx.x >> sh.cs_log2;
    now.set<VEC>(p, sh, t, first / sh.chunks, first % sh.chunks);
  }

  float masks[kMasks];
  for (int y = threadIdx.x; y < 2 * sh.R; y += sh.threads) bits[y] = 0;
  if (p.mask) load_masks(p, sh, t, now.b, masks);
  __syncthreads();
  if (p.mask) {
    set_bits(p, sh, t, now.b, masks, bits);
  } else if (t.tx == 0 && t.ty < sh.R) {
    bits[t.ty] = bits[sh.R + t.ty] = now.all;
  }
  __syncthreads();
  uint32_t on = now.here ? bits[t.ty] : 0;
  copy_rows<T, VEC>(x + (int64_t)now.b * p.xb + now.col, x_step, on, slots, sh.threads * V::BYTES);
  f32x2 weight[NP], bias[NP];
  int loaded = -1;  // the chunk whose weight and bias they are

  for (int odd = 0;; odd ^= 1) {
    int next_b = now.b + sh.step_boards, next_c = now.index + sh.step_chunks;
    if (next_c >= sh.chunks) next_c -= sh.chunks, next_b++;
    const bool more = next_b < p.n;
    if (more) next.set<VEC>(p, sh, t, next_b, next_c);
    const int groups = small_div(now.cw, p.cg);
    const uint32_t* bits_now = bits + odd * sh.R;
    uint32_t* bits_next = bits + (odd ^ 1) * sh.R;
    if (p.mask && more) load_masks(p, sh, t, next.b, masks);
    if (loaded != now.index && now.here) {
      load_params<VEC>(p.weight, 1.0f, sh.wvec, now.col, weight);
      load_params<VEC>(p.bias, 0.0f, sh.wvec, now.col, bias);
    }
    loaded = now.index;
    copies_done();

    // the thread's shares, in one pass around a value of its first row: the squares around the mean are the squares
    // around that value less its distance's, at most as many times larger as the share has values, since it is one
    // of them
    if (now.here) {
      const int cnt = __popc(on);
      f32x2 neg[NP], sum[NP], sq[NP];
      float ref[NU];
      {
        f32x2 v[NP] = {};
        if (on) V::unpack(slots[0], v);
#pragma unroll
        for (int u = 0; u < NU; u++) ref[u] = u * U % 2 ? v[u * U / 2].y : v[u * U / 2].x;
      }
#pragma unroll
      for (int j = 0; j < NP; j++) {
        neg[j] = {-ref[2 * j / U], VEC > 1 ? -ref[(2 * j + 1) / U] : 0.0f};
        sum[j] = sq[j] = {0.0f, 0.0f};
      }
      const typename V::Raw* slot = slots;
#pragma unroll 4
      for (int k = 0; k < cnt; k++, slot += sh.threads) {
        f32x2 v[NP];
        V::unpack(*slot, v);
#pragma unroll
        for (int j = 0; j < NP; j++) {
          const f32x2 d = add2(v[j], neg[j]);
          sum[j] = add2(sum[j], d);
          sq[j] = fma2(d, d, sq[j]);
        }
      }
      const float inv_n = cnt ? __fdividef(1.0f / U, (float)cnt) : 0.0f;
      auto lane_of = [](const f32x2 (&v)[NP], int c) { return c % 2 ? v[c / 2].y : v[c / 2].x; };
#pragma unroll
      for (int u = 0; u < NU; u++) {
        float m = lane_of(sum, u * U), q = lane_of(sq, u * U);
#pragma unroll
        for (int j = 1; j < U; j++) {
          m += lane_of(sum, u * U + j);
          q += lane_of(sq, u * U + j);
        }
        const float d = m * inv_n;
        q -= m * d;
        part[t.ty * units + t.tx * NU + u] = make_float2(ref[u] + d, q < 0.0f ? 0.0f : q);
      }
    }
    if (p.mask)  // last read before the previous board's second barrier
      for (int y = threadIdx.x; y < sh.R; y += sh.threads) bits_next[y] = 0;
    __syncthreads();

    // merged by group, a warp per group, around one share's mean: the correction by the mean's distance from it is
    // at most as many times the result as there are shares, since that share is one of them. (4 of 768 float32
    // channels 1e4 off the rest, one group: rstd off by 4.4e-6 of itself. A pass for the mean and one for the squares
    // leave 3e-8, but take 5% longer with one group a board and 22% with one channel a group.)
    int rows_on = 0;
    for (int i = lane; i < sh.R; i += 32) rows_on += __popc(bits_now[i]);
    rows_on = __reduce_add_sync(0xffffffffu, rows_on);
    int some = 0;  // a row lane with a point that is on
    while (some < sh.R - 1 && !bits_now[some]) some++;
    const float inv = rows_on ? __fdividef(1.0f, (float)rows_on * (float)p.cg) : 0.0f;
    float2* stats = p.stats && t.rank == 0 ? p.stats + (int64_t)now.b * p.G + small_div(now.c0, p.cg) : nullptr;
    float2* block_stats = mine + odd * all_groups;
    for (int g = warp; g < groups; g += warps) {
      const float2* gp = part + g * upg;
      const float ref = gp[some * units].x;
      float s = 0.0f, q = 0.0f;
      for (int y = y0, u = u0; y < sh.R;) {
        const float2 v = gp[y * units + u];
        const float k = (float)(__popc(bits_now[y]) * U), d = v.x - ref;
        if (k != 0.0f) {
          s += k * d;
          q += v.y + k * d * d;
        }
        y += dy;
        u += du;
        if (u >= upg) u -= upg, y++;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        q += __shfl_xor_sync(0xffffffffu, q, o);
      }
      if (lane == 0) {
        const float delta = s * inv;
        q -= s * delta;
        if (sh.cs == 1) fin[g] = final_stats(ref + delta, q * inv, rows_on, p.eps, stats, g);
        else block_stats[g] = make_float2(ref + delta, q < 0.0f ? 0.0f : q);
      }
    }
    if (p.mask && more) set_bits(p, sh, t, next.b, masks, bits_next);
    if (sh.cs > 1) {
      if (threadIdx.x == 0) counts[odd] = rows_on;
      __syncwarp();
      cluster_sync();
      for (int g = warp; g < groups; g += warps) {  // a lane per block of the cluster
        const float c = lane < sh.cs ? (float)ld_cluster(counts + odd, lane) : 0.0f;
        const float2 v = lane < sh.cs ? ld_cluster(block_stats + g, lane) : make_float2(0.0f, 0.0f);
        const float ref = block_stats[g].x;
        float n = c, s = c != 0.0f ? c * (v.x - ref) : 0.0f;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) {
          n += __shfl_xor_sync(0xffffffffu, n, o);
          s += __shfl_xor_sync(0xffffffffu, s, o);
        }
        const float delta = n != 0.0f ? s / n : 0.0f, d = v.x - ref - delta;
        float q = c != 0.0f ? v.y + c * (float)p.cg * d * d : 0.0f;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
        if (lane == 0)
          fin[g] = final_stats(ref + delta, n != 0.0f ? q / (n * (float)p.cg) : 0.0f, n != 0.0f, p.eps, stats, g);
      }
    }
    __syncthreads();

    if (now.here) {
      T* y = static_cast<T*>(p.y) + (int64_t)now.b * p.yb + (int64_t)(t.r0 + t.ty) * p.yr + now.col;
      f32x2 neg[NP], a[NP];
      float2 st[NU];
#pragma unroll
      for (int u = 0; u < NU; u++) st[u] = fin[small_div(t.tx * VEC + u * U, p.cg)];
#pragma unroll
      for (int j = 0; j < NP; j++) {
        const float2 lo = st[2 * j / U], hi = VEC > 1 ? st[(2 * j + 1) / U] : lo;
        neg[j] = {-lo.x, -hi.x};
        a[j] = mul2(weight[j], {lo.y, hi.y});
      }
      if (p.act == KC_ACT_MISH) apply_rows<T, VEC, KC_ACT_MISH>(on, slots, sh.threads, y, y_step, neg, a, bias);
      else if (p.act == KC_ACT_SILU) apply_rows<T, VEC, KC_ACT_SILU>(on, slots, sh.threads, y, y_step, neg, a, bias);
      else if (p.act == KC_ACT_RELU) apply_rows<T, VEC, KC_ACT_RELU>(on, slots, sh.threads, y, y_step, neg, a, bias);
      else apply_rows<T, VEC, KC_ACT_IDENTITY>(on, slots, sh.threads, y, y_step, neg, a, bias);
      // the slots have served; the zeros of the rows that are off can wait
      if (more) {
        const uint32_t on_next = next.here ? bits_next[t.ty] : 0;
        copy_rows<T, VEC>(x + (int64_t)next.b * p.xb + next.col, x_step, on_next, slots, sh.threads * V::BYTES);
      }
      zero_rows<T, VEC>(now.all & ~on, y, y_step);
    } else if (more && next.here) {
      copy_rows<T, VEC>(x + (int64_t)next.b * p.xb + next.col, x_step, bits_next[t.ty], slots, sh.threads * V::BYTES);
    }
    if (!more) break;
    on = next.here ? bits_next[t.ty] : 0;
    now = next;
  }
  if (sh.cs > 1) {  // a block's shared memory stays until the others have read it
    __syncwarp();
    cluster_sync();
  }
}

// Backward: x and dy of the rows that are on in slots of their own; gz (float32, so two planes of 16 bytes for eight
// 2-byte channels) takes dy's place when the thread has read it. The channels' sums go over rows first, then over the
// cluster, then into their groups.
template <typename T, int VEC>
struct BackSlots {
  using V = Vec<T, VEC>;
  using G = Vec<float, VEC < 4 ? VEC : 4>;
  static constexpr int PLANES = V::NP / G::NP;
  static_assert(sizeof(typename V::Raw) <= sizeof(typename G::Raw), "dy waits in the first plane of gz");
  typename V::Raw* x;
  typename G::Raw* g[PLANES];
  int step;
  __device__ __forceinline__ void next(int n) {
    x += n * step;
#pragma unroll
    for (int h = 0; h < PLANES; h++) g[h] += n * step;
  }
  __device__ __forceinline__ void store_g(int k, const f32x2 (&v)[V::NP]) {
#pragma unroll
    for (int h = 0; h < PLANES; h++) {
      f32x2 o[G::NP];
#pragma unroll
      for (int j = 0; j < G::NP; j++) o[j] = v[h * G::NP + j];
      g[h][k * step] = G::pack(o);
    }
  }
  __device__ __forceinline__ void load_g(int k, f32x2 (&v)[V::NP]) const {
#pragma unroll
    for (int h = 0; h < PLANES; h++) {
      f32x2 o[G::NP];
      G::unpack(g[h][k * step], o);
#pragma unroll
      for (int j = 0; j < G::NP; j++) v[h * G::NP + j] = o[j];
    }
  }
};

template <typename T, int VEC, int ACT, int N>
__device__ __forceinline__ void back_rows(BackSlots<T, VEC>& sl, const f32x2 (&neg_mean)[Vec<T, VEC>::NP],
                                          const f32x2 (&rstd)[Vec<T, VEC>::NP], const f32x2 (&w)[Vec<T, VEC>::NP],
                                          const f32x2 (&b)[Vec<T, VEC>::NP], f32x2 (&s1)[Vec<T, VEC>::NP],
                                          f32x2 (&s2)[Vec<T, VEC>::NP]) {
  using V = Vec<T, VEC>;
  f32x2 x[N][V::NP], g[N][V::NP];
#pragma unroll
  for (int k = 0; k < N; k++) {
    V::unpack(sl.x[k * sl.step], x[k]);
    V::unpack(*reinterpret_cast<const typename V::Raw*>(sl.g[0] + k * sl.step), g[k]);
  }
#pragma unroll
  for (int k = 0; k < N; k++)
#pragma unroll
    for (int j = 0; j < V::NP; j++) {
      const f32x2 xh = mul2(add2(x[k][j], neg_mean[j]), rstd[j]);
      const f32x2 z = fma2(xh, w[j], b[j]);
      f32x2& gz = g[k][j];
      if constexpr (ACT == KC_ACT_RELU) {
        gz.x = relu_on(z.x, x[k][j].x, -neg_mean[j].x, rstd[j].x, w[j].x, b[j].x) ? gz.x : 0.0f;
        gz.y = relu_on(z.y, x[k][j].y, -neg_mean[j].y, rstd[j].y, w[j].y, b[j].y) ? gz.y : 0.0f;
      } else {
        gz = mul2(gz, slope2<ACT>(z));
      }
      s1[j] = add2(s1[j], gz);
      s2[j] = fma2(gz, xh, s2[j]);
    }
#pragma unroll
  for (int k = 0; k < N; k++) sl.store_g(k, g[k]);
  sl.next(N);
}

template <typename T, int VEC, int ACT>
__device__ __forceinline__ void back_sums(BackSlots<T, VEC> sl, int cnt, const f32x2 (&neg_mean)[Vec<T, VEC>::NP],
                                          const f32x2 (&rstd)[Vec<T, VEC>::NP], const f32x2 (&w)[Vec<T, VEC>::NP],
                                          const f32x2 (&b)[Vec<T, VEC>::NP], f32x2 (&s1)[Vec<T, VEC>::NP],
                                          f32x2 (&s2)[Vec<T, VEC>::NP]) {
  for (; cnt >= 2; cnt -= 2) back_rows<T, VEC, ACT, 2>(sl, neg_mean, rstd, w, b, s1, s2);
  if (cnt) back_rows<T, VEC, ACT, 1>(sl, neg_mean, rstd, w, b, s1, s2);
}

// A block keeps one chunk and goes over boards blockIdx.y, blockIdx.y + gridDim.y, ..., as the forward kernel does.
template <typename T, int VEC, int U>
__global__ void __launch_bounds__(512) norm_resident_back_kernel(const __grid_constant__ NormParams p,
                                                                 const __grid_constant__ ResShape sh) {
  using V = Vec<T, VEC>;
  using S = BackSlots<T, VEC>;
  using G = typename S::G;
  constexpr int NU = VEC / U, NP = V::NP;
  const ResIds t = res_ids<VEC>(p, sh);
  Chunk at = {};
  at.set<VEC>(p, sh, t, 0, blockIdx.x >> sh.cs_log2);
  const int units = sh.cw / U;
  const int upg = p.cg / U, groups = small_div(at.cw, p.cg), all_groups = sh.cw / p.cg, g0 = small_div(at.c0, p.cg);
  const size_t vectors = (size_t)sh.slots * sh.threads, plane = vectors * sizeof(typename G::Raw);
  unsigned char* planes = norm_smem + round16(vectors * V::BYTES);
  S slots;
  slots.x = reinterpret_cast<typename V::Raw*>(norm_smem) + threadIdx.x;
  slots.step = sh.threads;
#pragma unroll
  for (int h = 0; h < S::PLANES; h++)
    slots.g[h] = reinterpret_cast<typename G::Raw*>(planes + h * plane) + threadIdx.x;
  float2* red = reinterpret_cast<float2*>(norm_smem);  // [R][cw] channel sums, when the slots have served
  float2* part = reinterpret_cast<float2*>(norm_smem + sh.slot_bytes);  // (ty, unit) sums of w gz, w gz xh
  float2* coef = part + sh.R * units;  // the groups' (c1, c2)
  float2* mine = coef + all_groups;    // [2][groups] the block's sums, of even and odd boards (cluster)
  uint32_t* bits = reinterpret_cast<uint32_t*>(mine + (sh.cs > 1 ? 2 * all_groups : 0));
  int* counts = reinterpret_cast<int*>(bits + 2 * sh.R);
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, warps = sh.threads / 32;
  const int y0 = small_div(lane, upg), u0 = lane - y0 * upg, dy = small_div(32, upg), du = 32 - dy * upg;
  const uint32_t x_step = (uint32_t)(sh.R * p.xr * sizeof(T)), y_step = (uint32_t)(sh.R * p.yr * sizeof(T));
  const int64_t x_at = (int64_t)(t.r0 + t.ty) * p.xr + at.col, y_at = (int64_t)(t.r0 + t.ty) * p.yr + at.col;
  const uint32_t all = at.all;
  auto copy_board = [&](int b, uint32_t on) {
    copy_rows<T, VEC>(static_cast<const T*>(p.x) + (int64_t)b * p.xb + x_at, x_step, on, slots.x,
                      sh.threads * V::BYTES);
    copy_rows<T, VEC>(static_cast<const T*>(p.dy) + (int64_t)b * p.yb + y_at, y_step, on, slots.g[0],
                      sh.threads * (int)sizeof(typename G::Raw));
  };

  float masks[kMasks];
  for (int y = threadIdx.x; y < 2 * sh.R; y += sh.threads) bits[y] = 0;
  if (p.mask) load_masks(p, sh, t, blockIdx.y, masks);
  __syncthreads();
  if (p.mask) {
    set_bits(p, sh, t, blockIdx.y, masks, bits);
  } else if (t.tx == 0 && t.ty < sh.R) {
    bits[t.ty] = bits[sh.R + t.ty] = all;
  }
  __syncthreads();
  uint32_t on = at.here ? bits[t.ty] : 0;
  copy_board(blockIdx.y, on);
  f32x2 w[NP], bias[NP], sum1[NP], sum2[NP];  // sums over the block's boards
#pragma unroll
  for (int j = 0; j < NP; j++) sum1[j] = sum2[j] = {0.0f, 0.0f};
  if (at.here) {
    load_params<VEC>(p.weight, 1.0f, sh.wvec, at.col, w);
    load_params<VEC>(p.bias, 0.0f, sh.wvec, at.col, bias);
    if (VEC == 1) w[0].y = 0.0f;
  }

  int odd = 0;
  for (int b = blockIdx.y; b < p.n; b += gridDim.y, odd ^= 1) {
    const int next = b + gridDim.y;
    const bool more = next < p.n;
    const uint32_t* bits_now = bits + odd * sh.R;
    uint32_t* bits_next = bits + (odd ^ 1) * sh.R;
    if (p.mask && more) load_masks(p, sh, t, next, masks);
    f32x2 neg[NP], rstd[NP];
    if (at.here) {
      const float2* stats = p.stats + (int64_t)b * p.G + g0;
      float2 st[NU];
#pragma unroll
      for (int u = 0; u < NU; u++) st[u] = stats[small_div(t.tx * VEC + u * U, p.cg)];
#pragma unroll
      for (int j = 0; j < NP; j++) {
        const float2 lo = st[2 * j / U], hi = VEC > 1 ? st[(2 * j + 1) / U] : make_float2(0.0f, 0.0f);
        neg[j] = {-lo.x, -hi.x};
        rstd[j] = {lo.y, hi.y};
      }
      copies_done();
      f32x2 s1[NP], s2[NP];
#pragma unroll
      for (int j = 0; j < NP; j++) s1[j] = s2[j] = {0.0f, 0.0f};
      const int cnt = __popc(on);
      if (p.act == KC_ACT_MISH) back_sums<T, VEC, KC_ACT_MISH>(slots, cnt, neg, rstd, w, bias, s1, s2);
      else if (p.act == KC_ACT_SILU) back_sums<T, VEC, KC_ACT_SILU>(slots, cnt, neg, rstd, w, bias, s1, s2);
      else if (p.act == KC_ACT_RELU) back_sums<T, VEC, KC_ACT_RELU>(slots, cnt, neg, rstd, w, bias, s1, s2);
      else back_sums<T, VEC, KC_ACT_IDENTITY>(slots, cnt, neg, rstd, w, bias, s1, s2);
#pragma unroll
      for (int j = 0; j < NP; j++) {
        sum1[j] = add2(sum1[j], s1[j]);
        sum2[j] = add2(sum2[j], s2[j]);
        s1[j] = mul2(s1[j], w[j]);
        s2[j] = mul2(s2[j], w[j]);
      }
      auto lane_of = [](const f32x2 (&v)[NP], int c) { return c % 2 ? v[c / 2].y : v[c / 2].x; };
#pragma unroll
      for (int u = 0; u < NU; u++) {
        float2 o = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < U; j++) {
          o.x += lane_of(s1, u * U + j);
          o.y += lane_of(s2, u * U + j);
        }
        part[t.ty * units + t.tx * NU + u] = o;
      }
    }
    if (p.mask)
      for (int y = threadIdx.x; y < sh.R; y += sh.threads) bits_next[y] = 0;
    __syncthreads();

    // the groups' sums, a warp per group
    int rows_on = 0;
    for (int i = lane; i < sh.R; i += 32) rows_on += __popc(bits_now[i]);
    rows_on = __reduce_add_sync(0xffffffffu, rows_on);
    const float inv = rows_on ? 1.0f / ((float)rows_on * (float)p.cg) : 0.0f;
    float2* block_sums = mine + odd * all_groups;
    for (int g = warp; g < groups; g += warps) {
      const float2* gp = part + g * upg;
      float c1 = 0.0f, c2 = 0.0f;
      for (int y = y0, u = u0; y < sh.R;) {
        const float2 v = gp[y * units + u];
        c1 += v.x;
        c2 += v.y;
        y += dy;
        u += du;
        if (u >= upg) u -= upg, y++;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        c1 += __shfl_xor_sync(0xffffffffu, c1, o);
        c2 += __shfl_xor_sync(0xffffffffu, c2, o);
      }
      if (lane == 0) {
        if (sh.cs == 1) coef[g] = make_float2(c1 * inv, c2 * inv);
        else block_sums[g] = make_float2(c1, c2);
      }
    }
    if (p.mask && more) set_bits(p, sh, t, next, masks, bits_next);
    if (sh.cs > 1) {
      if (threadIdx.x == 0) counts[odd] = rows_on;
      __syncwarp();
      cluster_sync();
      for (int g = warp; g < groups; g += warps) {  // a lane per block of the cluster
        float n = lane < sh.cs ? (float)ld_cluster(counts + odd, lane) : 0.0f;
        float2 c = lane < sh.cs ? ld_cluster(block_sums + g, lane) : make_float2(0.0f, 0.0f);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) {
          n += __shfl_xor_sync(0xffffffffu, n, o);
          c.x += __shfl_xor_sync(0xffffffffu, c.x, o);
          c.y += __shfl_xor_sync(0xffffffffu, c.y, o);
        }
        const float f = n != 0.0f ? 1.0f / (n * (float)p.cg) : 0.0f;
        if (lane == 0) coef[g] = make_float2(c.x * f, c.y * f);
      }
    }
    __syncthreads();

    const uint32_t on_next = at.here && more ? bits_next[t.ty] : 0;
    if (at.here) {
      T* dx = static_cast<T*>(p.y) + (int64_t)b * p.xb + x_at;
      f32x2 k1[NP], k2[NP], wr[NP];  // dx = gz (rstd w) - rstd c1 - xh (rstd c2)
      float2 co[NU];
#pragma unroll
      for (int u = 0; u < NU; u++) co[u] = coef[small_div(t.tx * VEC + u * U, p.cg)];
#pragma unroll
      for (int j = 0; j < NP; j++) {
        const float2 lo = co[2 * j / U], hi = VEC > 1 ? co[(2 * j + 1) / U] : lo;
        wr[j] = mul2(w[j], rstd[j]);
        k1[j] = mul2({-lo.x, -hi.x}, rstd[j]);
        k2[j] = mul2({-lo.y, -hi.y}, rstd[j]);
      }
      S sl = slots;
      each_on<2>(on, [&](const auto& i) {
        constexpr int N = sizeof(i) / sizeof(int);
        f32x2 o[N][NP], g[N][NP];
#pragma unroll
        for (int k = 0; k < N; k++) {
          V::unpack(sl.x[k * sl.step], o[k]);
          sl.load_g(k, g[k]);
        }
        sl.next(N);
#pragma unroll
        for (int k = 0; k < N; k++)
#pragma unroll
          for (int j = 0; j < NP; j++) {
            const f32x2 xh = mul2(add2(o[k][j], neg[j]), rstd[j]);
            o[k][j] = fma2(g[k][j], wr[j], fma2(xh, k2[j], k1[j]));
          }
#pragma unroll
        for (int k = 0; k < N; k++) *reinterpret_cast<typename V::Raw*>(nth_row(dx, i[k], x_step)) = V::pack(o[k]);
      });
      if (more) copy_board(next, on_next);
      zero_rows<T, VEC>(all & ~on, dx, x_step);
    }
    on = on_next;
  }
  if (sh.cs > 1) {
    __syncwarp();
    cluster_sync();
  }
  if (!p.sums) return;

  // the channels' sums over the block's boards: rows ty by `parts` threads per channel, then those
  __syncthreads();
  if (at.here) {
    float2* o = red + t.ty * sh.cw + t.tx * VEC;
#pragma unroll
    for (int j = 0; j < NP; j++) {
      o[2 * j] = make_float2(sum1[j].x, sum2[j].x);
      if (VEC > 1) o[2 * j + 1] = make_float2(sum1[j].y, sum2[j].y);
    }
  }
  __syncthreads();
  const int cw = at.cw, parts = min(sh.R, max(1, small_div(sh.threads, sh.cw)));
  const int mine_part = parts > 1 ? small_div(threadIdx.x, sh.cw) : 0;
  for (int c = threadIdx.x - mine_part * sh.cw; mine_part < parts && c < cw; c += parts > 1 ? sh.cw : sh.threads) {
    float2 s = make_float2(0.0f, 0.0f);
    for (int y = mine_part; y < sh.R; y += parts) {
      s.x += red[y * sh.cw + c].x;
      s.y += red[y * sh.cw + c].y;
    }
    red[mine_part * sh.cw + c] = s;  // row `mine_part` of this column is this thread's alone
  }
  __syncthreads();
  for (int c = threadIdx.x; c < cw; c += sh.threads) {
    float2 s = red[c];
    for (int k = 1; k < parts; k++) {
      s.x += red[k * sh.cw + c].x;
      s.y += red[k * sh.cw + c].y;
    }
    p.sums[((int64_t)blockIdx.y * sh.cs + t.rank) * p.C + at.c0 + c] = s;
  }
}

// ---------------------------------------------------------------------------------------------------------------
// The split path, for boards too large for one cluster of blocks: column vectors of VEC channels (lanes tx) by rows
// (ty), a tile of rows per block. grid (tiles * column blocks, boards modulo grid.y).
// ---------------------------------------------------------------------------------------------------------------
// Column vectors of a block: at most 64, the same number for every block.
__host__ __device__ __forceinline__ int tile_columns(int V) {
  const int blocks = (V + 63) / 64;
  return (V + blocks - 1) / blocks;
}

struct TileIds {
  int tile, col0, tx, ty, rows_at_once;
  bool active;
};

template <int VEC>
__device__ __forceinline__ TileIds tile_ids(const NormParams& p) {
  const int V = p.C / VEC, vc = tile_columns(V);
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

// Which of the next N rows of a thread are there and on; their masks are loaded before any of them is waited for.
// Backward fewer rows: they come in twos, with twice the constants.
constexpr int kRowsAhead = 4, kBackRows = 2;
template <int N>
__device__ __forceinline__ void rows_ahead(const NormParams& p, int b, int r, int step, int r1, bool (&on)[N]) {
  float m[N];
#pragma unroll
  for (int i = 0; i < N; i++) {
    const int ri = r + i * step;
    m[i] = ri < r1 ? (p.mask ? __ldg(p.mask + (int64_t)b * p.mb + ri) : 1.0f) : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < N; i++) on[i] = m[i] != 0.0f;
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
      for (int r = t.tile * p.tile_rows + t.ty; r < r1; r += kRowsAhead * t.rows_at_once) {
        float v[kRowsAhead][VEC];
        bool on[kRowsAhead];
        int k = 0;
        rows_ahead(p, b, r, t.rows_at_once, r1, on);
#pragma unroll
        for (int i = 0; i < kRowsAhead; i++)
          if (on[i]) {
            load_pack<T, VEC>(x + (int64_t)(r + i * t.rows_at_once) * p.xr, v[i]);
            k++;
          }
        if (!k) continue;
        const float ik = 1.0f / (float)k, share = (float)k / (float)(cnt + k);
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          float s = 0.0f, q = 0.0f;
#pragma unroll
          for (int i = 0; i < kRowsAhead; i++) s += on[i] ? v[i][j] : 0.0f;
          s *= ik;
#pragma unroll
          for (int i = 0; i < kRowsAhead; i++) {
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
      for (int j = 0; j < VEC; j++)
        red[(t.ty * VEC + j) * (kThreads / t.rows_at_once) + t.tx] = make_float2(mean[j], m2[j]);
      if (t.tx == 0) red_n[t.ty] = cnt;
    }
    __syncthreads();
    // a thread per channel; means as distances from one of them
    const int stride = kThreads / t.rows_at_once, first = t.col0 - t.tx * VEC;
    int N = 0, some = 0;
    for (int i = t.rows_at_once - 1; i >= 0; i--) {
      N += red_n[i];
      if (red_n[i]) some = i;
    }
    for (int c = threadIdx.x; c < tile_columns(p.C / VEC) * VEC && first + c < p.C; c += kThreads) {
      const int j = c % VEC, tx = c / VEC;
      const float ref = red[(some * VEC + j) * stride + tx].x;
      float s = 0.0f, q = 0.0f;
      for (int i = 0; i < t.rows_at_once; i++)
        if (red_n[i]) s += (float)red_n[i] * (red[(i * VEC + j) * stride + tx].x - ref);
      const float delta = N ? s / (float)N : 0.0f;
      for (int i = 0; i < t.rows_at_once; i++) {
        const float2 u = red[(i * VEC + j) * stride + tx];
        const float d = u.x - ref - delta;
        if (red_n[i]) q += u.y + d * d * (float)red_n[i];
      }
      p.part[((int64_t)b * p.tiles + t.tile) * p.C + first + c] = make_float2(N ? ref + delta : 0.0f, q);
    }
    if (first == 0 && threadIdx.x == 0) p.part_n[(int64_t)b * p.tiles + t.tile] = N;
    __syncthreads();
  }
}

// Sum over the threads of a block of whole warps, the same for all of them.
__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  v = (threadIdx.x & 31) < blockDim.x / 32 ? red[threadIdx.x & 31] : 0.0f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Merges the tiles and channels of one group: a block per (board, group), its threads over the channels of all tiles.
__global__ void __launch_bounds__(1024) norm_merge_stats_kernel(const __grid_constant__ NormParams p) {
  __shared__ float red[32];
  __shared__ int count[kMaxTiles];
  const int64_t id = blockIdx.x;
  const int b = (int)(id / p.G), g = (int)(id % p.G);
  const float2* part = p.part + (int64_t)b * p.tiles * p.C + (int64_t)g * p.cg;
  for (int t = threadIdx.x; t < p.tiles; t += blockDim.x) count[t] = p.part_n[(int64_t)b * p.tiles + t];
  __syncthreads();
  float N = 0.0f;
  int some = 0;
  for (int t = p.tiles - 1; t >= 0; t--) {
    N += (float)count[t];
    if (count[t]) some = t;
  }
  N *= (float)p.cg;
  const float ref = part[(int64_t)some * p.C].x;
  // thread -> (tile, channel) with the step of a block's threads
  const int lanes = min(p.cg, (int)blockDim.x), c0 = threadIdx.x % lanes, t0 = threadIdx.x / lanes;
  const int tiles_at_once = blockDim.x / lanes;
  float s = 0.0f;
  for (int t = t0; t < p.tiles && t0 < tiles_at_once; t += tiles_at_once)
    if (count[t])
#pragma unroll 4
      for (int c = c0; c < p.cg; c += lanes) s += (float)count[t] * (part[(int64_t)t * p.C + c].x - ref);
  s = block_sum(s, red);
  const float delta = N > 0.0f ? s / N : 0.0f;
  float q = 0.0f;
  for (int t = t0; t < p.tiles && t0 < tiles_at_once; t += tiles_at_once)
    if (count[t])
#pragma unroll 4
      for (int c = c0; c < p.cg; c += lanes) {
        const float2 u = part[(int64_t)t * p.C + c];
        const float d = u.x - ref - delta;
        q += u.y + d * d * (float)count[t];
      }
  q = block_sum(q, red);
  if (threadIdx.x == 0)
    p.coef[id] = final_stats(ref + delta, N > 0.0f ? q / N : 0.0f, N > 0.0f, p.eps, p.stats, id);
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
    for (int r = t.tile * p.tile_rows + t.ty; r < r1; r += kRowsAhead * t.rows_at_once) {
      float v[kRowsAhead][VEC] = {};
      bool on[kRowsAhead];
      rows_ahead(p, b, r, t.rows_at_once, r1, on);
#pragma unroll
      for (int i = 0; i < kRowsAhead; i++)
        if (on[i]) load_pack<T, VEC>(x + (int64_t)(r + i * t.rows_at_once) * p.xr, v[i]);
#pragma unroll
      for (int i = 0; i < kRowsAhead; i++) {
        const int ri = r + i * t.rows_at_once;
        if (ri >= r1) break;
        if (on[i]) {
#pragma unroll
          for (int j = 0; j < VEC; j++) v[i][j] = norm_act((v[i][j] - mean[j]) * a[j] + bias[j], p.act);
        }
        store_pack<T, VEC>(y + (int64_t)ri * p.yr, v[i]);
      }
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
      for (int r = t.tile * p.tile_rows + t.ty; r < r1; r += kBackRows * t.rows_at_once) {
        float v[kBackRows][VEC], g[kBackRows][VEC];
        bool on[kBackRows];
        rows_ahead(p, b, r, t.rows_at_once, r1, on);
#pragma unroll
        for (int i = 0; i < kBackRows; i++)
          if (on[i]) {
            load_pack<T, VEC>(x + (int64_t)(r + i * t.rows_at_once) * p.xr, v[i]);
            load_pack<T, VEC>(dy + (int64_t)(r + i * t.rows_at_once) * p.yr, g[i]);
          }
#pragma unroll
        for (int i = 0; i < kBackRows; i++) {
          if (!on[i]) continue;
          back_vec<VEC>(c, p.act, v[i], g[i]);
          cnt++;
#pragma unroll
          for (int j = 0; j < VEC; j++) {
            s1[j] += g[i][j];
            s2[j] += g[i][j] * v[i][j];
          }
        }
      }
    }
    if (t.active) {
#pragma unroll
      for (int j = 0; j < VEC; j++)
        red[(t.ty * VEC + j) * (kThreads / t.rows_at_once) + t.tx] = make_float2(s1[j], s2[j]);
      if (t.tx == 0) red_n[t.ty] = cnt;
    }
    __syncthreads();
    const int stride = kThreads / t.rows_at_once, first = t.col0 - t.tx * VEC;
    // a thread per channel
    for (int c = threadIdx.x; c < tile_columns(p.C / VEC) * VEC && first + c < p.C; c += kThreads) {
      float2 s = make_float2(0.0f, 0.0f);
      for (int i = 0; i < t.rows_at_once; i++) {
        const float2 u = red[(i * VEC + c % VEC) * stride + c / VEC];
        s.x += u.x;
        s.y += u.y;
      }
      p.part[((int64_t)b * p.tiles + t.tile) * p.C + first + c] = s;
    }
    if (first == 0 && threadIdx.x == 0) {
      int N = 0;
      for (int i = 0; i < t.rows_at_once; i++) N += red_n[i];
      p.part_n[(int64_t)b * p.tiles + t.tile] = N;
    }
    __syncthreads();
  }
}

// Adds the tiles of one group's channels and makes its c1, c2: a block per (board, group), its threads over channels.
__global__ void __launch_bounds__(1024) norm_merge_back_kernel(const __grid_constant__ NormParams p) {
  __shared__ float red[32];
  const int64_t id = blockIdx.x;
  const int b = (int)(id / p.G), g = (int)(id % p.G);
  float N = 0.0f;
  for (int t = 0; t < p.tiles; t++) N += (float)p.part_n[(int64_t)b * p.tiles + t];
  N *= (float)p.cg;
  float c1 = 0.0f, c2 = 0.0f;
  for (int i = threadIdx.x; i < p.cg; i += blockDim.x) {
    const int c = g * p.cg + i;
    const float2* part = p.part + (int64_t)b * p.tiles * p.C + c;
    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll 8
    for (int t = 0; t < p.tiles; t++) {
      const float2 u = part[(int64_t)t * p.C];
      s.x += u.x;
      s.y += u.y;
    }
    p.sums[(int64_t)b * p.C + c] = s;
    const float w = p.weight ? __ldg(p.weight + c) : 1.0f;
    c1 += w * s.x;
    c2 += w * s.y;
  }
  c1 = block_sum(c1, red);
  c2 = block_sum(c2, red);
  if (threadIdx.x == 0) p.coef[id] = N > 0.0f ? make_float2(c1 / N, c2 / N) : make_float2(0.0f, 0.0f);
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
    for (int r = t.tile * p.tile_rows + t.ty; r < r1; r += kBackRows * t.rows_at_once) {
      float v[kBackRows][VEC], g[kBackRows][VEC];
      bool on[kBackRows];
      rows_ahead(p, b, r, t.rows_at_once, r1, on);
#pragma unroll
      for (int i = 0; i < kBackRows; i++)
        if (on[i]) {
          load_pack<T, VEC>(x + (int64_t)(r + i * t.rows_at_once) * p.xr, v[i]);
          load_pack<T, VEC>(dy + (int64_t)(r + i * t.rows_at_once) * p.yr, g[i]);
        }
#pragma unroll
      for (int i = 0; i < kBackRows; i++) {
        const int ri = r + i * t.rows_at_once;
        if (ri >= r1) break;
        float o[VEC] = {};
        if (on[i]) {
          back_vec<VEC>(c, p.act, v[i], g[i]);
#pragma unroll
          for (int j = 0; j < VEC; j++) o[j] = (g[i][j] * c.w[j] - k[j].x - v[i][j] * k[j].y) * c.rstd[j];
        }
        store_pack<T, VEC>(dx + (int64_t)ri * p.xr, o);
      }
    }
  }
}

// dbias, dweight [c] = the rows' sums in a fixed order and in 64 bits: 8 channels a block, 32 lanes of rows each.
__global__ void __launch_bounds__(kThreads) norm_params_kernel(const float2* __restrict__ sums, int rows, int C,
                                                               float* __restrict__ dweight,
                                                               float* __restrict__ dbias) {
  __shared__ double2 red[32][8];
  const int tx = threadIdx.x & 7, ty = threadIdx.x / 8;
  const int c = blockIdx.x * 8 + tx;
  double2 s = make_double2(0.0, 0.0);
  if (c < C)
#pragma unroll 4
    for (int b = ty; b < rows; b += 32) {
      const float2 u = sums[(int64_t)b * C + c];
      s.x += u.x;
      s.y += u.y;
    }
  red[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && c < C) {
    for (int i = 1; i < 32; i++) {
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

Rows x_rows(const kc_group_norm_desc& d, const void* p) {
  return {p, d.n, d.points, d.channels, d.x_board_stride, d.x_row_stride, dtype_bytes(d.dtype)};
}
Rows y_rows(const kc_group_norm_desc& d, const void* p) {
  return {p, d.n, d.points, d.channels, d.y_board_stride, d.y_row_stride, dtype_bytes(d.dtype)};
}

// What the workspace query and the calls refuse alike: sizes and strides that the arithmetic of either cannot hold.
void check_desc(const kc_group_norm_desc* d) {
  if (!d) bad("null descriptor");
  if (d->dtype != KC_PRECISION_F32 && d->dtype != KC_PRECISION_F16 && d->dtype != KC_PRECISION_BF16)
    bad("dtype must be KC_PRECISION_F32, F16 or BF16");
  if (d->act < KC_ACT_IDENTITY || d->act > KC_ACT_SILU) bad("unknown activation");
  if (d->n < 0 || d->points < 0 || d->n > 1 << 30 || d->points > 1 << 30) bad("n and points must be 0 to 2^30");
  if (d->channels < 1 || d->groups < 1 || d->channels > 1 << 30) bad("channels must be 1 to 2^30, groups positive");
  if (d->channels % d->groups != 0) bad("channels must be a multiple of groups");
  if ((int64_t)d->n * d->channels > (int64_t)1 << 46) bad("n * channels must be at most 2^46");
  if (!(d->eps >= 0.0f) || !std::isfinite(d->eps)) bad("eps must be finite and not negative");
  if (d->reserved != 0) bad("reserved must be 0");
  if (!rows_in_range(x_rows(*d, nullptr)) || !rows_in_range(y_rows(*d, nullptr)))
    bad("strides must not be negative, nor reach past 2^46 elements");
}

// Tiles of rows of the split path: enough blocks for every SM several times over, of at least 32 rows.
void split_shape(const kc_group_norm_desc& d, int& tiles, int& tile_rows) {
  const int64_t per_board = std::max<int64_t>(1, 2048 / ((int64_t)std::max(1, d.n) * ((d.channels + 511) / 512)));
  const int64_t t = std::min<int64_t>({(int64_t)kMaxTiles, per_board, (d.points + 31) / 32});
  tile_rows = (int)((d.points + std::max<int64_t>(1, t) - 1) / std::max<int64_t>(1, t));
  tiles = (d.points + tile_rows - 1) / std::max(1, tile_rows);
}

// ---- resident path ----
int lcm_of(int a, int b) {
  int x = a, y = b;
  while (y) {
    const int r = x % y;
    x = y;
    y = r;
  }
  return (int)std::min<int64_t>((int64_t)a / x * b, 1 << 30);
}

// Shared memory of a block; sets slot_bytes.
size_t resident_smem(ResShape& s, int vec, int unit, int es, int cg, bool backward) {
  const size_t slots = (size_t)s.slots * s.threads, groups = s.cw / cg;
  size_t bytes = round16(slots * vec * es);
  if (backward) bytes = round16(std::max(bytes + slots * vec * 4, (size_t)s.R * s.cw * sizeof(float2)));
  s.slot_bytes = (int)bytes;
  return bytes + ((size_t)s.R * (s.cw / unit) + (s.cs > 1 ? 3 : 1) * groups) * sizeof(float2) +
         (2 * s.R + 2) * sizeof(int);
}

// Channels of a vector that are sure to lie in one group.
int unit_of(int vec, int cg) { return vec >= 4 && cg % vec == 0 ? vec : vec >= 4 && cg % 4 == 0 ? 4 : 1; }

// The chunk, cluster and block of a resident launch; false where a board's group does not fit 16 blocks.
bool resident_shape(const kc_group_norm_desc& d, int vec, bool backward, ResShape& s) {
  const int es = dtype_bytes(d.dtype), cg = d.channels / d.groups, unit = unit_of(vec, cg);
  const int base = lcm_of(cg, vec);
  if (d.channels > 1 << 18 || base > d.channels || base / vec > 512) return false;  // small_div's range
  // whole 64-byte pieces of a row
  int k = 1;
  while (base * k * es < 64 && base * k < d.channels) k++;
  s.cw = std::min(d.channels, base * k);
  if (s.cw / vec > 512) return false;
  const int64_t chunks = (d.channels + s.cw - 1) / s.cw;
  const int64_t row_step = d.points > 1 ? std::max(d.x_row_stride, d.y_row_stride) : 0;  // one row has no step
  auto fits = [&](int threads, int cs) {
    s.threads = threads;
    s.cs = cs;
    if (s.cw / vec > threads) return false;
    s.R = threads / (s.cw / vec);
    s.rows = (d.points + cs - 1) / cs;
    s.slots = (s.rows + s.R - 1) / s.R;
    const int64_t step = row_step * s.R * es;  // nth_row's
    return step <= 0xffffffffll && s.slots <= kMaxSlots &&
           resident_smem(s, vec, unit, es, cg, backward) <= (size_t)kMaxSmem;
  };
  bool ok = false;
  // the fewest blocks whose rows leave room for as many of them on an SM as their registers do: five of 128 threads
  // forward, two of 256 backward. (A limit of 18 and 9 rows a thread, which is that of 16-byte vectors at 361 points,
  // put 400 points into clusters of two: 256 boards x 400 x 384, bf16, 51 us instead of 37.5; 400 boards x 700 x 30,
  // bf16, 48 instead of 23 us, backward 78 instead of 30.)
  const size_t share = kMaxSmem / (backward ? 2 : 5) - 1024;
  for (int cs = 1; cs <= 8 && !ok; cs *= 2)
    ok = fits(backward ? 256 : 128, cs) && resident_smem(s, vec, unit, es, cg, backward) <= share;
  // larger boards: clusters of up to 16, where two blocks fit an SM before that where one does
  for (int cs = 2; cs <= 16 && !ok; cs *= 2)
    for (int threads = 256; threads <= 512 && !ok; threads *= 2)
      ok = fits(threads, cs) && resident_smem(s, vec, unit, es, cg, backward) <= (size_t)kMaxSmem / 2 - 1024;
  for (int cs = 2; cs <= 16 && !ok; cs *= 2) ok = fits(256, cs) || fits(512, cs);
  if (!ok) return false;
  // narrow vectors hold little each: many turns of large clusters, where tiles of rows take fewer (40 boards of 5,000 x
  // 99 channels, f16: 228 us in clusters of 16, 100 us in tiles)
  if (vec * es < 8 && s.cs > 4) return false;
  // few boards: spread one over more SMs
  while (s.cs < 8 && s.slots > 3 && (int64_t)d.n * chunks * s.cs < kSms) fits(s.threads, s.cs * 2);
  s.vdiv = (1u << 20) / (uint32_t)(s.cw / vec) + 1;
  // blocks that run together, by shared memory and registers. A forward block takes any chunks; a backward one keeps
  // its chunk (for the channels' sums) and the boards go evenly over them.
  const int64_t smem = resident_smem(s, vec, unit, es, cg, backward);
  const int by_registers = !backward && s.threads == 128 ? 5 : 512 / s.threads;
  const int64_t per_sm = std::max<int64_t>(1, std::min<int64_t>(kMaxSmem / (smem + 1024), by_registers));
  s.chunks = (int)chunks;
  s.blocks = (int)std::min<int64_t>(std::max<int64_t>(1, kSms * per_sm / s.cs), d.n * chunks);
  if (s.cs > 1 && per_sm > 1) {  // clusters start together only where SMs have room: no more than the turns need
    const int64_t tiles = d.n * chunks, turns = (tiles + s.blocks - 1) / s.blocks;
    s.blocks = (int)((tiles + turns - 1) / turns);
  }
  s.step_boards = s.blocks / s.chunks;
  s.step_chunks = s.blocks % s.chunks;
  const int64_t most = std::max<int64_t>(1, kSms * per_sm / (chunks * s.cs)), turns = (d.n + most - 1) / most;
  s.boards = (int)std::min<int64_t>((d.n + turns - 1) / turns, 65535);
  s.cs_log2 = 0;
  while (1 << s.cs_log2 < s.cs) s.cs_log2++;
  return chunks * s.cs <= 0x7fffffff;
}

struct Layout {
  size_t part = 0, part_n = 0, coef = 0, sums = 0, total = 0;
  bool resident = false;  // without the split path's parts
};
size_t round256(size_t v) { return (v + 255) / 256 * 256; }

Layout workspace_layout(const kc_group_norm_desc& d, bool backward) {
  Layout l;
  if (d.n == 0 || d.points == 0) return l;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += round256(bytes);
    return here;
  };
  // the split path's, unless the call is resident whatever its tensors' alignment
  bool resident = true;
  int64_t rows = 0;
  for (int v = 16 / dtype_bytes(d.dtype); v >= 1; v /= 2) {
    ResShape s;
    if (d.channels % v != 0) continue;
    if (resident_shape(d, v, backward, s)) rows = std::max<int64_t>(rows, (int64_t)s.boards * s.cs);
    else resident = false, rows = std::max<int64_t>(rows, d.n);
  }
  if (backward) l.sums = take((size_t)rows * d.channels * sizeof(float2));
  l.total = at;
  l.resident = resident;
  if (resident) return l;
  if ((int64_t)d.n * d.groups > 0x7fffffff) bad("n * groups above 2^31 - 1");  // a block each in the split path's merge
  int tiles, tile_rows;
  split_shape(d, tiles, tile_rows);
  l.part = take((size_t)d.n * tiles * d.channels * sizeof(float2));
  l.part_n = take((size_t)d.n * tiles * sizeof(int));
  l.coef = take((size_t)d.n * d.groups * sizeof(float2));
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

void launch_params(const NormParams& p, int rows, cudaStream_t st) {
  if (!p.dweight && !p.dbias) return;
  norm_params_kernel<<<(p.C + 7) / 8, kThreads, 0, st>>>(p.sums, rows, p.C, p.dweight, p.dbias);
  KC_CUDA(cudaGetLastError());
}

// A block per (board, group), of threads for its items.
unsigned merge_blocks(const NormParams& p) { return (unsigned)((int64_t)p.n * p.G); }  // workspace_layout: below 2^31
unsigned merge_threads(int64_t items) { return (unsigned)std::min<int64_t>(1024, (items + 31) / 32 * 32); }

template <typename T, int VEC>
void split_forward(const NormParams& p, cudaStream_t st) {
  const int V = p.C / VEC, vc = tile_columns(V);
  const dim3 grid((unsigned)(p.tiles * ((V + vc - 1) / vc)), (unsigned)std::min(p.n, 65535));
  norm_tile_stats_kernel<T, VEC><<<grid, kThreads, 0, st>>>(p);
  KC_CUDA(cudaGetLastError());
  norm_merge_stats_kernel<<<merge_blocks(p), merge_threads((int64_t)p.cg * p.tiles), 0, st>>>(p);
  KC_CUDA(cudaGetLastError());
  norm_tile_apply_kernel<T, VEC><<<grid, kThreads, 0, st>>>(p);
  KC_CUDA(cudaGetLastError());
}

template <typename T, int VEC>
void split_backward(const NormParams& p, cudaStream_t st) {
  const int V = p.C / VEC, vc = tile_columns(V);
  const dim3 grid((unsigned)(p.tiles * ((V + vc - 1) / vc)), (unsigned)std::min(p.n, 65535));
  norm_tile_back_kernel<T, VEC><<<grid, kThreads, 0, st>>>(p);
  KC_CUDA(cudaGetLastError());
  norm_merge_back_kernel<<<merge_blocks(p), merge_threads(p.cg), 0, st>>>(p);
  KC_CUDA(cudaGetLastError());
  norm_tile_dx_kernel<T, VEC><<<grid, kThreads, 0, st>>>(p);
  KC_CUDA(cudaGetLastError());
  launch_params(p, p.n, st);
}

template <auto kernel>
void launch_resident(const NormParams& p, const ResShape& s, bool backward, size_t smem, cudaStream_t st) {
  static std::atomic<uint64_t> allowed[2];  // devices on which this kernel may take more than 48 KB
  int dev = 0;
  KC_CUDA(cudaGetDevice(&dev));
  if (dev >= 128) bad("device index above 127");
  if (!(allowed[dev / 64].load(std::memory_order_acquire) >> (dev % 64) & 1)) {
    KC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem));
    KC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));  // clusters of 16
    // all of an SM's shared memory: the blocks that resident_shape counts on start together
    KC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                 cudaSharedmemCarveoutMaxShared));
    allowed[dev / 64].fetch_or(1ull << (dev % 64), std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = backward ? dim3((unsigned)(s.chunks * s.cs), (unsigned)s.boards) : dim3((unsigned)(s.blocks * s.cs));
  cfg.blockDim = dim3((unsigned)s.threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)s.cs;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = s.cs > 1 ? 1 : 0;
  KC_CUDA(cudaLaunchKernelEx(&cfg, kernel, p, s));
}

template <typename T, int VEC, int U>
void run_resident(const NormParams& p, ResShape s, bool backward, cudaStream_t st) {
  const size_t smem = resident_smem(s, VEC, U, sizeof(T), p.cg, backward);
  if (!backward && s.threads == 128)
    return launch_resident<norm_resident_kernel<T, VEC, U, 128>>(p, s, false, smem, st);
  if (!backward) return launch_resident<norm_resident_kernel<T, VEC, U, 512>>(p, s, false, smem, st);
  launch_resident<norm_resident_back_kernel<T, VEC, U>>(p, s, true, smem, st);
  launch_params(p, s.boards * s.cs, st);
}

template <typename T, int VEC>
void run_vec(const kc_group_norm_desc& d, const NormParams& p, bool backward, cudaStream_t st) {
  ResShape s;
  if (resident_shape(d, VEC, backward, s)) {
    s.wvec = aligned_to(p.weight, 16) && aligned_to(p.bias, 16);
    const int unit = unit_of(VEC, p.cg);
    if constexpr (VEC == 8)
      if (unit == 8) return run_resident<T, VEC, 8>(p, s, backward, st);
    if constexpr (VEC >= 4)
      if (unit == 4) return run_resident<T, VEC, 4>(p, s, backward, st);
    return run_resident<T, VEC, 1>(p, s, backward, st);
  }
  backward ? split_backward<T, VEC>(p, st) : split_forward<T, VEC>(p, st);
}

template <typename T>
void run_type(const kc_group_norm_desc& d, const NormParams& p, int vec, bool backward, cudaStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (vec == 8) return run_vec<T, 8>(d, p, backward, st);
  if (vec == 4) return run_vec<T, 4>(d, p, backward, st);
  if (vec == 2) return run_vec<T, 2>(d, p, backward, st);
  run_vec<T, 1>(d, p, backward, st);
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
  p.xr = d.points > 1 ? d.x_row_stride : 0;
  p.yb = d.y_board_stride;
  p.yr = d.points > 1 ? d.y_row_stride : 0;
  p.mb = d.mask_board_stride;
  split_shape(d, p.tiles, p.tile_rows);
  const Layout l = workspace_layout(d, backward);
  char* ws = static_cast<char*>(workspace);
  p.part = reinterpret_cast<float2*>(ws + l.part);
  p.part_n = reinterpret_cast<int*>(ws + l.part_n);
  p.coef = reinterpret_cast<float2*>(ws + l.coef);
  p.sums = p.dweight || p.dbias || !l.resident ? reinterpret_cast<float2*>(ws + l.sums) : nullptr;
  if (d.dtype == KC_PRECISION_F32) run_type<float>(d, p, vec, backward, st);
  else if (d.dtype == KC_PRECISION_F16) run_type<__half>(d, p, vec, backward, st);
  else run_type<__nv_bfloat16>(d, p, vec, backward, st);
}

void check_tensors(const kc_group_norm_desc& d, std::initializer_list<Rows> rows, const float* mask,
                   std::initializer_list<const void*> small) {
  const Rows m{mask, d.n, 1, d.points, d.mask_board_stride, 0, 4};
  if (mask && !rows_in_range(m)) bad("mask stride out of range");
  for (const Rows& r : rows)
    if (!aligned_to(r.p, r.bytes)) bad("a tensor is not aligned to its element");
  for (const void* s : small)
    if (!aligned_to(s, 4)) bad("a float32 tensor is not aligned to its element");
}

// Outputs share no memory with each other or with an input; only a tensor may be its own output.
void check_outputs(const kc_group_norm_desc& d, const Rows& out, std::initializer_list<Rows> ins, const float* mask,
                   std::initializer_list<Range> small_in, std::initializer_list<Range> small_out) {
  if (!rows_distinct(out)) bad("rows of the output share memory");
  for (const Rows& i : ins)
    if (rows_overlap(out, i) && !out.same(i)) bad("the output overlaps an input it does not match");
  const Rows m{mask, d.n, 1, d.points, d.mask_board_stride, 0, 4};
  if (rows_overlap(out, m)) bad("the output overlaps the mask");
  for (const Range& s : small_in)
    if (ranges_meet(s, out)) bad("the output overlaps another tensor of the call");
  for (const Range* o = small_out.begin(); o != small_out.end(); o++) {
    bool meets = ranges_meet(*o, out) || ranges_meet(*o, m);
    for (const Rows& i : ins) meets = meets || ranges_meet(*o, i);
    for (const Range& s : small_in) meets = meets || ranges_meet(*o, s);
    for (const Range* q = o + 1; q != small_out.end(); q++)
      meets = meets || ranges_meet(*o, *q);
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
    p.dweight = d_dweight;
    p.dbias = d_dbias;
    run(d, p, vec_of(d, {d_x, d_dy, d_dx}), true, d_workspace, st);
  });
}
