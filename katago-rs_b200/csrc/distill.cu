// Loss of a student's logits against a teacher's top logits, and the gradient of the logits (kc_distill_top,
// kc_distill_top_backward).
//
//   q = softmax(z / T), p_j = exp(t_j / T - L), L = log sum_j exp(t_j / T) over the row's entries or the teacher's own
//   loss = T^2 sum_j p_j (log p_j - log q_{id_j})
//   dz_i = dloss T (P q_i - sum_{j: id_j = i} p_j), P = sum_j p_j
//
// The teacher's side of a row is a few entries, held by the threads that share the row: exponentials of differences
// taken in 64 bits, and sums in 64 bits, since the loss is a difference of logarithms. With e_j = exp((t_j - max t) /
// T) the loss is T^2 (sum e_j x_j / sum e_j + log(s / sum e_j)), x_j = ((t_j - max t) - (z_{id_j} - m)) / T, from the
// row's largest logit m and s = sum exp((z - m) / T): one logarithm a row.
// Backward, the saved (m, s) make each element's gradient one exponential; the entries' classes are gathered before the
// row is written, so that the gradient may take the logits' place, and written over it at the end. Rows without entries
// are not read.
//
// Rows of at most 2,048 classes are a warp's, which keeps the row in shared memory while the next one is on its way
// there; longer ones a block's or, where rows are few, a cluster's (forward) or several blocks' (backward).
//
// What bounds it, measured on a B200 (6,549 GB/s copy), bytes that have to move / time:
//   backward, 4,096 rows x 32,000, 128 entries, bf16: 513 MB in 91.0 us, 5,640 GB/s (HBM)
//   forward, the same: 251 MB in 59.8 us, 4,200 GB/s. Neither the exponentials (16 a clock and SM: 29 us) nor issue
//     (51% of the slots) is full: a block lives for one row, whose first loads wait for the entries and a barrier, and
//     has nothing in flight while it ends
//   backward, 16,384 rows x 362, 64 entries, bf16: 32 MB in 14.3 us: 580 warp instructions a row, most of them the
//     entries'
//   forward, 60,000 rows x 362, 32 entries, bf16: 57 MB in 32 us: 424 warp instructions a row, 75% of the issue slots
//   more than 128 entries in rows of 362, which a block takes: 16,384 rows, 362 entries, bf16, forward 59 MB in 51.7
//     us, backward 71 MB in 60.5 us: 2,740 warp instructions a row, the entries' and the clearing of 8 KB of bits
// With loops over the entries in memory, all in 64 bits, these took 99, 67, 29 and 73 us.

#include <algorithm>
#include <cmath>
#include <string>

#include "../../include/katago_cuda.h"
#include "rows.cuh"

namespace kc {
namespace {

[[noreturn]] void bad(const std::string& what) { fail(KC_ERR_INVALID, "CUDA backend: top logits: " + what); }

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMostHeld = 4;        // entries of a thread (kernels are built for 1 to 4)
constexpr int kWarpClasses = 2048;  // rows up to this long, with up to 32 kMostHeld entries, are a warp's
constexpr int kWarpTop = 32 * kMostHeld;
constexpr int kMaxTop = kThreads * kMostHeld;
// Blocks to an SM of the kernels that give a row to a warp: 64 registers, or 80 for more entries.
constexpr int warp_kernel_blocks(int held) { return held <= 2 ? 4 : 3; }
// The loss is T^2 times a difference of logarithms that shrinks like 1 / T^2 while their error, the float32 sums',
// stays. Logits at distance 1 from the teacher's have a loss of 0.5, off by up to T^2 2^-18 (362 classes): 0.8% of it
// at T = 32. The worst of 2,000 rows measured: 0.02% at T = 20, 0.05% at 32, 2.5% at 256, 35% at 1,024, 490% at 4,096.
constexpr float kMostTemperature = 32.0f;
constexpr double kLightest = -690.0;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_huge_valf();

struct DistillParams {
  const void* z;
  const int32_t* ids;
  const float* top;
  const float* whole;
  float* loss;
  float2* stats;
  const float* dloss;
  void* dz;
  int64_t zs, ds, ts;
  int64_t rows;
  int classes, k;
  int splits, seg;  // blocks of a row, classes of each
  int row_bytes;    // of a warp's row in shared memory
  double temperature, inv;
  float c;          // log2(e) / T
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// exp of a 64-bit argument, or of `least`, to float32's precision; 0 below -104
__device__ __forceinline__ float exp_of(double x, double least = -200.0) {
  x = x < least ? least : x;
  const float hi = (float)x, e = expf(hi);
  return fmaf(e, (float)(x - hi), e);
}

__device__ __forceinline__ float warp_max(float v) {
  float m;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}
__device__ __forceinline__ float warp_sum(float v) { return lanes_sum(v, 32); }
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The largest value m (-inf: none) and s = sum of exp((z - m) / T).
struct Peak {
  float m, s;
};

// An exponent's base: 0 where there is only -inf, whose differences would be NaN.
__device__ __forceinline__ float base_of(float m) { return m == -kInf ? 0.0f : m; }

__device__ __forceinline__ Peak warp_peak(Peak a, float c) {
  const float m = warp_max(a.m);
  return {m, warp_sum(a.s * ex2((a.m - base_of(m)) * c))};
}

// 16 bytes of a row
template <typename T>
struct Chunk {
  static constexpr int VEC = 16 / sizeof(T), N = VEC / 2;
  using V = RowVec<T, VEC>;
  __device__ static __forceinline__ uint4 nothing() {  // elements of -inf
    const uint32_t w = std::is_same<T, float>::value ? 0xff800000u
                       : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
    return make_uint4(w, w, w, w);
  }
  __device__ static __forceinline__ float largest(const uint4& r) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
    if constexpr (std::is_same<T, float>::value) {
      return fmaxf(fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1])),
                   fmaxf(__uint_as_float(w[2]), __uint_as_float(w[3])));
    } else {
      using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      const T2* h = reinterpret_cast<const T2*>(&r);
      const T2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
      return fmaxf(to_f<T>(m.x), to_f<T>(m.y));
    }
  }
  // exp((z - base) / T) of the elements
  __device__ static __forceinline__ void exps(const uint4& r, float base, float c, f32x2 (&e)[N]) {
    float f[VEC];
    V::unpack(r, f);
#pragma unroll
    for (int j = 0; j < N; j++) {
      const f32x2 x = mul2(add2({f[2 * j], f[2 * j + 1]}, {-base, -base}), {c, c});
      e[j] = {ex2(x.x), ex2(x.y)};
    }
  }
  __device__ static __forceinline__ f32x2 sum(const uint4& r, float base, float c) {
    f32x2 e[N];
    exps(r, base, c, e);
#pragma unroll
    for (int o = N / 2; o > 0; o /= 2)
#pragma unroll
      for (int j = 0; j < o; j++) e[j] = add2(e[j], e[j + o]);
    return e[0];
  }
  __device__ static __forceinline__ uint4 gradient(const uint4& r, float base, float c, float a) {
    f32x2 e[N];
    exps(r, base, c, e);
    float f[VEC];
#pragma unroll
    for (int j = 0; j < N; j++) {
      const f32x2 v = mul2(e[j], {a, a});
      f[2 * j] = v.x;
      f[2 * j + 1] = v.y;
    }
    return V::pack(f);
  }
};

// Elements before an address that begin its 16 bytes.
template <typename T>
__device__ __forceinline__ int lead_of(const T* p) {
  return (int)(reinterpret_cast<uintptr_t>(p) % 16 / sizeof(T));
}

// ---- the teacher's entries ---------------------------------------------------------------------------------------
// Entry thread + i threads of a row in register i; id -1 and logit -inf where there is none.
template <int HELD>
struct Held {
  int id[HELD];
  float t[HELD];
  __device__ __forceinline__ void load(const DistillParams& p, int64_t r, int thread, int threads) {
#pragma unroll
    for (int i = 0; i < HELD; i++) {
      const int j = thread + i * threads;
      id[i] = -1;
      t[i] = -kInf;
      if (j < p.k && r < p.rows) {
        id[i] = __ldg(p.ids + r * p.ts + j);
        t[i] = __ldg(p.top + r * p.ts + j);
      }
    }
  }
  // once they have arrived: whether the thread has any
  __device__ __forceinline__ bool settle(const DistillParams& p) {
    bool some = false;
#pragma unroll
    for (int i = 0; i < HELD; i++) {
      if (id[i] < 0 || id[i] >= p.classes || t[i] == -kInf) {
        id[i] = -1;
        t[i] = -kInf;
      }
      some |= id[i] >= 0;
    }
    return some;
  }
  __device__ __forceinline__ float largest() const {
    float m = t[0];
#pragma unroll
    for (int i = 1; i < HELD; i++) m = fmaxf(m, t[i]);
    return m;
  }
};

// The entries' exponentials: of (t - largest) / T, or with the teacher's own log sum the probabilities themselves.
struct Teacher {
  double shift, inv;  // exp(t inv - shift)
  __device__ __forceinline__ Teacher(const DistillParams& p, int64_t r, float largest)
      : shift(p.whole ? (double)__ldg(p.whole + r) : largest * p.inv), inv(p.inv) {}
  __device__ __forceinline__ double at(float t) const { return t * inv - shift; }
};

// The sum of probabilities that were divided by their sum: 1, or NaN where an entry is NaN or +inf, which then is the
// whole row's gradient.
__device__ __forceinline__ double whole_of(double sum) { return (sum - sum) + 1.0; }

// A thread's share of sum e and of sum e x, where z are the entries' logits. An e is float32's least numbers at least
// (e^-100), so that at a class without probability its term is infinite; below kLightest (10^-300) it has no weight.
template <int HELD>
__device__ __forceinline__ void loss_terms(const Held<HELD>& h, const Teacher& teacher, const float (&z)[HELD], float m,
                                           double& se, double& sex) {
  se = sex = 0.0;
#pragma unroll
  for (int i = 0; i < HELD; i++) {
    if (h.id[i] < 0) continue;
    const double x = teacher.at(h.t[i]);
    const double e = exp_of(x, -100.0);
    se += e;
    if (x > kLightest) sex += e * (x - ((double)z[i] - (double)m) * teacher.inv);
  }
}
__device__ __forceinline__ void write_loss(const DistillParams& p, int64_t r, double se, double sex, Peak a) {
  const double loss = p.whole ? sex + se * log((double)a.s) : sex / se + log((double)a.s / se);
  p.loss[r] = (float)(loss * p.temperature * p.temperature);
  if (p.stats) p.stats[r] = make_float2(a.m, a.s);
}
__device__ __forceinline__ void write_nothing(const DistillParams& p, int64_t r) {
  p.loss[r] = 0.0f;
  if (p.stats) p.stats[r] = make_float2(0.0f, 0.0f);
}

// ---- rows of a warp ----------------------------------------------------------------------------------------------
// The aligned 16-byte pieces that hold a row, in shared memory (such a piece never leaves the allocation of the element
// in it); the elements of the first and last one that are not the row's become -inf.
template <typename T>
struct WarpRow {
  static constexpr int VEC = 16 / sizeof(T);
  static int bytes(int64_t classes) {
    return (int)std::min<int64_t>((classes * (int)sizeof(T) + 30) / 16 * 16, 1 << 16);
  }
  T* buf;
  __device__ __forceinline__ static int pieces(int lead, int classes) { return (lead + classes + VEC - 1) / VEC; }
  __device__ __forceinline__ void fetch(const T* z, int classes, int lane) const {
    const int lead = lead_of(z), n = pieces(lead, classes);
    const T* z0 = z - lead;
    for (int v = lane; v < n; v += 32) RowCopy<T, VEC>::copy(reinterpret_cast<uint4*>(buf) + v, z0 + v * VEC);
  }
  __device__ __forceinline__ void close(int lead, int classes, int lane) const {
    if (lane < lead) buf[lane] = from_f<T>(-kInf);
    const int tail = lead + classes + lane;
    if (tail < pieces(lead, classes) * VEC) buf[tail] = from_f<T>(-kInf);
    __syncwarp();
  }
};

template <typename T, int HELD>
__global__ void __launch_bounds__(kThreads, warp_kernel_blocks(HELD)) distill_warp_kernel(const DistillParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  auto row = [&](int turn) { return WarpRow<T>{reinterpret_cast<T*>(smem + (warp * 2 + turn) * p.row_bytes)}; };
  const int64_t step = (int64_t)gridDim.x * kWarps;
  int64_t r = (int64_t)blockIdx.x * kWarps + warp;
  const T* z = static_cast<const T*>(p.z);
  Held<HELD> next, later;  // the next row's entries, and those of the one behind it on their way
  next.load(p, r, lane, 32);
  bool some_next = __any_sync(0xffffffffu, next.settle(p));
  if (some_next) row(0).fetch(z + r * p.zs, p.classes, lane);
  copy_commit();
  later.load(p, r + step, lane, 32);
  // lane i keeps what the loss of the i-th of 32 rows is made of; they are written together
  int64_t own_r = -1;
  double own_se = 1.0, own_sex = 0.0;
  Peak own{0.0f, 0.0f};
  int kept = 0;
  for (int turn = 0; r < p.rows; r += step, turn ^= 1) {
    const Held<HELD> h = next;
    const bool some = some_next;
    next = later;
    some_next = __any_sync(0xffffffffu, next.settle(p));
    if (some_next) row(turn ^ 1).fetch(z + (r + step) * p.zs, p.classes, lane);
    copy_commit();
    later.load(p, r + 2 * step, lane, 32);
    if (!some) {
      if (lane == 0) write_nothing(p, r);
      continue;
    }
    copy_wait<1>();
    __syncwarp();
    const int lead = lead_of(z + r * p.zs), n = WarpRow<T>::pieces(lead, p.classes);
    const WarpRow<T> at = row(turn);
    at.close(lead, p.classes, lane);
    const uint4* piece = reinterpret_cast<const uint4*>(at.buf);
    float m = -kInf, zh[HELD];
    for (int v = lane; v < n; v += 32) m = fmaxf(m, Chunk<T>::largest(piece[v]));
    m = warp_max(m);
    const float base = base_of(m);
    f32x2 s2 = {0.0f, 0.0f};
    for (int v = lane; v < n; v += 32) s2 = add2(s2, Chunk<T>::sum(piece[v], base, p.c));
#pragma unroll
    for (int i = 0; i < HELD; i++) zh[i] = h.id[i] >= 0 ? to_f<T>(at.buf[lead + h.id[i]]) : 0.0f;
    const Teacher teacher(p, r, p.whole ? 0.0f : warp_max(h.largest()));
    double se, sex;
    loss_terms(h, teacher, zh, m, se, sex);
    const float s = warp_sum(s2.x + s2.y);
    se = warp_sum(se);
    sex = warp_sum(sex);
    if (lane == kept) own_r = r, own_se = se, own_sex = sex, own = {m, s};
    if (++kept == 32) {
      write_loss(p, own_r, own_se, own_sex, own);
      own_r = -1;
      kept = 0;
    }
    __syncwarp();  // the row's place is free
  }
  if (own_r >= 0) write_loss(p, own_r, own_se, own_sex, own);
  copy_wait<0>();
}

// ---- rows of a block ---------------------------------------------------------------------------------------------
// z[0, n) over a block's threads: whole 16-byte pieces from the first aligned address on, single elements around them.
template <typename T>
__device__ __forceinline__ Peak row_peak(const T* z, int n, float c) {
  constexpr int VEC = 16 / sizeof(T);
  Peak a{-kInf, 0.0f};
  auto raise = [&](float m) {
    m = fmaxf(a.m, m);
    if (m != a.m) a.s *= ex2((a.m - base_of(m)) * c);
    a.m = m;
    return base_of(m);
  };
  const int lead = lead_of(z), head = min(n, lead ? VEC - lead : 0), pieces = (n - head) / VEC, threads = blockDim.x;
  const uint4* zv = reinterpret_cast<const uint4*>(z + head);
  for (int v = threadIdx.x; v < pieces; v += 4 * threads) {
    uint4 raw[4];
#pragma unroll
    for (int i = 0; i < 4; i++) raw[i] = v + i * threads < pieces ? zv[v + i * threads] : Chunk<T>::nothing();
    const float base = raise(fmaxf(fmaxf(Chunk<T>::largest(raw[0]), Chunk<T>::largest(raw[1])),
                                   fmaxf(Chunk<T>::largest(raw[2]), Chunk<T>::largest(raw[3]))));
    f32x2 s = Chunk<T>::sum(raw[0], base, c);
#pragma unroll
    for (int i = 1; i < 4; i++)
      if (v + i * threads < pieces) s = add2(s, Chunk<T>::sum(raw[i], base, c));
    a.s += s.x + s.y;
  }
  for (int i = threadIdx.x; i < n - pieces * VEC; i += threads) {
    const float f = to_f<T>(z[i < head ? i : i + pieces * VEC]), base = raise(f);
    a.s += ex2((f - base) * c);
  }
  return a;
}

// A block, or a cluster of `splits` blocks, to a row; the first of them has the entries.
template <typename T, int HELD>
__global__ void __launch_bounds__(kThreads, 4) distill_block_kernel(const DistillParams p) {
  __shared__ Peak red[kWarps];
  __shared__ float red_t[kWarps];
  __shared__ double red_e[kWarps], red_x[kWarps];
  __shared__ Peak share;
  const int64_t r = blockIdx.x / p.splits;
  const int rank = blockIdx.x % p.splits, lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
  Held<HELD> h;
  h.load(p, r, threadIdx.x, blockDim.x);
  if (!__syncthreads_or(h.settle(p))) {  // all blocks of the row see the same
    if (rank == 0 && threadIdx.x == 0) write_nothing(p, r);
    return;
  }
  const T* z = static_cast<const T*>(p.z) + r * p.zs;
  float zh[HELD];
#pragma unroll
  for (int i = 0; i < HELD; i++) zh[i] = rank == 0 && h.id[i] >= 0 ? to_f<T>(z[h.id[i]]) : 0.0f;
  const int c0 = (int)min((int64_t)p.classes, (int64_t)rank * p.seg);
  const int c1 = (int)min((int64_t)p.classes, (int64_t)c0 + p.seg);
  Peak a = warp_peak(row_peak(z + c0, c1 - c0, p.c), p.c);
  const float mt = warp_max(h.largest());
  if (lane == 0) red[warp] = a, red_t[warp] = mt;
  __syncthreads();
  // every warp joins the warps' peaks for itself
  a = warp_peak(lane < warps ? red[lane] : Peak{-kInf, 0.0f}, p.c);
  if (p.splits > 1) {
    if (threadIdx.x == 0) share = a;
    cluster_sync();
    if (rank == 0) {
      a = {-kInf, 0.0f};
      if (lane < p.splits) {
        const uint32_t at = mapa_shared(smem_u32(&share), lane);
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(a.m), "=f"(a.s) : "r"(at) : "memory");
      }
      a = warp_peak(a, p.c);
    }
    cluster_sync();
    if (rank != 0) return;
  }
  const Teacher teacher(p, r, warp_max(lane < warps ? red_t[lane] : -kInf));
  double se, sex;
  loss_terms(h, teacher, zh, a.m, se, sex);
  se = warp_sum(se);
  sex = warp_sum(sex);
  if (lane == 0) red_e[warp] = se, red_x[warp] = sex;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < warps; w++) se += red_e[w], sex += red_x[w];
    write_loss(p, r, se, sex, a);
  }
}

// ---- backward ----------------------------------------------------------------------------------------------------
// Where entries of one class find each other: a bit for each class modulo `bits`, the bits that two entries share, and
// the entries for those that have to look.
struct Meet {
  uint32_t* seen;
  uint32_t* twice;
  int* id;
  float* p;
  uint32_t bits;
};

template <bool BLOCK>
__device__ __forceinline__ void sync_rows() {
  if (BLOCK) __syncthreads();
  else __syncwarp();
}
template <bool BLOCK>
__device__ __forceinline__ bool any_rows(bool v) {
  return BLOCK ? __syncthreads_or(v) : __any_sync(0xffffffffu, v);
}

template <bool BLOCK>
__device__ __forceinline__ void clear(const Meet& s, int thread, int threads) {
  for (uint32_t i = thread; i < s.bits / 32; i += threads) s.seen[i] = s.twice[i] = 0;
}

// `prob` of the first entry of a class becomes the sum over all of that class in their order, those of the others
// negative. The bits are clear.
template <bool BLOCK, int HELD>
__device__ __forceinline__ void join_equal(const Meet& s, const Held<HELD>& h, float (&prob)[HELD], int k, int thread,
                                           int threads) {
  bool again = false;
#pragma unroll
  for (int i = 0; i < HELD; i++) {
    if (h.id[i] < 0) continue;
    const uint32_t b = (uint32_t)h.id[i] & (s.bits - 1), bit = 1u << b % 32;
    if (atomicOr(&s.seen[b / 32], bit) & bit) {
      atomicOr(&s.twice[b / 32], bit);
      again = true;
    }
  }
  if (!any_rows<BLOCK>(again)) return;
#pragma unroll
  for (int i = 0; i < HELD; i++)
    if (thread + i * threads < k) s.id[thread + i * threads] = h.id[i], s.p[thread + i * threads] = prob[i];
  sync_rows<BLOCK>();
#pragma unroll
  for (int i = 0; i < HELD; i++) {
    if (h.id[i] < 0) continue;
    const uint32_t b = (uint32_t)h.id[i] & (s.bits - 1);
    if (!(s.twice[b / 32] >> b % 32 & 1)) continue;
    float sum = 0.0f;
    int low = -1;
    for (int j = 0; j < k; j++) {
      if (s.id[j] != h.id[i]) continue;
      if (low < 0) low = j;
      sum += s.p[j];
    }
    prob[i] = low == thread + i * threads ? sum : -1.0f;
  }
}

// dz[0, n) = a exp((z - base) / T) over a block's threads; WIDE: z and dz are equally far from 16 bytes
template <typename T, bool WIDE>
__device__ __forceinline__ void row_gradient(const T* z, T* dz, int n, float base, float c, float a) {
  constexpr int VEC = 16 / sizeof(T);
  const int threads = blockDim.x;
  int head = n, pieces = 0;
  if (WIDE) {
    const int lead = lead_of(z);
    head = min(n, lead ? VEC - lead : 0);
    pieces = (n - head) / VEC;
    const uint4* zv = reinterpret_cast<const uint4*>(z + head);
    uint4* dv = reinterpret_cast<uint4*>(dz + head);
    for (int v = threadIdx.x; v < pieces; v += 4 * threads) {
      uint4 raw[4];
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (v + i * threads < pieces) raw[i] = zv[v + i * threads];
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (v + i * threads < pieces) dv[v + i * threads] = Chunk<T>::gradient(raw[i], base, c, a);
    }
  }
  for (int i = threadIdx.x; i < n - pieces * VEC; i += threads) {
    const int at = i < head ? i : i + pieces * VEC;
    dz[at] = from_f<T>(a * ex2((to_f<T>(z[at]) - base) * c));
  }
}

template <typename T>
__device__ __forceinline__ void zero_row(T* dz, int n, int thread, int threads) {
  constexpr int VEC = 16 / sizeof(T);
  const int lead = lead_of(dz), head = min(n, lead ? VEC - lead : 0), pieces = (n - head) / VEC;
  for (int v = thread; v < pieces; v += threads) reinterpret_cast<uint4*>(dz + head)[v] = uint4{};
  for (int i = thread; i < n - pieces * VEC; i += threads) dz[i < head ? i : i + pieces * VEC] = from_f<T>(0.0f);
}

// The factors of a row's gradient: g (scale exp((z - base) / T) - p).
struct Factors {
  double g, scale;
  float base;
  __device__ __forceinline__ Factors(const DistillParams& p, int64_t r, double sum) {
    const float2 st = p.stats[r];
    g = (p.dloss ? (double)p.dloss[r] : 1.0) * p.temperature;
    scale = sum / st.y;
    base = base_of(st.x);
  }
  __device__ __forceinline__ float entry(float z, float prob, double inv) const {
    return (float)(g * (scale * exp_of(((double)z - base) * inv) - prob));
  }
};

template <typename T, bool WIDE, int HELD>
__global__ void __launch_bounds__(kThreads, warp_kernel_blocks(HELD)) distill_back_warp_kernel(const DistillParams p) {
  constexpr int VEC = 16 / sizeof(T), WORDS = kWarpClasses / 32;
  __shared__ uint32_t seen[kWarps][2][WORDS];
  __shared__ int ids[kWarps][kWarpTop];
  __shared__ float probs[kWarps][kWarpTop];
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const Meet meet{seen[warp][0], seen[warp][1], ids[warp], probs[warp], kWarpClasses};
  auto row = [&](int turn) { return WarpRow<T>{reinterpret_cast<T*>(smem + (warp * 2 + turn) * p.row_bytes)}; };
  const int64_t step = (int64_t)gridDim.x * kWarps;
  int64_t r = (int64_t)blockIdx.x * kWarps + warp;
  const T* z = static_cast<const T*>(p.z);
  Held<HELD> next, later;
  next.load(p, r, lane, 32);
  bool some_next = __any_sync(0xffffffffu, next.settle(p));
  if (some_next) row(0).fetch(z + r * p.zs, p.classes, lane);
  copy_commit();
  later.load(p, r + step, lane, 32);
  for (int turn = 0; r < p.rows; r += step, turn ^= 1) {
    const Held<HELD> h = next;
    const bool some = some_next;
    next = later;
    some_next = __any_sync(0xffffffffu, next.settle(p));
    if (some_next) row(turn ^ 1).fetch(z + (r + step) * p.zs, p.classes, lane);
    copy_commit();
    later.load(p, r + 2 * step, lane, 32);
    T* dz = static_cast<T*>(p.dz) + r * p.ds;
    if (!some) {
      zero_row(dz, p.classes, lane, 32);
      continue;
    }
    clear<false>(meet, lane, 32);
    const Teacher teacher(p, r, p.whole ? 0.0f : warp_max(h.largest()));
    float prob[HELD];
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < HELD; i++) {
      prob[i] = h.id[i] >= 0 ? exp_of(teacher.at(h.t[i])) : 0.0f;
      sum += prob[i];
    }
    sum = warp_sum(sum);
    if (!p.whole) {
      const double share = 1.0 / sum;
#pragma unroll
      for (int i = 0; i < HELD; i++) prob[i] = (float)(prob[i] * share);
      sum = whole_of(sum);
    }
    __syncwarp();
    join_equal<false>(meet, h, prob, p.k, lane, 32);
    const Factors f(p, r, sum);
    const float a = (float)(f.g * f.scale);
    copy_wait<1>();
    __syncwarp();
    const int lead = lead_of(z + r * p.zs), n = WarpRow<T>::pieces(lead, p.classes);
    const T* buf = row(turn).buf;
    // the pieces that are the row's alone as they are, the elements around them one at a time
    const int v0 = !WIDE ? n : lead ? 1 : 0, v1 = !WIDE ? n : (lead + p.classes) / VEC;
    for (int v = v0 + lane; v < v1; v += 32)
      reinterpret_cast<uint4*>(dz - lead)[v] =
          Chunk<T>::gradient(reinterpret_cast<const uint4*>(buf)[v], f.base, p.c, a);
    auto one = [&](int e) { dz[e] = from_f<T>(a * ex2((to_f<T>(buf[lead + e]) - f.base) * p.c)); };
    if (WIDE && v0 <= v1) {
      if (lead && lane < VEC - lead) one(lane);
      const int e = v1 * VEC - lead + lane;
      if (e < p.classes) one(e);
    } else {
      for (int e = lane; e < p.classes; e += 32) one(e);
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < HELD; i++)
      if (h.id[i] >= 0 && prob[i] >= 0.0f)
        dz[h.id[i]] = from_f<T>(f.entry(to_f<T>(buf[lead + h.id[i]]), prob[i], teacher.inv));
    __syncwarp();  // the row's place and the bits are free
  }
  copy_wait<0>();
}

template <typename T, bool WIDE, int HELD>
__global__ void __launch_bounds__(kThreads, 4) distill_back_block_kernel(const DistillParams p) {
  constexpr int kBits = 32768;
  __shared__ uint32_t seen[2][kBits / 32];
  __shared__ int ids[kMaxTop];
  __shared__ float probs[kMaxTop];
  __shared__ float red_t[kWarps];
  __shared__ double red_e[kWarps];
  const int64_t r = blockIdx.x / p.splits;
  const int rank = (int)(blockIdx.x % p.splits);
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
  const int c0 = (int)min((int64_t)p.classes, (int64_t)rank * p.seg);
  const int c1 = (int)min((int64_t)p.classes, (int64_t)c0 + p.seg);
  const T* z = static_cast<const T*>(p.z) + r * p.zs;
  T* dz = static_cast<T*>(p.dz) + r * p.ds;
  const Meet meet{seen[0], seen[1], ids, probs, kBits};
  Held<HELD> h;
  h.load(p, r, threadIdx.x, blockDim.x);
  clear<true>(meet, threadIdx.x, blockDim.x);
  const bool some = h.settle(p);
  const float mt = warp_max(h.largest());
  if (lane == 0) red_t[warp] = mt;
  if (!__syncthreads_or(some)) return zero_row(dz + c0, c1 - c0, threadIdx.x, blockDim.x);
  const Teacher teacher(p, r, warp_max(lane < warps ? red_t[lane] : -kInf));
  float prob[HELD], zh[HELD];
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < HELD; i++) {
    // the logits of this block's classes, before they may be written over
    zh[i] = h.id[i] >= c0 && h.id[i] < c1 ? to_f<T>(z[h.id[i]]) : 0.0f;
    prob[i] = h.id[i] >= 0 ? exp_of(teacher.at(h.t[i])) : 0.0f;
    sum += prob[i];
  }
  sum = warp_sum(sum);
  if (lane == 0) red_e[warp] = sum;
  __syncthreads();
  sum = red_e[0];
  for (int w = 1; w < warps; w++) sum += red_e[w];
  if (!p.whole) {
    const double share = 1.0 / sum;
#pragma unroll
    for (int i = 0; i < HELD; i++) prob[i] = (float)(prob[i] * share);
    sum = whole_of(sum);
  }
  join_equal<true>(meet, h, prob, p.k, threadIdx.x, blockDim.x);  // with a barrier: all logits are gathered
  const Factors f(p, r, sum);
  float entry[HELD];
#pragma unroll
  for (int i = 0; i < HELD; i++) entry[i] = f.entry(zh[i], prob[i], teacher.inv);
  row_gradient<T, WIDE>(z + c0, dz + c0, c1 - c0, f.base, p.c, (float)(f.g * f.scale));
  __syncthreads();
#pragma unroll
  for (int i = 0; i < HELD; i++)
    if (h.id[i] >= c0 && h.id[i] < c1 && prob[i] >= 0.0f) dz[h.id[i]] = from_f<T>(entry[i]);
}

// ---- host --------------------------------------------------------------------------------------------------------

// Blocks to a row, so that few rows still fill the device: `most` of them, of 4,096 classes or more. Returns the
// threads of a block: as many as keep a few 16-byte pieces each, and hold the entries.
int split_rows(DistillParams& p, int most, int bytes) {
  const int64_t want = (8 * kSmCount + p.rows - 1) / p.rows;
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({want, most, p.classes / 4096}));
  int pow2 = 1;
  while (2 * pow2 <= p.splits) pow2 *= 2;
  p.splits = pow2;
  p.seg = (int)(((int64_t)p.classes + p.splits - 1) / p.splits + 63) / 64 * 64;
  return (int64_t)p.seg * bytes <= 16384 && p.k <= kMaxTop / 2 ? kThreads / 2 : kThreads;
}

bool warp_rows(const DistillParams& p) { return p.classes <= kWarpClasses && p.k <= kWarpTop; }

// Blocks of warps that go over the rows: as many as run at once, by registers and shared memory (16 KB for the
// entries); one less than that backward in 2-byte types with more than 64 entries (60 and 64 registers).
unsigned warp_blocks(const DistillParams& p, int held) {
  const int by_rows = kMaxBlockSmem / (2 * kWarps * p.row_bytes + 16384);
  const int64_t most = (int64_t)kSmCount * std::max(1, std::min(warp_kernel_blocks(held), by_rows));
  return (unsigned)std::min<int64_t>((p.rows + kWarps - 1) / kWarps, most);
}

template <typename T, int HELD>
void forward_held(const DistillParams& p, int threads, cudaStream_t st) {
  if (warp_rows(p)) {
    allow_block_smem<distill_warp_kernel<T, HELD>>();
    distill_warp_kernel<T, HELD><<<warp_blocks(p, HELD), kThreads, (size_t)2 * kWarps * p.row_bytes, st>>>(p);
    KC_CUDA(cudaGetLastError());
    return;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.rows * p.splits));
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.splits > 1 ? 1 : 0;
  KC_CUDA(cudaLaunchKernelEx(&cfg, distill_block_kernel<T, HELD>, p));
}

template <typename T, bool WIDE, int HELD>
void backward_held(const DistillParams& p, int threads, cudaStream_t st) {
  if (warp_rows(p)) {
    allow_block_smem<distill_back_warp_kernel<T, WIDE, HELD>>();
    const size_t smem = (size_t)2 * kWarps * p.row_bytes;
    distill_back_warp_kernel<T, WIDE, HELD><<<warp_blocks(p, HELD), kThreads, smem, st>>>(p);
  } else {
    distill_back_block_kernel<T, WIDE, HELD><<<(unsigned)(p.rows * p.splits), threads, 0, st>>>(p);
  }
  KC_CUDA(cudaGetLastError());
}

template <typename T>
void forward(DistillParams p, cudaStream_t st) {
  p.row_bytes = WarpRow<T>::bytes(p.classes);
  const int threads = warp_rows(p) ? 32 : split_rows(p, 8, sizeof(T));
  if (p.k <= threads) forward_held<T, 1>(p, threads, st);
  else if (p.k <= 2 * threads) forward_held<T, 2>(p, threads, st);
  else if (p.k <= 3 * threads) forward_held<T, 3>(p, threads, st);
  else forward_held<T, 4>(p, threads, st);
}

template <typename T, bool WIDE>
void backward(DistillParams p, cudaStream_t st) {
  p.row_bytes = WarpRow<T>::bytes(p.classes);
  const int threads = warp_rows(p) ? 32 : split_rows(p, 256, sizeof(T));
  if (p.k <= threads) backward_held<T, WIDE, 1>(p, threads, st);
  else if (p.k <= 2 * threads) backward_held<T, WIDE, 2>(p, threads, st);
  else if (p.k <= 3 * threads) backward_held<T, WIDE, 3>(p, threads, st);
  else backward_held<T, WIDE, 4>(p, threads, st);
}

template <typename T>
void run_backward(const DistillParams& p, cudaStream_t st) {
  // 16-byte pieces where a row's logits and gradient are equally far from them
  const bool wide = ((uintptr_t)p.z - (uintptr_t)p.dz) % 16 == 0 &&
                    (p.rows == 1 || (p.zs - p.ds) * (int64_t)sizeof(T) % 16 == 0);
  wide ? backward<T, true>(p, st) : backward<T, false>(p, st);
}

Rows logit_rows(const kc_distill_desc& d, const void* p, int64_t stride) {
  return {p, d.rows, 1, d.classes, d.rows > 1 ? stride : 0, 0, dtype_bytes(d.dtype)};
}
Rows top_rows(const kc_distill_desc& d, const void* p) {
  return {p, d.rows, 1, d.top, d.rows > 1 ? d.top_stride : 0, 0, 4};
}

void check_desc(const kc_distill_desc* d) {
  if (!d) bad("null descriptor");
  if (d->dtype < KC_PRECISION_F32 || d->dtype > KC_PRECISION_BF16) bad("unknown dtype");
  if (d->rows < 0 || d->rows > 1 << 30) bad("rows must be 0 to 2^30");
  if (d->classes < 1 || d->classes > 1 << 30) bad("classes must be 1 to 2^30");
  if (d->top < 1 || d->top > kMaxTop) bad("top must be 1 to 1024");
  if (!(d->temperature >= 0x1p-20f && d->temperature <= kMostTemperature)) bad("temperature must be 2^-20 to 32");
}

void check_rows(const Rows& r) {
  if (!rows_in_range(r)) bad("strides must not be negative, nor reach elements beyond 2^46");
  if (!aligned_to(r.p, r.bytes)) bad("a tensor is not aligned to its element");
}

DistillParams params_of(const kc_distill_desc& d) {
  DistillParams p{};
  p.rows = d.rows;
  p.classes = d.classes;
  p.k = d.top;
  p.zs = d.rows > 1 ? d.logits_stride : 0;
  p.ds = d.rows > 1 ? d.dlogits_stride : 0;
  p.ts = d.rows > 1 ? d.top_stride : 0;
  p.temperature = d.temperature;
  p.inv = 1.0 / p.temperature;
  p.c = kLog2e / d.temperature;
  return p;
}

}  // namespace
}  // namespace kc

extern "C" int kc_distill_top(const kc_distill_desc* desc, const void* d_logits, const int32_t* d_ids,
                              const float* d_top_logits, const float* d_teacher_log_sum, float* d_loss, float* d_stats,
                              void* stream) {
  return kc::guard_entry([&] {
    using namespace kc;
    check_desc(desc);
    const kc_distill_desc d = *desc;
    const Rows z = logit_rows(d, d_logits, d.logits_stride), ids = top_rows(d, d_ids), top = top_rows(d, d_top_logits);
    for (const Rows& r : {z, ids, top}) check_rows(r);
    if (d.rows == 0) return;
    if (!d_logits || !d_ids || !d_top_logits || !d_loss) bad("null tensor");
    if (!aligned_to(d_teacher_log_sum, 4) || !aligned_to(d_loss, 4)) bad("a tensor is not aligned to its element");
    if (!aligned_to(d_stats, 8)) bad("the statistics must be 8-byte aligned");
    const Range loss{d_loss, 4 * d.rows}, stats{d_stats, 8 * d.rows}, whole{d_teacher_log_sum, 4 * d.rows};
    for (const Range& o : {loss, stats}) {
      for (const Rows& r : {z, ids, top})
        if (ranges_meet(o, r)) bad("an output overlaps an input");
      if (ranges_meet(o, whole)) bad("an output overlaps an input");
    }
    if (ranges_meet(loss, stats)) bad("the outputs overlap");
    TensorDevice dev("top logits", {d_logits, d_ids, d_top_logits, d_teacher_log_sum, d_loss, d_stats});
    DistillParams p = params_of(d);
    p.z = d_logits;
    p.ids = d_ids;
    p.top = d_top_logits;
    p.whole = d_teacher_log_sum;
    p.loss = d_loss;
    p.stats = reinterpret_cast<float2*>(d_stats);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (d.dtype == KC_PRECISION_F32) forward<float>(p, st);
    else if (d.dtype == KC_PRECISION_F16) forward<__half>(p, st);
    else forward<__nv_bfloat16>(p, st);
  });
}

extern "C" int kc_distill_top_backward(const kc_distill_desc* desc, const void* d_logits, const int32_t* d_ids,
                                       const float* d_top_logits, const float* d_teacher_log_sum, const float* d_stats,
                                       const float* d_dloss, void* d_dlogits, void* stream) {
  return kc::guard_entry([&] {
    using namespace kc;
    check_desc(desc);
    const kc_distill_desc d = *desc;
    const Rows z = logit_rows(d, d_logits, d.logits_stride), dz = logit_rows(d, d_dlogits, d.dlogits_stride),
               ids = top_rows(d, d_ids), top = top_rows(d, d_top_logits);
    for (const Rows& r : {z, dz, ids, top}) check_rows(r);
    if (d.rows == 0) return;
    if (!d_logits || !d_ids || !d_top_logits || !d_stats || !d_dlogits) bad("null tensor");
    if (!aligned_to(d_teacher_log_sum, 4) || !aligned_to(d_dloss, 4)) bad("a tensor is not aligned to its element");
    if (!aligned_to(d_stats, 8)) bad("the statistics must be 8-byte aligned");
    if (!rows_distinct(dz)) bad("rows of the output share memory");
    if (rows_overlap(dz, z) && !dz.same(z)) bad("the output overlaps an input it does not match");
    if (rows_overlap(dz, ids) || rows_overlap(dz, top)) bad("the output overlaps an input");
    for (const Range& s :
         {Range{d_stats, 8 * d.rows}, Range{d_dloss, 4 * d.rows}, Range{d_teacher_log_sum, 4 * d.rows}})
      if (ranges_meet(s, dz)) bad("the output overlaps an input");
    TensorDevice dev("top logits", {d_logits, d_ids, d_top_logits, d_teacher_log_sum, d_stats, d_dloss, d_dlogits});
    DistillParams p = params_of(d);
    p.z = d_logits;
    p.ids = d_ids;
    p.top = d_top_logits;
    p.whole = d_teacher_log_sum;
    p.stats = const_cast<float2*>(reinterpret_cast<const float2*>(d_stats));
    p.dloss = d_dloss;
    p.dz = d_dlogits;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (d.dtype == KC_PRECISION_F32) run_backward<float>(p, st);
    else if (d.dtype == KC_PRECISION_F16) run_backward<__half>(p, st);
    else run_backward<__nv_bfloat16>(p, st);
  });
}
