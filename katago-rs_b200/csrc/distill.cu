// Loss of a student's logits against a teacher's top logits, and the gradient of the logits (kc_distill_top,
// kc_distill_top_backward).
//
//   q = softmax(z / T), p_j = exp(t_j / T - L), L = log sum_j exp(t_j / T) over the row's entries or the teacher's own
//   loss = T^2 sum_j p_j (log p_j - log q_{id_j})
//   dz_i = dloss T (P q_i - sum_{j: id_j = i} p_j), P = sum_j p_j
//
// Forward, one pass over a row's logits keeps the largest and the sum of exp((z - largest) / T) in every thread and
// merges them; the entries' terms, differences of logarithms, are in 64 bits. Backward, the saved pair makes each
// element's gradient one exponential; a row's entries (their classes gathered before the row is written, so that the
// gradient may take the logits' place) are written over it at the end. Rows without entries are not read.

#include <algorithm>
#include <cmath>
#include <string>

#include "../../include/katago_cuda.h"
#include "rows.cuh"

namespace kc {
namespace {

[[noreturn]] void bad(const std::string& what) { fail(KC_ERR_INVALID, "CUDA backend: top logits: " + what); }

constexpr int kThreads = 256;
constexpr int kWarpClasses = 2048;  // rows up to this long are a warp's
constexpr int kWarpTop = 128;       // entries that a warp of the backward pass keeps in shared memory
constexpr int kMaxTop = 1024;
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
  double temperature;
  float c;          // log2(e) / T
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The largest value m (-inf: none) and s = sum of exp((z - m) / T).
struct Peak {
  float m, s;
};

// An exponent's base: 0 where there is only -inf, whose differences would be NaN.
__device__ __forceinline__ float base_of(float m) { return m == -kInf ? 0.0f : m; }

__device__ __forceinline__ Peak merge(Peak a, Peak b, float c) {
  const float m = fmaxf(a.m, b.m), base = base_of(m);
  return {m, a.s * ex2((a.m - base) * c) + b.s * ex2((b.m - base) * c)};
}

template <int N>
__device__ __forceinline__ void add_values(Peak& a, const float (&v)[N], float c) {
  float m = a.m;
#pragma unroll
  for (int j = 0; j < N; j++) m = fmaxf(m, v[j]);
  const float base = base_of(m);
  if (m != a.m) a.s *= ex2((a.m - base) * c);
  a.m = m;
#pragma unroll
  for (int j = 0; j < N; j++) a.s += ex2((v[j] - base) * c);
}

__device__ __forceinline__ Peak warp_peak(Peak a, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    a = merge(a, {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o)}, c);
  return a;
}

// z[0, n) over `threads` threads: whole 16-byte vectors from the first aligned address on, single elements around them.
template <typename T>
__device__ __forceinline__ Peak row_peak(const T* z, int n, int thread, int threads, float c) {
  constexpr int VEC = 16 / sizeof(T);
  using V = RowVec<T, VEC>;
  Peak a{-kInf, 0.0f};
  const int head = min(n, (int)((16 - (uintptr_t)z % 16) % 16 / sizeof(T)));
  const int nvec = (n - head) / VEC;
  const T* zv = z + head;
  int v = thread;
  for (; v + 3 * threads < nvec; v += 4 * threads) {
    typename V::Raw raw[4];
#pragma unroll
    for (int i = 0; i < 4; i++) raw[i] = V::load(zv + (int64_t)(v + i * threads) * VEC);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float f[VEC];
      V::unpack(raw[i], f);
      add_values(a, f, c);
    }
  }
  for (; v < nvec; v += threads) {
    float f[VEC];
    V::unpack(V::load(zv + (int64_t)v * VEC), f);
    add_values(a, f, c);
  }
  for (int i = thread; i < n - nvec * VEC; i += threads) {
    const float f[1] = {to_f<T>(z[i < head ? i : i + nvec * VEC])};
    add_values(a, f, c);
  }
  return a;
}

// The teacher's entries of a row.
struct Entries {
  const int32_t* ids;
  const float* top;
  __device__ __forceinline__ Entries(const DistillParams& p, int64_t r) : ids(p.ids + r * p.ts), top(p.top + r * p.ts) {}
  __device__ __forceinline__ bool there(const DistillParams& p, int j) const {
    const int id = __ldg(ids + j);
    return id >= 0 && id < p.classes && __ldg(top + j) != -kInf;
  }
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// L of a row, by a warp.
__device__ __forceinline__ double teacher_log_sum(const DistillParams& p, const Entries& e, int64_t r) {
  if (p.whole) return p.whole[r];
  const int lane = threadIdx.x % 32;
  float m = -kInf;
  for (int j = lane; j < p.k; j += 32)
    if (e.there(p, j)) m = fmaxf(m, __ldg(e.top + j));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  double s = 0.0;
  for (int j = lane; j < p.k; j += 32)
    if (e.there(p, j)) s += exp(((double)__ldg(e.top + j) - m) / p.temperature);
  return m / p.temperature + log(warp_sum(s));
}

// The loss of a row by a warp, from its logits' (m, s).
template <typename T>
__device__ __forceinline__ double row_loss(const DistillParams& p, const Entries& e, int64_t r, const T* z, Peak a) {
  const double log_sum = teacher_log_sum(p, e, r), log_s = log((double)a.s);
  double loss = 0.0;
  for (int j = threadIdx.x % 32; j < p.k; j += 32) {
    if (!e.there(p, j)) continue;
    const double log_p = __ldg(e.top + j) / p.temperature - log_sum, prob = exp(log_p);
    const double log_q = ((double)to_f<T>(z[__ldg(e.ids + j)]) - a.m) / p.temperature - log_s;
    if (prob != 0.0) loss += prob * (log_p - log_q);
  }
  return warp_sum(loss) * p.temperature * p.temperature;
}

__device__ __forceinline__ void write_row(const DistillParams& p, int64_t r, double loss, Peak a) {
  p.loss[r] = (float)loss;
  if (p.stats) p.stats[r] = make_float2(a.m, a.s);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) distill_warp_kernel(const DistillParams p) {
  const int lane = threadIdx.x % 32;
  const int64_t step = (int64_t)gridDim.x * (kThreads / 32);
  for (int64_t r = (int64_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32; r < p.rows; r += step) {
    const Entries e(p, r);
    bool some = false;
    for (int j = lane; j < p.k; j += 32) some |= e.there(p, j);
    if (!__any_sync(0xffffffffu, some)) {
      if (lane == 0) write_row(p, r, 0.0, {0.0f, 0.0f});
      continue;
    }
    const T* z = static_cast<const T*>(p.z) + r * p.zs;
    const Peak a = warp_peak(row_peak(z, p.classes, lane, 32, p.c), p.c);
    const double loss = row_loss(p, e, r, z, a);
    if (lane == 0) write_row(p, r, loss, a);
  }
}

// A block, or a cluster of `splits` blocks, to a row.
template <typename T>
__global__ void __launch_bounds__(kThreads) distill_block_kernel(const DistillParams p) {
  __shared__ Peak red[kThreads / 32];
  __shared__ Peak share;
  const int64_t r = blockIdx.x / p.splits;
  const int rank = blockIdx.x % p.splits, lane = threadIdx.x % 32;
  const Entries e(p, r);
  bool some = false;
  for (int j = threadIdx.x; j < p.k; j += kThreads) some |= e.there(p, j);
  if (!__syncthreads_or(some)) {  // all blocks of the row see the same
    if (rank == 0 && threadIdx.x == 0) write_row(p, r, 0.0, {0.0f, 0.0f});
    return;
  }
  const T* z = static_cast<const T*>(p.z) + r * p.zs;
  const int c0 = (int)min((int64_t)p.classes, (int64_t)rank * p.seg), c1 = (int)min((int64_t)p.classes, (int64_t)c0 + p.seg);
  Peak a = warp_peak(row_peak(z + c0, c1 - c0, threadIdx.x, kThreads, p.c), p.c);
  if (lane == 0) red[threadIdx.x / 32] = a;
  __syncthreads();
  if (threadIdx.x < 32) {
    a = warp_peak(lane < kThreads / 32 ? red[lane] : Peak{-kInf, 0.0f}, p.c);
    if (lane == 0) share = a;
  }
  if (p.splits > 1) {
    cluster_sync();
    if (rank == 0 && threadIdx.x < 32) {
      a = {-kInf, 0.0f};
      if (lane < p.splits) {
        const uint32_t at = mapa_shared(smem_u32(&share), lane);
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(a.m), "=f"(a.s) : "r"(at) : "memory");
      }
      a = warp_peak(a, p.c);
    }
    cluster_sync();
  }
  if (rank == 0 && threadIdx.x < 32) {
    const double loss = row_loss(p, e, r, z, a);
    if (lane == 0) write_row(p, r, loss, a);
  }
}

// ---- backward ----------------------------------------------------------------------------------------------------
// The entries of a row in shared memory, held by a warp or a block.
struct EntryStore {
  int* id;          // -1: absent
  float* p;         // probability, and in the end the gradient
  float* total;     // of all entries of that class; negative where an earlier entry stands for it
  uint32_t* seen;   // a bit for each class modulo `bits`
  uint32_t bits;
};

template <bool BLOCK>
__device__ __forceinline__ void sync_rows() {
  if (BLOCK) __syncthreads();
  else __syncwarp();
}

// Entries of one class become one. A class whose bit is set before it is looked for among all entries.
template <bool BLOCK>
__device__ __forceinline__ void join_equal(const EntryStore& s, int k, int thread, int threads) {
  for (uint32_t i = thread; i < s.bits / 32; i += threads) s.seen[i] = 0;
  sync_rows<BLOCK>();
  uint32_t again = 0;  // this thread's entries (at most 32) whose bit was set
  for (int j = thread, n = 0; j < k; j += threads, n++) {
    if (s.id[j] < 0) continue;
    const uint32_t b = (uint32_t)s.id[j] & (s.bits - 1);
    if (atomicOr(&s.seen[b / 32], 1u << b % 32) >> b % 32 & 1) again |= 1u << n;
  }
  for (int j = thread, n = 0; j < k; j += threads, n++) {
    if (!(again >> n & 1)) continue;
    int low = -1, count = 0;
    float sum = 0.0f;
    for (int i = 0; i < k; i++) {
      if (s.id[i] != s.id[j]) continue;
      if (low < 0) low = i;
      sum += s.p[i];
      count++;
    }
    if (count > 1)  // all threads that come here for this class write the same
      for (int i = low; i < k; i++)
        if (s.id[i] == s.id[j]) s.total[i] = i == low ? sum : -1.0f;
  }
  sync_rows<BLOCK>();
}

// dz[0, n) = a exp((z - m) / T)
template <typename T, int VEC>
__device__ __forceinline__ void row_gradient(const T* z, T* dz, int n, int thread, int threads, float m, float c, float a) {
  using V = RowVec<T, VEC>;
  const int head = VEC == 1 ? 0 : min(n, (int)((16 - (uintptr_t)z % 16) % 16 / sizeof(T)));
  const int nvec = (n - head) / VEC;
  int v = thread;
  auto one = [&](typename V::Raw raw, int at) {
    float f[VEC];
    V::unpack(raw, f);
#pragma unroll
    for (int j = 0; j < VEC; j++) f[j] = a * ex2((f[j] - m) * c);
    V::store(dz + head + (int64_t)at * VEC, V::pack(f));
  };
  for (; v + 3 * threads < nvec; v += 4 * threads) {
    typename V::Raw raw[4];
#pragma unroll
    for (int i = 0; i < 4; i++) raw[i] = V::load(z + head + (int64_t)(v + i * threads) * VEC);
#pragma unroll
    for (int i = 0; i < 4; i++) one(raw[i], v + i * threads);
  }
  for (; v < nvec; v += threads) one(V::load(z + head + (int64_t)v * VEC), v);
  for (int i = thread; i < n - nvec * VEC; i += threads) {
    const int at = i < head ? i : i + nvec * VEC;
    dz[at] = from_f<T>(a * ex2((to_f<T>(z[at]) - m) * c));
  }
}

// A row's classes [c0, c1) by a warp or a block. `log_sum` and `prob` are the same in all its threads.
template <typename T, int VEC, bool BLOCK>
__device__ __forceinline__ void back_row(const DistillParams& p, int64_t r, int c0, int c1, const EntryStore& s,
                                         int thread, int threads, double prob) {
  const T* z = static_cast<const T*>(p.z) + r * p.zs;
  T* dz = static_cast<T*>(p.dz) + r * p.ds;
  join_equal<BLOCK>(s, p.k, thread, threads);
  const float2 st = p.stats[r];
  const double g = (p.dloss ? (double)p.dloss[r] : 1.0) * p.temperature, scale = prob / st.y;
  const float base = base_of(st.x);
  for (int j = thread; j < p.k; j += threads) {
    const int id = s.id[j];
    if (id < c0 || id >= c1) continue;
    s.p[j] = (float)(g * (scale * exp(((double)to_f<T>(z[id]) - base) / p.temperature) - (double)s.total[j]));
  }
  sync_rows<BLOCK>();
  row_gradient<T, VEC>(z + c0, dz + c0, c1 - c0, thread, threads, base, p.c, (float)(g * scale));
  sync_rows<BLOCK>();
  for (int j = thread; j < p.k; j += threads) {
    const int id = s.id[j];
    if (id >= c0 && id < c1 && s.total[j] >= 0.0f) dz[id] = from_f<T>(s.p[j]);
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void zero_row(T* dz, int n, int thread, int threads) {
  using V = RowVec<T, VEC>;
  const int head = VEC == 1 ? 0 : min(n, (int)((16 - (uintptr_t)dz % 16) % 16 / sizeof(T)));
  const int nvec = (n - head) / VEC;
  for (int v = thread; v < nvec; v += threads) V::store(dz + head + (int64_t)v * VEC, typename V::Raw{});
  for (int i = thread; i < n - nvec * VEC; i += threads) dz[i < head ? i : i + nvec * VEC] = from_f<T>(0.0f);
}

// The entries and their probabilities into shared memory; the sum of these. Every warp finds L for itself.
template <bool BLOCK>
__device__ __forceinline__ double load_entries(const DistillParams& p, const Entries& e, int64_t r, const EntryStore& s,
                                               int thread, int threads, double* red) {
  const double log_sum = teacher_log_sum(p, e, r);
  double sum = 0.0;
  for (int j = thread; j < p.k; j += threads) {
    const bool there = e.there(p, j);
    const double prob = there ? exp(__ldg(e.top + j) / p.temperature - log_sum) : 0.0;
    s.id[j] = there ? __ldg(e.ids + j) : -1;
    s.p[j] = s.total[j] = (float)prob;
    sum += prob;
  }
  sum = warp_sum(sum);
  if (BLOCK) {
    if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = sum;
    __syncthreads();
    sum = 0.0;
    for (int w = 0; w < kThreads / 32; w++) sum += red[w];
  }
  return sum;
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) distill_back_warp_kernel(const DistillParams p) {
  __shared__ int id[kThreads / 32][kWarpTop];
  __shared__ float prob[kThreads / 32][kWarpTop], total[kThreads / 32][kWarpTop];
  __shared__ uint32_t seen[kThreads / 32][kWarpClasses / 32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const EntryStore s{id[warp], prob[warp], total[warp], seen[warp], kWarpClasses};
  const int64_t step = (int64_t)gridDim.x * (kThreads / 32);
  for (int64_t r = (int64_t)blockIdx.x * (kThreads / 32) + warp; r < p.rows; r += step) {
    const Entries e(p, r);
    bool some = false;
    for (int j = lane; j < p.k; j += 32) some |= e.there(p, j);
    if (!__any_sync(0xffffffffu, some)) {
      zero_row<T, VEC>(static_cast<T*>(p.dz) + r * p.ds, p.classes, lane, 32);
      continue;
    }
    __syncwarp();  // the last row's entries have been written
    const double sum = load_entries<false>(p, e, r, s, lane, 32, nullptr);
    back_row<T, VEC, false>(p, r, 0, p.classes, s, lane, 32, sum);
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) distill_back_block_kernel(const DistillParams p) {
  constexpr int kBits = 32768;
  __shared__ int id[kMaxTop];
  __shared__ float prob[kMaxTop], total[kMaxTop];
  __shared__ uint32_t seen[kBits / 32];
  __shared__ double red[kThreads / 32];
  const int64_t r = blockIdx.x / p.splits;
  const int rank = (int)(blockIdx.x % p.splits);
  const int c0 = (int)min((int64_t)p.classes, (int64_t)rank * p.seg), c1 = (int)min((int64_t)p.classes, (int64_t)c0 + p.seg);
  const Entries e(p, r);
  bool some = false;
  for (int j = threadIdx.x; j < p.k; j += kThreads) some |= e.there(p, j);
  if (!__syncthreads_or(some)) {
    zero_row<T, VEC>(static_cast<T*>(p.dz) + r * p.ds + c0, c1 - c0, threadIdx.x, kThreads);
    return;
  }
  const EntryStore s{id, prob, total, seen, kBits};
  const double sum = load_entries<true>(p, e, r, s, threadIdx.x, kThreads, red);
  back_row<T, VEC, true>(p, r, c0, c1, s, threadIdx.x, kThreads, sum);
}

// ---- host --------------------------------------------------------------------------------------------------------

// Blocks to a row, so that few rows still fill the device: `most` of them, of 4,096 classes or more.
void split_rows(DistillParams& p, int most) {
  const int64_t want = (8 * kSmCount + p.rows - 1) / p.rows;
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({want, most, p.classes / 4096}));
  int pow2 = 1;
  while (2 * pow2 <= p.splits) pow2 *= 2;
  p.splits = pow2;
  p.seg = (int)(((int64_t)p.classes + p.splits - 1) / p.splits + 63) / 64 * 64;
}

unsigned warp_blocks(int64_t rows) {
  return (unsigned)std::min<int64_t>((rows + kThreads / 32 - 1) / (kThreads / 32), 1 << 20);
}

template <typename T>
void forward(DistillParams p, cudaStream_t st) {
  if (p.classes <= kWarpClasses) {
    distill_warp_kernel<T><<<warp_blocks(p.rows), kThreads, 0, st>>>(p);
    KC_CUDA(cudaGetLastError());
    return;
  }
  split_rows(p, 8);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.rows * p.splits));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.splits > 1 ? 1 : 0;
  KC_CUDA(cudaLaunchKernelEx(&cfg, distill_block_kernel<T>, p));
}

template <typename T, int VEC>
void backward(DistillParams p, cudaStream_t st) {
  if (p.classes <= kWarpClasses && p.k <= kWarpTop) {
    distill_back_warp_kernel<T, VEC><<<warp_blocks(p.rows), kThreads, 0, st>>>(p);
  } else {
    split_rows(p, 256);
    distill_back_block_kernel<T, VEC><<<(unsigned)(p.rows * p.splits), kThreads, 0, st>>>(p);
  }
  KC_CUDA(cudaGetLastError());
}

template <typename T>
void run_backward(const DistillParams& p, cudaStream_t st) {
  // vectors where a row's logits and gradient are equally far from 16 bytes
  const bool wide = ((uintptr_t)p.z - (uintptr_t)p.dz) % 16 == 0 && (p.rows == 1 || (p.zs - p.ds) * (int64_t)sizeof(T) % 16 == 0);
  wide ? backward<T, 16 / sizeof(T)>(p, st) : backward<T, 1>(p, st);
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
  if (!(d->temperature >= 0x1p-20f && d->temperature <= 0x1p20f)) bad("temperature must be 2^-20 to 2^20");
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
    for (const Range& s : {Range{d_stats, 8 * d.rows}, Range{d_dloss, 4 * d.rows}, Range{d_teacher_log_sum, 4 * d.rows}})
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
