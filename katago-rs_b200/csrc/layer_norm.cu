// Norm of each token's row of channels (layer norm and RMS norm) on channels-last board tokens, forward and backward
// (kc_layer_norm, kc_layer_norm_backward).
//
//   mean = sum x / C (RMS: 0), var = sum (x - mean)^2 / C, rstd = 1 / sqrt(var + eps), xh = (x - mean) rstd,
//   y = xh w + b where the token is on, 0 elsewhere
//   g = dy w, c1 = sum g / C (RMS: 0), c2 = sum g xh / C, dx = rstd (g - c1 - xh c2) where on,
//   dweight = sum over tokens of dy xh, dbias = of dy
//
// A row stays in the registers of a group of lanes (2 to 32 of a warp, or a block) between the sums and the output:
// one read, one write. Forward, the variance is taken around the float32 mean of the first pass, whose own error the
// second pass finds (the sum of the distances), so that a large mean costs neither digits of the variance nor of
// x - mean. Backward, x - mean is from the saved mean, one float32: xh is off by up to |mean| rstd 2^-24 in a whole row
// (6e-4 under a mean of 10^4 times the spread), and dx and dweight with it. A block goes over many rows there and keeps
// the channels' sums in registers; a second launch adds the blocks' in their order (few rows: a cluster adds its own).
// Rows that registers do not hold (more than 16,384 channels forward, 8,192 backward) are read again for each pass.
//
// What bounds it: HBM in the large, with 341 warp instructions a pair of rows of 384 next to it (62% of the issue
// slots), of 16 to 24 warps an SM that hold their rows and sums in registers. The rows behind the one at hand are on
// their way into shared memory (loads straight into registers, one row at a time: 62 us where the ring takes 27); a
// mask is looked at a row after it was asked for (34 us without). Measured on a B200 (6,549 GB/s copy), bytes that have
// to move / time:
//   forward, 256 boards x 361 x 384, layer norm, masked: bf16 120 MB in 25.6 us, 4,680 GB/s; float32 239 MB in 43.1 us,
//     5,540 GB/s
//   the same, RMS norm, no mask: bf16 143 MB in 25.9 us, 5,510 GB/s; float32 285 MB in 50.4 us, 5,650 GB/s
//   forward, 64 x 361 x 768, layer norm, float32: 142 MB in 24.5 us, 5,800 GB/s
//   backward, 128 x 361 x 768, RMS norm, bf16: 213 MB in 41.4 us, 5,160 GB/s
//   backward, 256 x 361 x 384, RMS norm, float32: 427 MB in 74.5 us, 5,730 GB/s
//   the same, layer norm, masked: bf16 168 MB in 39.2 us, 4,280 GB/s; float32 334 MB in 63.5 us, 5,260 GB/s
// further from it: 2-byte rows of 16 elements a lane (forward, 256 x 361 x 128, 256 and 512, RMS norm, bf16: 12.0, 20.2
// and 36.4 us of 7.3, 14.6 and 29.0), rows that begin anywhere (forward 256 x 361 x 384 of 387: 42.5 us, a window of 19
// instructions each way a vector), rows of a block (forward 9,000 x 4,096, bf16, RMS: 36.5 us of 22.5; barriers),
// single elements there (5,000 x 4,099: 93 us of 12.5), rows read again (backward 1,000 x 20,000, float32: 150 us of
// 37).

#include <algorithm>
#include <cmath>
#include <string>

#include "../../include/katago_cuda.h"
#include "rows.cuh"

namespace kc {
namespace {

[[noreturn]] void bad(const std::string& what) { fail(KC_ERR_INVALID, "CUDA backend: layer norm: " + what); }

constexpr int kThreads = 256;
constexpr int kLongThreads = 512;

struct LayerParams {
  const void* x;
  const float* mask;
  const float* weight;
  const float* bias;
  void* y;         // forward: y; backward: dx
  const void* dy;
  float2* stats;   // (mean, rstd) of a token: written by the forward pass (may be null), read by the backward
  float* part;     // backward: the blocks' sums of dy xh and of dy, [blocks][2][slots] (PartShape)
  float* dweight;
  float* dbias;
  RowMap xm, ym, mm;
  int64_t rows;
  int C, lanes;
  int kind;
  int wide;        // weight and bias are 16-byte aligned
  int cluster;     // backward: all blocks are one cluster of so many, which adds their sums itself; 0: `part`
  float eps, least, slack;  // rstd_of
};

__device__ __forceinline__ float token_mask(const LayerParams& p, int64_t r) {
  return p.mask ? __ldg(p.mask + p.mm(r)) : 1.0f;
}
__device__ __forceinline__ bool token_on(const LayerParams& p, int64_t r) { return token_mask(p, r) != 0.0f; }

// 1 / sqrt(var + eps) of a sum of squares around a value that is `delta` from the mean; NaN where the squares passed
// float32's range. Without an eps NaN too where the variance is 0. A row of equal values has the same distance from its
// first mean everywhere, mostly not 0, and a variance that is the rounding of two sums of its square: `slack` (1 with
// an eps) makes that negative, and `least` (0 with an eps, otherwise -inf) leaves it so.
__device__ __forceinline__ float rstd_of(const LayerParams& p, float squares, float inv, float delta) {
  const float var = squares * inv - delta * p.slack * delta;
  if (!(squares <= 3.402823466e38f)) return __int_as_float(0x7fffffff);
  return __frsqrt_rn(fmaxf(var, p.least) + p.eps);
}

// A row's lanes: `lanes` neighbours of a warp, or a block.
template <bool BLOCK>
struct Group {
  int lane, lanes;
  int64_t first, step;
  __device__ __forceinline__ explicit Group(int row_lanes) {
    if (BLOCK) {
      lanes = blockDim.x;
      lane = threadIdx.x;
      first = blockIdx.x;
      step = gridDim.x;
    } else {
      lanes = row_lanes;
      lane = threadIdx.x & (row_lanes - 1);
      const int per = kThreads / row_lanes;
      first = (int64_t)blockIdx.x * per + threadIdx.x / row_lanes;
      step = (int64_t)gridDim.x * per;
    }
  }
  template <typename F>
  __device__ __forceinline__ F sum(F v, float2* red) const {
    return BLOCK ? block_sum(v, red) : lanes_sum(v, lanes);
  }
};

// A warp's lanes stay together for the sums: a group behind the last row takes part with nothing.
template <bool BLOCK>
__device__ __forceinline__ bool rows_left(int64_t r, int64_t rows) {
  return BLOCK ? r < rows : __any_sync(0xffffffffu, r < rows);
}

// A thread's NV vectors as pairs of elements, for the two-lane float32 arithmetic: a unit is a vector, or two vectors
// of one element. Pair j of unit u has elements 2 j and 2 j + 1 of both vectors' elements.
template <int VEC, int NV>
struct Units {
  static_assert(NV * VEC % 2 == 0, "whole pairs");
  static constexpr int U = VEC == 1 ? NV / 2 : NV, N = VEC == 1 ? 1 : VEC / 2;
  f32x2 v[U][N];

  __device__ __forceinline__ void fill(float f) {
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int j = 0; j < N; j++) v[u][j] = {f, f};
  }
  __device__ __forceinline__ float element(int e) const {
    const f32x2 q = v[e / (2 * N)][e / 2 % N];
    return e % 2 ? q.y : q.x;
  }
};

// Rows of a ring, whose thread takes `row` bytes for each.
constexpr int ring_depth(int row, bool backward) { return !backward && row * 4 <= 420 ? 4 : row * 3 <= 420 ? 3 : 2; }

// A thread's vectors of the next rows, on their way into shared memory of its own (DEPTH rows, the one at hand among
// them; no more than what 512 threads of an SM have room for). Rows that are off are not copied.
// SHIFT: rows that begin anywhere. The aligned 16-byte pieces that hold the row are copied (such a piece never leaves
// the allocation of the element in it), and a vector is a window over its own piece and the next one, which a neighbour
// has; its warp's lanes have to be done with a row before the next one takes its place.
template <typename T, int VEC, int NV, bool BLOCK, int TENSORS, bool SHIFT>
struct Ring {
  using Copy = RowCopy<T, VEC>;
  using Slot = typename Copy::Slot;
  static constexpr int SLOTS = SHIFT ? NV + 1 : NV;  // of a tensor's row
  static constexpr int ROW = TENSORS * SLOTS * (int)sizeof(Slot);
  static constexpr int DEPTH = ring_depth(ROW, TENSORS == 2);
  static size_t bytes(int threads) { return (size_t)DEPTH * ROW * threads; }

  Slot* mine;
  int stage = 0;      // of the row at hand
  int64_t next;       // the row to copy next
  float next_mask;    // looked at a row later, when it has arrived
  uint32_t on = 0;    // a bit for each stage
  // 4 bits for each stage: where the row begins in its first piece; or whether the thread's single 2-byte elements (its
  // lanes are an even number apart) are the upper halves of 4 bytes
  uint32_t begin[TENSORS] = {};

  __device__ __forceinline__ Slot* at(int s, int tensor, int i) const {
    return mine + (s * TENSORS * SLOTS + tensor * SLOTS + i) * (BLOCK ? (int)blockDim.x : kThreads);
  }
  __device__ __forceinline__ void look(const LayerParams& p) { next_mask = next < p.rows ? token_mask(p, next) : 0.0f; }
  __device__ __forceinline__ void fetch_row(const T* row, int tensor, const Group<BLOCK>& g, int C, int s) {
    const T* src = row + g.lane * VEC;
    int n = C / VEC;
    if constexpr (SHIFT || Copy::BYTES == 2) {
      const uint32_t low = SHIFT ? (uint32_t)reinterpret_cast<uintptr_t>(row) & 15u
                                 : (uint32_t)(reinterpret_cast<uintptr_t>(src) >> 1) & 1u;
      begin[tensor] = (begin[tensor] & ~(15u << 4 * s)) | low << 4 * s;
      if (SHIFT) {
        src = reinterpret_cast<const T*>(reinterpret_cast<uintptr_t>(row) - low) + g.lane * VEC;
        n = (int)(low + C * sizeof(T) + 15) / 16;
      }
    }
    src = Copy::base(src);
#pragma unroll
    for (int i = 0; i < SLOTS; i++, src += g.lanes * VEC)
      if (g.lane + i * g.lanes < n) Copy::copy(at(s, tensor, i), src);
  }
  __device__ __forceinline__ void fetch(const LayerParams& p, const Group<BLOCK>& g, int s) {
    const bool next_on = next_mask != 0.0f;
    on = (on & ~(1u << s)) | (next_on ? 1u << s : 0u);
    if (next_on) {
      fetch_row(static_cast<const T*>(p.x) + p.xm(next), 0, g, p.C, s);
      if (TENSORS == 2) fetch_row(static_cast<const T*>(p.dy) + p.ym(next), TENSORS - 1, g, p.C, s);
    }
    copy_commit();
    next += g.step;
    look(p);
  }
  __device__ __forceinline__ void start(const LayerParams& p, const Group<BLOCK>& g, void* smem) {
    mine = static_cast<Slot*>(smem) + threadIdx.x;
    next = g.first;
    look(p);
#pragma unroll
    for (int s = 0; s < DEPTH - 1; s++) fetch(p, g, s);
  }
  // The row at hand is there afterwards, and one more is on its way.
  __device__ __forceinline__ bool arrive(const LayerParams& p, const Group<BLOCK>& g) {
    if (SHIFT) __syncwarp();
    fetch(p, g, stage == 0 ? DEPTH - 1 : stage - 1);
    copy_wait<DEPTH - 1>();
    if (SHIFT) __syncwarp();
    return on >> stage & 1;
  }
  // unit u of the row at hand; of a vector that ends behind the row, `rest` elements. What stands beside them is 0, but
  // in the backward pass's x another element of the row: 0 is so far from a large mean that its xh may pass float32.
  __device__ __forceinline__ void get(int tensor, int u, const Group<BLOCK>& g, int nvec, int rest,
                                      f32x2 (&v)[Units<VEC, NV>::N]) const {
    float f[VEC];
    if constexpr (VEC == 1) {
      float e[2];
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const int i = 2 * u + k, c = g.lane + i * g.lanes;
        f[0] = k == 1 && TENSORS == 2 && tensor == 0 ? e[0] : 0.0f;
        if (c < nvec) Copy::unpack(*at(stage, tensor, i), begin[tensor] >> 4 * stage & 1, f);
        e[k] = f[0];
      }
      v[0] = {e[0], e[1]};
      return;
    }
    if constexpr (SHIFT) {
      // the last of the group's lanes goes on at the first one's next slot
      const Slot* own = at(stage, tensor, u);
      const Slot* other = g.lane == g.lanes - 1 ? at(stage, tensor, u + 1) - (g.lanes - 1) : own + 1;
      uint4 raw = window<sizeof(T), false>(*own, *other, begin[tensor] >> 4 * stage & 15);
      if (rest && g.lane + u * g.lanes == nvec - 1) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&raw);
        const uint32_t first = sizeof(T) == 4 ? w[0] : w[0] << 16 | (w[0] & 0xffffu);
        const uint32_t fill = TENSORS == 2 && tensor == 0 ? first : 0u;
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int bytes = rest * (int)sizeof(T) - 4 * k;
          w[k] = bytes >= 4 ? w[k] : bytes <= 0 ? fill : (w[k] & 0xffffu) | (fill & 0xffff0000u);
        }
      }
      Copy::unpack(raw, false, f);
    } else {
      Copy::unpack(*at(stage, tensor, u), false, f);
    }
    if constexpr (VEC > 1) {
#pragma unroll
      for (int j = 0; j < VEC / 2; j++) v[j] = {f[2 * j], f[2 * j + 1]};
    }
  }
  __device__ __forceinline__ void leave() { stage = stage == DEPTH - 1 ? 0 : stage + 1; }
};

// A thread's place in a row: which of its units there are, and their way out.
template <int VEC, int NV, bool BLOCK, bool SHIFT>
struct Place {
  using U = Units<VEC, NV>;
  const Group<BLOCK>& g;
  int nvec, rest;  // vectors of the row; SHIFT: elements of the last one, 0 where it is whole
  __device__ __forceinline__ Place(const Group<BLOCK>& group, int C)
      : g(group), nvec(SHIFT ? (C + VEC - 1) / VEC : C / VEC), rest(SHIFT ? C % VEC : 0) {}
  __device__ __forceinline__ bool has(int i) const { return g.lane + i * g.lanes < nvec; }  // vector i
  __device__ __forceinline__ bool has_unit(int u) const { return has(VEC == 1 ? 2 * u : u); }
  // `f` in the elements of pair j of unit u that there are
  __device__ __forceinline__ f32x2 both(int u, int j, float f) const {
    if (VEC == 1) return {f, has(2 * u + 1) ? f : 0.0f};
    if (SHIFT && rest && g.lane + u * g.lanes == nvec - 1)
      return {2 * j < rest ? f : 0.0f, 2 * j + 1 < rest ? f : 0.0f};
    return {f, f};
  }
  template <typename T>
  __device__ __forceinline__ static typename RowVec<T, VEC>::Raw pack(const f32x2 (&v)[U::N]) {
    float f[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) f[j] = j % 2 ? v[j / 2].y : v[j / 2].x;
    return RowVec<T, VEC>::pack(f);
  }
  template <typename T>
  __device__ __forceinline__ void store(T* row, int u, const f32x2 (&v)[U::N], uint32_t keep) const {
    using V = RowVec<T, VEC>;
    if constexpr (VEC == 1) {
      const float a[1] = {v[0].x}, b[1] = {v[0].y};
      V::store(row + g.lane + 2 * u * g.lanes, masked(V::pack(a), keep));
      if (has(2 * u + 1)) V::store(row + g.lane + (2 * u + 1) * g.lanes, masked(V::pack(b), keep));
    } else {
      V::store(row + (g.lane + u * g.lanes) * VEC, masked(pack<T>(v), keep));
    }
  }
  template <typename T>
  __device__ __forceinline__ void zero(T* row) const {
#pragma unroll
    for (int i = 0; i < NV; i++)
      if (has(i)) RowVec<T, VEC>::store(row + (g.lane + i * g.lanes) * VEC, typename RowVec<T, VEC>::Raw{});
  }
  // SHIFT: all vectors of a row that begins anywhere, by all lanes of the warp: a piece is a window over the vector
  // before and its own; the pieces that hold other rows' elements go out element by element. Nothing where `here` is
  // false.
  template <typename T>
  __device__ __forceinline__ void store_shifted(T* row, int C, const uint4 (&raw)[NV], bool here) const {
    const uint32_t low = (uint32_t)reinterpret_cast<uintptr_t>(row) & 15u;
    const int skip = (int)(low / sizeof(T)), from = g.lane == 0 ? g.lanes - 1 : g.lane - 1;
    const bool last = g.lane == g.lanes - 1;
    uint4* out = reinterpret_cast<uint4*>(reinterpret_cast<uintptr_t>(row) - low);
#pragma unroll
    for (int i = 0; i <= NV; i++) {
      const uint4 own = i < NV ? raw[i < NV ? i : 0] : uint4{};
      const uint4 give = last && i > 0 ? raw[i > 0 ? i - 1 : 0] : own;
      uint4 before;
      before.x = __shfl_sync(0xffffffffu, give.x, from, g.lanes);
      before.y = __shfl_sync(0xffffffffu, give.y, from, g.lanes);
      before.z = __shfl_sync(0xffffffffu, give.z, from, g.lanes);
      before.w = __shfl_sync(0xffffffffu, give.w, from, g.lanes);
      const uint4 piece = window<sizeof(T), true>(before, own, 16 - low);
      const int v = g.lane + i * g.lanes, c = v * VEC - skip;
      if (!here || c >= C) continue;
      if (c >= 0 && c + VEC <= C) {
        out[v] = piece;
      } else {
        const T* e = reinterpret_cast<const T*>(&piece);
#pragma unroll
        for (int j = 0; j < VEC; j++)
          if (c + j >= 0 && c + j < C) row[c + j] = e[j];
      }
    }
  }
  __device__ __forceinline__ void load(U& w, const float* p, float otherwise, bool wide) const {
    w.fill(otherwise);
    if (!p) return;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      if (!has(i)) continue;
      const float* q = p + (g.lane + i * g.lanes) * VEC;
      float f[VEC];
      if (SHIFT && rest && g.lane + i * g.lanes == nvec - 1) {
#pragma unroll
        for (int j = 0; j < VEC; j++) f[j] = j < rest ? __ldg(q + j) : otherwise;
      } else {
        load_params<VEC>(q, wide, f);
      }
      if constexpr (VEC == 1) {
        if (i % 2) w.v[i / 2][0].y = f[0];
        else w.v[i / 2][0].x = f[0];
      } else {
#pragma unroll
        for (int j = 0; j < VEC / 2; j++) w.v[i][j] = {f[2 * j], f[2 * j + 1]};
      }
    }
  }
};

// y = xh w + b of the units of a thread, with its weights and biases in registers or, SHARED, in the block's shared
// memory (16-byte parts of all vectors side by side, each read without a conflict). Shared where that makes room for a
// third block on an SM: 24 elements of 2 bytes a lane, 256 boards x 361 x 384 layer norm, bf16, 25.6 us and 27.2 in
// registers; float32 rows, whose ring leaves room for two blocks, lose (64 x 361 x 768: 32.6 and 24.8 us), and so do 8
// elements, which registers let run four blocks at once (2,000,000 x 16, bf16: 40.7 and 33.3 us). 16 elements of 2
// bytes run two blocks from registers and would gain too, which is not made use of yet (256 boards x 361 x 128, 256 and
// 512, layer norm, bf16, masked: 14.2, 22.9 and 40.5 us, from shared memory 12.9, 20.2 and 35.2).
template <int VEC, int NV, bool BLOCK, bool SHIFT, bool SHARED>
struct Affine {
  using At = Place<VEC, NV, BLOCK, SHIFT>;
  using U = Units<VEC, NV>;
  static size_t bytes(int C) { return SHARED ? 2 * C * sizeof(float) : 0; }
  U w, b;
  const float4* ws;
  __device__ __forceinline__ void start(const At& at, const LayerParams& p, void* smem) {
    if constexpr (SHARED) {
      constexpr int Q = VEC / 4;
      float4* to = static_cast<float4*>(smem);
      ws = to;
      for (int i = threadIdx.x; i < p.C / 4; i += kThreads) {
        float wi[4] = {1.0f, 1.0f, 1.0f, 1.0f}, bi[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (p.weight) load_params<4>(p.weight + 4 * i, p.wide, wi);
        if (p.bias) load_params<4>(p.bias + 4 * i, p.wide, bi);
        to[i % Q * at.nvec + i / Q] = make_float4(wi[0], wi[1], wi[2], wi[3]);
        to[(Q + i % Q) * at.nvec + i / Q] = make_float4(bi[0], bi[1], bi[2], bi[3]);
      }
      __syncthreads();
    } else {
      at.load(w, p.weight, 1.0f, p.wide);
      at.load(b, p.bias, 0.0f, p.wide);
    }
  }
  __device__ __forceinline__ void apply(const At& at, int u, f32x2 (&x)[U::N]) const {
    if constexpr (SHARED) {
      constexpr int Q = VEC / 4;
      const float4* mine = ws + at.g.lane + u * at.g.lanes;
#pragma unroll
      for (int q = 0; q < Q; q++) {
        const float4 wq = mine[q * at.nvec], bq = mine[(Q + q) * at.nvec];
        x[2 * q] = fma2(x[2 * q], {wq.x, wq.y}, {bq.x, bq.y});
        x[2 * q + 1] = fma2(x[2 * q + 1], {wq.z, wq.w}, {bq.z, bq.w});
      }
    } else {
#pragma unroll
      for (int j = 0; j < U::N; j++) x[j] = fma2(x[j], w.v[u][j], b.v[u][j]);
    }
  }
};
constexpr bool shared_params(int vec, int nv, bool block, bool shift) {
  return !block && !shift && vec == 8 && nv == 3;
}

constexpr int kBlockThreads = 512;  // of blocks that share a row, at most: 128 registers each

template <typename T, int VEC, int NV, bool BLOCK, bool SHIFT>
__global__ void __launch_bounds__(BLOCK ? kBlockThreads : kThreads,
                                  BLOCK ? 1 : shared_params(VEC, NV, BLOCK, SHIFT) ? 3 : 2)
    layer_norm_kernel(const LayerParams p) {
  using U = Units<VEC, NV>;
  __shared__ float2 red[2][32];
  extern __shared__ __align__(16) uint8_t smem[];
  const Group<BLOCK> g(p.lanes);
  const Place<VEC, NV, BLOCK, SHIFT> at(g, p.C);
  const float inv = 1.0f / (float)p.C;
  const bool layer = p.kind == KC_NORM_LAYER;
  Ring<T, VEC, NV, BLOCK, 1, SHIFT> ring;
  ring.start(p, g, smem);
  Affine<VEC, NV, BLOCK, SHIFT, shared_params(VEC, NV, BLOCK, SHIFT)> affine;
  affine.start(at, p, smem + decltype(ring)::DEPTH * decltype(ring)::ROW * kThreads);
  int turn = 0;  // a block's sums in a row take turns with `red`
  for (int64_t r = g.first; rows_left<BLOCK>(r, p.rows); r += g.step, ring.leave()) {
    const bool here = r < p.rows, on = ring.arrive(p, g);
    T* out = static_cast<T*>(p.y) + (here ? p.ym(r) : 0);
    if (BLOCK ? !on : !__any_sync(0xffffffffu, on)) {
      if (here && p.stats && g.lane == 0) p.stats[r] = make_float2(0.0f, 0.0f);
      if constexpr (SHIFT) {
        const uint4 nothing[NV] = {};
        at.store_shifted(out, p.C, nothing, here);
      } else if (here) {
        at.zero(out);
      }
      continue;
    }
    // a warp whose rows are on in part goes over all of them; what its other slots hold is dropped in the end
    U x;
    f32x2 s1 = {0.0f, 0.0f}, s2 = s1;
#pragma unroll
    for (int u = 0; u < U::U; u++) {
      if (!at.has_unit(u)) continue;
      ring.get(0, u, g, at.nvec, at.rest, x.v[u]);
      if (layer)
#pragma unroll
        for (int j = 0; j < U::N; j++) s1 = add2(s1, x.v[u][j]);
    }
    float m0 = 0.0f, delta = 0.0f, squares;
    if (layer) {
      m0 = g.sum(s1.x + s1.y, red[turn ^= 1]) * inv;
      s1 = {0.0f, 0.0f};
#pragma unroll
      for (int u = 0; u < U::U; u++) {
        if (!at.has_unit(u)) continue;
#pragma unroll
        for (int j = 0; j < U::N; j++) {
          x.v[u][j] = add2(x.v[u][j], at.both(u, j, -m0));
          s1 = add2(s1, x.v[u][j]);
          s2 = fma2(x.v[u][j], x.v[u][j], s2);
        }
      }
      const float2 s = g.sum(make_float2(s1.x + s1.y, s2.x + s2.y), red[turn ^= 1]);
      delta = s.x * inv;
      squares = s.y;
    } else {
#pragma unroll
      for (int u = 0; u < U::U; u++) {
        if (!at.has_unit(u)) continue;
#pragma unroll
        for (int j = 0; j < U::N; j++) s2 = fma2(x.v[u][j], x.v[u][j], s2);
      }
      squares = g.sum(s2.x + s2.y, red[turn ^= 1]);
    }
    if (!SHIFT && !here) continue;
    const float rstd = rstd_of(p, squares, inv, delta);
    if (here && p.stats && g.lane == 0) p.stats[r] = on ? make_float2(m0 + delta, rstd) : make_float2(0.0f, 0.0f);
    const f32x2 scale = {rstd, rstd}, shift = {-delta * rstd, -delta * rstd};
    const uint32_t keep = on ? 0xffffffffu : 0u;
    uint4 raw[SHIFT ? NV : 1];
#pragma unroll
    for (int u = 0; u < U::U; u++) {
      if constexpr (SHIFT) raw[u] = uint4{};
      if (!at.has_unit(u)) continue;
#pragma unroll
      for (int j = 0; j < U::N; j++) x.v[u][j] = fma2(x.v[u][j], scale, shift);
      affine.apply(at, u, x.v[u]);
      if constexpr (SHIFT) raw[u] = masked(at.template pack<T>(x.v[u]), keep);
      else at.store(out, u, x.v[u], keep);
    }
    if constexpr (SHIFT) at.store_shifted(out, p.C, raw, here);
  }
  copy_wait<0>();
}

// LEAN: RMS norm without a bias, which needs no sum of g and none of dy.
// 128 registers do not hold 24 elements a lane of rows that begin anywhere: LEAN spills 188 bytes a thread (2-byte
// types; 128 x 361 x 767, bf16: 82.5 us of 32.5) or 452 (float32: 117 us of 65); without LEAN float32 spills 72 and,
// with 16 elements, 88.
template <typename T, int VEC, int NV, bool BLOCK, bool SHIFT, bool LEAN>
__global__ void __launch_bounds__(BLOCK ? kBlockThreads : kThreads, BLOCK ? 1 : 2)
    layer_norm_back_kernel(const LayerParams p) {
  using U = Units<VEC, NV>;
  constexpr bool AGAIN = !LEAN && (BLOCK || NV * VEC > 16);  // xh and g are made twice where registers do not hold them
  __shared__ float2 red[2][32];
  extern __shared__ __align__(16) uint8_t smem[];
  const Group<BLOCK> g(p.lanes);
  const Place<VEC, NV, BLOCK, SHIFT> at(g, p.C);
  const float inv = 1.0f / (float)p.C;
  pdl_trigger();
  Ring<T, VEC, NV, BLOCK, 2, SHIFT> ring;
  ring.start(p, g, smem);
  U aw, ab, w;
  aw.fill(0.0f);
  ab.fill(0.0f);
  at.load(w, p.weight, 1.0f, p.wide);
  int turn = 0;  // a block's sums of the rows that are on take turns with `red`
  float2 st_next = g.first < p.rows ? p.stats[g.first] : make_float2(0.0f, 0.0f);
  for (int64_t r = g.first; rows_left<BLOCK>(r, p.rows); r += g.step, ring.leave()) {
    const bool here = r < p.rows, on = ring.arrive(p, g);
    const float2 st = st_next;
    if (r + g.step < p.rows) st_next = p.stats[r + g.step];
    T* out = static_cast<T*>(p.y) + (here ? p.xm(r) : 0);
    if (BLOCK ? !on : !__any_sync(0xffffffffu, on)) {
      if constexpr (SHIFT) {
        const uint4 nothing[NV] = {};
        at.store_shifted(out, p.C, nothing, here);
      } else if (here) {
        at.zero(out);
      }
      continue;
    }
    // xh and g of the row, for its sums and then for dx (where dy has no element it is 0, and xh plays no part)
    U xh, gw;
    f32x2 s1 = {0.0f, 0.0f}, s2 = s1;
    const f32x2 back = {-st.x, -st.x}, scale = {st.y, st.y};
    if (on) {
#pragma unroll
      for (int u = 0; u < U::U; u++) {
        if (!at.has_unit(u)) continue;
        ring.get(0, u, g, at.nvec, at.rest, xh.v[u]);
        f32x2 d[U::N];
        ring.get(1, u, g, at.nvec, at.rest, d);
#pragma unroll
        for (int j = 0; j < U::N; j++) {
          xh.v[u][j] = mul2(add2(xh.v[u][j], back), scale);
          const f32x2 gj = mul2(d[j], w.v[u][j]);
          aw.v[u][j] = fma2(d[j], xh.v[u][j], aw.v[u][j]);
          s2 = fma2(gj, xh.v[u][j], s2);
          if constexpr (!LEAN) {
            ab.v[u][j] = add2(ab.v[u][j], d[j]);
            s1 = add2(s1, gj);
          }
          if constexpr (!AGAIN) gw.v[u][j] = gj;
        }
      }
    }
    float2 s;
    if constexpr (LEAN) s = make_float2(0.0f, g.sum(s2.x + s2.y, red[turn ^= 1]));
    else s = g.sum(make_float2(s1.x + s1.y, s2.x + s2.y), red[turn ^= 1]);
    if (!SHIFT && !here) continue;
    // rstd (g - c1 - xh c2)
    const float k1 = p.kind == KC_NORM_LAYER ? -s.x * inv * st.y : 0.0f, k2 = -s.y * inv * st.y;
    const f32x2 c1 = {k1, k1}, c2 = {k2, k2};
    const uint32_t keep = on ? 0xffffffffu : 0u;
    if constexpr (AGAIN) asm volatile("" ::: "memory");
    uint4 raw[SHIFT ? NV : 1];
#pragma unroll
    for (int u = 0; u < U::U; u++) {
      if constexpr (SHIFT) raw[u] = uint4{};
      if (!at.has_unit(u)) continue;
      f32x2 o[U::N];
      if constexpr (AGAIN) {
        ring.get(1, u, g, at.nvec, at.rest, o);
        ring.get(0, u, g, at.nvec, at.rest, xh.v[u]);
      }
#pragma unroll
      for (int j = 0; j < U::N; j++) {
        if (AGAIN) xh.v[u][j] = mul2(add2(xh.v[u][j], back), scale);
        const f32x2 gj = AGAIN ? mul2(o[j], w.v[u][j]) : gw.v[u][j];
        o[j] = fma2(gj, scale, fma2(xh.v[u][j], c2, c1));
      }
      if constexpr (SHIFT) raw[u] = masked(at.template pack<T>(o), keep);
      else at.store(out, u, o, keep);
    }
    if constexpr (SHIFT) at.store_shifted(out, p.C, raw, here);
  }
  copy_wait<0>();
  if (!p.dweight && !p.dbias) return;
  // slot (which, i, j, lane) holds the sum of channel (lane + i lanes) VEC + j (element i VEC + j)
  constexpr int E = NV * VEC;
  const int slots = E * g.lanes;
  float* part = p.part + (size_t)blockIdx.x * 2 * slots;
  if (BLOCK) {
#pragma unroll
    for (int e = 0; e < E; e++) {
      part[e * g.lanes + g.lane] = aw.element(e);
      if (!LEAN) part[slots + e * g.lanes + g.lane] = ab.element(e);
    }
    return;
  }
  // a warp's groups in registers, then the warps' sums in shared memory, where the rows were
  __syncthreads();
  float* sums = reinterpret_cast<float*>(smem);
  const int warp = threadIdx.x / 32;
#pragma unroll
  for (int e = 0; e < E; e++) {
    float a = aw.element(e), b = ab.element(e);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      if (o >= g.lanes) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        if (!LEAN) b += __shfl_xor_sync(0xffffffffu, b, o);
      }
    if (threadIdx.x % 32 < g.lanes) {
      sums[(warp * 2 * E + e) * g.lanes + g.lane] = a;
      if (!LEAN) sums[((warp * 2 + 1) * E + e) * g.lanes + g.lane] = b;
    }
  }
  __syncthreads();
  const int all = (LEAN ? 1 : 2) * slots;
  for (int k = threadIdx.x; k < all; k += kThreads) {
    float s = 0.0f;
#pragma unroll
    for (int v = 0; v < kThreads / 32; v++) s += sums[v * 2 * slots + k];
    if (p.cluster) sums[k] = s;  // read by this thread alone so far
    else part[k] = s;
  }
  if (!p.cluster) return;
  // each block of the cluster adds a share of the slots over all of them
  cluster_sync();
  for (int k = blockIdx.x * kThreads + threadIdx.x; k < all; k += p.cluster * kThreads) {
    float s = 0.0f;
    for (int t = 0; t < p.cluster; t++) {
      float v;
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(smem_u32(sums + k), t)) : "memory");
      s += v;
    }
    const int slot = k < slots ? k : k - slots, e = slot / g.lanes;
    const int c = (slot % g.lanes + e / VEC * g.lanes) * VEC + e % VEC;
    float* out = k < slots ? p.dweight : p.dbias;
    if (out && c < p.C) out[c] = s;
  }
  cluster_sync();  // no block's shared memory goes before it has been read
}

// Rows that registers do not hold: a block to a row, read again for each pass.
template <typename T, int VEC>
__global__ void __launch_bounds__(kLongThreads) layer_norm_long_kernel(const LayerParams p) {
  using V = RowVec<T, VEC>;
  __shared__ float2 red[2][32];
  const float inv = 1.0f / (float)p.C;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const bool on = token_on(p, r);
    const T* row = static_cast<const T*>(p.x) + p.xm(r);
    float2 s = make_float2(0.0f, 0.0f);
    float m0 = 0.0f;
    if (on && p.kind == KC_NORM_LAYER) {
      for (int c = threadIdx.x * VEC; c < p.C; c += kLongThreads * VEC) {
        float v[VEC];
        V::unpack(V::load(row + c), v);
#pragma unroll
        for (int j = 0; j < VEC; j++) s.x += v[j];
      }
      m0 = block_sum(s, red[0]).x * inv;
    }
    s = make_float2(0.0f, 0.0f);
    if (on)
      for (int c = threadIdx.x * VEC; c < p.C; c += kLongThreads * VEC) {
        float v[VEC];
        V::unpack(V::load(row + c), v);
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          v[j] -= m0;
          s.x += v[j];
          s.y = fmaf(v[j], v[j], s.y);
        }
      }
    s = block_sum(s, red[1]);
    const float delta = p.kind == KC_NORM_LAYER ? s.x * inv : 0.0f;
    const float rstd = rstd_of(p, s.y, inv, delta);
    if (p.stats && threadIdx.x == 0) p.stats[r] = on ? make_float2(m0 + delta, rstd) : make_float2(0.0f, 0.0f);
    T* out = static_cast<T*>(p.y) + p.ym(r);
    for (int c = threadIdx.x * VEC; c < p.C; c += kLongThreads * VEC) {
      float o[VEC], w[VEC], b[VEC];
#pragma unroll
      for (int j = 0; j < VEC; j++) o[j] = 0.0f, w[j] = 1.0f, b[j] = 0.0f;
      if (on) {
        V::unpack(V::load(row + c), o);
        if (p.weight) load_params<VEC>(p.weight + c, p.wide, w);
        if (p.bias) load_params<VEC>(p.bias + c, p.wide, b);
#pragma unroll
        for (int j = 0; j < VEC; j++) o[j] = fmaf((o[j] - m0 - delta) * rstd, w[j], b[j]);
      }
      V::store(out + c, V::pack(o));
    }
    __syncthreads();  // red
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kLongThreads) layer_norm_long_back_kernel(const LayerParams p) {
  using V = RowVec<T, VEC>;
  __shared__ float2 red[32];
  const float inv = 1.0f / (float)p.C;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const bool on = token_on(p, r);
    const T* x = static_cast<const T*>(p.x) + p.xm(r);
    const T* dy = static_cast<const T*>(p.dy) + p.ym(r);
    float2 s = make_float2(0.0f, 0.0f), st = s;
    if (on) {
      st = p.stats[r];
      for (int c = threadIdx.x * VEC; c < p.C; c += kLongThreads * VEC) {
        float a[VEC], d[VEC], w[VEC];
        V::unpack(V::load(x + c), a);
        V::unpack(V::load(dy + c), d);
        if (p.weight) load_params<VEC>(p.weight + c, p.wide, w);
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          const float gw = p.weight ? d[j] * w[j] : d[j];
          s.x += gw;
          s.y = fmaf(gw, (a[j] - st.x) * st.y, s.y);
        }
      }
    }
    s = block_sum(s, red);
    const float c1 = p.kind == KC_NORM_LAYER ? s.x * inv : 0.0f, c2 = s.y * inv;
    T* out = static_cast<T*>(p.y) + p.xm(r);
    for (int c = threadIdx.x * VEC; c < p.C; c += kLongThreads * VEC) {
      float o[VEC];
#pragma unroll
      for (int j = 0; j < VEC; j++) o[j] = 0.0f;
      if (on) {
        float a[VEC], d[VEC], w[VEC];
        V::unpack(V::load(x + c), a);
        V::unpack(V::load(dy + c), d);
        if (p.weight) load_params<VEC>(p.weight + c, p.wide, w);
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          const float gw = p.weight ? d[j] * w[j] : d[j];
          o[j] = st.y * (gw - fmaf((a[j] - st.x) * st.y, c2, c1));
        }
      }
      V::store(out + c, V::pack(o));
    }
    __syncthreads();  // red
  }
}

// The channels' sums of long rows: a block to 32 channels and a share of the rows (before dx may take x's place).
template <typename T>
__global__ void __launch_bounds__(kThreads) layer_norm_long_sums_kernel(const LayerParams p) {
  __shared__ float2 red[kThreads / 32][32];
  const int tx = threadIdx.x % 32, ty = threadIdx.x / 32;
  for (int64_t c0 = (int64_t)blockIdx.x * 32; c0 < p.C; c0 += (int64_t)gridDim.x * 32) {
    const int64_t c = c0 + tx;
    float2 s = make_float2(0.0f, 0.0f);
    if (c < p.C)
      for (int64_t r = (int64_t)blockIdx.y * (kThreads / 32) + ty; r < p.rows;
           r += (int64_t)gridDim.y * (kThreads / 32)) {
        if (!token_on(p, r)) continue;
        const float2 st = p.stats[r];
        const float d = to_f<T>(static_cast<const T*>(p.dy)[p.ym(r) + c]);
        s.x = fmaf(d, (to_f<T>(static_cast<const T*>(p.x)[p.xm(r) + c]) - st.x) * st.y, s.x);
        s.y += d;
      }
    red[ty][tx] = s;
    __syncthreads();
    if (ty == 0 && c < p.C) {
      for (int i = 1; i < kThreads / 32; i++) s.x += red[i][tx].x, s.y += red[i][tx].y;
      p.part[(size_t)blockIdx.y * 2 * p.C + c] = s.x;
      p.part[(size_t)blockIdx.y * 2 * p.C + p.C + c] = s.y;
    }
    __syncthreads();
  }
}

// dweight and dbias from the blocks' sums, in the blocks' order. 32 slots to a block, 32 threads share the blocks.
struct PartShape {
  int blocks, slots;     // slots: of a block's sums of dy xh, those of dy behind them
  int C, nv, vec, lanes; // slot (i, j, lane) is channel (lane + i lanes) vec + j
};

__global__ void __launch_bounds__(1024) layer_norm_params_kernel(const float* part, const PartShape s, float* dweight,
                                                                 float* dbias) {
  __shared__ float red[32][33];
  pdl_wait();
  const int tx = threadIdx.x % 32, ty = threadIdx.x / 32;
  const int64_t first = dweight ? 0 : s.slots, end = dbias ? 2 * (int64_t)s.slots : s.slots;
  for (int64_t k0 = first + (int64_t)blockIdx.x * 32; k0 < end; k0 += (int64_t)gridDim.x * 32) {
    const int64_t k = k0 + tx;
    float sum = 0.0f;
    if (k < end)
#pragma unroll 8
      for (int b = ty; b < s.blocks; b += 32) sum += part[(size_t)b * 2 * s.slots + k];
    red[ty][tx] = sum;
    __syncthreads();
    // thread (tx, ty) adds lane tx's sum of slot ty
    float v = red[tx][ty];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int64_t at = k0 + ty;
    if (tx == 0 && at < end) {
      const int slot = (int)(at < s.slots ? at : at - s.slots), e = slot / s.lanes;
      const int c = (slot % s.lanes + e / s.vec * s.lanes) * s.vec + e % s.vec;
      if (c < s.C) (at < s.slots ? dweight : dbias)[c] = v;
    }
    __syncthreads();
  }
}

// ---- host --------------------------------------------------------------------------------------------------------

// How a call goes over its rows.
struct Shape {
  int vec, nv;
  bool shift;    // rows that begin anywhere
  bool block;    // a block to a row, otherwise `lanes` lanes of a warp
  bool is_long;
  int threads, lanes;
  int64_t blocks;
};

// 16-byte vectors of a warp's lane: up to 24 elements (weight, bias and the row in registers, or weight, row, gradient
// and the channels' sums). A block's thread has 16 or, forward, 32 elements.
constexpr int kNvs[] = {1, 2, 3, 4, 6};
constexpr bool warp_nv(int vec, int nv) { return vec * nv <= 24 && (vec == 4 || nv <= 3); }

// `bytes` of an element; `vec`: the widest vectors to which channels, strides and addresses are aligned.
Shape shape_of(int64_t rows, int C, int bytes, int vec, bool backward) {
  Shape s{};
  const int whole = 16 / bytes;
  s.vec = whole;
  s.shift = vec < whole;
  const int64_t nvec = ((int64_t)C + whole - 1) / whole;
  // the fewest lanes in a row that leave no more than an eighth of them idle, with as many vectors each as are built:
  // few shuffles for a sum, many loads in flight
  int64_t best = -1;
  for (int lanes = 2; lanes <= 32; lanes *= 2)
    for (int nv : kNvs) {
      if (!warp_nv(whole, nv) || (int64_t)lanes * nv < nvec) continue;
      const int64_t waste = (int64_t)lanes * nv * 8 - nvec * 8 > nvec ? (int64_t)lanes * nv - nvec : 0;
      const int64_t cost = waste * 64 + lanes;
      if (best < 0 || cost < best) best = cost, s.lanes = lanes, s.nv = nv;
    }
  if (best >= 0) {
    s.threads = kThreads;
    const int64_t per = kThreads / s.lanes, all = (rows + per - 1) / per;
    // about as many blocks as run at once, by registers and by the ring. Of float32 rows of 9 to 16 channels, and of
    // 2-byte rows of up to 16 that begin anywhere, registers let one less to an SM run than are launched: the last ones
    // wait (2,000,000 x 16 and x 13, float32: 58.3 and 94.7 us; 51.1 and 85.2 with a block less)
    const int by_registers = backward ? 2 : s.nv * whole <= 8 ? (s.shift ? 3 : 4)
                                          : shared_params(s.vec, s.nv, false, s.shift) ? 3 : 2;
    const int row = (backward ? 2 : 1) * (s.nv + (s.shift ? 1 : 0)) * 16;
    const int by_ring = kMaxBlockSmem / (ring_depth(row, backward) * row * kThreads + 1024);
    s.blocks = std::min<int64_t>(all, kSmCount * std::min(by_registers, by_ring));
    return s;
  }
  s.shift = false;
  s.vec = vec;
  s.block = true;
  for (int elements = 16; elements <= (backward ? 16 : 32); elements *= 2) {
    s.nv = elements / vec;
    const int64_t threads = ((int64_t)C / vec + s.nv - 1) / s.nv;
    s.threads = (int)std::min<int64_t>((threads + 31) / 32 * 32, 1 << 20);
    if (s.threads > kBlockThreads) continue;
    s.blocks = std::min<int64_t>(rows, kSmCount * (kBlockThreads / s.threads));
    return s;
  }
  s.block = false;
  s.is_long = true;
  s.threads = kLongThreads;
  s.blocks = std::min<int64_t>(rows, 1 << 20);
  return s;
}

// Shares of the rows in the long rows' channel sums.
int64_t long_shares(int64_t rows, int C) {
  const int64_t most = std::max<int64_t>(1, 8 * kSmCount / ((C + 31) / 32));
  return std::max<int64_t>(1, std::min<int64_t>(most, rows / 8));
}

// The blocks' sums; long rows have a slot to a channel.
PartShape part_shape(const Shape& s, int64_t rows, int C) {
  if (s.is_long) return {(int)long_shares(rows, C), C, C, 1, 1, C};
  const int lanes = s.block ? s.threads : s.lanes;
  return {(int)s.blocks, s.nv * s.vec * lanes, C, s.nv, s.vec, lanes};
}

template <typename T, int VEC, int NV, bool BLOCK, bool SHIFT, bool LEAN>
void launch_back(const LayerParams& p, const Shape& s, cudaStream_t st) {
  // the ring, and in its place the warps' sums
  const size_t sums = BLOCK ? 0 : (size_t)kThreads / 32 * 2 * NV * VEC * s.lanes * sizeof(float);
  const size_t smem = std::max(Ring<T, VEC, NV, BLOCK, 2, SHIFT>::bytes(s.threads), sums);
  allow_block_smem<layer_norm_back_kernel<T, VEC, NV, BLOCK, SHIFT, LEAN>, !BLOCK>();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)s.blocks);
  cfg.blockDim = dim3(s.threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.cluster ? 1 : 0;
  KC_CUDA(cudaLaunchKernelEx(&cfg, layer_norm_back_kernel<T, VEC, NV, BLOCK, SHIFT, LEAN>, p));
}

template <typename T, int VEC, int NV, bool BLOCK, bool SHIFT>
void launch_rows(const LayerParams& p, const Shape& s, bool backward, cudaStream_t st) {
  if (backward) {
    if constexpr (!BLOCK || NV * VEC <= 16) {
      if (p.kind == KC_NORM_RMS && !p.dbias) launch_back<T, VEC, NV, BLOCK, SHIFT, true>(p, s, st);
      else launch_back<T, VEC, NV, BLOCK, SHIFT, false>(p, s, st);
    }
  } else {
    const size_t smem = Ring<T, VEC, NV, BLOCK, 1, SHIFT>::bytes(s.threads) +
                        Affine<VEC, NV, BLOCK, SHIFT, shared_params(VEC, NV, BLOCK, SHIFT)>::bytes(p.C);
    allow_block_smem<layer_norm_kernel<T, VEC, NV, BLOCK, SHIFT>>();
    layer_norm_kernel<T, VEC, NV, BLOCK, SHIFT><<<(unsigned)s.blocks, s.threads, smem, st>>>(p);
  }
  KC_CUDA(cudaGetLastError());
}

template <typename T, int NV>
bool launch_warp(const LayerParams& p, const Shape& s, bool backward, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(T);
  if constexpr (warp_nv(VEC, NV)) {
    if (s.nv != NV) return false;
    s.shift ? launch_rows<T, VEC, NV, false, true>(p, s, backward, st)
            : launch_rows<T, VEC, NV, false, false>(p, s, backward, st);
    return true;
  }
  return false;
}

template <typename T, int... NVS>
void launch_warps(std::integer_sequence<int, NVS...>, const LayerParams& p, const Shape& s, bool backward,
                  cudaStream_t st) {
  (launch_warp<T, NVS>(p, s, backward, st) || ...);
}

template <typename T, int VEC>
void run_vec(const LayerParams& p, const Shape& s, bool backward, cudaStream_t st) {
  if (s.is_long) {
    if (!backward) {
      layer_norm_long_kernel<T, VEC><<<(unsigned)s.blocks, kLongThreads, 0, st>>>(p);
    } else {
      if (p.part) {
        const dim3 grid((unsigned)std::min<int64_t>(((int64_t)p.C + 31) / 32, 1 << 20),
                        (unsigned)long_shares(p.rows, p.C));
        layer_norm_long_sums_kernel<T><<<grid, kThreads, 0, st>>>(p);
        KC_CUDA(cudaGetLastError());
      }
      layer_norm_long_back_kernel<T, VEC><<<(unsigned)s.blocks, kLongThreads, 0, st>>>(p);
    }
    KC_CUDA(cudaGetLastError());
  } else if (!s.block) {
    launch_warps<T>(std::integer_sequence<int, 1, 2, 3, 4, 6>{}, p, s, backward, st);
  } else if (s.nv == 16 / VEC) {
    launch_rows<T, VEC, 16 / VEC, true, false>(p, s, backward, st);
  } else {
    launch_rows<T, VEC, 32 / VEC, true, false>(p, s, backward, st);
  }
}

template <typename T>
void run_type(const LayerParams& p, const Shape& s, bool backward, cudaStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (s.vec == 8) return run_vec<T, 8>(p, s, backward, st);
  if (s.vec == 4) return run_vec<T, 4>(p, s, backward, st);
  if (s.vec == 2) return run_vec<T, 2>(p, s, backward, st);
  run_vec<T, 1>(p, s, backward, st);
}

void run(const kc_layer_norm_desc& d, LayerParams p, int vec, bool backward, cudaStream_t st) {
  p.rows = (int64_t)d.n * d.points;
  p.C = d.channels;
  p.kind = d.kind;
  p.eps = d.eps;
  p.slack = 1.0f;
  if (p.eps == 0.0f) {
    // a sum is made of at most 42 + C / 512 additions: three such errors and the products', each 2^-24. The least
    // negative number for an eps: a variance of 0 becomes NaN, others stay
    p.slack += (3.0f * (42.0f + (float)p.C / 512.0f) + 16.0f) * 0x1p-24f;
    p.least = -HUGE_VALF;
    p.eps = -0x1p-149f;
  }
  p.wide = aligned_to(p.weight, 16) && aligned_to(p.bias, 16);
  p.xm = row_map(d.n, d.points, d.x_board_stride, d.x_row_stride);
  p.ym = row_map(d.n, d.points, d.y_board_stride, d.y_row_stride);
  p.mm = row_map(d.n, d.points, d.mask_board_stride, 1);
  Shape s = shape_of(p.rows, p.C, dtype_bytes(d.dtype), vec, backward);
  p.lanes = s.lanes;
  // few rows: one cluster of up to 16 blocks, whose groups of lanes have 4 rows each at most, and no second launch (361
  // x 384, RMS, bf16, with the call's time on the host: 21.0 us, 23.5 in two launches; 8.3 and 7.9 us on the device.
  // With 16 rows a group, 7,261 x 100, f16, took 29 us on the device, 10.5 over all SMs)
  if (p.part && !s.block && !s.is_long) {
    const int64_t groups = kThreads / s.lanes;
    if (p.rows <= 16 * 4 * groups) {
      p.cluster = 1;
      while (p.cluster < 16 && p.cluster * groups < p.rows) p.cluster *= 2;
      s.blocks = p.cluster;
    }
  }
  if (d.dtype == KC_PRECISION_F32) run_type<float>(p, s, backward, st);
  else if (d.dtype == KC_PRECISION_F16) run_type<__half>(p, s, backward, st);
  else run_type<__nv_bfloat16>(p, s, backward, st);
  if (!p.part || p.cluster) return;
  const PartShape q = part_shape(s, p.rows, p.C);
  const int64_t slots = (int64_t)q.slots * ((p.dweight ? 1 : 0) + (p.dbias ? 1 : 0));
  const dim3 grid((unsigned)std::min<int64_t>((slots + 31) / 32, 1 << 20));
  launch_after(layer_norm_params_kernel, grid, dim3(1024), 0, st, (const float*)p.part, q, p.dweight, p.dbias);
}

Rows x_rows(const kc_layer_norm_desc& d, const void* p) {
  return {p, d.n, d.points, d.channels, d.n > 1 ? d.x_board_stride : 0, d.points > 1 ? d.x_row_stride : 0,
          dtype_bytes(d.dtype)};
}
Rows y_rows(const kc_layer_norm_desc& d, const void* p) {
  return {p, d.n, d.points, d.channels, d.n > 1 ? d.y_board_stride : 0, d.points > 1 ? d.y_row_stride : 0,
          dtype_bytes(d.dtype)};
}
Rows mask_rows(const kc_layer_norm_desc& d, const void* p) {
  return {p, d.n, 1, d.points, d.n > 1 ? d.mask_board_stride : 0, 0, 4};
}

void check_desc(const kc_layer_norm_desc* d) {
  if (!d) bad("null descriptor");
  if (d->dtype < KC_PRECISION_F32 || d->dtype > KC_PRECISION_BF16) bad("unknown dtype");
  if (d->kind != KC_NORM_LAYER && d->kind != KC_NORM_RMS) bad("unknown kind");
  if (d->n < 0 || d->points < 0 || d->n > 1 << 30 || d->points > 1 << 30) bad("n and points must be 0 to 2^30");
  if ((int64_t)d->n * d->points > (int64_t)1 << 46) bad("n * points above 2^46");
  if (d->channels < 1 || d->channels > 1 << 30) bad("channels must be 1 to 2^30");
  if (!(d->eps >= 0.0f) || !std::isfinite(d->eps)) bad("eps must be finite and not negative");
  for (const Rows& r : {x_rows(*d, d), y_rows(*d, d), mask_rows(*d, d)})
    if (!rows_in_range(r)) bad("strides must not be negative, nor reach elements beyond 2^46");
}

int vec_of(const kc_layer_norm_desc& d, std::initializer_list<const void*> ptrs) {
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

// Of the parameter gradients' sums, whatever the tensors' alignment.
size_t back_workspace(const kc_layer_norm_desc& d) {
  const int64_t rows = (int64_t)d.n * d.points;
  if (rows == 0) return 0;
  size_t floats = 0;
  for (int v = 16 / dtype_bytes(d.dtype); v >= 1; v /= 2) {
    if (d.channels % v != 0) continue;
    const PartShape q = part_shape(shape_of(rows, d.channels, dtype_bytes(d.dtype), v, true), rows, d.channels);
    floats = std::max(floats, (size_t)q.blocks * 2 * q.slots);
  }
  return (floats * sizeof(float) + 255) / 256 * 256;
}

// Outputs share no memory with each other or with an input; only a tensor may be its own output.
void check_outputs(const Rows& out, std::initializer_list<Rows> ins, const Rows& mask,
                   std::initializer_list<Range> small_in, std::initializer_list<Range> small_out) {
  if (!rows_distinct(out)) bad("rows of the output share memory");
  for (const Rows& i : ins)
    if (rows_overlap(out, i) && !out.same(i)) bad("the output overlaps an input it does not match");
  if (rows_overlap(out, mask)) bad("the output overlaps the mask");
  for (const Range& s : small_in)
    if (ranges_meet(s, out)) bad("the output overlaps another tensor of the call");
  for (const Range* o = small_out.begin(); o != small_out.end(); o++) {
    bool meets = ranges_meet(*o, out) || ranges_meet(*o, mask);
    for (const Rows& i : ins) meets = meets || ranges_meet(*o, i);
    for (const Range& s : small_in) meets = meets || ranges_meet(*o, s);
    for (const Range* q = o + 1; q != small_out.end(); q++) meets = meets || ranges_meet(*o, *q);
    if (meets) bad("the statistics, parameter gradients or workspace overlap another tensor of the call");
  }
}

void check_aligned(std::initializer_list<Rows> rows, std::initializer_list<const void*> small, const void* stats) {
  for (const Rows& r : rows)
    if (!aligned_to(r.p, r.bytes)) bad("a tensor is not aligned to its element");
  for (const void* s : small)
    if (!aligned_to(s, 4)) bad("a float32 tensor is not aligned to its element");
  if (!aligned_to(stats, 8)) bad("the statistics must be 8-byte aligned");
}

}  // namespace
}  // namespace kc

extern "C" int kc_layer_norm(const kc_layer_norm_desc* desc, const void* d_x, const float* d_mask,
                             const float* d_weight, const float* d_bias, void* d_y, float* d_stats, void* stream) {
  return kc::guard_entry([&] {
    using namespace kc;
    check_desc(desc);
    const kc_layer_norm_desc d = *desc;
    if (d.n == 0 || d.points == 0) return;
    if (!d_x || !d_y) bad("null tensor");
    const Rows x = x_rows(d, d_x), y = y_rows(d, d_y);
    const int64_t ch = 4 * (int64_t)d.channels, sb = 8 * (int64_t)d.n * d.points;
    check_aligned({x, y}, {d_mask, d_weight, d_bias}, d_stats);
    check_outputs(y, {x}, mask_rows(d, d_mask), {{d_weight, ch}, {d_bias, ch}}, {{d_stats, sb}});
    TensorDevice dev("layer norm", {d_x, d_mask, d_weight, d_bias, d_y, d_stats});
    LayerParams p{};
    p.x = d_x;
    p.mask = d_mask;
    p.weight = d_weight;
    p.bias = d_bias;
    p.y = d_y;
    p.stats = reinterpret_cast<float2*>(d_stats);
    run(d, p, vec_of(d, {d_x, d_y}), false, static_cast<cudaStream_t>(stream));
  });
}

extern "C" int kc_layer_norm_backward_workspace(const kc_layer_norm_desc* desc, size_t* bytes) {
  return kc::guard_entry([&] {
    kc::check_desc(desc);
    if (!bytes) kc::bad("null result");
    *bytes = kc::back_workspace(*desc);
  });
}

extern "C" int kc_layer_norm_backward(const kc_layer_norm_desc* desc, const void* d_x, const float* d_mask,
                                      const float* d_weight, const float* d_stats, const void* d_dy, void* d_dx,
                                      float* d_dweight, float* d_dbias, void* d_workspace, size_t workspace_bytes,
                                      void* stream) {
  return kc::guard_entry([&] {
    using namespace kc;
    check_desc(desc);
    const kc_layer_norm_desc d = *desc;
    const bool none = d.n == 0 || d.points == 0, params = d_dweight || d_dbias;
    if (!none && (!d_x || !d_dy || !d_dx || !d_stats)) bad("null tensor");
    const Rows x = x_rows(d, d_x), dy = y_rows(d, d_dy), dx = x_rows(d, d_dx);
    const int64_t ch = 4 * (int64_t)d.channels, sb = 8 * (int64_t)d.n * d.points;
    const size_t need = params ? back_workspace(d) : 0;
    check_aligned({x, dy, dx}, {d_mask, d_weight, d_dweight, d_dbias}, d_stats);
    check_outputs(dx, {x, dy}, mask_rows(d, d_mask), {{d_weight, ch}, {d_stats, sb}},
                  {{d_dweight, ch}, {d_dbias, ch}, {need ? d_workspace : nullptr, (int64_t)need}});
    if (need && (!d_workspace || workspace_bytes < need)) bad("workspace of " + std::to_string(need) + " bytes needed");
    if (need && !aligned_to(d_workspace, 16)) bad("the workspace must be 16-byte aligned");
    if (none && !params) return;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    TensorDevice dev("layer norm", {d_x, d_mask, d_weight, d_stats, d_dy, d_dx, d_dweight, d_dbias,
                                    need ? d_workspace : nullptr});
    if (none) {
      if (d_dweight) KC_CUDA(cudaMemsetAsync(d_dweight, 0, (size_t)ch, st));
      if (d_dbias) KC_CUDA(cudaMemsetAsync(d_dbias, 0, (size_t)ch, st));
      return;
    }
    LayerParams p{};
    p.x = d_x;
    p.mask = d_mask;
    p.weight = d_weight;
    p.y = d_dx;
    p.dy = d_dy;
    p.stats = const_cast<float2*>(reinterpret_cast<const float2*>(d_stats));
    p.part = need ? static_cast<float*>(d_workspace) : nullptr;
    p.dweight = d_dweight;
    p.dbias = d_dbias;
    run(d, p, vec_of(d, {d_x, d_dy, d_dx}), true, st);
  });
}
