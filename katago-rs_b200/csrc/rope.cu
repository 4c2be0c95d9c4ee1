// Rotary positions with several axes on Q and K heads, forward and backward (kc_rope_axes, kc_rope_axes_backward).
//
//   angle[t][tb][j] = sum_a pos[t][a] freqs[tb][j][a], (y1, y2) = (x1 cos - x2 sin, x1 sin + x2 cos)
//   backward: dx = the gradient turned by -angle; d angle = dx2 x1 - dx1 x2;
//   dfreqs[tb][j][a] = sum_t pos[t][a] sum over the table's heads of d angle
//
// Angles are float64 sums brought to [-1/2, 1/2] turns before sine and cosine, so that far positions keep their
// digits. A thread owns the pair vector (VP neighbouring pairs) of one token and one table, makes its angles once and
// turns a run of the table's heads (Q and K) with them.

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
  int run, runs;                  // heads of a table a thread turns; such runs per table
  float* partial;                 // backward: [blocks][tables][pairs][axes]
  float* dfreqs;
  int blocks;
  float sign;                     // +1 forward, -1 backward
};

template <typename T, int N>
struct alignas(N * sizeof(T)) Pack {
  T v[N];
};

// sin and cos of VP pairs' angles at one token.
template <typename T, int VP>
__device__ __forceinline__ void angles(const RopeParams& p, int64_t t, int table, int j0, float (&c)[VP], float (&s)[VP]) {
  double pos[KC_ROPE_MAX_AXES];
#pragma unroll
  for (int a = 0; a < KC_ROPE_MAX_AXES; a++) pos[a] = a < p.axes ? (double)__ldg(p.pos + t * p.axes + a) : 0.0;
  const float* f = p.freqs + ((int64_t)table * p.pairs + j0) * p.axes;
#pragma unroll
  for (int j = 0; j < VP; j++) {
    double angle = 0.0;
#pragma unroll
    for (int a = 0; a < KC_ROPE_MAX_AXES; a++)
      if (a < p.axes) angle += pos[a] * (double)__ldg(f + j * p.axes + a);
    const double turns = angle * 0.15915494309189533577;  // 1 / (2 pi)
    const float part = (float)(turns - rint(turns));
    sincospif(2.0f * part, &s[j], &c[j]);
    s[j] *= p.sign;
  }
}

// The two halves of VP pairs of a head that starts at h: pair j of [j0, j0 + VP).
template <typename T, int VP, int LAYOUT>
__device__ __forceinline__ void load_pairs(const T* h, int j0, int pairs, float (&a)[VP], float (&b)[VP]) {
  if constexpr (LAYOUT == KC_ROPE_HALVES) {
    const Pack<T, VP> u = *reinterpret_cast<const Pack<T, VP>*>(h + j0);
    const Pack<T, VP> v = *reinterpret_cast<const Pack<T, VP>*>(h + pairs + j0);
#pragma unroll
    for (int j = 0; j < VP; j++) {
      a[j] = to_f<T>(u.v[j]);
      b[j] = to_f<T>(v.v[j]);
    }
  } else {
    const Pack<T, VP>* u = reinterpret_cast<const Pack<T, VP>*>(h + 2 * j0);
    const Pack<T, VP> lo = u[0], hi = u[1];
    T e[2 * VP];
#pragma unroll
    for (int j = 0; j < VP; j++) {
      e[j] = lo.v[j];
      e[VP + j] = hi.v[j];
    }
#pragma unroll
    for (int j = 0; j < VP; j++) {
      a[j] = to_f<T>(e[2 * j]);
      b[j] = to_f<T>(e[2 * j + 1]);
    }
  }
}

template <typename T, int VP, int LAYOUT>
__device__ __forceinline__ void store_pairs(T* h, int j0, int pairs, const float (&a)[VP], const float (&b)[VP]) {
  Pack<T, VP> u, v;
  if constexpr (LAYOUT == KC_ROPE_HALVES) {
#pragma unroll
    for (int j = 0; j < VP; j++) {
      u.v[j] = from_f<T>(a[j]);
      v.v[j] = from_f<T>(b[j]);
    }
    *reinterpret_cast<Pack<T, VP>*>(h + j0) = u;
    *reinterpret_cast<Pack<T, VP>*>(h + pairs + j0) = v;
  } else {
    T e[2 * VP];
#pragma unroll
    for (int j = 0; j < VP; j++) {
      e[2 * j] = from_f<T>(a[j]);
      e[2 * j + 1] = from_f<T>(b[j]);
    }
#pragma unroll
    for (int j = 0; j < VP; j++) {
      u.v[j] = e[j];
      v.v[j] = e[VP + j];
    }
    Pack<T, VP>* o = reinterpret_cast<Pack<T, VP>*>(h + 2 * j0);
    o[0] = u;
    o[1] = v;
  }
}

// Head i of a table's Q heads and K heads.
template <typename T>
__device__ __forceinline__ void head_of(const RopeParams& p, int64_t t, int table, int i, const T*& in, T*& out,
                                        const T*& x) {
  const bool is_q = i < p.q.per_table;
  const Heads& h = is_q ? p.q : p.k;
  const int64_t n = (int64_t)table * h.per_table + (is_q ? i : i - p.q.per_table);
  in = static_cast<const T*>(h.in) + t * h.in_t + n * h.in_h;
  out = static_cast<T*>(h.out) + t * h.out_t + n * h.out_h;
  x = static_cast<const T*>(h.x) + (h.x ? t * h.x_t + n * h.x_h : 0);
}

// A thread per (token, table, run of heads, pair vector); behind the pair vectors those of the unrotated rest.
template <typename T, int VP, int LAYOUT>
__global__ void __launch_bounds__(kThreads) rope_axes_kernel(const __grid_constant__ RopeParams p) {
  const int pv = p.pairs / VP, cols = pv + p.rest / VP;
  const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t per_token = (int64_t)p.tables * p.runs * cols;
  const int64_t t = id / per_token;
  if (t >= p.tokens) return;
  int r = (int)(id - t * per_token);
  const int col = r % cols;
  r /= cols;
  const int table = r / p.runs, i0 = (r % p.runs) * p.run;
  const int i1 = min(i0 + p.run, p.q.per_table + p.k.per_table);
  const T *in, *x;
  T* out;
  if (col >= pv) {
    const int d = 2 * p.pairs + (col - pv) * VP;
    for (int i = i0; i < i1; i++) {
      head_of<T>(p, t, table, i, in, out, x);
      if (in != out) *reinterpret_cast<Pack<T, VP>*>(out + d) = *reinterpret_cast<const Pack<T, VP>*>(in + d);
    }
    return;
  }
  float c[VP], s[VP];
  angles<T, VP>(p, t, table, col * VP, c, s);
  for (int i = i0; i < i1; i++) {
    head_of<T>(p, t, table, i, in, out, x);
    float a[VP], b[VP], ya[VP], yb[VP];
    load_pairs<T, VP, LAYOUT>(in, col * VP, p.pairs, a, b);
#pragma unroll
    for (int j = 0; j < VP; j++) {
      ya[j] = a[j] * c[j] - b[j] * s[j];
      yb[j] = a[j] * s[j] + b[j] * c[j];
    }
    store_pairs<T, VP, LAYOUT>(out, col * VP, p.pairs, ya, yb);
  }
}

// Backward with the frequencies' gradient: block x takes every blocks-th group of tokens, its threads are lanes of
// tokens by columns (table, pair vector; block y further columns). A thread adds pos * d angle over its tokens in
// float32, the block's lanes are added in order into the block's partial sums.
template <typename T, int VP, int LAYOUT>
__global__ void __launch_bounds__(kThreads) rope_axes_back_kernel(const __grid_constant__ RopeParams p) {
  __shared__ float red[kThreads * VP];
  const int pv = p.pairs / VP, cols = p.tables * pv, width = min(cols, kThreads), lanes = kThreads / width;
  const int tx = threadIdx.x % width, lane = threadIdx.x / width;
  const int col = blockIdx.y * width + tx;
  const bool active = lane < lanes && col < cols;
  const int table = active ? col / pv : 0, j0 = active ? (col % pv) * VP : 0;
  const int heads = p.q.per_table + p.k.per_table;
  float acc[KC_ROPE_MAX_AXES][VP] = {};
  if (active) {
    for (int64_t t = (int64_t)blockIdx.x * lanes + lane; t < p.tokens; t += (int64_t)p.blocks * lanes) {
      float c[VP], s[VP], turn[VP] = {};
      angles<T, VP>(p, t, table, j0, c, s);
      for (int i = 0; i < heads; i++) {
        const T *in, *x;
        T* out;
        head_of<T>(p, t, table, i, in, out, x);
        float a[VP], b[VP], xa[VP], xb[VP];
        load_pairs<T, VP, LAYOUT>(in, j0, p.pairs, a, b);
        load_pairs<T, VP, LAYOUT>(x, j0, p.pairs, xa, xb);
#pragma unroll
        for (int j = 0; j < VP; j++) {
          const float da = a[j] * c[j] - b[j] * s[j], db = a[j] * s[j] + b[j] * c[j];
          turn[j] += db * xa[j] - da * xb[j];
          a[j] = da;
          b[j] = db;
        }
        store_pairs<T, VP, LAYOUT>(out, j0, p.pairs, a, b);
      }
#pragma unroll
      for (int k = 0; k < KC_ROPE_MAX_AXES; k++) {
        if (k >= p.axes) break;
        const float pos = (float)__ldg(p.pos + t * p.axes + k);
#pragma unroll
        for (int j = 0; j < VP; j++) acc[k][j] += pos * turn[j];
      }
    }
  }
#pragma unroll
  for (int k = 0; k < KC_ROPE_MAX_AXES; k++) {
    if (k >= p.axes) break;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < VP; j++) red[j * kThreads + threadIdx.x] = acc[k][j];
    __syncthreads();
    if (active && lane == 0) {
      float* o = p.partial + (((int64_t)blockIdx.x * p.tables + table) * p.pairs + j0) * p.axes + k;
#pragma unroll
      for (int j = 0; j < VP; j++) {
        float v = 0.0f;
        for (int l = 0; l < lanes; l++) v += red[j * kThreads + l * width + tx];
        o[(int64_t)j * p.axes] = v;
      }
    }
  }
}

// The unrotated rest of the heads of a backward pass with the frequencies' gradient.
template <typename T, int VP>
__global__ void __launch_bounds__(kThreads) rope_rest_kernel(const __grid_constant__ RopeParams p) {
  const int cols = p.rest / VP, heads = p.q.per_table + p.k.per_table;
  const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t per_token = (int64_t)p.tables * heads * cols;
  const int64_t t = id / per_token;
  if (t >= p.tokens) return;
  const int r = (int)(id - t * per_token);
  const T *in, *x;
  T* out;
  head_of<T>(p, t, r / cols / heads, r / cols % heads, in, out, x);
  const int d = 2 * p.pairs + r % cols * VP;
  if (in != out) *reinterpret_cast<Pack<T, VP>*>(out + d) = *reinterpret_cast<const Pack<T, VP>*>(in + d);
}

// dfreqs = the blocks' partial sums, in order and in 64 bits: 32 frequencies a block, 8 lanes of blocks each.
__global__ void __launch_bounds__(kThreads) rope_freqs_kernel(const float* __restrict__ partial, int blocks, int count,
                                                              float* __restrict__ dfreqs) {
  __shared__ double red[8][32];
  const int tx = threadIdx.x & 31, ty = threadIdx.x / 32;
  const int i = blockIdx.x * 32 + tx;
  double s = 0.0;
  if (i < count)
    for (int b = ty; b < blocks; b += 8) s += partial[(int64_t)b * count + i];
  red[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && i < count) {
    for (int k = 1; k < 8; k++) s += red[k][tx];
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
  if (d->q_heads < 1 || d->k_heads < 0 || d->q_heads > 65536 || d->k_heads > 65536) bad("1 to 65536 q heads, 0 to 65536 k heads");
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

int64_t back_blocks(const kc_rope_desc& d) {
  return std::min<int64_t>(148 * 4, std::max<int64_t>(1, d.tokens));
}
size_t back_bytes(const kc_rope_desc& d) {
  if (d.tokens == 0) return 0;
  return (size_t)back_blocks(d) * d.tables * (d.rotary_dim / 2) * d.axes * sizeof(float);
}

RopeParams params(const kc_rope_desc& d, const int32_t* pos, const float* freqs, float sign) {
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

template <typename T, int VP, int LAYOUT>
void launch(RopeParams p, cudaStream_t st) {
  const int heads = p.q.per_table + p.k.per_table;
  p.run = heads;
  p.runs = 1;
  if (p.dfreqs) {
    const int cols = p.tables * (p.pairs / VP), width = std::min(cols, kThreads);
    rope_axes_back_kernel<T, VP, LAYOUT><<<dim3(p.blocks, (cols + width - 1) / width), kThreads, 0, st>>>(p);
    KC_CUDA(cudaGetLastError());
    if (p.rest) {
      rope_rest_kernel<T, VP><<<grid_of(p.tokens * p.tables * heads * (p.rest / VP)), kThreads, 0, st>>>(p);
      KC_CUDA(cudaGetLastError());
    }
    const int count = p.tables * p.pairs * p.axes;
    rope_freqs_kernel<<<(count + 31) / 32, kThreads, 0, st>>>(p.partial, p.blocks, count, p.dfreqs);
    KC_CUDA(cudaGetLastError());
    return;
  }
  const int64_t cols = p.pairs / VP + p.rest / VP;
  rope_axes_kernel<T, VP, LAYOUT><<<grid_of(p.tokens * p.tables * p.runs * cols), kThreads, 0, st>>>(p);
  KC_CUDA(cudaGetLastError());
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
    RopeParams p = params(d, d_pos, d_freqs, 1.0f);
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
    RopeParams p = params(d, d_pos, d_freqs, -1.0f);
    p.q = heads(in[0], out[0], x[0], d.tables);
    p.k = heads(in[1], out[1], x[1], d.tables);
    p.dfreqs = d_dfreqs;
    p.partial = static_cast<float*>(d_workspace);
    p.blocks = (int)back_blocks(d);
    run(d, p, vec_of(d, {in[0], in[1], out[0], out[1], x[0], x[1]}), st);
  });
}
