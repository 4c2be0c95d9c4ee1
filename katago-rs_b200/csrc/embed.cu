// Learned rows looked up by token, and the gradient of their table (kc_embed_rows, kc_embed_rows_backward).
//
//   y[t] = x[t] + scale table[id[t]]            (x may be absent; an id outside the table adds nothing)
//   dtable[v] = scale sum_{t: id[t] = v} dy[t]  (0 for rows that no token has)
//
// Forward, a few lanes of a warp take a token's row. Backward, the tokens are sorted by id (a stable radix sort of the
// ids, so that a row's sum has the tokens' order whatever the timing) and the sorted list is cut into equal pieces
// whatever the rows' shares of it, so that a row that most tokens have costs no more than many rows that few have: a
// group of lanes sums its piece run by run, writes the runs that lie inside it, and leaves its first and last run to
// its block, which joins those of its pieces; a last launch joins runs over blocks. Sums are float32: chains of at most
// a piece, then the pieces of a block, then the blocks.
//
// What bounds it, measured on a B200 (6,549 GB/s copy), bytes that have to move / time:
//   forward, 57,767 tokens x 768 added to a sequence, bf16: 187 MB in 36.5 us, 5,110 GB/s (HBM)
//   backward, 92,416 tokens x 384, 362 rows, bf16: 72 MB in 38.2 us: sort 15 us, sums 18 us (66% of the issue slots),
//     joins 6 us, the launches overlapping. The sort is 16 SMs' work: 5 us of ranks, 3 us for the exchange of the
//     counts, 4 us to write 8-byte entries a sector each
//   backward, 20,011 tokens x 512, 50,000 rows, float32: 143 MB in 48.0 us: sort 13 us, sums and zeros 26 us, joins 7
//     us
//   rows that begin anywhere: forward, 57,767 x 768 of 771, bf16: 63 us (72 us an element or two at a time); backward,
//     92,416 x 384 of 387, bf16: 52.5 us (75 us)
// Not kept: zeros written by the SMs that the sort leaves idle (50.1 us), dy asked into L2 by them (45.8 us, but the
// 92,416 tokens 40.2 us).

#include <algorithm>
#include <cmath>
#include <string>

#include "../../include/katago_cuda.h"
#include "rows.cuh"

namespace kc {
namespace {

[[noreturn]] void bad(const std::string& what) { fail(KC_ERR_INVALID, "CUDA backend: looked-up rows: " + what); }

constexpr int kThreads = 256;
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxBits = 9;          // of a digit: no more digits than threads; 32 warps x 512 counts are 64 KB
constexpr int kTile = 2048;          // tokens of a block of the sort, at least
constexpr int kRounds = 8;           // entries of a lane of the sort that stay in registers between its two passes
// Sorted in one launch by a cluster of up to 16 blocks; more by two launches a digit over all SMs.
constexpr int kClusterTokens = 16 * kSortThreads * kRounds;
constexpr int kFewTokens = 2048;     // sorted and summed in one launch, with digits of up to 8 bits
constexpr int kFewBits = 8;
constexpr int kUnroll = 4;           // tokens whose rows a lane has in flight

struct EmbedParams {
  const int32_t* ids;
  const void* table;
  const void* x;
  void* y;
  int64_t tokens, table_rows;
  int64_t ts, xs, ys;
  int C, lanes;
  float scale;
};

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) embed_kernel(const EmbedParams p) {
  using V = RowVec<T, VEC>;
  const int lane = threadIdx.x & (p.lanes - 1), per = kThreads / p.lanes, nvec = p.C / VEC;
  for (int64_t t = (int64_t)blockIdx.x * per + threadIdx.x / p.lanes; t < p.tokens; t += (int64_t)gridDim.x * per) {
    const int id = __ldg(p.ids + t);
    const bool there = id >= 0 && id < p.table_rows;
    const T* row = static_cast<const T*>(p.table) + (there ? id * p.ts : 0);
    const T* x = p.x ? static_cast<const T*>(p.x) + t * p.xs : nullptr;
    T* y = static_cast<T*>(p.y) + t * p.ys;
    for (int v0 = lane; v0 < nvec; v0 += 4 * p.lanes) {
      typename V::Raw a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int v = v0 + i * p.lanes;
        if (v >= nvec) continue;
        if (there) a[i] = V::load(row + v * VEC);
        if (x) b[i] = V::load(x + v * VEC);
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int v = v0 + i * p.lanes;
        if (v >= nvec) continue;
        float f[VEC], o[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j++) o[j] = 0.0f;
        if (x) V::unpack(b[i], o);
        if (there) {
          V::unpack(a[i], f);
#pragma unroll
          for (int j = 0; j < VEC; j++) o[j] = fmaf(f[j], p.scale, o[j]);
        }
        V::store(y + v * VEC, V::pack(o));
      }
    }
  }
}

// The same for rows that begin anywhere: aligned 16-byte pieces of the rows are read and written, each by a lane; a
// vector is a window over a lane's piece and the next lane's, and a piece to write one over the lane before's vector
// and its own. So lanes 1 to lanes - 2 of a group write; lane 0 has the last vector of the pieces before. (In place, no
// piece is read after its row's elements have been written.)
template <typename T>
__global__ void __launch_bounds__(kThreads) embed_shift_kernel(const EmbedParams p) {
  constexpr int VEC = 16 / sizeof(T), BATCH = 2;
  using V = RowVec<T, VEC>;
  const int lanes = p.lanes, lane = threadIdx.x & (lanes - 1), per = kThreads / lanes, mine = lanes - 2;
  const int pieces = (p.C + VEC - 1) / VEC + 1, bytes = p.C * (int)sizeof(T);
  auto low_of = [](const void* q) { return (uint32_t)reinterpret_cast<uintptr_t>(q) & 15u; };
  auto piece_of = [](const T* row, uint32_t low, int q) {
    return *reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(row) - low + 16 * (intptr_t)q);
  };
  auto from = [&](const uint4& w, int source) {
    return make_uint4(__shfl_sync(0xffffffffu, w.x, source, lanes), __shfl_sync(0xffffffffu, w.y, source, lanes),
                      __shfl_sync(0xffffffffu, w.z, source, lanes), __shfl_sync(0xffffffffu, w.w, source, lanes));
  };
  for (int64_t t0 = (int64_t)blockIdx.x * per; t0 < p.tokens; t0 += (int64_t)gridDim.x * per) {
    const int64_t t = t0 + threadIdx.x / lanes;
    const bool here = t < p.tokens;
    const int id = here ? __ldg(p.ids + t) : -1;
    const bool there = id >= 0 && id < p.table_rows;
    const T* row = static_cast<const T*>(p.table) + (there ? id * p.ts : 0);
    const T* x = static_cast<const T*>(p.x) + (here ? t * p.xs : 0);
    T* y = static_cast<T*>(p.y) + (here ? t * p.ys : 0);
    const uint32_t low_t = low_of(row), low_x = low_of(x), low_y = low_of(y);
    const int skip = (int)(low_y / sizeof(T));
    uint4 carry{};
    for (int v0 = 0; v0 < pieces; v0 += BATCH * mine) {
      uint4 a[BATCH], b[BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; k++) {
        const int q = v0 + k * mine + lane - 1;
        a[k] = there && lane > 0 && 16 * q < (int)low_t + bytes ? piece_of(row, low_t, q) : uint4{};
        if (p.x) b[k] = here && lane > 0 && 16 * q < (int)low_x + bytes ? piece_of(x, low_x, q) : uint4{};
      }
#pragma unroll
      for (int k = 0; k < BATCH; k++) {
        const int q = v0 + k * mine + lane - 1;
        float f[VEC], o[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j++) o[j] = 0.0f;
        if (p.x) V::unpack(window<sizeof(T), false>(b[k], from(b[k], lane + 1), low_x), o);
        V::unpack(window<sizeof(T), false>(a[k], from(a[k], lane + 1), low_t), f);
        if (there)
#pragma unroll
          for (int j = 0; j < VEC; j++) o[j] = fmaf(f[j], p.scale, o[j]);
        const uint4 vec = lane == 0 ? carry : V::pack(o);
        carry = from(vec, lanes - 2);
        const uint4 piece = window<sizeof(T), true>(from(vec, lane - 1), vec, 16 - low_y);
        const int c = q * VEC - skip;
        if (!here || lane == 0 || lane == lanes - 1 || c >= p.C) continue;
        if (c >= 0 && c + VEC <= p.C) {
          *reinterpret_cast<uint4*>(y + c) = piece;
        } else {
          const T* e = reinterpret_cast<const T*>(&piece);
#pragma unroll
          for (int j = 0; j < VEC; j++)
            if (c + j >= 0 && c + j < p.C) y[c + j] = e[j];
        }
      }
    }
  }
}

// ---- tokens sorted by id -----------------------------------------------------------------------------------------
// Entries are (key, token); the key of an id outside the table is table_rows, behind all rows. Each pass orders by one
// digit and keeps the order of equal ones.
struct SortParams {
  const int32_t* ids;  // the first pass's input, otherwise `in`
  const int2* in;
  int2* out;
  int* hist;           // [tiles][1 << bits]
  int tokens, rows;
  int shift, bits;
  int tiles, tile;     // tokens of a tile
};

enum class SortIn { kTiles, kCluster, kBlock };  // over launches, over a cluster, in a block's shared memory

template <SortIn IN>
__device__ __forceinline__ int2 sort_entry(const SortParams& p, int i) {
  if (!p.ids) return IN == SortIn::kBlock ? p.in[i] : __ldcg(p.in + i);  // other blocks' of the cluster
  const int id = __ldg(p.ids + i);
  return make_int2(id >= 0 && id < p.rows ? id : p.rows, i);
}

__global__ void __launch_bounds__(kSortThreads) embed_count_kernel(const SortParams p) {
  __shared__ int count[1 << kMaxBits];
  pdl_wait();
  pdl_trigger();
  const int bins = 1 << p.bits;
  for (int b = threadIdx.x; b < bins; b += kSortThreads) count[b] = 0;
  __syncthreads();
  const int i0 = blockIdx.x * p.tile, i1 = min(p.tokens, i0 + p.tile);
  const int lane = threadIdx.x % 32;
  for (int i = i0 + threadIdx.x; i - lane < i1; i += kSortThreads) {  // a warp's lanes stay together
    const int d = i < i1 ? sort_entry<SortIn::kTiles>(p, i).x >> p.shift & (bins - 1) : bins;
    const uint32_t peers = __match_any_sync(0xffffffffu, d);
    if (d < bins && lane == __ffs(peers) - 1) atomicAdd(&count[d], __popc(peers));
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kSortThreads) p.hist[(size_t)blockIdx.x * bins + b] = count[b];
}

// The two halves of cluster_sync.
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Places the tile's entries. Each warp owns a share of consecutive entries: it counts its digits, takes its places
// behind those of the tiles and warps before it, and goes over them again. The tiles' counts are in p.hist; a cluster
// with a block to each tile exchanges them (`totals`, [tiles][bins]).
template <SortIn IN, int THREADS>
__device__ __forceinline__ void place_tile(const SortParams& p, int tile, int* count, int* scan, int* totals) {
  constexpr int WARPS = THREADS / 32;
  const int bins = 1 << p.bits, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int b = threadIdx.x; b < WARPS * bins / 4; b += THREADS)
    reinterpret_cast<int4*>(count)[b] = make_int4(0, 0, 0, 0);
  __syncthreads();
  const int i0 = tile * p.tile, i1 = min(p.tokens, i0 + p.tile);
  const int share = ((max(i1 - i0, 0) + WARPS - 1) / WARPS + 31) / 32 * 32;
  const int w0 = i0 + warp * share, w1 = min(i1, w0 + share);
  int* mine = count + warp * bins;
  // an entry's place among those of its digit in the warp's share; a share of few rounds keeps its entries and places
  auto place = [&](int d) {
    // the lanes with this digit, a bit at a time
    uint32_t peers = __ballot_sync(0xffffffffu, d < bins);
#pragma unroll
    for (int b = 0; b < kMaxBits; b++) {
      if (b >= p.bits) break;
      const bool one = d >> b & 1;
      const uint32_t ones = __ballot_sync(0xffffffffu, one);
      peers &= one ? ones : ~ones;
    }
    int n = 0;
    if (d < bins) n = mine[d];
    __syncwarp();
    if (d < bins && lane == __ffs(peers) - 1) mine[d] = n + __popc(peers);
    __syncwarp();
    return n + __popc(peers & ((1u << lane) - 1));
  };
  auto digit = [&](int key, int i) { return i < w1 ? key >> p.shift & (bins - 1) : bins; };
  const bool kept = share <= 32 * kRounds;
  int2 e[kRounds];
  int at_digit[kRounds];
  for (int j = w0 + lane; j - lane < w1; j += 32 * kRounds) {
#pragma unroll
    for (int k = 0; k < kRounds; k++) e[k] = j + 32 * k < w1 ? sort_entry<IN>(p, j + 32 * k) : make_int2(0, 0);
#pragma unroll
    for (int k = 0; k < kRounds; k++)
      if (j - lane + 32 * k < w1) at_digit[k] = place(digit(e[k].x, j + 32 * k));
  }
  __syncthreads();
  // thread b: digit b's places
  int before = 0, total = 0;
  if (IN != SortIn::kTiles) {
    // no block writes into another one's shared memory before that has started (embed_sort_kernel)
    if (IN == SortIn::kCluster && p.ids && p.tiles > 1) cluster_wait();
    if (threadIdx.x < bins) {
#pragma unroll
      for (int w = 0; w < WARPS; w++) total += count[w * bins + threadIdx.x];
      if (p.tiles > 1)  // to all blocks of the cluster
        for (int t = 0; t < p.tiles; t++)
          asm volatile("st.shared::cluster.u32 [%0], %1;"
                       ::"r"(mapa_shared(smem_u32(totals + tile * bins + threadIdx.x), t)), "r"(total) : "memory");
    }
    if (p.tiles > 1) {
      cluster_sync();
      total = 0;
      if (threadIdx.x < bins) {
#pragma unroll 8
        for (int t = 0; t < p.tiles; t++) {
          const int h = totals[t * bins + threadIdx.x];
          if (t < tile) before += h;
          total += h;
        }
      }
    }
  } else if (threadIdx.x < bins) {
#pragma unroll 8
    for (int t = 0; t < p.tiles; t++) {
      const int h = p.hist[(size_t)t * bins + threadIdx.x];
      if (t < tile) before += h;
      total += h;
    }
  }
  // exclusive sums of the totals over the digits
  int sum = total;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int v = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += v;
  }
  if (lane == 31) scan[warp] = sum;
  __syncthreads();
  if (threadIdx.x < bins) {
    int at = sum - total + before;
    for (int w = 0; w < warp; w++) at += scan[w];
#pragma unroll 8
    for (int w = 0; w < WARPS; w++) {
      const int n = count[w * bins + threadIdx.x];
      count[w * bins + threadIdx.x] = at;
      at += n;
    }
  }
  __syncthreads();
  if (kept) {
#pragma unroll
    for (int k = 0; k < kRounds; k++) {
      const int i = w0 + lane + 32 * k;
      if (i < w1) p.out[mine[digit(e[k].x, i)] + at_digit[k]] = e[k];
    }
    return;
  }
  for (int j = w0 + lane; j - lane < w1; j += 32 * kRounds) {
#pragma unroll
    for (int k = 0; k < kRounds; k++) e[k] = j + 32 * k < w1 ? sort_entry<IN>(p, j + 32 * k) : make_int2(0, 0);
#pragma unroll
    for (int k = 0; k < kRounds; k++) {
      if (j - lane + 32 * k >= w1) continue;
      const int n = place(digit(e[k].x, j + 32 * k));
      if (j + 32 * k < w1) p.out[n] = e[k];
    }
  }
}

__global__ void __launch_bounds__(kSortThreads) embed_place_kernel(const SortParams p) {
  extern __shared__ __align__(16) int count[];
  __shared__ int scan[kSortWarps];
  pdl_wait();
  pdl_trigger();
  place_tile<SortIn::kTiles, kSortThreads>(p, blockIdx.x, count, scan, nullptr);
}

// All passes of a list that a cluster sorts, a tile to a block.
__global__ void __launch_bounds__(kSortThreads) embed_sort_kernel(SortParams p, int passes, int2* a, int2* b) {
  extern __shared__ __align__(16) int count[];
  __shared__ int scan[kSortWarps];
  int* totals = count + (kSortWarps << p.bits);
  pdl_trigger();
  if (p.tiles > 1) cluster_arrive();
  for (int i = 0; i < passes; i++) {
    p.out = (passes - i) % 2 ? a : b;  // the last pass ends in a
    p.shift = i * p.bits;
    place_tile<SortIn::kCluster, kSortThreads>(p, blockIdx.x, count, scan, totals);
    if (p.tiles > 1) cluster_sync();  // the entries are written, and the totals have been read
    else __syncthreads();
    p.ids = nullptr;
    p.in = p.out;
  }
}

// ---- sums of sorted rows -----------------------------------------------------------------------------------------
struct SumParams {
  const int2* list;  // sorted entries
  const void* dy;
  float* dtable;
  float* part;       // [blocks][2][C]: the first and last run of a block's pieces
  int2* part_ids;    // [blocks]: their keys; y = -1 where one run is all
  int64_t ys;
  int tokens, rows, C, lanes;
  int piece;         // entries of a group's piece, a multiple of kUnroll
  int blocks;        // over the list; those behind them write the rows that no token has
  int wide;          // dtable's rows are 16-byte aligned
  float scale;
};

template <int VEC>
__device__ __forceinline__ void store_row(const SumParams& p, int id, int c, const float (&v)[VEC]) {
  if (id >= p.rows) return;
  float* out = p.dtable + (size_t)id * p.C + c;
  if (VEC % 4 == 0 && p.wide) {  // channels are a multiple of 4: whole float4s, of which the row may end behind one
#pragma unroll
    for (int i = 0; i < VEC / 4; i++)
      if (c + 4 * i < p.C)
        reinterpret_cast<float4*>(out)[i] = make_float4(v[4 * i] * p.scale, v[4 * i + 1] * p.scale,
                                                        v[4 * i + 2] * p.scale, v[4 * i + 3] * p.scale);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i++)
      if (c + i < p.C) out[i] = v[i] * p.scale;
  }
}

// The kThreads rows from `row0` on that the list lacks: a thread looks for each, then all write them.
__device__ __forceinline__ void absent_rows(const SumParams& p, int row0, int columns, int* absent) {
  __shared__ int n;
  if (threadIdx.x == 0) n = 0;
  __syncthreads();
  const int row = row0 + threadIdx.x;
  if (row < p.rows) {
    int lo = 0, hi = p.tokens;  // the first entry whose key is not below row
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (p.list[mid].x < row) lo = mid + 1;
      else hi = mid;
    }
    if (lo == p.tokens || p.list[lo].x != row) absent[atomicAdd(&n, 1)] = row;
  }
  __syncthreads();
  const int c0 = blockIdx.y * columns, c1 = min(p.C, c0 + columns);
  const int width = p.wide ? (c1 - c0) / 4 : c1 - c0;
  for (int i = threadIdx.x; i < n * width; i += kThreads) {
    float* out = p.dtable + (size_t)absent[i / width] * p.C + c0;
    if (p.wide) reinterpret_cast<float4*>(out)[i % width] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    else out[i % width] = 0.0f;
  }
}

// The block's pieces of the list. WHOLE: they are all there is, and no run goes on in another block.
// SHIFT: rows of dy that begin anywhere. A lane reads an aligned 16-byte piece of the row (which never leaves the
// allocation of the element in it); its vector is a window over that and the next lane's, so that the last lane of a
// group has none. What lies behind the row's end is summed into channels that are not written.
// slot: [first, last][group][lane][VEC], key: [first, last][group]
template <typename T, int VEC, bool SHIFT, bool WHOLE>
__device__ __forceinline__ void sum_pieces(const SumParams& p, float* slot, int (*key)[kThreads / 2]) {
  using V = RowVec<T, VEC>;
  constexpr int SLOTS = kThreads * VEC;
  const int lanes = p.lanes, lane = threadIdx.x & (lanes - 1), group = threadIdx.x / lanes, groups = kThreads / lanes;
  const int per = SHIFT ? lanes - 1 : lanes;  // vectors of a group
  const int v = blockIdx.y * per + lane, c = v * VEC;
  const bool here = lane < per && c < p.C;
  const T* dy = static_cast<const T*>(p.dy) + (SHIFT ? 0 : c);
  // where a token's row begins in its first piece
  auto begin = [&](int token) {
    return ((uint32_t)reinterpret_cast<uintptr_t>(dy) + (uint32_t)token * (uint32_t)p.ys * (uint32_t)sizeof(T)) & 15u;
  };
  auto row = [&](int token) {
    if constexpr (SHIFT) {
      const uint32_t low = begin(token);
      const T* piece = reinterpret_cast<const T*>(reinterpret_cast<uintptr_t>(dy + token * p.ys) - low) + c;
      return 16 * v < (int)(low + p.C * sizeof(T)) ? V::load(piece) : typename V::Raw{};
    } else {
      return here ? V::load(dy + token * p.ys) : typename V::Raw{};
    }
  };
  const int64_t i0 = ((int64_t)(WHOLE ? 0 : blockIdx.x) * groups + group) * p.piece;
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; j++) acc[j] = 0.0f;
  int cur = -1, first = -1;  // the run at hand, and the piece's first one once it is over
  int2 later[kUnroll];       // the next entries, on their way while the rows of these are
  auto look = [&](int e0) {
#pragma unroll
    for (int u = 0; u < kUnroll; u++)
      later[u] = e0 < p.piece && i0 + e0 + u < p.tokens ? p.list[i0 + e0 + u] : make_int2(p.rows, 0);
  };
  look(0);
  for (int e0 = 0; e0 < p.piece; e0 += kUnroll) {
    int2 e[kUnroll];
    typename V::Raw raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; u++) e[u] = later[u];
#pragma unroll
    for (int u = 0; u < kUnroll; u++) raw[u] = e[u].x < p.rows ? row(e[u].y) : typename V::Raw{};
    look(e0 + kUnroll);
#pragma unroll
    for (int u = 0; u < kUnroll; u++) {
      if (e[u].x != cur) {
        if (cur >= 0) {
          if (first < 0) {
            first = cur;
#pragma unroll
            for (int j = 0; j < VEC; j++) slot[threadIdx.x * VEC + j] = acc[j];
          } else if (here) {
            store_row<VEC>(p, cur, c, acc);
          }
        }
        cur = e[u].x;
#pragma unroll
        for (int j = 0; j < VEC; j++) acc[j] = 0.0f;
      }
      if constexpr (SHIFT) {
        uint4 next;
        next.x = __shfl_down_sync(0xffffffffu, raw[u].x, 1, lanes);
        next.y = __shfl_down_sync(0xffffffffu, raw[u].y, 1, lanes);
        next.z = __shfl_down_sync(0xffffffffu, raw[u].z, 1, lanes);
        next.w = __shfl_down_sync(0xffffffffu, raw[u].w, 1, lanes);
        raw[u] = window<sizeof(T), false>(raw[u], next, begin(e[u].y));
      }
      if (here && cur < p.rows) {
        float f[VEC];
        V::unpack(raw[u], f);
#pragma unroll
        for (int j = 0; j < VEC; j++) acc[j] += f[j];
      }
    }
  }
  const int last = first < 0 ? 0 : 1;
#pragma unroll
  for (int j = 0; j < VEC; j++) slot[last * SLOTS + threadIdx.x * VEC + j] = acc[j];
  if (lane == 0) {
    key[0][group] = first < 0 ? cur : first;
    key[1][group] = first < 0 ? -1 : cur;
  }
  __syncthreads();
  // the groups' first and last runs in order, a thread to a channel
  const int width = lanes * VEC;
  for (int j = threadIdx.x; j < per * VEC; j += kThreads) {
    const int col = blockIdx.y * per * VEC + j;
    if (col >= p.C) continue;
    float* part = WHOLE ? nullptr : p.part + (size_t)blockIdx.x * 2 * p.C + col;
    float sum = 0.0f;
    int run = key[0][0], head = -1;
    for (int g = 0; g < groups; g++)
      for (int k = 0; k < 2; k++) {
        const int id = key[k][g];
        if (id < 0) continue;
        if (id != run) {
          if (!WHOLE && head < 0) head = run, part[0] = sum;
          else if (run < p.rows) p.dtable[(size_t)run * p.C + col] = sum * p.scale;
          run = id;
          sum = 0.0f;
        }
        sum += slot[k * SLOTS + g * width + j];
      }
    if (WHOLE) {
      if (run < p.rows) p.dtable[(size_t)run * p.C + col] = sum * p.scale;
    } else {
      part[head < 0 ? 0 : p.C] = sum;
      if (col == 0) p.part_ids[blockIdx.x] = make_int2(head < 0 ? run : head, head < 0 ? -1 : run);
    }
  }
}

template <typename T, int VEC, bool SHIFT>
__global__ void __launch_bounds__(kThreads, 4) embed_sum_kernel(const SumParams p) {
  __shared__ float slot[2 * kThreads * VEC];
  __shared__ int key[2][kThreads / 2];
  pdl_wait();
  pdl_trigger();
  if (blockIdx.x >= p.blocks)
    return absent_rows(p, (blockIdx.x - p.blocks) * kThreads, (p.lanes - SHIFT) * VEC, key[0]);
  sum_pieces<T, VEC, SHIFT, false>(p, slot, key);
}

// Few tokens in one launch: every block sorts them in its shared memory, the first of each column of blocks sums, and
// all share the rows that no token has.
template <typename T, int VEC, bool SHIFT>
__global__ void __launch_bounds__(kThreads) embed_few_kernel(SumParams p, SortParams q, int passes) {
  __shared__ __align__(16) int2 list[2][kFewTokens];
  __shared__ __align__(16) int count[kThreads / 32 << kFewBits];
  __shared__ int scan[kThreads / 32], absent[kThreads], key[2][kThreads / 2];
  static_assert(sizeof(list[1]) >= 2 * kThreads * VEC * sizeof(float), "the slots take the place of the other list");
  for (int i = 0; i < passes; i++) {
    q.out = list[(passes - i) % 2 ? 0 : 1];  // the last pass ends in list[0]
    q.shift = i * q.bits;
    place_tile<SortIn::kBlock, kThreads>(q, 0, count, scan, nullptr);
    __syncthreads();
    q.ids = nullptr;
    q.in = q.out;
  }
  p.list = list[0];
  if (blockIdx.x == 0) sum_pieces<T, VEC, SHIFT, true>(p, reinterpret_cast<float*>(list[1]), key);
  for (int64_t row0 = (int64_t)blockIdx.x * kThreads; row0 < p.rows; row0 += (int64_t)gridDim.x * kThreads) {
    absent_rows(p, (int)row0, (p.lanes - SHIFT) * VEC, absent);
    __syncthreads();
  }
}

// Runs over blocks. Block i of the list takes those that start in its first run (where the block before ends with
// another key) and in its last one: the sum of that and of the first runs behind it with the same key. A block to 32
// channels, 8 threads share a run's blocks.
__global__ void __launch_bounds__(kThreads) embed_join_kernel(const SumParams p) {
  __shared__ float red[kThreads / 32][33];
  __shared__ int stop;
  pdl_wait();
  const int tx = threadIdx.x % 32, ty = threadIdx.x / 32, c = blockIdx.y * 32 + tx;
  const int2 own = p.part_ids[blockIdx.x];
  int2 prev = make_int2(-1, -1);
  if (blockIdx.x > 0) prev = p.part_ids[blockIdx.x - 1];
  for (int k = 0; k < 2; k++) {
    const int id = k ? own.y : own.x;
    if (id < 0 || id >= p.rows) continue;
    if (k == 0 && id == (prev.y < 0 ? prev.x : prev.y)) continue;
    // blocks [blockIdx.x + 1, stop) begin with the run; it goes beyond this block only if it is its last one
    int end = blockIdx.x + 1;
    if (k == 1 || own.y < 0) {
      for (bool more = true; more; end += kThreads) {
        if (threadIdx.x == 0) stop = kThreads;
        __syncthreads();
        const int j = end + threadIdx.x;
        int2 q = make_int2(-1, -1);
        if (j < p.blocks) q = p.part_ids[j];
        const bool begins = j < p.blocks && q.x == id;
        if (!begins || q.y >= 0) atomicMin(&stop, (int)threadIdx.x + (begins ? 1 : 0));
        __syncthreads();
        more = stop == kThreads;
        if (!more) end += stop - kThreads;
        // a run that ends with the last block looked at goes on there as nothing: the next round stops at once
        __syncthreads();
      }
    }
    float s = 0.0f;
    if (c < p.C)
#pragma unroll 4
      for (int j = blockIdx.x + 1 + ty; j < end; j += kThreads / 32) s += p.part[(size_t)j * 2 * p.C + c];
    red[ty][tx] = s;
    __syncthreads();
    if (ty == 0 && c < p.C) {
      s = p.part[(size_t)blockIdx.x * 2 * p.C + k * p.C + c];
      for (int i = 0; i < kThreads / 32; i++) s += red[i][tx];
      p.dtable[(size_t)id * p.C + c] = s * p.scale;
    }
    __syncthreads();
  }
}

// ---- host --------------------------------------------------------------------------------------------------------

// Lanes of a row, `idle` of which have no vector: the groups that need the fewest lanes in all, the widest of them; the
// narrowest of those with two idle lanes (60,000 tokens x 377, bf16, forward: 56 us with 32 lanes).
int lanes_of(int nvec, int idle) {
  int best = 32;
  auto all = [&](int lanes) { return (int64_t)(nvec + lanes - idle - 1) / (lanes - idle) * lanes; };
  for (int lanes = 16; lanes >= 8; lanes /= 2)
    if (all(lanes) < all(best) || (idle == 2 && all(lanes) == all(best))) best = lanes;
  return best;
}

struct SumShape {
  int lanes, chunks, piece, blocks;
};
// `shift`: a group's last lane has no vector
SumShape sum_shape(int64_t tokens, int C, int vec, bool shift) {
  SumShape s;
  const int nvec = (C + vec - 1) / vec;
  s.lanes = lanes_of(nvec, shift);
  s.chunks = (nvec + s.lanes - shift - 1) / (s.lanes - shift);
  const int groups = kThreads / s.lanes;
  // four blocks to an SM, of pieces of up to 256 entries
  const int64_t want = (tokens * s.chunks + (int64_t)4 * kSmCount * groups - 1) / ((int64_t)4 * kSmCount * groups);
  s.piece = (int)std::min<int64_t>(256, std::max<int64_t>(kUnroll, (want + kUnroll - 1) / kUnroll * kUnroll));
  s.blocks = (int)((tokens + (int64_t)s.piece * groups - 1) / ((int64_t)s.piece * groups));
  return s;
}

struct SortShape {
  int passes, bits, tiles, tile;
  bool cluster;
};
SortShape sort_shape(int64_t tokens, int64_t rows) {
  SortShape s;
  int bits = 1;  // of keys 0 .. rows
  while (rows >> bits) bits++;
  s.passes = (bits + kMaxBits - 1) / kMaxBits;
  s.bits = (bits + s.passes - 1) / s.passes;
  s.cluster = tokens <= kClusterTokens;
  if (s.cluster) {
    s.tiles = 1;
    while (s.tiles < 16 && (int64_t)s.tiles * kTile < tokens) s.tiles *= 2;
    s.tile = (int)((tokens + s.tiles - 1) / s.tiles);
    return s;
  }
  // few tiles, so that a block soon has all their counts, of few entries, which go out one 32-byte sector each (400,000
  // tokens, 17 bits: 79 us in all with a tile to each SM, 74 us in tiles of 8,192; 300,000, 2 bits: 52 and 57 us)
  s.tile = (int)std::max<int64_t>(2 * kTile, (tokens + kSmCount - 1) / kSmCount);
  s.tiles = (int)((tokens + s.tile - 1) / s.tile);
  return s;
}

struct Layout {
  size_t a = 0, b = 0, hist = 0, part = 0, ids = 0, total = 0;
};
Layout layout(const kc_embed_desc& d) {
  Layout l;
  if (d.tokens == 0) return l;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  const SortShape s = sort_shape(d.tokens, d.table_rows);
  int blocks = 0;
  for (bool shift : {false, true})
    blocks = std::max(blocks, sum_shape(d.tokens, d.channels, 16 / dtype_bytes(d.dtype), shift).blocks);
  l.a = take((size_t)d.tokens * sizeof(int2));
  if (s.passes > 1) l.b = take((size_t)d.tokens * sizeof(int2));
  if (!s.cluster) l.hist = take(((size_t)s.tiles << s.bits) * sizeof(int));
  l.part = take((size_t)blocks * 2 * d.channels * sizeof(float));
  l.ids = take((size_t)blocks * sizeof(int2));
  l.total = at;
  return l;
}

void sort_tokens(const kc_embed_desc& d, const int32_t* ids, int2* a, int2* b, int* hist, cudaStream_t st) {
  const SortShape s = sort_shape(d.tokens, d.table_rows);
  SortParams p{ids, nullptr, nullptr, hist, (int)d.tokens, (int)d.table_rows, 0, s.bits, s.tiles, s.tile};
  const size_t smem = ((size_t)kSortWarps << s.bits) * sizeof(int);
  if (s.cluster) {
    allow_block_smem<embed_sort_kernel, true>();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(s.tiles);
    cfg.blockDim = dim3(kSortThreads);
    cfg.dynamicSmemBytes = smem + ((size_t)s.tiles << s.bits) * sizeof(int);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)s.tiles;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = s.tiles > 1 ? 1 : 0;
    KC_CUDA(cudaLaunchKernelEx(&cfg, embed_sort_kernel, p, s.passes, a, b));
    return;
  }
  allow_block_smem<embed_place_kernel>();
  for (int i = 0; i < s.passes; i++) {
    p.out = (s.passes - i) % 2 ? a : b;  // the last pass ends in a
    p.shift = i * s.bits;
    if (i == 0) {
      embed_count_kernel<<<s.tiles, kSortThreads, 0, st>>>(p);
      KC_CUDA(cudaGetLastError());
    } else {
      launch_after(embed_count_kernel, dim3(s.tiles), dim3(kSortThreads), 0, st, p);
    }
    launch_after(embed_place_kernel, dim3(s.tiles), dim3(kSortThreads), smem, st, p);
    p.ids = nullptr;
    p.in = p.out;
  }
}

template <typename T, int VEC, bool SHIFT>
void launch_sum(const SumParams& p, const SumShape& s, cudaStream_t st) {
  const unsigned absent = (unsigned)((p.rows + (int64_t)kThreads - 1) / kThreads);
  const dim3 grid((unsigned)s.blocks + absent, (unsigned)s.chunks);
  launch_after(embed_sum_kernel<T, VEC, SHIFT>, grid, dim3(kThreads), 0, st, p);
  launch_after(embed_join_kernel, dim3((unsigned)s.blocks, (unsigned)((p.C + 31) / 32)), dim3(kThreads), 0, st, p);
}

template <typename T>
void run_type(const EmbedParams& p, bool shift, unsigned blocks, cudaStream_t st) {
  if (shift) embed_shift_kernel<T><<<blocks, kThreads, 0, st>>>(p);
  else embed_kernel<T, 16 / sizeof(T)><<<blocks, kThreads, 0, st>>>(p);
  KC_CUDA(cudaGetLastError());
}

// One launch where groups of four lanes, 32 tokens to a group at most, have all tokens in a block (361 tokens x 384,
// 362 rows, f16: 13.7 us, 12.0 us in three launches, but 16 and 22 us with the calls' time on the host).
template <typename T, int VEC, bool SHIFT>
bool launch_few(SumParams p, const int32_t* ids, cudaStream_t st) {
  p.lanes = 4;
  const int groups = kThreads / p.lanes, per = p.lanes - SHIFT, nvec = (p.C + VEC - 1) / VEC;
  const int chunks = (nvec + per - 1) / per;
  if (p.tokens > std::min(kFewTokens, 32 * groups) || chunks > 2 * kSmCount) return false;
  p.piece = (p.tokens + groups * kUnroll - 1) / (groups * kUnroll) * kUnroll;
  int bits = 1;
  while ((int64_t)p.rows >> bits) bits++;
  const int passes = (bits + kFewBits - 1) / kFewBits;
  const SortParams q{ids, nullptr, nullptr, nullptr, p.tokens, p.rows, 0, (bits + passes - 1) / passes, 1, p.tokens};
  const int64_t rows = (p.rows + (int64_t)kThreads - 1) / kThreads, most = std::max(1, 4 * kSmCount / chunks);
  const dim3 grid((unsigned)std::min(rows, most), (unsigned)chunks);
  embed_few_kernel<T, VEC, SHIFT><<<grid, kThreads, 0, st>>>(p, q, passes);
  KC_CUDA(cudaGetLastError());
  return true;
}

template <typename T, bool SHIFT>
void sum_type(SumParams p, const kc_embed_desc& d, const int32_t* ids, int2* a, int2* b, int* hist, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(T);
  if (launch_few<T, VEC, SHIFT>(p, ids, st)) return;
  sort_tokens(d, ids, a, b, hist, st);
  const SumShape s = sum_shape(d.tokens, d.channels, VEC, SHIFT);
  p.list = a;
  p.lanes = s.lanes;
  p.piece = s.piece;
  p.blocks = s.blocks;
  launch_sum<T, VEC, SHIFT>(p, s, st);
}

Rows rows_of(const kc_embed_desc& d, const void* p, int64_t count, int64_t stride) {
  return {p, count, 1, d.channels, count > 1 ? stride : 0, 0, dtype_bytes(d.dtype)};
}

void check_desc(const kc_embed_desc* d) {
  if (!d) bad("null descriptor");
  if (d->dtype < KC_PRECISION_F32 || d->dtype > KC_PRECISION_BF16) bad("unknown dtype");
  if (d->tokens < 0 || d->tokens > 1 << 30) bad("tokens must be 0 to 2^30");
  if (d->table_rows < 1 || d->table_rows > 1 << 30) bad("table_rows must be 1 to 2^30");
  if (d->channels < 1 || d->channels > 1 << 20) bad("channels must be 1 to 2^20");
  if (!std::isfinite(d->scale)) bad("scale must be finite");
}

void check_rows(const Rows& r) {
  if (!rows_in_range(r)) bad("strides must not be negative, nor reach elements beyond 2^46");
  if (!aligned_to(r.p, r.bytes)) bad("a tensor is not aligned to its element");
}

int vec_of(const kc_embed_desc& d, std::initializer_list<Rows> rows) {
  const int es = dtype_bytes(d.dtype);
  for (int v = 16 / es; v > 1; v /= 2) {
    bool ok = d.channels % v == 0;
    for (const Rows& r : rows) ok = ok && aligned_to(r.p, (size_t)v * es) && r.outer_stride % v == 0;
    if (ok) return v;
  }
  return 1;
}

}  // namespace
}  // namespace kc

extern "C" int kc_embed_rows(const kc_embed_desc* desc, const int32_t* d_ids, const void* d_table, const void* d_x,
                             void* d_y, void* stream) {
  return kc::guard_entry([&] {
    using namespace kc;
    check_desc(desc);
    const kc_embed_desc d = *desc;
    const Rows table = rows_of(d, d_table, d.table_rows, d.table_stride), x = rows_of(d, d_x, d.tokens, d.x_stride),
               y = rows_of(d, d_y, d.tokens, d.y_stride);
    check_rows(table);
    if (d_x) check_rows(x);
    check_rows(y);
    if (d.tokens == 0) return;
    if (!d_ids || !d_table || !d_y) bad("null tensor");
    if (!aligned_to(d_ids, 4)) bad("the ids are not aligned to their element");
    if (!rows_distinct(y)) bad("rows of the output share memory");
    if (rows_overlap(y, table) || ranges_meet(Range{d_ids, 4 * d.tokens}, y)) bad("the output overlaps an input");
    if (rows_overlap(y, x) && !y.same(x)) bad("the output overlaps an input it does not match");
    TensorDevice dev("looked-up rows", {d_ids, d_table, d_x, d_y});
    EmbedParams p{d_ids, d_table, d_x, d_y, d.tokens, d.table_rows, table.outer_stride, x.outer_stride,
                  y.outer_stride, d.channels, 0, d.scale};
    const int whole = 16 / dtype_bytes(d.dtype);
    const bool shift = (d_x ? vec_of(d, {table, x, y}) : vec_of(d, {table, y})) < whole;
    const int nvec = (d.channels + whole - 1) / whole;
    p.lanes = lanes_of(shift ? nvec + 1 : nvec, shift ? 2 : 0);
    const int64_t per = kThreads / p.lanes;
    const unsigned blocks = (unsigned)std::min<int64_t>((d.tokens + per - 1) / per, 1 << 20);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (d.dtype == KC_PRECISION_F32) run_type<float>(p, shift, blocks, st);
    else if (d.dtype == KC_PRECISION_F16) run_type<__half>(p, shift, blocks, st);
    else run_type<__nv_bfloat16>(p, shift, blocks, st);
  });
}

extern "C" int kc_embed_rows_backward_workspace(const kc_embed_desc* desc, size_t* bytes) {
  return kc::guard_entry([&] {
    kc::check_desc(desc);
    if (!bytes) kc::bad("null result");
    *bytes = kc::layout(*desc).total;
  });
}

extern "C" int kc_embed_rows_backward(const kc_embed_desc* desc, const int32_t* d_ids, const void* d_dy,
                                      float* d_dtable, void* d_workspace, size_t workspace_bytes, void* stream) {
  return kc::guard_entry([&] {
    using namespace kc;
    check_desc(desc);
    const kc_embed_desc d = *desc;
    const Rows dy = rows_of(d, d_dy, d.tokens, d.y_stride);
    check_rows(dy);
    if (!d_dtable || (d.tokens && (!d_ids || !d_dy))) bad("null tensor");
    if (!aligned_to(d_ids, 4) || !aligned_to(d_dtable, 4)) bad("a tensor is not aligned to its element");
    const Layout l = layout(d);
    const Range table{d_dtable, 4 * d.table_rows * d.channels}, ids{d_ids, 4 * d.tokens},
        space{l.total ? d_workspace : nullptr, (int64_t)l.total};
    if (ranges_meet(table, dy) || ranges_meet(table, ids)) bad("the output overlaps an input");
    if (ranges_meet(space, dy) || ranges_meet(space, ids) || ranges_meet(space, table))
      bad("the workspace overlaps another tensor of the call");
    if (l.total && (!d_workspace || workspace_bytes < l.total))
      bad("workspace of " + std::to_string(l.total) + " bytes needed");
    if (l.total && !aligned_to(d_workspace, 16)) bad("the workspace must be 16-byte aligned");
    TensorDevice dev("looked-up rows", {d_ids, d_dy, d_dtable, space.p});
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (d.tokens == 0) {
      KC_CUDA(cudaMemsetAsync(d_dtable, 0, (size_t)table.bytes, st));
      return;
    }
    char* ws = static_cast<char*>(d_workspace);
    int2 *a = reinterpret_cast<int2*>(ws + l.a), *b = reinterpret_cast<int2*>(ws + l.b);
    int* hist = reinterpret_cast<int*>(ws + l.hist);
    const bool shift = vec_of(d, {dy}) * dy.bytes < 16;
    SumParams p{};
    p.dy = d_dy;
    p.dtable = d_dtable;
    p.part = reinterpret_cast<float*>(ws + l.part);
    p.part_ids = reinterpret_cast<int2*>(ws + l.ids);
    p.ys = dy.outer_stride;
    p.tokens = (int)d.tokens;
    p.rows = (int)d.table_rows;
    p.C = d.channels;
    p.wide = d.channels % 4 == 0 && aligned_to(d_dtable, 16);
    p.scale = d.scale;
    auto run = [&](auto zero) {
      using T = decltype(zero);
      shift ? sum_type<T, true>(p, d, d_ids, a, b, hist, st) : sum_type<T, false>(p, d, d_ids, a, b, hist, st);
    };
    if (d.dtype == KC_PRECISION_F32) run(0.0f);
    else if (d.dtype == KC_PRECISION_F16) run(__half{});
    else run(__nv_bfloat16{});
  });
}
