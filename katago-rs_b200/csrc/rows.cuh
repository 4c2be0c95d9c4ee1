// What the kernels over rows of consecutive elements share: vectors of 1 to 16 bytes of float32, f16 or bf16, sums over
// the lanes of a warp and over a block, and the addresses of rows that lie in boards.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>
#include <utility>

#include "gemm_pair.cuh"
#include "ops_common.h"

namespace kc {

// VEC neighbouring elements as one load or store.
template <typename T, int VEC>
struct RowVec {
  static constexpr int BYTES = VEC * (int)sizeof(T);
  using Raw = typename std::conditional<BYTES == 16, uint4, typename std::conditional<BYTES == 8, uint2,
              typename std::conditional<BYTES == 4, uint32_t, uint16_t>::type>::type>::type;

  __device__ static __forceinline__ Raw load(const T* p) { return *reinterpret_cast<const Raw*>(p); }
  __device__ static __forceinline__ void store(T* p, Raw r) { *reinterpret_cast<Raw*>(p) = r; }
  __device__ static __forceinline__ void unpack(const Raw& r, float (&v)[VEC]) {
    if constexpr (BYTES == 2) {
      v[0] = to_f<T>(*reinterpret_cast<const T*>(&r));
    } else {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
      if constexpr (std::is_same<T, float>::value) {
#pragma unroll
        for (int i = 0; i < VEC; i++) v[i] = __uint_as_float(w[i]);
      } else {
#pragma unroll
        for (int i = 0; i < VEC / 2; i++) {
          if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
          } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
          }
        }
      }
    }
  }
  __device__ static __forceinline__ Raw pack(const float (&v)[VEC]) {
    Raw r;
    if constexpr (BYTES == 2) {
      *reinterpret_cast<T*>(&r) = from_f<T>(v[0]);
    } else {
      uint32_t* w = reinterpret_cast<uint32_t*>(&r);
      if constexpr (std::is_same<T, float>::value) {
#pragma unroll
        for (int i = 0; i < VEC; i++) w[i] = __float_as_uint(v[i]);
      } else {
#pragma unroll
        for (int i = 0; i < VEC / 2; i++) w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
      }
    }
    return r;
  }
};

// Copies into shared memory by the thread that reads them there: no barrier, and loads in flight that take no
// registers. copy_commit() closes a group; copy_wait<N>() returns when all but the last N groups have arrived. A single
// 2-byte element comes with the 4 aligned bytes around it (`src` is the address of those: base()).
template <typename T, int VEC>
struct RowCopy {
  using V = RowVec<T, VEC>;
  static constexpr int BYTES = V::BYTES;
  using Slot = typename std::conditional<BYTES == 2, uint32_t, typename V::Raw>::type;
  __device__ static __forceinline__ const T* base(const T* p) {
    return BYTES == 2 ? reinterpret_cast<const T*>(reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)3) : p;
  }
  __device__ static __forceinline__ void copy(Slot* dst, const T* src) {
    if constexpr (BYTES == 16)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
    else
      asm volatile("cp.async.ca.shared.global [%0], [%1], %2;"
                   ::"r"(smem_u32(dst)), "l"(src), "n"(BYTES == 2 ? 4 : BYTES) : "memory");
  }
  // `high`: a single 2-byte element is the upper half of its 4 bytes
  __device__ static __forceinline__ void unpack(const Slot& s, bool high, float (&v)[VEC]) {
    if constexpr (BYTES == 2) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        v[0] = __uint_as_float((high ? s : s << 16) & 0xffff0000u);
      } else {
        const uint16_t h = (uint16_t)(high ? s >> 16 : s);
        v[0] = to_f<T>(*reinterpret_cast<const T*>(&h));
      }
    } else {
      V::unpack(s, v);
    }
  }
};
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// `r` where keep is all ones, zeros where it is 0
template <typename Raw>
__device__ __forceinline__ Raw masked(Raw r, uint32_t keep) {
  if constexpr (sizeof(Raw) == 2) {
    return r & (uint16_t)keep;
  } else {
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < (int)sizeof(Raw) / 4; i++) w[i] &= keep;
    return r;
  }
}

// VEC float32 parameters; `wide`: the array is 16-byte aligned, and `p` as far into it as VEC allows.
template <int VEC>
__device__ __forceinline__ void load_params(const float* p, bool wide, float (&v)[VEC]) {
  if (VEC % 4 == 0 && wide) {
#pragma unroll
    for (int i = 0; i < VEC / 4; i++) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(p) + i);
      v[4 * i] = f.x, v[4 * i + 1] = f.y, v[4 * i + 2] = f.z, v[4 * i + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i++) v[i] = __ldg(p + i);
  }
}

// A vector that begins `bytes` (0 to 15, UP: 1 to 16) into 32 bytes; ELEMENT bytes divide it.
template <int ELEMENT, bool UP>
__device__ __forceinline__ uint4 window(const uint4& lo, const uint4& hi, uint32_t bytes) {
  uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
  for (int k = 0; k < 6; k++) w[k] = bytes & 8 ? w[k + 2] : w[k];
#pragma unroll
  for (int k = 0; k < 5; k++) w[k] = bytes & 4 ? w[k + 1] : w[k];
  if (ELEMENT == 2) {
#pragma unroll
    for (int k = 0; k < 4; k++) w[k] = __funnelshift_r(w[k], w[k + 1], (bytes & 2) * 8);
  }
  return UP && bytes & 16 ? hi : make_uint4(w[0], w[1], w[2], w[3]);
}

// Sums over groups of `lanes` neighbouring lanes of a warp (a power of two; every lane of the warp takes part).
__device__ __forceinline__ float2 lanes_sum(float2 v, int lanes) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < lanes) {
      v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
  return v;
}

__device__ __forceinline__ float lanes_sum(float v, int lanes) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < lanes) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over a block of whole warps, the warps' sums in their order. `red` holds a value per warp; two calls in a row
// take different ones.
__device__ __forceinline__ float2 block_sum(float2 v, float2* red) {
  v = lanes_sum(v, 32);
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  v = red[0];
#pragma unroll 8
  for (int w = 1; w < blockDim.x / 32; w++) v.x += red[w].x, v.y += red[w].y;
  return v;
}

__device__ __forceinline__ float block_sum(float v, float2* red) {
  v = lanes_sum(v, 32);
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32].x = v;
  __syncthreads();
  v = red[0].x;
#pragma unroll 8
  for (int w = 1; w < blockDim.x / 32; w++) v += red[w].x;
  return v;
}

// Rows of `points` to a board. Boards whose rows go on at one stride are one long row of rows (points 0).
struct RowMap {
  int64_t points, board_stride, row_stride;
  __device__ __forceinline__ int64_t operator()(int64_t r) const {
    if (points == 0) return r * row_stride;
    int64_t b;
    if ((uint64_t)r <= 0xffffffffu) b = (uint32_t)r / (uint32_t)points;
    else b = r / points;
    return b * board_stride + (r - b * points) * row_stride;
  }
};
inline RowMap row_map(int64_t n, int64_t points, int64_t board_stride, int64_t row_stride) {
  if (n == 1) return {0, 0, row_stride};
  if (points == 1) return {0, 0, board_stride};
  if ((__int128)points * row_stride == board_stride) return {0, 0, row_stride};
  return {points, board_stride, row_stride};
}

// A launch that may start while the stream's last kernel ends; it waits (pdl_wait) before it reads what that one wrote.
template <typename... KArgs, typename... Args>
void launch_after(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  KC_CUDA(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...));
}

constexpr int kSmCount = 148;
constexpr int kMaxBlockSmem = 227 * 1024;

// Lets a kernel take all of a block's shared memory (and clusters of 16 blocks), once per device.
template <auto kernel, bool CLUSTERS = false>
void allow_block_smem() {
  static std::atomic<uint64_t> allowed[2];
  int dev = 0;
  KC_CUDA(cudaGetDevice(&dev));
  if (dev >= 128) fail(KC_ERR_INVALID, "CUDA backend: device index above 127");
  if (allowed[dev / 64].load(std::memory_order_acquire) >> (dev % 64) & 1) return;
  cudaFuncAttributes attr;
  KC_CUDA(cudaFuncGetAttributes(&attr, kernel));
  KC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               kMaxBlockSmem - (int)attr.sharedSizeBytes));
  KC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
  if (CLUSTERS) KC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  allowed[dev / 64].fetch_or(1ull << (dev % 64), std::memory_order_release);
}

}  // namespace kc
