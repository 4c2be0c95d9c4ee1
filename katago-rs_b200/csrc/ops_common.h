// What the standalone operators' entry points share: errors at the C boundary, the device their tensors live on,
// and the checks of strided tensors (all made on the host before any CUDA call).
#pragma once

#include <cstdint>
#include <exception>
#include <initializer_list>
#include <string>

#include <cuda_runtime.h>

#include "common.h"

namespace kc {

// Runs an entry point's body; nothing thrown in it crosses the C boundary.
template <typename F>
int guard_entry(F&& f) noexcept {
  try {
    f();
    set_last_error("");
    return KC_OK;
  } catch (const Error& e) {
    try { set_last_error(e.what()); } catch (...) {}
    return e.status;
  } catch (const std::exception& e) {
    try { set_last_error(std::string("CUDA backend: ") + e.what()); } catch (...) {}
    return KC_ERR_CUDA;
  } catch (...) {
    try { set_last_error("CUDA backend: unknown error"); } catch (...) {}
    return KC_ERR_CUDA;
  }
}

inline int dtype_bytes(int dtype) { return dtype == KC_PRECISION_F32 ? 4 : 2; }

// Makes the device that holds the operator's tensors current for the launch, and the caller's device again after it.
// Every pointer (null ones are skipped) has to be device memory of one device, or managed memory, which any device can
// use: the caller's where there is nothing else. A stream of another device makes the launch fail (a stream cannot be
// asked for its device while it is captured).
class TensorDevice {
 public:
  TensorDevice(const char* op, std::initializer_list<const void*> ptrs) {
    KC_CUDA(cudaGetDevice(&saved_));
    for (const void* p : ptrs) {
      if (!p) continue;
      cudaPointerAttributes a{};
      KC_CUDA(cudaPointerGetAttributes(&a, p));
      if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged)
        fail(KC_ERR_INVALID, std::string("CUDA backend: ") + op + ": a tensor is not in device memory");
      if (a.type == cudaMemoryTypeManaged) continue;
      if (dev_ >= 0 && a.device != dev_)
        fail(KC_ERR_INVALID, std::string("CUDA backend: ") + op + ": tensors on different devices");
      dev_ = a.device;
    }
    if (dev_ < 0) dev_ = saved_;
    if (dev_ != saved_) KC_CUDA(cudaSetDevice(dev_));
  }
  ~TensorDevice() {
    if (dev_ >= 0 && dev_ != saved_) cudaSetDevice(saved_);
  }
  TensorDevice(const TensorDevice&) = delete;
  TensorDevice& operator=(const TensorDevice&) = delete;
  int device() const { return dev_; }

 private:
  int saved_ = -1, dev_ = -1;
};

// A tensor of `outer` x `inner` rows of `width` consecutive elements; strides in elements.
struct Rows {
  const void* p;
  int64_t outer, inner, width, outer_stride, inner_stride;
  int bytes;  // per element

  int64_t last() const {  // elements from the first to one past the last
    return (outer - 1) * outer_stride + (inner - 1) * inner_stride + width;
  }
  bool empty() const { return !p || outer == 0 || inner == 0 || width == 0; }
  uintptr_t lo() const { return reinterpret_cast<uintptr_t>(p); }
  uintptr_t hi() const { return lo() + (uintptr_t)last() * bytes; }
  bool same(const Rows& o) const {
    return p == o.p && (outer == 1 || outer_stride == o.outer_stride) && (inner == 1 || inner_stride == o.inner_stride);
  }
};

// Whether two strided tensors share memory: exact where their outer strides are equal (slices of one wider buffer),
// otherwise whether their address ranges meet.
inline bool rows_overlap(const Rows& a, const Rows& b) {
  if (a.empty() || b.empty() || a.hi() <= b.lo() || b.hi() <= a.lo()) return false;
  // slices of one buffer of rows of S bytes: what each holds within a row
  auto apart = [](uintptr_t lo_a, int64_t ext_a, uintptr_t lo_b, int64_t ext_b, int64_t s) {
    if (s <= 0 || ext_a > s || ext_b > s) return false;
    const int64_t d = lo_b >= lo_a ? (int64_t)((lo_b - lo_a) % (uintptr_t)s)
                                   : (s - (int64_t)((lo_a - lo_b) % (uintptr_t)s)) % s;
    return d >= ext_a && d + ext_b <= s;
  };
  const int64_t sa = a.inner_stride * a.bytes, sb = b.inner_stride * b.bytes;
  const int64_t oa = a.outer_stride * a.bytes, ob = b.outer_stride * b.bytes;
  // the rows of both at one stride, in boards (tokens) of whole rows
  if (sa == sb && sa > 0 && (a.outer == 1 || oa % sa == 0) && (b.outer == 1 || ob % sb == 0) &&
      apart(a.lo(), a.width * a.bytes, b.lo(), b.width * b.bytes, sa))
    return false;
  // one outer stride: the whole inner extents apart within it
  if (oa == ob && apart(a.lo(), ((a.inner - 1) * a.inner_stride + a.width) * a.bytes, b.lo(),
                        ((b.inner - 1) * b.inner_stride + b.width) * b.bytes, oa))
    return false;
  return true;
}

// Whether the tensor's own rows share no memory (an output's must not).
inline bool rows_distinct(const Rows& a) {
  if (a.empty()) return true;
  const bool inner_ok = a.inner == 1 || a.inner_stride >= a.width;
  const int64_t inner_ext = (a.inner - 1) * a.inner_stride + a.width;
  if (inner_ok && (a.outer == 1 || a.outer_stride >= inner_ext)) return true;
  const bool outer_ok = a.outer == 1 || a.outer_stride >= a.width;  // rows of all outers side by side
  const int64_t outer_ext = (a.outer - 1) * a.outer_stride + a.width;
  return outer_ok && (a.inner == 1 || a.inner_stride >= outer_ext);
}

// Strides an operator can index with: none negative, all elements within 2^46 of the first.
inline bool rows_in_range(const Rows& a) {
  if (a.outer_stride < 0 || a.inner_stride < 0) return false;
  if (a.outer == 0 || a.inner == 0) return true;
  const __int128 last = (__int128)(a.outer - 1) * a.outer_stride + (__int128)(a.inner - 1) * a.inner_stride + a.width;
  return last <= ((__int128)1 << 46);
}

inline bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// A plain array.
struct Range {
  const void* p;
  int64_t bytes;
};

inline bool ranges_meet(const Range& a, const Rows& r) {
  if (!a.p || a.bytes <= 0 || r.empty()) return false;
  const uintptr_t lo = reinterpret_cast<uintptr_t>(a.p);
  return lo < r.hi() && r.lo() < lo + (uintptr_t)a.bytes;
}
inline bool ranges_meet(const Range& a, const Range& b) { return ranges_meet(a, Rows{b.p, 1, 1, b.bytes, 0, 0, 1}); }

}  // namespace kc
