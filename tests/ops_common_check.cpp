// The operators' shared host code (csrc/ops_common.h) against fakes of the CUDA calls it makes, without a GPU:
// argv[1] names the check, exit status 0 is success.
#include <cstdio>
#include <cstring>
#include <map>
#include <string>

#include "ops_common.h"

namespace {
std::map<const void*, cudaPointerAttributes> memory;
int current = 0;
cudaError_t pending = cudaSuccess;  // what the runtime remembers until it is asked
std::string message;
}  // namespace

extern "C" {
cudaError_t cudaGetDevice(int* d) { return *d = current, cudaSuccess; }
cudaError_t cudaSetDevice(int d) { return current = d, cudaSuccess; }
cudaError_t cudaPointerGetAttributes(cudaPointerAttributes* a, const void* p) {
  if (!memory.count(p)) return pending = cudaErrorInvalidValue;
  return *a = memory[p], cudaSuccess;
}
cudaError_t cudaGetLastError() {
  const cudaError_t e = pending;
  pending = cudaSuccess;
  return e;
}
const char* cudaGetErrorString(cudaError_t) { return "fake"; }
}

namespace kc {
void set_last_error(const std::string& msg) { message = msg; }
}  // namespace kc

namespace {
const void* add(uintptr_t p, cudaMemoryType type, int device) {
  cudaPointerAttributes a{};
  a.type = type;
  a.device = device;
  memory[reinterpret_cast<const void*>(p)] = a;
  return reinterpret_cast<const void*>(p);
}

#define EXPECT(c) \
  if (!(c)) return std::printf("%s:%d: %s (last message: %s)\n", __FILE__, __LINE__, #c, message.c_str()), 1

// Managed memory can be used from every device, so it decides on one only where no other tensor does, in any order.
int managed_memory() {
  const void* m = add(256, cudaMemoryTypeManaged, 0);
  const void* d1 = add(512, cudaMemoryTypeDevice, 1);
  const void* d0 = add(768, cudaMemoryTypeDevice, 0);
  int used = -1;
  auto call = [&](std::initializer_list<const void*> ptrs) {
    return kc::guard_entry([&] {
      kc::TensorDevice dev("op", ptrs);
      used = current;
    });
  };
  EXPECT(call({d1, m}) == KC_OK && used == 1 && current == 0);
  EXPECT(call({m, d1}) == KC_OK && used == 1 && current == 0);
  EXPECT(call({nullptr, m, m, d1, m}) == KC_OK && used == 1 && current == 0);
  EXPECT(call({m, nullptr}) == KC_OK && used == 0 && current == 0);
  EXPECT(call({m, d0, d1}) == KC_ERR_INVALID && current == 0);
  EXPECT(call({d1, m, d0}) == KC_ERR_INVALID && current == 0);
  EXPECT(call({add(1024, cudaMemoryTypeHost, 0), d1}) == KC_ERR_INVALID && current == 0);
  return 0;
}

// An error of a CUDA call belongs to the call of the operator that it failed, not to the next launch's check.
int failed_call() {
  const int rc = kc::guard_entry([] { KC_CUDA(pending = cudaErrorInvalidConfiguration); });
  EXPECT(rc == KC_ERR_CUDA && !message.empty());
  EXPECT(kc::guard_entry([] { KC_CUDA(cudaGetLastError()); }) == KC_OK);
  EXPECT(kc::guard_entry([] { kc::TensorDevice dev("op", {reinterpret_cast<const void*>(4096)}); }) == KC_ERR_CUDA);
  EXPECT(kc::guard_entry([] { KC_CUDA(cudaGetLastError()); }) == KC_OK);
  return 0;
}
}  // namespace

int main(int argc, char** argv) {
  if (argc == 2 && !std::strcmp(argv[1], "managed_memory")) return managed_memory();
  if (argc == 2 && !std::strcmp(argv[1], "failed_call")) return failed_call();
  return 2;
}
