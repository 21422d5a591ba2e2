// What the C entry points of libnetra_layers.so share: the error text, launches that stop behind
// a failed one, and checks of arguments.
#pragma once
#include "../../../include/netra_layers.h"

#include <hip/hip_runtime.h>

#include <string>

#include "../kernels/launch.h"

namespace {

thread_local std::string g_error;

// No exception leaves a C entry point: a message there is no memory for is lost.
int fail(int code, const char* name, const char* text) noexcept {
  try {
    g_error = std::string(name) + ": " + text;
  } catch (...) {
    g_error.clear();
  }
  return code;
}

// The launches of one call: behind one that failed there are no more.
class Launcher {
 public:
  explicit Launcher(hipStream_t stream) : stream_(stream) {}
  template <typename... A>
  void operator()(void (*kernel)(A...), dim3 grid, dim3 block, typename nk::Same<A>::type... args) noexcept {
    if (status_ == hipSuccess) status_ = nk::launch_kernel(kernel, grid, block, stream_, args...);
  }
  int result(const char* name) noexcept {
    if (status_ != hipSuccess) return fail(static_cast<int>(status_), name, hipGetErrorString(status_));
    g_error.clear();
    return 0;
  }

 private:
  hipStream_t stream_;
  hipError_t status_ = hipSuccess;
};

uint32_t elem(uint32_t type) { return type == NETRA_BF16 ? 2u : 4u; }
bool aligned(const void* p, uint64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

bool bad_type(uint32_t type) { return type != NETRA_BF16 && type != NETRA_F32; }
// A matrix's base has to be aligned to its elements.
bool bad_matrix(const void* p, uint32_t type, uint64_t stride, uint32_t cols) {
  return !p || bad_type(type) || stride < cols || !aligned(p, elem(type));
}

// Whether an output shares memory with an input: their byte ranges meet and they are
// not different columns of rows with one stride.
struct Span {
  const void* p;
  uint64_t stride, row, rows;  // bytes, bytes, count
};
bool share(const Span& a, const Span& b) {
  if (a.rows == 0 || b.rows == 0) return false;
  const uint64_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
  if (pa + (a.rows - 1u) * a.stride + a.row <= pb || pb + (b.rows - 1u) * b.stride + b.row <= pa) return false;
  if (a.stride != b.stride) return true;
  const uint64_t d = pb >= pa ? (pb - pa) % a.stride : (a.stride - (pa - pb) % a.stride) % a.stride;
  return d < a.row || d + b.row > a.stride;
}

bool bad_workspace(const void* p, uint64_t bytes, uint64_t need) {
  return bytes < need || (need && (!p || !aligned(p, 16)));
}

}  // namespace
