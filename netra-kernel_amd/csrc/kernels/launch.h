// A kernel launch with its own status: not what hipGetLastError() holds, which may
// be an error of some earlier call on the thread.
#pragma once
#include <hip/hip_runtime.h>

namespace nk {

template <typename T>
struct Same {
  using type = T;
};
template <typename... A>
hipError_t launch_kernel(void (*kernel)(A...), dim3 grid, dim3 block, hipStream_t stream,
                         typename Same<A>::type... args) noexcept {
  void* list[] = {const_cast<void*>(static_cast<const void*>(&args))...};
  const hipError_t status = hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, list, 0, stream);
  if (status != hipSuccess) (void)hipGetLastError();  // the caller of this reports it
  return status;
}

}  // namespace nk
