// Shared helpers of the training-step operators (include/purin_ops.h).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <exception>
#include <type_traits>
#include <utility>

#include "../../include/purin_ops.h"

namespace purin {

// The library's thread-local error message (capi.cu); never throws.
int32_t set_error(int32_t code, const char* message) noexcept;

namespace ops {

inline int32_t invalid(const char* message) {
  return set_error(PURIN_ERR_INVALID_ARGUMENT, message);
}

// Runs a C entry point's body: no exception leaves it.
template <typename F>
int32_t guarded(F&& body) noexcept {
  try {
    return body();
  } catch (const std::exception& e) {
    return set_error(PURIN_ERR_CUDA, e.what());
  } catch (...) {
    return set_error(PURIN_ERR_CUDA, "unknown C++ exception");
  }
}

// Makes `device` current and restores the caller's device on scope exit.
struct OnDevice {
  int previous = -1, device;
  cudaError_t error;
  explicit OnDevice(int to) : device(to) {
    if (cudaGetDevice(&previous) != cudaSuccess) previous = -1;
    error = previous == device ? cudaSuccess : cudaSetDevice(device);
    if (error != cudaSuccess) cudaGetLastError();  // reported here, not by the next launch
  }
  ~OnDevice() {
    if (previous >= 0 && previous != device) cudaSetDevice(previous);
  }
};

inline int32_t cuda_status(cudaError_t e) {
  return e == cudaSuccess ? PURIN_OK : set_error(PURIN_ERR_CUDA, cudaGetErrorString(e));
}
inline int32_t launched() { return cuda_status(cudaGetLastError()); }

inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
inline size_t dtype_bytes(int32_t dtype) {
  return dtype == PURIN_OPS_FLOAT64 ? 8 : dtype == PURIN_OPS_FLOAT32 ? 4 : 2;
}
inline bool known_dtype(int32_t dtype) {
  return dtype >= PURIN_OPS_FLOAT64 && dtype <= PURIN_OPS_FLOAT16;
}
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int sm_count(int device) {
  static std::atomic<int> known[64];
  if (device < 0 || device >= 64) return 148;
  int n = known[device].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      return 148;
    }
    known[device].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Blocks of a kernel that goes round its items: one round, of 32 blocks an SM at most.
inline unsigned grid_for(int64_t items, int64_t per_block, int sms) {
  const int64_t blocks = ceil_div(items, per_block), most = int64_t(sms) * 32;
  return unsigned(blocks < most ? (blocks > 0 ? blocks : 1) : most);
}

// Sums and products are held in 32 bits, in 64 for double.
template <typename T> struct Accumulator { using type = float; };
template <> struct Accumulator<double> { using type = double; };
template <typename T> using acc_t = typename Accumulator<T>::type;

__device__ __forceinline__ double widen(double x) { return x; }
__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
template <typename T, typename A> __device__ __forceinline__ T narrow(A x);
template <> __device__ __forceinline__ double narrow<double, double>(double x) { return x; }
template <> __device__ __forceinline__ float narrow<float, float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16, float>(float x) {
  return __float2bfloat16_rn(x);
}
template <> __device__ __forceinline__ __half narrow<__half, float>(float x) {
  return __float2half_rn(x);
}

// V adjacent elements, moved as one access.
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

// Outputs larger than this are stored past L2's kept lines (evict-first): they would not stay
// there for the next reader anyway, and what is being read does.
constexpr int64_t kStreamBytes = int64_t(64) << 20;  // half of L2

template <bool kStream, typename P>
__device__ __forceinline__ void store_pack(P* to, const P& p) {
  if constexpr (kStream && sizeof(P) == 16)
    __stcs(reinterpret_cast<int4*>(to), reinterpret_cast<const int4&>(p));
  else
    *to = p;
}

// Launches of one call follow each other closely: a kernel started by launch_after may begin
// while the previous one is still running, sets itself up, and reads and writes nothing of
// others before wait_for_previous(), which returns when the previous kernel has completed and
// its writes are visible.  Every kernel of a chain waits, so the wait covers those before.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... Parameters, typename... Arguments>
cudaError_t launch_after(void (*kernel)(Parameters...), dim3 grid, dim3 block, size_t shared,
                         cudaStream_t stream, Arguments&&... arguments) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = block;
  config.dynamicSmemBytes = shared;
  config.stream = stream;
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, std::forward<Arguments>(arguments)...);
}

// Quotient and remainder of a work item's index; 64-bit division is slow and rarely needed.
__device__ __forceinline__ void divide(int64_t at, int64_t by, bool fits32, int64_t& quotient, int64_t& rest) {
  quotient = fits32 ? int64_t(uint32_t(at) / uint32_t(by)) : at / by;
  rest = at - quotient * by;
}

// True if every row of the array can be read V elements at a time.
inline bool packable(const void* p, int64_t stride, int64_t dim, size_t element, int pack) {
  const size_t bytes = element * pack;
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && (stride * element) % bytes == 0 &&
         dim % pack == 0;
}

// Calls f with a value of the element type of `dtype`.
template <typename F>
int32_t with_dtype(int32_t dtype, F&& f) {
  switch (dtype) {
    case PURIN_OPS_FLOAT64: return f(double());
    case PURIN_OPS_FLOAT32: return f(float());
    case PURIN_OPS_BFLOAT16: return f(__nv_bfloat16());
    case PURIN_OPS_FLOAT16: return f(__half());
  }
  return invalid("unknown element type");
}

}  // namespace ops
}  // namespace purin
