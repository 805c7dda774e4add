// Shared helpers for the visionattn CUDA library: status codes, the per-thread
// error string, launch checking and bf16/f32 load/store helpers.
#pragma once

#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>
#include <stdio.h>

#include <algorithm>
#include <atomic>
#include <mutex>

#include "../../include/visionattn.h"

namespace va {

// Records `msg` as the calling thread's last error and returns `code`.
int set_error(int code, const char* fmt, ...);
void clear_error();

// Counts one kernel launch (reported by va_launch_count()).
void count_launch();

// Checks the launch that was just issued (invalid configuration, missing
// kernel image, …).  Asynchronous faults surface at the caller's next sync.
inline int check_launch(const char* what) {
  count_launch();
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(VA_ERR_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
  return VA_OK;
}

// Launches a kernel that may be set up while the previous one of the stream
// still runs its last blocks (programmatic dependent launch).  Such a kernel
// calls wait_for_previous() before its first access to global memory, which
// returns once all earlier work of the stream is complete and visible; the
// previous kernel may call let_next_start() at any time.
template <typename... P, typename... A>
int launch_behind(const char* what, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, A&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid, cfg.blockDim = block, cfg.dynamicSmemBytes = smem, cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr, cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  count_launch();
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(VA_ERR_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
  }
  return VA_OK;
}
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// One-time set-up that must run once on every device, such as
// cudaFuncSetAttribute(MaxDynamicSharedMemorySize), which applies to the
// current device only.  run(f) calls f() with the calling thread's current
// device unless it already succeeded there; safe from several host threads.
// Devices with an index ≥ 64 run f() on every call.
class PerDeviceOnce {
 public:
  template <typename F>
  int run(F&& f) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return set_error(VA_ERR_LAUNCH, "cudaGetDevice: %s", cudaGetErrorString(e));
    if (dev < 0 || dev >= 64) return f();
    const uint64_t bit = 1ull << dev;
    if (done_.load(std::memory_order_acquire) & bit) return VA_OK;
    std::lock_guard<std::mutex> lock(mu_);
    if (done_.load(std::memory_order_relaxed) & bit) return VA_OK;
    const int rc = f();
    if (rc == VA_OK) done_.fetch_or(bit, std::memory_order_release);
    return rc;
  }

 private:
  std::atomic<uint64_t> done_{0};
  std::mutex mu_;
};

inline int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// Scalar element access for the templated SIMT kernels (f32 or bf16 storage,
// f32 arithmetic).
template <typename T> __device__ __forceinline__ float ld(const T* p);
template <> __device__ __forceinline__ float ld<float>(const float* p) { return *p; }
template <> __device__ __forceinline__ float ld<__nv_bfloat16>(const __nv_bfloat16* p) {
  return __bfloat162float(*p);
}
template <typename T> __device__ __forceinline__ void st(T* p, float v);
template <> __device__ __forceinline__ void st<float>(float* p, float v) { *p = v; }
template <> __device__ __forceinline__ void st<__nv_bfloat16>(__nv_bfloat16* p, float v) {
  *p = __float2bfloat16_rn(v);
}

template <typename T> __device__ __forceinline__ float ldg(const T* p);
template <> __device__ __forceinline__ float ldg<float>(const float* p) { return __ldg(p); }
template <> __device__ __forceinline__ float ldg<__nv_bfloat16>(const __nv_bfloat16* p) {
  return __bfloat162float(*p);
}

// 16 bytes of f32, bf16 or f16 ↔ f32 values, two 16-bit elements an instruction
// (element by element the compiler spends several on each).
template <typename T> struct Bytes16;
template <> struct Bytes16<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const uint4& u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y), f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 put(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <> struct Bytes16<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  static __device__ __forceinline__ uint4 put(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 t = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&t);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Bytes16<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = t.x, f[2 * i + 1] = t.y;
    }
  }
  static __device__ __forceinline__ uint4 put(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 t = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&t);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

}  // namespace va

#define VA_CHECK_ARG(cond, ...)                                  \
  do {                                                           \
    if (!(cond)) return ::va::set_error(VA_ERR_SHAPE, __VA_ARGS__); \
  } while (0)
