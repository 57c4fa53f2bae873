// Shared helpers for the sm_100a kernels: storage types, conversions, warp/block reductions.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include <atomic>
#include <mutex>
#include <type_traits>
#include <utility>

#define OSB_API extern "C" __attribute__((visibility("default")))

// dtype codes used across the C interface
enum OsbDtype : int { OSB_F32 = 0, OSB_BF16 = 1 };

// error codes returned by the launch functions (besides cudaError values, which are < 10000)
enum OsbStatus : int {
  OSB_OK = 0,
  OSB_ERR_BAD_DTYPE = 10001,
  OSB_ERR_BAD_SHAPE = 10002,
  OSB_ERR_UNSUPPORTED = 10003,
  OSB_ERR_TOO_LARGE = 10004,
};

typedef __nv_bfloat16 bf16;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16 v) { return __bfloat162float(v); }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 from_f32<bf16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Sum over a block of up to 1024 threads; every thread gets the result. The order of the
// additions depends only on blockDim, so a row's result does not depend on what else is in the grid.
__device__ __forceinline__ float block_sum(float v, float* smem32) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nwarps = (blockDim.x + 31) >> 5;
  v = warp_sum(v);
  __syncthreads();  // protect smem32 from a previous use
  if (lane == 0) smem32[warp] = v;
  __syncthreads();
  float r = (lane < nwarps) ? smem32[lane] : 0.0f;
  r = warp_sum(r);
  return r;
}

__device__ __forceinline__ float block_max(float v, float* smem32) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nwarps = (blockDim.x + 31) >> 5;
  v = warp_max(v);
  __syncthreads();
  if (lane == 0) smem32[warp] = v;
  __syncthreads();
  float r = (lane < nwarps) ? smem32[lane] : -INFINITY;
  r = warp_max(r);
  return r;
}

static inline int osb_last_error() { return (int)cudaGetLastError(); }

// What a launch asks about the current device, asked once per device.
constexpr int OSB_MAX_DEVICES = 64;
static inline int osb_num_sms(int* out) {
  static std::atomic<int> known[OSB_MAX_DEVICES];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  int n = dev < OSB_MAX_DEVICES ? known[dev].load(std::memory_order_relaxed) : 0;
  if (n == 0) {
    e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return (int)e;
    if (dev < OSB_MAX_DEVICES) known[dev].store(n, std::memory_order_relaxed);
  }
  *out = n;
  return 0;
}
// Lets a kernel have this much dynamic shared memory. What it may have is never made less: a call that needs more may be between here and
// its launch, in another thread of the host.
template <auto Kernel> static inline int osb_allow_smem(size_t bytes) {
  static std::atomic<int> allowed[OSB_MAX_DEVICES];
  static std::mutex one_at_a_time;
  if (bytes <= 48 * 1024) return 0;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev >= OSB_MAX_DEVICES) return OSB_ERR_UNSUPPORTED;
  if (allowed[dev].load(std::memory_order_acquire) >= (int)bytes) return 0;
  std::lock_guard<std::mutex> lock(one_at_a_time);
  if (allowed[dev].load(std::memory_order_relaxed) >= (int)bytes) return 0;
  e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e != cudaSuccess) return (int)e;
  allowed[dev].store((int)bytes, std::memory_order_release);
  return 0;
}

// Programmatic dependent launch: a kernel launched through osb_launch may start while the kernel
// before it in the stream is finishing; it must call pdl_wait() before it reads or writes anything
// the earlier kernel touches (until then only its own set-up runs), and calls pdl_trigger() when the
// kernel after it may begin to launch. Without the launch attribute both are no-ops.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

inline int& osb_pdl_enabled() {
  static int v = 1;
  return v;
}

// cluster_x > 1 launches thread-block clusters of that many CTAs along x (gridDim.x must be a multiple).
template <typename... KArgs, typename... Args>
static inline int osb_launch_cluster(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem,
                                     cudaStream_t stream, int cluster_x, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (osb_pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  if (cluster_x > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)cluster_x;
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return (int)cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

template <typename... KArgs, typename... Args>
static inline int osb_launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                             Args&&... args) {
  return osb_launch_cluster(kernel, grid, block, smem, stream, 1, std::forward<Args>(args)...);
}

// An entry point a second time, with its arguments in an array of 64-bit words (pointers and integers as integers, numbers as doubles).
// A caller in Python packs them in half a microsecond; 26 arguments one by one are converted in four.
template <typename T> static inline T osb_word(const long long* w) {
  if constexpr (std::is_pointer<T>::value) {
    return reinterpret_cast<T>(static_cast<uintptr_t>(*w));
  } else if constexpr (std::is_floating_point<T>::value) {
    double d;
    memcpy(&d, w, sizeof d);
    return static_cast<T>(d);
  } else {
    return static_cast<T>(*w);
  }
}
template <typename R, typename... A, size_t... I>
static inline long long osb_call_packed(R (*f)(A...), const long long* words, std::index_sequence<I...>) {
  return f(osb_word<A>(words + I)...);
}
template <typename R, typename... A> static inline long long osb_call_packed(R (*f)(A...), const long long* words) {
  return osb_call_packed(f, words, std::index_sequence_for<A...>{});
}
#define OSB_PACKED(entry) \
  OSB_API long long entry##_packed(const long long* words) { return osb_call_packed(entry, words); }

// Dispatch over the two storage types: f(Tag<T>{}) is called with T = float or bf16.
template <typename T> struct Tag { typedef T type; };

template <typename F> static inline int osb_dispatch(int code, F&& f) {
  if (code == OSB_F32) return f(Tag<float>{});
  if (code == OSB_BF16) return f(Tag<bf16>{});
  return OSB_ERR_BAD_DTYPE;
}
#define OSB_T(tag) typename decltype(tag)::type
