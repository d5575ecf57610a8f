// Element types, argument structs and small helpers shared by the UNet
// operators (group norm, cross attention).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>

#include "nova_internal.h"

namespace nova {
namespace unet {

// Element type codes of the C ABI (NOVA_DTYPE_*).
enum DType : int { kF16 = 0, kBF16 = 1, kF32 = 2 };
inline bool dtype_ok(int t) { return t == kF16 || t == kBF16 || t == kF32; }
inline int dtype_bytes(int t) { return t == kF32 ? 4 : 2; }

// SMs of the current device, asked once for each device.
inline int device_sms() {
  static std::atomic<int> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  int sms = known[dev].load(std::memory_order_relaxed);
  if (sms == 0) {
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
    known[dev].store(sms, std::memory_order_relaxed);
  }
  return sms;
}

// Lets a kernel have up to `most` bytes of dynamic shared memory, once for each device.
template <typename Kernel>
cudaError_t allow_smem(Kernel* kernel, std::atomic<unsigned long long>* done, int most) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (dev & 63);
  if (done->load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  if (e == cudaSuccess) done->fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// Makes the device that `p` lives on, and its context, current for a call: the
// threads that run a backward pass may come without a context, and a tensor may
// live on another device than the caller's current one.
class OnDeviceOf {
 public:
  explicit OnDeviceOf(const void* p) {
    cudaPointerAttributes at{};
    status_ = cudaPointerGetAttributes(&at, p);
    if (status_ == cudaSuccess && at.type != cudaMemoryTypeDevice &&
        at.type != cudaMemoryTypeManaged)
      status_ = cudaErrorInvalidValue;
    if (status_ == cudaSuccess) status_ = cudaGetDevice(&before_);
    if (status_ == cudaSuccess) status_ = cudaSetDevice(at.device);
    device_ = at.device;
  }
  ~OnDeviceOf() {
    if (before_ >= 0 && before_ != device_) cudaSetDevice(before_);
  }
  OnDeviceOf(const OnDeviceOf&) = delete;
  OnDeviceOf& operator=(const OnDeviceOf&) = delete;
  cudaError_t status() const { return status_; }

 private:
  cudaError_t status_ = cudaSuccess;
  int before_ = -1, device_ = -1;
};

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }

// Element i of a small parameter array whose type is known at run time.
__device__ __forceinline__ float load_param(const void* p, int dtype, long long i) {
  if (dtype == kF32) return static_cast<const float*>(p)[i];
  if (dtype == kF16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_param(void* p, int dtype, long long i, float v) {
  if (dtype == kF32) static_cast<float*>(p)[i] = v;
  else if (dtype == kF16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// V consecutive elements kept as they lie in memory.  V * sizeof(T) is 16 (one
// 16-byte access) or V is 1.
template <typename T, int V>
struct alignas(V == 1 ? sizeof(T) : 16) Pack {
  T e[V];
};
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  return *reinterpret_cast<const Pack<T, V>*>(p);
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& v) {
  *reinterpret_cast<Pack<T, V>*>(p) = v;
}

}  // namespace unet
}  // namespace nova
