// Shared pieces of the embedding-head operators (hb_embed.cu, hb_norm.cu,
// hb_xent.cu, hb_clip.cu): element types, argument checks and the calling
// thread's last error. These operators work on device memory the caller
// owns, on the caller's stream, and allocate nothing: a call that needs
// scratch takes a workspace whose size a *_workspace function gives.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <string>

#include "../../include/hb_backend.h"

namespace hb {
namespace head {

// Records `what` as the calling thread's last head error and returns `st`.
hb_status fail(hb_status st, const std::string& what);
// Clears the calling thread's last head error.
void begin_call();
// SMs of the device (the caller has made it current).
int sm_count(int device);
// HB_OK, or HB_DEVICE_FAILED with the last launch's error text.
hb_status launched(const char* where);

// Makes `device` current for the call and puts the caller's device back.
class DeviceScope {
 public:
  explicit DeviceScope(int device) : ok_(cudaGetDevice(&prev_) == cudaSuccess && device >= 0) {
    if (ok_ && prev_ != device) {
      ok_ = cudaSetDevice(device) == cudaSuccess;
      moved_ = ok_;
    }
    if (!ok_) cudaGetLastError();
  }
  ~DeviceScope() {
    if (moved_) cudaSetDevice(prev_);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
  bool ok() const { return ok_; }

 private:
  int prev_ = 0;
  bool ok_, moved_ = false;
};

inline bool known_type(int32_t dtype) { return dtype >= HB_F32 && dtype <= HB_BF16; }
inline uint64_t size_of(int32_t dtype) { return dtype == HB_F32 ? 4 : 2; }
inline bool aligned(const void* p, uint64_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
inline uint64_t round_up(uint64_t n, uint64_t to) { return (n + to - 1) / to * to; }

__host__ __device__ inline float to_f32(float v) { return v; }
__host__ __device__ inline float to_f32(__half v) { return __half2float(v); }
__host__ __device__ inline float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V elements of T moved by one 16-byte load or store, or by two.
template <typename T, int V>
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Pack {
  T v[V];
};

// Lets kernel K have `bytes` of dynamic shared memory on the device (as much
// as there may be, once a device).
template <auto K>
void allow_shared(int device, uint32_t bytes) {
  static std::atomic<uint64_t> done{0};
  const uint64_t bit = 1ull << (device & 63);
  if (bytes <= 32 * 1024 || (done.load(std::memory_order_relaxed) & bit)) return;
  cudaFuncAttributes a;
  if (cudaFuncGetAttributes(&a, K) != cudaSuccess) return;
  if (cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448 - (int)a.sharedSizeBytes) == cudaSuccess && device < 64)
    done.fetch_or(bit, std::memory_order_relaxed);
}

// Calls f with a value of the element type `dtype` names (checked before).
template <typename F>
auto with_type(int32_t dtype, F&& f) {
  if (dtype == HB_F32) return f(float{});
  if (dtype == HB_F16) return f(__half{});
  return f(__nv_bfloat16{});
}

}  // namespace head
}  // namespace hb

// Argument checks of an entry point: the first that fails names itself.
#define HB_HEAD_REQUIRE(cond, what) \
  do {                              \
    if (!(cond)) return hb::head::fail(HB_INVALID_ARGUMENT, what); \
  } while (0)
