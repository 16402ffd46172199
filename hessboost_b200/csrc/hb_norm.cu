// Layer norm of rows, forward and backward.
//
//   mean = sum x / D, rstd = 1 / sqrt(sum (x - mean)^2 / D + eps)
//   xh = (x - mean) rstd, y = xh w + b
//   g = dy w, dx = rstd (g - mean(g) - xh mean(g xh))
//   dw = sum over the rows of dy xh, db = sum over the rows of dy
//
// Statistics and sums are f32; each output is rounded once.
#include <algorithm>

#include "hb_head.h"

namespace hb {
namespace head {
namespace {

constexpr int kNormThreads = 128;

__device__ float row_sum(float v, float* s) {
  s[threadIdx.x] = v;
  __syncthreads();
  for (int o = kNormThreads / 2; o; o >>= 1) {
    if (threadIdx.x < o) s[threadIdx.x] += s[threadIdx.x + o];
    __syncthreads();
  }
  const float r = s[0];
  __syncthreads();
  return r;
}

template <typename T, typename P>
__global__ void __launch_bounds__(kNormThreads)
    k_norm_forward(const T* __restrict__ x, uint64_t x_stride, uint64_t n_rows, uint32_t width,
                   const P* __restrict__ w, const P* __restrict__ b, float eps, T* __restrict__ y,
                   float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float s[kNormThreads];
  for (uint64_t r = blockIdx.x; r < n_rows; r += gridDim.x) {
    const T* xr = x + r * x_stride;
    float a = 0.0f;
    for (uint32_t d = threadIdx.x; d < width; d += kNormThreads) a += to_f32(xr[d]);
    const float mu = row_sum(a, s) / (float)width;
    a = 0.0f;
    for (uint32_t d = threadIdx.x; d < width; d += kNormThreads) {
      const float c = to_f32(xr[d]) - mu;
      a = fmaf(c, c, a);
    }
    const float rs = 1.0f / sqrtf(row_sum(a, s) / (float)width + eps);
    for (uint32_t d = threadIdx.x; d < width; d += kNormThreads) {
      const float xh = (to_f32(xr[d]) - mu) * rs;
      y[r * width + d] = from_f32<T>(fmaf(xh, w ? to_f32(w[d]) : 1.0f, b ? to_f32(b[d]) : 0.0f));
    }
    if (threadIdx.x == 0) mean[r] = mu, rstd[r] = rs;
  }
}

template <typename T, typename P>
__global__ void __launch_bounds__(kNormThreads)
    k_norm_backward(const T* __restrict__ dy, uint64_t dy_stride, const T* __restrict__ x, uint64_t x_stride,
                    uint64_t n_rows, uint32_t width, const P* __restrict__ w, const float* __restrict__ mean,
                    const float* __restrict__ rstd, T* __restrict__ dx) {
  __shared__ float s[kNormThreads];
  for (uint64_t r = blockIdx.x; r < n_rows; r += gridDim.x) {
    const T *xr = x + r * x_stride, *gr = dy + r * dy_stride;
    const float mu = mean[r], rs = rstd[r];
    float a = 0.0f, c = 0.0f;
    for (uint32_t d = threadIdx.x; d < width; d += kNormThreads) {
      const float g = to_f32(gr[d]) * (w ? to_f32(w[d]) : 1.0f);
      a += g;
      c = fmaf(g, (to_f32(xr[d]) - mu) * rs, c);
    }
    a = row_sum(a, s) / (float)width;
    c = row_sum(c, s) / (float)width;
    for (uint32_t d = threadIdx.x; d < width; d += kNormThreads) {
      const float g = to_f32(gr[d]) * (w ? to_f32(w[d]) : 1.0f), xh = (to_f32(xr[d]) - mu) * rs;
      dx[r * width + d] = from_f32<T>(rs * (g - a - xh * c));
    }
  }
}

// Slice blockIdx.y of the rows, one column a thread.
template <typename T>
__global__ void k_norm_slices(const T* __restrict__ dy, uint64_t dy_stride, const T* __restrict__ x,
                              uint64_t x_stride, uint64_t n_rows, uint32_t width,
                              const float* __restrict__ mean, const float* __restrict__ rstd,
                              float* __restrict__ part) {
  const uint32_t d = blockIdx.x * blockDim.x + threadIdx.x;
  if (d >= width) return;
  const uint64_t r0 = n_rows * blockIdx.y / gridDim.y, r1 = n_rows * (blockIdx.y + 1) / gridDim.y;
  float aw = 0.0f, ab = 0.0f;
  for (uint64_t r = r0; r < r1; ++r) {
    const float g = to_f32(dy[r * dy_stride + d]);
    aw = fmaf(g, (to_f32(x[r * x_stride + d]) - mean[r]) * rstd[r], aw);
    ab += g;
  }
  part[(uint64_t)(2 * blockIdx.y) * width + d] = aw;
  part[(uint64_t)(2 * blockIdx.y + 1) * width + d] = ab;
}

template <typename P>
__global__ void k_norm_join(const float* __restrict__ part, int slices, uint32_t width, P* __restrict__ dw,
                            P* __restrict__ db) {
  const uint32_t d = blockIdx.x * blockDim.x + threadIdx.x;
  if (d >= width) return;
  float aw = 0.0f, ab = 0.0f;
  for (int i = 0; i < slices; ++i) {
    aw += part[(uint64_t)(2 * i) * width + d];
    ab += part[(uint64_t)(2 * i + 1) * width + d];
  }
  if (dw) dw[d] = from_f32<P>(aw);
  if (db) db[d] = from_f32<P>(ab);
}

constexpr int kSlices = 128;

// f(element tag, parameter tag): parameters are of x's type or f32.
template <typename F>
void with_types(int32_t dtype, int32_t param, F&& f) {
  with_type(dtype, [&](auto t) {
    if (param == HB_F32) f(t, float{});
    else f(t, t);
  });
}

hb_status check_norm(int32_t dtype, int32_t param, uint64_t n_rows, uint32_t width) {
  HB_HEAD_REQUIRE(known_type(dtype), "unknown element type");
  HB_HEAD_REQUIRE(param == dtype || param == HB_F32, "weight and bias have x's type or f32");
  HB_HEAD_REQUIRE(width >= 1, "width must be at least 1");
  HB_HEAD_REQUIRE(n_rows < (1ull << 40), "too many rows");
  return HB_OK;
}

}  // namespace
}  // namespace head
}  // namespace hb

using namespace hb::head;

extern "C" {

hb_status hb_layer_norm_forward(int32_t device, const void* x, int32_t dtype, uint64_t x_stride, uint64_t n_rows,
                                uint32_t width, const void* weight, const void* bias, int32_t param_type,
                                float eps, void* y, float* mean, float* rstd, void* stream) {
  begin_call();
  if (hb_status st = check_norm(dtype, param_type, n_rows, width)) return st;
  if (!n_rows) return HB_OK;
  HB_HEAD_REQUIRE(x && y && mean && rstd, "x, y, mean or rstd is NULL");
  HB_HEAD_REQUIRE(x_stride >= width || n_rows == 1 || x_stride == 0, "x_stride is below width");
  HB_HEAD_REQUIRE(eps >= 0.0f, "eps must be >= 0");
  HB_HEAD_REQUIRE(aligned(x, size_of(dtype)) && aligned(y, size_of(dtype)) && aligned(weight, size_of(param_type)) &&
                      aligned(bias, size_of(param_type)) && aligned(mean, 4) && aligned(rstd, 4),
                  "a buffer is not aligned to its type");
  DeviceScope dev(device);
  if (!dev.ok()) return fail(HB_REFUSED, "no such device");
  const int grid = (int)std::min<uint64_t>(n_rows, (uint64_t)sm_count(device) * 16);
  with_types(dtype, param_type, [&](auto t, auto p) {
    using T = decltype(t);
    using P = decltype(p);
    k_norm_forward<T, P><<<grid, kNormThreads, 0, (cudaStream_t)stream>>>(
        (const T*)x, x_stride, n_rows, width, (const P*)weight, (const P*)bias, eps, (T*)y, mean, rstd);
  });
  return launched("hb_layer_norm_forward");
}

hb_status hb_layer_norm_backward_workspace(uint64_t n_rows, uint32_t width, uint64_t* bytes) {
  begin_call();
  HB_HEAD_REQUIRE(bytes && width, "bytes is NULL or width 0");
  *bytes = 8ull * kSlices * width;
  return HB_OK;
}

hb_status hb_layer_norm_backward(int32_t device, const void* dy, uint64_t dy_stride, const void* x,
                                 uint64_t x_stride, int32_t dtype, uint64_t n_rows, uint32_t width,
                                 const void* weight, int32_t param_type, const float* mean, const float* rstd,
                                 void* dx, void* dweight, void* dbias, void* workspace,
                                 uint64_t workspace_bytes, void* stream) {
  begin_call();
  if (hb_status st = check_norm(dtype, param_type, n_rows, width)) return st;
  HB_HEAD_REQUIRE(!n_rows || (dy && x && mean && rstd && dx), "dy, x, mean, rstd or dx is NULL");
  HB_HEAD_REQUIRE((x_stride >= width || n_rows <= 1 || x_stride == 0) && (dy_stride >= width || n_rows <= 1 || dy_stride == 0),
                  "a stride is below width");
  HB_HEAD_REQUIRE(aligned(x, size_of(dtype)) && aligned(dy, size_of(dtype)) && aligned(dx, size_of(dtype)) &&
                      aligned(weight, size_of(param_type)) && aligned(dweight, size_of(param_type)) &&
                      aligned(dbias, size_of(param_type)) && aligned(mean, 4) && aligned(rstd, 4),
                  "a buffer is not aligned to its type");
  const bool sums = dweight || dbias;
  HB_HEAD_REQUIRE(!sums || (workspace && aligned(workspace, 16) && workspace_bytes >= 8ull * kSlices * width),
                  "workspace is too small or not 16-byte aligned");
  DeviceScope dev(device);
  if (!dev.ok()) return fail(HB_REFUSED, "no such device");
  cudaStream_t s = (cudaStream_t)stream;
  const int grid = (int)std::min<uint64_t>(n_rows, (uint64_t)sm_count(device) * 16);
  with_types(dtype, param_type, [&](auto t, auto p) {
    using T = decltype(t);
    using P = decltype(p);
    if (n_rows)
      k_norm_backward<T, P><<<grid, kNormThreads, 0, s>>>((const T*)dy, dy_stride, (const T*)x, x_stride, n_rows, width,
                                                      (const P*)weight, mean, rstd, (T*)dx);
    if (sums) {
      const dim3 g((width + 127) / 128, kSlices);
      k_norm_slices<T><<<g, 128, 0, s>>>((const T*)dy, dy_stride, (const T*)x, x_stride, n_rows, width, mean, rstd,
                                     (float*)workspace);
      k_norm_join<P><<<(width + 127) / 128, 128, 0, s>>>((const float*)workspace, kSlices, width, (P*)dweight, (P*)dbias);
    }
  });
  return launched("hb_layer_norm_backward");
}

}  // extern "C"
