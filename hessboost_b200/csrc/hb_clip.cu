// Global gradient norm over many tensors, and clipping by it.
//
//   norm = sqrt(sum over the tensors, and their elements, of g^2)
//   out  = g * min(1, max_norm / (norm + 1e-6))
//
// A norm that is not finite passes into every output through the factor.
#include <algorithm>

#include "hb_head.h"

namespace hb {
namespace head {
namespace {

constexpr int kClipThreads = 256;
constexpr uint64_t kChunk = 65536;  // elements of one CTA's share of a tensor
constexpr int kTable = 512;         // tensors of one launch

// The tensors of one launch, passed as a kernel argument (no device copy of
// the table). first[i] = chunks before tensor i.
struct Table {
  const void* in[kTable];
  void* out[kTable];
  uint64_t size[kTable];
  uint32_t first[kTable + 1];
  uint8_t dtype[kTable];
  int n;
};

__device__ __forceinline__ int tensor_of(const Table& t, uint32_t chunk) {
  int lo = 0, hi = t.n - 1;  // last tensor whose first chunk is <= chunk
  while (lo < hi) {
    const int m = (lo + hi + 1) >> 1;
    if (t.first[m] <= chunk) lo = m; else hi = m - 1;
  }
  return lo;
}

template <typename T>
__device__ float square_sum(const void* p, uint64_t b, uint64_t e) {
  const T* v = (const T*)p;
  float acc = 0.0f;
  for (uint64_t i = b + threadIdx.x; i < e; i += kClipThreads) {
    const float x = to_f32(v[i]);
    acc = fmaf(x, x, acc);
  }
  return acc;
}

__device__ double block_sum(double v) {
  __shared__ double s[kClipThreads];
  s[threadIdx.x] = v;
  __syncthreads();
  for (int o = kClipThreads / 2; o; o >>= 1) {
    if (threadIdx.x < o) s[threadIdx.x] += s[threadIdx.x + o];
    __syncthreads();
  }
  return s[0];
}

__global__ void __launch_bounds__(kClipThreads) k_square_sums(const __grid_constant__ Table t, double* __restrict__ sums) {
  const int i = tensor_of(t, blockIdx.x);
  const uint64_t b = (uint64_t)(blockIdx.x - t.first[i]) * kChunk, e = min(b + kChunk, t.size[i]);
  const float v = t.dtype[i] == HB_F32   ? square_sum<float>(t.in[i], b, e)
                  : t.dtype[i] == HB_F16 ? square_sum<__half>(t.in[i], b, e)
                                         : square_sum<__nv_bfloat16>(t.in[i], b, e);
  const double all = block_sum((double)v);
  if (threadIdx.x == 0) sums[blockIdx.x] = all;
}

__global__ void __launch_bounds__(kClipThreads) k_norm(const double* __restrict__ sums, uint64_t n, float* __restrict__ norm) {
  double v = 0.0;
  for (uint64_t i = threadIdx.x; i < n; i += kClipThreads) v += sums[i];
  v = block_sum(v);
  if (threadIdx.x == 0) *norm = (float)sqrt(v);
}

template <typename T>
__device__ void scale_chunk(const void* in, void* out, uint64_t b, uint64_t e, float by) {
  const T* v = (const T*)in;
  T* o = (T*)out;
  for (uint64_t i = b + threadIdx.x; i < e; i += kClipThreads) o[i] = from_f32<T>(to_f32(v[i]) * by);
}

__global__ void __launch_bounds__(kClipThreads) k_clip(const __grid_constant__ Table t, const float* __restrict__ norm, float max_norm) {
  const float q = max_norm / (*norm + 1e-6f);
  const float by = q > 1.0f ? 1.0f : q;  // NaN stays NaN
  const int i = tensor_of(t, blockIdx.x);
  const uint64_t b = (uint64_t)(blockIdx.x - t.first[i]) * kChunk, e = min(b + kChunk, t.size[i]);
  if (t.dtype[i] == HB_F32) scale_chunk<float>(t.in[i], t.out[i], b, e, by);
  else if (t.dtype[i] == HB_F16) scale_chunk<__half>(t.in[i], t.out[i], b, e, by);
  else scale_chunk<__nv_bfloat16>(t.in[i], t.out[i], b, e, by);
}

hb_status check_tensors(int32_t n, const void* const* tensors, const uint64_t* sizes, const int32_t* dtypes) {
  HB_HEAD_REQUIRE(n >= 0, "n_tensors is negative");
  HB_HEAD_REQUIRE(n == 0 || (tensors && sizes && dtypes), "tensors, sizes or dtypes is NULL");
  for (int i = 0; i < n; ++i) {
    HB_HEAD_REQUIRE(known_type(dtypes[i]), "unknown element type");
    HB_HEAD_REQUIRE(sizes[i] < (1ull << 46), "a tensor is too large");
    HB_HEAD_REQUIRE(tensors[i] || !sizes[i], "a tensor is NULL");
    HB_HEAD_REQUIRE(aligned(tensors[i], size_of(dtypes[i])), "a tensor is not aligned to its type");
  }
  return HB_OK;
}

uint64_t chunks_of(int32_t n, const uint64_t* sizes) {
  uint64_t c = 0;
  for (int i = 0; i < n; ++i) c += (sizes[i] + kChunk - 1) / kChunk;
  return c;
}

// f(table, chunks, first chunk of the launch) for every group of kTable tensors.
template <typename F>
void each_table(int32_t n, const void* const* tensors, void* const* outs, const uint64_t* sizes, const int32_t* dtypes, F&& f) {
  uint64_t before = 0;
  Table t;
  for (int a = 0; a < n;) {
    t.n = 0;
    uint32_t c = 0;
    for (; a < n && t.n < kTable && c < (1u << 30); ++a) {
      if (!sizes[a]) continue;
      t.in[t.n] = tensors[a];
      t.out[t.n] = outs ? outs[a] : nullptr;
      t.size[t.n] = sizes[a];
      t.dtype[t.n] = (uint8_t)dtypes[a];
      t.first[t.n++] = c;
      c += (uint32_t)((sizes[a] + kChunk - 1) / kChunk);
    }
    if (c) f(t, c, before);
    before += c;
  }
}

hb_status norm_launch(int32_t n, const void* const* tensors, const uint64_t* sizes, const int32_t* dtypes,
                      float* norm, double* sums, cudaStream_t s) {
  uint64_t total = 0;
  each_table(n, tensors, nullptr, sizes, dtypes, [&](const Table& t, uint32_t chunks, uint64_t before) {
    k_square_sums<<<chunks, kClipThreads, 0, s>>>(t, sums + before);
    total = before + chunks;
  });
  k_norm<<<1, kClipThreads, 0, s>>>(sums, total, norm);
  return launched("hb_grad_norm");
}

}  // namespace
}  // namespace head
}  // namespace hb

using namespace hb::head;

extern "C" {

hb_status hb_grad_norm_workspace(int32_t n_tensors, const uint64_t* sizes, uint64_t* bytes) {
  begin_call();
  HB_HEAD_REQUIRE(bytes && n_tensors >= 0 && (sizes || !n_tensors), "sizes or bytes is NULL, or n_tensors negative");
  *bytes = 8 * std::max<uint64_t>(1, chunks_of(n_tensors, sizes));
  return HB_OK;
}

hb_status hb_grad_norm(int32_t device, int32_t n_tensors, const void* const* tensors, const uint64_t* sizes,
                       const int32_t* dtypes, float* norm, void* workspace, uint64_t workspace_bytes,
                       void* stream) {
  begin_call();
  if (hb_status st = check_tensors(n_tensors, tensors, sizes, dtypes)) return st;
  HB_HEAD_REQUIRE(norm && aligned(norm, 4), "norm is NULL or not aligned");
  HB_HEAD_REQUIRE(workspace && aligned(workspace, 8) && workspace_bytes >= 8 * std::max<uint64_t>(1, chunks_of(n_tensors, sizes)),
                  "workspace is too small or not 8-byte aligned");
  DeviceScope dev(device);
  if (!dev.ok()) return fail(HB_REFUSED, "no such device");
  return norm_launch(n_tensors, tensors, sizes, dtypes, norm, (double*)workspace, (cudaStream_t)stream);
}

hb_status hb_clip_grad_norm(int32_t device, int32_t n_tensors, const void* const* tensors, void* const* outs,
                            const uint64_t* sizes, const int32_t* dtypes, float max_norm, float* norm,
                            void* workspace, uint64_t workspace_bytes, void* stream) {
  begin_call();
  if (hb_status st = check_tensors(n_tensors, tensors, sizes, dtypes)) return st;
  HB_HEAD_REQUIRE(max_norm >= 0.0f, "max_norm must be >= 0");
  HB_HEAD_REQUIRE(norm && aligned(norm, 4), "norm is NULL or not aligned");
  HB_HEAD_REQUIRE(outs || !n_tensors, "outs is NULL");
  for (int i = 0; i < n_tensors; ++i)
    HB_HEAD_REQUIRE((outs[i] || !sizes[i]) && aligned(outs[i], size_of(dtypes[i])), "an output is NULL or not aligned to its type");
  HB_HEAD_REQUIRE(workspace && aligned(workspace, 8) && workspace_bytes >= 8 * std::max<uint64_t>(1, chunks_of(n_tensors, sizes)),
                  "workspace is too small or not 8-byte aligned");
  DeviceScope dev(device);
  if (!dev.ok()) return fail(HB_REFUSED, "no such device");
  cudaStream_t s = (cudaStream_t)stream;
  if (hb_status st = norm_launch(n_tensors, tensors, sizes, dtypes, norm, (double*)workspace, s)) return st;
  each_table(n_tensors, tensors, outs, sizes, dtypes, [&](const Table& t, uint32_t chunks, uint64_t) {
    k_clip<<<chunks, kClipThreads, 0, s>>>(t, norm, max_norm);
  });
  return launched("hb_clip_grad_norm");
}

}  // extern "C"
