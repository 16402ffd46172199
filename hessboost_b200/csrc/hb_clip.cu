// Global gradient norm over many tensors, and clipping by it.
//
//   norm = sqrt(sum over the tensors, and their elements, of g^2)
//   out  = g * min(1, max_norm / (norm + 1e-6))
//
// A norm that is not finite passes into every output through the factor.
// Squares and the sums of a chunk (up to 32 squares a thread) are f32 where
// they are inside its range, f64 where not; the rest of the sum is f64, in an
// order that the sizes alone decide.
//
// Bound by memory: everything is read, and for clipping read again and
// written. Tensors are cut into chunks of 1,024 vectors of 16 bytes, dealt to
// the CTAs in turn, whatever the tensors' sizes (a CTA with a run of chunks of
// its own, or loads that each had a bound to check, kept to 3.4 TB/s; this is
// 5.3). Clipping has no kernel for the norm between its two passes: every CTA
// adds the first one's sums itself.
#include <algorithm>
#include <cmath>
#include <memory>
#include <new>

#include "hb_head.h"

namespace hb {
namespace head {
namespace {

constexpr int kClipThreads = 256;
constexpr int kEach = 4;                               // vectors a thread of a chunk
constexpr uint32_t kChunk = kClipThreads * kEach;      // vectors
constexpr int kSmall = 24, kLarge = 512;               // tensors of a launch
constexpr int kCtasPerSm = 4;                          // all there at once, by their registers

// The tensors of a launch, passed as a kernel argument (no device copy of
// the table). first[i] = chunks before tensor i.
template <int kTable>
struct Table {
  const void* in[kTable];
  void* out[kTable];
  uint64_t n[kTable];
  uint32_t first[kTable + 1];
  uint8_t dtype[kTable];
  int count;
};

// A tensor's vectors: elements [head, head + V count) on 16-byte boundaries
// of `at`, of which in[] is `shift` elements past such a boundary. With a
// shift a vector comes from two units of the input, both wholly inside it.
// The elements before and after are taken singly.
struct Span {
  uint64_t head, count;
  uint32_t shift;
};
template <typename T>
__device__ __forceinline__ Span span_of(const T* in, const T* at, uint64_t n) {
  constexpr uint32_t V = 16 / sizeof(T);
  Span s;
  s.head = (16 - (reinterpret_cast<uintptr_t>(at) & 15)) % 16 / sizeof(T);
  if (s.head >= n) return {n, 0, 0};
  s.shift = (uint32_t)(reinterpret_cast<uintptr_t>(in + s.head) & 15) / sizeof(T);
  if (s.shift > s.head) s.head += V;  // the first unit begins before the tensor
  const uint64_t left = n > s.head ? n - s.head : 0;
  s.count = s.shift ? (left + s.shift) / V : left / V;
  if (s.shift) s.count = s.count ? s.count - 1 : 0;
  return s;
}

// The 16 bytes `shift` bytes into the 32 of a and b (a multiple of 2, below 16).
__device__ __forceinline__ uint4 shifted(uint4 a, uint4 b, uint32_t shift) {
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  if (shift & 8) {
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  }
  if (shift & 4) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  }
  if (shift & 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The block's sum of v, for every thread.
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double s[kClipThreads / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s[0];
#pragma unroll
  for (int w = 1; w < kClipThreads / 32; ++w) v += s[w];
  return v;
}

// This thread's squares of a chunk, in f64.
template <typename T>
__device__ __noinline__ double squares_f64(const T* in, uint64_t n, uint32_t chunk) {
  constexpr int V = 16 / sizeof(T);
  const Span s = span_of(in, in, n);
  double sum = 0.0;
  const auto add = [&](T v) {
    const double x = (double)to_f32(v);
    if (x != 0.0) sum = fma(x, x, sum);
  };
  const Pack<T, V>* from = reinterpret_cast<const Pack<T, V>*>(in + s.head);
  for (uint64_t i = (uint64_t)chunk * kChunk + threadIdx.x, k = 0; k < kEach && i < s.count; ++k, i += kClipThreads) {
    const Pack<T, V> q = from[i];
    for (int j = 0; j < V; ++j) add(q.v[j]);
  }
  if (chunk == 0)
    for (uint64_t k = threadIdx.x; k < n - s.count * V; k += kClipThreads) add(in[k < s.head ? k : k + s.count * V]);
  return sum;
}
// The same in f32, where no square leaves its range: a sum that is not finite
// may hold finite elements above 2^64, one below 2^-100 may lack squares that
// were too small for f32 (32 of them add 2^-144 to a larger sum at most).
// Those are formed again in f64: 120M bf16 take 97 us where all are, 47 else.
template <typename T>
__device__ __forceinline__ double squares(const T* in, uint64_t n, uint32_t chunk) {
  constexpr int V = 16 / sizeof(T);
  const Span s = span_of(in, in, n);
  const Pack<T, V>* from = reinterpret_cast<const Pack<T, V>*>(in + s.head) + (uint64_t)chunk * kChunk + threadIdx.x;
  const int64_t left = (int64_t)s.count - (int64_t)((uint64_t)chunk * kChunk + threadIdx.x);
  float acc[4] = {};
  bool zero = false;  // a whole chunk of zeros, as an embedding's gradient has many
  const auto add = [&](const Pack<T, V>& q) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float x = to_f32(q.v[k]);
      acc[k & 3] = fmaf(x, x, acc[k & 3]);
    }
  };
  if ((uint64_t)(chunk + 1) * kChunk <= s.count) {  // a whole chunk: its loads go out together
    Pack<T, V> q[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) q[i] = from[i * kClipThreads];
#pragma unroll
    for (int i = 0; i < kEach; ++i) add(q[i]);
    if ((acc[0] + acc[1]) + (acc[2] + acc[3]) == 0.0f) {
      zero = true;
#pragma unroll
      for (int i = 0; i < kEach; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) zero = zero && to_f32(q[i].v[k]) == 0.0f;
    }
  } else {
    for (int i = 0; i < kEach; ++i)
      if (i * kClipThreads < left) add(from[i * kClipThreads]);
  }
  if (chunk == 0) {
    const uint64_t ends = n - s.count * V;  // single elements: s.head before the vectors, the others after
    for (uint64_t k = threadIdx.x; k < ends; k += kClipThreads) {
      const float x = to_f32(in[k < s.head ? k : k + s.count * V]);
      acc[0] = fmaf(x, x, acc[0]);
      zero = zero && x == 0.0f;
    }
  }
  const float sum = (acc[0] + acc[1]) + (acc[2] + acc[3]);
  return zero || (sum >= 0x1p-100f && sum < INFINITY) ? (double)sum : squares_f64(in, n, chunk);
}

template <int kTable>
__global__ void __launch_bounds__(kClipThreads, kCtasPerSm) k_square_sums(const __grid_constant__ Table<kTable> t, double* __restrict__ sums) {
  const uint32_t chunks = t.first[t.count];
  double v = 0.0;
  int i = 0;
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    while (c >= t.first[i + 1]) ++i;
    const uint32_t k = c - t.first[i];
    v += t.dtype[i] == HB_F32   ? squares((const float*)t.in[i], t.n[i], k)
         : t.dtype[i] == HB_F16 ? squares((const __half*)t.in[i], t.n[i], k)
                                : squares((const __nv_bfloat16*)t.in[i], t.n[i], k);
  }
  v = block_sum(v);
  if (threadIdx.x == 0) sums[blockIdx.x] = v;
}

// The norm from the CTAs' sums, for every thread of the block.
__device__ __forceinline__ float norm_of(const double* __restrict__ sums, uint32_t n) {
  double v = 0.0;
  for (uint32_t i = threadIdx.x; i < n; i += kClipThreads) v += sums[i];
  return (float)sqrt(block_sum(v));
}

__global__ void __launch_bounds__(kClipThreads) k_norm(const double* __restrict__ sums, uint32_t n, float* __restrict__ norm) {
  const float v = norm_of(sums, n);
  if (threadIdx.x == 0) *norm = v;
}

template <typename T>
__device__ __forceinline__ void scale_chunk(const T* in, T* out, uint64_t n, uint32_t chunk, float by) {
  constexpr int V = 16 / sizeof(T);
  const Span s = span_of(in, out, n);
  const uint64_t first = (uint64_t)chunk * kChunk + threadIdx.x;
  const uint4* from = reinterpret_cast<const uint4*>(in + s.head - s.shift) + first;
  uint4* to = reinterpret_cast<uint4*>(out + s.head) + first;
  const uint32_t shift = s.shift * sizeof(T);
  const auto put = [&](int i, uint4 u) {
    Pack<T, V>& q = reinterpret_cast<Pack<T, V>&>(u);
#pragma unroll
    for (int k = 0; k < V; ++k) q.v[k] = from_f32<T>(to_f32(q.v[k]) * by);
    __stcs(to + i * kClipThreads, u);  // not read again: the cache is for what is
  };
  if ((uint64_t)(chunk + 1) * kChunk <= s.count) {
    uint4 a[kEach], b[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) a[i] = from[i * kClipThreads];
    if (shift) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) b[i] = from[i * kClipThreads + 1];
#pragma unroll
      for (int i = 0; i < kEach; ++i) a[i] = shifted(a[i], b[i], shift);
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) put(i, a[i]);
  } else {
    for (int i = 0; i < kEach; ++i)
      if (first + i * kClipThreads < s.count) {
        const uint4 a = from[i * kClipThreads];
        put(i, shift ? shifted(a, from[i * kClipThreads + 1], shift) : a);
      }
  }
  if (chunk == 0) {
    const uint64_t ends = n - s.count * V;
    for (uint64_t k = threadIdx.x; k < ends; k += kClipThreads) {
      const uint64_t at = k < s.head ? k : k + s.count * V;
      out[at] = from_f32<T>(to_f32(in[at]) * by);
    }
  }
}

// out = in for a launch's tensors, scaled by the norm of all launches' sums;
// in and out may be the same tensors.
template <int kTable>
__global__ void __launch_bounds__(kClipThreads, kCtasPerSm)
    k_clip(const __grid_constant__ Table<kTable> t, const double* __restrict__ sums, uint32_t n_sums, float max_norm, float* __restrict__ norm) {
  const float all = norm_of(sums, n_sums);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = all;
  const float q = max_norm / (all + 1e-6f);
  const float by = q > 1.0f ? 1.0f : q;  // NaN stays NaN
  const uint32_t chunks = t.first[t.count];
  int i = 0;
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    while (c >= t.first[i + 1]) ++i;
    const uint32_t k = c - t.first[i];
    if (t.dtype[i] == HB_F32) scale_chunk((const float*)t.in[i], (float*)t.out[i], t.n[i], k, by);
    else if (t.dtype[i] == HB_F16) scale_chunk((const __half*)t.in[i], (__half*)t.out[i], t.n[i], k, by);
    else scale_chunk((const __nv_bfloat16*)t.in[i], (__nv_bfloat16*)t.out[i], t.n[i], k, by);
  }
}

hb_status check_tensors(int32_t n, const void* const* tensors, const uint64_t* sizes, const int32_t* dtypes) {
  HB_HEAD_REQUIRE(n >= 0, "n_tensors is negative");
  HB_HEAD_REQUIRE(n == 0 || (tensors && sizes && dtypes), "tensors, sizes or dtypes is NULL");
  for (int i = 0; i < n; ++i) {
    HB_HEAD_REQUIRE(known_type(dtypes[i]), "unknown element type");
    HB_HEAD_REQUIRE(sizes[i] < (1ull << 42), "a tensor is too large");
    HB_HEAD_REQUIRE(tensors[i] || !sizes[i], "a tensor is NULL");
    HB_HEAD_REQUIRE(aligned(tensors[i], size_of(dtypes[i])), "a tensor is not aligned to its type");
  }
  return HB_OK;
}

// No output may overlap another output, nor an input but its own, which it
// then is: the chunks of a call run in no order, so an element that two of them
// wrote, or one read and one wrote, would be scaled once or twice by chance.
hb_status check_apart(int32_t n, const void* const* tensors, void* const* outs, const uint64_t* sizes, const int32_t* dtypes) {
  struct Range {
    uintptr_t begin, end;
  };
  if (!n) return HB_OK;
  const std::unique_ptr<Range[]> ranges(new (std::nothrow) Range[n]);
  if (!ranges) return fail(HB_REFUSED, "out of host memory");
  const auto range = [&](int i, const void* p) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    return Range{at, at + sizes[i] * size_of(dtypes[i])};
  };
  int count = 0;
  for (int i = 0; i < n; ++i)
    if (sizes[i]) ranges[count++] = range(i, outs[i]);
  std::sort(ranges.get(), ranges.get() + count, [](const Range& a, const Range& b) { return a.begin < b.begin; });
  for (int i = 1; i < count; ++i) HB_HEAD_REQUIRE(ranges[i].begin >= ranges[i - 1].end, "two outputs overlap");
  for (int i = 0; i < n; ++i) {
    if (!sizes[i] || tensors[i] == outs[i]) continue;  // its own output, which is apart from the others
    const Range r = range(i, tensors[i]);
    // the last output that begins before the input's end: those before it end before it begins
    const Range* after = std::lower_bound(ranges.get(), ranges.get() + count, r.end, [](const Range& a, uintptr_t v) { return a.begin < v; });
    HB_HEAD_REQUIRE(after == ranges.get() || after[-1].end <= r.begin, "an output overlaps an input that is not its own");
  }
  return HB_OK;
}

// Chunks of a tensor: of its vectors, one at least for its other elements.
uint32_t chunks_of(uint64_t n, int32_t dtype) {
  return (uint32_t)std::max<uint64_t>(1, (n * size_of(dtype) / 16 + kChunk - 1) / kChunk);
}
uint32_t ctas_of(uint32_t chunks, int sms) { return std::min(chunks, (uint32_t)(sms * kCtasPerSm)); }

// f(table of the next tensors, CTAs) for group after group of them.
template <int kTable, typename F>
void each_table(int32_t n, const void* const* tensors, void* const* outs, const uint64_t* sizes, const int32_t* dtypes, int sms, F&& f) {
  Table<kTable> t;
  for (int a = 0; a < n;) {
    t.count = 0;
    uint32_t c = 0;
    for (; a < n && t.count < kTable && c < (1u << 30); ++a) {
      if (!sizes[a]) continue;
      t.in[t.count] = tensors[a];
      t.out[t.count] = outs ? outs[a] : nullptr;
      t.n[t.count] = sizes[a];
      t.dtype[t.count] = (uint8_t)dtypes[a];
      t.first[t.count++] = c;
      c += chunks_of(sizes[a], dtypes[a]);
    }
    t.first[t.count] = c;
    if (c) f(t, ctas_of(c, sms));
  }
}
// Sums that a call's launches leave, at most: a launch's tensors are full
// groups but the last's.
uint64_t most_sums(int32_t n, int sms) { return (uint64_t)(n / kLarge + 2) * sms * kCtasPerSm; }

template <int kTable>
uint32_t sum_launches(int32_t n, const void* const* tensors, const uint64_t* sizes, const int32_t* dtypes, double* sums, int sms, cudaStream_t s) {
  uint32_t before = 0;
  each_table<kTable>(n, tensors, nullptr, sizes, dtypes, sms, [&](const Table<kTable>& t, uint32_t ctas) {
    k_square_sums<kTable><<<ctas, kClipThreads, 0, s>>>(t, sums + before);
    before += ctas;
  });
  return before;
}

}  // namespace
}  // namespace head
}  // namespace hb

using namespace hb::head;

extern "C" {

hb_status hb_grad_norm_workspace(int32_t device, int32_t n_tensors, uint64_t* bytes) {
  begin_call();
  HB_HEAD_REQUIRE(bytes && n_tensors >= 0, "bytes is NULL or n_tensors negative");
  *bytes = 8 * most_sums(n_tensors, sm_count(device));
  return HB_OK;
}

hb_status hb_grad_norm(int32_t device, int32_t n_tensors, const void* const* tensors, const uint64_t* sizes,
                       const int32_t* dtypes, float* norm, void* workspace, uint64_t workspace_bytes,
                       void* stream) {
  begin_call();
  if (hb_status st = check_tensors(n_tensors, tensors, sizes, dtypes)) return st;
  HB_HEAD_REQUIRE(norm && aligned(norm, 4), "norm is NULL or not aligned");
  const int sms = sm_count(device);
  HB_HEAD_REQUIRE(workspace && aligned(workspace, 8) && workspace_bytes >= 8 * most_sums(n_tensors, sms),
                  "workspace is too small or not 8-byte aligned");
  DeviceScope dev(device);
  if (!dev.ok()) return fail(HB_REFUSED, "no such device");
  cudaStream_t s = (cudaStream_t)stream;
  double* sums = (double*)workspace;
  const uint32_t n = n_tensors <= kSmall ? sum_launches<kSmall>(n_tensors, tensors, sizes, dtypes, sums, sms, s)
                                         : sum_launches<kLarge>(n_tensors, tensors, sizes, dtypes, sums, sms, s);
  k_norm<<<1, kClipThreads, 0, s>>>(sums, n, norm);
  return launched("hb_grad_norm");
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
  if (hb_status st = check_apart(n_tensors, tensors, outs, sizes, dtypes)) return st;
  const int sms = sm_count(device);
  HB_HEAD_REQUIRE(workspace && aligned(workspace, 8) && workspace_bytes >= 8 * most_sums(n_tensors, sms),
                  "workspace is too small or not 8-byte aligned");
  DeviceScope dev(device);
  if (!dev.ok()) return fail(HB_REFUSED, "no such device");
  cudaStream_t s = (cudaStream_t)stream;
  double* sums = (double*)workspace;
  const auto run = [&](auto table) {
    constexpr int kTable = decltype(table)::value;
    const uint32_t n = sum_launches<kTable>(n_tensors, tensors, sizes, dtypes, sums, sms, s);
    float* to = norm;  // the first launch writes it
    each_table<kTable>(n_tensors, tensors, outs, sizes, dtypes, sms, [&](const Table<kTable>& t, uint32_t ctas) {
      k_clip<kTable><<<ctas, kClipThreads, 0, s>>>(t, sums, n, max_norm, to);
      to = nullptr;
    });
    if (to) k_norm<<<1, kClipThreads, 0, s>>>(sums, n, norm);  // no element at all
  };
  if (n_tensors <= kSmall) run(std::integral_constant<int, kSmall>{});
  else run(std::integral_constant<int, kLarge>{});
  return launched("hb_clip_grad_norm");
}

}  // extern "C"
