// Layer norm of rows, forward and backward.
//
//   mean = sum x / D, rstd = 1 / sqrt(sum (x - mean)^2 / D + eps)
//   xh = (x - mean) rstd, y = xh w + b
//   g = dy w, dx = rstd (g - mean(g) - xh mean(g xh))
//   dw = sum over the rows of dy xh, db = sum over the rows of dy
//
// Statistics and sums are f32; each output is rounded once.
//
// Bound by memory: a row is read once (x, and dy in the backward pass), and
// everything else is formed from registers. CTAs go over the rows; each
// thread's next rows are on their way into its own part of shared memory by
// asynchronous copies (a ring of 3 or 4 rows, no barrier: a thread waits for its
// own copies alone), and what is issued for an element is kept small: columns
// at constant distances, a path without bounds for warps whose columns are
// all there, two f32 at a time where a vector holds them, weights kept in
// registers. Three shapes by the row's width, the number of registers its
// threads have for it:
//   group  a power of two of a warp's lanes holds a row, up to 16 elements a
//          lane;
//   block  a CTA holds a row, up to 16 elements a thread (more do not leave
//          the backward pass registers for its column sums);
//   loop   a CTA reads a wider row again for each of its sums.
// A vector is 16 bytes where every row starts on such a boundary. Other rows
// are copied as the 16-byte units they touch, a warp's (or group's) share of
// the row to a piece of shared memory, and taken from there singly.
//
// dw and db: a thread sums its columns over the rows its CTA takes, a CTA
// writes one row of partial sums, and k_norm_join adds those in order. The
// rows are dealt to a number of CTAs that does not depend on their speed,
// so the sums' order is fixed.
#include <algorithm>
#include <type_traits>

#include "hb_head.h"

namespace hb {
namespace head {
namespace {

constexpr int kGroupThreads = 256;
// Who holds a row: a group of lanes, a CTA of which there are two an SM (the
// forward pass alone: 8,191 x 4,097 f32 take it 50 us, 78 with one; the
// backward pass's column sums then spill, 116 us for 96), or a larger one. The
// most threads of each, by the registers of 16 elements a thread: two CTAs end
// at 4,608 columns. From 600 to there, 67M elements, they are 6 to 45% faster
// in bf16 (as fast at 4,608) and 2 to 30% off 16-byte boundaries, where f32 of
// 600 columns is 6% slower; f32 vectors are 22% faster at 600 and 1 to 9%
// slower from 1,000.
enum Holder { kByGroup, kBySmall, kByLarge };
constexpr int max_threads(int holder) { return holder == kByGroup ? kGroupThreads : holder == kBySmall ? 288 : 512; }
constexpr int kLoopThreads = 512;
constexpr uint64_t kParts = 640; // rows of partial sums at most

template <typename T, int V>
__device__ __forceinline__ void unpack(const Pack<T, V>& q, float (&v)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = to_f32(q.v[j]);
}
template <typename T, int V>
__device__ __forceinline__ void load(const T* p, float (&v)[V]) {
  unpack(*reinterpret_cast<const Pack<T, V>*>(p), v);
}
template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float (&v)[V]) {
  Pack<T, V> q;
  if constexpr (V > 1 && sizeof(T) == 2) {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      if constexpr (std::is_same<T, __half>::value) *reinterpret_cast<__half2*>(&q.v[j]) = __floats2half2_rn(v[j], v[j + 1]);
      else *reinterpret_cast<__nv_bfloat162*>(&q.v[j]) = __floats2bfloat162_rn(v[j], v[j + 1]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) q.v[j] = from_f32<T>(v[j]);
  }
  *reinterpret_cast<Pack<T, V>*>(p) = q;
}

// Element by element over V floats, two to an instruction where V is even.
union Two {
  float2 f;
  unsigned long long u;
};
__device__ __forceinline__ unsigned long long two(float x, float y) {
  Two t;
  t.f = make_float2(x, y);
  return t.u;
}
// d = a b + c
template <int V>
__device__ __forceinline__ void fma_v(float (&d)[V], const float (&a)[V], const float (&b)[V], const float (&c)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      Two t;
      asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(t.u) : "l"(two(a[j], a[j + 1])), "l"(two(b[j], b[j + 1])), "l"(two(c[j], c[j + 1])));
      d[j] = t.f.x, d[j + 1] = t.f.y;
    }
  } else {
    d[0] = fmaf(a[0], b[0], c[0]);
  }
}
template <int V>
__device__ __forceinline__ void add_v(float (&d)[V], const float (&a)[V], const float (&b)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      Two t;
      asm("add.rn.f32x2 %0, %1, %2;" : "=l"(t.u) : "l"(two(a[j], a[j + 1])), "l"(two(b[j], b[j + 1])));
      d[j] = t.f.x, d[j + 1] = t.f.y;
    }
  } else {
    d[0] = a[0] + b[0];
  }
}
template <int V>
__device__ __forceinline__ void mul_v(float (&d)[V], const float (&a)[V], const float (&b)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      Two t;
      asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(t.u) : "l"(two(a[j], a[j + 1])), "l"(two(b[j], b[j + 1])));
      d[j] = t.f.x, d[j + 1] = t.f.y;
    }
  } else {
    d[0] = a[0] * b[0];
  }
}
template <int V>
struct Same {  // V copies of one value
  float v[V];
  __device__ __forceinline__ explicit Same(float x) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = x;
  }
};
// The sum of V floats and what is in them already.
template <int V>
__device__ __forceinline__ float total(const float (&v)[V]) {
  float t = v[0];
#pragma unroll
  for (int j = 1; j < V; ++j) t += v[j];
  return t;
}

// The threads of one row: a group of lanes, or a CTA.
struct Lanes {
  int size;
  __device__ __forceinline__ float2 sum(float2 v) const {
    for (int o = size >> 1; o; o >>= 1) {
      v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    return v;
  }
  __device__ __forceinline__ float sum(float v) const {
    for (int o = size >> 1; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
};
struct Cta {
  float2 (*s)[32];  // two buffers: a sum's readers may still be there when the next one is written
  int warps, turn = 0;
  // Every warp's v, one in each of the first `warps` lanes, 0 in the others.
  __device__ __forceinline__ float2 gather(float2 v) {
    if ((threadIdx.x & 31) == 0) s[turn][threadIdx.x >> 5] = v;
    // not __syncthreads: the warps may be in different copies of the loop
    asm volatile("barrier.sync 0;" ::: "memory");
    v = (threadIdx.x & 31) < warps ? s[turn][threadIdx.x & 31] : make_float2(0.0f, 0.0f);
    turn ^= 1;
    return v;
  }
  __device__ __forceinline__ float2 sum(float2 v) { return Lanes{32}.sum(gather(Lanes{32}.sum(v))); }
};

// Stages of the ring: as many as fit beside 16 elements a thread of two
// tensors (one CTA of 512 threads), or of one (two of 288).
template <int kHolder>
constexpr int kRingStages = kHolder == kByLarge ? 3 : 4;
__device__ __forceinline__ void copy_async_4(void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
// 16 bytes, of which the first `bytes` are read and the others zero.
__device__ __forceinline__ void copy_async_16(void* to, const void* from, uint32_t bytes = 16) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// The copies of all but the last kPending commits have landed.
template <int kPending>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory"); }

// A thread's part of a row: vectors at columns first + i * apart, `there` of
// them inside the row; `lanes` threads with consecutive vectors share a
// chunk of the row (a warp of a block, or a group), this one the `lane`th.
template <int V, int N, bool kBlock>
struct Part {
  uint32_t first, apart, chunk, chunk_n;  // the chunk's first column, and how many it has
  int lane, lanes, there;
  bool full;  // all vectors of the warp's threads are inside
  __device__ __forceinline__ Part(int size, uint32_t width) {
    lanes = kBlock ? 32 : size;
    lane = threadIdx.x & (lanes - 1);
    apart = lanes * V;
    chunk = kBlock ? (threadIdx.x >> 5) * (32 * N * V) : 0;
    chunk_n = chunk < width ? min((uint32_t)(lanes * N * V), width - chunk) : 0;
    first = chunk + lane * V;
    there = first < width ? min(N, (int)((width - first - 1) / apart) + 1) : 0;
    full = __all_sync(0xffffffffu, there == N);
  }
};

// A ring of kStages rows of M tensors. Vectors: a thread's own slots. Single
// elements: a chunk's units, its first element up to 15 bytes into the first.
template <typename T, int V, int N, int M, int kStages, bool kBlock>
struct RowRing {
  unsigned char* base;
  uint32_t apart;
  __device__ __forceinline__ RowRing(unsigned char* raw, const Part<V, N, kBlock>& p) {
    if constexpr (V > 1) {
      base = raw + threadIdx.x * 16;
      apart = (kBlock ? blockDim.x : kGroupThreads) * 16;
    } else {
      apart = chunk_bytes(p.lanes);
      base = raw + threadIdx.x / p.lanes * (M * kStages) * apart;
    }
  }
  __host__ __device__ static constexpr uint32_t chunk_bytes(uint32_t lanes) { return (lanes * N * (uint32_t)sizeof(T) + 15) / 16 * 16 + 16; }
  static constexpr uint32_t bytes(uint32_t threads, uint32_t lanes) {
    return V > 1 ? kStages * M * N * threads * 16 : kStages * M * (threads / lanes) * chunk_bytes(lanes);
  }
  // Starts the copy of this thread's share of the chunk at `from` (vectors:
  // of its own vectors); nothing before `begin` is read.
  template <bool kFull>
  __device__ __forceinline__ void fetch(int stage, int tensor, const T* from, const Part<V, N, kBlock>& p, const T* begin) const {
    if constexpr (V > 1) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (kFull || i < p.there) copy_async_16(base + ((stage * M + tensor) * N + i) * apart, from + i * p.apart);
    } else {
      unsigned char* to = base + (stage * M + tensor) * apart;
      const uint32_t offset = (uint32_t)(reinterpret_cast<uintptr_t>(from) & 15), total = offset + p.chunk_n * sizeof(T);
      const unsigned char* unit = reinterpret_cast<const unsigned char*>(from) - offset;
      for (uint32_t q = p.lane * 16; q < total; q += p.lanes * 16) {
        if (q == 0 && unit < reinterpret_cast<const unsigned char*>(begin)) {
          for (uint32_t k = 0; offset + k * sizeof(T) < 16 && k < p.chunk_n; ++k) reinterpret_cast<T*>(to + offset)[k] = from[k];
        } else {
          copy_async_16(to + q, unit + q, min(16u, total - q));
        }
      }
    }
  }
  // This thread's vector i of the chunk that was fetched from `from`.
  __device__ __forceinline__ void get(int stage, int tensor, int i, const T* from, const Part<V, N, kBlock>& p, float (&v)[V]) const {
    if constexpr (V > 1) {
      load<T, V>(reinterpret_cast<const T*>(base + ((stage * M + tensor) * N + i) * apart), v);
    } else {
      const uint32_t offset = (uint32_t)(reinterpret_cast<uintptr_t>(from) & 15);
      v[0] = to_f32(reinterpret_cast<const T*>(base + (stage * M + tensor) * apart + offset)[p.lane + i * p.lanes]);
    }
  }
};

// kBlock: a CTA a row, else groups of `size` lanes; N vectors a thread. The
// CTA's rows are base + group for base = blockIdx.x * rows, + the grid's, ...
template <typename T, typename P, int V, int N, int kHolder>
__global__ void __launch_bounds__(max_threads(kHolder), kHolder == kByLarge ? 1 : kHolder == kBySmall || (V == 1 && N == 16) ? 2 : 3)
    k_norm_forward(const T* __restrict__ x, uint64_t x_stride, uint64_t n_rows, uint32_t width, int size,
                   const P* __restrict__ w, const P* __restrict__ b, float eps, T* __restrict__ y,
                   float* __restrict__ mean, float* __restrict__ rstd) {
  constexpr bool kBlock = kHolder != kByGroup;
  constexpr int kStages = kRingStages<kHolder>;
  __shared__ float2 s[2][32];
  extern __shared__ __align__(16) unsigned char raw[];
  const Part<V, N, kBlock> p(size, width);
  const RowRing<T, V, N, 1, kStages, kBlock> ring(raw, p);
  const uint32_t rows = kBlock ? 1 : kGroupThreads / size, group = kBlock ? 0 : threadIdx.x / size;
  const uint32_t step = gridDim.x * rows;
  Cta cta{s, (int)blockDim.x >> 5};
  const Lanes lanes{size};
  const float count = (float)width, over = 1.0f / count;
  // elements of this warp, and of warp (lane of this one)
  const auto elements = [&](int warp) { return (float)max(0, min(32 * N * V, (int)width - warp * 32 * N * V)); };
  const float n_warp = kBlock ? elements(threadIdx.x >> 5) : 0.0f, over_warp = n_warp > 0.0f ? 1.0f / n_warp : 0.0f;
  const float n_of = kBlock && (int)(threadIdx.x & 31) < cta.warps ? elements(threadIdx.x & 31) : 0.0f;
  const float over_of = n_of > 0.0f ? 1.0f / n_of : 0.0f;
  float ww[N][V], bb[N][V];
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int j = 0; j < V; ++j) ww[i][j] = 1.0f, bb[i][j] = 0.0f;
    if (i < p.there) {
      if (w) load<P, V>(w + p.first + i * p.apart, ww[i]);
      if (b) load<P, V>(b + p.first + i * p.apart, bb[i]);
    }
  }
  // this thread's row, where it is, and the row whose copy starts next
  uint32_t r = blockIdx.x * rows + group, r_ahead = r;
  const T *at = x + (uint64_t)r * x_stride + (V > 1 ? p.first : p.chunk), *ahead = at;
  T* out = y + (uint64_t)r * width + p.first;
  const auto go = [&](auto full_tag) {
    constexpr bool kFull = decltype(full_tag)::value;
    const auto has = [&](int i) { return kFull || i < p.there; };
    const auto fetch = [&](int stage) {
      if (r_ahead < n_rows) ring.template fetch<kFull>(stage, 0, ahead, p, x);
      copy_commit();
      r_ahead += step, ahead += (uint64_t)step * x_stride;
    };
    for (int k = 0; k < kStages; ++k) fetch(k);
    for (uint32_t base = blockIdx.x * rows, stage = 0; base < n_rows; base += step) {
      const bool in = kBlock || r < n_rows;
      copy_wait<kStages - 1>();
      if constexpr (V == 1) __syncwarp();
      float v[N][V], sums[V] = {};
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (in && has(i)) {
          ring.get(stage, 0, i, at, p, v[i]);
          add_v<V>(sums, sums, v[i]);
        }
      float a = total<V>(sums);
      // the squares' sum about a mean: the row's, or first the warp's, so that
      // a CTA meets once: sum over the warps of sq + n (mean - the row's)^2
      float mu;
      if constexpr (kBlock) {
        a = Lanes{32}.sum(a);
        mu = a * over_warp;
      } else {
        mu = lanes.sum(a) / count;
      }
#pragma unroll
      for (int j = 0; j < V; ++j) sums[j] = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (in && has(i)) {
          float c[V];
          add_v<V>(c, v[i], Same<V>(-mu).v);
          fma_v<V>(sums, c, c, sums);
        }
      float sq = total<V>(sums);
      if constexpr (kBlock) {
        sq = Lanes{32}.sum(sq);
        const float2 of = cta.gather(make_float2(a, sq));  // of warp (lane of this one)
        mu = Lanes{32}.sum(of.x) / count;
        const float d = n_of > 0.0f ? fmaf(of.x, over_of, -mu) : 0.0f;
        sq = Lanes{32}.sum(fmaf(n_of * d, d, of.y));
      } else {
        sq = lanes.sum(sq);
      }
      const float rs = rsqrtf(fmaf(sq, over, eps));
      fetch(stage);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (in && has(i)) {
          add_v<V>(v[i], v[i], Same<V>(-mu).v);
          mul_v<V>(v[i], v[i], Same<V>(rs).v);
          fma_v<V>(v[i], v[i], ww[i], bb[i]);
          store<T, V>(out + i * p.apart, v[i]);
        }
      if (in && (kBlock ? threadIdx.x == 0 : p.lane == 0)) mean[r] = mu, rstd[r] = rs;
      r += step, out += (uint64_t)step * width, at += (uint64_t)step * x_stride;
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
  };
  // a CTA's warps meet inside, whichever way each one takes
  if (p.full) go(std::true_type{}); else go(std::false_type{});
}

// As k_norm_forward over the rows; their dw and db sums go to
// part[CTA][2][width], or where the grid is one CTA to dw and db.
template <typename T, typename P, int V, int N, int kHolder>
__global__ void __launch_bounds__(max_threads(kHolder), kHolder == kByGroup ? 2 : 1)
    k_norm_backward(const T* __restrict__ dy, uint64_t dy_stride, const T* __restrict__ x, uint64_t x_stride,
                    uint64_t n_rows, uint32_t width, int size, const P* __restrict__ w,
                    const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx,
                    float* __restrict__ part, P* __restrict__ dw, P* __restrict__ db) {
  constexpr bool kBlock = kHolder != kByGroup;
  constexpr int kStages = kRingStages<kHolder>;
  __shared__ float2 s[2][32];
  __shared__ float2 s_stats[kStages][kGroupThreads];  // of a group's row; block: a copy a warp
  extern __shared__ __align__(16) unsigned char raw[];
  const Part<V, N, kBlock> p(size, width);
  const RowRing<T, V, N, 2, kStages, kBlock> ring(raw, p);
  const uint32_t rows = kBlock ? 1 : kGroupThreads / size, group = kBlock ? 0 : threadIdx.x / size;
  const uint32_t holder = threadIdx.x / p.lanes;
  const uint32_t step = gridDim.x * rows;
  Cta cta{s, (int)blockDim.x >> 5};
  const Lanes lanes{size};
  const float over = 1.0f / (float)width;
  float ww[N][V], acc_w[N][V], acc_b[N][V];
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int j = 0; j < V; ++j) ww[i][j] = 1.0f, acc_w[i][j] = acc_b[i][j] = 0.0f;
    if (w && i < p.there) load<P, V>(w + p.first + i * p.apart, ww[i]);
  }
  uint32_t r = blockIdx.x * rows + group, r_ahead = r;
  const uint32_t start = V > 1 ? p.first : p.chunk;
  const T *at_x = x + (uint64_t)r * x_stride + start, *at_y = dy + (uint64_t)r * dy_stride + start;
  const T *ahead_x = at_x, *ahead_y = at_y;
  T* out = dx + (uint64_t)r * width + p.first;
  const auto go = [&](auto full_tag) {
    constexpr bool kFull = decltype(full_tag)::value;
    const auto has = [&](int i) { return kFull || i < p.there; };
    const auto fetch = [&](int stage) {
      if (r_ahead < n_rows) {
        if (p.lane == 0) {
          copy_async_4(&s_stats[stage][holder].x, mean + r_ahead);
          copy_async_4(&s_stats[stage][holder].y, rstd + r_ahead);
        }
        ring.template fetch<kFull>(stage, 0, ahead_x, p, x);
        ring.template fetch<kFull>(stage, 1, ahead_y, p, dy);
      }
      copy_commit();
      r_ahead += step, ahead_x += (uint64_t)step * x_stride, ahead_y += (uint64_t)step * dy_stride;
    };
    for (int k = 0; k < kStages; ++k) fetch(k);
    for (uint32_t base = blockIdx.x * rows, stage = 0; base < n_rows; base += step) {
      const bool in = kBlock || r < n_rows;
      copy_wait<kStages - 1>();
      __syncwarp();
      float xh[N][V], g[N][V], sum_g[V] = {}, sum_x[V] = {};
      const float2 st = in ? s_stats[stage][holder] : make_float2(0.0f, 0.0f);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (in && has(i)) {
          ring.get(stage, 0, i, at_x, p, xh[i]);
          ring.get(stage, 1, i, at_y, p, g[i]);
          add_v<V>(xh[i], xh[i], Same<V>(-st.x).v);
          mul_v<V>(xh[i], xh[i], Same<V>(st.y).v);
          fma_v<V>(acc_w[i], g[i], xh[i], acc_w[i]);
          add_v<V>(acc_b[i], acc_b[i], g[i]);
          mul_v<V>(g[i], g[i], ww[i]);
          add_v<V>(sum_g, sum_g, g[i]);
          fma_v<V>(sum_x, g[i], xh[i], sum_x);
        }
      float2 a = make_float2(total<V>(sum_g), total<V>(sum_x));
      if constexpr (kBlock) a = cta.sum(a); else a = lanes.sum(a);
      fetch(stage);  // after the sum: every lane has read the row's stats and elements
      // dx = rstd (g - xh mean(g xh)) - rstd mean(g)
      const float shift = -st.y * (a.x * over), slope = -(a.y * over);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (in && has(i)) {
          fma_v<V>(g[i], xh[i], Same<V>(slope).v, g[i]);
          fma_v<V>(g[i], g[i], Same<V>(st.y).v, Same<V>(shift).v);
          store<T, V>(out + i * p.apart, g[i]);
        }
      r += step, out += (uint64_t)step * width, at_x += (uint64_t)step * x_stride, at_y += (uint64_t)step * dy_stride;
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
  };
  if (p.full) go(std::true_type{}); else go(std::false_type{});
  if (!part && !dw && !db) return;
  const auto put = [&](uint32_t d, float2 v) {
    if (gridDim.x == 1) {
      if (dw) dw[d] = from_f32<P>(v.x);
      if (db) db[d] = from_f32<P>(v.y);
    } else {
      part[(uint64_t)(2 * blockIdx.x) * width + d] = v.x;
      part[(uint64_t)(2 * blockIdx.x + 1) * width + d] = v.y;
    }
  };
  if constexpr (kBlock) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < p.there) {
#pragma unroll
        for (int j = 0; j < V; ++j) put(p.first + i * p.apart + j, make_float2(acc_w[i][j], acc_b[i][j]));
      }
  } else {
    // the groups of a warp, then the warps in order; the ring is free by now
    float2* s_col = reinterpret_cast<float2*>(raw);  // [warp][width]
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j)
        for (int o = size; o < 32; o <<= 1) {
          acc_w[i][j] += __shfl_xor_sync(0xffffffffu, acc_w[i][j], o);
          acc_b[i][j] += __shfl_xor_sync(0xffffffffu, acc_b[i][j], o);
        }
    __syncthreads();
    if ((threadIdx.x & 31) < size) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < p.there) {
#pragma unroll
          for (int j = 0; j < V; ++j)
            s_col[(threadIdx.x >> 5) * width + p.first + i * p.apart + j] = make_float2(acc_w[i][j], acc_b[i][j]);
        }
    }
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < width; d += kGroupThreads) {
      float2 t = s_col[d];
      for (int k = 1; k < kGroupThreads / 32; ++k) t.x += s_col[k * width + d].x, t.y += s_col[k * width + d].y;
      put(d, t);
    }
  }
}

// ---- loop: rows too wide for a CTA's registers --------------------------
template <typename T, typename P>
__global__ void __launch_bounds__(kLoopThreads)
    k_norm_forward_loop(const T* __restrict__ x, uint64_t x_stride, uint64_t n_rows, uint32_t width,
                        const P* __restrict__ w, const P* __restrict__ b, float eps, T* __restrict__ y,
                        float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float2 s[2][32];
  Cta cta{s, kLoopThreads / 32};
  for (uint64_t r = blockIdx.x; r < n_rows; r += gridDim.x) {
    const T* xr = x + r * x_stride;
    float a = 0.0f;
    for (uint32_t d = threadIdx.x; d < width; d += kLoopThreads) a += to_f32(xr[d]);
    const float mu = cta.sum(make_float2(a, 0.0f)).x / (float)width;
    a = 0.0f;
    for (uint32_t d = threadIdx.x; d < width; d += kLoopThreads) {
      const float c = to_f32(xr[d]) - mu;
      a = fmaf(c, c, a);
    }
    const float rs = 1.0f / sqrtf(cta.sum(make_float2(a, 0.0f)).x / (float)width + eps);
    for (uint32_t d = threadIdx.x; d < width; d += kLoopThreads) {
      const float xh = (to_f32(xr[d]) - mu) * rs;
      y[r * width + d] = from_f32<T>(fmaf(xh, w ? to_f32(w[d]) : 1.0f, b ? to_f32(b[d]) : 0.0f));
    }
    if (threadIdx.x == 0) mean[r] = mu, rstd[r] = rs;
  }
}

template <typename T, typename P>
__global__ void __launch_bounds__(kLoopThreads)
    k_norm_backward_loop(const T* __restrict__ dy, uint64_t dy_stride, const T* __restrict__ x, uint64_t x_stride,
                         uint64_t n_rows, uint32_t width, const P* __restrict__ w, const float* __restrict__ mean,
                         const float* __restrict__ rstd, T* __restrict__ dx) {
  __shared__ float2 s[2][32];
  Cta cta{s, kLoopThreads / 32};
  for (uint64_t r = blockIdx.x; r < n_rows; r += gridDim.x) {
    const T *xr = x + r * x_stride, *gr = dy + r * dy_stride;
    const float mu = mean[r], rs = rstd[r];
    float2 a = make_float2(0.0f, 0.0f);
    for (uint32_t d = threadIdx.x; d < width; d += kLoopThreads) {
      const float g = to_f32(gr[d]) * (w ? to_f32(w[d]) : 1.0f);
      a.x += g;
      a.y = fmaf(g, (to_f32(xr[d]) - mu) * rs, a.y);
    }
    a = cta.sum(a);
    a.x /= (float)width, a.y /= (float)width;
    for (uint32_t d = threadIdx.x; d < width; d += kLoopThreads) {
      const float g = to_f32(gr[d]) * (w ? to_f32(w[d]) : 1.0f), xh = (to_f32(xr[d]) - mu) * rs;
      dx[r * width + d] = from_f32<T>(rs * (g - a.x - xh * a.y));
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

// dw and db from the parts' sums: 32 columns a CTA, its warps each a share
// of the parts in order, then the warps in order.
constexpr int kJoinWarps = 16;
template <typename P>
__global__ void __launch_bounds__(32 * kJoinWarps)
    k_norm_join(const float* __restrict__ part, int parts, uint32_t width, P* __restrict__ dw, P* __restrict__ db) {
  __shared__ float2 s[kJoinWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t d = blockIdx.x * 32 + lane;
  float2 a = make_float2(0.0f, 0.0f);
  if (d < width) {
    const int p0 = parts * warp / kJoinWarps, p1 = parts * (warp + 1) / kJoinWarps;
#pragma unroll 4
    for (int i = p0; i < p1; ++i) {
      a.x += part[(uint64_t)(2 * i) * width + d];
      a.y += part[(uint64_t)(2 * i + 1) * width + d];
    }
  }
  s[warp][lane] = a;
  __syncthreads();
  if (warp || d >= width) return;
  for (int i = 1; i < kJoinWarps; ++i) a.x += s[i][lane].x, a.y += s[i][lane].y;
  if (dw) dw[d] = from_f32<P>(a.x);
  if (db) db[d] = from_f32<P>(a.y);
}

// ---- which shape ----------------------------------------------------------
enum NormShape { kGroup, kCta, kLoop };
struct NormPlan {
  NormShape shape;
  bool vec;     // 16-byte vectors
  int items;    // vectors a thread
  int size;     // threads of a row
};
NormPlan norm_plan(uint32_t width, uint64_t elem, bool vec) {
  NormPlan p;
  p.vec = vec;
  const int v = vec ? (int)(16 / elem) : 1;
  const uint32_t n = width / v;
  const uint32_t most = 16 / v;  // vectors of a thread
  if (n > 32 * most) {
    p.items = (int)most;
    p.size = (int)round_up((n + most - 1) / most, 32);
    p.shape = p.size <= max_threads(kByLarge) ? kCta : kLoop;
    return p;
  }
  p.shape = kGroup;
  // vectors: all 16 elements a lane, for the fewest steps between lanes; single
  // elements: as many lanes as there are, for the longest runs in memory
  p.items = 1;
  while (vec ? p.items < (int)std::min(most, n) : n > 32u * p.items) p.items *= 2;
  p.size = 1;
  while ((uint32_t)(p.size * p.items) < n) p.size *= 2;
  return p;
}

// f(vector length, vectors a thread, who holds the row) as constants.
template <typename T, bool kBackward, typename F>
void with_shape(const NormPlan& p, F&& f) {
  using std::integral_constant;
  const auto items = [&](auto v) {
    constexpr int kMost = 16 / decltype(v)::value;
    const integral_constant<int, kByGroup> group;
    if constexpr (!kBackward)
      if (p.shape == kCta && p.size <= max_threads(kBySmall)) return f(v, integral_constant<int, kMost>{}, integral_constant<int, kBySmall>{});
    if (p.shape == kCta) return f(v, integral_constant<int, kMost>{}, integral_constant<int, kByLarge>{});
    if (p.items == 1) return f(v, integral_constant<int, 1>{}, group);
    if (p.items == 2) return f(v, integral_constant<int, 2>{}, group);
    if constexpr (kMost >= 4)
      if (p.items == 4) return f(v, integral_constant<int, 4>{}, group);
    if constexpr (kMost >= 16) {
      if (p.items == 8) return f(v, integral_constant<int, 8>{}, group);
      return f(v, integral_constant<int, 16>{}, group);
    }
  };
  if (p.vec) items(integral_constant<int, 16 / sizeof(T)>{});
  else items(integral_constant<int, 1>{});
}

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
  HB_HEAD_REQUIRE(width >= 1 && width < (1u << 30), "width must be in [1, 2^30)");
  HB_HEAD_REQUIRE(n_rows < (1ull << 31) - (1u << 20), "at most 2^31 - 2^20 - 1 rows");
  return HB_OK;
}

// CTAs on an SM at a time, about: by threads, shared memory and registers.
uint64_t resident(int threads, uint32_t bytes, int regs) {
  return (uint64_t)std::max(1, std::min({1536 / threads, (int)(220000 / (bytes + 9000)), 65536 / (threads * regs)}));
}
// Rows of partial sums of a backward call.
uint64_t norm_parts(uint64_t n_rows) { return std::max<uint64_t>(1, std::min(n_rows, kParts)); }

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
  const uint64_t e = size_of(dtype);
  const bool vec = aligned(x, 16) && aligned(y, 16) && aligned(weight, 16) && aligned(bias, 16) && x_stride * e % 16 == 0 &&
                   width * e % 16 == 0;
  const NormPlan p = norm_plan(width, e, vec);
  cudaStream_t s = (cudaStream_t)stream;
  const uint64_t sms = (uint64_t)sm_count(device);
  with_types(dtype, param_type, [&](auto t, auto q) {
    using T = decltype(t);
    using P = decltype(q);
    if (p.shape == kLoop) {
      const int grid = (int)std::min<uint64_t>(n_rows, sms * 4);
      k_norm_forward_loop<T, P><<<grid, kLoopThreads, 0, s>>>((const T*)x, x_stride, n_rows, width, (const P*)weight,
                                                          (const P*)bias, eps, (T*)y, mean, rstd);
      return;
    }
    with_shape<T, false>(p, [&](auto v, auto n, auto holder) {
      constexpr int V = decltype(v)::value, N = decltype(n)::value;
      constexpr int kHolder = decltype(holder)::value;
      constexpr bool kBlock = kHolder != kByGroup;
      const uint64_t rows = kBlock ? 1 : kGroupThreads / p.size;
      const int threads = kBlock ? p.size : kGroupThreads;
      const uint32_t bytes = RowRing<T, V, N, 1, kRingStages<kHolder>, kBlock>::bytes(threads, kBlock ? 32 : p.size);
      const uint64_t grid = std::min<uint64_t>((n_rows + rows - 1) / rows, resident(threads, bytes, kHolder == kBySmall ? 112 : N * V * 3 + 30) * sms);
      allow_shared<k_norm_forward<T, P, V, N, kHolder>>(device, bytes);
      k_norm_forward<T, P, V, N, kHolder><<<(unsigned)grid, threads, bytes, s>>>(
          (const T*)x, x_stride, n_rows, width, p.size, (const P*)weight, (const P*)bias, eps, (T*)y, mean, rstd);
    });
  });
  return launched("hb_layer_norm_forward");
}

hb_status hb_layer_norm_backward_workspace(uint64_t n_rows, uint32_t width, uint64_t* bytes) {
  begin_call();
  HB_HEAD_REQUIRE(bytes && width, "bytes is NULL or width 0");
  *bytes = 8 * norm_parts(n_rows) * width;
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
  HB_HEAD_REQUIRE(!sums || (workspace && aligned(workspace, 16) && workspace_bytes >= 8 * norm_parts(n_rows) * width),
                  "workspace is too small or not 16-byte aligned");
  DeviceScope dev(device);
  if (!dev.ok()) return fail(HB_REFUSED, "no such device");
  cudaStream_t s = (cudaStream_t)stream;
  const uint64_t e = size_of(dtype), pe = size_of(param_type);
  if (!n_rows) {
    bool ok = true;
    for (void* out : {dweight, dbias})
      if (out) ok = cudaMemsetAsync(out, 0, width * pe, s) == cudaSuccess && ok;
    return ok ? HB_OK : launched("hb_layer_norm_backward");
  }
  const bool vec = aligned(x, 16) && aligned(dy, 16) && aligned(dx, 16) && aligned(weight, 16) && x_stride * e % 16 == 0 &&
                   dy_stride * e % 16 == 0 && width * e % 16 == 0;
  const NormPlan p = norm_plan(width, e, vec);
  float* part = sums ? (float*)workspace : nullptr;
  const uint64_t sms = (uint64_t)sm_count(device);
  with_types(dtype, param_type, [&](auto t, auto q) {
    using T = decltype(t);
    using P = decltype(q);
    uint64_t grid = 1;
    if (p.shape == kLoop) {
      grid = std::min<uint64_t>(n_rows, sms * 4);
      k_norm_backward_loop<T, P><<<(unsigned)grid, kLoopThreads, 0, s>>>((const T*)dy, dy_stride, (const T*)x, x_stride, n_rows, width,
                                                                   (const P*)weight, mean, rstd, (T*)dx);
      grid = norm_parts(n_rows) < 64 ? norm_parts(n_rows) : 64;
      if (sums)
        k_norm_slices<T><<<dim3((width + 127) / 128, (unsigned)grid), 128, 0, s>>>((const T*)dy, dy_stride, (const T*)x, x_stride,
                                                                             n_rows, width, mean, rstd, part);
    } else {
      with_shape<T, true>(p, [&](auto v, auto n, auto holder) {
        constexpr int V = decltype(v)::value, N = decltype(n)::value;
        constexpr int kHolder = decltype(holder)::value;
      constexpr bool kBlock = kHolder != kByGroup;
        const uint64_t rows = kBlock ? 1 : kGroupThreads / p.size;
        const int threads = kBlock ? p.size : kGroupThreads;
        const uint32_t ring = RowRing<T, V, N, 2, kRingStages<kHolder>, kBlock>::bytes(threads, kBlock ? 32 : p.size);
        const uint32_t bytes = kBlock ? ring : std::max<uint32_t>(ring, 8 * (kGroupThreads / 32) * width);
        const uint64_t most = std::min<uint64_t>(kParts, resident(threads, bytes, N * V * 5 + 35) * sms);
        grid = std::min<uint64_t>((n_rows + rows - 1) / rows, most);
        allow_shared<k_norm_backward<T, P, V, N, kHolder>>(device, bytes);
        k_norm_backward<T, P, V, N, kHolder><<<(unsigned)grid, threads, bytes, s>>>(
            (const T*)dy, dy_stride, (const T*)x, x_stride, n_rows, width, p.size, (const P*)weight, mean, rstd, (T*)dx, part,
            (P*)dweight, (P*)dbias);
      });
      if (grid == 1) return;  // one CTA has written dw and db itself
    }
    if (sums) k_norm_join<P><<<(width + 31) / 32, 32 * kJoinWarps, 0, s>>>(part, (int)grid, width, (P*)dweight, (P*)dbias);
  });
  return launched("hb_layer_norm_backward");
}

}  // extern "C"
