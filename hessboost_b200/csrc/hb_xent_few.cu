// Linear softmax cross entropy over a few classes in f32, where the logits of
// a row fit a thread's registers: x is read once forward and once backward,
// without the three-piece products (hb_xent_mma.cu) that f32 takes there.
//
// A CTA keeps the weights in shared memory, [column][class]; a thread has one
// row of a tile of 128. x comes in pieces of 32 columns by asynchronous
// copies into a ring of kHeld pieces, all of them at once where the width
// allows; backward then takes x from there again. A thread turns its logits
// into its row of G; for each piece a warp sums dw over its 32 rows in order
// and the warps' sums are added in order to the CTA's, and each thread forms
// its row's piece of dx in x's place. The CTAs' sums of dw are added in order
// at the end.
//
// Bound by the broadcast reads of the weights (a 16-byte one for four products
// of a row): 131,072 x 100 rows and 10 classes take 43 us forward and 102 us
// backward, where x's bytes alone would take 8 and 16.
#include <algorithm>
#include <cmath>

#include "hb_xent.h"

namespace hb {
namespace head {
namespace {

constexpr int kFewThreads = 128;        // and rows of a tile
constexpr int kWarps = kFewThreads / 32;
constexpr int kPiece = 32;              // columns of a piece
constexpr int kHeld = 4;                // pieces in shared memory
constexpr int kRowStride = kPiece + 1;  // of a piece's row
constexpr uint32_t kPieceFloats = kFewThreads * kRowStride;

struct FewParams {
  const float *x, *w;
  const void* labels;
  uint64_t x_stride, w_stride, n_rows;
  uint32_t width;
  int n_classes, label_type;
  float *loss, *lse;         // forward writes both, backward reads lse
  const float* dloss;
  uint64_t dloss_stride;
  float *dx, *dw;
  float* part;               // [CTA][classes][width]
  __device__ __forceinline__ int label(uint64_t row) const {
    const int64_t v = label_type == HB_I32 ? (int64_t)((const int32_t*)labels)[row] : ((const int64_t*)labels)[row];
    return v >= 0 && v < n_classes ? (int)v : -1;
  }
};

__host__ __device__ constexpr uint32_t pieces_of(uint32_t width) { return (width + kPiece - 1) / kPiece; }
// Floats of shared memory: the weights, the pieces, and backward dw's sums,
// the warps' parts of them and G.
template <int kClasses>
struct Few {
  static constexpr int kGStride = kClasses + 4;  // whole 16-byte units
  static uint32_t weights(uint32_t width) { return pieces_of(width) * kPiece * kClasses; }
  static uint32_t held(uint32_t width) { return std::min<uint32_t>(kHeld, pieces_of(width)) * kPieceFloats; }
  static uint32_t forward_bytes(uint32_t width) { return 4 * (weights(width) + held(width)); }
  static uint32_t backward_bytes(uint32_t width) {
    return forward_bytes(width) + 4 * (weights(width) + kWarps * kPiece * kClasses + kFewThreads * kGStride);
  }
};

// The weights, [column][class], zeros past either's end.
template <int kClasses>
__device__ __forceinline__ void load_weights(const FewParams& p, float* s_w) {
  const uint32_t columns = pieces_of(p.width) * kPiece;
  for (uint32_t i = threadIdx.x; i < columns * kClasses; i += kFewThreads) {
    const uint32_t v = i / columns, d = i - v * columns;
    s_w[d * kClasses + v] = v < (uint32_t)p.n_classes && d < p.width ? p.w[v * p.w_stride + d] : 0.0f;
  }
}

// The ring of a tile's pieces: load k is of piece k mod pieces, into place k
// mod kHeld; `loads` of them in all.
struct Pieces {
  float* s_x;
  uint32_t pieces, loads;
  __device__ __forceinline__ float* at(uint32_t k) const { return s_x + k % kHeld * kPieceFloats; }
  // Starts load k, a warp a row at a time (zeros past either end), or nothing.
  __device__ __forceinline__ void load(const FewParams& p, uint64_t row0, uint32_t k) const {
    if (k < loads) {
      const int lane = threadIdx.x & 31;
      const uint32_t d = k % pieces * kPiece + lane;
      const uint32_t rows = (uint32_t)min((uint64_t)kFewThreads, p.n_rows - row0);
      const float* from = p.x + row0 * p.x_stride + d;
      float* to = at(k) + lane;
#pragma unroll 8
      for (uint32_t r = threadIdx.x >> 5; r < kFewThreads; r += kWarps) {
        if (r < rows && d < p.width)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(to + r * kRowStride)),
                       "l"(from + r * p.x_stride)
                       : "memory");
        else
          to[r * kRowStride] = 0.0f;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  __device__ __forceinline__ void begin(const FewParams& p, uint64_t row0) const {
    for (uint32_t k = 0; k < kHeld; ++k) load(p, row0, k);
  }
  // The oldest load but kHeld - 1 has landed, for every thread.
  __device__ __forceinline__ void wait() const {
    asm volatile("cp.async.wait_group %0;" ::"n"(kHeld - 1) : "memory");
    __syncthreads();
  }
};

__device__ __forceinline__ void fma2(float& a0, float& a1, float b0, float b1, float c) {
  float2 a = make_float2(a0, a1), b = make_float2(b0, b1), cc = make_float2(c, c);
  asm("fma.rn.f32x2 %0, %1, %2, %0;"
      : "+l"(reinterpret_cast<unsigned long long&>(a))
      : "l"(reinterpret_cast<unsigned long long&>(b)), "l"(reinterpret_cast<unsigned long long&>(cc)));
  a0 = a.x, a1 = a.y;
}

// The logits of the thread's row; load k is used and load k + kHeld started.
template <int kClasses>
__device__ __forceinline__ void logits(const FewParams& p, const float* s_w, const Pieces& x, uint64_t row0, float (&z)[kClasses]) {
#pragma unroll
  for (int v = 0; v < kClasses; ++v) z[v] = 0.0f;
  for (uint32_t k = 0; k < x.pieces; ++k) {
    x.wait();
    const float* mine = x.at(k) + threadIdx.x * kRowStride;
    const float4* w = reinterpret_cast<const float4*>(s_w + k * kPiece * kClasses);
#pragma unroll 8
    for (int d = 0; d < kPiece; ++d) {
      const float a = mine[d];
#pragma unroll
      for (int v = 0; v < kClasses / 4; ++v) {
        const float4 q = w[d * (kClasses / 4) + v];
        fma2(z[4 * v], z[4 * v + 1], q.x, q.y, a);
        fma2(z[4 * v + 2], z[4 * v + 3], q.z, q.w, a);
      }
    }
    if (k + kHeld < x.loads) __syncthreads();
    x.load(p, row0, k + kHeld);
  }
}

template <int kClasses>
__global__ void __launch_bounds__(kFewThreads) k_few_forward(const FewParams p) {
  extern __shared__ __align__(16) float sm[];
  const uint32_t pieces = pieces_of(p.width);
  float* s_w = sm;
  const Pieces x{s_w + pieces * kPiece * kClasses, pieces, pieces};
  uint64_t row0 = (uint64_t)blockIdx.x * kFewThreads;
  x.begin(p, row0);
  load_weights<kClasses>(p, s_w);
  while (true) {
    const uint64_t r = row0 + threadIdx.x, next = row0 + (uint64_t)gridDim.x * kFewThreads;
    const int label = r < p.n_rows ? p.label(r) : -1;
    float z[kClasses];
    logits<kClasses>(p, s_w, x, row0, z);
    if (next < p.n_rows) {
      __syncthreads();
      x.begin(p, next);
    }
    if (r < p.n_rows) {
      float top = -INFINITY, at = 0.0f, s = 0.0f;
#pragma unroll
      for (int v = 0; v < kClasses; ++v) {
        if (v < p.n_classes) top = fmaxf(top, z[v]);
        if (v == label) at = z[v];
      }
      const float from = top == -INFINITY ? 0.0f : top;
#pragma unroll
      for (int v = 0; v < kClasses; ++v)
        if (v < p.n_classes) s += expf(z[v] - from);
      const float lse = from + logf(s);
      p.lse[r] = lse;
      p.loss[r] = label >= 0 ? lse - at : 0.0f;
    }
    if (next >= p.n_rows) break;
    row0 = next;
  }
}

template <int kClasses>
__global__ void __launch_bounds__(kFewThreads) k_few_backward(const FewParams p) {
  using F = Few<kClasses>;
  extern __shared__ __align__(16) float sm[];
  const uint32_t pieces = pieces_of(p.width), weights = pieces * kPiece * kClasses;
  float* s_w = sm;
  float* s_dw = s_w + weights;                          // [column][class]
  float* s_sum = s_dw + weights;                        // [warp][class][column of the piece]
  float* s_g = s_sum + kWarps * kPiece * kClasses;      // [row][kGStride]
  const bool held = pieces <= kHeld;                    // x stays for the second pass
  const Pieces x{s_g + kFewThreads * F::kGStride, pieces, held ? pieces : 2 * pieces};
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t row0 = (uint64_t)blockIdx.x * kFewThreads;
  x.begin(p, row0);
  load_weights<kClasses>(p, s_w);
  for (uint32_t i = threadIdx.x; i < weights; i += kFewThreads) s_dw[i] = 0.0f;
  while (true) {
    const uint64_t r = row0 + threadIdx.x, next = row0 + (uint64_t)gridDim.x * kFewThreads;
    const int label = r < p.n_rows ? p.label(r) : -1;
    const float each = label >= 0 ? p.dloss[r * p.dloss_stride] : 0.0f, lse = label >= 0 ? p.lse[r] : 0.0f;
    float g[kClasses];
    logits<kClasses>(p, s_w, x, row0, g);
#pragma unroll
    for (int v = 0; v < kClasses; ++v)
      g[v] = label >= 0 && v < p.n_classes ? each * (expf(g[v] - lse) - (v == label ? 1.0f : 0.0f)) : 0.0f;
#pragma unroll
    for (int v = 0; v < kClasses; v += 4)
      *reinterpret_cast<float4*>(s_g + threadIdx.x * F::kGStride + v) = make_float4(g[v], g[v + 1], g[v + 2], g[v + 3]);
    for (uint32_t k = 0; k < pieces; ++k) {
      const uint32_t load = held ? k : pieces + k;
      if (!held) x.wait();
      float* s_x = x.at(load);
      // a row without a label adds nothing to dw, whatever it holds
      if (label < 0)
        for (int d = 0; d < kPiece; ++d) s_x[threadIdx.x * kRowStride + d] = 0.0f;
      __syncwarp();
      // dw: column `lane` over the warp's rows (its own: their G is there too)
      float acc[kClasses];
#pragma unroll
      for (int v = 0; v < kClasses; ++v) acc[v] = 0.0f;
#pragma unroll 4
      for (int i = 0; i < 32; ++i) {
        const float a = s_x[(warp * 32 + i) * kRowStride + lane];
        const float4* gr = reinterpret_cast<const float4*>(s_g + (warp * 32 + i) * F::kGStride);
#pragma unroll
        for (int v = 0; v < kClasses / 4; ++v) {
          const float4 q = gr[v];
          fma2(acc[4 * v], acc[4 * v + 1], q.x, q.y, a);
          fma2(acc[4 * v + 2], acc[4 * v + 3], q.z, q.w, a);
        }
      }
#pragma unroll
      for (int v = 0; v < kClasses; ++v) s_sum[(warp * kClasses + v) * kPiece + lane] = acc[v];
      __syncwarp();
      // dx of the thread's row, in x's place
      const float4* w = reinterpret_cast<const float4*>(s_w + k * kPiece * kClasses);
#pragma unroll 8
      for (int d = 0; d < kPiece; ++d) {
        float a = 0.0f, b = 0.0f;
#pragma unroll
        for (int v = 0; v < kClasses / 4; ++v) {
          const float4 q = w[d * (kClasses / 4) + v];
          a = fmaf(g[4 * v], q.x, a), b = fmaf(g[4 * v + 1], q.y, b);
          a = fmaf(g[4 * v + 2], q.z, a), b = fmaf(g[4 * v + 3], q.w, b);
        }
        s_x[threadIdx.x * kRowStride + d] = a + b;
      }
      __syncthreads();
      for (int v = warp; v < kClasses; v += kWarps) {
        float t = s_sum[v * kPiece + lane];
#pragma unroll
        for (int q = 1; q < kWarps; ++q) t += s_sum[(q * kClasses + v) * kPiece + lane];
        s_dw[(k * kPiece + lane) * kClasses + v] += t;
      }
      const uint32_t d = k * kPiece + lane;
      if (d < p.width) {
        const uint32_t rows = (uint32_t)min((uint64_t)kFewThreads, p.n_rows - row0);
        float* out = p.dx + row0 * p.width + d;
#pragma unroll 8
        for (uint32_t i = warp; i < rows; i += kWarps) out[(uint64_t)i * p.width] = s_x[i * kRowStride + lane];
      }
      __syncthreads();
      if (!held) x.load(p, row0, load + kHeld);
    }
    if (next >= p.n_rows) break;
    row0 = next;
    // (not held: the loads past the last were empty, as begin's first ones wait for nothing)
    x.begin(p, row0);
  }
  const uint32_t all = (uint32_t)p.n_classes * p.width;
  for (uint32_t i = threadIdx.x; i < all; i += kFewThreads) {
    const uint32_t v = i / p.width, d = i - v * p.width;
    const float q = s_dw[d * kClasses + v];
    if (gridDim.x == 1) p.dw[i] = q;
    else p.part[(uint64_t)blockIdx.x * all + i] = q;
  }
}

// dw from the CTAs' sums: 32 elements a CTA, its warps each a share of the
// sums in order, then the warps in order.
constexpr int kJoinWarps = 8;
__global__ void __launch_bounds__(32 * kJoinWarps) k_few_join(const float* __restrict__ part, int parts, uint32_t n, float* __restrict__ dw) {
  __shared__ float s[kJoinWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t i = blockIdx.x * 32 + lane;
  float a = 0.0f;
  if (i < n) {
#pragma unroll 8
    for (int k = parts * warp / kJoinWarps; k < parts * (warp + 1) / kJoinWarps; ++k) a += part[(uint64_t)k * n + i];
  }
  s[warp][lane] = a;
  __syncthreads();
  if (warp || i >= n) return;
  for (int k = 1; k < kJoinWarps; ++k) a += s[k][lane];
  dw[i] = a;
}

// f(padded number of classes) as a constant.
template <typename F>
void with_classes(int n, F&& f) {
  using std::integral_constant;
  if (n <= 4) f(integral_constant<int, 4>{});
  else if (n <= 8) f(integral_constant<int, 8>{});
  else if (n <= 12) f(integral_constant<int, 12>{});
  else if (n <= 16) f(integral_constant<int, 16>{});
  else if (n <= 24) f(integral_constant<int, 24>{});
  else f(integral_constant<int, 32>{});
}

constexpr uint64_t kFewClasses = 32;
constexpr uint64_t kFewWeights = 2048;       // padded classes x padded width
constexpr uint64_t kPartBytes = 16ull << 20; // of the CTAs' sums of dw
// CTAs: one a tile, or as many as leave no more than kPartBytes.
uint64_t few_ctas(uint64_t n_rows, uint64_t n_classes, uint32_t width, int sms) {
  const uint64_t most = std::max<uint64_t>(2 * sms, std::min<uint64_t>(16 * sms, kPartBytes / (4 * n_classes * width)));
  return std::min((n_rows + kFewThreads - 1) / kFewThreads, most);
}

}  // namespace

// f32 alone: bf16 products take one pass of the tensor cores, and 131,072 x
// 64 rows with 16 classes take them 75 us backward, this 72. In f32 that is 72
// us against 157; with 32 classes of 128 columns it is 273 against 212.
bool few_applies(int32_t dtype, uint32_t width, uint64_t n_classes) {
  if (dtype != HB_F32 || n_classes > kFewClasses) return false;
  uint64_t weights = 0;
  with_classes((int)n_classes, [&](auto c) { weights = (uint64_t)decltype(c)::value * pieces_of(width) * kPiece; });
  return weights <= kFewWeights;
}

uint64_t few_bytes(uint64_t n_rows, uint32_t width, uint64_t n_classes, int sms) {
  const uint64_t ctas = few_ctas(n_rows, n_classes, width, sms);
  return ctas > 1 ? 4 * ctas * n_classes * width : 0;
}

void few_forward(const XentCall& c, float* loss, float* lse, int device, int sms, cudaStream_t s) {
  const FewParams p{(const float*)c.x, (const float*)c.w, c.labels, c.x_stride, c.w_stride, c.n_rows, c.width, (int)c.n_classes, c.label_type,
                    loss, lse};
  const unsigned ctas = (unsigned)few_ctas(c.n_rows, c.n_classes, c.width, sms);
  with_classes(p.n_classes, [&](auto n) {
    constexpr int kClasses = decltype(n)::value;
    const uint32_t bytes = Few<kClasses>::forward_bytes(c.width);
    allow_shared<k_few_forward<kClasses>>(device, bytes);
    k_few_forward<kClasses><<<ctas, kFewThreads, bytes, s>>>(p);
  });
}

void few_backward(const XentCall& c, const float* dloss, uint64_t dloss_stride, const float* lse, void* dx, void* dw, void* workspace,
                  int device, int sms, cudaStream_t s) {
  const FewParams p{(const float*)c.x, (const float*)c.w, c.labels, c.x_stride, c.w_stride, c.n_rows, c.width, (int)c.n_classes, c.label_type,
                    nullptr, const_cast<float*>(lse), dloss, dloss_stride, (float*)dx, (float*)dw, (float*)workspace};
  const unsigned ctas = (unsigned)few_ctas(c.n_rows, c.n_classes, c.width, sms);
  with_classes(p.n_classes, [&](auto n) {
    constexpr int kClasses = decltype(n)::value;
    const uint32_t bytes = Few<kClasses>::backward_bytes(c.width);
    allow_shared<k_few_backward<kClasses>>(device, bytes);
    k_few_backward<kClasses><<<ctas, kFewThreads, bytes, s>>>(p);
  });
  const uint32_t all = (uint32_t)(c.n_classes * c.width);
  if (ctas > 1) k_few_join<<<(all + 31) / 32, 32 * kJoinWarps, 0, s>>>(p.part, (int)ctas, all, p.dw);
}

}  // namespace head
}  // namespace hb
