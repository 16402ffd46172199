// Linear softmax cross entropy over a few classes in f32: x is read once
// forward and once backward, without the three-piece products
// (hb_xent_mma.cu) that f32 takes there.
//
// A warp keeps the weights in registers, a lane those of columns lane, lane +
// 32, ... and takes a few rows at a time, as many as make 32 logits. Each lane
// forms its columns' share of every logit; the shares are summed over the
// lanes so that lane l ends up with logit l (31 exchanges for the 32), and the
// softmax of a row is a few more between its lanes. Backward, the lanes hand
// their element of G round, and every lane forms dx of its columns and adds to
// its columns' part of dw, also in registers. The warps' parts of dw are
// added in order, then the CTAs'.
//
// Bound by issuing and by the exchanges' latency: of 131,072 x 100 rows with
// 10 classes x's bytes alone would take 8 us forward and 16 us backward; they
// take 39 and 60. With the weights in shared memory and a thread a row, the
// reads of them took 43 and 102 us, the tensor cores' pieces 87 and 250.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "hb_xent.h"

namespace hb {
namespace head {
namespace {

constexpr int kFewThreads = 128;
constexpr int kWarps = kFewThreads / 32;

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

// kClasses (a multiple of 4) classes over kLanes lanes, kRows rows at a time.
template <int kClasses>
struct Few {
  static constexpr int kLanes = kClasses <= 4 ? 4 : kClasses <= 8 ? 8 : kClasses <= 16 ? 16 : 32;
  static constexpr int kRows = 32 / kLanes;
};

__device__ __forceinline__ void fma2(float& a0, float& a1, float b0, float b1, float c) {
  float2 a = make_float2(a0, a1), b = make_float2(b0, b1), cc = make_float2(c, c);
  asm("fma.rn.f32x2 %0, %1, %2, %0;"
      : "+l"(reinterpret_cast<unsigned long long&>(a))
      : "l"(reinterpret_cast<unsigned long long&>(b)), "l"(reinterpret_cast<unsigned long long&>(cc)));
  a0 = a.x, a1 = a.y;
}

// The lane's columns lane + 32 j of the weights.
template <int kClasses, int J>
__device__ __forceinline__ void load_weights(const FewParams& p, float (&w)[J][kClasses]) {
  const uint32_t lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int v = 0; v < kClasses; ++v)
      w[j][v] = lane + 32 * j < p.width && v < p.n_classes ? p.w[v * p.w_stride + lane + 32 * j] : 0.0f;
}

// The lane's columns of the rows row0 + k, zeros where there are none.
template <int kRows, int J>
__device__ __forceinline__ void load_rows(const FewParams& p, uint64_t row0, float (&x)[kRows][J]) {
  const uint32_t lane = threadIdx.x & 31;
  const float* from = p.x + row0 * p.x_stride + lane;
#pragma unroll
  for (int k = 0; k < kRows; ++k)
#pragma unroll
    for (int j = 0; j < J; ++j) x[k][j] = row0 + k < p.n_rows && lane + 32 * j < p.width ? from[k * p.x_stride + 32 * j] : 0.0f;
}

// Logit (row l / kLanes, class l mod kLanes) of the warp's rows, in lane l.
template <int kClasses, int J>
__device__ __forceinline__ float logits(const float (&w)[J][kClasses], const float (&x)[Few<kClasses>::kRows][J]) {
  using F = Few<kClasses>;
  const int lane = threadIdx.x & 31;
  float a[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) a[i] = 0.0f;
#pragma unroll
  for (int k = 0; k < F::kRows; ++k)
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int v = 0; v < kClasses; v += 2) fma2(a[k * F::kLanes + v], a[k * F::kLanes + v + 1], w[j][v], w[j][v + 1], x[k][j]);
  // lane l keeps the half of the values that l's bit names, and gets the
  // other lane's share of it
#pragma unroll
  for (int s = 16; s; s >>= 1)
#pragma unroll
    for (int i = 0; i < s; ++i) {
      const bool up = lane & s;
      const float keep = up ? a[i + s] : a[i], give = up ? a[i] : a[i + s];
      a[i] = keep + __shfl_xor_sync(0xffffffffu, give, s);
    }
  return a[0];
}

template <int kClasses, int J>
__global__ void __launch_bounds__(kFewThreads) k_few_forward(const FewParams p) {
  using F = Few<kClasses>;
  const int lane = threadIdx.x & 31, v = lane % F::kLanes, k = lane / F::kLanes;
  float w[J][kClasses], x[F::kRows][J], next[F::kRows][J];
  load_weights(p, w);
  const uint64_t step = (uint64_t)gridDim.x * kWarps * F::kRows;
  uint64_t row0 = ((uint64_t)blockIdx.x * kWarps + (threadIdx.x >> 5)) * F::kRows;
  load_rows(p, row0, next);
  for (; row0 < p.n_rows; row0 += step) {
#pragma unroll
    for (int i = 0; i < F::kRows; ++i)
#pragma unroll
      for (int j = 0; j < J; ++j) x[i][j] = next[i][j];
    const uint64_t r = row0 + k;
    const bool in = r < p.n_rows;
    const int label = in ? p.label(r) : -1;
    load_rows(p, row0 + step, next);
    const float z = logits(w, x);
    const bool there = v < p.n_classes;
    float top = there ? z : -INFINITY;
#pragma unroll
    for (int s = F::kLanes / 2; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    const float from = top == -INFINITY ? 0.0f : top;
    float sum = there ? expf(z - from) : 0.0f;
#pragma unroll
    for (int s = F::kLanes / 2; s; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    const float at = __shfl_sync(0xffffffffu, z, k * F::kLanes + max(label, 0));
    if (v == 0 && in) {
      const float rest = logf(sum);
      p.lse[r] = from + rest;
      p.loss[r] = label >= 0 ? (from - at) + rest : 0.0f;  // lse's rounding, of the logits' size, plays no part
    }
  }
}

template <int kClasses, int J>
__global__ void __launch_bounds__(kFewThreads) k_few_backward(const FewParams p) {
  using F = Few<kClasses>;
  extern __shared__ float s_dw[];  // [warp][class][32 J]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, v = lane % F::kLanes, k = lane / F::kLanes;
  float w[J][kClasses], dw[J][kClasses], x[F::kRows][J], next[F::kRows][J];
  load_weights(p, w);
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int c = 0; c < kClasses; ++c) dw[j][c] = 0.0f;
  const uint64_t step = (uint64_t)gridDim.x * kWarps * F::kRows;
  uint64_t row0 = ((uint64_t)blockIdx.x * kWarps + warp) * F::kRows;
  load_rows(p, row0, next);
  for (; row0 < p.n_rows; row0 += step) {
#pragma unroll
    for (int i = 0; i < F::kRows; ++i)
#pragma unroll
      for (int j = 0; j < J; ++j) x[i][j] = next[i][j];
    const uint64_t r = row0 + k;
    const int label = r < p.n_rows ? p.label(r) : -1;
    const float each = label >= 0 ? p.dloss[r * p.dloss_stride] : 0.0f, lse = label >= 0 ? p.lse[r] : 0.0f;
    load_rows(p, row0 + step, next);
    const float z = logits(w, x);
    const float mine = label >= 0 && v < p.n_classes ? each * (expf(z - lse) - (v == label ? 1.0f : 0.0f)) : 0.0f;
#pragma unroll
    for (int i = 0; i < F::kRows; ++i) {
      // a row without a label adds nothing to dw, whatever it holds
      const bool labelled = __shfl_sync(0xffffffffu, label, i * F::kLanes) >= 0;
      float g[kClasses];
#pragma unroll
      for (int c = 0; c < kClasses; ++c) g[c] = __shfl_sync(0xffffffffu, mine, i * F::kLanes + c);
      float* out = p.dx + (row0 + i) * p.width + lane;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const float a = labelled ? x[i][j] : 0.0f;
        float d = 0.0f, e = 0.0f;
#pragma unroll
        for (int c = 0; c < kClasses; c += 2) {
          fma2(dw[j][c], dw[j][c + 1], g[c], g[c + 1], a);
          d = fmaf(g[c], w[j][c], d), e = fmaf(g[c + 1], w[j][c + 1], e);
        }
        if (row0 + i < p.n_rows && lane + 32 * j < p.width) out[32 * j] = d + e;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int c = 0; c < kClasses; ++c) s_dw[(warp * kClasses + c) * (32 * J) + 32 * j + lane] = dw[j][c];
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < (uint32_t)p.n_classes * (32 * J); i += kFewThreads) {
    const uint32_t c = i / (32 * J), d = i % (32 * J);
    if (d >= p.width) continue;
    float t = s_dw[i];
#pragma unroll
    for (int q = 1; q < kWarps; ++q) t += s_dw[q * kClasses * (32 * J) + i];
    if (gridDim.x == 1) p.dw[c * p.width + d] = t;
    else p.part[((uint64_t)blockIdx.x * p.n_classes + c) * p.width + d] = t;
  }
}

// dw from the CTAs' sums: 32 elements a CTA, its warps each a share of the
// sums in order, then the warps in order.
constexpr int kJoinWarps = 16;
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

// f(padded classes, columns a lane) as constants, where both fit a lane's
// registers (64 weights); whether they do.
template <typename F>
bool with_few(uint64_t n_classes, uint32_t width, F&& f) {
  using std::integral_constant;
  const auto columns = [&](auto c) {
    constexpr int kMost = 64 / decltype(c)::value;
    if (width <= 32) return f(c, integral_constant<int, 1>{}), true;
    if (width <= 64) return f(c, integral_constant<int, 2>{}), true;
    if constexpr (kMost >= 4)
      if (width <= 128) return f(c, integral_constant<int, 4>{}), true;
    if constexpr (kMost >= 8)
      if (width <= 256) return f(c, integral_constant<int, 8>{}), true;
    return false;
  };
  if (n_classes <= 4) return columns(integral_constant<int, 4>{});
  if (n_classes <= 8) return columns(integral_constant<int, 8>{});
  if (n_classes <= 12) return columns(integral_constant<int, 12>{});
  if (n_classes <= 16) return columns(integral_constant<int, 16>{});
  if (n_classes <= 24) return columns(integral_constant<int, 24>{});
  if (n_classes <= 32) return columns(integral_constant<int, 32>{});
  return false;
}

// CTAs: at most as many as are there at once, about, by their registers.
uint64_t few_ctas(uint64_t n_rows, uint64_t n_classes, uint32_t width, int sms, bool backward) {
  uint64_t n = 0;
  with_few(n_classes, width, [&](auto c, auto j) {
    constexpr int kHeld = decltype(c)::value * decltype(j)::value;
    const uint64_t rows = kWarps * Few<decltype(c)::value>::kRows;
    const int regs = 60 + (backward ? 9 * kHeld / 4 : kHeld), fit = std::max(2, 512 / regs);
    n = std::min<uint64_t>((n_rows + rows - 1) / rows, (uint64_t)fit * sms);
  });
  return n;
}

}  // namespace

// f32 alone: bf16 products take one pass of the tensor cores.
bool few_applies(int32_t dtype, uint32_t width, uint64_t n_classes) {
  return dtype == HB_F32 && with_few(n_classes, width, [](auto, auto) {});
}

uint64_t few_bytes(uint64_t n_rows, uint32_t width, uint64_t n_classes, int sms) {
  const uint64_t ctas = few_ctas(n_rows, n_classes, width, sms, true);
  return ctas > 1 ? 4 * ctas * n_classes * width : 0;
}

void few_forward(const XentCall& c, float* loss, float* lse, int sms, cudaStream_t s) {
  const FewParams p{(const float*)c.x, (const float*)c.w, c.labels, c.x_stride, c.w_stride, c.n_rows, c.width, (int)c.n_classes, c.label_type,
                    loss, lse};
  const unsigned ctas = (unsigned)few_ctas(c.n_rows, c.n_classes, c.width, sms, false);
  with_few(c.n_classes, c.width, [&](auto n, auto j) {
    k_few_forward<decltype(n)::value, decltype(j)::value><<<ctas, kFewThreads, 0, s>>>(p);
  });
}

void few_backward(const XentCall& c, const float* dloss, uint64_t dloss_stride, const float* lse, void* dx, void* dw, void* workspace,
                  int sms, cudaStream_t s) {
  const FewParams p{(const float*)c.x, (const float*)c.w, c.labels, c.x_stride, c.w_stride, c.n_rows, c.width, (int)c.n_classes, c.label_type,
                    nullptr, const_cast<float*>(lse), dloss, dloss_stride, (float*)dx, (float*)dw, (float*)workspace};
  const unsigned ctas = (unsigned)few_ctas(c.n_rows, c.n_classes, c.width, sms, true);
  with_few(c.n_classes, c.width, [&](auto n, auto j) {
    constexpr int kClasses = decltype(n)::value, J = decltype(j)::value;
    k_few_backward<kClasses, J><<<ctas, kFewThreads, 4 * kWarps * kClasses * 32 * J, s>>>(p);
  });
  const uint32_t all = (uint32_t)(c.n_classes * c.width);
  if (ctas > 1) k_few_join<<<(all + 31) / 32, 32 * kJoinWarps, 0, s>>>(p.part, (int)ctas, all, p.dw);
}

}  // namespace head
}  // namespace hb
