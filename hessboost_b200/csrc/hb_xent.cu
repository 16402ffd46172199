// Softmax cross entropy of a linear layer, without its logits.
//
//   z = x W^T, lse = log(sum over the classes of exp z), loss = lse - z[label]
//   G = dloss (exp(z - lse) - [class = label]), dx = G W, dW = G^T x
//
// A label outside [0, n_classes) is a row without a label: its loss is 0
// and it takes no part in the gradients. The forward pass keeps only lse;
// the backward pass computes the logits again, a piece of the classes at a
// time.
#include <algorithm>
#include <cmath>

#include "hb_head.h"

namespace hb {
namespace head {
namespace {

constexpr int kTile = 64;    // rows and classes of a CTA's tile of logits
constexpr int kStep = 16;    // columns of a step
constexpr int kSplits = 64;  // parts of the classes in the forward pass

// c[4][4] += A[row0 + 4 ty + i][k] B[col0 + 4 tx + j][k] over k in [0, kn),
// A and B read through element (row, k) functions that give 0 outside.
template <typename FA, typename FB>
__device__ __forceinline__ void tile_product(uint64_t kn, FA a, FB b, float (&c)[4][4], float (*sa)[kTile + 1],
                                             float (*sb)[kTile + 1]) {
  const int t = threadIdx.x, tx = t & 15, ty = t >> 4;
  for (uint64_t k0 = 0; k0 < kn; k0 += kStep) {
    for (int i = t; i < kTile * kStep; i += 256) {
      const int r = i / kStep, k = i % kStep;
      sa[k][r] = k0 + k < kn ? a(r, k0 + k) : 0.0f;
      sb[k][r] = k0 + k < kn ? b(r, k0 + k) : 0.0f;
    }
    __syncthreads();
    for (int k = 0; k < kStep; ++k)
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) c[i][j] = fmaf(sa[k][4 * ty + i], sb[k][4 * tx + j], c[i][j]);
    __syncthreads();
  }
}

template <typename L>
__device__ __forceinline__ int64_t label_of(const L* labels, uint64_t r, uint64_t n_classes) {
  const int64_t v = (int64_t)labels[r];
  return v >= 0 && v < (int64_t)n_classes ? v : -1;
}

// Split blockIdx.y of the classes: each row's maximum, sum of exp(z - max)
// and, where the split holds it, its label's logit.
template <typename T, typename L>
__global__ void __launch_bounds__(256)
    k_xent_parts(const T* __restrict__ x, uint64_t x_stride, const T* __restrict__ w, uint64_t w_stride,
                 const L* __restrict__ labels, uint64_t n_rows, uint32_t width, uint64_t n_classes,
                 float2* __restrict__ part, float* __restrict__ at_label) {
  __shared__ float sa[kStep][kTile + 1], sb[kStep][kTile + 1];
  __shared__ float2 sp[kTile][16];
  const uint64_t row0 = (uint64_t)blockIdx.x * kTile;
  const uint64_t tiles = (n_classes + kTile - 1) / kTile;
  const uint64_t t0 = tiles * blockIdx.y / gridDim.y, t1 = tiles * (blockIdx.y + 1) / gridDim.y;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float m[4], s[4];
  int64_t label[4];
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY, s[i] = 0.0f;
    const uint64_t r = row0 + 4 * ty + i;
    label[i] = r < n_rows ? label_of(labels, r, n_classes) : -1;
  }
  for (uint64_t tl = t0; tl < t1; ++tl) {
    const uint64_t col0 = tl * kTile;
    float c[4][4] = {};
    tile_product(
        width, [&](int r, uint64_t k) { return row0 + r < n_rows ? to_f32(x[(row0 + r) * x_stride + k]) : 0.0f; },
        [&](int r, uint64_t k) { return col0 + r < n_classes ? to_f32(w[(col0 + r) * w_stride + k]) : 0.0f; }, c, sa, sb);
    for (int i = 0; i < 4; ++i)
      for (int j = 0; j < 4; ++j) {
        const uint64_t v = col0 + 4 * tx + j;
        if (v >= n_classes) continue;
        const float z = c[i][j];
        if ((int64_t)v == label[i]) at_label[row0 + 4 * ty + i] = z;
        const float top = fmaxf(m[i], z);
        s[i] = (m[i] == top ? s[i] : s[i] * expf(m[i] - top)) + (z == top ? 1.0f : expf(z - top));
        m[i] = top;
      }
  }
  for (int i = 0; i < 4; ++i) sp[4 * ty + i][tx] = make_float2(m[i], s[i]);
  __syncthreads();
  if (threadIdx.x < kTile && row0 + threadIdx.x < n_rows) {
    float2 a = sp[threadIdx.x][0];
    for (int j = 1; j < 16; ++j) {
      const float2 b = sp[threadIdx.x][j];
      const float top = fmaxf(a.x, b.x);
      a.y = (a.x == top ? a.y : a.y * expf(a.x - top)) + (b.x == top ? b.y : b.y * expf(b.x - top));
      a.x = top;
    }
    part[(uint64_t)blockIdx.y * n_rows + row0 + threadIdx.x] = a;
  }
}

template <typename L>
__global__ void k_xent_join(const float2* __restrict__ part, int splits, const float* __restrict__ at_label,
                            const L* __restrict__ labels, uint64_t n_rows, uint64_t n_classes,
                            float* __restrict__ loss, float* __restrict__ lse) {
  const uint64_t r = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (r >= n_rows) return;
  float2 a = part[r];
  for (int i = 1; i < splits; ++i) {
    const float2 b = part[(uint64_t)i * n_rows + r];
    const float top = fmaxf(a.x, b.x);
    a.y = (a.x == top ? a.y : a.y * expf(a.x - top)) + (b.x == top ? b.y : b.y * expf(b.x - top));
    a.x = top;
  }
  const float l = a.x + logf(a.y);
  lse[r] = l;
  loss[r] = label_of(labels, r, n_classes) >= 0 ? l - at_label[r] : 0.0f;
}

// G of the classes [v0, v0 + vn): g[r][v - v0], f32.
template <typename T, typename L>
__global__ void __launch_bounds__(256)
    k_xent_grad(const T* __restrict__ x, uint64_t x_stride, const T* __restrict__ w, uint64_t w_stride,
                const L* __restrict__ labels, const float* __restrict__ dloss, uint64_t dloss_stride,
                const float* __restrict__ lse, uint64_t n_rows, uint32_t width, uint64_t n_classes, uint64_t v0,
                uint64_t vn, float* __restrict__ g) {
  __shared__ float sa[kStep][kTile + 1], sb[kStep][kTile + 1];
  const uint64_t row0 = (uint64_t)blockIdx.x * kTile, col0 = (uint64_t)blockIdx.y * kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float c[4][4] = {};
  tile_product(
      width, [&](int r, uint64_t k) { return row0 + r < n_rows ? to_f32(x[(row0 + r) * x_stride + k]) : 0.0f; },
      [&](int r, uint64_t k) { return col0 + r < vn ? to_f32(w[(v0 + col0 + r) * w_stride + k]) : 0.0f; }, c, sa, sb);
  for (int i = 0; i < 4; ++i) {
    const uint64_t r = row0 + 4 * ty + i;
    if (r >= n_rows) continue;
    const int64_t label = label_of(labels, r, n_classes);
    const float each = label >= 0 ? dloss[r * dloss_stride] : 0.0f, l = lse[r];
    for (int j = 0; j < 4; ++j) {
      const uint64_t v = col0 + 4 * tx + j;
      if (v < vn) g[r * vn + v] = label < 0 ? 0.0f : each * (expf(c[i][j] - l) - ((int64_t)(v0 + v) == label ? 1.0f : 0.0f));
    }
  }
}

// acc[r][d] (+)= sum over v of g[r][v] W[v0 + v][d]
template <typename T>
__global__ void __launch_bounds__(256)
    k_xent_dx(const float* __restrict__ g, const T* __restrict__ w, uint64_t w_stride, uint64_t n_rows,
              uint32_t width, uint64_t v0, uint64_t vn, float* __restrict__ acc, T* __restrict__ dx, int first, int last) {
  __shared__ float sa[kStep][kTile + 1], sb[kStep][kTile + 1];
  const uint64_t row0 = (uint64_t)blockIdx.x * kTile, col0 = (uint64_t)blockIdx.y * kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float c[4][4] = {};
  tile_product(
      vn, [&](int r, uint64_t k) { return row0 + r < n_rows ? g[(row0 + r) * vn + k] : 0.0f; },
      [&](int r, uint64_t k) { return col0 + r < width ? to_f32(w[(v0 + k) * w_stride + col0 + r]) : 0.0f; }, c, sa, sb);
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const uint64_t r = row0 + 4 * ty + i, d = col0 + 4 * tx + j;
      if (r >= n_rows || d >= width) continue;
      const float v = first ? c[i][j] : acc[r * width + d] + c[i][j];
      if (last) dx[r * width + d] = from_f32<T>(v);
      else acc[r * width + d] = v;
    }
}

// dW[v0 + v][d] = sum over r of g[r][v] x[r][d]
template <typename T>
__global__ void __launch_bounds__(256)
    k_xent_dw(const float* __restrict__ g, const T* __restrict__ x, uint64_t x_stride, uint64_t n_rows,
              uint32_t width, uint64_t v0, uint64_t vn, T* __restrict__ dw) {
  __shared__ float sa[kStep][kTile + 1], sb[kStep][kTile + 1];
  const uint64_t row0 = (uint64_t)blockIdx.x * kTile, col0 = (uint64_t)blockIdx.y * kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float c[4][4] = {};
  tile_product(
      n_rows, [&](int r, uint64_t k) { return row0 + r < vn ? g[k * vn + row0 + r] : 0.0f; },
      [&](int r, uint64_t k) { return col0 + r < width ? to_f32(x[k * x_stride + col0 + r]) : 0.0f; }, c, sa, sb);
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const uint64_t v = row0 + 4 * ty + i, d = col0 + 4 * tx + j;
      if (v < vn && d < width) dw[(v0 + v) * width + d] = from_f32<T>(c[i][j]);
    }
}

// Classes of a piece: G of a piece takes about 64 MiB.
uint64_t piece_of(uint64_t n_rows, uint64_t n_classes) {
  const uint64_t most = (16ull << 20) / std::max<uint64_t>(n_rows, 1) / kTile * kTile;
  return std::min(n_classes, std::min<uint64_t>(65535ull * kTile, std::max<uint64_t>(most, kTile)));
}

hb_status check_xent(const void* x, uint64_t x_stride, const void* w, uint64_t w_stride, int32_t dtype, const void* labels,
                     int32_t label_type, uint64_t n_rows, uint32_t width, uint64_t n_classes) {
  HB_HEAD_REQUIRE(dtype == HB_F32 || dtype == HB_BF16, "x and w are f32 or bf16");
  HB_HEAD_REQUIRE(label_type == HB_I32 || label_type == HB_I64, "unknown label type");
  HB_HEAD_REQUIRE(width >= 1 && width <= (1u << 20), "width must be in [1, 2^20]");
  HB_HEAD_REQUIRE(n_classes >= 1 && n_classes < (1ull << 31), "n_classes must be in [1, 2^31)");
  HB_HEAD_REQUIRE(n_rows < (1ull << 31), "at most 2^31 - 1 rows");
  HB_HEAD_REQUIRE(w && (!n_rows || (x && labels)), "x, w or labels is NULL");
  HB_HEAD_REQUIRE(x_stride >= width || n_rows <= 1, "x_stride is below width");
  HB_HEAD_REQUIRE(w_stride >= width || n_classes <= 1, "w_stride is below width");
  HB_HEAD_REQUIRE(aligned(x, size_of(dtype)) && aligned(w, size_of(dtype)) && aligned(labels, label_type == HB_I32 ? 4 : 8),
                  "a buffer is not aligned to its type");
  return HB_OK;
}

uint64_t forward_bytes(uint64_t n_rows) { return round_up(4 * n_rows, 256) + 8 * kSplits * n_rows; }
uint64_t backward_bytes(uint64_t n_rows, uint32_t width, uint64_t n_classes) {
  return round_up(4 * n_rows * piece_of(n_rows, n_classes), 256) + 4 * n_rows * width;
}

template <typename F>
void with_xent_types(int32_t dtype, int32_t label_type, F&& f) {
  auto g = [&](auto t) { if (label_type == HB_I32) f(t, int32_t{}); else f(t, int64_t{}); };
  if (dtype == HB_F32) g(float{}); else g(__nv_bfloat16{});
}

}  // namespace
}  // namespace head
}  // namespace hb

using namespace hb::head;

extern "C" {

hb_status hb_linear_xent_forward_workspace(uint64_t n_rows, uint32_t width, uint64_t n_classes, int32_t dtype, uint64_t* bytes) {
  begin_call();
  HB_HEAD_REQUIRE(bytes && n_rows < (1ull << 31), "bytes is NULL or too many rows");
  *bytes = forward_bytes(n_rows);
  return HB_OK;
}

hb_status hb_linear_xent_forward(int32_t device, const void* x, uint64_t x_stride, const void* w, uint64_t w_stride,
                                 int32_t dtype, const void* labels, int32_t label_type, uint64_t n_rows,
                                 uint32_t width, uint64_t n_classes, float* loss, float* lse, void* workspace,
                                 uint64_t workspace_bytes, void* stream) {
  begin_call();
  if (hb_status st = check_xent(x, x_stride, w, w_stride, dtype, labels, label_type, n_rows, width, n_classes)) return st;
  if (!n_rows) return HB_OK;
  HB_HEAD_REQUIRE(loss && lse && aligned(loss, 4) && aligned(lse, 4), "loss or lse is NULL or not aligned");
  HB_HEAD_REQUIRE(workspace && aligned(workspace, 256) && workspace_bytes >= forward_bytes(n_rows),
                  "workspace is too small or not 256-byte aligned");
  DeviceScope dev(device);
  if (!dev.ok()) return fail(HB_REFUSED, "no such device");
  cudaStream_t s = (cudaStream_t)stream;
  float* at_label = (float*)workspace;
  float2* part = (float2*)((char*)workspace + round_up(4 * n_rows, 256));
  const int splits = (int)std::min<uint64_t>(kSplits, (n_classes + kTile - 1) / kTile);
  with_xent_types(dtype, label_type, [&](auto t, auto l) {
    using T = decltype(t);
    using L = decltype(l);
    k_xent_parts<T, L><<<dim3((unsigned)((n_rows + kTile - 1) / kTile), splits), 256, 0, s>>>(
        (const T*)x, x_stride, (const T*)w, w_stride, (const L*)labels, n_rows, width, n_classes, part, at_label);
    k_xent_join<L><<<(int)((n_rows + 255) / 256), 256, 0, s>>>(part, splits, at_label, (const L*)labels, n_rows, n_classes, loss, lse);
  });
  return launched("hb_linear_xent_forward");
}

hb_status hb_linear_xent_backward_workspace(uint64_t n_rows, uint32_t width, uint64_t n_classes, int32_t dtype, uint64_t* bytes) {
  begin_call();
  HB_HEAD_REQUIRE(bytes && n_rows < (1ull << 31) && n_classes < (1ull << 31) && width <= (1u << 20), "bytes is NULL or sizes out of range");
  *bytes = backward_bytes(n_rows, width, n_classes);
  return HB_OK;
}

hb_status hb_linear_xent_backward(int32_t device, const float* dloss, uint64_t dloss_stride, const void* x,
                                  uint64_t x_stride, const void* w, uint64_t w_stride, int32_t dtype,
                                  const void* labels, int32_t label_type, const float* lse, uint64_t n_rows,
                                  uint32_t width, uint64_t n_classes, void* dx, void* dw, void* workspace,
                                  uint64_t workspace_bytes, void* stream) {
  begin_call();
  if (hb_status st = check_xent(x, x_stride, w, w_stride, dtype, labels, label_type, n_rows, width, n_classes)) return st;
  HB_HEAD_REQUIRE(dw && (!n_rows || (dloss && lse && dx)), "dloss, lse, dx or dw is NULL");
  HB_HEAD_REQUIRE(aligned(dloss, 4) && aligned(lse, 4) && aligned(dx, size_of(dtype)) && aligned(dw, size_of(dtype)),
                  "a buffer is not aligned to its type");
  HB_HEAD_REQUIRE(!n_rows || (workspace && aligned(workspace, 256) && workspace_bytes >= backward_bytes(n_rows, width, n_classes)),
                  "workspace is too small or not 256-byte aligned");
  DeviceScope dev(device);
  if (!dev.ok()) return fail(HB_REFUSED, "no such device");
  cudaStream_t s = (cudaStream_t)stream;
  if (!n_rows) {
    cudaMemsetAsync(dw, 0, n_classes * width * size_of(dtype), s);
    return launched("hb_linear_xent_backward");
  }
  const uint64_t piece = piece_of(n_rows, n_classes);
  float* g = (float*)workspace;
  float* acc = (float*)((char*)workspace + round_up(4 * n_rows * piece, 256));
  const unsigned row_tiles = (unsigned)((n_rows + kTile - 1) / kTile), d_tiles = (width + kTile - 1) / kTile;
  with_xent_types(dtype, label_type, [&](auto t, auto l) {
    using T = decltype(t);
    using L = decltype(l);
    for (uint64_t v0 = 0; v0 < n_classes; v0 += piece) {
      const uint64_t vn = std::min(piece, n_classes - v0);
      const unsigned v_tiles = (unsigned)((vn + kTile - 1) / kTile);
      k_xent_grad<T, L><<<dim3(row_tiles, v_tiles), 256, 0, s>>>((const T*)x, x_stride, (const T*)w, w_stride, (const L*)labels,
                                                             dloss, dloss_stride, lse, n_rows, width, n_classes, v0, vn, g);
      k_xent_dx<T><<<dim3(row_tiles, d_tiles), 256, 0, s>>>(g, (const T*)w, w_stride, n_rows, width, v0, vn, acc, (T*)dx,
                                                        v0 == 0, v0 + vn == n_classes);
      k_xent_dw<T><<<dim3(v_tiles, d_tiles), 256, 0, s>>>(g, (const T*)x, x_stride, n_rows, width, v0, vn, (T*)dw);
    }
  });
  return launched("hb_linear_xent_backward");
}

}  // extern "C"
