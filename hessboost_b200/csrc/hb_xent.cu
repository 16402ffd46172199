// Softmax cross entropy of a linear layer, without its logits.
//
//   z = x W^T, lse = log(sum over the classes of exp z), loss = lse - z[label]
//   G = dloss (exp(z - lse) - [class = label]), dx = G W, dW = G^T x
//
// A label outside [0, n_classes) is a row without a label: its loss is 0
// and it takes no part in the gradients. The forward pass keeps only lse;
// the backward pass computes the logits again, a piece of the classes (and a
// chunk of the rows) at a time, so that what is held of G stays below a fixed
// number of elements. The products are hb_xent_mma.cu's.
#include <algorithm>
#include <cmath>

#include "hb_xent.h"

namespace hb {
namespace head {
namespace {

// Elements of G's pieces held at a time (160 MiB in bf16): with half as many,
// twice the launches, 8,192 x 1,024 bf16 rows with 50,021 classes take 4.7 ms
// for 4.3 (a burst of passes), 2,048 x 2,048 with 32,000 classes 1.23 for
// 1.30. In f32 as many would take 3% off 4,099 x 257 rows with 12,289 classes
// and double the accumulators of dx and dw.
constexpr int64_t kGradElementsBf16 = 80ll << 20, kGradElementsF32 = 40ll << 20;
constexpr uint64_t kPartBytes = 64ull << 20;   // of the stats' parts held at a time
constexpr int kFinishThreads = 256;

template <typename L>
__device__ __forceinline__ int64_t label_of(const L* labels, uint64_t r, uint64_t n_classes) {
  const int64_t v = (int64_t)labels[r];
  return v >= 0 && v < (int64_t)n_classes ? v : -1;
}

// x in bf16 pieces, out[plane][row][padded], zero past `width`; where labels
// are given, rows without one are zero (whatever they hold, a product with
// their zero row of G is to add nothing).
// A thread makes 8 columns of a row.
template <typename T, typename L, int kPlanes>
__global__ void k_xent_pack(const T* __restrict__ x, uint64_t x_stride, uint64_t n_rows, uint32_t width,
                            uint32_t padded, int vec, const L* __restrict__ labels, uint64_t n_classes,
                            __nv_bfloat16* __restrict__ out) {
  const uint32_t groups = padded / 8;
  const uint64_t total = n_rows * groups;
  for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (uint64_t)gridDim.x * blockDim.x) {
    const uint64_t r = total >> 32 ? i / groups : (uint32_t)i / groups;
    const uint32_t d = (uint32_t)(i - r * groups) * 8;
    float v[8] = {};
    if (d < width && (!labels || label_of(labels, r, n_classes) >= 0)) {
      const T* from = x + r * x_stride + d;
      if (vec && d + 8 <= width) {
        constexpr int kPer = 16 / sizeof(T);
#pragma unroll
        for (int j = 0; j < 8; j += kPer) {
          const Pack<T, kPer> q = *reinterpret_cast<const Pack<T, kPer>*>(from + j);
#pragma unroll
          for (int k = 0; k < kPer; ++k) v[j + k] = to_f32(q.v[k]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (d + j < width) v[j] = to_f32(from[j]);
      }
    }
#pragma unroll
    for (int q = 0; q < kPlanes; ++q) {
      Pack<__nv_bfloat16, 8> b;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        // f32 past bf16's largest value: the first piece is that, not infinity
        const float most = 0x1.fep127f, size = fabsf(v[j]);
        b.v[j] = __float2bfloat16_rn(kPlanes > 1 && size > most && size < INFINITY ? copysignf(most, v[j]) : v[j]);
        if (q + 1 < kPlanes) v[j] -= __bfloat162float(b.v[j]);
      }
      *reinterpret_cast<Pack<__nv_bfloat16, 8>*>(out + (q * n_rows + r) * padded + d) = b;
    }
  }
}

// Joins the tiles' (max, sum) of each row: a CTA's 32 rows, each warp its
// share of the tiles in class order, then the warps in theirs.
constexpr int kJoinWarps = 16;
__device__ __forceinline__ float2 joined(float2 a, float2 b) {
  const float top = fmaxf(a.x, b.x);
  a.y = (a.x == top ? a.y : a.y * expf(a.x - top)) + (b.x == top ? b.y : b.y * expf(b.x - top));
  a.x = top;
  return a;
}
template <typename L>
__global__ void __launch_bounds__(32 * kJoinWarps)
    k_xent_join(const float2* __restrict__ part, int parts, const float* __restrict__ at_label,
                const L* __restrict__ labels, uint64_t n_rows, uint64_t n_classes, float* __restrict__ loss,
                float* __restrict__ lse) {
  __shared__ float2 sh[kJoinWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint64_t r = (uint64_t)blockIdx.x * 32 + lane;
  float2 a = make_float2(-INFINITY, 0.0f);
  if (r < n_rows) {
    const int p0 = parts * warp / kJoinWarps, p1 = parts * (warp + 1) / kJoinWarps;
#pragma unroll 8
    for (int i = p0; i < p1; ++i) a = joined(a, part[(uint64_t)i * n_rows + r]);
  }
  sh[warp][lane] = a;
  __syncthreads();
  if (warp || r >= n_rows) return;
  for (int i = 1; i < kJoinWarps; ++i) a = joined(a, sh[i][lane]);
  // a.y is at least 1, the maximum's own term, and the label's logit at most
  // the maximum: the loss is not below 0
  const float rest = logf(a.y);
  lse[r] = a.x + rest;
  loss[r] = label_of(labels, r, n_classes) >= 0 ? (a.x - at_label[r]) + rest : 0.0f;
}

// out[r][d] = the sum of the splits' accumulators, in their order; a thread
// makes 4 columns of a row.
template <typename T>
__global__ void k_xent_finish(const float* __restrict__ acc, int splits, uint64_t split_rows, uint64_t n_rows,
                              uint32_t width, uint32_t acc_stride, int vec, T* __restrict__ out) {
  const uint32_t groups = acc_stride / 4;
  const uint64_t total = n_rows * groups;
  for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (uint64_t)gridDim.x * blockDim.x) {
    const uint64_t r = total >> 32 ? i / groups : (uint32_t)i / groups;
    const uint32_t d = (uint32_t)(i - r * groups) * 4;
    const float* from = acc + r * acc_stride + d;
    float4 v = *reinterpret_cast<const float4*>(from);
#pragma unroll 4
    for (int s = 1; s < splits; ++s) {
      const float4 u = *reinterpret_cast<const float4*>(from + s * split_rows * acc_stride);
      v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
    }
    T* to = out + r * width + d;
    const T q[4] = {from_f32<T>(v.x), from_f32<T>(v.y), from_f32<T>(v.z), from_f32<T>(v.w)};
    if (vec) {
      *reinterpret_cast<Pack<T, 4>*>(to) = Pack<T, 4>{{q[0], q[1], q[2], q[3]}};
    } else {
      for (int j = 0; j < 4; ++j)
        if (d + j < width) to[j] = q[j];
    }
  }
}

// ---- plans ---------------------------------------------------------------
struct Operand {
  bool packed;
  uint64_t bytes;  // of its packed form
};
struct Sizes {
  uint64_t n_rows, n_classes;
  uint32_t width, padded;
  int planes, g_planes;
};

Sizes sizes_of(int32_t dtype, uint64_t n_rows, uint32_t width, uint64_t n_classes) {
  const bool f32 = dtype == HB_F32;
  return {n_rows, n_classes, width, (uint32_t)round_up(width, 64), f32 ? 3 : 1, f32 ? kGradPlanesF32 : kGradPlanesBf16};
}
// bf16 rows of whole 64-column blocks are read as they lie where the address
// and the row stride are whole 16-byte units, as TMA wants them. Others are
// copied in every call: with 32,000 classes, 1,000 columns take 291 us for the
// 255 of 1,024 forward over 4,096 rows, and 200 for 135 forward and back over 64.
Operand operand_of(const Sizes& z, int32_t dtype, const void* p, uint64_t stride, uint64_t rows, bool always) {
  const bool packed = always || dtype != HB_BF16 || !aligned(p, 16) || stride % 8 || z.width % 64;
  return {packed, packed ? round_up(2ull * z.planes * rows * z.padded, 256) : 0};
}

// Whether pairs of CTAs (256-row tiles) do the work: where rows, classes and
// width fill such tiles, and enough of them for every pair.
bool use_pairs(uint64_t rows, uint64_t classes, uint32_t width, int sms) {
  return rows >= 256 && classes >= 256 && width >= 128 && ((rows + 255) / 256) * ((classes + 255) / 256) >= (uint64_t)sms / 2;
}

int stages_of(uint64_t k) { return (int)((k + 64 * kMmaDepth - 1) / (64 * kMmaDepth)); }
// Columns of a tile: as few whole tiles of at most 256 as there need be, all
// alike (multiples of `unit`), or narrower ones where there are not enough
// tiles for the workers.
int tile_cols(uint64_t cols, uint64_t m_tiles, int workers, int unit, uint64_t most = 256) {
  uint64_t n = (cols + most - 1) / most;
  while (m_tiles * n < (uint64_t)workers && (cols + n) / (n + 1) > 64) ++n;
  const auto size = [&](uint64_t k) { return round_up((cols + k - 1) / k, unit); };
  return (int)size(n);
}
// The most columns of a tile of logits: where k is summed in chunks, as many
// as an epilogue warp can hold the sums of.
uint64_t z_cols(const Sizes& z) { return z_chunked(z.planes, z.width) ? 128 : 256; }

// Columns of the last of the tiles of n columns: 16 a CTA, 32, 64, or all,
// where that is enough (each CTA's share then lies in whole blocks of 64, or
// inside one).
int last_cols(uint64_t cols, int n, bool pair) {
  const int ctas = pair ? 2 : 1, left = (int)((cols - 1) % n + 1);
  for (int share : {16, 32, 64})
    if (share * ctas >= left && share * ctas <= n) return share * ctas;
  return n;
}
// Parts of k: enough tiles for the workers, at least 4 steps of 64 each, and
// none longer than its type's sums may be, since the tensor cores' own sums
// round towards zero: 0.7 U of what is summed so far on average (U = 2^-24) in
// each step of 16. In f32 that is 512: dw of 131,072 to 600,000 rows is then
// 6 to 16 U off (plain f32 sums 3 to 11) where parts of 1,024 made it 15 to 23,
// of 2,600 50 to 99, of 8,100 140 to 500, and dx over 16,918 classes 13 U for
// 17 to 22 (plain 12). (4,099 x 257 rows with 12,289 classes: 850 us, 816 with
// parts of 1,024, 964 of 256.) In bf16 it is 32,768, some 2^-12 of the result.
int k_splits(uint64_t tiles, int k_blocks, int workers, int planes) {
  const int want = tiles >= (uint64_t)workers ? 1 : (int)((workers + tiles - 1) / tiles);
  const int by_tiles = std::max(1, std::min(want, k_blocks * kMmaDepth / 4));
  const int longest = (planes == 1 ? 32768 : 512) / (64 * kMmaDepth);  // in k_blocks
  return std::max(by_tiles, (k_blocks + longest - 1) / longest);
}

struct Forward {
  Operand x, w;
  bool pair;
  int n_size, n_tiles;
  uint64_t chunk, part, at_label, bytes;
};
Forward forward_plan(const Sizes& z, int32_t dtype, const void* x, uint64_t x_stride, const void* w, uint64_t w_stride, int sms) {
  Forward f;
  f.x = operand_of(z, dtype, x, x_stride, z.n_rows, false);
  f.w = operand_of(z, dtype, w, w_stride, z.n_classes, false);
  f.pair = use_pairs(z.n_rows, z.n_classes, z.width, sms);
  const int m = f.pair ? 256 : 128;
  f.n_size = tile_cols(z.n_classes, (z.n_rows + m - 1) / m, f.pair ? sms / 2 : sms, f.pair ? 128 : 64, z_cols(z));
  f.n_tiles = (int)((z.n_classes + f.n_size - 1) / f.n_size);
  f.chunk = std::min<uint64_t>(z.n_rows, std::max<uint64_t>(256, kPartBytes / (8ull * f.n_tiles) / 256 * 256));
  f.part = round_up(8ull * f.n_tiles * f.chunk, 256);
  f.at_label = round_up(4 * f.chunk, 256);
  f.bytes = f.x.bytes + f.w.bytes + f.part + f.at_label;
  return f;
}

struct Backward {
  Operand x, w;
  bool pair;
  uint64_t piece, chunk, pieces, chunks;
  uint64_t g_stride;                      // elements of a row of G
  int grad_n, out_n;                      // tile columns of grad, and of dx and dw
  int dx_splits, dw_splits;
  bool dx_acc, dw_acc;
  uint32_t acc_stride;
  uint64_t dw_rows;                       // rows of a dw accumulator
  uint64_t g_bytes, dx_bytes, dw_bytes, bytes;  // g_bytes of one piece: there are two where there are two pieces
};
Backward backward_plan(const Sizes& z, int32_t dtype, const void* x, uint64_t x_stride, const void* w, uint64_t w_stride, int sms) {
  Backward b;
  b.x = operand_of(z, dtype, x, x_stride, z.n_rows, true);
  b.w = operand_of(z, dtype, w, w_stride, z.n_classes, false);
  const uint64_t most = (uint64_t)(z.planes == 1 ? kGradElementsBf16 : kGradElementsF32) / z.g_planes;
  // `least`: classes of a piece, where there are as many
  const auto chunk_of = [&](uint64_t least) { return std::min(z.n_rows, std::max<uint64_t>(most / std::min(z.n_classes, least) / 256 * 256, 256)); };
  b.chunk = chunk_of(2048);
  // several chunks of rows keep dw's accumulators of all the classes between
  // them, in f32 one for each 512 rows: chunks of about 2,048 (8,192 x 1,024
  // f32 rows with 20,000 classes: 711 MB of workspace for 1,080, 8.6 ms for 8.8)
  if (z.planes > 1 && b.chunk < z.n_rows) b.chunk = chunk_of(most / 2048);
  b.chunks = (z.n_rows + b.chunk - 1) / b.chunk;
  b.chunk = std::min(b.chunk, round_up((z.n_rows + b.chunks - 1) / b.chunks, 256));
  b.piece = std::min(z.n_classes, std::max<uint64_t>(most / b.chunk / 256 * 256, 256));
  b.pieces = (z.n_classes + b.piece - 1) / b.piece;
  b.piece = std::min(b.piece, round_up((z.n_classes + b.pieces - 1) / b.pieces, 256));
  b.pair = use_pairs(b.chunk, b.piece, z.width, sms);
  const int m = b.pair ? 256 : 128, workers = b.pair ? sms / 2 : sms;
  b.g_stride = round_up(b.piece, 64);
  const uint64_t row_tiles = (b.chunk + m - 1) / m, class_tiles = (b.piece + m - 1) / m;
  b.grad_n = tile_cols(b.piece, row_tiles, workers, b.pair ? 128 : 64, z_cols(z));
  b.out_n = tile_cols(z.width, row_tiles + class_tiles, workers, b.pair ? 128 : 64);
  // two tiles of which one would be mostly empty: whole ones and a narrow last
  if (z.width > 256 && z.width % 256 <= 128) b.out_n = 256;
  const uint64_t out_tiles = (z.width + b.out_n - 1) / b.out_n;
  b.dx_splits = k_splits(row_tiles * out_tiles, stages_of(b.piece), workers, z.planes);
  b.dw_splits = k_splits(class_tiles * out_tiles, stages_of(b.chunk), workers, z.planes);
  b.dx_acc = b.dx_splits > 1 || b.pieces > 1;
  b.dw_acc = b.dw_splits > 1 || b.chunks > 1;
  b.acc_stride = (uint32_t)round_up(z.width, 4);
  b.dw_rows = b.chunks > 1 ? z.n_classes : b.piece;
  b.g_bytes = round_up(2ull * z.g_planes * b.chunk * b.g_stride, 256);
  b.dx_bytes = b.dx_acc ? round_up(4ull * b.dx_splits * b.chunk * b.acc_stride, 256) : 0;
  b.dw_bytes = b.dw_acc ? round_up(4ull * b.dw_splits * b.dw_rows * b.acc_stride, 256) : 0;
  b.bytes = b.x.bytes + b.w.bytes + (b.pieces * b.chunks > 1 ? 2 : 1) * b.g_bytes + b.dx_bytes + b.dw_bytes;
  return b;
}

template <typename F>
void with_xent_types(int32_t dtype, int32_t label_type, F&& f) {
  auto g = [&](auto t) { if (label_type == HB_I32) f(t, int32_t{}); else f(t, int64_t{}); };
  if (dtype == HB_F32) g(float{}); else g(__nv_bfloat16{});
}

int grid_for(uint64_t threads, int block, int sms) {
  return (int)std::max<uint64_t>(1, std::min<uint64_t>((threads + block - 1) / block, (uint64_t)sms * 16));
}

// The operand as the products read it, after packing it to `at` where that
// is needed.
struct Lay {
  const void* p;
  uint64_t rows, stride, plane;
  int planes, blocks;
  bool map(CUtensorMap* m, int box_rows, int box_blocks) const {
    return mma_map(m, p, blocks, rows, planes, stride, plane, box_rows, box_blocks);
  }
};
Lay operand(const Operand& o, const Sizes& z, int32_t dtype, const void* p, uint64_t stride, uint64_t rows, const void* labels,
            int32_t label_type, void* at, int sms, cudaStream_t s) {
  if (!o.packed) return {p, rows, stride, stride, 1, (int)(z.width / 64)};
  const uint64_t total = rows * z.padded;
  with_xent_types(dtype, label_type, [&](auto t, auto l) {
    using T = decltype(t);
    using L = decltype(l);
    constexpr int kPlanes = sizeof(T) == 4 ? 3 : 1;
    k_xent_pack<T, L, kPlanes><<<grid_for(total / 8, 256, sms), 256, 0, s>>>((const T*)p, stride, rows, z.width, z.padded,
                                                                   aligned(p, 16) && stride * sizeof(T) % 16 == 0,
                                                                   (const L*)labels, z.n_classes, (__nv_bfloat16*)at);
  });
  return {at, rows, z.padded, total, z.planes, (int)(z.padded / 64)};
}

hb_status check_xent(const void* x, uint64_t x_stride, const void* w, uint64_t w_stride, int32_t dtype, uint64_t n_rows,
                     uint32_t width, uint64_t n_classes) {
  HB_HEAD_REQUIRE(dtype == HB_F32 || dtype == HB_BF16, "x and w are f32 or bf16");
  HB_HEAD_REQUIRE(width >= 1 && width <= (1u << 20), "width must be in [1, 2^20]");
  HB_HEAD_REQUIRE(n_classes >= 1 && n_classes < (1ull << 31) - 512, "n_classes must be in [1, 2^31 - 512)");
  HB_HEAD_REQUIRE(n_rows < (1ull << 31) - 512, "at most 2^31 - 513 rows");
  HB_HEAD_REQUIRE(w && (!n_rows || x), "x or w is NULL");
  HB_HEAD_REQUIRE(x_stride >= width || n_rows <= 1, "x_stride is below width");
  HB_HEAD_REQUIRE(w_stride >= width || n_classes <= 1, "w_stride is below width");
  HB_HEAD_REQUIRE(x_stride < (1ull << 38) && w_stride < (1ull << 38), "a stride is too large");
  HB_HEAD_REQUIRE(aligned(x, size_of(dtype)) && aligned(w, size_of(dtype)), "a buffer is not aligned to its type");
  return HB_OK;
}
hb_status check_labels(const void* labels, int32_t label_type, uint64_t n_rows) {
  HB_HEAD_REQUIRE(label_type == HB_I32 || label_type == HB_I64, "unknown label type");
  HB_HEAD_REQUIRE(labels || !n_rows, "labels is NULL");
  HB_HEAD_REQUIRE(aligned(labels, label_type == HB_I32 ? 4 : 8), "labels is not aligned to its type");
  return HB_OK;
}

}  // namespace
}  // namespace head
}  // namespace hb

using namespace hb::head;

extern "C" {

hb_status hb_linear_xent_forward_workspace(int32_t device, const void* x, uint64_t x_stride, const void* w, uint64_t w_stride,
                                           int32_t dtype, uint64_t n_rows, uint32_t width, uint64_t n_classes,
                                           uint64_t* bytes) {
  begin_call();
  if (hb_status st = check_xent(x, x_stride, w, w_stride, dtype, n_rows, width, n_classes)) return st;
  HB_HEAD_REQUIRE(bytes, "bytes is NULL");
  *bytes = !n_rows || few_applies(dtype, width, n_classes) ? 0 : forward_plan(sizes_of(dtype, n_rows, width, n_classes), dtype, x, x_stride, w, w_stride, sm_count(device)).bytes;
  return HB_OK;
}

hb_status hb_linear_xent_forward(int32_t device, const void* x, uint64_t x_stride, const void* w, uint64_t w_stride,
                                 int32_t dtype, const void* labels, int32_t label_type, uint64_t n_rows,
                                 uint32_t width, uint64_t n_classes, float* loss, float* lse, void* workspace,
                                 uint64_t workspace_bytes, void* stream) {
  begin_call();
  if (hb_status st = check_xent(x, x_stride, w, w_stride, dtype, n_rows, width, n_classes)) return st;
  if (hb_status st = check_labels(labels, label_type, n_rows)) return st;
  if (!n_rows) return HB_OK;
  HB_HEAD_REQUIRE(loss && lse && aligned(loss, 4) && aligned(lse, 4), "loss or lse is NULL or not aligned");
  const Sizes z = sizes_of(dtype, n_rows, width, n_classes);
  const int sms = sm_count(device);
  if (few_applies(dtype, width, n_classes)) {
    DeviceScope dev(device);
    if (!dev.ok()) return fail(HB_REFUSED, "no such device");
    few_forward(XentCall{x, w, labels, x_stride, w_stride, n_rows, n_classes, width, label_type}, loss, lse, sms,
                (cudaStream_t)stream);
    return launched("hb_linear_xent_forward");
  }
  const Forward f = forward_plan(z, dtype, x, x_stride, w, w_stride, sms);
  HB_HEAD_REQUIRE(workspace && aligned(workspace, 256) && workspace_bytes >= f.bytes,
                  "workspace is too small or not 256-byte aligned");
  DeviceScope dev(device);
  if (!dev.ok()) return fail(HB_REFUSED, "no such device");
  cudaStream_t s = (cudaStream_t)stream;
  char* at = (char*)workspace;
  MmaParams p{};
  const Lay lx = operand(f.x, z, dtype, x, x_stride, n_rows, nullptr, label_type, at, sms, s);
  const Lay lw = operand(f.w, z, dtype, w, w_stride, n_classes, nullptr, label_type, at + f.x.bytes, sms, s);
  if (!lx.map(&p.x_k, 128, kMmaDepth) || !lw.map(&p.w_k, f.pair ? f.n_size / 2 : f.n_size, kMmaDepth))
    return fail(HB_DEVICE_FAILED, "tensor map");
  at += f.x.bytes + f.w.bytes;
  p.part = (float2*)at;
  p.at_label = (float*)(at + f.part);
  p.planes = z.planes;
  p.all_classes = (int64_t)n_classes;
  p.width = (int)width;
  p.labels = labels;
  p.label_type = label_type;
  p.n_jobs = 1;
  const int m = f.pair ? 256 : 128;
  for (uint64_t r0 = 0; r0 < n_rows; r0 += f.chunk) {
    const uint64_t rows = std::min(f.chunk, n_rows - r0);
    p.part_stride = rows;
    p.jobs[0] = MmaJob{kJobStats, (int)((rows + m - 1) / m), f.n_tiles, f.n_size, f.n_size, (int)width, stages_of(width), 1, 1,
                       (int)r0, (int)rows, 0, (int)n_classes, {}};
    if (hb_status st = mma_launch(p, f.pair, sms, s)) return st;
    with_xent_types(dtype, label_type, [&](auto, auto l) {
      using L = decltype(l);
      k_xent_join<L><<<(int)((rows + 31) / 32), 32 * kJoinWarps, 0, s>>>(p.part, f.n_tiles, p.at_label, (const L*)labels + r0, rows, n_classes,
                                                           loss + r0, lse + r0);
    });
  }
  return launched("hb_linear_xent_forward");
}

hb_status hb_linear_xent_backward_workspace(int32_t device, const void* x, uint64_t x_stride, const void* w, uint64_t w_stride,
                                            int32_t dtype, uint64_t n_rows, uint32_t width, uint64_t n_classes,
                                            uint64_t* bytes) {
  begin_call();
  if (hb_status st = check_xent(x, x_stride, w, w_stride, dtype, n_rows, width, n_classes)) return st;
  HB_HEAD_REQUIRE(bytes, "bytes is NULL");
  const int sms = sm_count(device);
  *bytes = !n_rows ? 0
           : few_applies(dtype, width, n_classes)
               ? few_bytes(n_rows, width, n_classes, sms)
               : backward_plan(sizes_of(dtype, n_rows, width, n_classes), dtype, x, x_stride, w, w_stride, sms).bytes;
  return HB_OK;
}

hb_status hb_linear_xent_backward(int32_t device, const float* dloss, uint64_t dloss_stride, const void* x,
                                  uint64_t x_stride, const void* w, uint64_t w_stride, int32_t dtype,
                                  const void* labels, int32_t label_type, const float* lse, uint64_t n_rows,
                                  uint32_t width, uint64_t n_classes, void* dx, void* dw, void* workspace,
                                  uint64_t workspace_bytes, void* stream) {
  begin_call();
  if (hb_status st = check_xent(x, x_stride, w, w_stride, dtype, n_rows, width, n_classes)) return st;
  if (hb_status st = check_labels(labels, label_type, n_rows)) return st;
  HB_HEAD_REQUIRE(dw && (!n_rows || (dloss && lse && dx)), "dloss, lse, dx or dw is NULL");
  HB_HEAD_REQUIRE(aligned(dloss, 4) && aligned(lse, 4) && aligned(dx, size_of(dtype)) && aligned(dw, size_of(dtype)),
                  "a buffer is not aligned to its type");
  const Sizes z = sizes_of(dtype, n_rows, width, n_classes);
  const int sms = sm_count(device);
  if (n_rows && few_applies(dtype, width, n_classes)) {
    const uint64_t bytes = few_bytes(n_rows, width, n_classes, sms);
    HB_HEAD_REQUIRE(!bytes || (workspace && aligned(workspace, 256) && workspace_bytes >= bytes),
                    "workspace is too small or not 256-byte aligned");
    DeviceScope dev(device);
    if (!dev.ok()) return fail(HB_REFUSED, "no such device");
    few_backward(XentCall{x, w, labels, x_stride, w_stride, n_rows, n_classes, width, label_type}, dloss, dloss_stride, lse, dx, dw,
                 workspace, sms, (cudaStream_t)stream);
    return launched("hb_linear_xent_backward");
  }
  Backward b{};
  if (n_rows) {
    b = backward_plan(z, dtype, x, x_stride, w, w_stride, sms);
    HB_HEAD_REQUIRE(workspace && aligned(workspace, 256) && workspace_bytes >= b.bytes,
                    "workspace is too small or not 256-byte aligned");
  }
  DeviceScope dev(device);
  if (!dev.ok()) return fail(HB_REFUSED, "no such device");
  cudaStream_t s = (cudaStream_t)stream;
  if (!n_rows) {
    if (cudaMemsetAsync(dw, 0, n_classes * width * size_of(dtype), s) != cudaSuccess) return launched("hb_linear_xent_backward");
    return HB_OK;
  }
  char* at = (char*)workspace;
  MmaParams p{};
  const Lay lx = operand(b.x, z, dtype, x, x_stride, n_rows, labels, label_type, at, sms, s);
  const Lay lw = operand(b.w, z, dtype, w, w_stride, n_classes, nullptr, label_type, at + b.x.bytes, sms, s);
  const int ctas = b.pair ? 2 : 1, k_rows = 64 * kMmaDepth, out_blocks = b.out_n / ctas / 64;
  if (!lx.map(&p.x_k, 128, kMmaDepth) || !lw.map(&p.w_k, b.grad_n / ctas, kMmaDepth) || !lx.map(&p.x_mn, k_rows, out_blocks) ||
      !lw.map(&p.w_mn, k_rows, out_blocks))
    return fail(HB_DEVICE_FAILED, "tensor map");
  at += b.x.bytes + b.w.bytes;
  const uint64_t steps = b.chunks * b.pieces;
  char* const g[2] = {at, steps > 1 ? at + b.g_bytes : at};
  at = g[1] + b.g_bytes;
  float* dx_acc = (float*)at;
  float* dw_acc = (float*)(at + b.dx_bytes);
  p.planes = z.planes;
  p.all_classes = (int64_t)n_classes;
  p.width = (int)width;
  p.labels = labels;
  p.label_type = label_type;
  p.dloss = dloss;
  p.dloss_stride = dloss_stride;
  p.lse = lse;
  const uint64_t e = size_of(dtype);
  const int out_type = dtype == HB_F32 ? kOutF32 : kOutBf16, m = b.pair ? 256 : 128;
  const int out_tiles = (int)((width + b.out_n - 1) / b.out_n), last = last_cols(width, b.out_n, b.pair);
  const auto vec = [&](const void* q) { return (int)(aligned(q, 16) && width * e % 16 == 0 && b.out_n * e % 16 == 0); };
  // dx or dw of `rows` rows from `splits` accumulators
  const auto finish = [&](const float* acc, int splits, uint64_t split_rows, uint64_t rows, void* to) {
    const int grid = grid_for(rows * (b.acc_stride / 4), kFinishThreads, sms), wide = aligned(to, 4 * e) && width % 4 == 0;
    if (dtype == HB_F32)
      k_xent_finish<float><<<grid, kFinishThreads, 0, s>>>(acc, splits, split_rows, rows, width, b.acc_stride, wide, (float*)to);
    else
      k_xent_finish<__nv_bfloat16><<<grid, kFinishThreads, 0, s>>>(acc, splits, split_rows, rows, width, b.acc_stride, wide, (__nv_bfloat16*)to);
  };
  // Step i is piece i mod pieces of chunk i / pieces. A launch takes dw and
  // dx of one step's G and forms the next step's, whose small tiles fill up
  // the workers that the large ones leave uneven.
  for (uint64_t i = 0; i <= steps; ++i) {
    p.n_jobs = 0;
    const auto sizes = [&](MmaJob& job, uint64_t step) {
      const uint64_t r0 = step / b.pieces * b.chunk, v0 = step % b.pieces * b.piece;
      job.row0 = (int)r0, job.n_rows = (int)std::min(b.chunk, n_rows - r0);
      job.class0 = (int)v0, job.n_classes = (int)std::min(b.piece, n_classes - v0);
    };
    const auto g_lay = [&](const MmaJob& job, uint64_t step) {
      return Lay{g[step & 1], (uint64_t)job.n_rows, b.g_stride, b.chunk * b.g_stride, z.g_planes, (job.n_classes + 63) / 64};
    };
    MmaJob done{};
    void *dx_to = nullptr, *dw_to = nullptr;
    float* acc = nullptr;
    const uint64_t c = (i - 1) / b.pieces, q = (i - 1) % b.pieces;  // of the step done, where i > 0
    if (i > 0) {
      sizes(done, i - 1);
      const Lay lg = g_lay(done, i - 1);
      if (!lg.map(&p.g_k, 128, kMmaDepth) || !lg.map(&p.g_mn, k_rows, 2)) return fail(HB_DEVICE_FAILED, "tensor map");
      dx_to = (char*)dx + (uint64_t)done.row0 * width * e;
      dw_to = (char*)dw + (uint64_t)done.class0 * width * e;
      acc = b.chunks > 1 ? dw_acc + (uint64_t)done.class0 * b.acc_stride : dw_acc;
      // a last piece or chunk may have fewer steps of k than splits: the
      // splits without any add 0
      MmaJob& jw = p.jobs[p.n_jobs++] = done;
      jw.n_last = last;
      jw.kind = kJobDw, jw.m_tiles = (done.n_classes + m - 1) / m, jw.n_tiles = out_tiles, jw.n_size = b.out_n;
      jw.k_total = done.n_rows, jw.k_blocks = stages_of(done.n_rows), jw.splits = b.dw_splits;
      jw.out = MmaOut{b.dw_acc ? kOutAcc : out_type, c > 0, vec(dw_to), (int)b.dw_rows, (int)b.acc_stride, acc, dw_to};
      MmaJob& jx = p.jobs[p.n_jobs++] = done;
      jx.n_last = last;
      jx.kind = kJobDx, jx.m_tiles = (done.n_rows + m - 1) / m, jx.n_tiles = out_tiles, jx.n_size = b.out_n;
      jx.k_total = done.n_classes, jx.k_blocks = stages_of(done.n_classes), jx.splits = b.dx_splits;
      jx.out = MmaOut{b.dx_acc ? kOutAcc : out_type, q > 0, vec(dx_to), (int)b.chunk, (int)b.acc_stride, dx_acc, dx_to};
    }
    if (i < steps) {
      MmaJob& jg = p.jobs[p.n_jobs++] = MmaJob{};
      sizes(jg, i);
      if (!g_lay(jg, i).map(&p.g_out, 32, 1)) return fail(HB_DEVICE_FAILED, "tensor map");
      jg.kind = kJobGrad, jg.m_tiles = (jg.n_rows + m - 1) / m, jg.n_tiles = (jg.n_classes + b.grad_n - 1) / b.grad_n;
      jg.n_size = jg.n_last = b.grad_n, jg.k_total = (int)width, jg.k_blocks = stages_of(width), jg.splits = 1, jg.m_fast = 1;
    }
    if (hb_status st = mma_launch(p, b.pair, sms, s)) return st;
    if (i > 0 && b.dw_acc && c + 1 == b.chunks) finish(acc, b.dw_splits, b.dw_rows, done.n_classes, dw_to);
    if (i > 0 && b.dx_acc && q + 1 == b.pieces) finish(dx_acc, b.dx_splits, b.chunk, done.n_rows, dx_to);
  }
  return launched("hb_linear_xent_backward");
}

}  // extern "C"
