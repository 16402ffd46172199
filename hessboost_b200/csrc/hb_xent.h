// The linear softmax cross entropy's tensor-core products (hb_xent_mma.cu)
// as its entry points (hb_xent.cu) launch them.
#pragma once

#include <cuda.h>

#include "hb_head.h"

namespace hb {
namespace head {

enum MmaKind { kJobStats = 0, kJobGrad = 1, kJobDx = 2, kJobDw = 3 };
enum MmaOutType { kOutAcc = 0, kOutF32 = 1, kOutBf16 = 2 };

// Where a dx or dw tile goes: f32 accumulators [splits][split_rows]
// [acc_stride] (added to what an earlier launch left, or set), or the result
// itself, rows of the layer's width (vec: 16-byte stores will do).
struct MmaOut {
  int type, add, vec;
  int split_rows, acc_stride;
  float* acc;
  void* to;
};

// Pieces (bf16) of G. One, rounded as dx and dw are, would not do for bf16
// layers either: a row of G sums to 0 over the classes, so what their weights
// share cancels in dx, but the roundings of G times it do not. Weights of 8
// with a spread of 0.25 then leave 6% of dx; with two pieces it is 2^-8 of
// that, and bf16 weights have no finer spread. Both products are done twice
// for it: 8,192 x 1,024 rows with 50,021 classes take 4.5 ms pass after pass,
// 3.0 with one.
constexpr int kGradPlanesBf16 = 2, kGradPlanesF32 = 3;
constexpr int kMmaDepth = 2;  // blocks of 64 of k in a stage
// Stages of z's k that are summed in the tensor cores, and whether there are more.
constexpr int kXentChunkF32 = 4, kXentChunkBf16 = 16;
constexpr bool z_chunked(int planes, uint32_t width) {
  return (width + 64 * kMmaDepth - 1) / (64 * kMmaDepth) > (planes > 1 ? kXentChunkF32 : kXentChunkBf16);
}

// m_tiles x n_tiles tiles of (128 x CTAs) x n_size (the last ones n_last), k (k_total of it) in
// k_blocks stages shared among `splits` tiles each; m_fast: consecutive tiles go down the rows.
// The job's rows are [row0, row0 + n_rows) of the call's, its classes
// [class0, class0 + n_classes) of the layer's.
struct MmaJob {
  int kind, m_tiles, n_tiles, n_size, n_last, k_total, k_blocks, splits, m_fast;
  int row0, n_rows, class0, n_classes;
  MmaOut out;
};

constexpr int kMaxJobs = 3;
constexpr int kMaxWorkers = 160;

struct MmaParams {
  // the operands (bf16), with the boxes of their two uses: k along memory,
  // and their own rows along memory
  CUtensorMap x_k, x_mn, w_k, w_mn, g_k, g_mn;
  CUtensorMap g_out;           // what grad writes (dx and dw read an earlier launch's)
  MmaJob jobs[kMaxJobs];
  int n_jobs;
  int planes;                  // of x and w 1: bf16; 3: f32 in three pieces
  int width;
  const void* labels;          // of the call's rows, as the next three
  int label_type;
  int64_t all_classes;
  const float* dloss;
  uint64_t dloss_stride;
  const float* lse;
  float2* part;                // stats: [n_tiles][part_stride]
  uint64_t part_stride;
  float* at_label;             // stats: of the job's rows
  // worker u (a CTA, or a pair) takes tiles [first[j][u], first[j][u + 1]) of job j
  int first[kMaxJobs][kMaxWorkers + 1];

  // The row's label, -1 where it has none.
  __device__ __forceinline__ int64_t label(int64_t row) const {
    const int64_t v = label_type == HB_I32 ? (int64_t)((const int32_t*)labels)[row] : ((const int64_t*)labels)[row];
    return v >= 0 && v < all_classes ? v : -1;
  }
};

// A map of bf16 [planes][rows][64 * blocks] as [planes][blocks][rows][64],
// with boxes of box_blocks x box_rows x 64; strides in elements, multiples
// of 8, the address 16-byte aligned.
bool mma_map(CUtensorMap* map, const void* p, uint64_t blocks, uint64_t rows, uint64_t planes, uint64_t row_stride,
             uint64_t plane_stride, int box_rows, int box_blocks);
// Runs the jobs by single CTAs or (pair) by pairs of them; shares the tiles out.
hb_status mma_launch(MmaParams& p, bool pair, int sms, cudaStream_t s);

// ---- few classes (hb_xent_few.cu) -------------------------------------------

// x, w and the labels of a call.
struct XentCall {
  const void *x, *w, *labels;
  uint64_t x_stride, w_stride, n_rows, n_classes;
  uint32_t width;
  int32_t label_type;
};

// Whether the layer is one for these (a rule on its sizes).
bool few_applies(int32_t dtype, uint32_t width, uint64_t n_classes);
// Workspace of the backward call.
uint64_t few_bytes(uint64_t n_rows, uint32_t width, uint64_t n_classes, int sms);
void few_forward(const XentCall& c, float* loss, float* lse, int sms, cudaStream_t s);
void few_backward(const XentCall& c, const float* dloss, uint64_t dloss_stride, const float* lse, void* dx, void* dw, void* workspace,
                  int sms, cudaStream_t s);

}  // namespace head
}  // namespace hb
