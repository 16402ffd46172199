// The matrix products of the linear softmax cross entropy on the 5th
// generation tensor cores (tcgen05, bf16 operands, f32 accumulators):
//
//   stats  z = x w^T, each row's (max, sum of exp(z - max)) over a tile's classes
//   grad   z again, G = dloss (exp(z - lse) - [class = label]) of a piece of the classes
//   dx     G w      (k: the piece's classes)
//   dw     G^T x    (k: the rows)
//
// One persistent kernel runs a list of such jobs, whose tiles share_out deals to
// the CTAs, or pairs of them, in runs of about equal work. A CTA's warp 0 feeds
// 128-deep stages of both operands through a ring in shared memory by TMA, warp
// 1 issues the MMAs of a 128 x n tile (a pair's is 256 x n, n <= 256) into one
// of two TMEM accumulators, and warps 4 to 11 work the other one off. Operands
// are read as they lie, whether k or their own rows run along memory, so G is
// written once, row by row, and read by dx (k along memory) and by dw (its
// classes along memory).
//
// Every operand is seen as [plane][block of 64 columns][row][64 columns], so
// that one copy brings a CTA's whole share of an operand for a stage: with
// 64 x 64 copies (8 KiB each) the copies themselves were the limit, 990
// TFLOP/s on 8,192 x 1,024 x 50,021 against 1,330 with 128 x 64 ones, both
// before the clocks fall. Bound by the tensor cores and then by power: the
// logits of that size take 599 us cold (1.40 PFLOP/s, tensor pipe 77% busy), a
// piece's dx and dw with the next one's G 317 (82%); the whole call's 5.0
// TFLOP, pass after pass, 4.5 ms (1.1 PFLOP/s at the clocks of the power cap).
// It takes rows of whole blocks: columns past an operand's width are zeros.
//
// f32 operands are three bf16 pieces (v = p0 + p1 + p2, each the rounding of
// what the ones before leave), and a product is the six products of pieces
// whose orders add up to at most 2: what is left out is below 2^-24 of the
// operands' product. The smallest are summed first.
//
// The tensor cores round their sums towards zero, so the logits' k, where it
// is long, is summed in chunks that are added up in f32 arithmetic: f32 in
// chunks of 512 (z over 1,233 columns in one go left 8e-6 of the gradients),
// bf16, whose loss is f32 too, in chunks of 2,048: over 16,384 columns in one
// go the loss was 48 U off (U = 2^-24), now it is 5.3, as over 2,048. An
// epilogue warp then holds 64 columns' sums, so the tiles are at most 128 wide
// and fetch more: 2,048 x 4,096 bf16 rows with 32,000 classes take 805 us
// forward, 515 in one go. (For dx and dw, whose k is cut up anyway, see
// k_splits.)
#include <algorithm>
#include <cmath>
#include <string>

#include "hb_mma.cuh"
#include "hb_xent.h"

namespace hb {
namespace head {
namespace {

using namespace hb::mma;

constexpr int kThreads = 384;  // copies, MMAs, two idle warps, 8 warps of the epilogue
constexpr uint32_t kRow = 128;  // bytes of 64 columns
// A stage holds kDepth blocks of 64 of k: 128 rows of A and the CTA's share
// of up to 256 of B.
template <bool kPair>
struct Shape {
  static constexpr int kCtas = kPair ? 2 : 1;
  static constexpr uint32_t kABytes = 128 * kRow * kMmaDepth;
  static constexpr uint32_t kStageBytes = kABytes + 256 / kCtas * kRow * kMmaDepth;
  static constexpr int kStages = 196608 / kStageBytes;
  static constexpr uint32_t kSmemBytes = 1024 + kStages * kStageBytes + 8 * 4096 + 256;
};
constexpr float kLog2e = 1.4426950408889634f;

// exp(x), and a = exp(a - ref), b = exp(b - ref). The softmax statistics take
// the difference first, in which logits near the maximum are exact, and the
// maximum's own term is 1 whatever its size: a term of 2^(x log2(e) - the
// rounded ref log2(e)) made the loss of certain rows negative and overflowed
// with logits near the type's limits.
__device__ __forceinline__ float exp_fast(float x) { return exp2_fast(x * kLog2e); }
__device__ __forceinline__ void exp_fast2(float& a, float& b, float ref) {
  float2 v = make_float2(a, b), r = make_float2(-ref, -ref), l = make_float2(kLog2e, kLog2e);
  unsigned long long& u = reinterpret_cast<unsigned long long&>(v);
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(u) : "l"(reinterpret_cast<unsigned long long&>(r)));
  asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(u) : "l"(reinterpret_cast<unsigned long long&>(l)));
  a = exp2_fast(v.x), b = exp2_fast(v.y);
}

// (piece of A, piece of B) of the products, smallest first; the last one
// alone for bf16 operands' logits, the last two where A is bf16's G.
__constant__ int kPairA[6] = {2, 0, 1, 0, 1, 0};
__constant__ int kPairB[6] = {0, 2, 1, 1, 0, 0};

// The chunks that a tile's k is summed in.
template <bool kSplit, bool kChunked>
__device__ __forceinline__ int chunks_of(const MmaJob& job, int k0, int k1) {
  constexpr int kChunk = kSplit ? kXentChunkF32 : kXentChunkBf16;
  return kChunked && (job.kind == kJobStats || job.kind == kJobGrad) ? max(1, (k1 - k0 + kChunk - 1) / kChunk) : 1;
}

template <int kStages>
struct Ring {
  int stage = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void next() {
    if (++stage == kStages) stage = 0, parity ^= 1u;
  }
};

struct TileAt {
  int m, n, cols, k0, k1, split;  // k in stages
};

__device__ __forceinline__ TileAt tile_at(const MmaJob& job, int t) {
  TileAt a;
  const int plane = job.m_tiles * job.n_tiles;
  a.split = t / plane;
  t -= a.split * plane;
  if (job.m_fast) a.n = t / job.m_tiles, a.m = t - a.n * job.m_tiles;
  else a.m = t / job.n_tiles, a.n = t - a.m * job.n_tiles;
  a.cols = a.n + 1 == job.n_tiles ? job.n_last : job.n_size;
  a.k0 = (int)((long long)job.k_blocks * a.split / job.splits);
  a.k1 = (int)((long long)job.k_blocks * (a.split + 1) / job.splits);
  return a;
}

// Calls f(job, tile) for each of worker u's tiles until it returns false.
template <typename F>
__device__ __forceinline__ void each_tile(const MmaParams& p, int u, F&& f) {
  for (int j = 0; j < p.n_jobs; ++j)
    for (int t = p.first[j][u], end = p.first[j][u + 1]; t < end; ++t)
      if (!f(p.jobs[j], tile_at(p.jobs[j], t))) return;
}

template <typename T>
__device__ __forceinline__ void store32(T* dst, const float (&v)[32], int n, bool vec) {
  if (vec && n == 32) {
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 32; i += kPer) {
      Pack<T, kPer> q;
#pragma unroll
      for (int j = 0; j < kPer; ++j) q.v[j] = from_f32<T>(v[i + j]);
      *reinterpret_cast<Pack<T, kPer>*>(dst + i) = q;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < n) dst[i] = from_f32<T>(v[i]);
  }
}

// kSplit: f32 operands in three pieces. kChunked: z's k may be longer than a
// chunk, tiles of z are at most 128 columns wide.
template <bool kPair, bool kSplit, bool kChunked>
__global__ void __launch_bounds__(kThreads, 1) k_xent_mma(const __grid_constant__ MmaParams p) {
  using S = Shape<kPair>;
  constexpr int kChunk = kSplit ? kXentChunkF32 : kXentChunkBf16;
  constexpr int kStages = S::kStages, kGradPlanes = kSplit ? kGradPlanesF32 : kGradPlanesBf16;
  extern __shared__ unsigned char raw[];
  const uint32_t base = (smem_addr(raw) + 1023u) & ~1023u;
  const uint32_t staging = base + kStages * S::kStageBytes;
  const uint32_t bars = staging + 8 * 4096;
  // full: copies landed (a pair's in its first CTA); empty: the MMAs have
  // read a stage; acc_full, acc_empty: the same of an accumulator
  const auto full = [&](int s) { return bars + 8u * s; };
  const auto empty = [&](int s) { return bars + 8u * (kStages + s); };
  const auto acc_full = [&](int b) { return bars + 8u * (2 * kStages + b); };
  const auto acc_empty = [&](int b) { return bars + 8u * (2 * kStages + 2 + b); };
  __shared__ uint32_t s_tmem;
  __shared__ volatile uint32_t s_gave_up;
  const auto pairs_of = [&](const MmaJob& job) { return kSplit ? 6 : job.kind == kJobDx || job.kind == kJobDw ? kGradPlanes : 1; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = kPair ? blockIdx.x & 1 : 0, worker = blockIdx.x / S::kCtas;
  if (threadIdx.x == 0) {
    s_gave_up = 0u;
    for (int s = 0; s < kStages; ++s) bar_init(full(s), 1), bar_init(empty(s), 1);
    for (int b = 0; b < 2; ++b) bar_init(acc_full(b), 1), bar_init(acc_empty(b), 8 * S::kCtas);
    bar_init_fence();
    tma_prefetch(&p.x_k), tma_prefetch(&p.w_k);
  }
  if (warp == 2) tmem_alloc<kPair>(smem_addr(&s_tmem), 512);
  fence_before();
  if constexpr (kPair) cluster_sync(); else __syncthreads();
  fence_after();
  const uint32_t tmem = s_tmem;

  if (warp == 0 && lane == 0) {
    Ring<kStages> r;
    uint32_t issued = 0;  // stages with a copy in flight or landed
    bool ok = true;
    each_tile(p, worker, [&](const MmaJob& job, const TileAt& at) {
      const int share = at.cols / S::kCtas;  // this CTA's rows of B
      const bool a_mn = job.kind == kJobDw, b_mn = job.kind == kJobDx || job.kind == kJobDw;
      const CUtensorMap* ma = job.kind == kJobDw ? &p.g_mn : job.kind == kJobDx ? &p.g_k : &p.x_k;
      const CUtensorMap* mb = job.kind == kJobDw ? &p.x_mn : job.kind == kJobDx ? &p.w_mn : &p.w_k;
      // a copy is of the whole tile's share, whatever lies past the last one's
      const uint32_t bytes = S::kABytes + job.n_size / S::kCtas * kRow * kMmaDepth;
      // rows of the operands in their tensors: x starts at the job's first
      // row and w at its first class where those are its rows or its k
      const int a_row = (at.m * S::kCtas + rank) * 128 + (ma == &p.x_k ? job.row0 : 0);
      const int b_row = at.n * job.n_size + rank * share + (mb == &p.w_k ? job.class0 : 0);
      const int bk0 = mb == &p.w_mn ? job.class0 : mb == &p.x_mn ? job.row0 : 0;
      const int chunks = chunks_of<kSplit, kChunked>(job, at.k0, at.k1), pairs = pairs_of(job);
      for (int c = 0; c < chunks * pairs; ++c) {
        const int q = 6 - pairs + c % pairs, pa = kPairA[q], pb = kPairB[q];
        const int k0 = chunks > 1 ? at.k0 + c / pairs * kChunk : at.k0, k1 = chunks > 1 ? min(at.k1, k0 + kChunk) : at.k1;
        for (int k = k0; k < k1; ++k) {
          if (!(ok = bar_wait(empty(r.stage), r.parity ^ 1u, &s_gave_up))) return false;
          const uint32_t dst = base + r.stage * S::kStageBytes;
          const uint32_t bar = kPair ? peer_addr(full(r.stage), 0) : full(r.stage);
          if (rank == 0) bar_expect(full(r.stage), bytes * S::kCtas);
          issued |= 1u << r.stage;
          // coordinates: column in the block, row, block, plane
          if (a_mn) tma_load<kPair>(dst, ma, bar, 0, k * 64 * kMmaDepth, a_row >> 6, pa);
          else tma_load<kPair>(dst, ma, bar, 0, a_row, k * kMmaDepth, pa);
          if (b_mn) tma_load<kPair>(dst + S::kABytes, mb, bar, b_row & 63, bk0 + k * 64 * kMmaDepth, b_row >> 6, pb);
          else tma_load<kPair>(dst + S::kABytes, mb, bar, 0, b_row, k * kMmaDepth, pb);
          r.next();
        }
      }
      return true;
    });
    if (!ok && rank == 0) {
      // let the copies in flight land before the shared memory goes (a pair
      // leaves together, and its first CTA counts both CTAs' copies)
      for (int s = 0; s < kStages; ++s)
        if (issued >> s & 1u) {
          const uint32_t parity = s < r.stage ? r.parity : r.parity ^ 1u;
          for (uint32_t i = 0; i < kWaitTries / 64 && !bar_try(full(s), parity); ++i) {
          }
        }
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    Ring<kStages> r;
    int tile = 0;
    each_tile(p, worker, [&](const MmaJob& job, const TileAt& at) {
      const bool a_mn = job.kind == kJobDw, b_mn = job.kind == kJobDx || job.kind == kJobDw;
      const uint32_t idesc = instr_desc(128 * S::kCtas, at.cols, a_mn, b_mn), sa = k_step(a_mn), sb = k_step(b_mn);
      // k-major: 16 of k are 32 bytes on, the next block of 64 one block of
      // rows on; mn-major: 16 of k are 16 rows of 128 bytes on
      const uint32_t share = job.n_size / S::kCtas;  // k-major tiles are all alike
      const uint32_t block_a = a_mn ? 64 * kRow >> 4 : 128 * kRow >> 4, block_b = b_mn ? 64 * kRow >> 4 : share * kRow >> 4;
      const int chunks = chunks_of<kSplit, kChunked>(job, at.k0, at.k1);
      for (int c = 0; c < chunks; ++c, ++tile) {
        const int buf = tile & 1;
        if (!bar_wait<kPair>(acc_empty(buf), ((tile >> 1) & 1) ^ 1, &s_gave_up)) return false;
        fence_after();
        const uint32_t d = tmem + buf * 256;
        bool add = false;
        const int k0 = chunks > 1 ? at.k0 + c * kChunk : at.k0, k1 = chunks > 1 ? min(at.k1, k0 + kChunk) : at.k1;
        for (int q = pairs_of(job); q > 0; --q)
        for (int k = k0; k < k1; ++k) {
          if (!bar_wait(full(r.stage), r.parity, &s_gave_up)) return false;
          fence_after();
          const uint32_t dst = base + r.stage * S::kStageBytes;
          const uint64_t da = tile_desc(dst, a_mn, 64 * kMmaDepth), db = tile_desc(dst + S::kABytes, b_mn, 64 * kMmaDepth);
          const int left = job.k_total - k * 64 * kMmaDepth;
#pragma unroll
          for (int i = 0; i < 4 * kMmaDepth; ++i) {
            if (16 * i >= left) break;
            mma_f16<kPair>(d, da + (i >> 2) * block_a + (i & 3) * sa, db + (i >> 2) * block_b + (i & 3) * sb, idesc, add);
            add = true;
          }
          mma_commit<kPair>(empty(r.stage));
          r.next();
        }
        mma_commit<kPair>(acc_full(buf));
      }
      return true;
    });
  } else if (warp >= 4) {
    // Two warps for each 32 rows, one for each half of the columns: with one,
    // its waits for TMEM, for exp2 and for its own sums leave the SM idle
    // while a short k's next tile is ready.
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const uint32_t stage = staging + (warp - 4) * 4096;
    int tile = 0;
    each_tile(p, worker, [&](const MmaJob& job, const TileAt& at) {
      const int cut = min(at.cols, (at.cols / 2 + 63) & ~63), c0 = half ? cut : 0, c1 = half ? at.cols : cut;
      const int chunks = chunks_of<kSplit, kChunked>(job, at.k0, at.k1);
      const auto release = [&](int buf) {
        fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (kPair) bar_arrive_at(peer_addr(acc_empty(buf), 0)); else bar_arrive(acc_empty(buf));
        }
      };
      // the chunks but the last, of the warp's 64 columns (tiles are 128 wide at most)
      float sum[kChunked ? 64 : 1] = {};
      bool ok = true;
      if constexpr (kChunked) {
        for (int c = 0; c + 1 < chunks; ++c, ++tile) {
          const int buf = tile & 1;
          ok = bar_wait(acc_full(buf), (tile >> 1) & 1, &s_gave_up) && ok;
          __syncwarp();
          fence_after();
          if (c0 < c1) {
            float v[32];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              tmem_load32(tmem + buf * 256 + ((uint32_t)(quarter * 32) << 16) + c0 + 32 * h, v);
#pragma unroll
              for (int i = 0; i < 32; ++i) sum[32 * h + i] += v[i];
            }
          }
          release(buf);
        }
      }
      const int buf = tile & 1;
      ok = bar_wait(acc_full(buf), (tile >> 1) & 1, &s_gave_up) && ok;
      __syncwarp();
      fence_after();
      const uint32_t acc = tmem + buf * 256 + ((uint32_t)(quarter * 32) << 16);
      // adds the chunks before to the accumulators of columns c and on
      const auto add_chunks = [&](int c, float* v) {
        if constexpr (kChunked) {
          if (chunks > 1) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] += c == c0 ? sum[i] : sum[32 + i];
          }
        }
      };
      const int row0 = (at.m * S::kCtas + rank) * 128 + quarter * 32, row = row0 + lane;
      const int col0 = at.n * job.n_size;
      if (job.kind == kJobStats) {
        const bool in = row < job.n_rows;
        const int64_t rel = (in ? p.label((int64_t)job.row0 + row) : -1) - job.class0 - col0;
        float m = -INFINITY, s = 0.0f;
        for (int c = c0; c < c1; c += 32) {
          const int left = job.n_classes - (col0 + c);
          if (left <= 0) break;
          float v[32];
          tmem_load32(acc + c, v);
          add_chunks(c, v);
          if (left < 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = i < left ? v[i] : -INFINITY;
          }
          if (rel >= c && rel < c + 32) {
            const int hit = (int)rel - c;
            float z = 0.0f;
#pragma unroll
            for (int i = 0; i < 32; ++i) z = hit == i ? v[i] : z;
            p.at_label[row] = z;
          }
          float t[4] = {m, v[0], v[1], v[2]};
#pragma unroll
          for (int i = 3; i < 32; ++i) t[i & 3] = fmaxf(t[i & 3], v[i]);
          const float top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
          const float ref = top == -INFINITY ? 0.0f : top;
          float add[4] = {s * exp_fast(m - ref), 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            exp_fast2(v[i], v[i + 1], ref);
            add[i & 3] += v[i], add[(i & 3) + 1] += v[i + 1];
          }
          s = (add[0] + add[1]) + (add[2] + add[3]);
          m = top;
        }
        // a half that gave up shows in the sum, whichever half it is
        s = ok ? s : NAN;
        // the halves meet in the second warp's staging, which no stats tile uses
        const uint32_t meet = staging + (4 + quarter) * 4096 + buf * 256 + lane * 8;
        if (half) asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(meet), "f"(m), "f"(s) : "memory");
        asm volatile("bar.sync %0, 64;" ::"r"(quarter + 1) : "memory");
        if (!half && in) {
          float2 o;
          asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(o.x), "=f"(o.y) : "r"(meet) : "memory");
          const float top = fmaxf(m, o.x), ref = top == -INFINITY ? 0.0f : top;
          s = s * exp_fast(m - ref) + o.y * exp_fast(o.x - ref);
          p.part[(size_t)at.n * p.part_stride + row] = make_float2(top, s);
        }
      } else if (job.kind == kJobGrad) {
        const bool in = row < job.n_rows;
        const int64_t label = in ? p.label((int64_t)job.row0 + row) : -1;
        const int64_t rel = label - job.class0 - col0;
        // a row without a label: logits and lse 0 (its operand row is 0), factor 0
        const float each = !ok ? NAN : label >= 0 ? p.dloss[(size_t)(job.row0 + row) * p.dloss_stride] : 0.0f;
        // exp(z - lse) = 2^(z log2(e) - lse log2(e)). For f32, whose rounding of
        // that difference (about -13 here and there) would be 3e-7 of the
        // result: lse log2(e) = hi + lo with hi a multiple of 2^-9, whole parts
        // taken out exactly, 2^x of what is left
        const float l = label >= 0 ? p.lse[job.row0 + row] : 0.0f, product = l * kLog2e;
        const float hi = kSplit ? rintf(product * 512.0f) * (1.0f / 512.0f) : product;
        const float lo = kSplit ? fmaf(l, kLog2e, -hi) : 0.0f;
        for (int c = c0; c < c1; c += 64) {
          const int left = job.n_classes - (col0 + c);
          if (left <= 0) break;  // nothing of G there
          float v[64];
          tmem_load32(acc + c, reinterpret_cast<float(&)[32]>(v[0]));
          tmem_load32(acc + c + 32, reinterpret_cast<float(&)[32]>(v[32]));
          add_chunks(c, v);
          add_chunks(c + 32, v + 32);
#pragma unroll
          for (int i = 0; i < 64; ++i) {
            const float g = fmaf(v[i], kLog2e, -hi);
            if (kSplit) {
              const float whole = fminf(fmaxf(rintf(g), -126.0f), 127.0f);
              v[i] = exp2_fast(fmaf(v[i], kLog2e, -(hi + whole)) - lo) * __int_as_float(((int)whole + 127) << 23);
            } else {
              v[i] = exp2_fast(g);
            }
          }
          if (rel >= c && rel < c + 64) {
            const int hit = (int)rel - c;
#pragma unroll
            for (int i = 0; i < 64; ++i) v[i] -= hit == i ? 1.0f : 0.0f;
          }
#pragma unroll
          for (int i = 0; i < 64; ++i) v[i] *= each;
          if (left < 64) {  // zeros up to the block's end: dx reads it whole
#pragma unroll
            for (int i = 0; i < 64; ++i) v[i] = i < left ? v[i] : 0.0f;
          }
#pragma unroll 1
          for (int q = 0; q < kGradPlanes; ++q) {
            if (lane == 0) tma_wait_read<0>();
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              uint32_t h[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const __nv_bfloat162 b = __floats2bfloat162_rn(v[8 * i + 2 * j], v[8 * i + 2 * j + 1]);
                h[j] = *reinterpret_cast<const uint32_t*>(&b);
                v[8 * i + 2 * j] -= __low2float(b);
                v[8 * i + 2 * j + 1] -= __high2float(b);
              }
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 128 + ((i ^ (lane & 7)) << 4)), "r"(h[0]),
                           "r"(h[1]), "r"(h[2]), "r"(h[3])
                           : "memory");
            }
            proxy_fence();
            __syncwarp();
            if (lane == 0 && row0 < job.n_rows) {
              tma_store(&p.g_out, stage, 0, row0, (col0 + c) >> 6, q);
              tma_commit();
            }
          }
        }
      } else {
        const int rows = job.kind == kJobDx ? job.n_rows : job.n_classes;
        const MmaOut& o = job.out;
        // no step of k fell to an empty split: its accumulator is not written
        const bool none = at.k0 == at.k1;
        for (int c = c0; c < c1; c += 32) {
          const int left = p.width - (col0 + c);
          if (left <= 0) break;
          float v[32];
          tmem_load32(acc + c, v);
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = !ok ? NAN : none ? 0.0f : v[i];
          if (row < rows) {
            const int n = left < 32 ? left : 32;
            if (o.type == kOutAcc) {
              // accumulators' rows are padded to whole groups of four; each
              // element is added to once a launch, so the order is the launches'
              float* q = o.acc + ((size_t)at.split * o.split_rows + row) * o.acc_stride + col0 + c;
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (4 * i < n) {
                  if (o.add)
                    asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(q + 4 * i), "f"(v[4 * i]),
                                 "f"(v[4 * i + 1]), "f"(v[4 * i + 2]), "f"(v[4 * i + 3])
                                 : "memory");
                  else
                    *reinterpret_cast<float4*>(q + 4 * i) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                }
            } else if (o.type == kOutF32) {
              store32((float*)o.to + (size_t)row * p.width + col0 + c, v, n, o.vec);
            } else {
              store32((__nv_bfloat16*)o.to + (size_t)row * p.width + col0 + c, v, n, o.vec);
            }
          }
          __syncwarp();
        }
      }
      release(buf);
      ++tile;
      return true;
    });
    if (lane == 0) tma_wait_all();
  }
  __syncwarp();
  fence_before();
  if constexpr (kPair) cluster_sync(); else __syncthreads();
  fence_after();
  if (warp == 2) tmem_free<kPair>(tmem, 512);
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encoder() {
  static const EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return (EncodeFn)f;
  }();
  return fn;
}

}  // namespace

bool mma_map(CUtensorMap* map, const void* p, uint64_t blocks, uint64_t rows, uint64_t planes, uint64_t row_stride,
             uint64_t plane_stride, int box_rows, int box_blocks) {
  const EncodeFn fn = encoder();
  if (!fn) return false;
  const cuuint64_t dims[4] = {64, rows, blocks, planes};
  const cuuint64_t strides[3] = {2 * row_stride, 128, 2 * plane_stride};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, (cuuint32_t)box_blocks, 1}, step[4] = {1, 1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

namespace {

// Shares the jobs' tiles out among the workers in the jobs' order: each
// job's tiles go where the least work is so far (a tile's work: its blocks
// of k, times the products of pieces, and about three more), as far as whole
// tiles allow.
void share_out(MmaParams& p, int workers) {
  long long load[kMaxWorkers] = {};
  for (int j = 0; j < p.n_jobs; ++j) {
    const MmaJob& job = p.jobs[j];
    const long long tiles = (long long)job.m_tiles * job.n_tiles * job.splits;
    const long long pairs = p.planes > 1 ? 6 : job.kind == kJobDx || job.kind == kJobDw ? kGradPlanesBf16 : 1;
    const long long cost = pairs * kMmaDepth * job.k_blocks / job.splits + 3;
    const auto below = [&](long long level) {
      long long n = 0;
      for (int u = 0; u < workers; ++u) n += level > load[u] ? (level - load[u]) / cost : 0;
      return n;
    };
    // the lowest level under which all the tiles fit
    long long lo = 0, hi = cost * (tiles / workers + 2);
    for (int u = 0; u < workers; ++u) hi = load[u] > hi - cost * (tiles / workers + 2) ? load[u] + cost * (tiles / workers + 2) : hi;
    while (lo < hi) {
      const long long m = (lo + hi) / 2;
      if (below(m) >= tiles) hi = m; else lo = m + 1;
    }
    long long spare = below(lo) - tiles;  // tiles that the level has room for beyond ours
    int at = 0;
    for (int u = 0; u < workers; ++u) {
      long long n = lo > load[u] ? (lo - load[u]) / cost : 0;
      if (spare > 0 && n > 0 && load[u] + n * cost == lo) --n, --spare;
      p.first[j][u] = at;
      at += (int)n;
      load[u] += n * cost;
    }
    p.first[j][workers] = at;
  }
}

template <bool kPair, bool kSplit, bool kChunked>
hb_status launch(const MmaParams& p, int workers, cudaStream_t s) {
  using S = Shape<kPair>;
  static thread_local int ready = -1;
  int device = 0;
  cudaGetDevice(&device);
  if (ready != device) {
    if (cudaFuncSetAttribute(k_xent_mma<kPair, kSplit, kChunked>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmemBytes) != cudaSuccess)
      return fail(HB_DEVICE_FAILED, "shared memory of the product kernel");
    ready = device;
  }
  cudaLaunchConfig_t c{};
  c.gridDim = dim3(workers * S::kCtas);
  c.blockDim = dim3(kThreads);
  c.dynamicSmemBytes = S::kSmemBytes;
  c.stream = s;
  cudaLaunchAttribute a[1];
  a[0].id = cudaLaunchAttributeClusterDimension;
  a[0].val.clusterDim = {S::kCtas, 1, 1};
  c.attrs = a;
  c.numAttrs = kPair ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&c, k_xent_mma<kPair, kSplit, kChunked>, p);
  if (e == cudaSuccess) return HB_OK;
  cudaGetLastError();
  return fail(HB_DEVICE_FAILED, std::string("product kernel: ") + cudaGetErrorString(e));
}

}  // namespace

hb_status mma_launch(MmaParams& p, bool pair, int sms, cudaStream_t s) {
  long long tiles = 0;
  for (int j = 0; j < p.n_jobs; ++j) tiles += (long long)p.jobs[j].m_tiles * p.jobs[j].n_tiles * p.jobs[j].splits;
  if (!tiles) return HB_OK;
  const int most = std::min(pair ? sms / 2 : sms, kMaxWorkers);
  const int workers = (int)std::min<long long>(tiles, std::max(most, 1));
  share_out(p, workers);
  if (p.planes > 1) return pair ? launch<true, true, true>(p, workers, s) : launch<false, true, true>(p, workers, s);
  if (z_chunked(p.planes, p.width)) return pair ? launch<true, false, true>(p, workers, s) : launch<false, false, true>(p, workers, s);
  return pair ? launch<true, false, false>(p, workers, s) : launch<false, false, false>(p, workers, s);
}

}  // namespace head
}  // namespace hb
