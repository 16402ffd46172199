// The matrix products of the linear softmax cross entropy on the 5th
// generation tensor cores (tcgen05, bf16 operands, f32 accumulators):
//
//   stats  z = x w^T, each row's (max, sum of exp(z - max)) over a tile's classes
//   grad   z again, G = dloss (exp(z - lse) - [class = label]) of a piece of the classes
//   dx     G w      (k: the piece's classes)
//   dw     G^T x    (k: the rows)
//
// One persistent kernel runs a list of such jobs: tile t of the list goes to
// CTA t mod grid. A CTA's warp 0 feeds 64-deep steps of both operands
// through a ring of shared-memory stages by TMA, warp 1 issues the MMAs of a
// 128 x n tile (n <= 256) into one of two TMEM accumulators, and warps 4 to 7
// work the other one off. An operand tile is a stack of 64 x 64 blocks
// whether k or its rows run along memory (tile_desc), so G is written once,
// row by row, and read as it is by dx (k along memory) and by dw (its
// classes along memory), and x and w are read as they lie as well.
//
// f32 operands are three bf16 pieces (v = p0 + p1 + p2, each the rounding of
// what the ones before leave), and a product is the six products of pieces
// whose orders add up to at most 2: what is left out is below 2^-24 of the
// operands' product. The smallest are summed first.
#include <algorithm>
#include <cmath>
#include <string>

#include "hb_mma.cuh"
#include "hb_xent.h"

namespace hb {
namespace head {
namespace {

using namespace hb::mma;

constexpr uint32_t kBlock = 8192;  // bytes of a 64 x 64 block
constexpr int kThreads = 256;
// A stage holds 128 rows of A and the CTA's share of up to 256 of B.
template <bool kPair>
struct Shape {
  static constexpr int kCtas = kPair ? 2 : 1;
  static constexpr int kStages = kPair ? 6 : 4;
  static constexpr uint32_t kStageBytes = (kPair ? 4 : 6) * kBlock;
  static constexpr uint32_t kSmemBytes = 1024 + kStages * kStageBytes + 4 * 2 * 4096 + 256;
};
constexpr float kLog2e = 1.4426950408889634f;

// (piece of A, piece of B) of the products, smallest first; the last one
// alone for bf16 operands.
__constant__ int kPairA[6] = {2, 0, 1, 1, 0, 0};
__constant__ int kPairB[6] = {0, 2, 1, 0, 1, 0};

// The mantissa, in [1, 2), of the first row's factor: G is formed in units
// of it and dx and dw multiplied by it again in f32. A factor that is the
// same for every row (a mean) then does not round each element of a bf16 G
// the same way, which would not average out: with random factors the
// gradients are 1.41 of one rounding off, with 1 / n up to 2.4.
__device__ __forceinline__ float unit_of(const MmaParams& p) {
  const uint32_t bits = __float_as_uint(p.dloss[0]);
  const uint32_t e = bits >> 23 & 0xffu;
  return p.planes > 1 || e == 0u || e == 0xffu ? 1.0f : __uint_as_float((bits & 0x7fffffu) | 0x3f800000u);
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
  int m, n, k0, k1, split;
};

__device__ __forceinline__ TileAt tile_at(const MmaJob& job, int t) {
  TileAt a;
  const int plane = job.m_tiles * job.n_tiles;
  a.split = t / plane;
  t -= a.split * plane;
  if (job.m_fast) a.n = t / job.m_tiles, a.m = t - a.n * job.m_tiles;
  else a.m = t / job.n_tiles, a.n = t - a.m * job.n_tiles;
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

template <bool kPair>
__global__ void __launch_bounds__(kThreads, 1) k_xent_mma(const __grid_constant__ MmaParams p) {
  using S = Shape<kPair>;
  constexpr int kStages = S::kStages;
  extern __shared__ unsigned char raw[];
  const uint32_t base = (smem_addr(raw) + 1023u) & ~1023u;
  const uint32_t staging = base + kStages * S::kStageBytes;
  const uint32_t bars = staging + 4 * 2 * 4096;
  // full: copies landed (a pair's in its first CTA); empty: the MMAs have
  // read a stage; acc_full, acc_empty: the same of an accumulator
  const auto full = [&](int s) { return bars + 8u * s; };
  const auto empty = [&](int s) { return bars + 8u * (kStages + s); };
  const auto acc_full = [&](int b) { return bars + 8u * (2 * kStages + b); };
  const auto acc_empty = [&](int b) { return bars + 8u * (2 * kStages + 2 + b); };
  __shared__ uint32_t s_tmem;
  __shared__ volatile uint32_t s_gave_up;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = kPair ? blockIdx.x & 1 : 0, worker = blockIdx.x / S::kCtas;
  if (threadIdx.x == 0) {
    s_gave_up = 0u;
    for (int s = 0; s < kStages; ++s) bar_init(full(s), 1), bar_init(empty(s), 1);
    for (int b = 0; b < 2; ++b) bar_init(acc_full(b), 1), bar_init(acc_empty(b), 4 * S::kCtas);
    bar_init_fence();
    tma_prefetch(&p.x), tma_prefetch(&p.w);
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
      const int share = job.n_size / S::kCtas, nb = (share + 63) / 64;  // this CTA's rows of B, and their blocks
      const CUtensorMap* ma = job.kind == kJobDx || job.kind == kJobDw ? &p.g : &p.x;
      const CUtensorMap* mb = job.kind == kJobDw ? &p.x : &p.w;
      const bool a_mn = job.kind == kJobDw, b_mn = job.kind == kJobDx || job.kind == kJobDw;
      // rows of the operands in their tensors: x starts at the job's first
      // row and w at its first class where those are its rows or its k
      const int a_row = (at.m * S::kCtas + rank) * 128 + (ma == &p.x ? job.row0 : 0);
      const int b_row = at.n * job.n_size + rank * share + (mb == &p.w && !b_mn ? job.class0 : 0);
      const int bk0 = mb == &p.w && b_mn ? job.class0 : mb == &p.x ? job.row0 : 0;
      for (int q = 6 - p.pairs; q < 6; ++q) {
        const int pa = kPairA[q], pb = kPairB[q];
        for (int k = at.k0; k < at.k1; ++k) {
          if (!(ok = bar_wait(empty(r.stage), r.parity ^ 1u, &s_gave_up))) return false;
          const uint32_t dst = base + r.stage * S::kStageBytes;
          const uint32_t bar = kPair ? peer_addr(full(r.stage), 0) : full(r.stage);
          if (rank == 0) bar_expect(full(r.stage), (2 + nb) * kBlock * S::kCtas);
          issued |= 1u << r.stage;
          for (int b = 0; b < 2; ++b) {
            if (a_mn) tma_load<kPair>(dst + b * kBlock, ma, bar, a_row + 64 * b, k * 64, pa);
            else tma_load<kPair>(dst + b * kBlock, ma, bar, k * 64, a_row + 64 * b, pa);
          }
          for (int b = 0; b < nb; ++b) {
            if (b_mn) tma_load<kPair>(dst + (2 + b) * kBlock, mb, bar, b_row + 64 * b, bk0 + k * 64, pb);
            else tma_load<kPair>(dst + (2 + b) * kBlock, mb, bar, k * 64, b_row + 64 * b, pb);
          }
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
      const uint32_t idesc = instr_desc(128 * S::kCtas, job.n_size, a_mn, b_mn), sa = k_step(a_mn), sb = k_step(b_mn);
      const int buf = tile & 1;
      if (!bar_wait<kPair>(acc_empty(buf), ((tile >> 1) & 1) ^ 1, &s_gave_up)) return false;
      fence_after();
      const uint32_t d = tmem + buf * 256;
      bool add = false;
      for (int i = p.pairs * (at.k1 - at.k0); i > 0; --i) {
        if (!bar_wait(full(r.stage), r.parity, &s_gave_up)) return false;
        fence_after();
        const uint32_t dst = base + r.stage * S::kStageBytes;
        const uint64_t da = tile_desc(dst, a_mn), db = tile_desc(dst + 2 * kBlock, b_mn);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          mma_f16<kPair>(d, da + k * sa, db + k * sb, idesc, add);
          add = true;
        }
        mma_commit<kPair>(empty(r.stage));
        r.next();
      }
      mma_commit<kPair>(acc_full(buf));
      ++tile;
      return true;
    });
  } else if (warp >= 4) {
    const int w4 = warp - 4;
    const uint32_t stage = staging + w4 * 8192;
    int tile = 0, stored = 0;
    each_tile(p, worker, [&](const MmaJob& job, const TileAt& at) {
      const int buf = tile & 1;
      const bool ok = bar_wait(acc_full(buf), (tile >> 1) & 1, &s_gave_up);
      __syncwarp();
      fence_after();
      const uint32_t acc = tmem + buf * 256 + ((uint32_t)(w4 * 32) << 16);
      const int row0 = (at.m * S::kCtas + rank) * 128 + w4 * 32, row = row0 + lane;
      const int col0 = at.n * job.n_size;
      if (job.kind == kJobStats || job.kind == kJobGrad) {
        const bool in = row < job.n_rows;
        const int64_t label = in ? p.label((int64_t)job.row0 + row) : -1;
        const int64_t rel = label - job.class0 - col0;
        if (job.kind == kJobStats) {
          float m = -INFINITY, s = 0.0f;
          for (int c = 0; c < job.n_size; c += 32) {
            float v[32];
            tmem_load32(acc + c, v);
            if (!ok) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = NAN;
            }
            const int left = job.n_classes - (col0 + c);
            if (left <= 0) break;
            if (left < 32) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = i < left ? v[i] : -INFINITY;
            }
            if (rel >= c && rel < c + 32) {
              float z = 0.0f;
#pragma unroll
              for (int i = 0; i < 32; ++i) z = rel == c + i ? v[i] : z;
              p.at_label[row] = z;
            }
            float top = m;
#pragma unroll
            for (int i = 0; i < 32; ++i) top = fmaxf(top, v[i]);
            const float ref = top == -INFINITY ? 0.0f : top * kLog2e;
            float add = 0.0f;
#pragma unroll
            for (int i = 0; i < 32; ++i) add += exp2_fast(fmaf(v[i], kLog2e, -ref));
            s = fmaf(s, exp2_fast(fmaf(m, kLog2e, -ref)), add);
            m = top;
          }
          if (in) p.part[(size_t)at.n * p.part_stride + row] = make_float2(m, s);
        } else {
          const float each = label >= 0 ? p.dloss[(size_t)(job.row0 + row) * p.dloss_stride] / unit_of(p) : 0.0f;
          // lse log2(e) as a rounded value and what the rounding left
          const float l = in ? p.lse[job.row0 + row] : 0.0f;
          const float hi = l * kLog2e, lo = fmaf(l, kLog2e, -hi);
          for (int c = 0; c < job.n_size; c += 64) {
            float v[64];
            tmem_load32(acc + c, reinterpret_cast<float(&)[32]>(v[0]));
            tmem_load32(acc + c + 32, reinterpret_cast<float(&)[32]>(v[32]));
#pragma unroll
            for (int i = 0; i < 64; ++i) {
              float g = exp2_fast(fmaf(v[i], kLog2e, -hi) - lo);
              if (rel == c + i) g -= 1.0f;
              v[i] = label < 0 ? 0.0f : ok ? each * g : NAN;
            }
            if (col0 + c >= job.n_classes) break;  // nothing of G there
            for (int q = 0; q < p.planes; ++q) {
              const uint32_t out = stage + (stored & 1) * 4096;
              if (lane == 0) tma_wait_read<1>();
              __syncwarp();
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                uint32_t h[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const __nv_bfloat162 b = __floats2bfloat162_rn(v[8 * i + 2 * j], v[8 * i + 2 * j + 1]);
                  h[j] = *reinterpret_cast<const uint32_t*>(&b);
                  if (p.planes > 1) {
                    v[8 * i + 2 * j] -= __low2float(b);
                    v[8 * i + 2 * j + 1] -= __high2float(b);
                  }
                }
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(out + lane * 128 + ((i ^ (lane & 7)) << 4)), "r"(h[0]),
                             "r"(h[1]), "r"(h[2]), "r"(h[3])
                             : "memory");
              }
              proxy_fence();
              __syncwarp();
              if (lane == 0 && row0 < job.n_rows) {
                tma_store(&p.g_out, out, col0 + c, row0, q);
                tma_commit();
              }
              ++stored;
            }
          }
        }
      } else {
        const int rows = job.kind == kJobDx ? job.n_rows : job.n_classes;
        const MmaOut& o = job.out;
        const float unit = unit_of(p);
        for (int c = 0; c < job.n_size; c += 32) {
          float v[32];
          tmem_load32(acc + c, v);
          if (!ok || at.k0 == at.k1) {  // no step of k fell to this split
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = ok ? 0.0f : NAN;
          }
          const int left = p.width - (col0 + c);
          if (left <= 0) break;
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] *= unit;
          if (row < rows) {
            const int n = left < 32 ? left : 32;
            if (o.type == kOutAcc) {
              // accumulators' rows are padded to whole groups of four
              float4* q = reinterpret_cast<float4*>(o.acc + ((size_t)at.split * o.split_rows + row) * o.acc_stride + col0 + c);
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (4 * i < n) {
                  float4 u = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                  if (o.add) {
                    const float4 b = q[i];
                    u.x += b.x, u.y += b.y, u.z += b.z, u.w += b.w;
                  }
                  q[i] = u;
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
      fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (kPair) bar_arrive_at(peer_addr(acc_empty(buf), 0)); else bar_arrive(acc_empty(buf));
      }
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

bool mma_map(CUtensorMap* map, const void* p, uint64_t cols, uint64_t rows, uint64_t planes, uint64_t row_stride,
             uint64_t plane_stride, int box_rows) {
  const EncodeFn fn = encoder();
  if (!fn) return false;
  const cuuint64_t dims[3] = {cols, rows, planes};
  const cuuint64_t strides[2] = {2 * row_stride, 2 * plane_stride};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, step[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

namespace {

// Shares the jobs' tiles out among the workers in the jobs' order: each
// job's tiles go where the least work is so far (a tile's work: its steps of
// k and about three more), as far as whole tiles allow.
void share_out(MmaParams& p, int workers) {
  long long load[kMaxWorkers] = {};
  for (int j = 0; j < p.n_jobs; ++j) {
    const MmaJob& job = p.jobs[j];
    const long long tiles = (long long)job.m_tiles * job.n_tiles * job.splits;
    const long long cost = (long long)p.pairs * job.k_blocks / job.splits + 3;
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

template <bool kPair>
hb_status launch(const MmaParams& p, int workers, cudaStream_t s) {
  using S = Shape<kPair>;
  static thread_local int ready = -1;
  int device = 0;
  cudaGetDevice(&device);
  if (ready != device) {
    if (cudaFuncSetAttribute(k_xent_mma<kPair>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmemBytes) != cudaSuccess)
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
  const cudaError_t e = cudaLaunchKernelEx(&c, k_xent_mma<kPair>, p);
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
  return pair ? launch<true>(p, workers, s) : launch<false>(p, workers, s);
}

}  // namespace head
}  // namespace hb
