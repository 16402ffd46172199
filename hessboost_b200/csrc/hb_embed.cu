// Embedding of token bags and the table's gradient.
//
//   forward   out[n]    = scale * sum over the cells c of row n of table[t_c]
//   backward  dtable[v] = scale * sum over the cells c with t_c = v of grad[row(c)]
//
// A token id outside [0, n_tokens) is an absent cell (a missing value of the
// binned matrix): it contributes nothing, and a row of nothing but absent
// cells is 0. Sums are f32 in a fixed order (cell order), rounded once to
// the table's type, so results do not change from run to run.
//
// The gradient sorts the cells by token (a stable radix sort, so that each
// token's cells stay in order) and sums each token's run of rows.
#include <algorithm>

#include "hb_head.h"

namespace hb {
namespace head {
namespace {

template <typename Tok>
__device__ __forceinline__ uint32_t token_of(const Tok* tokens, uint64_t c, uint64_t n_tokens) {
  // negative ids and ids past the table become n_tokens: absent
  const uint64_t t = (uint64_t)(int64_t)tokens[c];
  return (uint32_t)(t < n_tokens ? t : n_tokens);
}

// One thread per (row, column).
template <typename T, typename Tok>
__global__ void k_embed_forward(const Tok* __restrict__ tokens, const int64_t* __restrict__ row_ptr,
                                uint64_t n_rows, uint64_t n_cells, uint64_t per_row,
                                const T* __restrict__ table, uint64_t n_tokens, uint32_t width,
                                uint64_t table_stride, float scale, T* __restrict__ out) {
  const uint64_t total = n_rows * width;
  for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (uint64_t)gridDim.x * blockDim.x) {
    const uint64_t r = i / width;
    const uint32_t d = (uint32_t)(i - r * width);
    int64_t c0 = (int64_t)(r * per_row), c1 = c0 + (int64_t)per_row;
    if (row_ptr) {
      c0 = max((int64_t)0, row_ptr[r]);
      c1 = min((int64_t)n_cells, row_ptr[r + 1]);
    }
    float acc = 0.0f;
    for (int64_t c = c0; c < c1; ++c) {
      const uint32_t t = token_of(tokens, (uint64_t)c, n_tokens);
      if (t < n_tokens) acc += to_f32(table[(uint64_t)t * table_stride + d]);
    }
    out[i] = from_f32<T>(acc * scale);
  }
}

// ---- stable radix sort of (token, row) pairs --------------------------
constexpr int kSortThreads = 256;
constexpr int kSortItems = 8;                       // a thread's cells, consecutive
constexpr int kSortTile = kSortThreads * kSortItems;
constexpr int kDigitBits = 4;
constexpr int kDigits = 1 << kDigitBits;

// Cells to (token, row) pairs; the cells outside every bag of a ragged
// batch keep the absent token that k_no_rows gave them.
template <typename Tok>
__global__ void k_pairs_uniform(const Tok* __restrict__ tokens, uint64_t n_cells, uint64_t per_row,
                                uint64_t n_tokens, uint32_t* __restrict__ key, uint32_t* __restrict__ row) {
  for (uint64_t c = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; c < n_cells;
       c += (uint64_t)gridDim.x * blockDim.x) {
    key[c] = token_of(tokens, c, n_tokens);
    row[c] = (uint32_t)(c / per_row);
  }
}
__global__ void k_no_rows(uint64_t n_cells, uint64_t n_tokens, uint32_t* __restrict__ key,
                          uint32_t* __restrict__ row) {
  for (uint64_t c = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; c < n_cells;
       c += (uint64_t)gridDim.x * blockDim.x) {
    key[c] = (uint32_t)n_tokens;
    row[c] = 0u;
  }
}
template <typename Tok>
__global__ void k_pairs_ragged(const Tok* __restrict__ tokens, const int64_t* __restrict__ row_ptr,
                               uint64_t n_rows, uint64_t n_cells, uint64_t n_tokens,
                               uint32_t* __restrict__ key, uint32_t* __restrict__ row) {
  // a warp per row
  const uint32_t lane = threadIdx.x & 31u;
  for (uint64_t r = ((uint64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5; r < n_rows;
       r += ((uint64_t)gridDim.x * blockDim.x) >> 5) {
    const int64_t c0 = max((int64_t)0, row_ptr[r]), c1 = min((int64_t)n_cells, row_ptr[r + 1]);
    for (int64_t c = c0 + lane; c < c1; c += 32) {
      key[c] = token_of(tokens, (uint64_t)c, n_tokens);
      row[c] = (uint32_t)r;
    }
  }
}

// counts[d * tiles + tile] = cells of the tile whose digit is d.
__global__ void k_digit_counts(const uint32_t* __restrict__ key, uint64_t n, int shift,
                               uint32_t* __restrict__ counts) {
  __shared__ uint32_t s[kDigits];
  if (threadIdx.x < kDigits) s[threadIdx.x] = 0u;
  __syncthreads();
  const uint64_t base = (uint64_t)blockIdx.x * kSortTile;
  for (int i = threadIdx.x; i < kSortTile; i += kSortThreads)
    if (base + i < n) atomicAdd(&s[(key[base + i] >> shift) & (kDigits - 1)], 1u);
  __syncthreads();
  if (threadIdx.x < kDigits) counts[(uint64_t)threadIdx.x * gridDim.x + blockIdx.x] = s[threadIdx.x];
}

// In place exclusive prefix sum by one CTA of 1,024 threads.
__global__ void k_scan(uint32_t* __restrict__ v, uint64_t n) {
  __shared__ uint32_t s[1024];
  uint32_t carry = 0u;
  for (uint64_t b = 0; b < n; b += 1024) {
    const uint64_t i = b + threadIdx.x;
    const uint32_t x = i < n ? v[i] : 0u;
    s[threadIdx.x] = x;
    __syncthreads();
    for (int o = 1; o < 1024; o <<= 1) {
      const uint32_t y = threadIdx.x >= o ? s[threadIdx.x - o] : 0u;
      __syncthreads();
      s[threadIdx.x] += y;
      __syncthreads();
    }
    if (i < n) v[i] = carry + s[threadIdx.x] - x;
    carry += s[1023];
    __syncthreads();
  }
}

// Moves a tile's pairs to their digit's place, keeping their order: thread t
// owns kSortItems consecutive cells, and the counts of (digit, thread) are
// scanned digit-major.
__global__ void k_digit_scatter(const uint32_t* __restrict__ key, const uint32_t* __restrict__ row,
                                uint64_t n, int shift, const uint32_t* __restrict__ offsets,
                                uint32_t* __restrict__ key_out, uint32_t* __restrict__ row_out) {
  __shared__ uint32_t s[kDigits][kSortThreads + 1];
  const int t = threadIdx.x;
  const uint64_t base = (uint64_t)blockIdx.x * kSortTile + (uint64_t)t * kSortItems;
  for (int d = 0; d < kDigits; ++d) s[d][t] = 0u;
  uint32_t k[kSortItems];
  for (int i = 0; i < kSortItems; ++i)
    if (base + i < n) {
      k[i] = key[base + i];
      ++s[(k[i] >> shift) & (kDigits - 1)][t];
    }
  __syncthreads();
  if (t < kDigits) {
    uint32_t run = offsets[(uint64_t)t * gridDim.x + blockIdx.x];
    for (int j = 0; j < kSortThreads; ++j) {
      const uint32_t c = s[t][j];
      s[t][j] = run;
      run += c;
    }
  }
  __syncthreads();
  for (int i = 0; i < kSortItems; ++i)
    if (base + i < n) {
      const uint32_t to = s[(k[i] >> shift) & (kDigits - 1)][t]++;
      key_out[to] = k[i];
      row_out[to] = row[base + i];
    }
}

// starts[v] = first sorted cell with a token >= v, for v in [0, n_tokens].
__global__ void k_starts(const uint32_t* __restrict__ key, uint64_t n, uint64_t n_tokens,
                         uint32_t* __restrict__ starts) {
  for (uint64_t v = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; v <= n_tokens;
       v += (uint64_t)gridDim.x * blockDim.x) {
    uint64_t lo = 0, hi = n;
    while (lo < hi) {
      const uint64_t m = (lo + hi) >> 1;
      if (key[m] < v) lo = m + 1; else hi = m;
    }
    starts[v] = (uint32_t)lo;
  }
}

// A warp per token: its run of rows summed in order.
template <typename T>
__global__ void k_embed_backward(const uint32_t* __restrict__ row, const uint32_t* __restrict__ starts,
                                 const T* __restrict__ grad, uint64_t grad_stride, uint64_t n_tokens,
                                 uint32_t width, float scale, T* __restrict__ dtable) {
  const uint32_t lane = threadIdx.x & 31u;
  for (uint64_t v = ((uint64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5; v < n_tokens;
       v += ((uint64_t)gridDim.x * blockDim.x) >> 5) {
    const uint32_t c0 = starts[v], c1 = starts[v + 1];
    for (uint32_t d = lane; d < width; d += 32) {
      float acc = 0.0f;
      for (uint32_t c = c0; c < c1; ++c) acc += to_f32(grad[(uint64_t)row[c] * grad_stride + d]);
      dtable[v * width + d] = from_f32<T>(acc * scale);
    }
  }
}

struct BackwardPlan {
  uint64_t tiles, counts, pairs, starts, bytes;
  int passes;
};
BackwardPlan backward_plan(uint64_t n_cells, uint64_t n_tokens) {
  BackwardPlan p;
  p.tiles = (n_cells + kSortTile - 1) / kSortTile;
  p.passes = 0;
  while (p.passes * kDigitBits < 33 && (n_tokens >> (p.passes * kDigitBits))) ++p.passes;
  p.pairs = round_up(4 * n_cells, 256);
  p.counts = round_up(4 * p.tiles * kDigits, 256);
  p.starts = round_up(4 * (n_tokens + 1), 256);
  p.bytes = 4 * p.pairs + p.counts + p.starts;
  return p;
}

int grid_for(uint64_t threads, int block, int sms) {
  return (int)std::max<uint64_t>(1, std::min<uint64_t>((threads + block - 1) / block, (uint64_t)sms * 16));
}

hb_status check_tokens(const void* tokens, int32_t token_type, const int64_t* row_ptr, uint64_t n_rows,
                       uint64_t n_cells, uint64_t n_tokens, uint32_t width, int32_t dtype) {
  HB_HEAD_REQUIRE(known_type(dtype), "unknown element type");
  HB_HEAD_REQUIRE(token_type == HB_I32 || token_type == HB_I64, "unknown token type");
  HB_HEAD_REQUIRE(width >= 1, "width must be at least 1");
  HB_HEAD_REQUIRE(n_tokens >= 1 && n_tokens < 0xffffffffull, "n_tokens must be in [1, 2^32 - 1)");
  HB_HEAD_REQUIRE(n_rows < 0xffffffffull && n_cells < 0xffffffffull, "at most 2^32 - 2 rows and cells");
  HB_HEAD_REQUIRE(row_ptr || (n_rows ? n_cells % n_rows == 0 : n_cells == 0),
                  "without row_ptr every row has n_cells / n_rows cells");
  HB_HEAD_REQUIRE(tokens || !n_cells, "tokens is NULL");
  HB_HEAD_REQUIRE(aligned(tokens, token_type == HB_I32 ? 4 : 8), "tokens is not aligned to its type");
  HB_HEAD_REQUIRE(aligned(row_ptr, 8), "row_ptr is not 8-byte aligned");
  return HB_OK;
}

}  // namespace
}  // namespace head
}  // namespace hb

using namespace hb::head;

extern "C" {

hb_status hb_embed_forward(int32_t device, const void* tokens, int32_t token_type,
                           const int64_t* row_ptr, uint64_t n_rows, uint64_t n_cells,
                           const void* table, int32_t dtype, uint64_t n_tokens, uint32_t width,
                           uint64_t table_stride, float scale, void* out, void* stream) {
  begin_call();
  if (hb_status st = check_tokens(tokens, token_type, row_ptr, n_rows, n_cells, n_tokens, width, dtype)) return st;
  HB_HEAD_REQUIRE(table && (out || !n_rows), "table or out is NULL");
  HB_HEAD_REQUIRE(table_stride >= width, "table_stride is below width");
  HB_HEAD_REQUIRE(aligned(table, size_of(dtype)) && aligned(out, size_of(dtype)), "table or out is not aligned to its type");
  if (!n_rows) return HB_OK;
  DeviceScope dev(device);
  if (!dev.ok()) return fail(HB_REFUSED, "no such device");
  const uint64_t per_row = row_ptr ? 0 : n_cells / n_rows;
  const int grid = grid_for(n_rows * width, 256, sm_count(device));
  with_type(dtype, [&](auto tag) {
    using T = decltype(tag);
    if (token_type == HB_I32)
      k_embed_forward<T, int32_t><<<grid, 256, 0, (cudaStream_t)stream>>>(
          (const int32_t*)tokens, row_ptr, n_rows, n_cells, per_row, (const T*)table, n_tokens, width,
          table_stride, scale, (T*)out);
    else
      k_embed_forward<T, int64_t><<<grid, 256, 0, (cudaStream_t)stream>>>(
          (const int64_t*)tokens, row_ptr, n_rows, n_cells, per_row, (const T*)table, n_tokens, width,
          table_stride, scale, (T*)out);
  });
  return launched("hb_embed_forward");
}

hb_status hb_embed_backward_workspace(uint64_t n_rows, uint64_t n_cells, uint64_t n_tokens, uint32_t width,
                                      uint64_t* bytes) {
  begin_call();
  HB_HEAD_REQUIRE(bytes, "bytes is NULL");
  HB_HEAD_REQUIRE(n_rows < 0xffffffffull && n_cells < 0xffffffffull && n_tokens < 0xffffffffull && width,
                  "sizes out of range");
  *bytes = backward_plan(n_cells, n_tokens).bytes;
  return HB_OK;
}

hb_status hb_embed_backward(int32_t device, const void* tokens, int32_t token_type,
                            const int64_t* row_ptr, uint64_t n_rows, uint64_t n_cells, const void* grad,
                            int32_t dtype, uint64_t grad_stride, uint64_t n_tokens, uint32_t width,
                            float scale, void* dtable, void* workspace, uint64_t workspace_bytes,
                            void* stream) {
  begin_call();
  if (hb_status st = check_tokens(tokens, token_type, row_ptr, n_rows, n_cells, n_tokens, width, dtype)) return st;
  HB_HEAD_REQUIRE((grad || !n_rows) && dtable, "grad or dtable is NULL");
  HB_HEAD_REQUIRE(grad_stride >= width || n_rows <= 1 || grad_stride == 0, "grad_stride is below width");
  HB_HEAD_REQUIRE(aligned(grad, size_of(dtype)) && aligned(dtable, size_of(dtype)), "grad or dtable is not aligned to its type");
  const BackwardPlan p = backward_plan(n_cells, n_tokens);
  HB_HEAD_REQUIRE(workspace_bytes >= p.bytes && workspace && aligned(workspace, 256),
                  "workspace is too small or not 256-byte aligned");
  DeviceScope dev(device);
  if (!dev.ok()) return fail(HB_REFUSED, "no such device");
  cudaStream_t s = (cudaStream_t)stream;
  const int sms = sm_count(device);
  char* at = (char*)workspace;
  auto take = [&](uint64_t bytes) { char* q = at; at += bytes; return (uint32_t*)q; };
  uint32_t *key[2], *row[2];
  for (int b = 0; b < 2; ++b) key[b] = take(p.pairs), row[b] = take(p.pairs);
  uint32_t* counts = take(p.counts);
  uint32_t* starts = take(p.starts);
  int cur = 0;
  if (n_cells) {
    auto pairs = [&](auto tok) {
      using Tok = decltype(tok);
      if (row_ptr) {
        k_no_rows<<<grid_for(n_cells, 256, sms), 256, 0, s>>>(n_cells, n_tokens, key[0], row[0]);
        if (n_rows)
          k_pairs_ragged<Tok><<<grid_for(n_rows * 32, 256, sms), 256, 0, s>>>((const Tok*)tokens, row_ptr, n_rows,
                                                                          n_cells, n_tokens, key[0], row[0]);
      } else {
        k_pairs_uniform<Tok><<<grid_for(n_cells, 256, sms), 256, 0, s>>>((const Tok*)tokens, n_cells, n_cells / n_rows,
                                                                     n_tokens, key[0], row[0]);
      }
    };
    if (token_type == HB_I32) pairs(int32_t{}); else pairs(int64_t{});
    for (int pass = 0; pass < p.passes; ++pass, cur ^= 1) {
      k_digit_counts<<<(int)p.tiles, kSortThreads, 0, s>>>(key[cur], n_cells, pass * kDigitBits, counts);
      k_scan<<<1, 1024, 0, s>>>(counts, p.tiles * kDigits);
      k_digit_scatter<<<(int)p.tiles, kSortThreads, 0, s>>>(key[cur], row[cur], n_cells, pass * kDigitBits, counts,
                                                        key[cur ^ 1], row[cur ^ 1]);
    }
  }
  k_starts<<<grid_for(n_tokens + 1, 256, sms), 256, 0, s>>>(key[cur], n_cells, n_tokens, starts);
  with_type(dtype, [&](auto tag) {
    using T = decltype(tag);
    k_embed_backward<T><<<grid_for(n_tokens * 32, 256, sms), 256, 0, s>>>(row[cur], starts, (const T*)grad, grad_stride,
                                                                     n_tokens, width, scale, (T*)dtable);
  });
  return launched("hb_embed_backward");
}

}  // extern "C"
