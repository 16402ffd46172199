// Embedding of token bags and the table's gradient.
//
//   forward   out[n]    = scale * sum over the cells c of row n of table[t_c]
//   backward  dtable[v] = scale * sum over the cells c with t_c = v of grad[row(c)]
//
// A token id outside [0, n_tokens) is an absent cell (a missing value of the
// binned matrix): it contributes nothing, and a row of nothing but absent
// cells is 0. Sums are f32 in a fixed order, rounded once to the table's
// type, so results do not change from run to run.
//
// Both directions move one row of `width` elements a cell through the L2 cache
// (the tables and gradients of a head fit there) and are bound by what is issued
// for a cell and by waiting for its row: 5.2M cells of 128 bf16 take 135 us
// forward, 11 TB/s of the L2 cache (43% of its rate) with an instruction issued
// in 65% of the cycles. So the lanes of a row load 8 tokens together and pass
// them round, a row's address is one multiply-add, and two f32 are added at a
// time; with every lane working out its own addresses it took 298 us.
//
// The gradient sorts the cells by token (a stable radix sort of (token, row)
// pairs, digits of at most 10 bits) and sums the sorted cells' rows in chunks
// of equal length, whatever the tokens' frequencies: a run of one token that
// lies inside a chunk is finished there; a run that crosses chunks leaves a
// part in each, and the parts are summed in order, by the same kernel where
// there are many of them (its input is then the parts), else by the warp of
// the chunk where the run begins.
#include <algorithm>
#include <type_traits>

#include "hb_head.h"

namespace hb {
namespace head {
namespace {

constexpr uint32_t kAbsent = 0xffffffffu;

template <typename Tok>
__device__ __forceinline__ uint32_t token_of(const Tok* tokens, uint64_t c, uint32_t n_tokens) {
  // negative ids and ids past the table become n_tokens: absent
  const uint64_t t = (uint64_t)(int64_t)tokens[c];
  return t < n_tokens ? (uint32_t)t : n_tokens;
}

// ---- vectors --------------------------------------------------------------
// V elements of T, at most 16 bytes, added into f32, two at a time.
template <typename T, int V>
__device__ __forceinline__ void add_to(float (&a)[V], const Pack<T, V>& q) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      float2 x = make_float2(a[j], a[j + 1]), y = make_float2(to_f32(q.v[j]), to_f32(q.v[j + 1]));
      unsigned long long& xu = reinterpret_cast<unsigned long long&>(x);
      asm("add.rn.f32x2 %0, %0, %1;" : "+l"(xu) : "l"(reinterpret_cast<unsigned long long&>(y)));
      a[j] = x.x, a[j + 1] = x.y;
    }
  } else {
    a[0] += to_f32(q.v[0]);
  }
}
// q, or zeros.
template <typename T, int V>
__device__ __forceinline__ void keep(Pack<T, V>& q, bool it) {
  if constexpr (sizeof(q) % 4 == 0) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&q);
#pragma unroll
    for (int i = 0; i < (int)sizeof(q) / 4; ++i) w[i] = it ? w[i] : 0u;
  } else {
    uint16_t& w = reinterpret_cast<uint16_t&>(q);
    w = it ? w : (uint16_t)0;
  }
}
template <typename T, int V>
__device__ __forceinline__ void put(T* to, const float (&a)[V], float scale) {
  Pack<T, V> q;
#pragma unroll
  for (int j = 0; j < V; ++j) q.v[j] = from_f32<T>(a[j] * scale);
  *reinterpret_cast<Pack<T, V>*>(to) = q;
}

// How a width is laid over lanes: vectors of V elements, groups of `lanes`
// (a power of two) for a row, each lane N vectors `lanes` apart; blockIdx.y
// counts pieces of lanes * N vectors.
struct Cover {
  int v, n, lanes, pieces;
};
Cover cover(uint32_t width, uint64_t elem, bool by16, bool by4) {
  Cover c;
  c.v = by16 ? (int)(16 / elem) : by4 ? (int)(4 / elem) : 1;
  const uint32_t vecs = width / c.v;
  c.lanes = 1;
  while (c.lanes < 32 && (uint32_t)c.lanes < vecs) c.lanes *= 2;
  c.n = vecs > 64 ? 4 : vecs > 32 ? 2 : 1;
  c.pieces = (int)((vecs + c.lanes * c.n - 1) / (c.lanes * c.n));
  return c;
}
// f(V, N) as constants.
template <typename T, typename F>
void with_cover(const Cover& c, F&& f) {
  using std::integral_constant;
  const auto n = [&](auto v) {
    if (c.n == 1) f(v, integral_constant<int, 1>{});
    else if (c.n == 2) f(v, integral_constant<int, 2>{});
    else f(v, integral_constant<int, 4>{});
  };
  if (c.v == (int)(16 / sizeof(T))) n(integral_constant<int, 16 / sizeof(T)>{});
  else if (sizeof(T) == 2 && c.v == 2) n(integral_constant<int, 2>{});
  else n(integral_constant<int, 1>{});
}

// 8 words of a list that the lanes of a group go through together. Groups of
// 8 lanes or more (kTogether) load a word a lane and pass it round.
constexpr int kBatch = 8;
template <bool kTogether>
struct Batch {
  uint32_t w[kTogether ? 1 : kBatch];
  template <typename F>
  __device__ __forceinline__ void load(F&& word) {
    if constexpr (kTogether) {
      w[0] = word(threadIdx.x & (kBatch - 1));
    } else {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) w[u] = word(u);
    }
  }
  // Whether all the words this lane holds satisfy f.
  template <typename F>
  __device__ __forceinline__ bool all(F&& f) const {
    bool ok = true;
#pragma unroll
    for (int u = 0; u < (kTogether ? 1 : kBatch); ++u) ok = ok && f(w[u]);
    return ok;
  }
  // Word u, the same u for every lane of the warp; `first` the group's first lane.
  __device__ __forceinline__ uint32_t get(int u, int first) const {
    if constexpr (kTogether) return __shfl_sync(0xffffffffu, w[0], first + u);
    else return w[u];
  }
};

// ---- forward ---------------------------------------------------------------
constexpr int kForwardThreads = 256;
// Vectors in flight a lane.
constexpr int kFlight = 4;

// A group of lanes a row, or `split` (a power of two) groups of one warp:
// group k takes cells k, k + split, ... and their sums meet in the warp.
template <typename T, typename Tok, int V, int N, bool kTogether>
__global__ void __launch_bounds__(kForwardThreads, N * V <= 8 ? 4 : N * V <= 16 ? 3 : 2)
    k_embed_forward(const Tok* __restrict__ tokens, const int64_t* __restrict__ row_ptr, uint64_t n_rows,
                    uint64_t n_cells, uint64_t per_row, const T* __restrict__ table, uint32_t n_tokens,
                    uint32_t width, uint32_t stride_bytes, float scale, int lanes, int split,
                    T* __restrict__ out) {
  const int lane = threadIdx.x & (lanes - 1), part = threadIdx.x / lanes & (split - 1);
  const uint64_t r = ((uint64_t)blockIdx.x * kForwardThreads + threadIdx.x) / (lanes * split);
  const uint32_t d0 = (blockIdx.y * lanes * N + lane) * V;
  // a lane past the width goes along with column 0
  const unsigned char* column[N];
#pragma unroll
  for (int i = 0; i < N; ++i) column[i] = reinterpret_cast<const unsigned char*>(table + (d0 + i * lanes * V < width ? d0 + i * lanes * V : 0));
  float a[N][V] = {};
  uint32_t begin = 0u, end = 0u;
  if (r < n_rows) {
    int64_t c0 = (int64_t)(r * per_row), c1 = c0 + (int64_t)per_row;
    if (row_ptr) {
      c0 = max((int64_t)0, row_ptr[r]);
      c1 = min((int64_t)n_cells, row_ptr[r + 1]);
    }
    if (c0 < c1) begin = (uint32_t)c0 + part, end = (uint32_t)c1;
  }
  const int first = threadIdx.x & 31 & ~(lanes - 1);
  Batch<kTogether> ids, next;
  const auto fetch = [&](uint32_t c) {
    next.load([&](int u) {
      const uint64_t at = (uint64_t)c + u * split;
      return at < end ? token_of(tokens, at, n_tokens) : n_tokens;
    });
  };
  const auto vector = [&](uint32_t t, int i) {
    return reinterpret_cast<const Pack<T, V>*>(column[i] + (uint64_t)t * stride_bytes);
  };
  fetch(begin);
  // the warp's lanes stay together: as many rounds as its longest row has
  int rounds = begin < end ? (int)((end - begin + kBatch * split - 1) / (kBatch * split)) : 0;
  rounds = __reduce_max_sync(0xffffffffu, rounds);
  // a group whose own row is through stays where it is: going on, `c` could
  // pass 2^32 and come back to cells before `end`
  for (uint32_t c = begin; rounds > 0; --rounds) {
    constexpr int U = kFlight / N;  // cells in flight
    ids = next;
    if (c < end) c += kBatch * split;  // less than 256 past the end, and 2^32 is 4,098 past it
    if (rounds > 1) fetch(c);
    const bool whole = __all_sync(0xffffffffu, ids.all([&](uint32_t t) { return t < n_tokens; }));
#pragma unroll
    for (int b = 0; b < kBatch; b += U) {
      uint32_t t[U];
      Pack<T, V> q[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u) t[u] = ids.get(b + u, first);
      if (whole) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < N; ++i) q[u][i] = *vector(t[u], i);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < N; ++i) add_to(a[i], q[u][i]);
      } else {
        // an absent cell reads row 0 and adds zeros: no branches between loads
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < N; ++i) q[u][i] = *vector(t[u] < n_tokens ? t[u] : 0u, i);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < N; ++i) {
            keep(q[u][i], t[u] < n_tokens);
            add_to(a[i], q[u][i]);
          }
      }
    }
  }
  for (int o = lanes; o < lanes * split; o <<= 1)
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) a[i][j] += __shfl_xor_sync(0xffffffffu, a[i][j], o);
  if (r < n_rows && part == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t d = d0 + i * lanes * V;
      if (d < width) put<T, V>(out + r * width + d, a[i], scale);
    }
  }
}

// ---- stable radix sort of (token, row) pairs --------------------------
constexpr int kSortThreads = 256;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortRounds = 8;                      // a warp's cells: 8 rounds of 32 in order
constexpr int kSortTile = kSortThreads * kSortRounds;
constexpr int kMostBits = 10;                       // of a digit
constexpr int kMostDigits = 1 << kMostBits;

// The row of every cell inside a bag (the others keep kAbsent): a warp a row.
__global__ void k_rows_ragged(const int64_t* __restrict__ row_ptr, uint64_t n_rows, uint64_t n_cells,
                              uint32_t* __restrict__ row) {
  const uint32_t lane = threadIdx.x & 31u;
  for (uint64_t r = ((uint64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5; r < n_rows;
       r += ((uint64_t)gridDim.x * blockDim.x) >> 5) {
    const int64_t c0 = max((int64_t)0, row_ptr[r]), c1 = min((int64_t)n_cells, row_ptr[r + 1]);
    for (int64_t c = c0 + lane; c < c1; c += 32) row[c] = (uint32_t)r;
  }
}

// Where a pass reads its pairs: the first pass the tokens (and the rows of
// a ragged batch), the others the pass before.
template <typename Tok>
struct FirstPass {
  const Tok* tokens;
  const uint32_t* rows;  // NULL: cell c is of row c / per_row
  uint32_t per_row, over, n_tokens;  // over: 2^32 / per_row, rounded down
  __device__ __forceinline__ uint32_t key(uint32_t c) const {
    const uint32_t t = token_of(tokens, c, n_tokens);
    return rows && rows[c] == kAbsent ? n_tokens : t;
  }
  __device__ __forceinline__ uint32_t row(uint32_t c) const {
    if (rows) return rows[c];
    const uint32_t q = __umulhi(c, over);  // the quotient, or one less
    return c - q * per_row >= per_row ? q + 1 : q;
  }
};
struct NextPass {
  const uint32_t *keys, *rows;
  __device__ __forceinline__ uint32_t key(uint32_t c) const { return keys[c]; }
  __device__ __forceinline__ uint32_t row(uint32_t c) const { return rows[c]; }
};

// counts[d * tiles + tile] = cells of the tile whose digit is d.
template <typename Source>
__global__ void __launch_bounds__(kSortThreads)
    k_digit_counts(const Source from, uint32_t n, int shift, int digits, uint32_t* __restrict__ counts) {
  __shared__ uint32_t s[kMostDigits];
  for (int d = threadIdx.x; d < digits; d += kSortThreads) s[d] = 0u;
  __syncthreads();
  const uint32_t base = blockIdx.x * kSortTile;
#pragma unroll 4
  for (int i = threadIdx.x; i < kSortTile; i += kSortThreads)
    if (base + i < n) atomicAdd(&s[(from.key(base + i) >> shift) & (digits - 1)], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += kSortThreads) counts[(uint64_t)d * gridDim.x + blockIdx.x] = s[d];
}

// Exclusive prefix sum of one value a thread; the sum of all in *all.
__device__ __forceinline__ uint32_t cta_scan(uint32_t v, uint32_t* all) {
  __shared__ uint32_t s[kSortWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) s[warp] = x;
  __syncthreads();
  uint32_t before = 0u, sum = 0u;
#pragma unroll
  for (int w = 0; w < kSortWarps; ++w) {
    before += w < warp ? s[w] : 0u;
    sum += s[w];
  }
  *all = sum;
  return before + x - v;
}

// A CTA a digit: its tiles' counts become their exclusive prefix sums.
__global__ void __launch_bounds__(kSortThreads)
    k_digit_scan(uint32_t* __restrict__ counts, uint32_t tiles, uint32_t* __restrict__ totals) {
  uint32_t* c = counts + (uint64_t)blockIdx.x * tiles;
  uint32_t carry = 0u;
  constexpr uint32_t kEach = 8;
  for (uint32_t b = 0; b < tiles; b += kSortThreads * kEach) {
    const uint32_t at = b + threadIdx.x * kEach;
    uint32_t v[kEach], sum = 0u, all;
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
      v[i] = at + i < tiles ? c[at + i] : 0u;
      sum += v[i];
    }
    uint32_t run = carry + cta_scan(sum, &all);
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
      if (at + i < tiles) c[at + i] = run;
      run += v[i];
    }
    carry += all;
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

// Moves a tile's pairs to their digit's place, keeping their order. Warp w
// has 256 consecutive cells in rounds of 32; a cell's rank among its digit's
// is the warps' before, its warp's rounds' before, its round's lanes' before.
// The tile is put in order in shared memory first, so that each digit's
// pairs go out together. totals NULL: the tile is all there is.
template <typename Source>
__global__ void __launch_bounds__(kSortThreads, 5)
    k_digit_scatter(const Source from, uint32_t n, int shift, int digits, const uint32_t* __restrict__ counts,
                    const uint32_t* __restrict__ totals, uint32_t* __restrict__ key_out,
                    uint32_t* __restrict__ row_out) {
  extern __shared__ uint32_t sm[];
  uint32_t* s_count = sm;                                // [kSortWarps][digits]
  uint32_t* s_to = sm + kSortWarps * digits;             // [digits]: place of the digit's first pair, less its place in the tile
  uint32_t* s_key = s_to + digits;                       // [kSortTile]
  uint32_t* s_row = s_key + kSortTile;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t base = blockIdx.x * kSortTile, here = min((uint32_t)kSortTile, n - base);
  for (int i = threadIdx.x; i < kSortWarps * digits; i += kSortThreads) s_count[i] = 0u;
  __syncthreads();
  uint32_t key[kSortRounds];
  uint16_t rank[kSortRounds];
  uint32_t* mine = s_count + warp * digits;
#pragma unroll
  for (int i = 0; i < kSortRounds; ++i) {
    const uint32_t c = warp * (32 * kSortRounds) + i * 32 + lane;
    key[i] = c < here ? from.key(base + c) : 0u;
  }
#pragma unroll
  for (int i = 0; i < kSortRounds; ++i) {
    const uint32_t c = warp * (32 * kSortRounds) + i * 32 + lane;
    const uint32_t d = c < here ? (key[i] >> shift) & (digits - 1) : kAbsent;
    // the lanes of the same digit, a bit at a time (20 us for 1.8M cells
    // against 24 with the match instruction, which slows with the number of
    // different digits)
    uint32_t same = __ballot_sync(0xffffffffu, c < here);
    if (c >= here) same = ~same;
    for (int b = digits >> 1; b; b >>= 1) {
      const uint32_t ones = __ballot_sync(0xffffffffu, d & b);
      same &= d & b ? ones : ~ones;
    }
    const uint32_t before = c < here ? mine[d] : 0u;
    rank[i] = (uint16_t)(before + __popc(same & ((1u << lane) - 1u)));
    __syncwarp();
    if (c < here && (same >> lane) == 1u) mine[d] = before + __popc(same);  // the last of its lanes
    __syncwarp();
  }
  __syncthreads();
  // digit by digit (kEach a thread): the warps' counts to their prefix sums in
  // the tile, and the digits' places
  constexpr int kEach = kMostDigits / kSortThreads;
  uint32_t count[kEach], sum = 0u, total = 0u, all;
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int d = threadIdx.x * kEach + k;
    count[k] = 0u;
    if (d < digits) {
      for (int w = 0; w < kSortWarps; ++w) count[k] += s_count[w * digits + d];
      sum += count[k];
      if (totals) total += totals[d];
    }
  }
  uint32_t in_tile = cta_scan(sum, &all), place = totals ? cta_scan(total, &all) : 0u;
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int d = threadIdx.x * kEach + k;
    if (d < digits) {
      s_to[d] = totals ? place + counts[(uint64_t)d * gridDim.x + blockIdx.x] - in_tile : 0u;
      if (totals) place += totals[d];
      uint32_t run = in_tile;
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t v = s_count[w * digits + d];
        s_count[w * digits + d] = run;
        run += v;
      }
      in_tile = run;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSortRounds; ++i) {
    const uint32_t c = warp * (32 * kSortRounds) + i * 32 + lane;
    if (c < here) {
      const uint32_t at = mine[(key[i] >> shift) & (digits - 1)] + rank[i];
      s_key[at] = key[i];
      s_row[at] = from.row(base + c);
    }
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < here; i += kSortThreads) {
    const uint32_t k = s_key[i], to = s_to[(k >> shift) & (digits - 1)] + i;
    key_out[to] = k;
    row_out[to] = s_row[i];
  }
}

// ---- sums of the sorted cells' rows ----------------------------------------
constexpr int kSumThreads = 256;

// What becomes of the runs that cross chunks: chunk j leaves a part of the
// run it begins in (slot 2 j) and of the run it ends in (2 j + 1), as rows of
// `width` f32, with their tokens. A slot whose chunk is all one run, already
// in the slot before, holds the token and no row (kAbsent); a slot without a
// run to hand on, no token.
struct Parts {
  float* sums;
  uint32_t *key, *row;
};

// A group of lanes sums a chunk of `chunk` (a multiple of 8) cells in order:
// runs that begin and end inside go to dtable, the others to the parts.
template <typename T, typename Out, int V, int N, bool kTogether>
__global__ void __launch_bounds__(kSumThreads, N * V <= 4 ? 4 : N * V <= 8 ? 3 : 2)
    k_run_sums(const uint32_t* __restrict__ key, const uint32_t* __restrict__ row, uint32_t n, uint32_t chunk,
               const T* __restrict__ in, uint32_t stride_bytes, uint32_t n_tokens, uint32_t width, float scale,
               int lanes, Out* __restrict__ dtable, const Parts parts) {
  const int lane = threadIdx.x & (lanes - 1);
  const uint32_t j = (uint32_t)(((uint64_t)blockIdx.x * kSumThreads + threadIdx.x) / lanes);
  const uint64_t begin = (uint64_t)j * chunk;
  // a group past the end goes along with its warp, over no cells
  const uint32_t c0 = (uint32_t)min((uint64_t)n, begin), c1 = (uint32_t)min((uint64_t)n, begin + chunk);
  const uint32_t d0 = (blockIdx.y * lanes * N + lane) * V;
  const unsigned char* column[N];
#pragma unroll
  for (int i = 0; i < N; ++i) column[i] = reinterpret_cast<const unsigned char*>(in + (d0 + i * lanes * V < width ? d0 + i * lanes * V : 0));
  float a[N][V] = {};
  uint32_t now = c0 < c1 ? key[c0] : kAbsent;
  const uint32_t after = c0 < c1 && c1 < n ? key[c1] : kAbsent;
  bool open = c0 < c1 && c0 > 0 && key[c0 - 1] == now;  // the run began before the chunk
  uint32_t tail_key = kAbsent, tail_row = kAbsent, head_key = kAbsent;
  const auto flush = [&](bool goes_on) {
    if (now < n_tokens) {
      if (open || goes_on) {
        const uint32_t slot = 2 * j + (open ? 0 : 1);
        if (open) head_key = now;
        else tail_row = slot;
        if (goes_on) tail_key = now;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const uint32_t d = d0 + i * lanes * V;
          if (d < width) {
#pragma unroll
            for (int k = 0; k < V; ++k) parts.sums[(uint64_t)slot * width + d + k] = a[i][k];
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const uint32_t d = d0 + i * lanes * V;
          if (d < width) put<Out, V>(dtable + (uint64_t)now * width + d, a[i], scale);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) a[i][k] = 0.0f;
    open = false;
  };
  const int first = threadIdx.x & 31 & ~(lanes - 1);
  Batch<kTogether> keys, rows, next_keys, next_rows;
  // a cell that is absent, or past the end, has no row
  const auto fetch = [&](uint32_t c) {
    next_keys.load([&](int u) { return (uint64_t)c + u < c1 ? key[c + u] : kAbsent; });
    next_rows.load([&](int u) { return (uint64_t)c + u < c1 && key[c + u] < n_tokens ? row[c + u] : kAbsent; });
  };
  const auto vector = [&](uint32_t r, int i) {
    return reinterpret_cast<const Pack<T, V>*>(column[i] + (uint64_t)r * stride_bytes);
  };
  fetch(c0);
  for (uint32_t c = c0, left = chunk; left > 0; left -= kBatch, c += kBatch) {
    constexpr int U = kFlight / N;
    keys = next_keys, rows = next_rows;
    if (left > kBatch) fetch(c + kBatch);
    // no token ends and no cell is absent in the batch, in any of the warp's groups
    const bool plain = keys.all([&](uint32_t k) { return k == now; }) && rows.all([](uint32_t r) { return r != kAbsent; });
    const bool whole = __all_sync(0xffffffffu, plain);
#pragma unroll 1
    for (int b = 0; b < kBatch; b += U) {
      uint32_t r[U];
      Pack<T, V> q[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u) r[u] = rows.get(b + u, first);
      if (whole) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < N; ++i) q[u][i] = *vector(r[u], i);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < N; ++i) add_to(a[i], q[u][i]);
        continue;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i) q[u][i] = *vector(r[u] != kAbsent ? r[u] : 0u, i);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t k = keys.get(b + u, first);
        if (k != now && (uint64_t)c + b + u < c1) {
          flush(false);
          now = k;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
          keep(q[u][i], r[u] != kAbsent);
          add_to(a[i], q[u][i]);
        }
        __syncwarp();
      }
    }
  }
  if (c0 >= c1) return;
  flush(after == now);
  if (blockIdx.y == 0 && lane == 0) {
    parts.key[2 * j] = head_key;
    parts.row[2 * j] = head_key == kAbsent ? kAbsent : 2 * j;
    parts.key[2 * j + 1] = tail_key;
    parts.row[2 * j + 1] = tail_row;
  }
}

// The parts of each run, in order: slot i begins a run where its token is
// not the slot's before. A warp looks at kJoinEach slots and takes their runs.
constexpr int kJoinEach = 4, kJoinSlotsCta = kSumThreads / 32 * kJoinEach;
template <typename Out>
__global__ void __launch_bounds__(kSumThreads)
    k_run_join(const Parts parts, uint32_t slots, uint32_t n_tokens, uint32_t width, float scale,
               Out* __restrict__ dtable) {
  const int lane = threadIdx.x & 31;
  const uint32_t warp = (blockIdx.x * kSumThreads + threadIdx.x) >> 5, i = warp * kJoinEach + lane;
  const uint32_t mine = lane < kJoinEach && i < slots ? parts.key[i] : kAbsent;
  uint32_t begins = __ballot_sync(0xffffffffu, mine < n_tokens && (i == 0 || parts.key[i - 1] != mine));
  while (begins) {
    const int l = __ffs(begins) - 1;
    begins &= begins - 1;
    const uint32_t s0 = warp * kJoinEach + l, token = __shfl_sync(0xffffffffu, mine, l);
    const uint32_t b = blockIdx.y * 128 + lane;
    float a[4] = {};
    // 32 slots at a time: whose they are, their rows, then the rows together
    for (uint32_t s = s0; s < slots; s += 32) {
      const bool ours = s + lane < slots && parts.key[s + lane] == token;
      const uint32_t row = ours ? parts.row[s + lane] : kAbsent;
      const uint32_t not_ours = ~__ballot_sync(0xffffffffu, ours);
      const int run = not_ours ? __ffs(not_ours) - 1 : 32;
      for (int u = 0; u < run; u += 8) {
        float v[8][4];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t at = __shfl_sync(0xffffffffu, row, u + k & 31);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            v[k][i] = u + k < run && at != kAbsent && b + i * 32 < width ? parts.sums[(uint64_t)at * width + b + i * 32] : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) a[i] += v[k][i];
      }
      if (run < 32) break;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (b + i * 32 < width) dtable[(uint64_t)token * width + b + i * 32] = from_f32<Out>(a[i] * scale);
  }
}

// ---- plan of the gradient ----------------------------------------------------
constexpr uint32_t kJoinSlots = 1024;  // parts that k_run_join takes; more are summed in chunks first

struct BackwardPlan {
  uint32_t tiles, chunk, chunks, chunk2, chunks2;  // the 2s: of the parts, where they are too many
  int passes, bits;                        // digits of `bits`
  uint64_t pairs, counts, totals, parts, parts2, bytes;
};
BackwardPlan backward_plan(uint64_t n_cells, uint64_t n_tokens, uint32_t width) {
  BackwardPlan p;
  p.tiles = (uint32_t)((n_cells + kSortTile - 1) / kSortTile);
  int bits = 1;
  while (n_tokens >> bits) ++bits;
  p.passes = (bits + kMostBits - 1) / kMostBits;
  p.bits = (bits + p.passes - 1) / p.passes;
  // longer chunks leave fewer parts (131,072 rows of about 40 cells, 128 bf16:
  // 521 us forward and back with chunks of 128, 570 of 32, 635 of 16), shorter
  // ones keep the SMs busy (400,000 single cells, 64 bf16: 157 us of 16, 177 of
  // 128): enough chunks for about 64 warps of each of the 148 SMs (the
  // workspace goes by them and is asked for without a device)
  p.chunk = 16;
  while (p.chunk < 128 && n_cells / p.chunk * std::min<uint64_t>(32, (width + 3) / 4) > 148 * 2048 * 2) p.chunk *= 2;
  p.chunks = (uint32_t)((n_cells + p.chunk - 1) / p.chunk);
  p.chunk2 = 32;  // 128 took 4% longer over 20M cells, 24% over 0.2M
  p.chunks2 = 2ull * p.chunks > kJoinSlots ? (uint32_t)((2ull * p.chunks + p.chunk2 - 1) / p.chunk2) : 0;
  p.pairs = round_up(4 * n_cells, 256);
  p.counts = p.tiles > 1 ? round_up(4ull * p.tiles << p.bits, 256) : 0;
  p.totals = round_up(4ull << p.bits, 256);
  const auto parts = [&](uint64_t chunks) { return round_up(8 * chunks * width, 256) + 2 * round_up(8 * chunks, 256); };
  p.parts = parts(p.chunks);
  p.parts2 = p.chunks2 ? parts(p.chunks2) : 0;
  p.bytes = 4 * p.pairs + p.counts + p.totals + p.parts + p.parts2;
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
  HB_HEAD_REQUIRE(width < (1u << 22), "width must be below 2^22");
  HB_HEAD_REQUIRE(n_rows < 0xffffffffull && n_cells < (1ull << 32) - 2 * kSortTile, "at most 2^32 - 4098 rows and cells");
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
  HB_HEAD_REQUIRE(table_stride < (1ull << 30), "table_stride must be below 2^30");
  HB_HEAD_REQUIRE(aligned(table, size_of(dtype)) && aligned(out, size_of(dtype)), "table or out is not aligned to its type");
  if (!n_rows) return HB_OK;
  DeviceScope dev(device);
  if (!dev.ok()) return fail(HB_REFUSED, "no such device");
  const uint64_t per_row = row_ptr ? 0 : n_cells / n_rows, e = size_of(dtype);
  const auto by = [&](uint64_t to) { return aligned(table, to) && aligned(out, to) && width * e % to == 0 && table_stride * e % to == 0; };
  const Cover c = cover(width, e, by(16), by(4));
  // a row's cells among the groups of a warp where the rows alone leave most
  // of the GPU idle: a row of 28 cells then takes 1 round of loads, not 4
  int split = 1;
  while (c.lanes * split < 32 && n_rows * c.lanes * split < (uint64_t)sm_count(device) * 512) split *= 2;
  const uint64_t ctas = (n_rows * c.lanes * split + kForwardThreads - 1) / kForwardThreads;
  HB_HEAD_REQUIRE(ctas < (1ull << 31), "too many rows of this width");
  const dim3 grid((unsigned)ctas, c.pieces);
  with_type(dtype, [&](auto tag) {
    using T = decltype(tag);
    with_cover<T>(c, [&](auto v, auto n) {
      constexpr int V = decltype(v)::value, N = decltype(n)::value;
      const auto run = [&](auto tok) {
        using Tok = decltype(tok);
        const auto kernel = c.lanes >= kBatch ? k_embed_forward<T, Tok, V, N, true> : k_embed_forward<T, Tok, V, N, false>;
        kernel<<<grid, kForwardThreads, 0, (cudaStream_t)stream>>>(
            (const Tok*)tokens, row_ptr, n_rows, n_cells, per_row, (const T*)table, (uint32_t)n_tokens, width,
            (uint32_t)(table_stride * e), scale, c.lanes, split, (T*)out);
      };
      if (token_type == HB_I32) run(int32_t{}); else run(int64_t{});
    });
  });
  return launched("hb_embed_forward");
}

hb_status hb_embed_backward_workspace(uint64_t n_rows, uint64_t n_cells, uint64_t n_tokens, uint32_t width,
                                      uint64_t* bytes) {
  begin_call();
  HB_HEAD_REQUIRE(bytes, "bytes is NULL");
  HB_HEAD_REQUIRE(n_rows < 0xffffffffull && n_cells < (1ull << 32) - 2 * kSortTile && n_tokens < 0xffffffffull && width,
                  "sizes out of range");
  *bytes = backward_plan(n_cells, n_tokens, width).bytes;
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
  HB_HEAD_REQUIRE(grad_stride < (1ull << 30), "grad_stride must be below 2^30");
  HB_HEAD_REQUIRE(aligned(grad, size_of(dtype)) && aligned(dtable, size_of(dtype)), "grad or dtable is not aligned to its type");
  const BackwardPlan p = backward_plan(n_cells, n_tokens, width);
  HB_HEAD_REQUIRE(workspace_bytes >= p.bytes && workspace && aligned(workspace, 256),
                  "workspace is too small or not 256-byte aligned");
  DeviceScope dev(device);
  if (!dev.ok()) return fail(HB_REFUSED, "no such device");
  cudaStream_t s = (cudaStream_t)stream;
  const int sms = sm_count(device);
  const uint64_t e = size_of(dtype);
  // tokens without a cell have a gradient of 0; the others' rows are written over
  if (cudaMemsetAsync(dtable, 0, n_tokens * width * e, s) != cudaSuccess) return launched("hb_embed_backward");
  if (!n_cells || !n_rows) return HB_OK;
  char* at = (char*)workspace;
  const auto take = [&](uint64_t bytes) { char* q = at; at += bytes; return (uint32_t*)q; };
  uint32_t *key[2], *row[2];
  for (int b = 0; b < 2; ++b) key[b] = take(p.pairs), row[b] = take(p.pairs);
  uint32_t *counts = take(p.counts), *totals = take(p.totals);
  const auto take_parts = [&](uint64_t chunks) {
    Parts q;
    q.sums = (float*)take(round_up(8 * chunks * width, 256));
    q.key = take(round_up(8 * chunks, 256)), q.row = take(round_up(8 * chunks, 256));
    return q;
  };
  const Parts parts = take_parts(p.chunks), parts2 = p.chunks2 ? take_parts(p.chunks2) : Parts{};
  const uint32_t n = (uint32_t)n_cells;
  if (row_ptr) {
    // the second buffer's rows: the first pass writes the first buffer's
    if (cudaMemsetAsync(row[1], 0xff, 4 * n_cells, s) != cudaSuccess) return launched("hb_embed_backward");
    k_rows_ragged<<<grid_for(n_rows * 32, 256, sms), 256, 0, s>>>(row_ptr, n_rows, n_cells, row[1]);
  }
  const int digits = 1 << p.bits;
  const uint32_t sort_bytes = 4u * ((kSortWarps + 1) * digits + 2 * kSortTile);
  const auto sort_pass = [&](auto from, int pass) {
    using Source = decltype(from);
    const int shift = pass * p.bits, to = pass & 1;
    if (p.tiles > 1) {
      k_digit_counts<<<p.tiles, kSortThreads, 0, s>>>(from, n, shift, digits, counts);
      k_digit_scan<<<digits, kSortThreads, 0, s>>>(counts, p.tiles, totals);
    }
    allow_shared<k_digit_scatter<Source>>(device, sort_bytes);
    k_digit_scatter<<<p.tiles, kSortThreads, sort_bytes, s>>>(from, n, shift, digits, counts, p.tiles > 1 ? totals : nullptr,
                                                          key[to], row[to]);
  };
  for (int pass = 0; pass < p.passes; ++pass) {
    const uint32_t* rows = row_ptr ? row[1] : nullptr;
    const uint32_t per_row = row_ptr ? 1u : (uint32_t)(n_cells / n_rows), over = per_row > 1 ? (uint32_t)((1ull << 32) / per_row) : 0xffffffffu, tokens_n = (uint32_t)n_tokens;
    if (pass > 0) sort_pass(NextPass{key[pass & 1 ^ 1], row[pass & 1 ^ 1]}, pass);
    else if (token_type == HB_I32) sort_pass(FirstPass<int32_t>{(const int32_t*)tokens, rows, per_row, over, tokens_n}, 0);
    else sort_pass(FirstPass<int64_t>{(const int64_t*)tokens, rows, per_row, over, tokens_n}, 0);
  }
  const int last = (p.passes - 1) & 1;
  const auto by = [&](uint64_t to) { return aligned(grad, to) && aligned(dtable, to) && width * e % to == 0 && grad_stride * e % to == 0; };
  const Cover c = cover(width, e, by(16), by(4));
  const auto ctas = [](uint64_t chunks, int lanes) { return (unsigned)((chunks * lanes + kSumThreads - 1) / kSumThreads); };
  with_type(dtype, [&](auto tag) {
    using T = decltype(tag);
    with_cover<T>(c, [&](auto v, auto w) {
      constexpr int V = decltype(v)::value, N = decltype(w)::value;
      const auto kernel = c.lanes >= kBatch ? k_run_sums<T, T, V, N, true> : k_run_sums<T, T, V, N, false>;
      kernel<<<dim3(ctas(p.chunks, c.lanes), c.pieces), kSumThreads, 0, s>>>(
          key[last], row[last], n, p.chunk, (const T*)grad, (uint32_t)(grad_stride * e), (uint32_t)n_tokens, width, scale, c.lanes, (T*)dtable, parts);
    });
    Parts of = parts;
    uint32_t slots = 2 * p.chunks;
    if (p.chunks2) {
      const Cover c2 = cover(width, 4, width % 4 == 0 && by(4 * e), true);
      with_cover<float>(c2, [&](auto v, auto w) {
        constexpr int V = decltype(v)::value, N = decltype(w)::value;
        const auto kernel = c2.lanes >= kBatch ? k_run_sums<float, T, V, N, true> : k_run_sums<float, T, V, N, false>;
        kernel<<<dim3(ctas(p.chunks2, c2.lanes), c2.pieces), kSumThreads, 0, s>>>(
            parts.key, parts.row, slots, p.chunk2, parts.sums, 4 * width, (uint32_t)n_tokens, width, scale, c2.lanes, (T*)dtable, parts2);
      });
      of = parts2;
      slots = 2 * p.chunks2;
    }
    k_run_join<T><<<dim3((slots + kJoinSlotsCta - 1) / kJoinSlotsCta, (width + 127) / 128), kSumThreads, 0, s>>>(of, slots, (uint32_t)n_tokens, width,
                                                                                                    scale, (T*)dtable);
  });
  return launched("hb_embed_backward");
}

}  // extern "C"
