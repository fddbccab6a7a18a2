// Expert routing for gfx950: the rows of tokens in the order of the experts that the tokens chose, and
// back, with weights applied, and the gradients of both.
//
// n tokens choose k experts each; pair a = t*k + j holds expert e[a].  A pair whose expert lies outside
// [0, E) is dropped (padding, or a pair over its expert's capacity).
//   plan      places = position of every pair in the stable order by (kept ? e : E); order = its inverse;
//             expert_offsets[e] = pairs of experts before e, expert_offsets[E] = pairs kept
//   dispatch  rows[places[t,j]] = x[t]                    (zeros for a dropped pair)
//   combine   y[t] = sum over kept j of w[t,j] * rows[places[t,j]]    (w = 1: dispatch's gradient)
//   combine's gradient   grad_rows[places[t,j]] = w[t,j] * g[t],  grad_w[t,j] = <rows[places[t,j]], g[t]>
// Nothing is added with atomics: every sum has one fixed order, so that two runs are bit-identical.

#include <algorithm>

#include "tbe_common.h"

namespace tbe {
namespace {

// ------------------------------------------------------------------------------------ plan
// A stable counting sort by expert.  Up to kSmallPairs pairs: one workgroup, one launch.  More: the
// counts of every tile of pairs, their prefix sums over the tiles of an expert, and a launch that
// ranks a tile's pairs with wavefront ballots (all lanes of one expert are found with one ballot per bit
// of the expert's number) and places them.  Pairs inside a tile are numbered (wavefront, item, lane),
// which the ranking keeps, so the order is stable.
constexpr int kMaxExperts = TBE_MAX_EXPERTS;  // and one bin more for the dropped pairs
constexpr int kTileWaves = 4, kTileItems = 8;
constexpr int kPlanTile = kTileWaves * kWave * kTileItems;
constexpr int kSmallWaves = 16, kSmallItems = 8;
constexpr int kSmallPairs = kSmallWaves * kWave * kSmallItems;
constexpr int kSmallExperts = 1023;  // widest single-workgroup plan: 16 wavefronts' counters in 64 KB of LDS

template <typename I> __device__ __forceinline__ int bin_of(I expert, int E) {
  return (expert >= 0 && expert < E) ? static_cast<int>(expert) : E;
}

template <typename I, int BINS>
__global__ __launch_bounds__(kBlockThreads) void expert_count_kernel(const I *__restrict__ ids, int64_t n, int E,
                                                                    int64_t tiles, int32_t *__restrict__ counts) {
  __shared__ int32_t s_count[BINS];
  for (int e = threadIdx.x; e <= E; e += kBlockThreads) s_count[e] = 0;
  __syncthreads();
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kPlanTile + threadIdx.x;
#pragma unroll
  for (int q = 0; q < kTileItems; ++q) {
    const int64_t a = base + q * kBlockThreads;
    if (a < n) atomicAdd(&s_count[bin_of(ids[a], E)], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e <= E; e += kBlockThreads) counts[e * tiles + blockIdx.x] = s_count[e];
}

// One wavefront per bin: exclusive prefix sums of its counts over the tiles, and its total.
__global__ __launch_bounds__(kBlockThreads) void expert_scan_kernel(int32_t *__restrict__ counts, int64_t tiles,
                                                                   int E, int32_t *__restrict__ totals) {
  const int lane = threadIdx.x & (kWave - 1);
  const int e = blockIdx.x * kWavesPerBlock + (threadIdx.x >> 6);
  if (e > E) return;
  int32_t *row = counts + e * tiles;
  int running = 0;
  for (int64_t i0 = 0; i0 < tiles; i0 += kWave) {
    const int c = i0 + lane < tiles ? row[i0 + lane] : 0;
    int x = c;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int y = __shfl_up(x, d, kWave);
      if (lane >= d) x += y;
    }
    if (i0 + lane < tiles) row[i0 + lane] = running + x - c;
    running += __shfl(x, kWave - 1, kWave);
  }
  if (lane == 0) totals[e] = running;
}

template <typename I, int WAVES, int ITEMS, int BINS, bool SINGLE>
__global__ __launch_bounds__(WAVES *kWave) void expert_place_kernel(
    const I *__restrict__ ids, int64_t n, int E, int bits, const int32_t *__restrict__ counts,
    const int32_t *__restrict__ totals, int64_t tiles, int32_t *__restrict__ expert_offsets,
    int32_t *__restrict__ order, int32_t *__restrict__ places) {
  constexpr int kThreads = WAVES * kWave;
  __shared__ int32_t s_count[WAVES][BINS];
  __shared__ int32_t s_start[BINS];
  __shared__ int32_t s_wave[WAVES];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = threadIdx.x >> 6;
  for (int e = lane; e <= E; e += kWave) s_count[wave][e] = 0;
  __syncthreads();

  const int64_t base = (static_cast<int64_t>(blockIdx.x) * WAVES + wave) * (kWave * ITEMS) + lane;
  int key[ITEMS], rank[ITEMS];
#pragma unroll
  for (int q = 0; q < ITEMS; ++q) {
    const int64_t a = base + q * kWave;
    key[q] = a < n ? bin_of(ids[a], E) : -1;
  }
#pragma unroll
  for (int q = 0; q < ITEMS; ++q) {
    uint64_t same = __ballot(key[q] >= 0);
    for (int b = 0; b < bits; ++b) {
      const bool set = (key[q] >> b) & 1;
      const uint64_t vote = __ballot(set);
      same &= set ? vote : ~vote;
    }
    rank[q] = 0;
    if (key[q] >= 0) {
      const int first = __ffsll(static_cast<unsigned long long>(same)) - 1;
      int before = 0;
      if (lane == first) before = atomicAdd(&s_count[wave][key[q]], __popcll(same));
      before = __shfl(before, first, kWave);
      rank[q] = before + __popcll(same & ((1ull << lane) - 1));
    }
  }
  __syncthreads();
  // counts of a bin: exclusive over the workgroup's wavefronts, then the bin's total over all tiles
  for (int e = threadIdx.x; e < BINS; e += kThreads) {
    int sum = 0;
    if (e <= E) {
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const int c = s_count[w][e];
        s_count[w][e] = sum;
        sum += c;
      }
      if constexpr (!SINGLE) sum = totals[e];
    }
    s_start[e] = sum;
  }
  __syncthreads();
  // exclusive prefix sum over the bins
  constexpr int kPer = BINS > kThreads ? BINS / kThreads : 1;
  int mine[kPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = threadIdx.x * kPer + i;
    mine[i] = e < BINS ? s_start[e] : 0;
    sum += mine[i];
  }
  int incl = sum;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int y = __shfl_up(incl, d, kWave);
    if (lane >= d) incl += y;
  }
  if (lane == kWave - 1) s_wave[wave] = incl;
  __syncthreads();
  int start = incl - sum;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) start += w < wave ? s_wave[w] : 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = threadIdx.x * kPer + i;
    if (e <= E) {
      if (blockIdx.x == 0) expert_offsets[e] = start;
      int first = start;
      if constexpr (!SINGLE) first += counts[e * tiles + blockIdx.x];
      s_start[e] = first;
    }
    start += mine[i];
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < ITEMS; ++q) {
    const int64_t a = base + q * kWave;
    if (a < n) {
      const int place = s_start[key[q]] + s_count[wave][key[q]] + rank[q];
      places[a] = place;
      order[place] = static_cast<int32_t>(a);
    }
  }
}

// ------------------------------------------------------------------------------- row traffic
// Rows are moved as vectors of VEC elements, the widest of 16, 8, 4 and 2 bytes that divides the row and
// every address.  A workgroup takes `group` whole tokens, or, for rows of more than a workgroup's
// vectors, one slice of one token (blockIdx.y); its threads are dealt to the (token, vector) pairs in
// order, so that no lane idles for a row that is no power of two.
struct RowTiles {
  int64_t tokens;
  int64_t groups;    // of `group` tokens; a workgroup takes every gridDim.x-th one
  int32_t choices;
  int32_t vectors;   // of a row
  int32_t group;     // tokens of a workgroup
  int32_t slice;     // vectors of a workgroup (group * vectors, or fewer than a row)
  uint32_t magic;    // i / vectors = (i * magic) >> shift for the i < 2^16 that occur
  int32_t shift;
};

__device__ __forceinline__ int divided(const RowTiles &r, int i) {
  return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(i)) * r.magic) >> r.shift);
}

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

// The row of a pair, or -1 for one that is dropped.
__device__ __forceinline__ bool is_kept(int32_t place, int32_t kept) {
  return static_cast<uint32_t>(place) < static_cast<uint32_t>(kept);
}

template <typename U, int ITER>
__global__ __launch_bounds__(kBlockThreads) void expert_dispatch_kernel(
    const U *__restrict__ x, int64_t x_stride, const int32_t *__restrict__ places,
    const int32_t *__restrict__ kept_rows, U *__restrict__ rows, RowTiles r) {
  const int col0 = blockIdx.y * r.slice;
  const int64_t pairs = r.tokens * r.choices;
  const int32_t kept = *kept_rows;
  for (int64_t group = blockIdx.x; group < r.groups; group += gridDim.x) {
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
      const int i = it * kBlockThreads + threadIdx.x;
      if (i >= r.slice) continue;
      const int t = r.group > 1 ? divided(r, i) : 0;
      const int col = col0 + i - t * r.vectors;
      const int64_t token = group * r.group + t;
      if (token >= r.tokens || col >= r.vectors) continue;
      const U v = x[token * x_stride + col];
      for (int j = 0; j < r.choices; ++j) {
        const int32_t place = places[token * r.choices + j];
        if (place < 0 || place >= pairs) continue;
        rows[static_cast<int64_t>(place) * r.vectors + col] = place < kept ? v : U{};
      }
    }
  }
}

template <typename T, typename W, int VEC, int ITER>
__global__ __launch_bounds__(kBlockThreads) void expert_combine_kernel(
    const T *__restrict__ rows, int64_t row_stride, const int32_t *__restrict__ places,
    const int32_t *__restrict__ kept_rows, const W *__restrict__ weights, T *__restrict__ out, RowTiles r) {
  using A = typename AccOf<T>::type;
  using P = Pack<T, VEC>;
  const int col0 = blockIdx.y * r.slice;
  const int32_t kept = static_cast<int32_t>(min(static_cast<int64_t>(*kept_rows), r.tokens * r.choices));
  for (int64_t group = blockIdx.x; group < r.groups; group += gridDim.x) {
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
      const int i = it * kBlockThreads + threadIdx.x;
      if (i >= r.slice) continue;
      const int t = r.group > 1 ? divided(r, i) : 0;
      const int col = col0 + i - t * r.vectors;
      const int64_t token = group * r.group + t;
      if (token >= r.tokens || col >= r.vectors) continue;
      A sum[VEC];
#pragma unroll
      for (int q = 0; q < VEC; ++q) sum[q] = A(0);
      for (int j = 0; j < r.choices; ++j) {
        const int64_t a = token * r.choices + j;
        const int32_t place = places[a];
        if (!is_kept(place, kept)) continue;
        const P v = *reinterpret_cast<const P *>(rows + place * row_stride + static_cast<int64_t>(col) * VEC);
        const A w = weights ? static_cast<A>(weights[a]) : A(1);
#pragma unroll
        for (int q = 0; q < VEC; ++q) sum[q] += w * static_cast<A>(v.v[q]);
      }
      P o;
#pragma unroll
      for (int q = 0; q < VEC; ++q) o.v[q] = static_cast<T>(sum[q]);
      *reinterpret_cast<P *>(out + (token * r.vectors + col) * VEC) = o;
    }
  }
}

// GROUP lanes per token (a workgroup per token for GROUP = 256): the token's gradient row is read once per
// kChoices choices, every chosen row is read and its gradient written once.  Without grad_weights the rows are
// not read, without grad_rows nothing is written to them.
template <typename T, typename W, int VEC, int GROUP>
__global__ __launch_bounds__(kBlockThreads) void expert_combine_backward_kernel(
    const T *__restrict__ grad, int64_t grad_stride, const T *__restrict__ rows, int64_t row_stride,
    const int32_t *__restrict__ places, const int32_t *__restrict__ kept_rows, const W *__restrict__ weights,
    T *__restrict__ grad_rows, W *__restrict__ grad_weights, int64_t tokens, int choices, int vectors) {
  using A = typename AccOf<T>::type;
  using P = Pack<T, VEC>;
  constexpr int kChoices = 4;
  __shared__ A s_part[kWavesPerBlock][kChoices];
  const int sub = threadIdx.x % GROUP;
  constexpr int kTokens = kBlockThreads / GROUP;
  const int64_t pairs = tokens * choices;
  const int32_t kept = static_cast<int32_t>(min(static_cast<int64_t>(*kept_rows), pairs));
  // (a group leaves as a whole; with GROUP = 256 the workgroup does, so that its barriers are met by all or none)
  for (int64_t token = static_cast<int64_t>(blockIdx.x) * kTokens + threadIdx.x / GROUP; token < tokens;
       token += static_cast<int64_t>(gridDim.x) * kTokens)
  for (int j0 = 0; j0 < choices; j0 += kChoices) {
    const T *g_row = grad + token * grad_stride;
    int32_t place[kChoices];
    A w[kChoices], dot[kChoices];
#pragma unroll
    for (int j = 0; j < kChoices; ++j) {
      const int64_t a = token * choices + j0 + j;
      place[j] = j0 + j < choices ? places[a] : -1;
      if (place[j] >= pairs) place[j] = -1;
      w[j] = is_kept(place[j], kept) ? static_cast<A>(weights[a]) : A(0);
      dot[j] = A(0);
    }
    for (int col = sub; col < vectors; col += GROUP) {
      const P gv = *reinterpret_cast<const P *>(g_row + static_cast<int64_t>(col) * VEC);
#pragma unroll
      for (int j = 0; j < kChoices; ++j) {
        if (place[j] < 0) continue;
        const bool keep = place[j] < kept;
        P o;
        if (keep && grad_weights) {
          const P v = *reinterpret_cast<const P *>(rows + place[j] * row_stride + static_cast<int64_t>(col) * VEC);
#pragma unroll
          for (int q = 0; q < VEC; ++q) dot[j] += static_cast<A>(v.v[q]) * static_cast<A>(gv.v[q]);
        }
        if (!grad_rows) continue;
#pragma unroll
        for (int q = 0; q < VEC; ++q) o.v[q] = keep ? static_cast<T>(w[j] * static_cast<A>(gv.v[q])) : T(0);
        *reinterpret_cast<P *>(grad_rows + (static_cast<int64_t>(place[j]) * vectors + col) * VEC) = o;
      }
    }
    if (!grad_weights) continue;
#pragma unroll
    for (int j = 0; j < kChoices; ++j) {
#pragma unroll
      for (int m = 1; m < (GROUP < kWave ? GROUP : kWave); m <<= 1) dot[j] += shfl_x(dot[j], m);
    }
    if constexpr (GROUP > kWave) {
      __syncthreads();
      if ((threadIdx.x & (kWave - 1)) == 0) {
#pragma unroll
        for (int j = 0; j < kChoices; ++j) s_part[threadIdx.x >> 6][j] = dot[j];
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kChoices; ++j) {
        dot[j] = A(0);
#pragma unroll
        for (int q = 0; q < kWavesPerBlock; ++q) dot[j] += s_part[q][j];
      }
    }
    if (sub == 0) {
#pragma unroll
      for (int j = 0; j < kChoices; ++j)
        if (j0 + j < choices) grad_weights[token * choices + j0 + j] = static_cast<W>(dot[j]);
    }
  }
}

// ------------------------------------------------------------------------------------ host
size_t element_size(int32_t dtype) {
  return dtype == TBE_DTYPE_F64 ? 8 : dtype == TBE_DTYPE_F32 ? 4 : 2;
}
bool float_dtype(int32_t dtype) {
  return dtype == TBE_DTYPE_F32 || dtype == TBE_DTYPE_F16 || dtype == TBE_DTYPE_F64 || dtype == TBE_DTYPE_BF16;
}

// Widest power of two up to 16 that divides all of the byte counts and addresses or'ed into `bits`.
int vector_bytes(uint64_t bits) {
  int v = 16;
  while (bits & (v - 1)) v >>= 1;
  return v;
}
uint64_t address(const void *p) { return reinterpret_cast<uint64_t>(p); }

constexpr int kRowIter = 4;  // vectors per thread
constexpr int64_t kMaxGrid = 1 << 22;  // workgroups of a launch: grid times workgroup stays below 2^32 threads

// (the division is exact: i < 2^16 and vectors <= 2^16 where it is used)
RowTiles row_tiles(int64_t tokens, int32_t choices, int64_t vectors, dim3 *grid) {
  RowTiles r;
  r.tokens = tokens;
  r.choices = choices;
  r.vectors = static_cast<int32_t>(vectors);
  constexpr int64_t kSpan = kBlockThreads * kRowIter;
  if (vectors >= kSpan) {
    r.group = 1;
    r.groups = tokens;
    r.slice = static_cast<int32_t>(kSpan);
    r.magic = 0;
    r.shift = 0;
    *grid = dim3(static_cast<unsigned>(std::min(tokens, kMaxGrid)), static_cast<unsigned>(ceil_div(vectors, kSpan)));
    return r;
  }
  r.group = static_cast<int32_t>(kSpan / vectors);
  r.slice = static_cast<int32_t>(r.group * vectors);
  int log2 = 0;
  while ((int64_t{1} << log2) < vectors) ++log2;
  r.shift = 16 + log2;
  r.magic = static_cast<uint32_t>(((uint64_t{1} << r.shift) + vectors - 1) / vectors);
  r.groups = ceil_div(tokens, r.group);
  *grid = dim3(static_cast<unsigned>(std::min(r.groups, kMaxGrid)));
  return r;
}

int plan_bits(int32_t experts) {  // bits of the largest bin number, `experts`
  int bits = 0;
  while ((1 << bits) <= experts) ++bits;
  return bits;
}

struct PlanRegions {
  uint64_t counts, totals, total_bytes;
  int64_t tiles;
};
PlanRegions plan_regions(int64_t pairs, int32_t experts) {
  PlanRegions p;
  p.tiles = 0;
  p.counts = p.totals = 0;
  p.total_bytes = 256;
  if (pairs <= kSmallPairs && experts <= kSmallExperts) return p;
  p.tiles = std::max<int64_t>(1, ceil_div(pairs, kPlanTile));
  p.totals = align_up(static_cast<uint64_t>(p.tiles) * (experts + 1) * 4, 256);
  p.total_bytes = p.totals + align_up((experts + 1) * 4ull, 256);
  return p;
}

template <typename I, int BINS>
void launch_plan_tiles(const I *ids, int64_t pairs, int32_t experts, const PlanRegions &p, void *workspace,
                       int32_t *expert_offsets, int32_t *order, int32_t *places, hipStream_t s) {
  int32_t *counts = reinterpret_cast<int32_t *>(static_cast<char *>(workspace) + p.counts);
  int32_t *totals = reinterpret_cast<int32_t *>(static_cast<char *>(workspace) + p.totals);
  const dim3 grid(static_cast<unsigned>(p.tiles));
  TBE_LAUNCH("expert_count", s, (expert_count_kernel<I, BINS>), grid, dim3(kBlockThreads), ids, pairs, experts,
             p.tiles, counts);
  TBE_LAUNCH("expert_scan", s, expert_scan_kernel, dim3(static_cast<unsigned>(ceil_div(experts + 1, kWavesPerBlock))),
             dim3(kBlockThreads), counts, p.tiles, experts, totals);
  TBE_LAUNCH("expert_place", s, (expert_place_kernel<I, kTileWaves, kTileItems, BINS, false>), grid,
             dim3(kTileWaves * kWave), ids, pairs, experts, plan_bits(experts), counts, totals, p.tiles,
             expert_offsets, order, places);
}

template <typename I>
void launch_plan(const void *expert_ids, int64_t pairs, int32_t experts, const PlanRegions &p, void *workspace,
                 int32_t *expert_offsets, int32_t *order, int32_t *places, hipStream_t s) {
  const I *ids = static_cast<const I *>(expert_ids);
  if (p.tiles == 0) {
    const int32_t *none = nullptr;
#define TBE_PLAN_SMALL(BINS)                                                                                     \
  TBE_LAUNCH("expert_place", s, (expert_place_kernel<I, kSmallWaves, kSmallItems, BINS, true>), dim3(1),         \
             dim3(kSmallWaves * kWave), ids, pairs, experts, plan_bits(experts), none, none, int64_t{1},         \
             expert_offsets, order, places)
    if (experts < 256) { TBE_PLAN_SMALL(256); }
    else { TBE_PLAN_SMALL(1024); }
#undef TBE_PLAN_SMALL
  } else if (experts < 256) {
    launch_plan_tiles<I, 256>(ids, pairs, experts, p, workspace, expert_offsets, order, places, s);
  } else if (experts < 1024) {
    launch_plan_tiles<I, 1024>(ids, pairs, experts, p, workspace, expert_offsets, order, places, s);
  } else {
    launch_plan_tiles<I, 4096>(ids, pairs, experts, p, workspace, expert_offsets, order, places, s);
  }
}

struct CombineCall {
  const void *rows;
  int64_t row_stride;
  const int32_t *places;
  const int32_t *kept;
  const void *weights;
  int64_t tokens;
  int32_t choices;
  int64_t D;
  hipStream_t stream;
};

template <typename T, typename W, int VEC>
void launch_combine(const CombineCall &c, void *output) {
  dim3 grid;
  const RowTiles r = row_tiles(c.tokens, c.choices, c.D / VEC, &grid);
  TBE_LAUNCH("expert_combine", c.stream, (expert_combine_kernel<T, W, VEC, kRowIter>), grid, dim3(kBlockThreads),
             static_cast<const T *>(c.rows), c.row_stride, c.places, c.kept, static_cast<const W *>(c.weights),
             static_cast<T *>(output), r);
}

template <typename T, typename W, int VEC>
void launch_combine_backward(const CombineCall &c, const void *grad, int64_t grad_stride, void *grad_rows,
                             void *grad_weights) {
  const int vectors = static_cast<int>(c.D / VEC);
#define TBE_COMBINE_BACKWARD(GROUP)                                                                                \
  TBE_LAUNCH("expert_combine_backward", c.stream, (expert_combine_backward_kernel<T, W, VEC, GROUP>),              \
             dim3(static_cast<unsigned>(std::min(ceil_div(c.tokens, kBlockThreads / GROUP), kMaxGrid))), dim3(kBlockThreads), \
             static_cast<const T *>(grad), grad_stride, static_cast<const T *>(c.rows), c.row_stride, c.places,    \
             c.kept, static_cast<const W *>(c.weights), static_cast<T *>(grad_rows),                               \
             static_cast<W *>(grad_weights), c.tokens, c.choices, vectors)
  if (vectors <= 16) { TBE_COMBINE_BACKWARD(16); }
  else if (vectors <= 256) { TBE_COMBINE_BACKWARD(64); }
  else { TBE_COMBINE_BACKWARD(256); }
#undef TBE_COMBINE_BACKWARD
}

// f(T{}, W{}, VEC) for the types and the vector width of a call
template <typename T, typename W, typename F> void with_vector(int bytes, F &&f) {
  const int vec = bytes / static_cast<int>(sizeof(T));
  if constexpr (sizeof(T) == 2) {
    if (vec >= 8) return f(T{}, W{}, std::integral_constant<int, 8>{});
  }
  if constexpr (sizeof(T) <= 4) {
    if (vec >= 4) return f(T{}, W{}, std::integral_constant<int, 4>{});
  }
  if (vec >= 2) return f(T{}, W{}, std::integral_constant<int, 2>{});
  return f(T{}, W{}, std::integral_constant<int, 1>{});
}
template <typename F> void with_types(int32_t dtype, int32_t weights_dtype, int bytes, F &&f) {
  const bool f32 = weights_dtype == TBE_DTYPE_F32;
  switch (dtype) {
    case TBE_DTYPE_F32: return with_vector<float, float>(bytes, f);
    case TBE_DTYPE_F16: return f32 ? with_vector<_Float16, float>(bytes, f) : with_vector<_Float16, _Float16>(bytes, f);
    case TBE_DTYPE_BF16: return f32 ? with_vector<__bf16, float>(bytes, f) : with_vector<__bf16, __bf16>(bytes, f);
    default: return f32 ? with_vector<double, float>(bytes, f) : with_vector<double, double>(bytes, f);
  }
}

int check_rows(const char *name, int32_t dtype, int64_t tokens, int32_t choices, int32_t experts, int64_t D) {
  TBE_REQUIRE(float_dtype(dtype), "%s: bad dtype %d", name, dtype);
  TBE_REQUIRE(tokens >= 0, "%s: num_tokens must not be negative", name);
  TBE_REQUIRE(choices > 0, "%s: choices must be positive (got %d)", name, choices);
  TBE_REQUIRE(experts > 0 && experts <= kMaxExperts, "%s: num_experts must be 1 to %d (got %d)", name, kMaxExperts,
              experts);
  TBE_REQUIRE(tokens < INT32_MAX / choices, "%s: num_tokens * choices out of range", name);
  TBE_REQUIRE(D > 0 && D <= (1 << 24), "%s: D must be 1 to 2^24 (got %lld)", name, (long long)D);
  return TBE_OK;
}

}  // namespace
}  // namespace tbe

extern "C" uint64_t tbe_expert_plan_workspace_bytes(int64_t num_pairs, int32_t num_experts) {
  if (num_pairs < 0 || num_pairs >= INT32_MAX || num_experts < 1 || num_experts > tbe::kMaxExperts) return 0;
  return tbe::plan_regions(num_pairs, num_experts).total_bytes;
}

extern "C" int tbe_expert_plan(const void *expert_ids, int32_t id_bytes, int64_t num_pairs, int32_t num_experts,
                               int32_t *expert_offsets, int32_t *order, int32_t *places, void *workspace,
                               uint64_t workspace_bytes, void *stream) {
  using namespace tbe;
  const char *name = "tbe_expert_plan";
  TBE_REQUIRE(id_bytes == 4 || id_bytes == 8, "%s: expert ids of 4 or 8 bytes (got %d)", name, id_bytes);
  TBE_REQUIRE(num_pairs >= 0 && num_pairs < INT32_MAX, "%s: num_pairs out of range", name);
  TBE_REQUIRE(num_experts > 0 && num_experts <= kMaxExperts, "%s: num_experts must be 1 to %d (got %d)", name,
              kMaxExperts, num_experts);
  TBE_REQUIRE(expert_offsets && (num_pairs == 0 || (expert_ids && order && places)), "%s: null pointer argument", name);
  const PlanRegions p = plan_regions(num_pairs, num_experts);
  if (!workspace || workspace_bytes < p.total_bytes)
    return fail(TBE_ERR_WORKSPACE, "%s: workspace of %llu bytes needed, %llu given", name,
                (unsigned long long)p.total_bytes, (unsigned long long)workspace_bytes);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (id_bytes == 4) launch_plan<int32_t>(expert_ids, num_pairs, num_experts, p, workspace, expert_offsets, order, places, s);
  else launch_plan<int64_t>(expert_ids, num_pairs, num_experts, p, workspace, expert_offsets, order, places, s);
  return check_launch(name);
}

extern "C" int tbe_expert_dispatch(const void *tokens, int64_t token_stride, int32_t dtype, int64_t num_tokens,
                                   int32_t choices, int32_t num_experts, int64_t D, const int32_t *places,
                                   const int32_t *expert_offsets, void *rows, void *stream) {
  using namespace tbe;
  const char *name = "tbe_expert_dispatch";
  if (int rc = check_rows(name, dtype, num_tokens, choices, num_experts, D)) return rc;
  TBE_REQUIRE(token_stride >= 0, "%s: token_stride must not be negative", name);
  if (num_tokens == 0) return TBE_OK;
  TBE_REQUIRE(tokens && places && expert_offsets && rows, "%s: null pointer argument", name);
  const uint64_t size = element_size(dtype);
  const int bytes = vector_bytes(D * size | token_stride * size | address(tokens) | address(rows));
  TBE_REQUIRE(bytes >= static_cast<int>(size), "%s: misaligned pointer", name);
  dim3 grid;
  const RowTiles r = row_tiles(num_tokens, choices, D * size / bytes, &grid);
  TBE_REQUIRE(grid.y <= 65535, "%s: D out of range", name);
  const int64_t stride = token_stride * size / bytes;
  const int32_t *kept = expert_offsets + num_experts;
  hipStream_t s = static_cast<hipStream_t>(stream);
#define TBE_DISPATCH(U)                                                                                           \
  TBE_LAUNCH("expert_dispatch", s, (expert_dispatch_kernel<U, kRowIter>), grid, dim3(kBlockThreads),              \
             static_cast<const U *>(tokens), stride, places, kept, static_cast<U *>(rows), r)
  if (bytes == 16) { TBE_DISPATCH(uint4); }
  else if (bytes == 8) { TBE_DISPATCH(uint2); }
  else if (bytes == 4) { TBE_DISPATCH(uint32_t); }
  else { TBE_DISPATCH(uint16_t); }
#undef TBE_DISPATCH
  return check_launch(name);
}

extern "C" int tbe_expert_combine(const void *rows, int64_t row_stride, int32_t dtype, int64_t num_tokens,
                                  int32_t choices, int32_t num_experts, int64_t D, const int32_t *places,
                                  const int32_t *expert_offsets, const void *weights, int32_t weights_dtype,
                                  void *output, void *stream) {
  using namespace tbe;
  const char *name = "tbe_expert_combine";
  if (int rc = check_rows(name, dtype, num_tokens, choices, num_experts, D)) return rc;
  TBE_REQUIRE(row_stride >= 0, "%s: row_stride must not be negative", name);
  TBE_REQUIRE(!weights || weights_dtype == TBE_DTYPE_F32 || weights_dtype == dtype,
              "%s: weights must be fp32 or of the rows' type", name);
  if (num_tokens == 0) return TBE_OK;
  TBE_REQUIRE(rows && places && expert_offsets && output, "%s: null pointer argument", name);
  const uint64_t size = element_size(dtype);
  const int bytes = vector_bytes(D * size | row_stride * size | address(rows) | address(output));
  TBE_REQUIRE(bytes >= static_cast<int>(size), "%s: misaligned pointer", name);
  const CombineCall c{rows, row_stride, places, expert_offsets + num_experts, weights, num_tokens, choices, D,
                      static_cast<hipStream_t>(stream)};
  with_types(dtype, weights ? weights_dtype : dtype, bytes, [&](auto t, auto w, auto vec) {
    launch_combine<decltype(t), decltype(w), decltype(vec)::value>(c, output);
  });
  return check_launch(name);
}

extern "C" int tbe_expert_combine_backward(const void *grad_output, int64_t grad_stride, const void *rows,
                                           int64_t row_stride, int32_t dtype, int64_t num_tokens, int32_t choices,
                                           int32_t num_experts, int64_t D, const int32_t *places,
                                           const int32_t *expert_offsets, const void *weights, int32_t weights_dtype,
                                           void *grad_rows, void *grad_weights, void *stream) {
  using namespace tbe;
  const char *name = "tbe_expert_combine_backward";
  if (int rc = check_rows(name, dtype, num_tokens, choices, num_experts, D)) return rc;
  TBE_REQUIRE(row_stride >= 0 && grad_stride >= 0, "%s: strides must not be negative", name);
  TBE_REQUIRE(weights_dtype == TBE_DTYPE_F32 || weights_dtype == dtype,
              "%s: weights must be fp32 or of the rows' type", name);
  if (num_tokens == 0) return TBE_OK;
  TBE_REQUIRE(grad_output && places && expert_offsets && weights && (rows || !grad_weights) &&
                  (grad_rows || grad_weights),
              "%s: null pointer argument", name);
  const uint64_t size = element_size(dtype);
  const int bytes = vector_bytes(D * size | row_stride * size | grad_stride * size | address(rows) |
                                 address(grad_output) | address(grad_rows));
  TBE_REQUIRE(bytes >= static_cast<int>(size), "%s: misaligned pointer", name);
  const CombineCall c{rows, row_stride, places, expert_offsets + num_experts, weights, num_tokens, choices, D,
                      static_cast<hipStream_t>(stream)};
  with_types(dtype, weights_dtype, bytes, [&](auto t, auto w, auto vec) {
    launch_combine_backward<decltype(t), decltype(w), decltype(vec)::value>(c, grad_output, grad_stride, grad_rows,
                                                                          grad_weights);
  });
  return check_launch(name);
}
