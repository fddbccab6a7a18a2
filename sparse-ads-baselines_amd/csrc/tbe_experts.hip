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
// A stable counting sort by expert.  What bounds it is latency: the whole input is a few MB at most, so launches,
// barriers and chains of dependent steps are kept few.
//   up to kFewPairs pairs   one workgroup, one launch
//   few tiles               two launches: the counts of every tile of pairs; then every tile adds up the counts of
//                           the tiles before it (and of all) itself.  Tiles of one pair a thread while that
//                           reads few counts, of four beyond
//   more                    three: a launch in between turns an expert's counts into prefix sums over the tiles
// (Measured, 8 / 64 / 256 experts: 8192 pairs in one workgroup of eight pairs a thread 9.1 / 10.9 / 12.9 us, in two
// launches with four pairs a thread 9.1 / 9.7 / 10.6, with one 6.3 / 6.7 / 7.6; 262144 pairs in two launches 7.3 / 9.0 / 14.2
// with one, 9.9 / 11.7 / 14.1 with four; 524288 with four 10.5 / 12.1 / 15.6 in two, 12.1 / 13.9 / 15.7 in three, with one
// 13.1 / 15.1 / 18.0 in three.)
// A tile's pairs are ranked with wavefront ballots (all lanes of one expert are found with one ballot per bit of the
// expert's number).  Pairs inside a tile are numbered (wavefront, item, lane), which the ranking keeps, so the
// order is stable.
constexpr int kMaxExperts = TBE_MAX_EXPERTS;  // and one bin more for the dropped pairs
constexpr int kTinyPairs = kWave;       // one wavefront
constexpr int kFewPairs = 16 * kWave;
constexpr int kFewExperts = 1023;       // widest plan with 16 wavefronts a workgroup: their counters take 64 KB of LDS
constexpr int kManyItems = 4;           // pairs a thread of the larger tiles
// wavefronts of a workgroup that ranks with `bins` counters per wavefront
constexpr int tile_waves(int bins) { return bins <= 1024 ? 16 : 4; }
constexpr int tile_pairs(int bins, int items) { return tile_waves(bins) * kWave * items; }

template <typename I> __device__ __forceinline__ int bin_of(I expert, int E) {
  return (expert >= 0 && expert < E) ? static_cast<int>(expert) : E;
}

// counts[tile][bin] (DIRECT) or counts[bin][tile]
template <typename I, int ITEMS, int BINS, bool DIRECT>
__global__ __launch_bounds__(tile_waves(BINS) * kWave) void expert_count_kernel(
    const I *__restrict__ ids, int64_t n, int E, int64_t tiles, int32_t *__restrict__ counts) {
  constexpr int kThreads = tile_waves(BINS) * kWave;
  __shared__ int32_t s_count[BINS];
  const int64_t base = static_cast<int64_t>(blockIdx.x) * tile_pairs(BINS, ITEMS) + threadIdx.x;
  I id[ITEMS];
#pragma unroll
  for (int q = 0; q < ITEMS; ++q) id[q] = base + q * kThreads < n ? ids[base + q * kThreads] : I(0);
  for (int e = threadIdx.x; e <= E; e += kThreads) s_count[e] = 0;
  __syncthreads();
#pragma unroll
  for (int q = 0; q < ITEMS; ++q)
    if (base + q * kThreads < n) atomicAdd(&s_count[bin_of(id[q], E)], 1);
  __syncthreads();
  for (int e = threadIdx.x; e <= E; e += kThreads)
    counts[DIRECT ? blockIdx.x * static_cast<int64_t>(E + 1) + e : e * tiles + blockIdx.x] = s_count[e];
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

enum { kPlanSingle, kPlanDirect, kPlanScanned };

template <typename I, int WAVES, int ITEMS, int BINS, int MODE>
__global__ __launch_bounds__(WAVES *kWave) void expert_place_kernel(
    const I *__restrict__ ids, int64_t n, int E, int bits, const int32_t *__restrict__ counts,
    const int32_t *__restrict__ totals, int64_t tiles, int32_t *__restrict__ expert_offsets,
    int32_t *__restrict__ order, int32_t *__restrict__ places) {
  constexpr int kThreads = WAVES * kWave;
  __shared__ int32_t s_count[WAVES][BINS];
  __shared__ int32_t s_start[BINS];
  __shared__ int32_t s_before[MODE == kPlanDirect ? BINS : 1];
  __shared__ int32_t s_wave[WAVES];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = threadIdx.x >> 6;

  const int64_t base = (static_cast<int64_t>(blockIdx.x) * WAVES + wave) * (kWave * ITEMS) + lane;
  int key[ITEMS], rank[ITEMS];
#pragma unroll
  for (int q = 0; q < ITEMS; ++q) {
    const int64_t a = base + q * kWave;
    key[q] = a < n ? bin_of(ids[a], E) : -1;
  }
  for (int e = lane; e <= E; e += kWave) s_count[wave][e] = 0;
  if constexpr (MODE == kPlanDirect) {
    for (int e = threadIdx.x; e < BINS; e += kThreads) s_start[e] = s_before[e] = 0;
  }
  __syncthreads();
  if constexpr (MODE == kPlanDirect) {
    // threads are dealt to (bin, every parts-th tile); sums of whole numbers, whose order does not matter
    const int wide = E + 1 < kThreads ? E + 1 : kThreads;
    const int parts = kThreads / wide;
    const int part = threadIdx.x / wide;
    if (part < parts) {
      for (int e = threadIdx.x - part * wide; e <= E; e += wide) {
        int total = 0, before = 0;
#pragma unroll 8
        for (int t = part; t < static_cast<int>(tiles); t += parts) {
          const int c = counts[t * (E + 1) + e];
          total += c;
          before += t < static_cast<int>(blockIdx.x) ? c : 0;
        }
        atomicAdd(&s_start[e], total);
        atomicAdd(&s_before[e], before);
      }
    }
  }
#pragma unroll
  for (int q = 0; q < ITEMS; ++q) {
    rank[q] = 0;
    if (base - lane + q * kWave >= n) continue;  // (the whole wavefront)
    uint64_t same = __ballot(key[q] >= 0);
    for (int b = 0; b < bits; ++b) {
      const bool set = (key[q] >> b) & 1;
      const uint64_t vote = __ballot(set);
      same &= set ? vote : ~vote;
    }
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
      if constexpr (MODE == kPlanScanned) sum = totals[e];
    }
    if constexpr (MODE != kPlanDirect) s_start[e] = sum;
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
      if constexpr (MODE == kPlanDirect) first += s_before[e];
      if constexpr (MODE == kPlanScanned) first += counts[e * tiles + blockIdx.x];
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
// What bounds these kernels is memory: they move rows and do next to nothing with them.
//
// Rows are moved 16 bytes a lane, whatever their width and alignment: the memory system takes 16-byte accesses at
// any element's address, and the last vector of a row is the one that ENDS with the row (it overlaps the one
// before it; both write the same bytes).  Measured, 32768 tokens, 8 rows each, bf16, 2046 elements a row:
// combined in 189 us that way, in 372 us with the 4-byte vectors that would divide the row.  Rows of fewer than
// 16 bytes are moved element by element.
//
// One thread per (token, vector), numbered token after token, so that no lane idles for a row that is no power
// of two wide; a thread asks for the places of up to eight choices, then for their eight rows, before it
// uses the first.
//
// Row sets that the 256 MB memory-side cache cannot hold anyway are moved with streaming accesses (read, and, where a
// row fills whole cache lines, written): 1.07 GB of rows of 4 KB dispatched in 205 us instead of 227, combined
// in 184 instead of 218; but 67 MB dispatched and combined again 30.2 us without, 28.7 to 32.4 with them, and rows
// of 4092 bytes 299 us streamed instead of 271 (partly written lines).
struct RowMap {
  int64_t tokens;
  int64_t first;      // of this launch
  int32_t choices;
  int32_t vectors;    // of a row
  int32_t D;          // elements of a row (bytes for dispatch)
  uint32_t count;     // (token, vector) pairs of this launch, < 2^31
  uint32_t magic;     // i / vectors = (i * magic) >> shift for i < 2^31
  int32_t shift;
};

// A dropped pair's place lies behind the rows kept; so do places that are none.
__device__ __forceinline__ bool is_kept(int32_t place, int32_t kept) {
  return static_cast<uint32_t>(place) < static_cast<uint32_t>(kept);
}
__device__ __forceinline__ int32_t rows_kept(const int32_t *kept_rows, int64_t pairs) {
  return static_cast<int32_t>(max(int64_t{0}, min(static_cast<int64_t>(*kept_rows), pairs)));
}

// U: what is moved per lane (Words16, or one element of 2, 4 or 8 bytes)
template <typename U, bool STREAM>
__global__ __launch_bounds__(kBlockThreads) void expert_dispatch_kernel(
    const char *__restrict__ x, int64_t x_stride, const int32_t *__restrict__ places,
    const int32_t *__restrict__ kept_rows, char *__restrict__ rows, RowMap m) {
  constexpr int kAhead = 8;
  const uint32_t i = blockIdx.x * kBlockThreads + threadIdx.x;
  if (i >= m.count) return;
  const uint32_t t = static_cast<uint32_t>((static_cast<uint64_t>(i) * m.magic) >> m.shift);
  const int col = min(static_cast<int>((i - t * m.vectors) * sizeof(U)), m.D - static_cast<int>(sizeof(U)));
  const int64_t token = m.first + t;
  const uint32_t pairs = static_cast<uint32_t>(m.tokens * m.choices);
  const int32_t kept = *kept_rows;
  const U v = *reinterpret_cast<const U *>(x + token * x_stride + col);
  const int32_t *mine = places + token * m.choices;
  for (int j0 = 0; j0 < m.choices; j0 += kAhead) {
    int32_t place[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) place[j] = j0 + j < m.choices ? mine[j0 + j] : -1;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (static_cast<uint32_t>(place[j]) >= pairs) continue;
      U *to = reinterpret_cast<U *>(rows + static_cast<int64_t>(place[j]) * m.D + col);
      const U o = place[j] < kept ? v : U{};
      if constexpr (STREAM) __builtin_nontemporal_store(o, to);
      else *to = o;
    }
  }
}

template <typename T, typename W, int VEC, int AHEAD, bool STREAM>
__global__ __launch_bounds__(kBlockThreads) void expert_combine_kernel(
    const T *__restrict__ rows, int64_t row_stride, const int32_t *__restrict__ places,
    const int32_t *__restrict__ kept_rows, const W *__restrict__ weights, T *__restrict__ out, RowMap m) {
  using A = typename AccOf<T>::type;
  using P = Pack<T, VEC>;
  const uint32_t i = blockIdx.x * kBlockThreads + threadIdx.x;
  if (i >= m.count) return;
  const uint32_t t = static_cast<uint32_t>((static_cast<uint64_t>(i) * m.magic) >> m.shift);
  const int col = min(static_cast<int>(i - t * m.vectors) * VEC, m.D - VEC);
  const int64_t token = m.first + t;
  const int32_t kept = rows_kept(kept_rows, m.tokens * m.choices);
  A sum[VEC];
#pragma unroll
  for (int q = 0; q < VEC; ++q) sum[q] = A(0);
  for (int j0 = 0; j0 < m.choices; j0 += AHEAD) {
    int32_t place[AHEAD];
    A w[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int64_t a = token * m.choices + min(j0 + j, m.choices - 1);  // clamped: no branch per load
      place[j] = places[a];
      w[j] = weights ? static_cast<A>(weights[a]) : A(1);
    }
    P v[AHEAD];
    bool keep[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      keep[j] = j0 + j < m.choices && is_kept(place[j], kept);
      // (a dropped pair asks for row 0, which stays in the caches, and drops it: no branch between the loads)
      v[j] = load_pack<T, VEC, STREAM>(rows + (keep[j] ? place[j] : 0) * row_stride + col);
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
#pragma unroll
      for (int q = 0; q < VEC; ++q) sum[q] = keep[j] ? sum[q] + w[j] * static_cast<A>(v[j].v[q]) : sum[q];
    }
  }
  P o;
#pragma unroll
  for (int q = 0; q < VEC; ++q) o.v[q] = static_cast<T>(sum[q]);
  store_pack<T, VEC, false>(out + token * m.D + col, o);
}

// GROUP lanes per pair (a workgroup per pair for GROUP = 256): the pair's row is read once, its gradient written
// once; the token's gradient row comes from the caches for all pairs of the token but the first.  (One group per
// token, its gradient row held in registers over four choices at a time, took 485 us where this takes 447: 32768
// tokens, 8 rows of 2048 bf16 each.)  Without grad_weights the rows are not read, without grad_rows nothing is
// written to them.
template <typename T, typename W, int VEC, int GROUP, bool STREAM>
__global__ __launch_bounds__(kBlockThreads) void expert_combine_backward_kernel(
    const T *__restrict__ grad, int64_t grad_stride, const T *__restrict__ rows, int64_t row_stride,
    const int32_t *__restrict__ places, const int32_t *__restrict__ kept_rows, const W *__restrict__ weights,
    T *__restrict__ grad_rows, W *__restrict__ grad_weights, uint32_t pairs, int64_t slots, int choices, int vectors,
    int D, uint32_t magic, int shift) {
  using A = typename AccOf<T>::type;
  using P = Pack<T, VEC>;
  constexpr int kPairs = kBlockThreads / GROUP;
  __shared__ A s_part[kWavesPerBlock];
  const int sub = threadIdx.x % GROUP;
  const int32_t kept = rows_kept(kept_rows, pairs);
  // (a group leaves as a whole; with GROUP = 256 the workgroup does, so that its barriers are met by all or none)
  for (int64_t at = static_cast<int64_t>(blockIdx.x) * kPairs + threadIdx.x / GROUP; at < slots;
       at += static_cast<int64_t>(gridDim.x) * kPairs) {
    int64_t pair = at;
    uint32_t token;
    if constexpr (GROUP > kWave) {
      // workgroups are dealt to the XCDs in turn: a token's pairs go to every eighth one, so that its gradient row is
      // fetched into one L2 and not into as many as the token has choices
      const uint32_t q = static_cast<uint32_t>((static_cast<uint64_t>(at >> 3) * magic) >> shift);  // of 8 * choices
      const uint32_t j = static_cast<uint32_t>(at >> 3) - q * choices;
      token = q * kNumXcd + static_cast<uint32_t>(at & (kNumXcd - 1));
      pair = static_cast<int64_t>(token) * choices + j;
      if (pair >= pairs) continue;
    } else {
      token = static_cast<uint32_t>((static_cast<uint64_t>(pair) * magic) >> shift);
    }
    const int32_t place = places[pair];
    const bool keep = is_kept(place, kept);
    const bool write = grad_rows && static_cast<uint32_t>(place) < pairs;
    const A w = keep ? static_cast<A>(weights[pair]) : A(0);
    const T *g_row = grad + token * grad_stride;
    const T *row = rows + place * row_stride;
    T *to = grad_rows + static_cast<int64_t>(place) * D;
    A dot = A(0);
    for (int c = sub; c < vectors; c += GROUP) {
      const int col = min(c * VEC, D - VEC);
      const int seen = c * VEC - col;  // elements that the row's last vector shares with the one before it
      P g, v;
      if (keep) {
        g = load_pack<T, VEC, false>(g_row + col);
        if (grad_weights) v = load_pack<T, VEC, STREAM>(row + col);
      }
      if (write) {
        P o;
#pragma unroll
        for (int q = 0; q < VEC; ++q) o.v[q] = keep ? static_cast<T>(w * static_cast<A>(g.v[q])) : T(0);
        store_pack<T, VEC, false>(to + col, o);
      }
      if (grad_weights && keep) {
#pragma unroll
        for (int q = 0; q < VEC; ++q) {
          const A term = static_cast<A>(v.v[q]) * static_cast<A>(g.v[q]);
          dot += q >= seen ? term : A(0);
        }
      }
    }
    if (!grad_weights) continue;
#pragma unroll
    for (int d = 1; d < (GROUP < kWave ? GROUP : kWave); d <<= 1) dot += shfl_x(dot, d);
    if constexpr (GROUP > kWave) {
      __syncthreads();
      if ((threadIdx.x & (kWave - 1)) == 0) s_part[threadIdx.x >> 6] = dot;
      __syncthreads();
      dot = A(0);
#pragma unroll
      for (int q = 0; q < kWavesPerBlock; ++q) dot += s_part[q];
    }
    if (sub == 0) grad_weights[pair] = static_cast<W>(dot);
  }
}

// ------------------------------------------------------------------------------------ host
size_t element_size(int32_t dtype) {
  return dtype == TBE_DTYPE_F64 ? 8 : dtype == TBE_DTYPE_F32 ? 4 : 2;
}
bool float_dtype(int32_t dtype) {
  return dtype == TBE_DTYPE_F32 || dtype == TBE_DTYPE_F16 || dtype == TBE_DTYPE_F64 || dtype == TBE_DTYPE_BF16;
}

uint64_t address(const void *p) { return reinterpret_cast<uint64_t>(p); }

// Rows that the memory-side cache (256 MB) does not hold are streamed.
bool streams(int64_t pairs, int64_t row_bytes) { return pairs * row_bytes > (int64_t{256} << 20); }
// Streamed stores: only where they fill whole cache lines.
bool whole_lines(const void *base, int64_t row_bytes) { return ((address(base) | row_bytes) & 127) == 0; }

// i / d = (i * magic) >> shift for i < 2^31: magic = ceil(2^(31 + s) / d) with s = ceil(log2 d) fits 32 bits, and its
// error of less than d / 2^(31 + s) <= 2^-31 a unit of i stays below 1 / d for every such i.
void division_by(int64_t d, uint32_t *magic, int32_t *shift) {
  int log2 = 0;
  while ((int64_t{1} << log2) < d) ++log2;
  *shift = 31 + log2;
  *magic = static_cast<uint32_t>(((uint64_t{1} << *shift) + static_cast<uint64_t>(d) - 1) / static_cast<uint64_t>(d));
}

// f(map, grid) for every launch of at most 2^31 - 1 threads, each over whole tokens.
template <typename F> void for_row_maps(int64_t tokens, int32_t choices, int64_t vectors, int64_t D, F &&f) {
  RowMap m;
  m.tokens = tokens;
  m.choices = choices;
  m.vectors = static_cast<int32_t>(vectors);
  m.D = static_cast<int32_t>(D);
  division_by(vectors, &m.magic, &m.shift);
  const int64_t most = std::max<int64_t>(1, (INT32_MAX - kBlockThreads) / vectors);
  for (m.first = 0; m.first < tokens; m.first += most) {
    m.count = static_cast<uint32_t>(std::min(most, tokens - m.first) * vectors);
    f(m, dim3(static_cast<unsigned>(ceil_div(m.count, kBlockThreads))));
  }
}

constexpr int64_t kMaxGrid = 1 << 22;  // workgroups of a launch: grid times workgroup stays below 2^32 threads

int plan_bits(int32_t experts) {  // bits of the largest bin number, `experts`
  int bits = 0;
  while ((1 << bits) <= experts) ++bits;
  return bits;
}

// Bins of the kernels that serve `experts`, which has to stay below them.
int plan_bins(int32_t experts) { return experts < 256 ? 256 : experts < 1024 ? 1024 : 4096; }

struct PlanRegions {
  uint64_t totals, total_bytes;  // (the counts come first)
  int64_t tiles;                 // 0: one workgroup
  int items;                     // pairs a thread
  bool direct;                   // no launch for the prefix sums
};
PlanRegions plan_regions(int64_t pairs, int32_t experts) {
  PlanRegions p{0, 0, 0, 1, true};
  if (pairs <= kFewPairs && experts <= kFewExperts) return p;
  const int bins = plan_bins(experts);
  // tiles whose counts each of them may add up itself
  const auto few = [&](int64_t most) { return std::min<int64_t>(most, (1 << 16) / (experts + 1)); };
  p.tiles = std::max<int64_t>(1, ceil_div(pairs, tile_pairs(bins, 1)));
  if (p.tiles > few(256)) {
    p.items = kManyItems;
    p.tiles = ceil_div(pairs, tile_pairs(bins, kManyItems));
    p.direct = p.tiles <= few(128);
  }
  p.totals = align_up(static_cast<uint64_t>(p.tiles) * (experts + 1) * 4, 256);
  // (at least what the smaller tiles take, so that a workspace sized for a maximum serves every smaller batch)
  const uint64_t smaller = p.items > 1 ? align_up(static_cast<uint64_t>(few(256)) * (experts + 1) * 4, 256) : 0;
  p.total_bytes = std::max(p.totals, smaller) + align_up((experts + 1) * 4ull, 256);
  return p;
}

template <typename I, int BINS>
void launch_plan_tiles(const I *ids, int64_t pairs, int32_t experts, const PlanRegions &p, void *workspace,
                       int32_t *expert_offsets, int32_t *order, int32_t *places, hipStream_t s) {
  int32_t *counts = static_cast<int32_t *>(workspace);
  int32_t *totals = reinterpret_cast<int32_t *>(static_cast<char *>(workspace) + p.totals);
  const dim3 grid(static_cast<unsigned>(p.tiles)), block(tile_waves(BINS) * kWave);
#define TBE_PLAN_COUNT(ITEMS, DIRECT)                                                                             \
  TBE_LAUNCH("expert_count", s, (expert_count_kernel<I, ITEMS, BINS, DIRECT>), grid, block, ids, pairs, experts, \
             p.tiles, counts)
#define TBE_PLAN_PLACE(ITEMS, MODE)                                                                               \
  TBE_LAUNCH("expert_place", s, (expert_place_kernel<I, tile_waves(BINS), ITEMS, BINS, MODE>), grid, block, ids,  \
             pairs, experts, plan_bits(experts), counts, totals, p.tiles, expert_offsets, order, places)
  if (p.items == 1) {
    TBE_PLAN_COUNT(1, true);
    TBE_PLAN_PLACE(1, kPlanDirect);
  } else if (p.direct) {
    TBE_PLAN_COUNT(kManyItems, true);
    TBE_PLAN_PLACE(kManyItems, kPlanDirect);
  } else {
    TBE_PLAN_COUNT(kManyItems, false);
    TBE_LAUNCH("expert_scan", s, expert_scan_kernel, dim3(static_cast<unsigned>(ceil_div(experts + 1, kWavesPerBlock))),
               dim3(kBlockThreads), counts, p.tiles, experts, totals);
    TBE_PLAN_PLACE(kManyItems, kPlanScanned);
  }
#undef TBE_PLAN_COUNT
#undef TBE_PLAN_PLACE
}

template <typename I>
void launch_plan(const void *expert_ids, int64_t pairs, int32_t experts, const PlanRegions &p, void *workspace,
                 int32_t *expert_offsets, int32_t *order, int32_t *places, hipStream_t s) {
  const I *ids = static_cast<const I *>(expert_ids);
  if (p.tiles == 0) {
    const int32_t *none = nullptr;
#define TBE_PLAN_FEW(WAVES, BINS)                                                                                \
  TBE_LAUNCH("expert_place", s, (expert_place_kernel<I, WAVES, 1, BINS, kPlanSingle>), dim3(1),                  \
             dim3(WAVES *kWave), ids, pairs, experts, plan_bits(experts), none, none, int64_t{1},                \
             expert_offsets, order, places)
    if (experts < 256 && pairs <= kTinyPairs) { TBE_PLAN_FEW(1, 256); }
    else if (experts < 256) { TBE_PLAN_FEW(16, 256); }
    else { TBE_PLAN_FEW(16, 1024); }
#undef TBE_PLAN_FEW
    return;
  }
  switch (plan_bins(experts)) {
    case 256: return launch_plan_tiles<I, 256>(ids, pairs, experts, p, workspace, expert_offsets, order, places, s);
    case 1024: return launch_plan_tiles<I, 1024>(ids, pairs, experts, p, workspace, expert_offsets, order, places, s);
    default: return launch_plan_tiles<I, 4096>(ids, pairs, experts, p, workspace, expert_offsets, order, places, s);
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

template <typename T, typename W, int VEC, int AHEAD, bool STREAM>
void launch_combine_as(const CombineCall &c, void *output) {
  for_row_maps(c.tokens, c.choices, ceil_div(c.D, VEC), c.D, [&](const RowMap &m, dim3 grid) {
    TBE_LAUNCH("expert_combine", c.stream, (expert_combine_kernel<T, W, VEC, AHEAD, STREAM>), grid, dim3(kBlockThreads),
               static_cast<const T *>(c.rows), c.row_stride, c.places, c.kept, static_cast<const W *>(c.weights),
               static_cast<T *>(output), m);
  });
}

template <typename T, typename W, int VEC> void launch_combine(const CombineCall &c, void *output) {
  if constexpr (VEC == 1) {
    launch_combine_as<T, W, 1, 4, false>(c, output);
  } else {
    const bool stream = streams(c.tokens * c.choices, c.D * sizeof(T));
#define TBE_COMBINE(AHEAD)                                                          \
  do {                                                                              \
    if (stream) launch_combine_as<T, W, VEC, AHEAD, true>(c, output);               \
    else launch_combine_as<T, W, VEC, AHEAD, false>(c, output);                     \
  } while (0)
    // as many rows ahead as a token has, in steps: a row ahead that is not there costs its request.  (2, 4 and 8 ahead,
    // 32768 tokens, rows of 2048 bf16, one choice 43, 48 and 76 us, two 77, 77 and 96, three 93, 88 and 115, four 112, 111
    // and 129, six 162, 167 and 163, eight 214, 211 and 211; 512 tokens, rows of 1024, eight choices 3.7, 3.2 and 3.2.)
    if (c.choices <= 2) TBE_COMBINE(2);
    else if (c.choices <= 4) TBE_COMBINE(4);
    else TBE_COMBINE(8);
#undef TBE_COMBINE
  }
}

constexpr int kWavefrontVectors = 352;  // widest row of a wavefront, see below
template <typename T, typename W, int VEC, bool STREAM>
void launch_combine_backward_as(const CombineCall &c, const void *grad, int64_t grad_stride, void *grad_rows,
                                void *grad_weights) {
  const int vectors = static_cast<int>(ceil_div(c.D, VEC));
  const int64_t pairs = c.tokens * c.choices;
  uint32_t magic;
  int shift;
  division_by(c.choices, &magic, &shift);
  int64_t slots = pairs;
#define TBE_COMBINE_BACKWARD(GROUP)                                                                                \
  TBE_LAUNCH("expert_combine_backward", c.stream, (expert_combine_backward_kernel<T, W, VEC, GROUP, STREAM>),      \
             dim3(static_cast<unsigned>(std::min(ceil_div(slots, kBlockThreads / GROUP), kMaxGrid))),              \
             dim3(kBlockThreads), static_cast<const T *>(grad), grad_stride, static_cast<const T *>(c.rows),       \
             c.row_stride, c.places, c.kept, static_cast<const W *>(c.weights), static_cast<T *>(grad_rows),       \
             static_cast<W *>(grad_weights), static_cast<uint32_t>(pairs), slots, c.choices, vectors,              \
             static_cast<int>(c.D), magic, shift)
  // The narrowest group that holds a row, a workgroup for rows of more than 352 vectors.  (A wavefront and a workgroup a
  // row: 16384 tokens, 4 rows each, of 192 vectors 89 and 116 us, 257: 146 and 159, 288: 139 and 153, 352: 171 and 174,
  // 384: 184 and 182, 448: 216 and 211, 512: 262 and 236, 1024: 508 and 493; 1024 tokens, 257: 8.4 and 9.4, 352: 10.4 and
  // 11.4, 512: 14 and 16, 768: 19.5 and 19.0; 32 rows alone, which leave the chip empty, 257: 4.6 and 3.4.)
  if (vectors <= 8) { TBE_COMBINE_BACKWARD(8); }
  else if (vectors <= 16) { TBE_COMBINE_BACKWARD(16); }
  else if (vectors <= 32) { TBE_COMBINE_BACKWARD(32); }
  else if (vectors <= kWavefrontVectors) { TBE_COMBINE_BACKWARD(64); }
  else {
    slots = ceil_div(c.tokens, kNumXcd) * kNumXcd * c.choices;
    TBE_COMBINE_BACKWARD(256);
  }
#undef TBE_COMBINE_BACKWARD
}

// (Streamed reads of the rows beyond what the memory-side cache holds, plain ones and these: 320 MB of rows of 2048 bf16
// 155 and 147 us, 1 GB 472 and 469; 732 MB of rows of 64 fp32 431 and 419.)
template <typename T, typename W, int VEC>
void launch_combine_backward(const CombineCall &c, const void *grad, int64_t grad_stride, void *grad_rows,
                             void *grad_weights) {
  if constexpr (VEC > 1) {
    if (streams(c.tokens * c.choices, c.D * sizeof(T)))
      return launch_combine_backward_as<T, W, VEC, true>(c, grad, grad_stride, grad_rows, grad_weights);
  }
  launch_combine_backward_as<T, W, VEC, false>(c, grad, grad_stride, grad_rows, grad_weights);
}

// f(T{}, W{}, VEC) for the types of a call: 16-byte vectors, single elements for rows that hold no vector
template <typename T, typename W, typename F> void with_vector(int64_t D, F &&f) {
  constexpr int kVec = 16 / static_cast<int>(sizeof(T));
  if (D >= kVec) return f(T{}, W{}, std::integral_constant<int, kVec>{});
  return f(T{}, W{}, std::integral_constant<int, 1>{});
}
template <typename F> void with_types(int32_t dtype, int32_t weights_dtype, int64_t D, F &&f) {
  const bool f32 = weights_dtype == TBE_DTYPE_F32;
  switch (dtype) {
    case TBE_DTYPE_F32: return with_vector<float, float>(D, f);
    case TBE_DTYPE_F16: return f32 ? with_vector<_Float16, float>(D, f) : with_vector<_Float16, _Float16>(D, f);
    case TBE_DTYPE_BF16: return f32 ? with_vector<__bf16, float>(D, f) : with_vector<__bf16, __bf16>(D, f);
    default: return f32 ? with_vector<double, float>(D, f) : with_vector<double, double>(D, f);
  }
}

// (addresses need the alignment of an element, whatever the vectors')
bool aligned(const void *p, int32_t dtype) { return address(p) % element_size(dtype) == 0; }

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
  if (p.total_bytes > 0 && (!workspace || workspace_bytes < p.total_bytes))
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
  TBE_REQUIRE(aligned(tokens, dtype) && aligned(rows, dtype), "%s: misaligned pointer", name);
  const int64_t size = static_cast<int64_t>(element_size(dtype));
  const int64_t row_bytes = D * size;
  const int64_t unit = row_bytes >= 16 ? 16 : size;
  const bool stream_out = streams(num_tokens * choices, row_bytes) && whole_lines(rows, row_bytes);
  const int32_t *kept = expert_offsets + num_experts;
  hipStream_t s = static_cast<hipStream_t>(stream);
#define TBE_DISPATCH(U, STREAM)                                                                                   \
  TBE_LAUNCH("expert_dispatch", s, (expert_dispatch_kernel<U, STREAM>), grid, dim3(kBlockThreads),                \
             static_cast<const char *>(tokens), token_stride * size, places, kept, static_cast<char *>(rows), m)
  for_row_maps(num_tokens, choices, ceil_div(row_bytes, unit), row_bytes, [&](const RowMap &m, dim3 grid) {
    if (unit == 16 && stream_out) { TBE_DISPATCH(Words16, true); }
    else if (unit == 16) { TBE_DISPATCH(Words16, false); }
    else if (unit == 8) { TBE_DISPATCH(uint64_t, false); }
    else if (unit == 4) { TBE_DISPATCH(uint32_t, false); }
    else { TBE_DISPATCH(uint16_t, false); }
  });
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
  TBE_REQUIRE(aligned(rows, dtype) && aligned(output, dtype), "%s: misaligned pointer", name);
  const CombineCall c{rows, row_stride, places, expert_offsets + num_experts, weights, num_tokens, choices, D,
                      static_cast<hipStream_t>(stream)};
  with_types(dtype, weights ? weights_dtype : dtype, D, [&](auto t, auto w, auto vec) {
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
  TBE_REQUIRE(aligned(grad_output, dtype) && aligned(rows, dtype) && aligned(grad_rows, dtype),
              "%s: misaligned pointer", name);
  const CombineCall c{rows, row_stride, places, expert_offsets + num_experts, weights, num_tokens, choices, D,
                      static_cast<hipStream_t>(stream)};
  with_types(dtype, weights_dtype, D, [&](auto t, auto w, auto vec) {
    launch_combine_backward<decltype(t), decltype(w), decltype(vec)::value>(c, grad_output, grad_stride, grad_rows,
                                                                          grad_weights);
  });
  return check_launch(name);
}
