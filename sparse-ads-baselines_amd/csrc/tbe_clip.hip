// The global norm of gradients and clipping to it, for gfx950:
//   norm    N = sqrt(sum over all tensors and elements of g^2)
//   scaled  g * min(1, max_norm / (N + 1e-6)); a norm that is no number makes every element one, and an infinite one
//           under an infinite limit scales nothing
// and, for a sorted batch of embedding lookups, the norm of the tables' exact gradient, which has one row
// per distinct index and is never stored:
//   N = sqrt(sum over rows r of || sum over lookups p of row r of (w_p *) g[bag(p)] ||^2)
// Squares are added up in 64 bits: no value that a 32-bit float holds overflows there, and the memory system,
// not the vector ALU, stays what these passes wait for.  Every sum has one fixed order (no atomics), so two runs
// of the same lists are bit-identical.

#include <algorithm>
#include <new>
#include <type_traits>
#include <vector>

#include "tbe_stages.h"

namespace tbe {
namespace {

// ------------------------------------------------------------------------------ lists of tensors
// A launch takes a list of tensors of one type by kernel argument (under 4 KB), cut into chunks of kChunkVectors
// 16-byte vectors.  Chunks begin at the first 16-byte boundary of the tensor that is written (read, for a sum): the
// elements before it, fewer than a vector, belong to the first chunk, those behind the last whole vector to the
// last one.  The other tensor of a pair may lie at any element's address, which the memory system takes.
// An entry is 12 bytes, 20 with an output of its own: a launch takes 320 tensors, or 192.
constexpr int kChunkVectors = 1024;  // 16 KB
constexpr int kListTensors = 320;    // read, or scaled in place
constexpr int kPairTensors = 192;    // with outputs of their own
constexpr int kShortList = kWave;    // calls of up to so many tensors pass short lists, which a launch copies
constexpr int kNoBoundary = 0x8000;
template <int N, bool PAIRS> struct TensorList {
  static constexpr int kTensors = N;
  static constexpr bool kPairs = PAIRS;
  uint64_t src[N];                  // address, and above its 48 bits the last chunk's `count`, or kNoBoundary | elements
  uint64_t dst[PAIRS ? N : 1];
  int32_t chunk_end[N];             // running number of chunks; INT32_MAX behind the last tensor
  int32_t chunks;
};
using ReadList = TensorList<kListTensors, false>;
using PairList = TensorList<kPairTensors, true>;
using ShortReadList = TensorList<kShortList, false>;
using ShortPairList = TensorList<kShortList, true>;
static_assert(sizeof(ReadList) < 3900 && sizeof(PairList) < 3900, "kernel arguments");

// The tensor that a chunk belongs to: every lane looks at some of the ends.
template <typename L> __device__ __forceinline__ int tensor_of_chunk(const L &list, int chunk) {
  const int lane = threadIdx.x & (kWave - 1);
  int before = 0;
#pragma unroll
  for (int i = 0; i < L::kTensors; i += kWave) before += __popcll(__ballot(list.chunk_end[i + lane] <= chunk));
  return __builtin_amdgcn_readfirstlane(before);
}

template <typename T> struct Piece {
  const T *src;   // of the chunk's first vector
  T *dst;
  int count;      // elements from there on
  int head;       // elements before it that belong to the chunk
};
// (elements before the first 16-byte boundary)
template <typename T> __host__ __device__ __forceinline__ int head_of(uint64_t address) {
  return static_cast<int>(((16 - (address & 15)) & 15) / sizeof(T));
}
template <typename T, typename L> __device__ __forceinline__ Piece<T> piece_of_chunk(const L &list, int chunk) {
  constexpr int kElements = kChunkVectors * (16 / static_cast<int>(sizeof(T)));
  const int t = tensor_of_chunk(list, chunk);
  const uint64_t packed = list.src[t];
  const uint64_t src = packed & ((uint64_t{1} << 48) - 1);
  const uint64_t dst = L::kPairs ? list.dst[L::kPairs ? t : 0] : src;
  const int in_tensor = chunk - (t ? list.chunk_end[t - 1] : 0);
  const int last = static_cast<int>(packed >> 48);
  Piece<T> p;
  int64_t first;
  if (last & kNoBoundary) {  // the whole tensor lies before the boundary
    p.head = last & ~kNoBoundary;
    p.count = 0;
    first = p.head;
  } else {
    const int head = head_of<T>(dst);
    p.head = in_tensor == 0 ? head : 0;
    p.count = chunk + 1 == list.chunk_end[t] ? last : kElements;
    first = head + static_cast<int64_t>(in_tensor) * kElements;
  }
  p.src = reinterpret_cast<const T *>(src) + first;
  p.dst = reinterpret_cast<T *>(dst) + first;
  return p;
}

__device__ __forceinline__ double square(double x) { return x * x; }

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) v += shfl_x(v, m);
  return v;
}
// Sum over the workgroup, in every thread.
template <int WAVES> __device__ __forceinline__ double block_sum(double v) {
  __shared__ double s_wave[WAVES];
  v = wave_sum(v);
  if ((threadIdx.x & (kWave - 1)) == 0) s_wave[threadIdx.x >> 6] = v;
  __syncthreads();
  double sum = 0.0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) sum += s_wave[w];
  return sum;
}

// This thread's squares of a chunk that THREADS threads share; AHEAD vectors are requested before the first is used.
template <typename T, int THREADS, int AHEAD, bool STREAM>
__device__ __forceinline__ double chunk_squares(const Piece<T> &p, int thread) {
  constexpr int kVec = 16 / sizeof(T);
  const T *src = p.src;
  const int vectors = p.count / kVec;
  double sum = 0.0;
  for (int i0 = thread; i0 < vectors; i0 += THREADS * AHEAD) {
    Pack<T, kVec> x[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int i = i0 + u * THREADS;
      x[u] = load_pack<T, kVec, STREAM>(src + min(i, vectors - 1) * kVec);  // clamped: no branch per load
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (i0 + u * THREADS >= vectors) break;
#pragma unroll
      for (int q = 0; q < kVec; ++q) sum += square(static_cast<double>(x[u].v[q]));
    }
  }
  const int rest = vectors * kVec + thread;
  if (rest < p.count) sum += square(static_cast<double>(src[rest]));
  if (thread < p.head) sum += square(static_cast<double>(src[thread - p.head]));
  return sum;
}

// dst = src * scale for a chunk that THREADS threads share: products in 32 bits for the types of up to 32, rounded
// once more for those of 16.
template <typename T, int THREADS, int AHEAD, bool STREAM_IN, bool STREAM_OUT>
__device__ __forceinline__ void chunk_scaled(const Piece<T> &p, typename AccOf<T>::type scale, int thread) {
  using A = typename AccOf<T>::type;
  constexpr int kVec = 16 / sizeof(T);
  const T *src = p.src;
  T *dst = p.dst;
  const int vectors = p.count / kVec;
  for (int i0 = thread; i0 < vectors; i0 += THREADS * AHEAD) {
    Pack<T, kVec> x[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      x[u] = load_pack<T, kVec, STREAM_IN>(src + min(i0 + u * THREADS, vectors - 1) * kVec);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int i = i0 + u * THREADS;
      if (i >= vectors) break;
#pragma unroll
      for (int q = 0; q < kVec; ++q) x[u].v[q] = static_cast<T>(static_cast<A>(x[u].v[q]) * scale);
      store_pack<T, kVec, STREAM_OUT>(dst + i * kVec, x[u]);
    }
  }
  const int rest = vectors * kVec + thread;
  if (rest < p.count) dst[rest] = static_cast<T>(static_cast<A>(src[rest]) * scale);
  if (thread < p.head) dst[thread - p.head] = static_cast<T>(static_cast<A>(src[thread - p.head]) * scale);
}

__device__ __forceinline__ void store_norm(void *norm, int f64, double value) {
  if (f64) *static_cast<double *>(norm) = value;
  else *static_cast<float *>(norm) = static_cast<float>(value);
}

// The norm is rounded once, to the type it is stored in; the scale is formed in 64 bits from it.
__device__ __forceinline__ double clip_scale(double norm, double max_norm) {
  const double scale = max_norm / (norm + 1e-6);
  // (no limit: nothing is scaled, infinities included)
  return scale > 1.0 || (isinf(max_norm) && isinf(norm)) ? 1.0 : scale;
}

// A grid that fills the chip once walks the chunks; a partial sum per workgroup.
template <typename T, typename L, bool STREAM>
__global__ __launch_bounds__(kBlockThreads) void square_sum_kernel(L list, double *__restrict__ partial) {
  double sum = 0.0;
  for (int chunk = blockIdx.x; chunk < list.chunks; chunk += gridDim.x)
    sum += chunk_squares<T, kBlockThreads, 4, STREAM>(piece_of_chunk<T>(list, chunk), threadIdx.x);
  sum = block_sum<kWavesPerBlock>(sum);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

constexpr int kWideThreads = 1024;
__global__ __launch_bounds__(kWideThreads) void norm_finish_kernel(const double *__restrict__ partial, int64_t count,
                                                                  void *norm, int f64) {
  double sum = 0.0;
  for (int64_t i = threadIdx.x; i < count; i += kWideThreads) sum += partial[i];
  sum = block_sum<kWideThreads / kWave>(sum);
  if (threadIdx.x == 0) store_norm(norm, f64, sqrt(sum));
}

// A vector per thread and chunk (reading and writing want many short requests: 300 tensors of 300 M fp32 elements in all,
// measured and scaled in place, 569 us, with four vectors a thread of smaller workgroups 602), a workgroup walking every
// kScaleBlocks-th chunk.  The grid is what a call within the limit pays for, in place: 600 M bf16 elements take 196 us with
// up to 16384 workgroups, 246 with one per chunk, 183 with 2048, 177 for the norm alone; scaled into others they take 568,
// 579 and 601.
template <typename T, typename L, bool STREAM_IN, bool STREAM_OUT>
__global__ __launch_bounds__(kWideThreads) void scale_kernel(L list, const void *norm, int f64, double max_norm) {
  using A = typename AccOf<T>::type;
  const double n = f64 ? *static_cast<const double *>(norm) : static_cast<double>(*static_cast<const float *>(norm));
  const A scale = static_cast<A>(clip_scale(n, max_norm));
  if (!L::kPairs && scale == A(1)) return;  // in place and within the limit: nothing changes
  for (int chunk = blockIdx.x; chunk < list.chunks; chunk += gridDim.x)
    chunk_scaled<T, kWideThreads, 1, STREAM_IN, STREAM_OUT>(piece_of_chunk<T>(list, chunk), scale, threadIdx.x);
}

// The same where the caches hold the gradients: every workgroup adds up the partial sums itself, in the order of
// norm_finish_kernel, and the first one writes the norm, in place of a launch in between.  Two workgroups per compute
// unit, which all run at once, walk the chunks.  (fp32, scaled in place, this way and with that launch: 4 M elements
// 11.7 and 13.1 us, 12 M 26.7 and 28.5, 60 M 107.9 and 105.5; within the limit 4 M 7.9 and 10.6, 12 M 13.7 and 16.4, 60 M
// 39.9 and 53.2.)
constexpr int kJoinedBlocks = 512;
constexpr int64_t kJoinedSums = 4 * kWideThreads;  // (each of a long list of lists' launches would add up all of them)
template <typename T, typename L, bool STREAM_OUT>
__global__ __launch_bounds__(kWideThreads) void scale_joined_kernel(L list, const double *__restrict__ partial,
                                                                    int64_t count, void *norm, int f64, double max_norm) {
  using A = typename AccOf<T>::type;
  double sum = 0.0;
  for (int64_t i = threadIdx.x; i < count; i += kWideThreads) sum += partial[i];
  const double root = sqrt(block_sum<kWideThreads / kWave>(sum));
  const double n = f64 ? root : static_cast<double>(static_cast<float>(root));
  if (blockIdx.x == 0 && threadIdx.x == 0) store_norm(norm, f64, root);
  const A scale = static_cast<A>(clip_scale(n, max_norm));
  if (!L::kPairs && scale == A(1)) return;
  for (int chunk = blockIdx.x; chunk < list.chunks; chunk += gridDim.x)
    chunk_scaled<T, kWideThreads, 1, false, STREAM_OUT>(piece_of_chunk<T>(list, chunk), scale, threadIdx.x);
}

// Few chunks: norm and scaling in one workgroup, two wavefronts per chunk (8 fp32 chunks: 4.2 us a pass, 5.0 with one
// wavefront each, 4.6 with four).  In place, where most passes have nothing to write, it serves up to three chunks a
// pair of wavefronts, with outputs of their own one: 11 chunks within the limit 5.5 us, 7.4 in two launches, 24 chunks
// 7.4 and 7.5, 32 chunks 9.0 and 7.4; written 8 chunks 6.9 and 7.5, 11 chunks 8.8 and 7.6.
constexpr int kFewChunks = 24;
constexpr int kFewWritten = 8;
template <typename T, typename L>
__global__ __launch_bounds__(kWideThreads) void clip_few_kernel(L list, int scaled, void *norm, int f64,
                                                                double max_norm) {
  using A = typename AccOf<T>::type;
  constexpr int kThreads = 2 * kWave;
  constexpr int kGroups = kWideThreads / kThreads;
  const int thread = threadIdx.x % kThreads;
  const int group = threadIdx.x / kThreads;
  double sum = 0.0;
  for (int chunk = group; chunk < list.chunks; chunk += kGroups)
    sum += chunk_squares<T, kThreads, 8, false>(piece_of_chunk<T>(list, chunk), thread);
  sum = block_sum<kWideThreads / kWave>(sum);
  const double root = sqrt(sum);
  if (threadIdx.x == 0) store_norm(norm, f64, root);
  if (!scaled) return;
  const double n = f64 ? root : static_cast<double>(static_cast<float>(root));
  const A scale = static_cast<A>(clip_scale(n, max_norm));
  if (!L::kPairs && scale == A(1)) return;
  for (int chunk = group; chunk < list.chunks; chunk += kGroups)
    chunk_scaled<T, kThreads, 8, false, false>(piece_of_chunk<T>(list, chunk), scale, thread);
}

// --------------------------------------------------------------------- norm of the tables' gradient
// One workgroup per tile of kTile consecutive sorted positions and column block of up to 64 vectors.  Its lane groups (one
// 16-byte vector of the row per lane) each walk a run of consecutive positions, adding the gradient rows of one
// segment and squaring the sum where the segment ends: a lane squares its own columns, so that no sum over lanes is
// needed before the very end.  A segment that crosses runs is joined by the group in whose run it begins: what the
// runs behind it have left of it is in LDS.  One that crosses tiles leaves partial rows (row 2 * tile: what ends in the
// tile or runs through it, row 2 * tile + 1: what begins in it and goes on), which the next launch joins from
// the tile where the segment begins.
// What bounds it is the gather of the gradient rows from the caches (5.2 M lookups of 512 bytes); the workgroups of an
// XCD walk one eighth of the positions in order, so that they work on one table's gradient rows, which its L2 holds.
constexpr int kTile = 256;
static_assert(kTile == kBlockThreads, "a thread per position");

template <typename T, int VEC, bool WEIGHTED>
__global__ __launch_bounds__(kBlockThreads) void table_norm_tiles_kernel(
    const T *__restrict__ grad, const T *__restrict__ psw, const int32_t *__restrict__ positions_sorted,
    const int32_t *__restrict__ grad_rows, const int32_t *__restrict__ segment_ids, int64_t n, int D,
    int64_t num_tiles, int64_t tiles_per_xcd, typename AccOf<T>::type *__restrict__ partial_rows,
    double *__restrict__ tile_sums) {
  using V = RowVec<T, VEC>;
  using A = typename V::A;
  using R = typename V::R;
  constexpr int kAhead = 8;
  constexpr int kEnds = INT32_MIN;
  __shared__ int32_t s_row[kTile];  // gradient row of every position, kEnds or'ed in where a segment ends
  __shared__ A s_weight[WEIGHTED ? kTile : 1];
  __shared__ A s_head[kBlockThreads][VEC];
  __shared__ int32_t s_through[kTile];  // whether one segment runs through a whole run
  const int64_t tile = xcd_contiguous(blockIdx.x, tiles_per_xcd);
  if (tile >= num_tiles) return;
  const int64_t p0 = tile * kTile;
  const int len = static_cast<int>(min(n - p0, static_cast<int64_t>(kTile)));
  {
    const int64_t p = min(p0 + threadIdx.x, n - 1);
    const int pos = positions_sorted[p];
    const bool ends = p + 1 == n || segment_ids[p] != segment_ids[min(p + 1, n - 1)];
    s_row[threadIdx.x] = grad_rows[pos] | (ends ? kEnds : 0);
    if constexpr (WEIGHTED) s_weight[threadIdx.x] = to_acc(psw[pos]);
  }
  const bool open_before = p0 > 0 && segment_ids[p0 - 1] == segment_ids[p0];
  __syncthreads();

  const int vectors = D / VEC - blockIdx.y * kWave;  // of the columns from this block's first on
  const int chunks = vectors < kWave ? vectors : kWave;
  const int groups = kWave / chunks;                 // of a wavefront
  const int lane = threadIdx.x & (kWave - 1);
  const int in_wave = lane / chunks;
  const int c = lane - in_wave * chunks;
  const int runs = groups * kWavesPerBlock;
  const int run = (len + runs - 1) / runs;
  const int r = (threadIdx.x >> 6) * groups + in_wave;
  const int64_t col = (static_cast<int64_t>(blockIdx.y) * kWave + c) * VEC;
  const int begin = min(r * run, len), end = min(begin + run, len);
  const bool active = in_wave < groups && begin < end;
  // whether the position before b (behind which a run begins) belongs to the segment of position b
  const auto opens = [&](int b) { return b == 0 ? open_before : s_row[b - 1] >= 0; };

  double squares = 0.0;
  V G;
  G.zero();
  bool head = active && opens(begin);  // the segment being added began before this run
  const auto square = [&](const A(&g)[VEC]) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) squares += static_cast<double>(g[k]) * static_cast<double>(g[k]);
  };
  const auto leave_head = [&] {
#pragma unroll
    for (int k = 0; k < VEC; ++k) s_head[r * chunks + c][k] = G.v[k];
  };
  if (active) {
    for (int i0 = begin; i0 < end; i0 += kAhead) {
      R raw[kAhead];
      int word[kAhead];
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        word[q] = s_row[min(i0 + q, end - 1)];  // clamped, not predicated: no branch per load
        raw[q] = V::load_raw(grad + static_cast<int64_t>(word[q] & ~kEnds) * D + col);
      }
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        if (i0 + q >= end) break;
        V x;
        x.unpack(raw[q]);
        A w = A(1);
        if constexpr (WEIGHTED) w = s_weight[i0 + q];
#pragma unroll
        for (int k = 0; k < VEC; ++k) G.v[k] += WEIGHTED ? x.v[k] * w : x.v[k];
        if (word[q] < 0) {
          if (head) leave_head();
          else square(G.v);
          head = false;
          G.zero();
        }
      }
    }
    if (head) leave_head();
    if (c == 0) s_through[r] = head;
  }
  __syncthreads();
  // The groups with a segment to join: the one in whose run it begins, and the first one for what comes from before.
  const bool begins_here = active && !head && s_row[end - 1] >= 0;
  for (int from = 0; from < 2; ++from) {
    const bool joins = from == 0 ? begins_here : (active && r == 0 && open_before);
    if (!joins) continue;
    if (from == 1) G.zero();
    bool open = true;
    int t = from == 0 ? r + 1 : 0;
    for (; open && t * run < len; ++t) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) G.v[k] += s_head[t * chunks + c][k];
      open = s_through[t];
    }
    if (from == 0 && !open) {
      square(G.v);
    } else {
      A *rows = partial_rows + (2 * tile + (from == 0 ? 1 : 0)) * D + col;
#pragma unroll
      for (int k = 0; k < VEC; ++k) rows[k] = G.v[k];
    }
  }
  squares = block_sum<kWavesPerBlock>(squares);
  if (threadIdx.x == 0) tile_sums[tile * gridDim.y + blockIdx.y] = squares;
}

// The partial rows first, first + step, ... up to `last` of the segment that begins in `tile`, for this lane's columns;
// eight are requested before the first is added.
template <int VEC, typename A>
__device__ __forceinline__ void add_partial_rows(const A *__restrict__ partial_rows, int D, int64_t tile, int64_t first,
                                                 int64_t step, int64_t last, int64_t col, A (&sum)[VEC]) {
  constexpr int kAhead = 8;
  for (int64_t t0 = first; t0 <= last; t0 += step * kAhead) {
    A part[kAhead][VEC];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int64_t t = min(t0 + a * step, last);
      const A *row = partial_rows + (2 * t + (t == tile ? 1 : 0)) * D + col;
#pragma unroll
      for (int k = 0; k < VEC; ++k) part[a][k] = row[k];
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const bool real = t0 + a * step <= last;
#pragma unroll
      for (int k = 0; k < VEC; ++k) sum[k] += real ? part[a][k] : A(0);
    }
  }
}

// The segments that cross tiles: a wavefront per tile, working where one begins and goes on, adds the
// partial rows of the tiles up to its end; a workgroup's wavefronts then add up their tiles' squares.  Segments of more
// than kLongTiles tiles are left to the workgroups behind `joins`, one for every kLongTiles tiles: it joins the
// segment whose first such tile is its own.  (One row looked up 5.2 million times: 201 us, 741 with a wavefront.)
constexpr int kLongTiles = 64;
template <typename T, int VEC>
__global__ __launch_bounds__(kBlockThreads) void table_norm_join_kernel(
    const int32_t *__restrict__ segment_ids, const int32_t *__restrict__ segment_starts, int64_t n, int D,
    int64_t num_tiles, int joins, const typename AccOf<T>::type *__restrict__ partial_rows,
    const double *__restrict__ tile_sums, int column_blocks, double *__restrict__ partial, void *norm, int f64) {
  using A = typename AccOf<T>::type;
  __shared__ A s_part[kWavesPerBlock][kWave][VEC];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = threadIdx.x >> 6;
  const bool is_long = static_cast<int>(blockIdx.x) >= joins;
  double squares = 0.0;  // (of this lane)
  const int64_t first = is_long ? (static_cast<int64_t>(blockIdx.x) - joins) * kLongTiles
                                : static_cast<int64_t>(blockIdx.x) * kWavesPerBlock + wave;
  const int64_t stride = is_long ? num_tiles : static_cast<int64_t>(joins) * kWavesPerBlock;
  for (int64_t at = first; at < num_tiles; at += stride) {
    if (!is_long)
      for (int b = lane; b < column_blocks; b += kWave) squares += tile_sums[at * column_blocks + b];
    const int64_t next = (at + 1) * kTile;
    if (next >= n) continue;
    const int segment = segment_ids[next - 1];
    if (segment_ids[next] != segment) continue;
    const int64_t tile = segment_starts[segment] / kTile;  // where it begins
    const int64_t last = (static_cast<int64_t>(segment_starts[segment + 1]) - 1) / kTile;
    if ((last - tile > kLongTiles) != is_long) continue;
    // (a segment that began in an earlier tile is joined by that one's wavefront, or the workgroup of the first kLongTiles-th
    // tile from there on; the conditions hold for a whole workgroup where the barriers are)
    if (is_long ? at - tile >= kLongTiles : at != tile) continue;
    for (int v0 = 0; v0 < D / VEC; v0 += kWave) {
      const int chunks = min(kWave, D / VEC - v0);
      const int groups = kWave / chunks;
      const int r = lane / chunks;
      const int c = lane - r * chunks;
      const int64_t col = static_cast<int64_t>(v0 + c) * VEC;
      A sum[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) sum[k] = A(0);
      if (r < groups)
        add_partial_rows<VEC, A>(partial_rows, D, tile, tile + (is_long ? wave * groups : 0) + r,
                                 is_long ? groups * kWavesPerBlock : groups, last, col, sum);
      for (int g = 1; g < groups; ++g) {
        const int from = min(lane + g * chunks, kWave - 1);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const A o = shfl_idx(sum[k], from);
          if (r == 0) sum[k] += o;
        }
      }
      if (is_long) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < VEC; ++k) s_part[wave][lane][k] = sum[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          sum[k] = A(0);
#pragma unroll
          for (int w = 0; w < kWavesPerBlock; ++w) sum[k] += s_part[w][lane][k];
        }
      }
      if (r == 0 && (!is_long || wave == 0)) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) squares += static_cast<double>(sum[k]) * static_cast<double>(sum[k]);
      }
    }
  }
  squares = block_sum<kWavesPerBlock>(squares);
  if (threadIdx.x != 0) return;
  if (gridDim.x == 1) store_norm(norm, f64, sqrt(squares));  // (no more launches: this is all of it)
  else partial[blockIdx.x] = squares;
}

// ------------------------------------------------------------------------------------------ host
constexpr int kMaxBlocks = 256 * 8;   // of a sum over a list: eight workgroups per compute unit
constexpr int kScaleBlocks = 1 << 14; // of a scaling launch (see scale_kernel)
constexpr int kJoinBlocks = 8192;
constexpr int kFewTiles = 8;

size_t size_of(int32_t dtype) { return dtype == TBE_DTYPE_F64 ? 8 : dtype == TBE_DTYPE_F32 ? 4 : 2; }

struct ListCall {
  const void *const *gradients;
  void *const *outputs;
  const int64_t *numels;
  const int32_t *dtypes;
  int32_t count;
};

// Chunks of a tensor whose boundaries are those of `address`, and what its last one holds.
struct Chunks {
  int64_t count;
  int last;
};
Chunks chunks_of(int64_t numel, uint64_t address, int32_t dtype) {
  const int64_t size = static_cast<int64_t>(size_of(dtype));
  const int64_t head = static_cast<int64_t>((16 - (address & 15)) & 15) / size;
  const int64_t elements = kChunkVectors * 16 / size;
  if (numel < head) return Chunks{1, kNoBoundary | static_cast<int>(numel)};
  const int64_t count = std::max<int64_t>(1, ceil_div(numel - head, elements));
  return Chunks{count, static_cast<int>(numel - head - (count - 1) * elements)};
}

bool in_place(const ListCall &c) {
  for (int32_t i = 0; i < c.count; ++i)
    if (c.numels[i] && c.outputs[i] != c.gradients[i]) return false;
  return true;
}

// A call's tensors of one type, in lists of at most L::kTensors.  f(list) is called for every one.
template <typename L, typename F> void for_lists(const ListCall &c, int32_t dtype, F &&f) {
  L list;
  int tensors = 0;
  list.chunks = 0;
  const auto emit = [&] {
    for (int i = tensors; i < L::kTensors; ++i) {
      list.chunk_end[i] = INT32_MAX;
      list.src[i] = 0;
    }
    f(list);
    tensors = list.chunks = 0;
  };
  for (int32_t i = 0; i < c.count; ++i) {
    if (c.dtypes[i] != dtype || c.numels[i] == 0) continue;
    const uint64_t src = reinterpret_cast<uint64_t>(c.gradients[i]);
    const uint64_t written = L::kPairs ? reinterpret_cast<uint64_t>(c.outputs[i]) : src;
    const Chunks chunks = chunks_of(c.numels[i], written, dtype);
    if (tensors == L::kTensors || list.chunks + chunks.count > INT32_MAX / 2) emit();
    list.src[tensors] = src | static_cast<uint64_t>(chunks.last) << 48;
    if constexpr (L::kPairs) list.dst[tensors] = written;
    list.chunks += static_cast<int32_t>(chunks.count);
    list.chunk_end[tensors++] = list.chunks;
  }
  if (tensors) emit();
}

// The lists of a call that reads, or scales in place, or (pairs) has outputs of its own.
template <typename F> void each_list(const ListCall &c, int32_t dtype, bool pairs, F &&f) {
  const bool small = c.count <= kShortList;
  if (pairs && small) for_lists<ShortPairList>(c, dtype, f);
  else if (pairs) for_lists<PairList>(c, dtype, f);
  else if (small) for_lists<ShortReadList>(c, dtype, f);
  else for_lists<ReadList>(c, dtype, f);
}

int check_list(const char *name, const ListCall &c, bool outputs) {
  TBE_REQUIRE(c.count >= 0, "%s: num_tensors must not be negative", name);
  TBE_REQUIRE(c.count == 0 || (c.gradients && c.numels && c.dtypes && (c.outputs || !outputs)),
              "%s: null pointer argument", name);
  for (int32_t i = 0; i < c.count; ++i) {
    TBE_REQUIRE(c.dtypes[i] >= TBE_DTYPE_F32 && c.dtypes[i] <= TBE_DTYPE_BF16, "%s: bad dtype %d", name, c.dtypes[i]);
    const uint64_t size = size_of(c.dtypes[i]);
    TBE_REQUIRE(c.numels[i] >= 0 && c.numels[i] <= (int64_t{1} << 40), "%s: element count of tensor %d out of range", name, i);
    if (c.numels[i] == 0) continue;
    TBE_REQUIRE(c.gradients[i] && (!outputs || c.outputs[i]), "%s: null pointer argument", name);
    TBE_REQUIRE((reinterpret_cast<uint64_t>(c.gradients[i]) >> 48) == 0, "%s: address of tensor %d out of range", name, i);
    TBE_REQUIRE(reinterpret_cast<uint64_t>(c.gradients[i]) % size == 0 &&
                    (!outputs || reinterpret_cast<uint64_t>(c.outputs[i]) % size == 0),
                "%s: misaligned pointer of tensor %d", name, i);
  }
  return TBE_OK;
}

// An output may be its own gradient; apart from that no output may share memory with another output or with
// another tensor's gradient: two workgroups would write there, or one read what another has scaled.
int check_overlap(const char *name, const ListCall &c) {
  struct Range {
    uint64_t begin, end;
    bool operator<(const Range &o) const { return begin < o.begin; }
  };
  try {
    std::vector<Range> written, read;  // (a gradient that is its own output counts as written only)
    written.reserve(c.count);
    for (int32_t i = 0; i < c.count; ++i) {
      if (c.numels[i] == 0) continue;
      const uint64_t bytes = static_cast<uint64_t>(c.numels[i]) * size_of(c.dtypes[i]);
      const uint64_t out = reinterpret_cast<uint64_t>(c.outputs[i]), in = reinterpret_cast<uint64_t>(c.gradients[i]);
      written.push_back(Range{out, out + bytes});
      if (in != out) read.push_back(Range{in, in + bytes});
    }
    // (the tensors of a bucket come in order: nothing to sort then)
    for (std::vector<Range> *v : {&written, &read})
      if (!std::is_sorted(v->begin(), v->end())) std::sort(v->begin(), v->end());
    size_t r = 0;
    uint64_t read_end = 0;  // of the ranges read that begin before the one written
    for (size_t w = 0; w < written.size(); ++w) {
      for (; r < read.size() && read[r].begin < written[w].end; ++r) {
        // it begins before this range's end: it has to end before its begin, and, beginning behind the ranges written
        // before, to begin behind their ends
        TBE_REQUIRE(w == 0 || read[r].begin >= written[w - 1].end, "%s: an output shares memory with another tensor's gradient", name);
        read_end = std::max(read_end, read[r].end);
      }
      TBE_REQUIRE(read_end <= written[w].begin, "%s: an output shares memory with another tensor's gradient", name);
      TBE_REQUIRE(w == 0 || written[w].begin >= written[w - 1].end, "%s: two outputs share memory", name);
    }
  } catch (const std::bad_alloc &) {
    return fail(TBE_ERR_INVALID, "%s: out of host memory", name);
  }
  return TBE_OK;
}

constexpr int32_t kDtypes[] = {TBE_DTYPE_F32, TBE_DTYPE_F16, TBE_DTYPE_BF16, TBE_DTYPE_F64};

// (every type of a list starts pieces of its own, so there are at most this many)
int64_t max_pieces(int32_t count) { return count / kListTensors + 4; }

template <typename F> void with_type(int32_t dtype, F &&f) {
  switch (dtype) {
    case TBE_DTYPE_F32: return f(float{});
    case TBE_DTYPE_F16: return f(_Float16{});
    case TBE_DTYPE_BF16: return f(__bf16{});
    default: return f(double{});
  }
}

uint64_t total_bytes(const ListCall &c) {
  uint64_t bytes = 0;
  for (int32_t i = 0; i < c.count; ++i) bytes += static_cast<uint64_t>(c.numels[i]) * size_of(c.dtypes[i]);
  return bytes;
}
// More than the 256 MB memory-side cache holds: the second pass finds little of what the first one read, so both are
// streamed (1.2 GB squared and scaled: 568 us, 629 with plain accesses; 240 MB 117 and 107 the other way round).
bool streams(uint64_t bytes) { return bytes > (uint64_t{256} << 20); }
// Outputs of their own push what the norm's pass has left out of the caches, unless they are streamed (240 MB squared and
// scaled: 112 us, 141 with plain stores, 160 MB 77 and 81, 40 to 128 MB no difference to 63 and 64; two sets of 96 MB in
// turn 49 and 57); small ones are left to whoever reads them next.
bool streams_out(bool same, uint64_t bytes) { return streams(bytes) || (!same && bytes > (uint64_t{32} << 20)); }

// The partial sums of all lists; returns their number.
int64_t launch_squares(const ListCall &c, double *partial, hipStream_t s) {
  int64_t used = 0;
  const bool stream = streams(total_bytes(c));
  for (const int32_t dtype : kDtypes) {
    each_list(c, dtype, false, [&](const auto &list) {
      using L = std::decay_t<decltype(list)>;
      const dim3 grid(static_cast<unsigned>(std::min(list.chunks, stream ? kMaxBlocks : kWideThreads))),
          block(kBlockThreads);
      with_type(dtype, [&](auto t) {
        using T = decltype(t);
        if (stream) TBE_LAUNCH("gradient_squares", s, (square_sum_kernel<T, L, true>), grid, block, list, partial + used);
        else TBE_LAUNCH("gradient_squares", s, (square_sum_kernel<T, L, false>), grid, block, list, partial + used);
      });
      used += grid.x;
    });
  }
  return used;
}

void launch_finish(const double *partial, int64_t used, void *norm, int32_t norm_dtype, hipStream_t s) {
  TBE_LAUNCH("gradient_norm", s, norm_finish_kernel, dim3(1), dim3(kWideThreads), partial, used, norm,
             norm_dtype == TBE_DTYPE_F64 ? 1 : 0);
}

void launch_scale(const ListCall &c, double max_norm, const void *norm, int32_t norm_dtype, hipStream_t s) {
  const int f64 = norm_dtype == TBE_DTYPE_F64 ? 1 : 0;
  const uint64_t bytes = total_bytes(c);
  const bool same = in_place(c);
  const bool stream_in = streams(bytes), stream_out = streams_out(same, bytes);
  for (const int32_t dtype : kDtypes) {
    with_type(dtype, [&](auto t) {
      using T = decltype(t);
      const auto launch = [&](const auto &list) {
        using L = std::decay_t<decltype(list)>;
        const dim3 grid(static_cast<unsigned>(std::min(list.chunks, kScaleBlocks))), block(kWideThreads);
        if (stream_in) TBE_LAUNCH("gradient_scale", s, (scale_kernel<T, L, true, true>), grid, block, list, norm, f64, max_norm);
        else if (stream_out) TBE_LAUNCH("gradient_scale", s, (scale_kernel<T, L, false, true>), grid, block, list, norm, f64, max_norm);
        else TBE_LAUNCH("gradient_scale", s, (scale_kernel<T, L, false, false>), grid, block, list, norm, f64, max_norm);
      };
      each_list(c, dtype, !same, launch);
    });
  }
}

// What a call's lists come to.
struct Lists {
  int32_t dtype = -1;     // -1: no elements; -2: several types
  int64_t chunks = 0;
  bool same;              // nothing is written, or in place
};
Lists count_lists(const ListCall &c) {
  Lists l;
  l.same = !c.outputs || in_place(c);
  for (int32_t i = 0; i < c.count; ++i) {
    if (c.numels[i] == 0) continue;
    l.dtype = l.dtype == -1 || l.dtype == c.dtypes[i] ? c.dtypes[i] : -2;
    l.chunks += chunks_of(c.numels[i], reinterpret_cast<uint64_t>(l.same ? c.gradients[i] : c.outputs[i]), c.dtypes[i]).count;
  }
  return l;
}

// Norm (c.outputs null) or norm and scaling of one list of few chunks, in one launch; whether it was one.
bool launch_few(const ListCall &c, const Lists &l, double max_norm, void *norm, int32_t norm_dtype, hipStream_t s) {
  if (l.dtype < 0 || l.chunks > (l.same ? kFewChunks : kFewWritten)) return false;
  with_type(l.dtype, [&](auto t) {
    const auto launch = [&](const auto &list) {
      TBE_LAUNCH("gradient_clip_few", s, (clip_few_kernel<decltype(t), std::decay_t<decltype(list)>>), dim3(1),
                 dim3(kWideThreads), list, c.outputs ? 1 : 0, norm, norm_dtype == TBE_DTYPE_F64 ? 1 : 0, max_norm);
    };
    each_list(c, l.dtype, !l.same, launch);
  });
  return true;
}

// Norm and scaling.  (The norm is written by every list's launch, the same value.)
void launch_clip(const ListCall &c, const Lists &l, double max_norm, void *workspace, void *norm, int32_t norm_dtype,
                 hipStream_t s) {
  const uint64_t bytes = total_bytes(c);
  double *partial = static_cast<double *>(workspace);
  const int64_t used = launch_squares(c, partial, s);
  if (streams(bytes) || used == 0 || used > kJoinedSums) {
    launch_finish(partial, used, norm, norm_dtype, s);
    launch_scale(c, max_norm, norm, norm_dtype, s);
    return;
  }
  const int f64 = norm_dtype == TBE_DTYPE_F64 ? 1 : 0;
  const bool stream_out = streams_out(l.same, bytes);
  for (const int32_t dtype : kDtypes) {
    with_type(dtype, [&](auto t) {
      using T = decltype(t);
      const auto launch = [&](const auto &list) {
        using L = std::decay_t<decltype(list)>;
        const dim3 grid(static_cast<unsigned>(std::min(list.chunks, kJoinedBlocks))), block(kWideThreads);
        if (stream_out)
          TBE_LAUNCH("gradient_scale", s, (scale_joined_kernel<T, L, true>), grid, block, list, partial, used, norm, f64, max_norm);
        else
          TBE_LAUNCH("gradient_scale", s, (scale_joined_kernel<T, L, false>), grid, block, list, partial, used, norm, f64, max_norm);
      };
      each_list(c, dtype, !l.same, launch);
    });
  }
}

int check_norm(const char *name, const void *norm, int32_t norm_dtype) {
  TBE_REQUIRE(norm, "%s: norm is null", name);
  TBE_REQUIRE(norm_dtype == TBE_DTYPE_F32 || norm_dtype == TBE_DTYPE_F64, "%s: the norm is F32 or F64 (got %d)", name, norm_dtype);
  return TBE_OK;
}

int check_workspace(const char *name, int32_t count, const void *workspace, uint64_t bytes) {
  const uint64_t need = tbe_gradient_norm_workspace_bytes(count);
  if (!workspace || bytes < need)
    return fail(TBE_ERR_WORKSPACE, "%s: workspace of %llu bytes needed, %llu given", name, (unsigned long long)need,
                (unsigned long long)bytes);
  return TBE_OK;
}

struct TableCall {
  const void *grad, *psw;
  const int32_t *positions_sorted, *grad_rows, *segment_ids, *segment_starts;
  int64_t n;
  int32_t D;
  void *partial_rows;
  double *tile_sums, *partial;
  void *norm;
  int f64;
  hipStream_t stream;
};

// Workgroups that join: a tile per wavefront, or one workgroup for what it does in the time of a launch; and those for the
// long segments behind them.
struct JoinGrid {
  int joins;
  int64_t blocks;
};
JoinGrid join_grid(int64_t tiles) {
  JoinGrid g;
  g.joins = tiles <= kFewTiles ? 1 : static_cast<int>(std::min<int64_t>(ceil_div(tiles, kWavesPerBlock), kJoinBlocks));
  g.blocks = g.joins + (tiles > kLongTiles ? ceil_div(tiles, kLongTiles) : 0);
  return g;
}

// Returns the number of partial sums left, 0 if the norm is written.
template <typename T, int VEC> unsigned launch_table(const TableCall &c, int64_t tiles, int column_blocks) {
  using A = typename AccOf<T>::type;
  const int64_t per_xcd = ceil_div(tiles, kNumXcd);
  const dim3 grid(static_cast<unsigned>(per_xcd * kNumXcd), column_blocks), block(kBlockThreads);
  const T *grad = static_cast<const T *>(c.grad), *psw = static_cast<const T *>(c.psw);
  A *rows = static_cast<A *>(c.partial_rows);
  if (psw)
    TBE_LAUNCH("table_norm_tiles", c.stream, (table_norm_tiles_kernel<T, VEC, true>), grid, block, grad, psw,
               c.positions_sorted, c.grad_rows, c.segment_ids, c.n, c.D, tiles, per_xcd, rows, c.tile_sums);
  else
    TBE_LAUNCH("table_norm_tiles", c.stream, (table_norm_tiles_kernel<T, VEC, false>), grid, block, grad, psw,
               c.positions_sorted, c.grad_rows, c.segment_ids, c.n, c.D, tiles, per_xcd, rows, c.tile_sums);
  const JoinGrid join = join_grid(tiles);
  TBE_LAUNCH("table_norm_join", c.stream, (table_norm_join_kernel<T, VEC>), dim3(static_cast<unsigned>(join.blocks)), block,
             c.segment_ids, c.segment_starts, c.n, c.D, tiles, join.joins, rows, c.tile_sums, column_blocks, c.partial,
             c.norm, c.f64);
  return join.blocks == 1 ? 0 : static_cast<unsigned>(join.blocks);
}

}  // namespace
}  // namespace tbe

extern "C" uint64_t tbe_gradient_norm_workspace_bytes(int32_t num_tensors) {
  if (num_tensors < 0) return 0;
  return static_cast<uint64_t>(tbe::max_pieces(num_tensors)) * tbe::kMaxBlocks * sizeof(double);
}

extern "C" int tbe_gradient_norm(const void *const *gradients, const int64_t *numels, const int32_t *dtypes,
                                 int32_t num_tensors, void *norm, int32_t norm_dtype, void *workspace,
                                 uint64_t workspace_bytes, void *stream) {
  using namespace tbe;
  const char *name = "tbe_gradient_norm";
  const ListCall c{gradients, nullptr, numels, dtypes, num_tensors};
  if (int rc = check_list(name, c, false)) return rc;
  if (int rc = check_norm(name, norm, norm_dtype)) return rc;
  if (int rc = check_workspace(name, num_tensors, workspace, workspace_bytes)) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (!launch_few(c, count_lists(c), 0.0, norm, norm_dtype, s)) {
    double *partial = static_cast<double *>(workspace);
    launch_finish(partial, launch_squares(c, partial, s), norm, norm_dtype, s);
  }
  return check_launch(name);
}

extern "C" int tbe_scale_gradients(const void *const *gradients, void *const *outputs, const int64_t *numels,
                                   const int32_t *dtypes, int32_t num_tensors, double max_norm, const void *norm,
                                   int32_t norm_dtype, void *stream) {
  using namespace tbe;
  const char *name = "tbe_scale_gradients";
  const ListCall c{gradients, outputs, numels, dtypes, num_tensors};
  if (int rc = check_list(name, c, true)) return rc;
  if (int rc = check_norm(name, norm, norm_dtype)) return rc;
  TBE_REQUIRE(max_norm >= 0.0, "%s: max_norm must not be negative", name);
  if (int rc = check_overlap(name, c)) return rc;
  launch_scale(c, max_norm, norm, norm_dtype, static_cast<hipStream_t>(stream));
  return check_launch(name);
}

extern "C" int tbe_clip_gradients(const void *const *gradients, void *const *outputs, const int64_t *numels,
                                  const int32_t *dtypes, int32_t num_tensors, double max_norm, void *norm,
                                  int32_t norm_dtype, void *workspace, uint64_t workspace_bytes, void *stream) {
  using namespace tbe;
  const char *name = "tbe_clip_gradients";
  const ListCall c{gradients, outputs, numels, dtypes, num_tensors};
  if (int rc = check_list(name, c, true)) return rc;
  if (int rc = check_norm(name, norm, norm_dtype)) return rc;
  TBE_REQUIRE(max_norm >= 0.0, "%s: max_norm must not be negative", name);
  if (int rc = check_workspace(name, num_tensors, workspace, workspace_bytes)) return rc;
  if (int rc = check_overlap(name, c)) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const Lists l = count_lists(c);
  if (!launch_few(c, l, max_norm, norm, norm_dtype, s)) launch_clip(c, l, max_norm, workspace, norm, norm_dtype, s);
  return check_launch(name);
}

extern "C" int tbe_table_gradient_norm(const void *grad_output, int32_t dtype, int32_t D, int32_t T, int32_t B,
                                       int64_t num_indices, const void *per_sample_weights, void *workspace,
                                       uint64_t workspace_bytes, void *norm, int32_t norm_dtype, void *stream) {
  using namespace tbe;
  const char *name = "tbe_table_gradient_norm";
  TBE_REQUIRE(T > 0 && B > 0, "%s: T and B must be positive (got %d, %d)", name, T, B);
  TBE_REQUIRE(D > 0 && D % 4 == 0, "%s: D must be a positive multiple of 4 (got %d)", name, D);
  TBE_REQUIRE(dtype >= TBE_DTYPE_F32 && dtype <= TBE_DTYPE_F64, "%s: bad dtype %d", name, dtype);
  TBE_REQUIRE(num_indices >= 0 && num_indices < INT32_MAX, "%s: num_indices out of range", name);
  TBE_REQUIRE(static_cast<int64_t>(T) * B < INT32_MAX, "%s: T*B out of range", name);
  TBE_REQUIRE(grad_output, "%s: null pointer argument", name);
  if (int rc = check_norm(name, norm, norm_dtype)) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int f64 = norm_dtype == TBE_DTYPE_F64 ? 1 : 0;
  if (num_indices == 0) {
    TBE_LAUNCH("gradient_norm", s, norm_finish_kernel, dim3(1), dim3(kWideThreads), nullptr, int64_t{0}, norm, f64);
    return check_launch(name);
  }
  tbe_workspace_layout_t l;
  backward_layout(num_indices, D, dtype, T, &l);
  if (!workspace || workspace_bytes < l.total_bytes)
    return fail(TBE_ERR_WORKSPACE, "%s: workspace of %llu bytes needed, %llu given", name,
                (unsigned long long)l.total_bytes, (unsigned long long)workspace_bytes);
  const RowGeometry g = row_geometry(dtype, D);
  const int64_t tiles = ceil_div(num_indices, kTile);
  const int64_t column_blocks = ceil_div(g.chunks, kWave);
  // The update's queues and partial rows are not in use between a plan and its update: the tiles' sums go to the
  // chunk records' room, the partial rows (two per kTile positions, like the update's) to their own.
  static_assert(kTile == kChunkLen, "two partial rows per tile fit the update's");
  const int64_t join_parts = join_grid(tiles).blocks;
  const uint64_t sums = static_cast<uint64_t>(tiles * column_blocks + join_parts) * sizeof(double);
  if (sums > l.partial_sums - l.chunk_segments || column_blocks > 65535)
    return fail(TBE_ERR_UNSUPPORTED, "%s: rows of %d elements are too wide", name, D);
  char *ws = static_cast<char *>(workspace);
  TableCall c;
  c.grad = grad_output;
  c.psw = per_sample_weights;
  c.positions_sorted = reinterpret_cast<const int32_t *>(ws + l.positions_sorted);
  c.grad_rows = reinterpret_cast<const int32_t *>(ws + l.grad_rows);
  c.segment_ids = reinterpret_cast<const int32_t *>(ws + l.segment_ids);
  c.segment_starts = reinterpret_cast<const int32_t *>(ws + l.segment_starts);
  c.n = num_indices;
  c.D = D;
  c.partial_rows = ws + l.partial_sums;
  c.partial = reinterpret_cast<double *>(ws + l.chunk_segments);
  c.tile_sums = c.partial + join_parts;
  c.norm = norm;
  c.f64 = f64;
  c.stream = s;
  unsigned parts;
  switch (dtype) {
    case TBE_DTYPE_F32: parts = launch_table<float, 4>(c, tiles, static_cast<int>(column_blocks)); break;
    case TBE_DTYPE_F16:
      parts = g.vec == 8 ? launch_table<__half, 8>(c, tiles, static_cast<int>(column_blocks))
                         : launch_table<__half, 4>(c, tiles, static_cast<int>(column_blocks));
      break;
    default: parts = launch_table<double, 2>(c, tiles, static_cast<int>(column_blocks)); break;
  }
  if (parts)
    TBE_LAUNCH("gradient_norm", s, norm_finish_kernel, dim3(1), dim3(kWideThreads), c.partial,
               static_cast<int64_t>(parts), norm, f64);
  return check_launch(name);
}
