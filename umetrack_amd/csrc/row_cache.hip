// Rows of state caches: copy, fork, free and compact.  A row is one hand track's state, a few buffers wide (2592 + 64
// bytes of temporal memory, 252 of smoothed landmarks, ...).
//
// The index work (who writes a row last, which rows are free, where a row goes) is integer arithmetic on a few bytes a
// row; the moves are bound by HBM: 2 x row bytes for every row that changes place, and rows that stay are not touched.
// A wave moves up to MOVE_BYTES of one buffer's row, all of its loads in flight before its first store, so that a few long
// rows fill the GPU as well as many short ones; buffers of a few words a row ride along with a row's first piece.
// Ranks come from per-block counts that every block adds up for itself, in one workgroup where the cache is small.
#include "umt_internal.h"

#include <algorithm>
#include <type_traits>

namespace umt {

constexpr int RT = 256;
constexpr int64_t MOVE_BYTES = 4096;       // 64 lanes x 16 bytes x 4 loads in flight
constexpr int ONE = 1024;                  // threads of a workgroup that ranks rows
constexpr int BLOCK = 4 * ONE;             // rows it takes at once
constexpr int LDS_BYTES = 64 * 1024;       // of a workgroup that stages rows

struct RowBuffers {
  char* data[UMT_ROW_BUFFERS_MAX];
  int64_t bytes[UMT_ROW_BUFFERS_MAX];      // a row's
  int64_t staged[UMT_ROW_BUFFERS_MAX];     // offset in a staged row
  int unit[UMT_ROW_BUFFERS_MAX];           // 16, 4 or 1: what data and row_bytes are multiples of
  int piece0[UMT_ROW_BUFFERS_MAX + 1];     // first piece of long buffer k in a row; [n_long] = pieces of a row
  int n, n_long;                           // long buffers first; the others have at most one unit a lane
  int64_t staged_bytes;
};

// Bytes in HBM and in LDS: addresses of their own kinds, or every access would be a generic one
using Global = __attribute__((address_space(1))) char*;
using Local = __attribute__((address_space(3))) char*;
template <typename P, typename U>
__device__ __forceinline__ U load_unit(P p, int i) {
  if constexpr (std::is_same_v<P, Global>)
    return ((const __attribute__((address_space(1))) U*)p)[i];
  else
    return ((const __attribute__((address_space(3))) U*)p)[i];
}
template <typename P, typename U>
__device__ __forceinline__ void store_unit(P p, int i, U v) {
  if constexpr (std::is_same_v<P, Global>)
    ((__attribute__((address_space(1))) U*)p)[i] = v;
  else
    ((__attribute__((address_space(3))) U*)p)[i] = v;
}
typedef uint32_t Quad __attribute__((ext_vector_type(4)));

template <typename U, typename TO, typename FROM>
__device__ __forceinline__ void move_units(TO to, FROM from, int n, int lane) {
  for (int i0 = 0; i0 < n; i0 += 256) {
    U r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i0 + lane + 64 * i < n) r[i] = load_unit<FROM, U>(from, i0 + lane + 64 * i);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i0 + lane + 64 * i < n) store_unit<TO, U>(to, i0 + lane + 64 * i, r[i]);
  }
}

// Where a row lies: in the caches, or in a staged row (16-byte aligned)
struct Cached {
  using P = Global;
  int64_t row;
  __device__ __forceinline__ P at(const RowBuffers& B, int k) const { return (Global)(B.data[k] + row * B.bytes[k]); }
};
template <typename A>
struct Staged {
  using P = A;
  A base;
  __device__ __forceinline__ P at(const RowBuffers& B, int k) const { return base + B.staged[k]; }
};

// Piece p of a row, by one wave.  Source and target are different rows, and no other wave writes the one or reads the other.
template <typename TO, typename FROM>
__device__ __forceinline__ void move_piece(const RowBuffers& B, int p, TO to, FROM from, int lane) {
  using T = typename TO::P;
  using F = typename FROM::P;
  uint32_t word[UMT_ROW_BUFFERS_MAX];
  Quad quad[UMT_ROW_BUFFERS_MAX];
  const bool tiny = p == 0;
  if (tiny) {
#pragma unroll
    for (int k = 0; k < UMT_ROW_BUFFERS_MAX; ++k) {
      if (k < B.n_long || k >= B.n) continue;
      const F f = from.at(B, k);
      if (lane * B.unit[k] < B.bytes[k]) {
        if (B.unit[k] == 16)
          quad[k] = load_unit<F, Quad>(f, lane);
        else
          word[k] = B.unit[k] == 4 ? load_unit<F, uint32_t>(f, lane) : (uint32_t)load_unit<F, uint8_t>(f, lane);
      }
    }
  }
  if (B.n_long) {
    int k = 0;
    while (k + 1 < B.n_long && p >= B.piece0[k + 1]) ++k;
    const int64_t off = (int64_t)(p - B.piece0[k]) * MOVE_BYTES, left = B.bytes[k] - off;
    const int n = (int)(left < MOVE_BYTES ? left : MOVE_BYTES);
    const T t = to.at(B, k) + off;
    const F f = from.at(B, k) + off;
    if (B.unit[k] == 16)
      move_units<Quad>(t, f, n / 16, lane);
    else if (B.unit[k] == 4)
      move_units<uint32_t>(t, f, n / 4, lane);
    else
      move_units<uint8_t>(t, f, n, lane);
  }
  if (tiny) {
#pragma unroll
    for (int k = 0; k < UMT_ROW_BUFFERS_MAX; ++k) {
      if (k < B.n_long || k >= B.n) continue;
      const T t = to.at(B, k);
      if (lane * B.unit[k] < B.bytes[k]) {
        if (B.unit[k] == 16)
          store_unit<T, Quad>(t, lane, quad[k]);
        else if (B.unit[k] == 4)
          store_unit<T, uint32_t>(t, lane, word[k]);
        else
          store_unit<T, uint8_t>(t, lane, (uint8_t)word[k]);
      }
    }
  }
}

// the same in all lanes of a wave: row numbers go into scalar registers, and with them every address of the row
__device__ __forceinline__ int64_t uniform(int64_t v) {
  return (int64_t)((uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)v));
}

__device__ __forceinline__ bool in_cache(int64_t r, int rows) { return r >= 0 && r < rows; }

// exclusive rank of v among the workgroup's ONE threads, in thread order, and the sum of all
__device__ __forceinline__ int rank_in_group(int v, int* total, int* lds) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  int incl = v;
  for (int o = 1; o < 64; o <<= 1) {
    const int w = __shfl_up(incl, o);
    incl += lane >= o ? w : 0;
  }
  __syncthreads();
  if (lane == 63) lds[wv] = incl;
  __syncthreads();
  int before = 0, all = 0;
  for (int k = 0; k < ONE / 64; ++k) {
    before += k < wv ? lds[k] : 0;
    all += lds[k];
  }
  *total = all;
  return before + incl - v;
}

// the same with the sums of two more numbers, behind one wait
struct RankAndSums {
  int rank, all, a, b;
};
__device__ __forceinline__ RankAndSums rank_and_sums(int v, int a, int b, int4* lds) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  int incl = v;
  for (int o = 1; o < 64; o <<= 1) {
    const int w = __shfl_up(incl, o);
    incl += lane >= o ? w : 0;
    a += __shfl_xor(a, o);
    b += __shfl_xor(b, o);
  }
  __syncthreads();
  if (lane == 63) lds[wv] = make_int4(incl, a, b, 0);
  __syncthreads();
  RankAndSums r{incl - v, 0, 0, 0};
  for (int k = 0; k < ONE / 64; ++k) {
    const int4 w = lds[k];
    r.rank += k < wv ? w.x : 0;
    r.all += w.x;
    r.a += w.y;
    r.b += w.z;
  }
  return r;
}

// bit i: live[r + i] is set, i < 4; rows at or past `end` are not
__device__ __forceinline__ int live4(const uint8_t* live, int64_t r, int64_t end) {
  int b = 0;
  if (((uint64_t)live & 3) == 0 && r + 4 <= end && (r & 3) == 0) {
    const uint32_t v = *reinterpret_cast<const uint32_t*>(live + r);
    for (int i = 0; i < 4; ++i) b |= (v >> (8 * i) & 0xff ? 1 : 0) << i;
  } else {
    for (int i = 0; i < 4; ++i)
      if (r + i < end) b |= (live[r + i] ? 1 : 0) << i;
  }
  return b;
}

// counts[block] = live rows of the block
__global__ __launch_bounds__(ONE) void count_rows_kernel(const uint8_t* __restrict__ live, int rows, int32_t* __restrict__ counts) {
  __shared__ int lds[ONE / 64];
  int all;
  rank_in_group(__popc(live4(live, (int64_t)blockIdx.x * BLOCK + threadIdx.x * 4, rows)), &all, lds);
  if (threadIdx.x == 0) counts[blockIdx.x] = all;
}
// sum of counts[0 .. upto) by the whole workgroup, in any order: they are integers
__device__ __forceinline__ int sum_counts(const int32_t* counts, int upto, int* lds) {
  int mine = 0, all;
  for (int i = threadIdx.x; i < upto; i += ONE) mine += counts[i];
  rank_in_group(mine, &all, lds);
  return all;
}

// ---------------------------------------------------------------- copy
// A few rows: one workgroup holds them all in LDS between reading and writing (calls replayed in a graph, this against the
// two launches below: 20 rows of 2908 bytes 17.0 and 17.2 us, 64 rows of 252 bytes 16.2 and 16.1, 200 of them 29.9 and 16.2).
constexpr int FEW = 64;
__global__ __launch_bounds__(ONE) void copy_few_kernel(RowBuffers B, const int64_t* __restrict__ src, const int64_t* __restrict__ dst, int n,
                                                       int rows, int32_t* __restrict__ status) {
  extern __shared__ uint4 stage[];
  __shared__ int64_t to[FEW];
  __shared__ int64_t from[FEW];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), pieces = B.piece0[B.n_long];
  for (int i = tid; i < n; i += ONE) {
    const bool ok = in_cache(src[i], rows) && in_cache(dst[i], rows);
    if (!ok && status) atomicOr(status, (int)UMT_STATUS_BAD_ROW);
    to[i] = ok ? dst[i] : -1;
    from[i] = ok ? src[i] : -1;
  }
  __syncthreads();
  for (int it = wv; it < n * pieces; it += ONE / 64) {
    const int i = it / pieces;
    if (to[i] >= 0) move_piece(B, it - i * pieces, Staged<Local>{(Local)stage + i * B.staged_bytes}, Cached{uniform(from[i])}, lane);
  }
  __syncthreads();
  for (int it = wv; it < n * pieces; it += ONE / 64) {
    const int i = it / pieces;
    if (to[i] < 0) continue;
    bool last = true;                       // of several writes to one row the highest i counts
    for (int o = i + 1 + lane; o < n; o += 64) last &= to[o] != to[i];
    if (__all(last)) move_piece(B, it - i * pieces, Cached{uniform(to[i])}, Staged<Local>{(Local)stage + i * B.staged_bytes}, lane);
  }
}

// More: two launches.  Every workgroup of the first marks all targets in a bit map of the cache in its LDS (64 KB of row
// numbers from L2 for 8191 copies), decides on copies of its own and brings those sources to safety that the call overwrites.
// plan[i]: what the second launch does.  8191 of 32768 rows of 2592 + 64 + 252 bytes, sources and
// targets drawn apart from each other: 5.3 + 10.9 us, where the five launches below take 25.  The limits are the bit map's LDS
// and the launch's share of the numbers; both are ahead of the five up to there (calls replayed in a graph: 16384 copies in
// 262144 rows 17.8 and 23.8 us, 300 in 262144 rows 16.5 and 17.7).
enum { COPY_NOT = 0, COPY_ROW = 1, COPY_STAGED = 2 };
constexpr int MAP_ROWS = 1 << 18;          // 32 KB of bits
constexpr int MAP_COPIES = 1 << 14, MAP_GROUPS = 128, MAP_EACH = MAP_COPIES / MAP_GROUPS;      // MAP_EACH <= ONE: a copy a thread
__global__ __launch_bounds__(ONE) void copy_plan_kernel(RowBuffers B, const int64_t* __restrict__ src, const int64_t* __restrict__ dst, int n,
                                                        int rows, uint8_t* __restrict__ plan, char* __restrict__ stage,
                                                        int32_t* __restrict__ status) {
  extern __shared__ uint32_t map[];
  __shared__ int twice, n_todo;             // some row is written by more than one copy; sources to bring to safety
  __shared__ uint16_t todo[MAP_EACH];
  __shared__ uint8_t late[MAP_EACH];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), pieces = B.piece0[B.n_long];
  for (int i = tid; i < (rows + 31) / 32; i += ONE) map[i] = 0;
  if (tid == 0) twice = n_todo = 0;
  const int each = (n + gridDim.x - 1) / gridDim.x, i0 = min(n, (int)blockIdx.x * each), i1 = min(n, i0 + each), mine = i0 + tid;
  int64_t s = -1, d = -1;                   // a thread's own copy
  if (mine < i1) {
    s = src[mine];
    d = dst[mine];
  }
  __syncthreads();
  constexpr int AHEAD = 8;
  for (int k0 = tid; k0 < n; k0 += AHEAD * ONE) {
    int64_t r[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) r[k] = k0 + k * ONE < n ? dst[k0 + k * ONE] : -1;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {      // of a copy that will not be made too: a source too many brought to safety, no more
      if (!in_cache(r[k], rows)) continue;
      const uint32_t bit = 1u << (r[k] & 31);
      if (atomicOr(map + (r[k] >> 5), bit) & bit) twice = 1;
    }
  }
  __syncthreads();
  if (twice) {                              // of several writes to one row the highest i counts
    for (int i = i0 + wv; i < i1; i += ONE / 64) {
      const int64_t to = uniform(dst[i]);
      bool last = true;
      for (int o = i + 1 + lane; o < n; o += 64) last &= dst[o] != to || !in_cache(src[o], rows);
      const bool counts = __all(last);
      if (lane == 0) late[i - i0] = !counts;
    }
    __syncthreads();
  }
  if (mine < i1) {
    int what = COPY_NOT;
    if (!in_cache(s, rows) || !in_cache(d, rows)) {
      if (status) atomicOr(status, (int)UMT_STATUS_BAD_ROW);
    } else if (s != d && !(twice && late[tid])) {
      what = map[s >> 5] >> (s & 31) & 1 ? COPY_STAGED : COPY_ROW;
    }
    plan[mine] = (uint8_t)what;
    if (what == COPY_STAGED) todo[atomicAdd(&n_todo, 1)] = (uint16_t)mine;   // any order: each has its own place
  }
  __syncthreads();
  for (int it = wv; it < n_todo * pieces; it += ONE / 64) {
    const int k = it / pieces, i = todo[k];
    move_piece(B, it - k * pieces, Staged<Global>{(Global)(stage + i * B.staged_bytes)}, Cached{uniform(src[i])}, lane);
  }
}
__global__ __launch_bounds__(RT) void copy_planned_kernel(RowBuffers B, const int64_t* __restrict__ src, const int64_t* __restrict__ dst, int n,
                                                          const uint8_t* __restrict__ plan, char* stage) {
  const int lane = threadIdx.x & 63, pieces = B.piece0[B.n_long];
  const unsigned item = blockIdx.x * (RT / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = (int)(item / (unsigned)pieces), p = (int)(item - (unsigned)i * (unsigned)pieces);
  if (i >= n) return;
  const int what = plan[i];
  const int64_t s = src[i], d = dst[i];
  if (what == COPY_STAGED)
    move_piece(B, p, Cached{uniform(d)}, Staged<Global>{(Global)(stage + i * B.staged_bytes)}, lane);
  else if (what == COPY_ROW)
    move_piece(B, p, Cached{uniform(d)}, Cached{uniform(s)}, lane);
}

// Any number: five launches, with a table of a word a row.
// last[r] = highest i that writes row r, -1 where none does; only rows that the call names are touched
__global__ __launch_bounds__(RT) void copy_clear_kernel(const int64_t* __restrict__ src, const int64_t* __restrict__ dst, int n,
                                                        int rows, int32_t* __restrict__ last, int32_t* __restrict__ todo,
                                                        int32_t* __restrict__ status) {
  const int i = blockIdx.x * RT + threadIdx.x;
  if (i == 0) todo[0] = 0;
  if (i >= n) return;
  if (!in_cache(src[i], rows) || !in_cache(dst[i], rows)) {
    if (status) atomicOr(status, (int)UMT_STATUS_BAD_ROW);
    return;
  }
  last[src[i]] = -1;
  last[dst[i]] = -1;
}
__global__ __launch_bounds__(RT) void copy_claim_kernel(const int64_t* __restrict__ src, const int64_t* __restrict__ dst, int n,
                                                        int rows, int32_t* __restrict__ last) {
  const int i = blockIdx.x * RT + threadIdx.x;
  if (i < n && in_cache(src[i], rows) && in_cache(dst[i], rows)) atomicMax(last + dst[i], i);
}
__device__ __forceinline__ bool copies(const int32_t* last, int64_t s, int64_t d, int i, int rows) {
  return in_cache(s, rows) && in_cache(d, rows) && s != d && last[d] == i;
}
// todo: [0] how many, then the copies whose source is overwritten by the call (in any order: each has its staging place)
__global__ __launch_bounds__(RT) void copy_list_kernel(const int64_t* __restrict__ src, const int64_t* __restrict__ dst, int n, int rows,
                                                       const int32_t* __restrict__ last, int32_t* __restrict__ todo) {
  const int i = blockIdx.x * RT + threadIdx.x;
  if (i < n && copies(last, src[i], dst[i], i, rows) && last[src[i]] >= 0) todo[4 + atomicAdd(todo, 1)] = i;
}
__global__ __launch_bounds__(RT) void copy_stage_kernel(RowBuffers B, const int64_t* __restrict__ src, const int32_t* __restrict__ todo,
                                                        char* __restrict__ stage) {
  const int lane = threadIdx.x & 63, pieces = B.piece0[B.n_long];
  const unsigned n = (unsigned)todo[0] * (unsigned)pieces, stride = gridDim.x * (RT / 64);
  for (unsigned item = blockIdx.x * (RT / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); item < n; item += stride) {
    const unsigned k = item / (unsigned)pieces;
    const int i = todo[4 + k];
    move_piece(B, (int)(item - k * pieces), Staged<Global>{(Global)(stage + i * B.staged_bytes)}, Cached{uniform(src[i])}, lane);
  }
}
__global__ __launch_bounds__(RT) void copy_move_kernel(RowBuffers B, const int64_t* __restrict__ src, const int64_t* __restrict__ dst, int n,
                                                       int rows, const int32_t* __restrict__ last, char* stage) {
  const int lane = threadIdx.x & 63, pieces = B.piece0[B.n_long];
  const unsigned item = blockIdx.x * (RT / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = (int)(item / (unsigned)pieces), p = (int)(item - (unsigned)i * (unsigned)pieces);
  if (i >= n) return;
  const int64_t s = src[i], d = dst[i];
  if (!copies(last, s, d, i, rows)) return;
  if (last[s] >= 0)
    move_piece(B, p, Cached{uniform(d)}, Staged<Global>{(Global)(stage + i * B.staged_bytes)}, lane);
  else
    move_piece(B, p, Cached{uniform(d)}, Cached{uniform(s)}, lane);
}

// ---------------------------------------------------------------- fork
// order[k] = the k-th source that is a live row; the k-th free row becomes its copy.
// sources of one block: appends to order from `wanted` on
__device__ __forceinline__ int order_sources(const uint8_t* live, int rows, const int64_t* src, int n, int64_t i0, int wanted, int64_t* ids,
                                             int32_t* order, int32_t* status, int* lds) {
  int ok = 0;
  for (int j = 0; j < 4; ++j) {
    const int64_t i = i0 + threadIdx.x * 4 + j;
    if (i >= n) break;
    const bool fine = in_cache(src[i], rows) && live[src[i]] != 0;
    if (!fine && status) atomicOr(status, (int)UMT_STATUS_BAD_ROW);
    ok |= fine << j;
    ids[i] = -1;
  }
  int all, k = wanted + rank_in_group(__popc(ok), &all, lds);
  for (int j = 0; j < 4; ++j)
    if (ok >> j & 1) order[k++] = (int)(i0 + threadIdx.x * 4 + j);
  return all;
}
// free rows of one block: hands them to the sources from `found` on
__device__ __forceinline__ int hand_out_rows(uint8_t* live, int rows, int64_t r0, int found, int wanted, int64_t* ids, const int32_t* order,
                                             int* lds) {
  const int64_t r = r0 + threadIdx.x * 4;
  const int there = (int)max((int64_t)0, min((int64_t)4, rows - r)), gone = ~live4(live, r, rows) & ((1 << there) - 1);
  int all, k = found + rank_in_group(__popc(gone), &all, lds);
  for (int j = 0; j < 4; ++j)
    if (gone >> j & 1) {
      if (k < wanted) {
        ids[order[k]] = r + j;
        live[r + j] = 1;
      }
      ++k;
    }
  return all;
}

// everything in one workgroup; `moves`: the copies too (6.7 us for 2 of 64 rows), where every wave has one at most (calls
// replayed in a graph, against another launch for them: 8 rows of 2908 bytes 16.8 and 17.8 us, 64 rows of 252 19.3 and 16.8)
__global__ __launch_bounds__(ONE) void fork_one_kernel(RowBuffers B, uint8_t* live, int rows, const int64_t* __restrict__ src, int n,
                                                       int64_t* ids, int32_t* order, int32_t* status, int moves) {
  __shared__ int lds[ONE / 64];
  int wanted = 0, found = 0;
  for (int64_t i0 = 0; i0 < n; i0 += BLOCK) wanted += order_sources(live, rows, src, n, i0, wanted, ids, order, status, lds);
  __syncthreads();                          // order and ids are complete, and no live flag has changed yet
  for (int64_t r0 = 0; r0 < rows && found < wanted; r0 += BLOCK) found += hand_out_rows(live, rows, r0, found, wanted, ids, order, lds);
  if (status && threadIdx.x == 0 && found < wanted) atomicOr(status, (int)UMT_STATUS_NO_FREE_ROW);
  if (!moves) return;
  __syncthreads();
  const int lane = threadIdx.x & 63, pieces = B.piece0[B.n_long];
  for (int it = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); it < n * pieces; it += ONE / 64) {
    const int i = it / pieces;
    if (ids[i] >= 0) move_piece(B, it - i * pieces, Cached{uniform(ids[i])}, Cached{uniform(src[i])}, lane);
  }
}
// the same in four launches: counts (live rows a block; good sources a block behind them), order, hand out, move
__global__ __launch_bounds__(ONE) void fork_count_kernel(const uint8_t* __restrict__ live, int rows, const int64_t* __restrict__ src, int n,
                                                         int row_blocks, int32_t* __restrict__ counts) {
  __shared__ int lds[ONE / 64];
  int mine = 0, all;
  if ((int)blockIdx.x < row_blocks) {
    mine = __popc(live4(live, (int64_t)blockIdx.x * BLOCK + threadIdx.x * 4, rows));
  } else {
    const int64_t i0 = (int64_t)(blockIdx.x - row_blocks) * BLOCK + threadIdx.x * 4;
    for (int j = 0; j < 4; ++j) mine += i0 + j < n && in_cache(src[i0 + j], rows) && live[src[i0 + j]] != 0;
  }
  rank_in_group(mine, &all, lds);
  if (threadIdx.x == 0) counts[blockIdx.x] = all;
}
__global__ __launch_bounds__(ONE) void fork_order_kernel(const uint8_t* __restrict__ live, int rows, const int64_t* __restrict__ src, int n,
                                                         const int32_t* __restrict__ counts, int row_blocks, int64_t* __restrict__ ids,
                                                         int32_t* __restrict__ order, int32_t* __restrict__ status) {
  __shared__ int lds[ONE / 64];
  const int before = sum_counts(counts + row_blocks, blockIdx.x, lds);
  order_sources(live, rows, src, n, (int64_t)blockIdx.x * BLOCK, before, ids, order, status, lds);
}
__global__ __launch_bounds__(ONE) void fork_rows_kernel(uint8_t* live, int rows, const int32_t* __restrict__ counts, int row_blocks,
                                                        int source_blocks, int64_t* ids, const int32_t* __restrict__ order,
                                                        int32_t* __restrict__ status) {
  __shared__ int lds[ONE / 64];
  const int64_t r0 = (int64_t)blockIdx.x * BLOCK;
  const int found = (int)(r0 - sum_counts(counts, blockIdx.x, lds));       // free rows before this block
  const int wanted = sum_counts(counts + row_blocks, source_blocks, lds);
  const int here = found < wanted ? hand_out_rows(live, rows, r0, found, wanted, ids, order, lds) : 0;
  if (status && blockIdx.x + 1 == gridDim.x && threadIdx.x == 0 && found + here < wanted) atomicOr(status, (int)UMT_STATUS_NO_FREE_ROW);
}

// sources are live rows and targets were free ones, so no row is both
__global__ __launch_bounds__(RT) void fork_move_kernel(RowBuffers B, const int64_t* __restrict__ src, const int64_t* __restrict__ ids, int n) {
  const int lane = threadIdx.x & 63, pieces = B.piece0[B.n_long];
  const unsigned item = blockIdx.x * (RT / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = (int)(item / (unsigned)pieces);
  if (i >= n || ids[i] < 0) return;
  move_piece(B, (int)(item - (unsigned)i * (unsigned)pieces), Cached{uniform(ids[i])}, Cached{uniform(src[i])}, lane);
}

// ---------------------------------------------------------------- free
__global__ __launch_bounds__(RT) void free_rows_kernel(uint8_t* __restrict__ live, int rows, const int64_t* __restrict__ row_ids,
                                                       int n, int32_t* __restrict__ status) {
  const int64_t i = (int64_t)blockIdx.x * RT + threadIdx.x;
  if (i >= n) return;
  const int64_t r = row_ids[i];
  if (in_cache(r, rows))
    live[r] = 0;
  else if (status)
    atomicOr(status, (int)UMT_STATUS_BAD_ROW);
}

// ---------------------------------------------------------------- compact
// lists: [0] = live rows c, [1] = moves, from [4] on the holes below c and behind them the live rows from c on, in order.
// counts may be null in a grid of one block.  (Workgroups that count all 65536 flags for themselves take 9.5 us, these two
// launches 2.9 + 6.6, and a call is no shorter for it.)  live is read only: the launch that moves writes it.
__global__ __launch_bounds__(ONE) void compact_list_kernel(const uint8_t* __restrict__ live, int rows, const int32_t* __restrict__ counts,
                                                           int64_t* __restrict__ now, int32_t* __restrict__ lists) {
  __shared__ int4 lds[ONE / 64];
  const int64_t r = (int64_t)blockIdx.x * BLOCK + threadIdx.x * 4;
  const int mine = live4(live, r, rows);
  int in_all = 0, before = 0;
  if (counts)
    for (int i = threadIdx.x; i < (int)gridDim.x; i += ONE) {
      const int n = counts[i];
      in_all += n;
      before += i < (int)blockIdx.x ? n : 0;
    }
  const RankAndSums first = rank_and_sums(__popc(mine), in_all, before, lds);
  const int c = counts ? first.a : first.all;
  // live rows below row c: whole blocks, and the part of the block that row c lies in
  const int cut = counts ? c / BLOCK : 0;
  int part = __popc(live4(live, (int64_t)cut * BLOCK + threadIdx.x * 4, c));
  for (int i = threadIdx.x; i < cut; i += ONE) part += counts[i];
  const int under = rank_and_sums(0, part, 0, lds).a;
  int32_t *holes = lists + 4, *movers = holes + rows;
  int k = first.rank + first.b;             // live rows before row r
  for (int i = 0; i < 4; ++i) {
    if (r + i >= rows) break;
    const bool lv = mine >> i & 1;
    if (r + i < c) {
      if (!lv) holes[r + i - k] = (int32_t)(r + i);
      now[r + i] = lv ? r + i : -1;
    } else if (lv) {
      movers[k - under] = (int32_t)(r + i);
    } else {
      now[r + i] = -1;
    }
    k += lv;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    lists[0] = c;
    lists[1] = c - under;
  }
}

// rows at or above the live count move to free rows below it: no row is both.  14600 of 65536 rows of 2592 + 64 + 252 bytes: 18 us, 4.6 TB/s.
__global__ __launch_bounds__(RT) void compact_move_kernel(RowBuffers B, const int32_t* __restrict__ lists, int rows, uint8_t* __restrict__ live,
                                                          int64_t* __restrict__ now, int64_t* __restrict__ count) {
  const int lane = threadIdx.x & 63, pieces = B.piece0[B.n_long], c = lists[0], moves = lists[1];
  const unsigned n = (unsigned)moves * (unsigned)pieces, stride = gridDim.x * (RT / 64);
  const int64_t all = (int64_t)gridDim.x * RT;
  const int32_t *holes = lists + 4, *movers = holes + rows;
  for (int64_t r = (int64_t)blockIdx.x * RT + threadIdx.x; r < rows; r += all) {
    live[r] = r < c;
    if (r < moves) now[movers[r]] = holes[r];
    if (r == 0) *count = c;
  }
  for (unsigned item = blockIdx.x * (RT / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); item < n; item += stride) {
    const unsigned k = item / (unsigned)pieces;
    move_piece(B, (int)(item - k * pieces), Cached{uniform(holes[k])}, Cached{uniform(movers[k])}, lane);
  }
}
__global__ void compact_nothing_kernel(int64_t* count) { *count = 0; }

static int row_buffers(const char* what, const umt_row_buffer* buffers, int n, int rows, RowBuffers* B) {
  UMT_REQUIRE(n > 0 && n <= UMT_ROW_BUFFERS_MAX && buffers && rows >= 0, UMT_ERR_INVALID, "%s: %d buffers of %d rows", what, n, rows);
  *B = RowBuffers{};
  B->n = n;
  for (int k = 0; k < n; ++k) {
    const umt_row_buffer& b = buffers[k];
    UMT_REQUIRE((b.data || rows == 0) && b.row_bytes > 0 && b.row_bytes <= (1LL << 40) / (rows > 0 ? rows : 1), UMT_ERR_INVALID,
                "%s: buffer %d is null or has %d rows of %lld bytes", what, k, rows, (long long)b.row_bytes);
    const uint64_t lo = (uint64_t)b.data;
    for (int j = 0; j < k && rows > 0; ++j) {
      const uint64_t o = (uint64_t)buffers[j].data;
      UMT_REQUIRE(o + (uint64_t)buffers[j].row_bytes * rows <= lo || lo + (uint64_t)b.row_bytes * rows <= o, UMT_ERR_INVALID,
                  "%s: buffers %d and %d overlap", what, j, k);
    }
  }
  int64_t pieces = 0, off = 0;
  int at = 0;
  for (int tiny = 0; tiny < 2; ++tiny)      // long buffers first
    for (int k = 0; k < n; ++k) {
      const umt_row_buffer& b = buffers[k];
      const uint64_t both = (uint64_t)b.data | (uint64_t)b.row_bytes;
      const int unit = both % 16 == 0 ? 16 : both % 4 == 0 ? 4 : 1;
      if ((b.row_bytes <= 64 * unit) != (tiny == 1)) continue;
      B->data[at] = (char*)b.data;
      B->bytes[at] = b.row_bytes;
      B->unit[at] = unit;
      B->staged[at] = off;
      off += round_up64(b.row_bytes, 16);
      if (!tiny) {
        B->piece0[at] = (int)pieces;
        pieces += (b.row_bytes + MOVE_BYTES - 1) / MOVE_BYTES;
        UMT_REQUIRE(pieces < (1 << 30), UMT_ERR_INVALID, "%s: rows of %lld bytes", what, (long long)b.row_bytes);
        B->n_long = at + 1;
      }
      ++at;
    }
  B->piece0[B->n_long] = pieces > 0 ? (int)pieces : 1;
  B->staged_bytes = off;
  return 0;
}

// Workgroups of a move of n rows, a wave per piece.  A launch counts its threads in 32 bits; where a launch of `most`
// workgroups goes through the pieces in rounds, the pieces are counted in 31.
static int move_grid(const char* what, const RowBuffers& B, int64_t n, int most, unsigned* grid) {
  const int64_t pieces = n * B.piece0[B.n_long], wg = (pieces + RT / 64 - 1) / (RT / 64);
  UMT_REQUIRE(pieces < (most ? 1LL << 31 : (1LL << 26) - RT), UMT_ERR_INVALID, "%s: %lld rows of %d pieces", what, (long long)n,
              B.piece0[B.n_long]);
  *grid = (unsigned)(most && wg > most ? most : wg);
  return 0;
}

static int need_workspace(const char* what, const void* ws, int64_t have, int64_t need) {
  UMT_REQUIRE(need == 0 || (ws && have >= need), UMT_ERR_WORKSPACE, "%s: workspace %lld < %lld bytes", what, (long long)have, (long long)need);
  return 0;
}

}  // namespace umt

using namespace umt;

static bool few_rows(const RowBuffers& B, int n) { return n <= FEW && n * B.staged_bytes <= LDS_BYTES - 16 * FEW; }
static bool planned(int rows, int n) { return rows <= MAP_ROWS && n <= MAP_COPIES; }
static int blocks_of(int64_t n) { return (int)((n + BLOCK - 1) / BLOCK); }

extern "C" int64_t umt_rows_copy_workspace_bytes(const umt_row_buffer* buffers, int n_buffers, int rows, int n) {
  RowBuffers B;
  if (n < 0 || row_buffers("rows copy", buffers, n_buffers, rows, &B) != 0) return -1;
  if (n == 0 || few_rows(B, n)) return 0;
  // the index part holds a place for every copy asked for, also where no row number can be good
  const int64_t index = planned(rows, n) ? round_up64(n, 16) : round_up64((int64_t)rows * 4, 16) + round_up64(16 + (int64_t)n * 4, 16);
  return index + (rows ? n * B.staged_bytes : 0);
}

extern "C" int umt_rows_copy(const umt_row_buffer* buffers, int n_buffers, int rows, const int64_t* src, const int64_t* dst, int n,
                             int32_t* status, void* workspace, int64_t workspace_bytes, void* stream) {
  RowBuffers B;
  UMT_TRY(row_buffers("rows copy", buffers, n_buffers, rows, &B));
  UMT_REQUIRE(n >= 0 && (n == 0 || (src && dst)), UMT_ERR_INVALID, "rows copy: n=%d or null pointer", n);
  if (n == 0) return 0;
  hipStream_t s = (hipStream_t)stream;
  if (few_rows(B, n)) {
    hipLaunchKernelGGL(copy_few_kernel, dim3(1), dim3(ONE), (size_t)(n * B.staged_bytes), s, B, src, dst, n, rows, status);
    UMT_CHECK_HIP(hipGetLastError());
    return 0;
  }
  UMT_TRY(need_workspace("rows copy", workspace, workspace_bytes, umt_rows_copy_workspace_bytes(buffers, n_buffers, rows, n)));
  unsigned grid = 0;
  UMT_TRY(move_grid("rows copy", B, n, 0, &grid));
  if (planned(rows, n)) {
    uint8_t* plan = (uint8_t*)workspace;
    char* stage = (char*)workspace + round_up64(n, 16);
    const int groups = std::min((n + ONE / 64 - 1) / (ONE / 64), MAP_GROUPS);       // at most MAP_EACH copies each
    hipLaunchKernelGGL(copy_plan_kernel, dim3(groups), dim3(ONE), (size_t)((rows + 31) / 32) * 4, s, B, src, dst, n, rows, plan, stage, status);
    hipLaunchKernelGGL(copy_planned_kernel, dim3(grid), dim3(RT), 0, s, B, src, dst, n, plan, stage);
    UMT_CHECK_HIP(hipGetLastError());
    return 0;
  }
  int32_t* last = (int32_t*)workspace;
  int32_t* todo = (int32_t*)((char*)workspace + round_up64((int64_t)rows * 4, 16));
  char* stage = (char*)todo + round_up64(16 + (int64_t)n * 4, 16);
  const dim3 per_pair((n + RT - 1) / RT);
  hipLaunchKernelGGL(copy_clear_kernel, per_pair, dim3(RT), 0, s, src, dst, n, rows, last, todo, status);
  hipLaunchKernelGGL(copy_claim_kernel, per_pair, dim3(RT), 0, s, src, dst, n, rows, last);
  hipLaunchKernelGGL(copy_list_kernel, per_pair, dim3(RT), 0, s, src, dst, n, rows, last, todo);
  hipLaunchKernelGGL(copy_stage_kernel, dim3(grid < 2048 ? grid : 2048), dim3(RT), 0, s, B, src, todo, stage);
  hipLaunchKernelGGL(copy_move_kernel, dim3(grid), dim3(RT), 0, s, B, src, dst, n, rows, last, stage);
  UMT_CHECK_HIP(hipGetLastError());
  return 0;
}

// One workgroup ranks this many rows or sources in the time of the other launches' start (calls replayed in a graph, one
// workgroup against the four launches: 1000 of 4096 rows 18.0 and 22.9 us; of 16384 rows 2 17.4 and 20.6, 1000 23.8 and 22.5;
// 1000 of 32768 rows 31.6 and 22.9)
static bool one_group(int rows, int n) { return rows <= 4 * BLOCK && n <= BLOCK; }

extern "C" int64_t umt_rows_fork_workspace_bytes(int rows, int n) {
  return rows < 0 || n < 0 ? -1 : n == 0 ? 0 : (int64_t)n * 4 + (one_group(rows, n) ? 0 : (blocks_of(rows) + blocks_of(n)) * 4);
}

extern "C" int umt_rows_fork(const umt_row_buffer* buffers, int n_buffers, int rows, uint8_t* live, const int64_t* src, int n,
                             int64_t* ids, int32_t* status, void* workspace, int64_t workspace_bytes, void* stream) {
  RowBuffers B;
  UMT_TRY(row_buffers("rows fork", buffers, n_buffers, rows, &B));
  UMT_REQUIRE(n >= 0 && (n == 0 || (src && ids)) && (live || rows == 0), UMT_ERR_INVALID, "rows fork: n=%d or null pointer", n);
  if (n == 0) return 0;
  UMT_TRY(need_workspace("rows fork", workspace, workspace_bytes, umt_rows_fork_workspace_bytes(rows, n)));
  unsigned grid = 0;
  UMT_TRY(move_grid("rows fork", B, n, 0, &grid));
  hipStream_t s = (hipStream_t)stream;
  int32_t *order = (int32_t*)workspace, *counts = order + n;
  if (one_group(rows, n)) {
    const int moves = (int64_t)n * B.piece0[B.n_long] <= ONE / 64;
    hipLaunchKernelGGL(fork_one_kernel, dim3(1), dim3(ONE), 0, s, B, live, rows, src, n, ids, order, status, moves);
    if (!moves) hipLaunchKernelGGL(fork_move_kernel, dim3(grid), dim3(RT), 0, s, B, src, ids, n);
  } else {
    const int rb = blocks_of(rows), sb = blocks_of(n);
    hipLaunchKernelGGL(fork_count_kernel, dim3(rb + sb), dim3(ONE), 0, s, live, rows, src, n, rb, counts);
    hipLaunchKernelGGL(fork_order_kernel, dim3(sb), dim3(ONE), 0, s, live, rows, src, n, counts, rb, ids, order, status);
    if (rb) hipLaunchKernelGGL(fork_rows_kernel, dim3(rb), dim3(ONE), 0, s, live, rows, counts, rb, sb, ids, order, status);
    hipLaunchKernelGGL(fork_move_kernel, dim3(grid), dim3(RT), 0, s, B, src, ids, n);
  }
  UMT_CHECK_HIP(hipGetLastError());
  return 0;
}

extern "C" int umt_rows_free(uint8_t* live, int rows, const int64_t* row_ids, int n, int32_t* status, void* stream) {
  UMT_REQUIRE(n >= 0 && rows >= 0 && (n == 0 || row_ids) && (live || rows == 0), UMT_ERR_INVALID, "rows free: n=%d rows=%d or null pointer", n, rows);
  if (n == 0) return 0;
  hipLaunchKernelGGL(free_rows_kernel, dim3((unsigned)(((int64_t)n + RT - 1) / RT)), dim3(RT), 0, (hipStream_t)stream, live, rows, row_ids, n, status);
  UMT_CHECK_HIP(hipGetLastError());
  return 0;
}

extern "C" int64_t umt_rows_compact_workspace_bytes(int rows) { return rows < 0 ? -1 : 16 + 8 * (int64_t)rows + 4 * (int64_t)blocks_of(rows); }

extern "C" int umt_rows_compact(const umt_row_buffer* buffers, int n_buffers, int rows, uint8_t* live, int64_t* now, int64_t* count,
                                void* workspace, int64_t workspace_bytes, void* stream) {
  RowBuffers B;
  UMT_TRY(row_buffers("rows compact", buffers, n_buffers, rows, &B));
  UMT_REQUIRE((live && now && count) || (rows == 0 && count), UMT_ERR_INVALID, "rows compact: null pointer");
  hipStream_t s = (hipStream_t)stream;
  if (rows == 0) {
    hipLaunchKernelGGL(compact_nothing_kernel, dim3(1), dim3(1), 0, s, count);
    UMT_CHECK_HIP(hipGetLastError());
    return 0;
  }
  UMT_TRY(need_workspace("rows compact", workspace, workspace_bytes, umt_rows_compact_workspace_bytes(rows)));
  unsigned grid = 0;
  UMT_TRY(move_grid("rows compact", B, rows / 2 + 1, 4096, &grid));              // at most half of the rows move
  int32_t *lists = (int32_t*)workspace, *counts = lists + 4 + 2 * (int64_t)rows;
  const int blocks = blocks_of(rows);
  const bool counted = blocks > 1;
  if (counted) hipLaunchKernelGGL(count_rows_kernel, dim3(blocks), dim3(ONE), 0, s, live, rows, counts);
  hipLaunchKernelGGL(compact_list_kernel, dim3(blocks), dim3(ONE), 0, s, live, rows, counted ? counts : (int32_t*)nullptr, now, lists);
  hipLaunchKernelGGL(compact_move_kernel, dim3(grid), dim3(RT), 0, s, B, lists, rows, live, now, count);
  UMT_CHECK_HIP(hipGetLastError());
  return 0;
}
