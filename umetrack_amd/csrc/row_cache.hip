// Rows of state caches: copy, fork, free and compact.  A row is one hand track's state, a few buffers wide (2592 + 64
// bytes of temporal memory, 252 of smoothed landmarks, ...).
//
// The index work (who writes a row last, which rows are free, where a row goes) is integer arithmetic on a few bytes a
// row; the moves are bound by HBM: 2 x row bytes for every row that changes place, and rows that stay are not touched.
// A move is cut into pieces of MOVE_BYTES over all buffers, one wave each, so that a few long rows fill the GPU as well as
// many short ones.
#include "umt_internal.h"

namespace umt {

constexpr int RT = 256;
constexpr int64_t MOVE_BYTES = 4096;       // 64 lanes x 16 bytes x 4 loads in flight

struct RowBuffers {
  char* data[UMT_ROW_BUFFERS_MAX];
  int64_t bytes[UMT_ROW_BUFFERS_MAX];      // a row's
  int64_t staged[UMT_ROW_BUFFERS_MAX];     // offset in a staged row
  int unit[UMT_ROW_BUFFERS_MAX];           // 16, 4 or 1: what data and row_bytes are multiples of
  int piece0[UMT_ROW_BUFFERS_MAX + 1];     // first piece of the buffer in a row
  int n;
  int64_t staged_bytes;
};

template <typename U>
__device__ __forceinline__ void move_units(char* __restrict__ to, const char* __restrict__ from, int n, int lane) {
  U* t = reinterpret_cast<U*>(to);
  const U* f = reinterpret_cast<const U*>(from);
  int i = lane;
  for (; i + 192 < n; i += 256) {
    const U a = f[i], b = f[i + 64], c = f[i + 128], d = f[i + 192];
    t[i] = a;
    t[i + 64] = b;
    t[i + 128] = c;
    t[i + 192] = d;
  }
  for (; i < n; i += 64) t[i] = f[i];
}

// piece p of a row; `to` / `from` null: the caches' row, else a staged row (16-byte aligned)
__device__ __forceinline__ void move_piece(const RowBuffers& B, int p, int64_t dst, char* to, int64_t src, const char* from, int lane) {
  int k = 0;
  while (k + 1 < B.n && p >= B.piece0[k + 1]) ++k;
  const int64_t at = (int64_t)(p - B.piece0[k]) * MOVE_BYTES, left = B.bytes[k] - at;
  const int n = (int)(left < MOVE_BYTES ? left : MOVE_BYTES);
  char* t = to ? to + B.staged[k] + at : B.data[k] + dst * B.bytes[k] + at;
  const char* f = from ? from + B.staged[k] + at : B.data[k] + src * B.bytes[k] + at;
  if (B.unit[k] == 16)
    move_units<uint4>(t, f, n / 16, lane);
  else if (B.unit[k] == 4)
    move_units<uint32_t>(t, f, n / 4, lane);
  else
    move_units<uint8_t>(t, f, n, lane);
}

__device__ __forceinline__ bool in_cache(int64_t r, int rows) { return r >= 0 && r < rows; }

// ---------------------------------------------------------------- copy
// last[r] = highest i that writes row r, -1 where none does; only rows that the call names are touched
__global__ __launch_bounds__(RT) void copy_clear_kernel(const int64_t* __restrict__ src, const int64_t* __restrict__ dst, int n,
                                                        int rows, int32_t* __restrict__ last, int32_t* __restrict__ status) {
  const int i = blockIdx.x * RT + threadIdx.x;
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
// phase 0: rows that are read and overwritten by this call go to their staging place; phase 1: every copy, from there
template <int PHASE>
__global__ __launch_bounds__(RT) void copy_move_kernel(RowBuffers B, const int64_t* __restrict__ src, const int64_t* __restrict__ dst,
                                                       int n, int rows, const int32_t* __restrict__ last, char* __restrict__ stage) {
  const int lane = threadIdx.x & 63, pieces = B.piece0[B.n];
  const int64_t item = (int64_t)blockIdx.x * (RT / 64) + (threadIdx.x >> 6);
  const int64_t i = item / pieces;
  if (i >= n) return;
  const int p = (int)(item - i * pieces);
  const int64_t s = src[i], d = dst[i];
  if (!in_cache(s, rows) || !in_cache(d, rows) || s == d || last[d] != i) return;
  const bool overwritten = last[s] >= 0;
  char* place = stage + i * B.staged_bytes;
  if (PHASE == 0) {
    if (overwritten) move_piece(B, p, 0, place, s, nullptr, lane);
  } else {
    move_piece(B, p, d, nullptr, s, overwritten ? place : nullptr, lane);
  }
}

// ---------------------------------------------------------------- fork
constexpr int ONE = 1024;                  // threads of the single workgroup that ranks rows

// exclusive rank of `flag` among the workgroup's threads, and the count of all
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

// order[k] = the k-th source that is a live row; the k-th free row becomes its copy
__global__ __launch_bounds__(ONE) void fork_rows_kernel(uint8_t* __restrict__ live, int rows, const int64_t* __restrict__ src, int n,
                                                        int64_t* __restrict__ ids, int32_t* __restrict__ order, int32_t* __restrict__ status) {
  __shared__ int lds[ONE / 64];
  const int tid = threadIdx.x;
  int wanted = 0;
  bool bad = false;
  for (int i0 = 0; i0 < n; i0 += ONE) {
    const int i = i0 + tid;
    bool ok = false;
    if (i < n) {
      ok = in_cache(src[i], rows) && live[src[i]] != 0;
      bad |= !ok;
      ids[i] = -1;
    }
    int all;
    const int k = rank_in_group(ok, &all, lds);
    if (ok) order[wanted + k] = i;
    wanted += all;
  }
  __syncthreads();                          // order and ids are complete, and no live flag has changed yet
  int found = 0;
  for (int r0 = 0; r0 < rows && found < wanted; r0 += ONE) {
    const int r = r0 + tid;
    const bool is_free = r < rows && live[r] == 0;
    int all;
    const int k = found + rank_in_group(is_free, &all, lds);
    if (is_free && k < wanted) {
      ids[order[k]] = r;
      live[r] = 1;
    }
    found += all;
  }
  if (status && bad) atomicOr(status, (int)UMT_STATUS_BAD_ROW);
  if (status && tid == 0 && found < wanted) atomicOr(status, (int)UMT_STATUS_NO_FREE_ROW);
}

// sources are live rows and targets were free ones, so no row is both
__global__ __launch_bounds__(RT) void fork_move_kernel(RowBuffers B, const int64_t* __restrict__ src, const int64_t* __restrict__ ids, int n) {
  const int lane = threadIdx.x & 63, pieces = B.piece0[B.n];
  const int64_t item = (int64_t)blockIdx.x * (RT / 64) + (threadIdx.x >> 6);
  const int64_t i = item / pieces;
  if (i >= n || ids[i] < 0) return;
  move_piece(B, (int)(item - i * pieces), ids[i], nullptr, src[i], nullptr, lane);
}

// ---------------------------------------------------------------- free
__global__ __launch_bounds__(RT) void free_rows_kernel(uint8_t* __restrict__ live, int rows, const int64_t* __restrict__ row_ids,
                                                       int n, int32_t* __restrict__ status) {
  const int i = blockIdx.x * RT + threadIdx.x;
  if (i >= n) return;
  const int64_t r = row_ids[i];
  if (in_cache(r, rows))
    live[r] = 0;
  else if (status)
    atomicOr(status, (int)UMT_STATUS_BAD_ROW);
}

// ---------------------------------------------------------------- compact
// moves: [0] = how many, then (hole, row) lists of rows entries each
__global__ __launch_bounds__(ONE) void compact_rows_kernel(uint8_t* __restrict__ live, int rows, int64_t* __restrict__ now,
                                                           int64_t* __restrict__ count, int32_t* __restrict__ moves) {
  __shared__ int lds[ONE / 64];
  const int tid = threadIdx.x;
  int mine = 0, c;
  for (int r = tid; r < rows; r += ONE) mine += live[r] != 0;
  rank_in_group(mine, &c, lds);
  int32_t *holes = moves + 4, *movers = holes + rows;
  int n_holes = 0, n_movers = 0;
  for (int r0 = 0; r0 < rows; r0 += ONE) {
    const int r = r0 + tid;
    const bool lv = r < rows && live[r] != 0;
    const bool hole = r < c && !lv, mover = r >= c && lv;
    int all;
    const int k = rank_in_group(hole | (mover << 16), &all, lds);
    if (hole) holes[n_holes + (k & 0xffff)] = r;
    if (mover) movers[n_movers + (k >> 16)] = r;
    n_holes += all & 0xffff;
    n_movers += all >> 16;
    if (r < rows) {
      if (!mover) now[r] = lv ? r : -1;
      live[r] = r < c;
    }
  }
  __syncthreads();                          // the lists are complete; n_holes == n_movers
  for (int k = tid; k < n_movers; k += ONE) now[movers[k]] = holes[k];
  if (tid == 0) {
    moves[0] = n_movers;
    *count = c;
  }
}

// rows at or above the live count move to free rows below it: no row is both
__global__ __launch_bounds__(RT) void compact_move_kernel(RowBuffers B, const int32_t* __restrict__ moves, int rows) {
  const int lane = threadIdx.x & 63, pieces = B.piece0[B.n];
  const int64_t n = (int64_t)moves[0] * pieces, stride = (int64_t)gridDim.x * (RT / 64);
  const int32_t *holes = moves + 4, *movers = holes + rows;
  for (int64_t item = (int64_t)blockIdx.x * (RT / 64) + (threadIdx.x >> 6); item < n; item += stride) {
    const int64_t k = item / pieces;
    move_piece(B, (int)(item - k * pieces), holes[k], nullptr, movers[k], nullptr, lane);
  }
}

static int row_buffers(const char* what, const umt_row_buffer* buffers, int n, int rows, RowBuffers* B) {
  UMT_REQUIRE(n > 0 && n <= UMT_ROW_BUFFERS_MAX && buffers && rows >= 0, UMT_ERR_INVALID, "%s: %d buffers of %d rows", what, n, rows);
  B->n = n;
  int64_t pieces = 0, off = 0;
  for (int k = 0; k < n; ++k) {
    const umt_row_buffer& b = buffers[k];
    UMT_REQUIRE((b.data || rows == 0) && b.row_bytes > 0 && b.row_bytes <= (1LL << 40), UMT_ERR_INVALID,
                "%s: buffer %d is null or its rows have %lld bytes", what, k, (long long)b.row_bytes);
    const uint64_t lo = (uint64_t)b.data, both = lo | (uint64_t)b.row_bytes;
    for (int j = 0; j < k && rows > 0; ++j) {
      const uint64_t o = (uint64_t)buffers[j].data;
      UMT_REQUIRE(o + (uint64_t)buffers[j].row_bytes * rows <= lo || lo + (uint64_t)b.row_bytes * rows <= o, UMT_ERR_INVALID,
                  "%s: buffers %d and %d overlap", what, j, k);
    }
    B->data[k] = (char*)b.data;
    B->bytes[k] = b.row_bytes;
    B->unit[k] = both % 16 == 0 ? 16 : both % 4 == 0 ? 4 : 1;
    B->staged[k] = off;
    off += round_up64(b.row_bytes, 16);
    B->piece0[k] = (int)pieces;
    pieces += (b.row_bytes + MOVE_BYTES - 1) / MOVE_BYTES;
    UMT_REQUIRE(pieces < (1 << 30), UMT_ERR_INVALID, "%s: rows of %lld bytes", what, (long long)b.row_bytes);
  }
  B->piece0[n] = (int)pieces;
  B->staged_bytes = off;
  return 0;
}

// workgroups of a move of n rows, a wave per piece
static int move_grid(const char* what, const RowBuffers& B, int64_t n, unsigned* grid) {
  const int64_t wg = (n * B.piece0[B.n] + RT / 64 - 1) / (RT / 64);
  UMT_REQUIRE(wg < (1LL << 31), UMT_ERR_INVALID, "%s: %lld rows of %d pieces", what, (long long)n, B.piece0[B.n]);
  *grid = (unsigned)wg;
  return 0;
}

static int need_workspace(const char* what, const void* ws, int64_t have, int64_t need) {
  UMT_REQUIRE(need == 0 || (ws && have >= need), UMT_ERR_WORKSPACE, "%s: workspace %lld < %lld bytes", what, (long long)have, (long long)need);
  return 0;
}

}  // namespace umt

using namespace umt;

extern "C" int64_t umt_rows_copy_workspace_bytes(const umt_row_buffer* buffers, int n_buffers, int rows, int n) {
  RowBuffers B;
  if (n < 0 || row_buffers("rows copy", buffers, n_buffers, rows, &B) != 0) return -1;
  return n == 0 || rows == 0 ? 0 : round_up64((int64_t)rows * 4, 16) + n * B.staged_bytes;
}

extern "C" int umt_rows_copy(const umt_row_buffer* buffers, int n_buffers, int rows, const int64_t* src, const int64_t* dst, int n,
                             int32_t* status, void* workspace, int64_t workspace_bytes, void* stream) {
  RowBuffers B;
  UMT_TRY(row_buffers("rows copy", buffers, n_buffers, rows, &B));
  UMT_REQUIRE(n >= 0 && (n == 0 || (src && dst)), UMT_ERR_INVALID, "rows copy: n=%d or null pointer", n);
  if (n == 0) return 0;
  UMT_TRY(need_workspace("rows copy", workspace, workspace_bytes, umt_rows_copy_workspace_bytes(buffers, n_buffers, rows, n)));
  unsigned grid = 0;
  UMT_TRY(move_grid("rows copy", B, n, &grid));
  hipStream_t s = (hipStream_t)stream;
  int32_t* last = (int32_t*)workspace;
  char* stage = (char*)workspace + round_up64((int64_t)rows * 4, 16);
  const dim3 per_pair((n + RT - 1) / RT);
  hipLaunchKernelGGL(copy_clear_kernel, per_pair, dim3(RT), 0, s, src, dst, n, rows, last, status);
  hipLaunchKernelGGL(copy_claim_kernel, per_pair, dim3(RT), 0, s, src, dst, n, rows, last);
  hipLaunchKernelGGL(copy_move_kernel<0>, dim3(grid), dim3(RT), 0, s, B, src, dst, n, rows, last, stage);
  hipLaunchKernelGGL(copy_move_kernel<1>, dim3(grid), dim3(RT), 0, s, B, src, dst, n, rows, last, stage);
  UMT_CHECK_HIP(hipGetLastError());
  return 0;
}

extern "C" int64_t umt_rows_fork_workspace_bytes(int rows, int n) { return rows < 0 || n < 0 ? -1 : (int64_t)n * 4; }

extern "C" int umt_rows_fork(const umt_row_buffer* buffers, int n_buffers, int rows, uint8_t* live, const int64_t* src, int n,
                             int64_t* ids, int32_t* status, void* workspace, int64_t workspace_bytes, void* stream) {
  RowBuffers B;
  UMT_TRY(row_buffers("rows fork", buffers, n_buffers, rows, &B));
  UMT_REQUIRE(n >= 0 && (n == 0 || (src && ids)) && (live || rows == 0), UMT_ERR_INVALID, "rows fork: n=%d or null pointer", n);
  if (n == 0) return 0;
  UMT_TRY(need_workspace("rows fork", workspace, workspace_bytes, umt_rows_fork_workspace_bytes(rows, n)));
  unsigned grid = 0;
  UMT_TRY(move_grid("rows fork", B, n, &grid));
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(fork_rows_kernel, dim3(1), dim3(ONE), 0, s, live, rows, src, n, ids, (int32_t*)workspace, status);
  hipLaunchKernelGGL(fork_move_kernel, dim3(grid), dim3(RT), 0, s, B, src, ids, n);
  UMT_CHECK_HIP(hipGetLastError());
  return 0;
}

extern "C" int umt_rows_free(uint8_t* live, int rows, const int64_t* row_ids, int n, int32_t* status, void* stream) {
  UMT_REQUIRE(n >= 0 && rows >= 0 && (n == 0 || row_ids) && (live || rows == 0), UMT_ERR_INVALID, "rows free: n=%d rows=%d or null pointer", n, rows);
  if (n == 0) return 0;
  hipLaunchKernelGGL(free_rows_kernel, dim3((n + RT - 1) / RT), dim3(RT), 0, (hipStream_t)stream, live, rows, row_ids, n, status);
  UMT_CHECK_HIP(hipGetLastError());
  return 0;
}

extern "C" int64_t umt_rows_compact_workspace_bytes(int rows) { return rows < 0 ? -1 : 16 + 8 * (int64_t)rows; }

extern "C" int umt_rows_compact(const umt_row_buffer* buffers, int n_buffers, int rows, uint8_t* live, int64_t* now, int64_t* count,
                                void* workspace, int64_t workspace_bytes, void* stream) {
  RowBuffers B;
  UMT_TRY(row_buffers("rows compact", buffers, n_buffers, rows, &B));
  UMT_REQUIRE((live && now && count) || (rows == 0 && count), UMT_ERR_INVALID, "rows compact: null pointer");
  UMT_TRY(need_workspace("rows compact", workspace, workspace_bytes, umt_rows_compact_workspace_bytes(rows)));
  hipStream_t s = (hipStream_t)stream;
  int32_t* moves = (int32_t*)workspace;
  hipLaunchKernelGGL(compact_rows_kernel, dim3(1), dim3(ONE), 0, s, live, rows, now, count, moves);
  if (rows > 1) {                           // at most half of the rows move
    unsigned grid = 0;
    UMT_TRY(move_grid("rows compact", B, rows / 2, &grid));
    hipLaunchKernelGGL(compact_move_kernel, dim3(grid < 4096 ? grid : 4096), dim3(RT), 0, s, B, moves, rows);
  }
  UMT_CHECK_HIP(hipGetLastError());
  return 0;
}
