// Gated linear recurrence over recordings, its gradients, and its one-frame form over a cache of rows.
//
//   h[t] = a h[t-1] + c x[t],   a = sigmoid(gate), c = 1 - a = sigmoid(-gate)
//
// One lane owns one (row, feature) and walks the time axis in stretches of UMT_GATED_KEEP steps whose loads are all in
// flight together; neighbouring lanes are neighbouring features, so every load of a wave is one run of memory.  There is
// nothing to reuse: the passes are bound by HBM once enough loads are in flight.
//
// Arithmetic.  With e = exp(-|gate|) the smaller of (a, c) is m = e / (1 + e), which keeps its relative precision however
// small it gets, and the larger one is 1 - m.  A step is base + m (other - base), where base is what the larger weight
// belongs to: one fma, and neither a slow decay (a near 1) nor the remainder of an old outlier (a near 0) is lost in
// 1 - m.  The sign bit of the stored m says which one the base is (set: the input).  m = 0 returns the base itself, so
// a masked frame or a dropped memory passes through exactly, whatever the other operand holds.
#include "umt_internal.h"

namespace umt {

constexpr int KEEP = UMT_GATED_KEEP;
constexpr int GT = 256;

__device__ __forceinline__ float load_value(const float* p) { return *p; }
__device__ __forceinline__ float load_value(const __bf16* p) { return (float)*p; }
__device__ __forceinline__ void store_value(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_value(__bf16* p, float v) { *p = (__bf16)v; }   // one rounding, to nearest even

// exp(-|g|) as exp2 of a product in two pieces: the first product's rounding, up to |g| 2^-24 of the result, is put back
__device__ __forceinline__ float gate_step(float g) {
  const float n = -fabsf(g);
  const float p = n * 1.44269504f;
  const float rest = fmaf(n, 1.44269504f, -p) + n * 1.925963e-8f;      // log2(e) = 1.44269504 + 1.9e-8
  const float e0 = __builtin_amdgcn_exp2f(p);
  const float e = e0 > 0.f ? fmaf(e0 * 0.6931472f, rest, e0) : e0;     // gate = +-inf or far: rest may be NaN
  return copysignf(e * __builtin_amdgcn_rcpf(1.f + e), g);
}

__device__ __forceinline__ float advance(float h, float x, float m) {
  const bool from_x = __float_as_uint(m) >> 31;
  const float am = fabsf(m), base = from_x ? x : h, other = from_x ? h : x;
  return am == 0.f ? base : fmaf(am, other - base, base);
}

// the step a mask asks for: hold = (x 0, m +0), drop = (x, m -0), both = (0, -0)
__device__ __forceinline__ void masked(bool use, bool valid, float& x, float& m) {
  x = valid ? x : 0.f;
  m = use ? (valid ? m : 0.f) : -0.f;
}

// backward factors of a step: c s, a s and c a for the stored m (masks folded in: m = +-0)
__device__ __forceinline__ float times_c(float m, float s) { return __float_as_uint(m) >> 31 ? fmaf(m, s, s) : m * s; }
__device__ __forceinline__ float times_a(float m, float s) { return __float_as_uint(m) >> 31 ? -m * s : fmaf(-m, s, s); }

struct Masks {
  const uint8_t* use;
  const uint8_t* valid;
};

// bits of one lane's stretch: bit j = mask[(t0 + j), row], steps past the end read as the last one
__device__ __forceinline__ unsigned mask_bits(const uint8_t* p, int64_t st, int t0, int T) {
  unsigned bits = 0;
#pragma unroll
  for (int j = 0; j < KEEP; ++j) {
    const int t = min(t0 + j, T - 1);
    bits |= (p[t * st] ? 1u : 0u) << j;
  }
  return bits;
}

template <typename V>
__global__ __launch_bounds__(GT) void gated_scan_kernel(umt_gated_shape S, const V* __restrict__ x, const V* __restrict__ gate,
                                                        Masks mk, const float* __restrict__ h0, V* __restrict__ h,
                                                        float* __restrict__ h_last, float* __restrict__ kept) {
  const int F = S.groups * S.share;
  const int64_t N = (int64_t)S.rows * F;
  const int64_t e = (int64_t)blockIdx.x * GT + threadIdx.x;
  if (e >= N) return;
  const int64_t row = e / F;
  const int f = (int)(e - row * F);
  const V* xp = x + row * S.x_row + f;
  const V* gp = gate + row * S.gate_row + f / S.share;
  V* hp = h + row * S.out_row + f;
  const uint8_t* up = mk.use ? mk.use + row * S.use_row : nullptr;
  const uint8_t* vp = mk.valid ? mk.valid + row * S.valid_row : nullptr;
  float cur = h0 ? h0[e] : 0.f;
  for (int t0 = 0; t0 < S.t; t0 += KEEP) {
    float xs[KEEP], ms[KEEP];
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
      const int t = min(t0 + j, S.t - 1);
      xs[j] = load_value(xp + t * S.x_t);
      ms[j] = load_value(gp + t * S.gate_t);
    }
    const unsigned ub = up ? mask_bits(up, S.use_t, t0, S.t) : ~0u, vb = vp ? mask_bits(vp, S.valid_t, t0, S.t) : ~0u;
    if (kept) kept[(int64_t)(t0 / KEEP) * N + e] = cur;
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
      float m = gate_step(ms[j]);
      masked(ub >> j & 1, vb >> j & 1, xs[j], m);
      if (t0 + j < S.t) {
        cur = advance(cur, xs[j], m);
        store_value(hp + (t0 + j) * S.out_t, cur);
      }
    }
  }
  if (h_last) h_last[e] = cur;
}

// Which features the lanes of a backward wave own.  share = 1: 64 in a row.  share <= 64: as many whole groups as fit, so
// that the sum over a group stays in its wave (21 landmarks of 3 coordinates: 63 lanes).  share > 64: one of `pieces` equal
// parts of one group; the parts' sums are added by a second launch in part order, so no order of arrival is in the result.
struct LaneMap {
  int pieces, width, groups_per_wave;     // pieces > 1: width = features of a piece
  int64_t waves;
};
static LaneMap lane_map(const umt_gated_shape& S) {
  LaneMap m{1, S.share, 1, 0};
  const int64_t G = (int64_t)S.rows * S.groups;
  if (S.share > 64) {
    m.pieces = (S.share + 63) / 64;
    m.width = (S.share + m.pieces - 1) / m.pieces;
    m.waves = G * m.pieces;
  } else {
    m.groups_per_wave = 64 / S.share;
    m.waves = (G + m.groups_per_wave - 1) / m.groups_per_wave;
  }
  return m;
}

// sum of the `len` lanes from this one on within its group or piece (`pos` = place in it): log2(len) exchanges in a fixed
// order, the group's first lane holds the whole sum
__device__ __forceinline__ float group_sum(float v, int pos, int len) {
  for (int o = 1; o < len; o <<= 1) {
    const float w = __shfl_down(v, o);
    v += pos + o < len ? w : 0.f;
  }
  return v;
}

template <typename V>
__global__ __launch_bounds__(GT) void gated_scan_backward_kernel(umt_gated_shape S, LaneMap L, const V* __restrict__ x,
                                                                 const V* __restrict__ gate, Masks mk,
                                                                 const float* __restrict__ kept, const V* __restrict__ dh,
                                                                 const float* __restrict__ dh_last, V* __restrict__ dx,
                                                                 V* __restrict__ dgate, float* __restrict__ part,
                                                                 float* __restrict__ dh0) {
  const int lane = threadIdx.x & 63;
  const int64_t wave = (int64_t)blockIdx.x * (GT / 64) + (threadIdx.x >> 6);
  if (wave >= L.waves) return;
  const int F = S.groups * S.share;
  const int64_t N = (int64_t)S.rows * F, G = (int64_t)S.rows * S.groups;
  int64_t group;
  int pos, len, first;                     // place in the group or piece, its length, feature of the piece's start in the group
  if (L.pieces > 1) {
    group = wave / L.pieces;
    first = (int)(wave - group * L.pieces) * L.width;
    len = min(L.width, S.share - first);
    pos = lane;
  } else {
    group = wave * L.groups_per_wave + lane / S.share;
    first = 0;
    len = S.share;
    pos = lane % S.share;
  }
  const bool on = pos < len && group < G && (L.pieces > 1 || lane < L.groups_per_wave * S.share);
  group = on ? group : G - 1;
  const int inner = on ? first + pos : S.share - 1;
  const int64_t row = group / S.groups;
  const int gi = (int)(group - row * S.groups);
  const int f = gi * S.share + inner;
  const int64_t e = row * F + f;
  const V* xp = x + row * S.x_row + f;
  const V* gp = gate + row * S.gate_row + gi;
  const V* dp = dh + row * S.dh_row + f;
  V* dxp = dx ? dx + row * S.out_row + f : nullptr;
  const uint8_t* up = mk.use ? mk.use + row * S.use_row : nullptr;
  const uint8_t* vp = mk.valid ? mk.valid + row * S.valid_row : nullptr;
  float v = dh_last ? dh_last[e] : 0.f;
  for (int t0 = (S.t - 1) / KEEP * KEEP; t0 >= 0; t0 -= KEEP) {
    float q[KEEP], ms[KEEP], ds[KEEP];
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
      const int t = min(t0 + j, S.t - 1);
      q[j] = load_value(xp + t * S.x_t);
      ms[j] = load_value(gp + t * S.gate_t);
      ds[j] = load_value(dp + t * S.dh_t);
    }
    const unsigned ub = up ? mask_bits(up, S.use_t, t0, S.t) : ~0u, vb = vp ? mask_bits(vp, S.valid_t, t0, S.t) : ~0u;
    float cur = kept[(int64_t)(t0 / KEEP) * N + e];
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {       // the states again; q becomes c a (h[t-1] - x[t]), the slope over the gate
      float m = gate_step(ms[j]), xv = q[j];
      masked(ub >> j & 1, vb >> j & 1, xv, m);
      const float am = fabsf(m);
      q[j] = am == 0.f ? 0.f : fmaf(-am, am, am) * (cur - xv);
      cur = advance(cur, xv, m);
      ms[j] = m;
    }
#pragma unroll
    for (int j = KEEP - 1; j >= 0; --j) {
      const int t = t0 + j;
      if (t >= S.t) continue;
      const float s = ds[j] + v;
      const float gx = (vb >> j & 1) ? times_c(ms[j], s) : 0.f;
      v = (ms[j] == 0.f && __float_as_uint(ms[j]) >> 31) ? 0.f : times_a(ms[j], s);
      if (on && dxp) store_value(dxp + t * S.out_t, gx);
      if (dgate) {
        const float sum = group_sum(on && q[j] != 0.f ? s * q[j] : 0.f, pos, len);
        if (on && pos == 0) {
          if (L.pieces > 1)
            part[((int64_t)t * G + group) * L.pieces + (wave - group * L.pieces)] = sum;
          else
            store_value(dgate + t * S.dgate_t + row * S.dgate_row + gi, sum);
        }
      }
    }
  }
  if (on && dh0) dh0[e] = v;
}

template <typename V>
__global__ __launch_bounds__(GT) void gate_parts_kernel(umt_gated_shape S, int pieces, const float* __restrict__ part,
                                                        V* __restrict__ dgate) {
  const int64_t G = (int64_t)S.rows * S.groups;
  const int64_t k = (int64_t)blockIdx.x * GT + threadIdx.x;
  if (k >= G * S.t) return;
  float s = 0.f;
  for (int p = 0; p < pieces; ++p) s += part[k * pieces + p];
  const int64_t t = k / G, g = k - t * G, row = g / S.groups;
  store_value(dgate + t * S.dgate_t + row * S.dgate_row + (g - row * S.groups), s);
}

// ---------------------------------------------------------------- one frame over a cache of rows
constexpr int STEP_SEG = 256;              // features one wave advances

// owner[r] = highest sample that names row r, named[r] = how many do; only rows that are named are touched
__global__ __launch_bounds__(GT) void step_clear_kernel(const int64_t* __restrict__ idx, int batch, int cache_rows,
                                                        int32_t* __restrict__ owner, int32_t* __restrict__ named) {
  const int b = blockIdx.x * GT + threadIdx.x;
  if (b >= batch) return;
  const int64_t r = idx[b];
  if (r < 0 || r >= cache_rows) return;
  owner[r] = -1;
  named[r] = 0;
}
__global__ __launch_bounds__(GT) void step_claim_kernel(const int64_t* __restrict__ idx, int batch, int cache_rows,
                                                        int32_t* __restrict__ owner, int32_t* __restrict__ named) {
  const int b = blockIdx.x * GT + threadIdx.x;
  if (b >= batch) return;
  const int64_t r = idx[b];
  if (r < 0 || r >= cache_rows) return;
  atomicMax(owner + r, b);                 // integers: the same whatever the order
  atomicAdd(named + r, 1);
}

struct StepArgs {
  const int64_t* idx;
  const uint8_t *use, *valid;
  int batch, groups, share, cache_rows, segs;
  float* state;
  const int32_t *owner, *named;
  int32_t* status;
};

template <typename V>
__device__ __forceinline__ float step_one(const StepArgs& A, const V* x, const V* gate, V* out, int b, int f, float prev, bool has_row) {
  const int F = A.groups * A.share;
  float xv = load_value(x + (int64_t)b * F + f);
  float m = gate_step(load_value(gate + (int64_t)b * A.groups + f / A.share));
  masked(has_row && (!A.use || A.use[b]), !A.valid || A.valid[b], xv, m);
  const float hv = advance(prev, xv, m);
  store_value(out + (int64_t)b * F + f, hv);
  return hv;
}

// One wave per (sample, segment of features).  A row that several samples name is advanced by the wave of the highest one:
// it reads the row once, computes the other samples' outputs from that, and writes the row last.
template <typename V>
__global__ __launch_bounds__(GT) void gated_step_kernel(StepArgs A, const V* __restrict__ x, const V* __restrict__ gate,
                                                        V* __restrict__ out) {
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * (GT / 64) + (threadIdx.x >> 6);
  const int b = (int)(item / A.segs), f0 = (int)(item - (int64_t)b * A.segs) * STEP_SEG;
  if (b >= A.batch) return;
  const int F = A.groups * A.share, f1 = min(F, f0 + STEP_SEG);
  const int64_t r = A.idx ? A.idx[b] : b;
  const bool has_row = r >= 0 && r < A.cache_rows;
  if (!has_row) {
    if (A.status && f0 == 0 && lane == 0) atomicOr(A.status, (int)UMT_STATUS_BAD_MEMORY_IDX);
    for (int f = f0 + lane; f < f1; f += 64) step_one(A, x, gate, out, b, f, 0.f, false);
    return;
  }
  bool shared = false;
  if (A.idx) {
    if (A.owner[r] != b) return;
    shared = A.named[r] > 1;
  }
  for (int f = f0 + lane; f < f1; f += 64) {
    float* sp = A.state + r * F + f;
    const float prev = *sp;
    if (shared)
      for (int o = 0; o < b; ++o)
        if (A.idx[o] == r) step_one(A, x, gate, out, o, f, prev, true);
    *sp = step_one(A, x, gate, out, b, f, prev, true);
  }
}

static int check_shape(const umt_gated_shape* S, bool backward) {
  UMT_REQUIRE(S, UMT_ERR_INVALID, "gated scan: null shape");
  UMT_REQUIRE(S->dtype == UMT_VALUES_F32 || S->dtype == UMT_VALUES_BF16, UMT_ERR_INVALID, "gated scan: dtype = %d", S->dtype);
  UMT_REQUIRE(S->t >= 0 && S->rows >= 0 && S->groups > 0 && S->share > 0, UMT_ERR_INVALID,
              "gated scan: t=%d rows=%d groups=%d share=%d", S->t, S->rows, S->groups, S->share);
  UMT_REQUIRE((int64_t)S->groups * S->share <= (1 << 24), UMT_ERR_INVALID, "gated scan: %d x %d features in a row", S->groups, S->share);
  UMT_REQUIRE((int64_t)S->rows * S->groups * S->share <= (1LL << 36), UMT_ERR_INVALID, "gated scan: %d rows of %d x %d features",
              S->rows, S->groups, S->share);
  UMT_REQUIRE(S->t <= (1 << 30) && (int64_t)S->rows * S->groups <= (1LL << 38) / (S->t > 0 ? S->t : 1), UMT_ERR_INVALID,
              "gated scan: %d steps of %d x %d gates", S->t, S->rows, S->groups);
  const int64_t st[] = {S->x_t, S->x_row, S->gate_t, S->gate_row, S->out_t, S->out_row, S->use_t, S->use_row, S->valid_t,
                        S->valid_row, S->dh_t, S->dh_row, S->dgate_t, S->dgate_row};
  for (int i = 0; i < (backward ? 14 : 10); ++i) UMT_REQUIRE(st[i] >= 0, UMT_ERR_INVALID, "gated scan: negative stride %lld", (long long)st[i]);
  return 0;
}

// a (t, rows, n) array that is written: one of the two strides steps over all of the other axis
static bool lies_apart(int64_t st_t, int64_t st_row, int t, int rows, int64_t n) {
  const bool rows_inner = (rows <= 1 || st_row >= n) && (t <= 1 || st_t >= (rows - 1) * st_row + n);
  const bool t_inner = (t <= 1 || st_t >= n) && (rows <= 1 || st_row >= (t - 1) * st_t + n);
  return rows_inner || t_inner;
}

static int copy_ends(float* to, const float* from, int64_t n, hipStream_t s);

__global__ __launch_bounds__(GT) void copy_or_zero_kernel(float* __restrict__ to, const float* __restrict__ from, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * GT + threadIdx.x;
  if (i < n) to[i] = from ? from[i] : 0.f;
}
static int copy_ends(float* to, const float* from, int64_t n, hipStream_t s) {
  if (!to || n == 0) return 0;
  hipLaunchKernelGGL(copy_or_zero_kernel, dim3((unsigned)((n + GT - 1) / GT)), dim3(GT), 0, s, to, from, n);
  UMT_CHECK_HIP(hipGetLastError());
  return 0;
}

template <typename V>
static int launch_scan(const umt_gated_shape& S, const void* x, const void* gate, Masks mk, const float* h0, void* h,
                       float* h_last, float* kept, hipStream_t s) {
  const int64_t N = (int64_t)S.rows * S.groups * S.share;
  hipLaunchKernelGGL((gated_scan_kernel<V>), dim3((unsigned)((N + GT - 1) / GT)), dim3(GT), 0, s, S, (const V*)x, (const V*)gate,
                     mk, h0, (V*)h, h_last, kept);
  UMT_CHECK_HIP(hipGetLastError());
  return 0;
}

template <typename V>
static int launch_backward(const umt_gated_shape& S, const void* x, const void* gate, Masks mk, const float* kept, const void* dh,
                           const float* dh_last, void* dx, void* dgate, float* dh0, float* part, hipStream_t s) {
  const LaneMap L = lane_map(S);
  const int waves = GT / 64;
  hipLaunchKernelGGL((gated_scan_backward_kernel<V>), dim3((unsigned)((L.waves + waves - 1) / waves)), dim3(GT), 0, s, S, L,
                     (const V*)x, (const V*)gate, mk, kept, (const V*)dh, dh_last, (V*)dx, (V*)dgate, part, dh0);
  if (dgate && L.pieces > 1) {
    const int64_t n = (int64_t)S.t * S.rows * S.groups;
    hipLaunchKernelGGL((gate_parts_kernel<V>), dim3((unsigned)((n + GT - 1) / GT)), dim3(GT), 0, s, S, L.pieces, part, (V*)dgate);
  }
  UMT_CHECK_HIP(hipGetLastError());
  return 0;
}

template <typename V>
static int launch_step(const StepArgs& A, const void* x, const void* gate, void* out, hipStream_t s) {
  const int64_t items = (int64_t)A.batch * A.segs;
  const int waves = GT / 64;
  hipLaunchKernelGGL((gated_step_kernel<V>), dim3((unsigned)((items + waves - 1) / waves)), dim3(GT), 0, s, A, (const V*)x,
                     (const V*)gate, (V*)out);
  UMT_CHECK_HIP(hipGetLastError());
  return 0;
}

}  // namespace umt

using namespace umt;

extern "C" int64_t umt_gated_scan_workspace_bytes(const umt_gated_shape* shape) {
  if (check_shape(shape, false) != 0) return -1;
  return 0;
}

extern "C" int umt_gated_scan(const umt_gated_shape* shape, const void* x, const void* gate, const uint8_t* use_memory,
                              const uint8_t* valid, const float* h0, void* h, float* h_last, float* kept, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  UMT_TRY(check_shape(shape, false));
  const umt_gated_shape& S = *shape;
  const int64_t N = (int64_t)S.rows * S.groups * S.share;
  hipStream_t s = (hipStream_t)stream;
  if (N == 0) return 0;
  if (S.t == 0) return copy_ends(h_last, h0, N, s);
  UMT_REQUIRE(x && gate && h, UMT_ERR_INVALID, "gated scan: null pointer");
  UMT_REQUIRE(lies_apart(S.out_t, S.out_row, S.t, S.rows, (int64_t)S.groups * S.share), UMT_ERR_INVALID,
              "gated scan: the output's strides %lld, %lld overlap", (long long)S.out_t, (long long)S.out_row);
  (void)workspace;
  (void)workspace_bytes;
  const Masks mk{use_memory, valid};
  return S.dtype == UMT_VALUES_BF16 ? launch_scan<__bf16>(S, x, gate, mk, h0, h, h_last, kept, s)
                                    : launch_scan<float>(S, x, gate, mk, h0, h, h_last, kept, s);
}

extern "C" int64_t umt_gated_scan_backward_workspace_bytes(const umt_gated_shape* shape) {
  if (check_shape(shape, false) != 0) return -1;
  const LaneMap L = lane_map(*shape);
  return L.pieces > 1 ? (int64_t)shape->t * shape->rows * shape->groups * L.pieces * (int64_t)sizeof(float) : 0;
}

extern "C" int umt_gated_scan_backward(const umt_gated_shape* shape, const void* x, const void* gate, const uint8_t* use_memory,
                                       const uint8_t* valid, const float* kept, const void* dh, const float* dh_last, void* dx,
                                       void* dgate, float* dh0, void* workspace, int64_t workspace_bytes, void* stream) {
  UMT_TRY(check_shape(shape, true));
  const umt_gated_shape& S = *shape;
  const int64_t N = (int64_t)S.rows * S.groups * S.share;
  hipStream_t s = (hipStream_t)stream;
  if (N == 0) return 0;
  if (S.t == 0) return copy_ends(dh0, dh_last, N, s);
  UMT_REQUIRE(x && gate && kept && dh, UMT_ERR_INVALID, "gated scan backward: null pointer");
  UMT_REQUIRE(!dx || lies_apart(S.out_t, S.out_row, S.t, S.rows, (int64_t)S.groups * S.share), UMT_ERR_INVALID,
              "gated scan backward: dx's strides %lld, %lld overlap", (long long)S.out_t, (long long)S.out_row);
  UMT_REQUIRE(!dgate || lies_apart(S.dgate_t, S.dgate_row, S.t, S.rows, S.groups), UMT_ERR_INVALID,
              "gated scan backward: dgate's strides %lld, %lld overlap", (long long)S.dgate_t, (long long)S.dgate_row);
  const int64_t need = umt_gated_scan_backward_workspace_bytes(shape);
  UMT_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), UMT_ERR_WORKSPACE, "gated scan backward: workspace %lld < %lld bytes",
              (long long)workspace_bytes, (long long)need);
  const Masks mk{use_memory, valid};
  return S.dtype == UMT_VALUES_BF16
             ? launch_backward<__bf16>(S, x, gate, mk, kept, dh, dh_last, dx, dgate, dh0, (float*)workspace, s)
             : launch_backward<float>(S, x, gate, mk, kept, dh, dh_last, dx, dgate, dh0, (float*)workspace, s);
}

extern "C" int64_t umt_gated_step_workspace_bytes(int batch, int cache_rows) {
  return batch > 0 && cache_rows > 0 ? 2 * (int64_t)cache_rows * (int64_t)sizeof(int32_t) : 0;
}

extern "C" int umt_gated_step(int dtype, const void* x, const void* gate, const int64_t* memory_idx, const uint8_t* use_memory,
                              const uint8_t* valid, int batch, int groups, int share, float* state, int cache_rows, void* out,
                              int32_t* status, void* workspace, int64_t workspace_bytes, void* stream) {
  UMT_REQUIRE(dtype == UMT_VALUES_F32 || dtype == UMT_VALUES_BF16, UMT_ERR_INVALID, "gated step: dtype = %d", dtype);
  UMT_REQUIRE(batch >= 0 && cache_rows >= 0 && groups > 0 && share > 0 && (int64_t)groups * share <= (1 << 24), UMT_ERR_INVALID,
              "gated step: batch=%d cache_rows=%d groups=%d share=%d", batch, cache_rows, groups, share);
  if (batch == 0) return 0;
  UMT_REQUIRE(x && gate && out && (state || cache_rows == 0), UMT_ERR_INVALID, "gated step: null pointer");
  UMT_REQUIRE(memory_idx || batch <= cache_rows, UMT_ERR_INVALID, "gated step: %d samples and %d rows without memory_idx", batch, cache_rows);
  const int64_t need = memory_idx ? umt_gated_step_workspace_bytes(batch, cache_rows) : 0;
  UMT_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), UMT_ERR_WORKSPACE, "gated step: workspace %lld < %lld bytes",
              (long long)workspace_bytes, (long long)need);
  const int F = groups * share, segs = (F + STEP_SEG - 1) / STEP_SEG;
  UMT_REQUIRE((int64_t)batch * segs <= (1LL << 32), UMT_ERR_INVALID, "gated step: %d samples of %d features", batch, F);
  hipStream_t s = (hipStream_t)stream;
  int32_t *owner = (int32_t*)workspace, *named = owner + cache_rows;
  if (memory_idx && cache_rows > 0) {
    const dim3 grid((batch + GT - 1) / GT);
    hipLaunchKernelGGL(step_clear_kernel, grid, dim3(GT), 0, s, memory_idx, batch, cache_rows, owner, named);
    hipLaunchKernelGGL(step_claim_kernel, grid, dim3(GT), 0, s, memory_idx, batch, cache_rows, owner, named);
  }
  const StepArgs A{memory_idx, use_memory, valid, batch, groups, share, cache_rows, segs, state, owner, named, status};
  return dtype == UMT_VALUES_BF16 ? launch_step<__bf16>(A, x, gate, out, s) : launch_step<float>(A, x, gate, out, s);
}
