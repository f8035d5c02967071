// Gated linear recurrence over recordings, its gradients, and its one-frame form over a cache of rows.
//
//   h[t] = a h[t-1] + c x[t],   a = sigmoid(gate), c = 1 - a = sigmoid(-gate)
//
// One lane owns one (row, feature); a wave loads UMT_GATED_KEEP steps of its 64 lanes at once, so neighbouring lanes read
// neighbouring features and 32 loads are in flight.  Where there are many lanes a wave walks the whole axis alone.  Where
// there are few, the waves of a workgroup take successive stretches of a tile (the recurrence over a stretch is itself a
// step, see join()), and beyond that the axis is cut into segments that workgroups of their own run, whose steps a first
// launch finds.  No order of arrival enters a result.
//
// Arithmetic.  With e = exp(-|gate|) the smaller of (a, c) is m = e / (1 + e), which keeps its relative precision however
// small it gets, and the larger one is 1 - m.  A step is base + m (other - base), where base is what the larger weight
// belongs to: one fma, and neither a slow decay (a near 1) nor the remainder of an old outlier (a near 0) is lost in
// 1 - m.  The sign bit of the stored m says which one the base is (set: the input).  A frame that is skipped is the step
// (x, m) = (0, +0), a dropped memory is m = -0 with the memory read as 0, so what lies under a mask enters nowhere.
#include "umt_internal.h"

#include <type_traits>

namespace umt {

constexpr int KEEP = UMT_GATED_KEEP;
constexpr int GT = 256;

__device__ __forceinline__ float as_value(float v) { return v; }
__device__ __forceinline__ float as_value(__bf16 v) { return (float)v; }
__device__ __forceinline__ float load_value(const float* p) { return *p; }
__device__ __forceinline__ float load_value(const __bf16* p) { return (float)*p; }
__device__ __forceinline__ void store_value(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_value(__bf16* p, float v) { *p = (__bf16)v; }   // one rounding, to nearest even

// The stored m of a gate.  exp2 of the rounded product |gate| log2(e) is off by up to |gate| + 2 units of 2^-24 relative,
// and as m <= exp(-|gate|) that is at most 1.5 such units absolute: less than the rounding of the state in the same step.
__device__ __forceinline__ float gate_step(float g) {
  const float e = __builtin_amdgcn_exp2f(-fabsf(g) * 1.44269504f);
  return copysignf(e * __builtin_amdgcn_rcpf(1.f + e), g);
}

__device__ __forceinline__ float advance(float h, float x, float m) {
  const bool from_x = __float_as_uint(m) >> 31;
  const float base = from_x ? x : h, other = from_x ? h : x;
  return fmaf(fabsf(m), other - base, base);
}

// all ones where bit j is set
__device__ __forceinline__ unsigned bit_mask(unsigned bits, int j) { return (unsigned)((int)(bits << (31 - j)) >> 31); }
__device__ __forceinline__ float masked_value(float v, unsigned mask) { return __uint_as_float(__float_as_uint(v) & mask); }
// the m of a masked step: keeps its value, +0 (skipped) or -0 (memory dropped)
__device__ __forceinline__ float masked_step(float m, unsigned use, unsigned valid) {
  return __uint_as_float((__float_as_uint(m) & valid & use) | (~use & 0x80000000u));
}

// backward factors of a step: c s and a s for the stored m
__device__ __forceinline__ float times_c(float m, float s) {
  const float p = fabsf(m) * s;
  return __float_as_uint(m) >> 31 ? s - p : p;
}
__device__ __forceinline__ float times_a(float m, float s) {
  const float p = fabsf(m) * s;
  return __float_as_uint(m) >> 31 ? p : s - p;
}

struct Masks {
  const uint8_t* use;
  const uint8_t* valid;
};

// A stretch of steps is a step itself: h_out = p + a h_in, with q = 1 - a carried on its own (the stretch's response to a
// memory of 0 and inputs of 1), because 1 - a of a rounded a has lost a slow decay.
struct Stretch {
  float a, q, p;
};
__device__ __forceinline__ float join(float h, const Stretch& s) {
  const float slow = h + fmaf(-s.q, h, s.p), fast = fmaf(s.a, h, s.p);
  return s.a == 0.f ? s.p : s.q <= 0.5f ? slow : fast;      // a = 0: the memory was dropped on the way, whatever h holds
}
__device__ __forceinline__ Stretch then(const Stretch& f, const Stretch& s) {
  return Stretch{f.a * s.a, join(f.q, Stretch{s.a, s.q, s.q}), join(f.p, s)};
}

// One stream of (t, row, feature) values as a wave addresses it: the step's place is the same in all lanes, a lane adds
// its distance from the wave's first row (OFF = 32 bits unless the rows lie further apart than that)
template <typename V, typename OFF>
struct Lanes {
  const V* at;             // step 0 of the wave's first row
  int64_t step;
  OFF mine;                // in bytes
  __device__ __forceinline__ V load(int64_t t) const {
    return *reinterpret_cast<const V*>(reinterpret_cast<const char*>(at + t * step) + mine);
  }
};

// Frame masks of KEEP steps, one bit a step.  Lane 16 k + j reads the byte of step j of the wave's row r0 + k and a ballot
// hands every lane the 16 bits of its own row: one load a stretch where a wave holds up to 4 rows, more only where the
// rows are shorter than that.
struct MaskLanes {
  const uint8_t* p;
  int64_t st, sr, r0;
  int rows, span, mine;    // rows of the call, rows of the wave, this lane's row among them
  __device__ __forceinline__ uint8_t fetch(int t0, int T, int k0) const {
    const int lane = threadIdx.x & 63;
    const int64_t r = r0 + k0 + (lane >> 4);
    const int t = t0 + (lane & 15);
    return p[(int64_t)(t < T ? t : T - 1) * st + (r < rows ? r : rows - 1) * sr];
  }
  // `first` = fetch(t0, T, 0), made ahead
  __device__ __forceinline__ unsigned bits(uint8_t first, int t0, int T) const {
    unsigned b = 0;
    for (int k0 = 0; k0 < span; k0 += 4) {
      const uint64_t all = __ballot((k0 ? fetch(t0, T, k0) : first) != 0);
      if ((mine >> 2) == (k0 >> 2)) b = (unsigned)(all >> (16 * (mine & 3))) & 0xffffu;
    }
    return b;
  }
};

// What one wave of the forward direction works on
template <typename V, typename OFF, bool MASK>
struct Walk {
  Lanes<V, OFF> x, g;
  MaskLanes um, vm;
  bool has_use, has_valid;
  int T;
  V rx[KEEP], rg[KEEP];
  uint8_t ru, rv;

  // e0: first element of the wave, e: this lane's (clamped into the call)
  __device__ __forceinline__ void place(const umt_gated_shape& S, const V* x_, const V* gate_, const Masks& mk, int64_t row0, int64_t row,
                                        int f, int gi, int64_t x_t, int64_t x_row) {
    T = S.t;
    x = {x_ + row0 * x_row, x_t, (OFF)(((row - row0) * x_row + f) * (int64_t)sizeof(V))};
    g = {gate_ + row0 * S.gate_row, S.gate_t, (OFF)(((row - row0) * S.gate_row + gi) * (int64_t)sizeof(V))};
    if (MASK) {
      const int mine = (int)(row - row0), span = __builtin_amdgcn_readfirstlane(wave_max(mine)) + 1;
      has_use = mk.use != nullptr;
      has_valid = mk.valid != nullptr;
      um = {mk.use, S.use_t, S.use_row, row0, S.rows, span, mine};
      vm = {mk.valid, S.valid_t, S.valid_row, row0, S.rows, span, mine};
    }
  }
  static __device__ __forceinline__ int wave_max(int v) {
    for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o));
    return v;
  }
  __device__ __forceinline__ void fetch(int t0) {
    if (MASK) {
      if (has_use) ru = um.fetch(t0, T, 0);
      if (has_valid) rv = vm.fetch(t0, T, 0);
    }
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
      const int t = t0 + j < T ? t0 + j : T - 1;
      rg[j] = g.load(t);
      rx[j] = x.load(t);
    }
  }
  // the fetched stretch: inputs, m of each step, mask bits (steps past the end are skipped frames)
  // back: xs are gradients, which no valid mask covers
  __device__ __forceinline__ void take(int t0, float (&xs)[KEEP], float (&ms)[KEEP], unsigned& ub, unsigned& vb, bool back) {
    ub = vb = 0xffffu;
    if (MASK) {
      if (has_use) ub = um.bits(ru, t0, T);
      if (has_valid) vb = vm.bits(rv, t0, T);
    }
    const int left = T - t0;
    unsigned past = 0;
    if (left < KEEP) {
      past = left <= 0 ? 0xffffu : 0xffffu << left & 0xffffu;
      ub |= past;
      vb &= ~past;
    }
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
      xs[j] = as_value(rx[j]);
      ms[j] = gate_step(as_value(rg[j]));
    }
    if (MASK || left < KEEP) {
#pragma unroll
      for (int j = 0; j < KEEP; ++j) {
        const unsigned v = bit_mask(vb, j);
        xs[j] = masked_value(xs[j], back ? ~bit_mask(past, j) : v);
        ms[j] = masked_step(ms[j], bit_mask(ub, j), v);
      }
    }
  }
};

template <bool MASK>
__device__ __forceinline__ float memory_of(float h, unsigned ub, int j) {
  return MASK ? masked_value(h, bit_mask(ub, j)) : h;
}

// Partners: the W waves of a workgroup take the KEEP-step stretches of a tile in turn; each hands its stretch over in LDS and
// joins those before it (after it, in the backward direction) to the state that entered the tile.
template <int W>
struct Partners {
  float (*lds)[W][3][64];
  int turn = 0;
  // state before this wave's stretch; `through` becomes the state behind the tile
  template <bool BACK>
  __device__ __forceinline__ float enter(const Stretch& mine, int tw, int lane, float& through) {
    float(*b)[3][64] = lds[turn];
    turn ^= 1;                              // two places: one barrier a tile
    b[tw][0][lane] = mine.a;
    b[tw][1][lane] = mine.q;
    b[tw][2][lane] = mine.p;
    __syncthreads();
    float cur = through, own = through;
    for (int i = 0; i < W; ++i) {
      const int w = BACK ? W - 1 - i : i;
      if (w == tw) own = cur;
      cur = join(cur, Stretch{b[w][0][lane], b[w][1][lane], b[w][2][lane]});
    }
    through = cur;
    return own;
  }
};

template <int W>
constexpr int group_threads() { return W == 1 ? GT : 64 * W; }

// the joined segments before (after) this one, [segment][a, q, p][lane] in `segs`: the waves join a run of them each
template <int W, bool BACK>
__device__ __forceinline__ float enter_segment(const float* __restrict__ segs, int seg, int n_segs, int64_t n, int64_t e, int tw, int lane,
                                               float first, Partners<W>& partners) {
  const int count = BACK ? n_segs - 1 - seg : seg, per = (count + W - 1) / W;
  const int a0 = min(count, tw * per), a1 = min(count, a0 + per);
  Stretch run{1.f, 0.f, 0.f};
  for (int i = a0; i < a1; ++i) {
    const float* s = segs + (int64_t)(BACK ? n_segs - 1 - i : i) * 3 * n + e;
    run = then(run, Stretch{s[0], s[n], s[2 * n]});
  }
  float through = first;
  partners.template enter<false>(run, tw, lane, through);
  return through;
}

template <typename V, typename OFF, int W, bool MASK>
__global__ __launch_bounds__(group_threads<W>()) void gated_scan_kernel(umt_gated_shape S, const V* __restrict__ x, const V* __restrict__ gate,
                                                                        Masks mk, const float* __restrict__ h0, const float* __restrict__ segs,
                                                                        int seg_tiles, V* __restrict__ h, float* __restrict__ h_last,
                                                                        float* __restrict__ kept) {
  __shared__ float lds[W > 1 ? 2 : 1][W][3][64];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int F = S.groups * S.share;
  const int64_t N = (int64_t)S.rows * F;
  const int64_t e0 = W == 1 ? ((int64_t)blockIdx.x * (GT / 64) + wv) * 64 : (int64_t)blockIdx.x * 64;
  const int tw = W == 1 ? 0 : wv;
  if (W == 1 && e0 >= N) return;
  const int64_t e = e0 + lane < N ? e0 + lane : N - 1;
  const bool on = e0 + lane < N;
  const int64_t row0 = e0 / F, row = e / F;
  const int f = (int)(e - row * F);
  Walk<V, OFF, MASK> w;
  w.place(S, x, gate, mk, row0, row, f, f / S.share, S.x_t, S.x_row);
  char* hp = reinterpret_cast<char*>(h + row0 * S.out_row);
  const OFF mine = (OFF)(((row - row0) * S.out_row + f) * (int64_t)sizeof(V));
  const int tiles = (S.t + KEEP * W - 1) / (KEEP * W);
  const int tile0 = blockIdx.y * seg_tiles, tile1 = min(tiles, tile0 + seg_tiles);
  w.fetch((tile0 * W + tw) * KEEP);
  float cur = h0 ? h0[e] : 0.f;
  Partners<W> partners{reinterpret_cast<float(*)[W][3][64]>(lds)};
  if (W > 1 && segs) cur = enter_segment<W, false>(segs, blockIdx.y, gridDim.y, N, e, tw, lane, cur, partners);
  for (int tile = tile0; tile < tile1; ++tile) {
    const int t0 = (tile * W + tw) * KEEP;
    float xs[KEEP], ms[KEEP];
    unsigned ub, vb;
    w.take(t0, xs, ms, ub, vb, false);
    if (tile + 1 < tile1) w.fetch(t0 + W * KEEP);
    float st = cur;
    if (W > 1) {
      Stretch own{1.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < KEEP; ++j) {
        own.a *= (__float_as_uint(ms[j]) >> 31) ? fabsf(ms[j]) : 1.f - ms[j];
        own.q = advance(memory_of<MASK>(own.q, ub, j), 1.f, ms[j]);
        own.p = advance(memory_of<MASK>(own.p, ub, j), xs[j], ms[j]);
      }
      st = partners.template enter<false>(own, tw, lane, cur);
      if (t0 >= S.t) continue;
    }
    if (kept && on) kept[(int64_t)(t0 / KEEP) * N + e] = st;
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
      st = advance(memory_of<MASK>(st, ub, j), xs[j], ms[j]);
      if (on && t0 + j < S.t) store_value(reinterpret_cast<V*>(hp + (int64_t)(t0 + j) * S.out_t * (int64_t)sizeof(V) + mine), st);
    }
    if (h_last && on && t0 + KEEP >= S.t) h_last[e] = st;
    if (W == 1) cur = st;
  }
}

// The steps that the first segments make of the state (of the gradient that enters from behind, for the last segments):
// a wave walks its share of the segment alone, the waves' stretches are joined at the end.
template <typename V, typename OFF, int W, bool MASK, bool BACK>
__global__ __launch_bounds__(64 * W) void gated_segment_kernel(umt_gated_shape S, const V* __restrict__ v, const V* __restrict__ gate, Masks mk,
                                                               int seg_tiles, int64_t v_t, int64_t v_row, float* __restrict__ segs) {
  __shared__ float lds[W][3][64];
  const int lane = threadIdx.x & 63, tw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int F = S.groups * S.share;
  const int64_t N = (int64_t)S.rows * F;
  const int64_t e0 = (int64_t)blockIdx.x * 64;
  const int64_t e = e0 + lane < N ? e0 + lane : N - 1;
  const int64_t row0 = e0 / F, row = e / F;
  const int f = (int)(e - row * F);
  Walk<V, OFF, MASK> w;
  w.place(S, v, gate, mk, row0, row, f, f / S.share, v_t, v_row);
  const int seg = blockIdx.y + (BACK ? 1 : 0);
  const int c0 = (seg * W + tw) * seg_tiles;               // stretches of this wave: c0 .. c0 + seg_tiles - 1
  Stretch own{1.f, 0.f, 0.f};
  w.fetch((BACK ? c0 + seg_tiles - 1 : c0) * KEEP);
  for (int k = 0; k < seg_tiles; ++k) {
    const int t0 = (BACK ? c0 + seg_tiles - 1 - k : c0 + k) * KEEP;
    float xs[KEEP], ms[KEEP];
    unsigned ub, vb;
    w.take(t0, xs, ms, ub, vb, BACK);
    if (k + 1 < seg_tiles) w.fetch(BACK ? t0 - KEEP : t0 + KEEP);
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
      const int j = BACK ? KEEP - 1 - i : i;
      own.a *= (__float_as_uint(ms[j]) >> 31) ? fabsf(ms[j]) : 1.f - ms[j];
      own.q = advance(memory_of<MASK>(own.q, ub, j), 1.f, ms[j]);
      own.p = BACK ? memory_of<MASK>(times_a(ms[j], xs[j] + own.p), ub, j) : advance(memory_of<MASK>(own.p, ub, j), xs[j], ms[j]);
    }
  }
  lds[tw][0][lane] = own.a;
  lds[tw][1][lane] = own.q;
  lds[tw][2][lane] = own.p;
  __syncthreads();
  if (tw != 0 || e0 + lane >= N) return;
  Stretch all{1.f, 0.f, 0.f};
  for (int i = 0; i < W; ++i) {
    const int k = BACK ? W - 1 - i : i;
    all = then(all, Stretch{lds[k][0][lane], lds[k][1][lane], lds[k][2][lane]});
  }
  float* o = segs + (int64_t)seg * 3 * N + e;
  o[0] = all.a;
  o[N] = all.q;
  o[2 * N] = all.p;
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

template <typename V, typename OFF, int W, bool MASK>
__global__ __launch_bounds__(group_threads<W>()) void gated_scan_backward_kernel(
    umt_gated_shape S, LaneMap L, const V* __restrict__ x, const V* __restrict__ gate, Masks mk, const float* __restrict__ kept,
    const V* __restrict__ dh, const float* __restrict__ dh_last, const float* __restrict__ segs, int seg_tiles, V* __restrict__ dx,
    V* __restrict__ dgate, float* __restrict__ part, float* __restrict__ dh0) {
  __shared__ float lds[W > 1 ? 2 : 1][W][3][64];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t wave = W == 1 ? (int64_t)blockIdx.x * (GT / 64) + wv : blockIdx.x;
  const int tw = W == 1 ? 0 : wv;
  if (wave >= L.waves) return;
  const int F = S.groups * S.share;
  const int64_t N = (int64_t)S.rows * F, G = (int64_t)S.rows * S.groups;
  // the wave's first group, and this lane's place in its group or piece
  int64_t group0, group;
  int pos, len, first;                     // place, length, and the feature of the group at which the piece starts
  if (L.pieces > 1) {
    group0 = group = wave / L.pieces;
    first = (int)(wave - group * L.pieces) * L.width;
    len = min(L.width, S.share - first);
    pos = lane;
  } else {
    group0 = wave * L.groups_per_wave;
    group = group0 + lane / S.share;
    first = 0;
    len = S.share;
    pos = lane % S.share;
  }
  const bool on = pos < len && group < G && (L.pieces > 1 || lane < L.groups_per_wave * S.share);
  group = on ? group : group0;
  const int64_t row0 = group0 / S.groups, row = group / S.groups;
  const int gi = (int)(group - row * S.groups);
  const int f = gi * S.share + (on ? first + pos : first);
  const int64_t e = row * F + f;
  Walk<V, OFF, MASK> w;
  w.place(S, x, gate, mk, row0, row, f, gi, S.x_t, S.x_row);
  const Lanes<V, OFF> d{dh + row0 * S.dh_row, S.dh_t, (OFF)(((row - row0) * S.dh_row + f) * (int64_t)sizeof(V))};
  char* dxp = dx ? reinterpret_cast<char*>(dx + row0 * S.out_row) : nullptr;
  const OFF mine = (OFF)(((row - row0) * S.out_row + f) * (int64_t)sizeof(V));
  const int tiles = (S.t + KEEP * W - 1) / (KEEP * W);
  const int tile0 = blockIdx.y * seg_tiles, tile1 = min(tiles, tile0 + seg_tiles);
  Partners<W> partners{reinterpret_cast<float(*)[W][3][64]>(lds)};
  float v = dh_last ? dh_last[e] : 0.f;
  if (W > 1 && segs) v = enter_segment<W, true>(segs, blockIdx.y, gridDim.y, N, e, tw, lane, v, partners);
  for (int tile = tile1 - 1; tile >= tile0; --tile) {
    const int t0 = (tile * W + tw) * KEEP;
    float q[KEEP], ms[KEEP], ds[KEEP];
    unsigned ub, vb;
    w.fetch(t0);
    V rd[KEEP];
#pragma unroll
    for (int j = 0; j < KEEP; ++j) rd[j] = d.load(t0 + j < S.t ? t0 + j : S.t - 1);
    float cur = t0 < S.t ? kept[(int64_t)(t0 / KEEP) * N + e] : 0.f;
    w.take(t0, q, ms, ub, vb, false);
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {        // the states again; q becomes c a (h[t-1] - x[t]), the slope over the gate
      const float am = fabsf(ms[j]), xv = q[j];
      cur = memory_of<MASK>(cur, ub, j);
      q[j] = fmaf(-am, am, am) * (cur - xv);
      if (MASK) q[j] = masked_value(q[j], bit_mask(ub & vb, j));
      cur = advance(cur, xv, ms[j]);
      ds[j] = t0 + j < S.t ? as_value(rd[j]) : 0.f;
    }
    float b = v;
    if (W > 1) {
      Stretch own{1.f, 0.f, 0.f};
#pragma unroll
      for (int j = KEEP - 1; j >= 0; --j) {
        own.a *= (__float_as_uint(ms[j]) >> 31) ? fabsf(ms[j]) : 1.f - ms[j];
        own.q = advance(memory_of<MASK>(own.q, ub, j), 1.f, ms[j]);
        own.p = memory_of<MASK>(times_a(ms[j], ds[j] + own.p), ub, j);
      }
      b = partners.template enter<true>(own, tw, lane, v);
      if (t0 >= S.t) continue;
    }
#pragma unroll
    for (int j = KEEP - 1; j >= 0; --j) {
      const int t = t0 + j;
      if (t >= S.t) continue;
      const float s = ds[j] + b;
      const float gx = masked_value(times_c(ms[j], s), MASK ? bit_mask(vb, j) : ~0u);
      b = memory_of<MASK>(times_a(ms[j], s), ub, j);
      if (on && dxp) store_value(reinterpret_cast<V*>(dxp + (int64_t)t * S.out_t * (int64_t)sizeof(V) + mine), gx);
      if (dgate) {
        const float slope = s * q[j];
        const float sum = group_sum(on && (!MASK || (ub & vb) >> j & 1) ? slope : 0.f, pos, len);
        if (on && pos == 0) {
          if (L.pieces > 1)
            part[((int64_t)t * G + group) * L.pieces + (wave - group * L.pieces)] = sum;
          else
            store_value(dgate + t * S.dgate_t + row * S.dgate_row + gi, sum);
        }
      }
    }
    if (on && dh0 && t0 == 0) dh0[e] = b;
    if (W == 1) v = b;
  }
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
  const unsigned use = has_row && (!A.use || A.use[b]) ? ~0u : 0u, valid = !A.valid || A.valid[b] ? ~0u : 0u;
  const float xv = masked_value(load_value(x + (int64_t)b * F + f), valid);
  const float m = masked_step(gate_step(load_value(gate + (int64_t)b * A.groups + f / A.share)), use, valid);
  const float hv = advance(masked_value(prev, use), xv, m);
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

// How the time axis is shared out.  `waves` = waves that 64 lanes each would make.  A wave that walks alone needs about four
// others on its CU to keep HBM busy; below that the workgroup's waves take turns, and where even 16 of them per 64 lanes
// leave CUs empty the axis is cut into segments of whole tiles, at the price of reading the inputs twice.
struct Split {
  int w, segs, seg_tiles;
};
static Split split_axis(int64_t waves, int t) {
  const int64_t stretches = t > 0 ? (t + KEEP - 1) / KEEP : 1;
  Split p{1, 1, 1};
  if (waves < 1024 && stretches > 1) p.w = waves >= 256 || stretches <= 4 ? 4 : 16;
  const int64_t tiles = (stretches + p.w - 1) / p.w;
  int64_t segs = 1;
  if (p.w == 16 && waves > 0 && waves < 128) segs = 256 / waves;
  if (segs > tiles / 2) segs = tiles / 2;
  if (segs < 1) segs = 1;
  p.seg_tiles = (int)((tiles + segs - 1) / segs);
  p.segs = (int)((tiles + p.seg_tiles - 1) / p.seg_tiles);
  return p;
}
static int64_t segment_floats(const umt_gated_shape& S, int64_t waves) {
  const Split p = split_axis(waves, S.t);
  return p.segs > 1 ? (int64_t)p.segs * 3 * S.rows * S.groups * S.share : 0;
}
static int64_t scan_waves(const umt_gated_shape& S) { return ((int64_t)S.rows * S.groups * S.share + 63) / 64; }

// whether a wave's lanes lie within 2^31 bytes of each other in every stream: 64 features are at most 64 rows
static bool near_rows(const umt_gated_shape& S, int64_t size) {
  const int F = S.groups * S.share;
  const int64_t rows = F >= 64 ? 2 : 64 / F + 2;
  const int64_t st[] = {S.x_row, S.gate_row, S.out_row, S.dh_row};
  for (int64_t r : st)
    if (r > ((1LL << 31) / size - F) / rows) return false;
  return true;
}

template <typename V, typename OFF, bool MASK>
static int launch_scan(const umt_gated_shape& S, const V* x, const V* gate, Masks mk, const float* h0, V* h, float* h_last, float* kept,
                       float* segs, hipStream_t s) {
  const int64_t waves = scan_waves(S);
  const Split p = split_axis(waves, S.t);
  const float* entering = p.segs > 1 ? segs : nullptr;
  if (p.w == 1) {
    hipLaunchKernelGGL((gated_scan_kernel<V, OFF, 1, MASK>), dim3((unsigned)((waves + 3) / 4)), dim3(GT), 0, s, S, x, gate, mk, h0, entering,
                       p.seg_tiles, h, h_last, kept);
  } else if (p.w == 4) {
    hipLaunchKernelGGL((gated_scan_kernel<V, OFF, 4, MASK>), dim3((unsigned)waves), dim3(256), 0, s, S, x, gate, mk, h0, entering,
                       p.seg_tiles, h, h_last, kept);
  } else {
    if (p.segs > 1)
      hipLaunchKernelGGL((gated_segment_kernel<V, OFF, 16, MASK, false>), dim3((unsigned)waves, p.segs - 1), dim3(1024), 0, s, S, x, gate, mk,
                         p.seg_tiles, S.x_t, S.x_row, segs);
    hipLaunchKernelGGL((gated_scan_kernel<V, OFF, 16, MASK>), dim3((unsigned)waves, p.segs), dim3(1024), 0, s, S, x, gate, mk, h0, entering,
                       p.seg_tiles, h, h_last, kept);
  }
  UMT_CHECK_HIP(hipGetLastError());
  return 0;
}

template <typename V, typename OFF, bool MASK>
static int launch_backward(const umt_gated_shape& S, const V* x, const V* gate, Masks mk, const float* kept, const V* dh,
                           const float* dh_last, V* dx, V* dgate, float* dh0, float* part, float* segs, hipStream_t s) {
  const LaneMap L = lane_map(S);
  const Split p = split_axis(L.waves, S.t);
  const float* entering = p.segs > 1 ? segs : nullptr;
  if (p.w == 1) {
    hipLaunchKernelGGL((gated_scan_backward_kernel<V, OFF, 1, MASK>), dim3((unsigned)((L.waves + 3) / 4)), dim3(GT), 0, s, S, L, x, gate, mk,
                       kept, dh, dh_last, entering, p.seg_tiles, dx, dgate, part, dh0);
  } else if (p.w == 4) {
    hipLaunchKernelGGL((gated_scan_backward_kernel<V, OFF, 4, MASK>), dim3((unsigned)L.waves), dim3(256), 0, s, S, L, x, gate, mk, kept, dh,
                       dh_last, entering, p.seg_tiles, dx, dgate, part, dh0);
  } else {
    if (p.segs > 1)
      hipLaunchKernelGGL((gated_segment_kernel<V, OFF, 16, MASK, true>), dim3((unsigned)scan_waves(S), p.segs - 1), dim3(1024), 0, s, S, dh,
                         gate, mk, p.seg_tiles, S.dh_t, S.dh_row, segs);
    hipLaunchKernelGGL((gated_scan_backward_kernel<V, OFF, 16, MASK>), dim3((unsigned)L.waves, p.segs), dim3(1024), 0, s, S, L, x, gate, mk,
                       kept, dh, dh_last, entering, p.seg_tiles, dx, dgate, part, dh0);
  }
  if (dgate && L.pieces > 1) {
    const int64_t n = (int64_t)S.t * S.rows * S.groups;
    hipLaunchKernelGGL((gate_parts_kernel<V>), dim3((unsigned)((n + GT - 1) / GT)), dim3(GT), 0, s, S, L.pieces, part, dgate);
  }
  UMT_CHECK_HIP(hipGetLastError());
  return 0;
}

static int64_t part_floats(const umt_gated_shape& S) {
  const LaneMap L = lane_map(S);
  return L.pieces > 1 ? (int64_t)S.t * S.rows * S.groups * L.pieces : 0;
}

// the kernel variants: value type, distance of the rows, masks
template <typename Call>
static int by_variant(const umt_gated_shape& S, bool masks, Call call) {
  const bool near = near_rows(S, S.dtype == UMT_VALUES_BF16 ? 2 : 4);
  auto typed = [&](auto v) {
    if (near) return masks ? call(v, (uint32_t)0, std::true_type()) : call(v, (uint32_t)0, std::false_type());
    return masks ? call(v, (uint64_t)0, std::true_type()) : call(v, (uint64_t)0, std::false_type());
  };
  return S.dtype == UMT_VALUES_BF16 ? typed((__bf16)0.f) : typed(0.f);
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
  return segment_floats(*shape, scan_waves(*shape)) * (int64_t)sizeof(float);
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
  const int64_t need = umt_gated_scan_workspace_bytes(shape);
  UMT_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), UMT_ERR_WORKSPACE, "gated scan: workspace %lld < %lld bytes",
              (long long)workspace_bytes, (long long)need);
  const Masks mk{use_memory, valid};
  return by_variant(S, use_memory || valid, [&](auto v, auto off, auto masked) {
    using V = decltype(v);
    return launch_scan<V, decltype(off), decltype(masked)::value>(S, (const V*)x, (const V*)gate, mk, h0, (V*)h, h_last, kept,
                                                                  (float*)workspace, s);
  });
}

extern "C" int64_t umt_gated_scan_backward_workspace_bytes(const umt_gated_shape* shape) {
  if (check_shape(shape, false) != 0) return -1;
  return (segment_floats(*shape, lane_map(*shape).waves) + part_floats(*shape)) * (int64_t)sizeof(float);
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
  float *part = (float*)workspace, *segs = part + part_floats(S);
  return by_variant(S, use_memory || valid, [&](auto v, auto off, auto masked) {
    using V = decltype(v);
    return launch_backward<V, decltype(off), decltype(masked)::value>(S, (const V*)x, (const V*)gate, mk, kept, (const V*)dh, dh_last, (V*)dx,
                                                                      (V*)dgate, dh0, part, segs, s);
  });
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
