// Gated linear recurrence over recordings, its gradients, and its one-frame form over a cache of rows.
//
//   h[t] = a h[t-1] + c x[t],   a = sigmoid(gate), c = 1 - a = sigmoid(-gate)
//
// About 8 operations a value against 6 to 12 bytes: bound by HBM where the call is large, by the launch where it is small.
// One lane owns one (row, feature), or two neighbouring ones of bfloat16 where they can be loaded together (pairs()); a wave
// loads UMT_GATED_KEEP steps of its 64 lanes at once, so neighbouring lanes read neighbouring features and 32 loads are in
// flight.  Where there are many lanes a wave walks the whole axis alone.  Where there are fewer, the waves of a workgroup
// take successive stretches of a tile (the recurrence over a stretch is itself a step, see join()).  Where there are few,
// the axis is cut into runs, a wave each: a first launch finds the step that each run is, a second one walks the runs from
// the states they begin with.  No order of arrival enters a result, and no workgroup waits for another.
//
// Arithmetic.  With e = exp(-|gate|) the smaller of (a, c) is m = e / (1 + e), which keeps its relative precision however
// small it gets, and the larger one is 1 - m.  A step is base + m (other - base), where base is what the larger weight
// belongs to: one fma, and neither a slow decay (a near 1) nor the remainder of an old outlier (a near 0) is lost in
// 1 - m.  It is formed as base + w (other / 2 - base / 2), w = 2 m: the same roundings (but for the last bit below 2^-125),
// and two finite values at the two ends of the range do not make an infinite difference.  The sign bit of the stored w says
// which one the base is (set: the input).  A frame that is skipped is the step (x, w) = (0, +0), a dropped memory is w = -0
// with the memory read as 0, so what lies under a mask enters nowhere.
#include "umt_internal.h"

#include <algorithm>
#include <type_traits>

namespace umt {

constexpr int KEEP = UMT_GATED_KEEP;
constexpr int GT = 256;
constexpr int RUN_WAVES = 8;               // runs of a workgroup

// E values that a lane loads and stores as one
template <typename V, int E>
struct Values;
template <>
struct Values<float, 1> {
  using Raw = float;
  static __device__ __forceinline__ void open(Raw r, float (&v)[1]) { v[0] = r; }
  static __device__ __forceinline__ Raw close(const float (&v)[1]) { return v[0]; }
};
template <>
struct Values<__bf16, 1> {
  using Raw = __bf16;
  static __device__ __forceinline__ void open(Raw r, float (&v)[1]) { v[0] = (float)r; }
  static __device__ __forceinline__ Raw close(const float (&v)[1]) { return (__bf16)v[0]; }      // one rounding, to nearest even
};
template <>
struct Values<__bf16, 2> {
  using Raw = uint32_t;
  static __device__ __forceinline__ void open(Raw r, float (&v)[2]) {
    v[0] = __uint_as_float(r << 16);
    v[1] = __uint_as_float(r & 0xffff0000u);
  }
  static __device__ __forceinline__ Raw close(const float (&v)[2]) {
    const __bf16 a = (__bf16)v[0], b = (__bf16)v[1];
    return (uint32_t)__builtin_bit_cast(uint16_t, a) | (uint32_t)__builtin_bit_cast(uint16_t, b) << 16;
  }
};
__device__ __forceinline__ float load_value(const float* p) { return *p; }
__device__ __forceinline__ float load_value(const __bf16* p) { return (float)*p; }
__device__ __forceinline__ void store_value(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_value(__bf16* p, float v) { *p = (__bf16)v; }   // one rounding, to nearest even

// The stored w = 2 m of a gate.  exp2 of the rounded product |gate| log2(e) is off by up to |gate| + 2 units of 2^-24
// relative, and as m <= exp(-|gate|) that is at most 1.5 such units absolute: less than the rounding of the state in the
// same step.
__device__ __forceinline__ float gate_step(float g) {
  const float e = __builtin_amdgcn_exp2f(-fabsf(g) * 1.44269504f);
  return copysignf(e * __builtin_amdgcn_rcpf(fmaf(0.5f, e, 0.5f)), g);
}
__device__ __forceinline__ bool from_input(float w) { return __float_as_uint(w) >> 31; }

// (h - x) / 2
__device__ __forceinline__ float half_apart(float h, float x) { return fmaf(0.5f, h, -0.5f * x); }
// An infinite base is what comes out: its difference is made from a finite one, as inf - inf is none.  (Two operations a value
// more than advance_finite: 230 -> 232 us for 512 steps of 512 rows of 648 bf16 values.)
constexpr float LARGEST = 3.402823466e38f;
__device__ __forceinline__ float advance(float h, float x, float w) {
  const float base = from_input(w) ? x : h, other = from_input(w) ? h : x;
  return fmaf(fabsf(w), half_apart(other, __builtin_amdgcn_fmed3f(base, -LARGEST, LARGEST)), base);
}
// the same bits where all is finite; an infinite base makes NaN
__device__ __forceinline__ float advance_finite(float h, float x, float w) { return fmaf(-w, half_apart(h, x), from_input(w) ? x : h); }

// all ones where bit j is set
__device__ __forceinline__ unsigned bit_mask(unsigned bits, int j) { return (unsigned)((int)(bits << (31 - j)) >> 31); }
__device__ __forceinline__ float masked_value(float v, unsigned mask) { return __uint_as_float(__float_as_uint(v) & mask); }
// the w of a masked step: keeps its value, +0 (skipped) or -0 (memory dropped)
__device__ __forceinline__ float masked_step(float w, unsigned use, unsigned valid) {
  return __uint_as_float((__float_as_uint(w) & valid & use) | (~use & 0x80000000u));
}
template <bool MASK>
__device__ __forceinline__ float memory_of(float h, unsigned ub, int j) {
  return MASK ? masked_value(h, bit_mask(ub, j)) : h;
}

// backward factors of a step: c s and a s for its signed m
__device__ __forceinline__ float times_c(float m, float s) {
  const float p = fabsf(m) * s;
  return from_input(m) ? s - p : p;
}
__device__ __forceinline__ float times_a(float m, float s) {
  const float p = fabsf(m) * s;
  return from_input(m) ? p : s - p;
}

// Both weights of a gate, a = 1 / (1 + e) and c = e a with e = exp(-gate), each to a few units of 2^-24 of itself.  The
// exponent stops at 2^126, where c is 1 and a as good as 0.
struct Weights {
  float a, c;
  static __device__ __forceinline__ Weights of_gate(float g) {
    const float e = __builtin_amdgcn_exp2f(__builtin_elementwise_minimum(g * -1.44269504f, 126.f));     // NaN stays NaN
    const float a = __builtin_amdgcn_rcpf(1.f + e);
    return {a, e * a};
  }
  static __device__ __forceinline__ Weights of_step(float m) {
    const float s = fabsf(m), l = 1.f - s;
    return {from_input(m) ? s : l, from_input(m) ? l : s};
  }
  // skipped: (1, 0); memory dropped: (0, 1)
  __device__ __forceinline__ Weights masked(unsigned use, unsigned valid) const {
    return {__uint_as_float(((__float_as_uint(a) & valid) | (~valid & 0x3f800000u)) & use),
            __uint_as_float((__float_as_uint(c) & valid & use) | (~use & 0x3f800000u))};
  }
};

// A stretch of steps is a step itself: h_out = p + a h_in.  q = 1 - a is carried on its own (the stretch's response to a
// memory of 0 and inputs of 1: sums of positive terms), because 1 - a of a rounded a has lost a slow decay.  p and q are
// made of the same weights, so a constant input keeps its value whatever their rounding.
struct Stretch {
  float a, q, p;
  template <bool MASK>
  __device__ __forceinline__ void forward(float x, const Weights& w, unsigned use) {
    a *= w.a;
    q = fmaf(w.a, q, w.c);
    p = fmaf(w.a, MASK ? masked_value(p, use) : p, w.c * x);
  }
  template <bool MASK>
  __device__ __forceinline__ void backward(float d, const Weights& w, unsigned use) {
    a *= w.a;
    q = fmaf(w.a, q, w.c);
    p = w.a * (d + p);
    if (MASK) p = masked_value(p, use);
  }
  // a = 0 is kept for a memory that was dropped (`ub`: the use bits of all steps): one that has merely faded below every
  // float still hands on what is not finite
  __device__ __forceinline__ void close(unsigned ub) { a = (ub & 0xffffu) != 0xffffu ? 0.f : fmaxf(a, FADED); }
  static constexpr float FADED = 1.4e-45f;
};
__device__ __forceinline__ float join(float h, const Stretch& s) {
  const float slow = h + fmaf(-s.q, h, s.p), fast = fmaf(s.a, h, s.p);       // an infinite h would meet itself in the slow one
  return s.a == 0.f ? s.p : s.q <= 0.5f && fabsf(h) <= LARGEST ? slow : fast; // a = 0: the memory was dropped on the way, whatever h holds
}
__device__ __forceinline__ Stretch then(const Stretch& f, const Stretch& s) {
  const float a = f.a == 0.f || s.a == 0.f ? 0.f : fmaxf(f.a * s.a, Stretch::FADED);
  return Stretch{a, join(f.q, Stretch{s.a, s.q, s.q}), join(f.p, s)};
}

struct Masks {
  const uint8_t* use;
  const uint8_t* valid;
};

using Global = __attribute__((address_space(1))) char*;     // or the integers below would make them generic addresses
__device__ __forceinline__ Global uniform(const void* p) {  // into scalar registers: the same in all lanes of the wave
  const uint64_t v = (uint64_t)p;
  return (Global)(((uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) |
                  (unsigned)__builtin_amdgcn_readfirstlane((int)v));
}

// One stream of (t, row, feature) values as a wave addresses it: a step's place is the same in all lanes, a lane adds its
// distance from the wave's first row (OFF = 32 bits unless steps or rows lie further apart than that)
template <typename V, int E, typename OFF>
struct Lanes {
  using Raw = typename Values<V, E>::Raw;
  using At = __attribute__((address_space(1))) Raw*;
  Global at;               // step 0 of the wave's first row
  OFF step, mine;          // bytes
  __device__ __forceinline__ Lanes(const V* p, int64_t t_stride, int64_t row_stride, int64_t row0, int64_t row, int64_t inner) {
    at = uniform(p + row0 * row_stride);
    step = (OFF)(t_stride * (int64_t)sizeof(V));
    mine = (OFF)(((row - row0) * row_stride + inner) * (int64_t)sizeof(V));
  }
  // `mine`, hidden from the compiler, which would add it to `at` ahead of the loops and then address every step by 64-bit
  // vector additions instead of a scalar base and a 32-bit offset
  __device__ __forceinline__ OFF here() const {
    OFF m = mine;
    asm volatile("" : "+v"(m));
    return m;
  }
  // steps t0 .. t0 + KEEP - 1; those past the end read the last one
  __device__ __forceinline__ void load(int t0, int T, Raw (&r)[KEEP]) const {
    Global p = at + (int64_t)(t0 < T ? t0 : T - 1) * (int64_t)step;
    const int more = T - 1 - t0;            // steps that follow the first
    const OFF m = here();
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
      r[j] = *(At)(p + m);
      p += j < more ? step : (OFF)0;
    }
  }
  __device__ __forceinline__ Global step_at(int t) const { return at + (int64_t)t * (int64_t)step; }
  __device__ __forceinline__ void store_at(Global p, OFF m, const float (&v)[E]) const { *(At)(p + m) = Values<V, E>::close(v); }
  __device__ __forceinline__ void store(int t0, int T, bool on, const float (&v)[KEEP][E]) const {
    Global p = at + (int64_t)t0 * (int64_t)step;
    if (!on) return;
    const OFF m = here();
    if (t0 + KEEP <= T) {
#pragma unroll
      for (int j = 0; j < KEEP; ++j, p += step) *(At)(p + m) = Values<V, E>::close(v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < KEEP; ++j, p += step)
        if (t0 + j < T) *(At)(p + m) = Values<V, E>::close(v[j]);
    }
  }
};

// Frame masks of KEEP steps, one bit a step.  Lane 16 k + j reads the byte of step j of the wave's row r0 + k and a ballot
// hands every lane the 16 bits of its own row: one load a stretch where a wave holds up to 4 rows, more only where the
// rows are shorter than that.
struct MaskLanes {
  const uint8_t* p;        // this lane's byte of step 0, of row r0 + lane / 16
  int64_t st, sr;
  __device__ __forceinline__ MaskLanes() = default;
  __device__ __forceinline__ MaskLanes(const uint8_t* m, int64_t st_, int64_t sr_, int64_t r0) : st(st_), sr(sr_) {
    p = m ? m + (r0 + ((threadIdx.x & 63) >> 4)) * sr_ : nullptr;
  }
  // rows past the call's last are not read (they have no lanes)
  __device__ __forceinline__ uint8_t fetch(int t0, int T, int k0, int rows) const {
    const int lane = threadIdx.x & 63, t = min(t0 + (lane & 15), T - 1);
    return k0 + (lane >> 4) < rows ? p[(int64_t)t * st + k0 * sr] : 0;
  }
  // `first` = fetch(t0, T, 0, rows), made ahead; rows: of the wave, from its first on; mine: this lane's
  __device__ __forceinline__ unsigned bits(uint8_t first, int t0, int T, int rows, int mine) const {
    unsigned b = 0;
    for (int k0 = 0; k0 < rows; k0 += 4) {
      const uint64_t all = __ballot((k0 ? fetch(t0, T, k0, rows) : first) != 0);
      if ((mine >> 2) == (k0 >> 2)) b = (unsigned)(all >> (16 * (mine & 3))) & 0xffffu;
    }
    return b;
  }
};

// The (row, feature) of a lane's first value.  A wave owns `per` consecutive values, from wave * per on; lanes without any
// stand in for the wave's first and write nothing.
template <int E, typename OFF>
struct Place {
  using Index = std::conditional_t<sizeof(OFF) == 4, uint32_t, int64_t>;      // 32-bit divisions where they do
  int64_t e0, e, row0, row;
  int f, gi;
  bool on;
  __device__ __forceinline__ Place(const umt_gated_shape& S, int64_t wave, int per) {
    const int mine = (threadIdx.x & 63) * E;
    const Index F = (Index)(S.groups * S.share), N = (Index)S.rows * F, first = (Index)wave * (Index)per, i = first + (Index)mine;
    on = mine < per && i < N;
    const Index k = on ? i : first, r0 = first / F, r = k / F;
    e0 = first;
    e = k;
    row0 = r0;
    row = r;
    f = (int)(k - r * F);
    gi = f / S.share;
  }
};

// The two streams that both directions go by (an input and its gate, GE = 2 gates for 2 values, 1 for all) with the masks
template <typename V, int E, int GE, typename OFF, bool MASK>
struct Walk {
  using X = Lanes<V, E, OFF>;
  using G = Lanes<V, GE, OFF>;
  // a stretch on its way
  struct Fetched {
    typename X::Raw x[KEEP];
    typename G::Raw g[KEEP];
    uint8_t use, valid;
  };
  X x;
  G g;
  MaskLanes um, vm;
  int T, rows, mine;       // rows of the wave, this lane's among them

  __device__ __forceinline__ Walk(const umt_gated_shape& S, const Place<E, OFF>& at, const V* x_, int64_t x_t, int64_t x_row, const V* gate_,
                                  const Masks& mk)
      : x(x_, x_t, x_row, at.row0, at.row, at.f), g(gate_, S.gate_t, S.gate_row, at.row0, at.row, at.gi), T(S.t) {
    if (MASK) {
      int span = mine = (int)(at.row - at.row0);
      for (int o = 32; o > 0; o >>= 1) span = max(span, __shfl_xor(span, o));
      rows = __builtin_amdgcn_readfirstlane(span) + 1;
      um = MaskLanes(mk.use, S.use_t, S.use_row, at.row0);
      vm = MaskLanes(mk.valid, S.valid_t, S.valid_row, at.row0);
    }
  }
  __device__ __forceinline__ void fetch(int t0, const Masks& mk, Fetched& r) const {
    if (MASK) {
      if (mk.use) r.use = um.fetch(t0, T, 0, rows);
      if (mk.valid) r.valid = vm.fetch(t0, T, 0, rows);
    }
    g.load(t0, T, r.g);
    x.load(t0, T, r.x);
  }
  // mask bits of a fetched stretch; steps past the end are skipped frames
  __device__ __forceinline__ void bits(const Fetched& r, int t0, const Masks& mk, unsigned& ub, unsigned& vb, unsigned& past) const {
    ub = vb = 0xffffu;
    if (MASK) {
      if (mk.use) ub = um.bits(r.use, t0, T, rows, mine);
      if (mk.valid) vb = vm.bits(r.valid, t0, T, rows, mine);
    }
    const int left = T - t0;
    past = left >= KEEP ? 0u : left <= 0 ? 0xffffu : 0xffffu << left & 0xffffu;
    ub |= past;
    vb &= ~past;
  }
  // the fetched stretch: inputs, w of each step, mask bits
  __device__ __forceinline__ void take(const Fetched& r, int t0, const Masks& mk, float (&xs)[KEEP][E], float (&ws)[KEEP][GE], unsigned& ub,
                                       unsigned& vb) const {
    unsigned past;
    bits(r, t0, mk, ub, vb, past);
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
      Values<V, E>::open(r.x[j], xs[j]);
      Values<V, GE>::open(r.g[j], ws[j]);
#pragma unroll
      for (int i = 0; i < GE; ++i) ws[j][i] = gate_step(ws[j][i]);
    }
    if (MASK || past) {
#pragma unroll
      for (int j = 0; j < KEEP; ++j) {
        const unsigned v = bit_mask(vb, j), u = bit_mask(ub, j);
#pragma unroll
        for (int i = 0; i < E; ++i) xs[j][i] = masked_value(xs[j][i], v);
#pragma unroll
        for (int i = 0; i < GE; ++i) ws[j][i] = masked_step(ws[j][i], u, v);
      }
    }
  }
  // the fetched stretch walked from state st on: states (a step's registers are free again behind it)
  __device__ __forceinline__ void follow(const Fetched& r, int t0, const Masks& mk, float (&st)[E], float (&hs)[KEEP][E]) const {
    unsigned ub, vb, past;
    bits(r, t0, mk, ub, vb, past);
    const bool some = MASK || past;
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
      const unsigned v = bit_mask(vb, j), u = bit_mask(ub, j);
      float xv[E], w[GE];
      Values<V, E>::open(r.x[j], xv);
      Values<V, GE>::open(r.g[j], w);
#pragma unroll
      for (int i = 0; i < GE; ++i) {
        w[i] = gate_step(w[i]);
        if (some) w[i] = masked_step(w[i], u, v);
      }
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if (some) xv[i] = masked_value(xv[i], v);
        hs[j][i] = st[i] = advance(MASK ? masked_value(st[i], u) : st[i], xv[i], w[i % GE]);
      }
    }
  }
};

// Partners: the W waves of a workgroup take the KEEP-step stretches of a tile in turn; each hands its stretch over in LDS and
// joins those before it (after it, in the backward direction) to the state that entered the tile.
template <int W, int E>
struct Partners {
  float (*lds)[W][3 * E][64];
  int turn = 0;
  // `own`: state before this wave's stretch; `through` becomes the state behind the tile
  template <bool BACK>
  __device__ __forceinline__ void enter(const Stretch (&mine)[E], int tw, int lane, float (&through)[E], float (&own)[E]) {
    float(*b)[3 * E][64] = lds[turn];
    turn ^= 1;                              // two places: one barrier a tile
#pragma unroll
    for (int i = 0; i < E; ++i) {
      b[tw][3 * i][lane] = mine[i].a;
      b[tw][3 * i + 1][lane] = mine[i].q;
      b[tw][3 * i + 2][lane] = mine[i].p;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < E; ++i) {
      float cur = through[i];
      own[i] = cur;
      for (int n = 0; n < W; ++n) {
        const int w = BACK ? W - 1 - n : n;
        if (w == tw) own[i] = cur;
        cur = join(cur, Stretch{b[w][3 * i][lane], b[w][3 * i + 1][lane], b[w][3 * i + 2][lane]});
      }
      through[i] = cur;
    }
  }
};

// How a call is shared out (split_axis)
struct Split {
  int per;                 // values of a wave
  int w;                   // waves that share a tile, 1: a wave walks alone
  int len;                 // stretches of a run, 0: the axis is not cut
  int groups;              // workgroups along the axis
  int64_t waves;           // of `per` values
};

// Workgroups go to the 8 XCDs in turn, and each XCD has an L2 of its own: neighbours among `all` pieces of work share the
// 128-byte lines that lie across their border, so each XCD gets an unbroken eighth of them.
constexpr unsigned XCDS = 8;
static unsigned xcd_grid(int64_t all) { return (unsigned)((all + XCDS - 1) / XCDS * XCDS); }
__device__ __forceinline__ unsigned xcd_piece() { return (blockIdx.x % XCDS) * (gridDim.x / XCDS) + blockIdx.x / XCDS; }

// Where a wave works: its lanes' wave, its first stretch, how many stretches, the distance between them
template <int W, bool RUNS>
struct Part {
  int64_t wave;
  int group;               // of runs
  int tw, first, count, by;
  bool none;               // nowhere: the same for a whole workgroup where it shares work
  __device__ __forceinline__ Part(const Split& P, int T) {
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), all = (T + KEEP - 1) / KEEP;
    const unsigned piece = xcd_piece();
    if (RUNS) {
      group = (int)(piece / (unsigned)P.waves);
      wave = piece - (unsigned)group * (unsigned)P.waves;
      none = group >= P.groups;
      tw = wv;
      first = (group * RUN_WAVES + wv) * P.len;
      count = max(0, min(P.len, all - first));
      by = 1;
    } else {
      wave = W == 1 ? (int64_t)piece * (GT / 64) + wv : piece;
      none = wave >= P.waves;
      tw = first = W == 1 ? 0 : wv;
      count = (all + W - 1) / W;            // the same for all waves of a workgroup, which meet at a barrier a tile
      by = W;
    }
  }
};

// ws: Stretch of every run [run][3][N], then of every workgroup's runs joined [group][3][N]
__device__ __forceinline__ float* run_at(float* ws, int64_t N, int run) { return ws + (int64_t)run * 3 * N; }
__device__ __forceinline__ Stretch load_stretch(const float* s, int64_t N, int64_t e) { return Stretch{s[e], s[N + e], s[2 * N + e]}; }
__device__ __forceinline__ void store_stretch(float* s, int64_t N, int64_t e, const Stretch& v) {
  s[e] = v.a;
  s[N + e] = v.q;
  s[2 * N + e] = v.p;
}

// The step that each run is (BACK: of the gradient that comes from behind).  108001 steps of 2 x 21 landmarks, fp32: 18.4 us
// for 72 MB, of which about 5 are the launch and the first loads.
template <typename V, int E, int GE, typename OFF, bool MASK, bool BACK>
__global__ __launch_bounds__(64 * RUN_WAVES) void gated_runs_kernel(umt_gated_shape S, Split P, const V* __restrict__ v, int64_t v_t, int64_t v_row,
                                                                    const V* __restrict__ gate, Masks mk, float* __restrict__ ws) {
  __shared__ float lds[RUN_WAVES][3 * E][64];
  using W = Walk<V, E, GE, OFF, MASK>;
  const int lane = threadIdx.x & 63;
  const Part<1, true> part(P, S.t);
  if (part.none) return;
  const Place<E, OFF> at(S, part.wave, P.per);
  const int64_t N = (int64_t)S.rows * S.groups * S.share;
  const W w(S, at, v, v_t, v_row, gate, mk);
  Stretch own[E];
#pragma unroll
  for (int i = 0; i < E; ++i) own[i] = {1.f, 0.f, 0.f};
  unsigned all_use = ~0u;
  const int last = part.first + part.count - 1;
  auto start = [&](int k) { return (BACK ? last - k : part.first + k) * KEEP; };
  auto walk = [&](int k, const typename W::Fetched& now, typename W::Fetched& next) __attribute__((always_inline)) {
    const int t0 = start(k);
    if (k + 1 < part.count) w.fetch(start(k + 1), mk, next);
    unsigned ub, vb, past;
    w.bits(now, t0, mk, ub, vb, past);
    all_use &= ub;
    const bool some = MASK || past;
#pragma unroll
    for (int n = 0; n < KEEP; ++n) {
      const int j = BACK ? KEEP - 1 - n : n;
      const unsigned u = bit_mask(ub, j), va = bit_mask(vb, j);
      float x[E], g[GE];
      Values<V, E>::open(now.x[j], x);
      Values<V, GE>::open(now.g[j], g);
      Weights wt[GE];
#pragma unroll
      for (int i = 0; i < GE; ++i) {
        wt[i] = Weights::of_gate(g[i]);
        if (some) wt[i] = wt[i].masked(u, va);
      }
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if (BACK) {
          if (past) x[i] = masked_value(x[i], ~bit_mask(past, j));           // gradients: no valid mask covers them
          own[i].template backward<MASK>(x[i], wt[i % GE], u);
        } else {
          if (some) x[i] = masked_value(x[i], va);
          own[i].template forward<MASK>(x[i], wt[i % GE], u);
        }
      }
    }
  };
  typename W::Fetched a, b;                // two in turn: no copies between them
  if (part.count > 0) w.fetch(start(0), mk, a);
  for (int k = 0; k < part.count; k += 2) {
    walk(k, a, b);
    if (k + 1 < part.count) walk(k + 1, b, a);
  }
#pragma unroll
  for (int i = 0; i < E; ++i) {
    own[i].close(all_use);
    lds[part.tw][3 * i][lane] = own[i].a;
    lds[part.tw][3 * i + 1][lane] = own[i].q;
    lds[part.tw][3 * i + 2][lane] = own[i].p;
    if (at.on) store_stretch(run_at(ws, N, part.group * RUN_WAVES + part.tw), N, at.e + i, own[i]);
  }
  __syncthreads();
  if (part.tw != 0 || !at.on) return;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    Stretch all{1.f, 0.f, 0.f};
    for (int n = 0; n < RUN_WAVES; ++n) {
      const int k = BACK ? RUN_WAVES - 1 - n : n;
      all = then(all, Stretch{lds[k][3 * i][lane], lds[k][3 * i + 1][lane], lds[k][3 * i + 2][lane]});
    }
    store_stretch(run_at(ws, N, P.groups * RUN_WAVES + part.group), N, at.e + i, all);
  }
}

// State with which this wave's run begins: the workgroups before it (BACK: behind it) are joined by the waves, an equal
// share each, then the runs before it in its own
template <bool BACK, int E>
__device__ __forceinline__ void enter_run(const float* ws, const Split& P, int group, int64_t N, int64_t e, int tw, int lane, float (&h)[E],
                                          Partners<RUN_WAVES, E>& partners) {
  const int count = BACK ? P.groups - 1 - group : group, each = (count + RUN_WAVES - 1) / RUN_WAVES;
  const int i0 = min(count, tw * each), i1 = min(count, i0 + each);
  const float* joined = ws + (int64_t)P.groups * RUN_WAVES * 3 * N;
  Stretch run[E], own[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    own[i] = load_stretch(ws + (int64_t)(group * RUN_WAVES + tw) * 3 * N, N, e + i);
    run[i] = {1.f, 0.f, 0.f};
#pragma unroll 4
    for (int n = i0; n < i1; ++n) run[i] = then(run[i], load_stretch(joined + (int64_t)(BACK ? P.groups - 1 - n : n) * 3 * N, N, e + i));
  }
  float unused[E], begin[E];
  partners.template enter<false>(run, tw, lane, h, unused);
  partners.template enter<BACK>(own, tw, lane, h, begin);
#pragma unroll
  for (int i = 0; i < E; ++i) h[i] = begin[i];
}

template <int W, bool RUNS>
constexpr int partner_waves() { return RUNS ? RUN_WAVES : W; }
template <int W, bool RUNS>
constexpr int group_threads() { return RUNS ? 64 * RUN_WAVES : W == 1 ? GT : 64 * W; }

// A wave alone (512 steps of 512 rows of 648 bf16 values, a gate each): 235 us for 1.02 GB, 4.3 TB/s where a copy reaches 5.06.
// Tiles (64 steps of 128 x 21 landmarks, fp32): 6 us.  Runs (108001 steps of 2 x 21 landmarks): 27 us for 127 MB, about 6 of
// them the launch, the first loads and the joining; the inputs have been read once before.
template <typename V, int E, int GE, typename OFF, int W, bool MASK, bool RUNS>
__global__ __launch_bounds__((group_threads<W, RUNS>())) void gated_scan_kernel(umt_gated_shape S, Split P, const V* __restrict__ x,
                                                                                const V* __restrict__ gate, Masks mk,
                                                                                const float* __restrict__ h0, const float* __restrict__ ws,
                                                                                V* __restrict__ h, float* __restrict__ h_last,
                                                                                float* __restrict__ kept) {
  constexpr int PW = partner_waves<W, RUNS>();
  __shared__ float lds[PW > 1 ? 2 : 1][PW][3 * E][64];
  const int lane = threadIdx.x & 63;
  const Part<W, RUNS> part(P, S.t);
  if (part.none) return;
  const Place<E, OFF> at(S, part.wave, P.per);
  const int64_t N = (int64_t)S.rows * S.groups * S.share;
  using Wk = Walk<V, E, GE, OFF, MASK>;
  const Wk w(S, at, x, S.x_t, S.x_row, gate, mk);
  const Lanes<V, E, OFF> out(h, S.out_t, S.out_row, at.row0, at.row, at.f);
  typename Wk::Fetched fa, fb;             // two in turn: no copies between them
  if (part.count > 0) w.fetch(part.first * KEEP, mk, fa);
  Partners<PW, E> partners{reinterpret_cast<float(*)[PW][3 * E][64]>(lds)};
  float cur[E];
#pragma unroll
  for (int i = 0; i < E; ++i) cur[i] = h0 ? h0[at.e + i] : 0.f;
  if constexpr (RUNS) enter_run<false>(ws, P, part.group, N, at.e, part.tw, lane, cur, partners);
  auto keep = [&](int c, const float(&st)[E]) __attribute__((always_inline)) {
    if (kept && at.on)
#pragma unroll
      for (int i = 0; i < E; ++i) kept[(int64_t)c * N + at.e + i] = st[i];
  };
  auto walk = [&](int k, const typename Wk::Fetched& now, typename Wk::Fetched& next) __attribute__((always_inline)) {
    const int c = part.first + k * part.by, t0 = c * KEEP;
    float hs[KEEP][E], st[E];
    if (k + 1 < part.count) w.fetch(t0 + part.by * KEEP, mk, next);
    if constexpr (W > 1) {
      float steps[KEEP][GE];
      unsigned ub, vb;
      w.take(now, t0, mk, hs, steps, ub, vb);
      Stretch own[E];
#pragma unroll
      for (int i = 0; i < E; ++i) own[i] = {1.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < KEEP; ++j)
#pragma unroll
        for (int i = 0; i < E; ++i) own[i].template forward<MASK>(hs[j][i], Weights::of_step(0.5f * steps[j][i % GE]), bit_mask(ub, j));
#pragma unroll
      for (int i = 0; i < E; ++i) own[i].close(ub);
      partners.template enter<false>(own, part.tw, lane, cur, st);
      if (t0 >= S.t) return;
      keep(c, st);
#pragma unroll
      for (int j = 0; j < KEEP; ++j)
#pragma unroll
        for (int i = 0; i < E; ++i) hs[j][i] = st[i] = advance(memory_of<MASK>(st[i], ub, j), hs[j][i], steps[j][i % GE]);
    } else {
      keep(c, cur);
      w.follow(now, t0, mk, cur, hs);
#pragma unroll
      for (int i = 0; i < E; ++i) st[i] = cur[i];
    }
    out.store(t0, S.t, at.on, hs);
    if (h_last && at.on && t0 + KEEP >= S.t)
#pragma unroll
      for (int i = 0; i < E; ++i) h_last[at.e + i] = st[i];
  };
  for (int k = 0; k < part.count; k += 2) {
    walk(k, fa, fb);
    if (k + 1 < part.count) walk(k + 1, fb, fa);
  }
}

// ---------------------------------------------------------------- backward
// Sums over the features of a gate.  A wave's lanes hold consecutive features, so a gate's are a run of lanes (a lane's own
// two are added first; `share` and `per` count lanes here).  The KEEP steps' products go through the wave's own LDS rows.
// Gates of 16 lanes and more: lane 16 k + j reads the 16 products of step j that lanes 16 k .. 16 k + 15 left, at most two
// gates' of which the second begins at `bound`, and the four such parts of a step are added across the wave (255 steps of
// 384 x 18 gates of 18 lanes: 18 us of the kernel, 32 with the gates one after the other).  Smaller gates: with n of them in
// the wave, lane n i + k adds up gate k of the steps i, i + 64 / n, ..., and neighbouring lanes write neighbouring gates.  A
// gate that reaches into other waves leaves its part in `part`, and a second launch adds the parts in order (7.5 us there).
constexpr int SUM_ROW = 68;                // floats of a step's row: 16-byte reads of 16 steps lie in different banks
constexpr int SUM_ROWS = KEEP * SUM_ROW + 64;      // reads past a gate's end are thrown away, but made
constexpr int WIDE_GATE = 16;
constexpr int WIDE_GATES = 5;              // that a wave can hold parts of

// v of the lanes 16 and 32 away added: the same sum in all four
__device__ __forceinline__ float add_quarters(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

template <typename V>
struct GateSums {
  int gi0, groups;         // the wave's first gate in its row, gates of a row
  int left;                // gates from the wave's first to the call's last
  int count, lead, per;    // gates that the wave holds, lanes of the first that lie before it, lanes
  int share, slots, slot0; // slot0: waves that hold the first gate before this one
  int step;                // this lane's first step: lane & 15, or of gates of fewer than WIDE_GATE lanes lane / count
  int wide0, bound;        // wide gates: that of lane (lane & ~15), and how many lanes on the next begins
  int lo, n;               // smaller ones: the first product of gate lane % count, and how many the wave has
  bool whole;              // all of them, so this is the sum
  int64_t off;             // and where it goes
  int64_t row_step;        // of dgate
  V* to;                   // the first gate's places at this lane's first step
  float* part;
  __device__ __forceinline__ GateSums(const umt_gated_shape& S, int64_t row0, int64_t e0, int E, int per_, int slots_, V* dgate, float* parts) {
    const int lane = threadIdx.x & 63;
    const int64_t G = (int64_t)S.rows * S.groups, inner = e0 - row0 * (S.groups * S.share);
    gi0 = (int)inner / S.share;
    groups = S.groups;
    const int64_t group0 = row0 * S.groups + gi0;
    left = (int)(G - group0 < 1 << 20 ? G - group0 : 1 << 20);
    share = S.share / E;
    per = per_ / E;
    lead = ((int)inner - gi0 * S.share) / E;
    slots = slots_;
    slot0 = (lead + per - 1) / per;
    count = share ? (lead + per + share - 1) / share : 0;
    row_step = S.dgate_row;
    step = lane & 15;
    if (share >= WIDE_GATE) {
      const int from = lead + (lane & 48);
      wide0 = from / share;
      bound = (wide0 + 1) * share - from;
    } else if (share > 0) {
      step = lane / count;
      const int k = lane - step * count, at = k * share - lead;
      lo = max(0, at);
      n = min(per, at + share) - lo;
      whole = n == share;
      off = whole ? place(k) : part_place(k);
      if (step >= 64 / count || k >= left) step = KEEP;    // nothing to do
    }
    to = dgate + step * S.dgate_t + row0 * S.dgate_row + gi0;
    part = parts + ((int64_t)step * G + group0) * slots;
  }
  // gate k of the wave from its first: one row further where rows have as many as the 64 that a wave may hold
  __device__ __forceinline__ int64_t place(int k) const {
    const int row_on = gi0 + k < groups ? 0 : groups >= 64 ? 1 : (int)((unsigned)(gi0 + k) / (unsigned)groups);
    return row_on * row_step + (k - row_on * groups);
  }
  __device__ __forceinline__ int64_t part_place(int k) const { return (int64_t)k * slots + (k == 0 ? slot0 : 0); }
};

// v: this lane's products of KEEP steps; rows: the wave's LDS; the steps from t0 on lie to_t0 and part_t0 elements on, to_t and
// part_t from one to the next
template <typename V>
__device__ __forceinline__ void sum_gates(const GateSums<V>& A, float* rows, const float (&v)[KEEP][1], bool on, int steps, int64_t to_t0,
                                          int64_t to_t, int64_t part_t0, int64_t part_t) {
  const int lane = threadIdx.x & 63, k0 = lane >> 4;
#pragma unroll
  for (int i = 0; i < KEEP; ++i) rows[i * SUM_ROW + lane] = on ? v[i][0] : 0.f;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  if (A.share >= WIDE_GATE) {
    const float* row = rows + A.step * SUM_ROW;
    float4 r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = *reinterpret_cast<const float4*>(row + 16 * k0 + 4 * i);
    float lo[4], hi[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const bool next = 4 * i + m >= A.bound;
        lo[m] = (i ? lo[m] : 0.f) + (next ? 0.f : p[m]);
        hi[m] = (i ? hi[m] : 0.f) + (next ? p[m] : 0.f);
      }
    }
    const float first = (lo[0] + lo[1]) + (lo[2] + lo[3]), second = (hi[0] + hi[1]) + (hi[2] + hi[3]);
    float mine = 0.f, fifth = 0.f;           // gate k0; gate 4 where there is one
#pragma unroll
    for (int k = 0; k < WIDE_GATES; ++k) {
      if (k >= A.count) break;
      const float sum = add_quarters(A.wide0 == k ? first : A.wide0 + 1 == k ? second : 0.f);
      if (k < 4)
        mine = k0 == k ? sum : mine;
      else
        fifth = sum;
    }
    auto put = [&](int k, float sum) __attribute__((always_inline)) {
      if (A.step >= steps || k >= A.left || k >= A.count) return;
      if (min(A.per, (k + 1) * A.share - A.lead) - max(0, k * A.share - A.lead) == A.share)
        store_value(A.to + to_t0 + A.place(k), sum);
      else
        A.part[part_t0 + A.part_place(k)] = sum;
    };
    put(k0, mine);
    if (A.count > 4 && k0 == 0) put(4, fifth);
  } else {
    const int by = 64 / A.count;             // steps at once: neighbouring lanes write neighbouring gates
    V* to = A.to + (to_t0 + A.off);
    float* part = A.part + (part_t0 + A.off);
    for (int i = A.step; i < min(steps, KEEP); i += by, to += by * to_t, part += by * part_t) {
      const float* row = rows + i * SUM_ROW + A.lo;
      float sum = 0.f;
      for (int m = 0; m < A.share; m += 4) {               // four reads in flight, added in a fixed order
        float r[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) r[q] = row[m + q];
#pragma unroll
        for (int q = 0; q < 4; ++q) r[q] = m + q < A.n ? r[q] : 0.f;
        sum += (r[0] + r[1]) + (r[2] + r[3]);
      }
      if (A.whole)
        store_value(to, sum);
      else
        *part = sum;
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <typename V>
__global__ __launch_bounds__(GT) void gate_parts_kernel(umt_gated_shape S, int per, int slots, const float* __restrict__ part,
                                                        V* __restrict__ dgate) {
  const int64_t G = (int64_t)S.rows * S.groups;
  const int64_t g = (int64_t)blockIdx.x * GT + threadIdx.x;
  if (g >= G) return;
  const int n = (int)(((g + 1) * S.share - 1) / per - g * S.share / per) + 1;
  if (n == 1) return;
  const int64_t row = g / S.groups, at = row * S.dgate_row + (g - row * S.groups);
  for (int64_t t = blockIdx.y; t < S.t; t += gridDim.y) {
    float s = 0.f;
    for (int p = 0; p < n; ++p) s += part[(t * G + g) * slots + p];
    store_value(dgate + t * S.dgate_t + at, s);
  }
}

// From the last stretch to the first: the states of a stretch again from the kept one before it, then the gradients down.
//   s = dh + v,  dx = c s,  dgate = sum a c s (h' - x),  v' = a s
// 512 steps of 512 rows of 648 bf16 values with a gate each: 380 us for 1.74 GB (4.6 TB/s).  255 steps of 384 rows of 18 x 36
// values: 112 us for 0.40 GB (3.5 TB/s): two waves a SIMD, of which the vector operations alone take 70 us (about 65 for the
// two values of a lane and step); the gate sums are 18 of the 112.  A stretch of inputs ahead is what fits: gradients ahead too spill
// (x1.4 to x3.7).  Both weights a step in the place of m: 3 % less there, 3 % more with a gate a value.
template <typename V, int E, int GE, typename OFF, int W, bool MASK, bool RUNS>
__global__ __launch_bounds__((group_threads<W, RUNS>()), 2) void gated_scan_backward_kernel(
    umt_gated_shape S, Split P, int slots, const V* __restrict__ x, const V* __restrict__ gate, Masks mk, const float* __restrict__ kept,
    const V* __restrict__ dh, const float* __restrict__ dh_last, const float* __restrict__ ws, V* __restrict__ dx, V* __restrict__ dgate,
    float* __restrict__ parts, float* __restrict__ dh0) {
  constexpr int PW = partner_waves<W, RUNS>(), GW = group_threads<W, RUNS>() / 64;
  __shared__ float lds[PW > 1 ? 2 : 1][PW][3 * E][64];
  __shared__ alignas(16) float sums[GW][SUM_ROWS];
  const int lane = threadIdx.x & 63;
  const Part<W, RUNS> part(P, S.t);
  if (part.none) return;
  const Place<E, OFF> at(S, part.wave, P.per);
  const int64_t N = (int64_t)S.rows * S.groups * S.share;
  using Wk = Walk<V, E, GE, OFF, MASK>;
  const Wk w(S, at, x, S.x_t, S.x_row, gate, mk);
  const Lanes<V, E, OFF> d(dh, S.dh_t, S.dh_row, at.row0, at.row, at.f), out(dx, S.out_t, S.out_row, at.row0, at.row, at.f);
  const Lanes<V, GE, OFF> single(dgate, S.dgate_t, S.dgate_row, at.row0, at.row, at.gi);
  const GateSums<V> A(S, at.row0, at.e0, E, P.per, slots, dgate, parts);
  Partners<PW, E> partners{reinterpret_cast<float(*)[PW][3 * E][64]>(lds)};
  float v[E];
#pragma unroll
  for (int i = 0; i < E; ++i) v[i] = dh_last ? dh_last[at.e + i] : 0.f;
  if constexpr (RUNS) enter_run<true>(ws, P, part.group, N, at.e, part.tw, lane, v, partners);
  typename Wk::Fetched now;                // a stretch ahead; its gradients are asked for when it begins and needed last
  typename Lanes<V, E, OFF>::Raw rd[KEEP];
  float first[E];
  auto fetch = [&](int k) __attribute__((always_inline)) {
    const int c = part.first + k * part.by;
    w.fetch(c * KEEP, mk, now);
#pragma unroll
    for (int i = 0; i < E; ++i) first[i] = c * KEEP < S.t ? kept[(int64_t)c * N + at.e + i] : 0.f;
  };
  if (part.count > 0) fetch(part.count - 1);
  for (int k = part.count - 1; k >= 0; --k) {
    const int t0 = (part.first + k * part.by) * KEEP;
    float q[KEEP][E], ms[KEEP][GE], cur[E];
    unsigned ub, vb, past;
    d.load(t0, S.t, rd);
    w.bits(now, t0, mk, ub, vb, past);
    const bool some = MASK || past;
#pragma unroll
    for (int i = 0; i < E; ++i) cur[i] = first[i];
    // the states again; q is c a (h[t-1] - x[t]), the slope over the gate; the halved difference serves both.  (An infinite
    // state becomes NaN here rather than stay: the slopes behind it are not finite either way, and it ends where it is dropped.)
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
      const unsigned va = bit_mask(vb, j), u = bit_mask(ub, j);
      float step[GE];
      Values<V, E>::open(now.x[j], q[j]);
      Values<V, GE>::open(now.g[j], step);
#pragma unroll
      for (int i = 0; i < GE; ++i) {
        step[i] = gate_step(step[i]);
        if (some) step[i] = masked_step(step[i], u, va);
        ms[j][i] = 0.5f * step[i];
      }
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float aw = fabsf(step[i % GE]), x = some ? masked_value(q[j][i], va) : q[j][i];
        if (MASK) cur[i] = masked_value(cur[i], u);
        q[j][i] = fmaf(-aw, fabsf(ms[j][i % GE]), aw) * half_apart(cur[i], x);
        cur[i] = advance_finite(cur[i], x, step[i % GE]);
      }
    }
    if (k > 0) fetch(k - 1);
    auto gradient = [&](int j, float(&g)[E]) __attribute__((always_inline)) {
      Values<V, E>::open(rd[j], g);
      if (past)
#pragma unroll
        for (int i = 0; i < E; ++i) g[i] = masked_value(g[i], ~bit_mask(past, j));
    };
    float b[E];
    if constexpr (W > 1) {
      Stretch own[E];
#pragma unroll
      for (int i = 0; i < E; ++i) own[i] = {1.f, 0.f, 0.f};
#pragma unroll
      for (int j = KEEP - 1; j >= 0; --j) {
        float g[E];
        gradient(j, g);
#pragma unroll
        for (int i = 0; i < E; ++i) own[i].template backward<MASK>(g[i], Weights::of_step(ms[j][i % GE]), bit_mask(ub, j));
      }
#pragma unroll
      for (int i = 0; i < E; ++i) own[i].close(ub);
      partners.template enter<true>(own, part.tw, lane, v, b);
      if (t0 >= S.t) continue;
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) b[i] = v[i];
    }
    float slope[KEEP][GE];
    asm volatile("" : "+v"(ub), "+v"(vb));  // the mask words anew: 32 registers of them across the two loops cost more
    auto down = [&](auto usual) __attribute__((always_inline)) {
      constexpr bool USUAL = decltype(usual)::value;
      Global xp = out.step_at(t0 + KEEP - 1), gp = single.step_at(t0 + KEEP - 1);
      const OFF xm = out.here(), gm = single.here();
#pragma unroll
      for (int j = KEEP - 1; j >= 0; --j) {
        const Global xa = xp, ga = gp;
        xp -= out.step;
        gp -= single.step;
        if (!USUAL && t0 + j >= S.t) continue;
        float g[E], x[E];
        Values<V, E>::open(rd[j], g);
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const float m = ms[j][i % GE], s = g[i] + b[i], l = s * q[j][i];
          if (i < GE)
            slope[j][i] = l;
          else
            slope[j][0] += l;
          x[i] = times_c(m, s);
          if (MASK) x[i] = masked_value(x[i], bit_mask(vb, j));
          b[i] = memory_of<MASK>(times_a(m, s), ub, j);
        }
        if (MASK)
#pragma unroll
          for (int i = 0; i < GE; ++i) slope[j][i] = masked_value(slope[j][i], bit_mask(ub & vb, j));
        if (USUAL || dx) out.store_at(xa, xm, x);
        if (GE == 2 && (USUAL || dgate)) single.store_at(ga, gm, slope[j]);
      }
    };
    if (at.on) {
      if (t0 + KEEP <= S.t && dx && (GE == 1 || dgate))
        down(std::true_type());             // without a question a step
      else
        down(std::false_type());
    }
    if (E == 1 && dgate && S.share == 1) single.store(t0, S.t, at.on, slope);
    if constexpr (GE == 1)
      if (dgate && S.share > 1)
        sum_gates(A, sums[threadIdx.x >> 6], slope, at.on, S.t - t0, (int64_t)t0 * S.dgate_t, S.dgate_t, (int64_t)t0 * S.rows * S.groups * slots,
                  (int64_t)S.rows * S.groups * slots);
    if (dh0 && at.on && t0 == 0)
#pragma unroll
      for (int i = 0; i < E; ++i) dh0[at.e + i] = b[i];
    if (W == 1)
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = b[i];
  }
}

// ---------------------------------------------------------------- one frame over a cache of rows
constexpr int STEP_SEG = 256;              // features one wave advances
// Samples among which a wave looks for its row's other names itself, rather than wait for two launches that make a table (calls
// replayed in a graph, looking against the table: rows of 648 values, 512 samples 16.2 and 16.3 us, 1024 15.9 and 16.1, 1500
// 18.4 and 16.7, 4096 58 and 22; of 63 values, 1500 16.7 and 16.9, 4096 27.5 and 16.1).
constexpr int STEP_LOOK = 1024;

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
  const int32_t *owner, *named;             // null: every wave looks through idx itself
  int32_t* status;
};

// STEP_SEG features of sample b, from f0 on; prev: the row's values.  -> the new state
template <typename V>
__device__ __forceinline__ void step_values(const StepArgs& A, const V* x, const V* gate, V* out, int b, int f0,
                                            bool has_row, const float (&prev)[STEP_SEG / 64], float (&h)[STEP_SEG / 64]) {
  const int lane = threadIdx.x & 63, F = A.groups * A.share;
  const unsigned use = has_row && (!A.use || A.use[b]) ? ~0u : 0u, valid = !A.valid || A.valid[b] ? ~0u : 0u;
  float xv[STEP_SEG / 64], gv[STEP_SEG / 64];
#pragma unroll
  for (int i = 0; i < STEP_SEG / 64; ++i) {
    const int f = min(f0 + 64 * i + lane, F - 1);
    xv[i] = load_value(x + (int64_t)b * F + f);
    gv[i] = load_value(gate + (int64_t)b * A.groups + f / A.share);
  }
#pragma unroll
  for (int i = 0; i < STEP_SEG / 64; ++i) {
    h[i] = advance(masked_value(prev[i], use), masked_value(xv[i], valid), masked_step(gate_step(gv[i]), use, valid));
    if (f0 + 64 * i + lane < F) store_value(out + (int64_t)b * F + f0 + 64 * i + lane, h[i]);
  }
}

// One wave per (sample, segment of features).  A row that several samples name is advanced by the wave of the highest one:
// it reads the row once, computes the other samples' outputs from that, and writes the row last.  Who that is a small batch
// finds by looking through memory_idx (64 a load, from L2), a large one in the owner table of two launches before.
// 2 samples of 63 values: 2.6 us.  8191 of 16384 rows of 648 fp32 values: 18.7 us for 106 MB (a part of it in the cache
// behind L2) and 2.6 + 2.6 for the table.
template <typename V>
__global__ __launch_bounds__(GT) void gated_step_kernel(StepArgs A, const V* x, const V* gate, V* out) {
  constexpr int K = STEP_SEG / 64;
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * (GT / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = (int)(item / A.segs), f0 = (int)(item - (int64_t)b * A.segs) * STEP_SEG;
  if (b >= A.batch) return;
  const int F = A.groups * A.share;
  const int64_t r = A.idx ? A.idx[b] : b;
  const bool has_row = r >= 0 && r < A.cache_rows;
  bool shared = false;
  if (A.idx && has_row) {
    if (A.owner) {
      if (A.owner[r] != b) return;
      shared = A.named[r] > 1;
    } else {
      for (int o = 0; o < A.batch; o += 64) {
        const uint64_t same = __ballot(o + lane < A.batch && A.idx[min(o + lane, A.batch - 1)] == r);
        const int at = b - o;                                  // this sample's place among the 64
        if (at < 0 ? same != 0 : at < 63 && same >> (at + 1) != 0) return;
        if (same & (at >= 64 ? ~0ull : at <= 0 ? 0ull : (1ull << at) - 1)) shared = true;
      }
    }
  }
  if (!has_row && A.status && f0 == 0 && lane == 0) atomicOr(A.status, (int)UMT_STATUS_BAD_MEMORY_IDX);
  float prev[K] = {}, h[K];
  float* sp = A.state + (has_row ? r : 0) * F;
  if (has_row && (shared || !A.use || A.use[b])) {             // a memory that is dropped is not read
#pragma unroll
    for (int i = 0; i < K; ++i) prev[i] = sp[min(f0 + 64 * i + lane, F - 1)];
  }
  if (shared)
    for (int o = 0; o < b; ++o)
      if (A.idx[o] == r) step_values(A, x, gate, out, o, f0, true, prev, h);
  step_values(A, x, gate, out, b, f0, has_row, prev, h);
  if (!has_row) return;
#pragma unroll
  for (int i = 0; i < K; ++i)
    if (f0 + 64 * i + lane < F) sp[f0 + 64 * i + lane] = h[i];
}

static int check_shape(const umt_gated_shape* S, bool backward) {
  UMT_REQUIRE(S, UMT_ERR_INVALID, "gated scan: null shape");
  UMT_REQUIRE(S->dtype == UMT_VALUES_F32 || S->dtype == UMT_VALUES_BF16, UMT_ERR_INVALID, "gated scan: dtype = %d", S->dtype);
  UMT_REQUIRE(S->t >= 0 && S->rows >= 0 && S->groups > 0 && S->share > 0, UMT_ERR_INVALID,
              "gated scan: t=%d rows=%d groups=%d share=%d", S->t, S->rows, S->groups, S->share);
  UMT_REQUIRE((int64_t)S->groups * S->share <= (1 << 24), UMT_ERR_INVALID, "gated scan: %d x %d features in a row", S->groups, S->share);
  // a launch counts its threads in 32 bits, and no lane owns less than a feature
  UMT_REQUIRE((int64_t)S->rows * S->groups * S->share <= (1LL << 31), UMT_ERR_INVALID, "gated scan: %d rows of %d x %d features",
              S->rows, S->groups, S->share);
  UMT_REQUIRE(S->t <= (1 << 30) && (int64_t)S->rows * S->groups <= (1LL << 38) / (S->t > 0 ? S->t : 1), UMT_ERR_INVALID,
              "gated scan: %d steps of %d x %d gates", S->t, S->rows, S->groups);
  const int64_t st[] = {S->x_t, S->x_row, S->gate_t, S->gate_row, S->out_t, S->out_row, S->use_t, S->use_row, S->valid_t,
                        S->valid_row, S->dh_t, S->dh_row, S->dgate_t, S->dgate_row};
  for (int i = 0; i < (backward ? 14 : 10); ++i) {          // t strides and row strides in turn; no array reaches over 2^48 values
    const int n = i % 2 ? S->rows : S->t;
    UMT_REQUIRE(st[i] >= 0 && (n <= 1 || st[i] <= (1LL << 48) / n), UMT_ERR_INVALID, "gated scan: stride %lld over %d", (long long)st[i], n);
  }
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

// How the axis is shared out, for waves of `per` values (times: fp32, forward / backward in us, calls replayed in a graph).
// * A wave that walks alone needs about four others on its CU to keep HBM busy; below 1024 the waves of a workgroup take
//   turns.  Alone against four: 1000 steps of 900 waves 132 / 245 and 169 / 260, of 1024 152 / 260 and 176 / 274, of 1200
//   233 / 366 and 208 / 366; 250 steps of 700 waves 33 / 56 and 31 / 49, of 1024 39 / 70 and 39 / 73.  (From 1024 on the lone
//   waves come in rounds, and which is ahead goes with what is left for the last round.)
// * Eight waves take turns where tiles leave CUs free, else four.  600 steps of 200 waves: 28 / 40 in eights, 32 / 49 in fours;
//   of 300 waves 45 / 69 and 42 / 59.  Four where they cover the axis: 48 steps of 300 waves 15 in fours, 21 in eights, backward.
// * With a tile on fewer than two thirds of the CUs, an axis of more than two tiles is cut into runs, at the price of reading
//   the inputs twice.  Tiles against runs: 3000 steps of 148 waves 92 / 169 and 82 / 144; 2000 steps of 197 waves 64 / 122 and
//   78 / 135; of 40 waves 300 steps 17 / 23 and 16 / 19, of 100 waves 300 steps 18 / 24 and 22 / 28, 600 steps 25 / 35 and
//   27 / 35; up to 256 steps they are within 2 us of each other.
// * Eight runs are a workgroup, and as many of them as fill the CUs evenly run at once: of one to four per CU what has the
//   shortest way, with a stretch more for the start of each.  3000 steps of 99 waves: 57 / 89 in 495 workgroups, 79 / 129 in 297.
constexpr int CUS = 256;
static Split split_axis(const umt_gated_shape& S, int per) {
  const int64_t N = (int64_t)S.rows * S.groups * S.share;
  const int all = S.t > 0 ? (S.t + KEEP - 1) / KEEP : 1;
  Split p{per, 1, 0, 1, (N + per - 1) / per};
  if (p.waves >= 1024 || all == 1 || p.waves == 0) return p;
  if (p.waves >= 2 * CUS / 3 || all <= 16) {
    p.w = p.waves >= 256 || all <= 4 ? 4 : 8;
    return p;
  }
  int64_t best = 0;
  for (int each = 1; each <= 4; ++each) {   // workgroups per CU
    const int64_t runs = each * CUS / p.waves * RUN_WAVES, len = (all + runs - 1) / runs;
    if (best && each * (len + 1) >= best) continue;
    best = each * (len + 1);
    p.len = (int)len;
  }
  p.groups = (all + p.len * RUN_WAVES - 1) / (p.len * RUN_WAVES);
  return p;
}
static int64_t run_floats(const umt_gated_shape& S, int per) {
  const Split p = split_axis(S, per);
  return p.len ? (int64_t)p.groups * (RUN_WAVES + 1) * 3 * S.rows * S.groups * S.share : 0;
}
// Values of a forward wave whose lanes hold E: 64 E, or as many whole rows as fit where rows lie further apart than steps and
// that leaves at most 4 lanes idle (300 steps of 2000 rows of 63 fp32 values, rows first: 91 -> 81 us; with steps further
// apart 78 -> 82).
static int forward_values(const umt_gated_shape& S, int E) {
  const int F = S.groups * S.share / E, whole = S.x_row > S.x_t && F > 0 && F <= 64 ? 64 / F * F : 0;
  return (whole >= 60 ? whole : 64) * E;
}
// Values of a backward wave whose lanes hold E: 64 E, or as many whole gates as fit (21 landmarks of 3 coordinates: 63
// lanes) where that leaves at most 4 lanes idle, so that their sums need no second launch.
static int backward_values(const umt_gated_shape& S, int E) {
  const int share = S.share / E, whole = share > 0 && share <= 64 ? 64 / share * share : 0;
  return (whole >= 60 ? whole : 64) * E;
}
// parts of a gate's sum: waves that its features may lie in, 0 where they always lie in one
static int gate_slots(const umt_gated_shape& S, int per) { return per % S.share == 0 ? 0 : (S.share + per - 2) / per + 1; }
static int64_t part_floats(const umt_gated_shape& S, int per) { return (int64_t)S.t * S.rows * S.groups * gate_slots(S, per); }

// Whether lanes can hold two values: they, and the gates where every feature has its own, lie in pairs at even places.
// 4-byte loads in the place of 2-byte ones: 512 steps of 512 rows of 648 features 267 -> 251 us.
static bool pairable(const umt_gated_shape& S) {
  return S.dtype == UMT_VALUES_BF16 && S.groups * S.share % 2 == 0 && (S.share == 1 || S.share % 2 == 0);
}
static bool even(int64_t a, int64_t b, const void* p) { return a % 2 == 0 && b % 2 == 0 && (uint64_t)p % 4 == 0; }
static bool pairs(const umt_gated_shape& S, const void* x, const void* gate, const void* out, const void* dh, const void* dgate) {
  return pairable(S) && even(S.x_t, S.x_row, x) && even(S.out_t, S.out_row, out) && (!dh || even(S.dh_t, S.dh_row, dh)) &&
         (S.share > 1 || (even(S.gate_t, S.gate_row, gate) && (!dgate || even(S.dgate_t, S.dgate_row, dgate))));
}

// whether 32 bits hold a step's distance and a lane's from its wave's first row in every stream (128 features are at most
// 128 rows), and count the features of the call
static bool near_rows(const umt_gated_shape& S, int64_t size) {
  const int F = S.groups * S.share;
  const int64_t rows = F >= 128 ? 2 : 128 / F + 2;
  const int64_t by_row[] = {S.x_row, S.gate_row, S.out_row, S.dh_row, S.dgate_row}, by_step[] = {S.x_t, S.gate_t, S.out_t, S.dh_t, S.dgate_t};
  for (int64_t r : by_row)
    if (r > ((1LL << 31) / size - F) / rows) return false;
  for (int64_t t : by_step)
    if (t >= (1LL << 31) / size) return false;
  return (int64_t)S.rows * F < (1LL << 31) - 128;
}

template <typename V, int E, int GE, typename OFF, bool MASK>
static int launch_scan(const umt_gated_shape& S, const V* x, const V* gate, Masks mk, const float* h0, V* h, float* h_last, float* kept,
                       float* ws, hipStream_t s) {
  const Split p = split_axis(S, forward_values(S, E));
  const dim3 runs(xcd_grid(p.waves * p.groups)), tiles(xcd_grid(p.waves)), alone(xcd_grid((p.waves + 3) / 4));
#define UMT_SCAN(W, RUNS, GRID, THREADS)                                                                                              \
  hipLaunchKernelGGL((gated_scan_kernel<V, E, GE, OFF, W, MASK, RUNS>), GRID, dim3(THREADS), 0, s, S, p, x, gate, mk, h0, ws, h, h_last, \
                     kept)
  if (p.len) {
    hipLaunchKernelGGL((gated_runs_kernel<V, E, GE, OFF, MASK, false>), runs, dim3(64 * RUN_WAVES), 0, s, S, p, x, S.x_t, S.x_row,
                       gate, mk, ws);
    UMT_SCAN(1, true, runs, 64 * RUN_WAVES);
  } else if (p.w == 1) {
    UMT_SCAN(1, false, alone, GT);
  } else if (p.w == 4) {
    UMT_SCAN(4, false, tiles, 256);
  } else {
    UMT_SCAN(8, false, tiles, 512);
  }
#undef UMT_SCAN
  UMT_CHECK_HIP(hipGetLastError());
  return 0;
}

template <typename V, int E, int GE, typename OFF, bool MASK>
static int launch_backward(const umt_gated_shape& S, const V* x, const V* gate, Masks mk, const float* kept, const V* dh,
                           const float* dh_last, V* dx, V* dgate, float* dh0, float* ws, hipStream_t s) {
  const int per = backward_values(S, E), slots = gate_slots(S, per);
  const Split p = split_axis(S, per);
  const dim3 runs(xcd_grid(p.waves * p.groups)), tiles(xcd_grid(p.waves)), alone(xcd_grid((p.waves + 3) / 4));
  float* parts = ws + run_floats(S, per);
#define UMT_SCAN(W, RUNS, GRID, THREADS)                                                                                               \
  hipLaunchKernelGGL((gated_scan_backward_kernel<V, E, GE, OFF, W, MASK, RUNS>), GRID, dim3(THREADS), 0, s, S, p, slots, x, gate, mk, kept, \
                     dh, dh_last, ws, dx, dgate, parts, dh0)
  if (p.len) {
    hipLaunchKernelGGL((gated_runs_kernel<V, E, GE, OFF, MASK, true>), runs, dim3(64 * RUN_WAVES), 0, s, S, p, dh, S.dh_t,
                       S.dh_row, gate, mk, ws);
    UMT_SCAN(1, true, runs, 64 * RUN_WAVES);
  } else if (p.w == 1) {
    UMT_SCAN(1, false, alone, GT);
  } else if (p.w == 4) {
    UMT_SCAN(4, false, tiles, 256);
  } else {
    UMT_SCAN(8, false, tiles, 512);
  }
#undef UMT_SCAN
  if (dgate && slots) {
    // a thread per gate and a few steps: 4096 workgroups where there are that many
    const int64_t across = ((int64_t)S.rows * S.groups + GT - 1) / GT, along = std::min<int64_t>(S.t, std::max<int64_t>(1, 4096 / across));
    hipLaunchKernelGGL((gate_parts_kernel<V>), dim3((unsigned)across, (unsigned)along), dim3(GT), 0, s, S, per, slots, parts, dgate);
  }
  UMT_CHECK_HIP(hipGetLastError());
  return 0;
}

template <int N>
using Count = std::integral_constant<int, N>;
// the kernel variants: value type, values and gates of a lane, distance of the rows, masks
template <typename Call>
static int by_variant(const umt_gated_shape& S, bool two, bool masks, Call call) {
  const bool near = near_rows(S, S.dtype == UMT_VALUES_BF16 ? 2 : 4);
  auto typed = [&](auto v, auto e, auto ge) {
    if (near) return masks ? call(v, e, ge, (uint32_t)0, std::true_type()) : call(v, e, ge, (uint32_t)0, std::false_type());
    return masks ? call(v, e, ge, (uint64_t)0, std::true_type()) : call(v, e, ge, (uint64_t)0, std::false_type());
  };
  if (S.dtype == UMT_VALUES_F32) return typed(0.f, Count<1>(), Count<1>());
  if (!two) return typed((__bf16)0.f, Count<1>(), Count<1>());
  return S.share == 1 ? typed((__bf16)0.f, Count<2>(), Count<2>()) : typed((__bf16)0.f, Count<2>(), Count<1>());
}

static bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  return na > 0 && nb > 0 && (const char*)a < (const char*)b + nb && (const char*)b < (const char*)a + na;
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
  int64_t n = 0;                                            // whichever way the tensors' places allow
  for (int E = 1; E <= (pairable(*shape) ? 2 : 1); ++E) n = std::max(n, run_floats(*shape, forward_values(*shape, E)));
  return n * (int64_t)sizeof(float);
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
  return by_variant(S, pairs(S, x, gate, h, nullptr, nullptr), use_memory || valid, [&](auto v, auto e, auto ge, auto off, auto masked) {
    using V = decltype(v);
    return launch_scan<V, decltype(e)::value, decltype(ge)::value, decltype(off), decltype(masked)::value>(
        S, (const V*)x, (const V*)gate, mk, h0, (V*)h, h_last, kept, (float*)workspace, s);
  });
}

extern "C" int64_t umt_gated_scan_backward_workspace_bytes(const umt_gated_shape* shape) {
  if (check_shape(shape, false) != 0) return -1;
  int64_t n = 0;
  for (int E = 1; E <= (pairable(*shape) ? 2 : 1); ++E) {
    const int per = backward_values(*shape, E);
    n = std::max(n, run_floats(*shape, per) + part_floats(*shape, per));
  }
  return n * (int64_t)sizeof(float);
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
  return by_variant(S, pairs(S, x, gate, dx, dh, dgate), use_memory || valid, [&](auto v, auto e, auto ge, auto off, auto masked) {
    using V = decltype(v);
    return launch_backward<V, decltype(e)::value, decltype(ge)::value, decltype(off), decltype(masked)::value>(
        S, (const V*)x, (const V*)gate, mk, kept, (const V*)dh, dh_last, (V*)dx, (V*)dgate, dh0, (float*)workspace, s);
  });
}

extern "C" int64_t umt_gated_step_workspace_bytes(int batch, int cache_rows) {
  return batch > STEP_LOOK && cache_rows > 0 ? 2 * (int64_t)cache_rows * (int64_t)sizeof(int32_t) : 0;
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
  UMT_REQUIRE((int64_t)batch * segs < (1LL << 26) - GT, UMT_ERR_INVALID, "gated step: %d samples of %d features", batch, F);      // waves
  // a row may be written while another sample's values are read; an output only by the wave that has read its place
  const int64_t size = dtype == UMT_VALUES_BF16 ? 2 : 4, values = (int64_t)batch * F * size, gates = (int64_t)batch * groups * size;
  const int64_t rows = (int64_t)cache_rows * F * (int64_t)sizeof(float);
  UMT_REQUIRE(!overlap(state, rows, x, values) && !overlap(state, rows, gate, gates) && !overlap(state, rows, out, values), UMT_ERR_INVALID,
              "gated step: state overlaps x, gate or out");
  UMT_REQUIRE((out == x || !overlap(out, values, x, values)) && ((out == gate && share == 1) || !overlap(out, values, gate, gates)),
              UMT_ERR_INVALID, "gated step: out overlaps a part of x or gate");
  hipStream_t s = (hipStream_t)stream;
  int32_t *owner = need ? (int32_t*)workspace : nullptr, *named = need ? owner + cache_rows : nullptr;
  if (need) {
    const dim3 grid((batch + GT - 1) / GT);
    hipLaunchKernelGGL(step_clear_kernel, grid, dim3(GT), 0, s, memory_idx, batch, cache_rows, owner, named);
    hipLaunchKernelGGL(step_claim_kernel, grid, dim3(GT), 0, s, memory_idx, batch, cache_rows, owner, named);
  }
  const StepArgs A{memory_idx, use_memory, valid, batch, groups, share, cache_rows, segs, state, owner, named, status};
  return dtype == UMT_VALUES_BF16 ? launch_step<__bf16>(A, x, gate, out, s) : launch_step<float>(A, x, gate, out, s);
}
