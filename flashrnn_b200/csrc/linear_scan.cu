// Gated linear recurrence: per channel (head, unit) of a batch row
//   c_t = f_t c_{t-1} + v_t,   f_t = sigmoid(x_f + b_f),   u_t = 1 - f_t
//   leaky (f, z):       v = u z,                      hidden = c
//   lstm  (i, f, z, o): v = sigmoid(i) tanh(z),       hidden = sigmoid(o) tanh(c)
// with x the gate pre-activations Wx[B,T,G,N,D]. There is no recurrent matrix, so a span of steps is the map
// c -> A c + H with A = prod f, and spans compose: (A2, H2) o (A1, H1) = (A2 A1, A2 H1 + H2). A step is c + (v - u c) where
// f is 1/2 or more and f c + v where it is less: u keeps its digits where f is next to one, which is where errors would add up over the most
// steps, f keeps them where it is next to zero, where a large state has to vanish behind a small input.
//
// Backward: with dc_t the gradient that reaches c_t through hidden_t, g_t = dc_t + f_{t+1} g_{t+1}; the same scan in reverse
// time over e_t = f_t (dc_t + e_{t+1}). The gates' gradients need c_{t-1}: it is recomputed from Wx, which has to be read
// anyway, and from the state at the start of every tile, which the forward pass keeps: 4 bytes per channel and tile, 1/64 (LSTM 1/32) of what the
// hidden states take in bf16.
//
// Few channels: time is cut. One CTA takes a tile of 128 (LSTM: 64) steps x 64 channels of a batch row, read once into registers:
// a thread has L steps of VEC neighbouring channels, scans them, the tile's spans are joined by shuffles and through shared memory,
// and the second walk over the registers starts from the right state. Tiles of a row are joined through global memory: a tile
// publishes its (A, H), in groups of 8 tiles every tile composes the maps of those in front of it, in order, with the state at the
// start of its group, and the last tile of a group publishes the state at the start of the next. The order of the sums does not
// depend on timing, so two calls give the same bits. CTAs take their tiles from a counter, earlier steps first: whoever is waited for
// has started. Many channels, or next to no time: a thread walks its channels through the whole sequence (below).
//
// The floor is the bytes: leaky bf16 6 a step and channel forward, 10 backward; lstm 10 and 18. With many channels tiles reach 50 % of it in bf16
// (leaky, B8 T2048 N32 D128: 120 us of 61 forward, 209 of 103 backward) and 83 - 86 % in fp32 (B4 T4096: 149 of 123, 237 of 205); small
// layers less (fp32 B13 T333 N2 D200: 9 of 3, 17 of 5). Per step and channel 34 instructions forward (ncu), 0.52 issued a cycle, in a
// chain of load, scan, two barriers and a fetch from other tiles, with 24 warps to an SM. Walks reach 75 % (leaky, B32 T2048 N32 D128: 331 of
// 246, 539 of 410).
#include "../../include/flashrnn_b200.h"

#include "column_sum.cuh"
#include "frnn_common.cuh"

namespace frnn {

namespace {

constexpr int kGroup = 8;    // tiles of a group
constexpr unsigned long long kDefaultWaitNs = 2000000000ull;

struct LinParams {
  const void* wx;         // [B][T][G][ND]
  const float* bias;      // [G][ND]
  const float* initial;   // [B][ND] or null: zeros
  const int* lengths;     // [B] or null: T
  float* starts;          // [B][tiles - 1][ND]: state before every tile but the first; null: not kept
  int* err;
  uint8_t* exchange;      // all ones; the tile counter, the maps, the states between groups; null: one tile
  unsigned long long wait_limit_ns;
  int B, T, ND, n_cg, n_tiles;
  // forward
  void* hidden;           // [B][T][ND]
  float* last;            // [B][ND]
  // backward
  const void* d_hidden;   // [B][T][ND]
  const float* d_last;    // [B][ND] or null: zeros
  void* d_wx;             // [B][T][G][ND]
  float* db_part;         // [B * tiles][G][ND]
  float* d_initial;       // [B][ND] or null
};

// N fp32 values of neighbouring channels; two share an instruction where N is even.
template <int N>
struct Vec {
  float v[N];
  __device__ __forceinline__ float& operator[](int i) { return v[i]; }
  __device__ __forceinline__ float operator[](int i) const { return v[i]; }
};
template <int N>
__device__ __forceinline__ Vec<N> splat(float x) {
  Vec<N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r.v[i] = x;
  return r;
}
template <int N>
__device__ __forceinline__ Vec<N> fma_(const Vec<N>& a, const Vec<N>& b, const Vec<N>& c) {
  Vec<N> r;
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2)
      asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n fma.rn.f32x2 x, x, y, z;\n"
          " mov.b64 {%0, %1}, x;\n}"
          : "=f"(r.v[i]), "=f"(r.v[i + 1])
          : "f"(a.v[i]), "f"(a.v[i + 1]), "f"(b.v[i]), "f"(b.v[i + 1]), "f"(c.v[i]), "f"(c.v[i + 1]));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = __fmaf_rn(a.v[i], b.v[i], c.v[i]);
  }
  return r;
}
template <int N>
__device__ __forceinline__ Vec<N> mul_(const Vec<N>& a, const Vec<N>& b) {
  Vec<N> r;
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2)
      asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
          : "=f"(r.v[i]), "=f"(r.v[i + 1])
          : "f"(a.v[i]), "f"(a.v[i + 1]), "f"(b.v[i]), "f"(b.v[i + 1]));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = __fmul_rn(a.v[i], b.v[i]);
  }
  return r;
}
template <int N>
__device__ __forceinline__ Vec<N> add_(const Vec<N>& a, const Vec<N>& b) {
  Vec<N> r;
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2)
      asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
          : "=f"(r.v[i]), "=f"(r.v[i + 1])
          : "f"(a.v[i]), "f"(a.v[i + 1]), "f"(b.v[i]), "f"(b.v[i + 1]));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = __fadd_rn(a.v[i], b.v[i]);
  }
  return r;
}
template <int N>
__device__ __forceinline__ Vec<N> exp2_(const Vec<N>& a) {
  Vec<N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r.v[i] = exp2_fast(a.v[i]);
  return r;
}
template <int N>
__device__ __forceinline__ Vec<N> rcp_(const Vec<N>& a) {
  Vec<N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r.v[i] = rcp_fast(a.v[i]);
  return r;
}
// min that keeps a NaN
template <int N>
__device__ __forceinline__ Vec<N> min_(const Vec<N>& a, float b) {
  Vec<N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) asm("min.NaN.f32 %0, %1, %2;" : "=f"(r.v[i]) : "f"(a.v[i]), "f"(b));
  return r;
}
template <int N>
__device__ __forceinline__ Vec<N> load_(const float* p) {
  Vec<N> r;
  ld_f32_vec<N>(p, r.v);
  return r;
}

// N neighbouring values of a row, as they lie in memory.
template <int N, bool BF16>
struct Pack {
  static constexpr int kBytes = N * (BF16 ? 2 : 4);
  uint32_t w[kBytes < 4 ? 1 : kBytes / 4];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (uint32_t& x : w) x = 0u;
  }
  __device__ __forceinline__ void load(const uint8_t* p) {
    if constexpr (kBytes == 2) {
      w[0] = __ldg(reinterpret_cast<const unsigned short*>(p));
    } else if constexpr (kBytes == 4) {
      w[0] = __ldg(reinterpret_cast<const unsigned*>(p));
    } else if constexpr (kBytes == 8) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = v.x; w[1] = v.y;
    } else {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    }
  }
  __device__ __forceinline__ Vec<N> get() const {
    Vec<N> r;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (BF16) r.v[i] = __uint_as_float((i & 1) ? (w[i >> 1] & 0xffff0000u) : (w[i >> 1] << 16));
      else r.v[i] = __uint_as_float(w[i]);
    }
    return r;
  }
  // one rounding, to the type of Wx, of values computed in fp32
  __device__ __forceinline__ void set(const Vec<N>& v) {
    if constexpr (!BF16) {
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = __float_as_uint(v.v[i]);
    } else if constexpr (N == 1) {
      w[0] = __bfloat16_as_ushort(__float2bfloat16_rn(v.v[0]));
    } else {
#pragma unroll
      for (int i = 0; i < N; i += 2) w[i / 2] = pack_bf16x2(v.v[i], v.v[i + 1]);
    }
  }
  __device__ __forceinline__ void store(uint8_t* p) const {
    if constexpr (kBytes == 2) *reinterpret_cast<unsigned short*>(p) = static_cast<unsigned short>(w[0]);
    else if constexpr (kBytes == 4) *reinterpret_cast<unsigned*>(p) = w[0];
    else if constexpr (kBytes == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};

constexpr float kLog2e = 1.4426950408889634f;
// tanh(y) as num / den, from b = -2 log2(e) y: with e = 2^-|b| it is (1 - e) / (1 + e) with the sign of y. That difference loses the digits of
// a small y: below 1/8 it is y - y^3/3 + 2 y^5/15, the start of tanh's series; what is left out of it is 2^-22 of y.
template <int N>
__device__ __forceinline__ void tanh_(const Vec<N>& b, Vec<N>& e, Vec<N>& num, Vec<N>& den) {
  constexpr float k = 0.34657359027997264f, kSmall = 0.125f / k;  // y = -k b
#pragma unroll
  for (int i = 0; i < N; ++i) e[i] = exp2_fast(-fabsf(b[i]));
  const Vec<N> one = splat<N>(1.0f), w = mul_(b, b), far = fma_(e, splat<N>(-1.0f), one);
  den = add_(one, e);
  Vec<N> near = fma_(w, splat<N>(-k * k * k * k * k * 2.0f / 15.0f), splat<N>(k * k * k / 3.0f));
  near = mul_(mul_(fma_(w, near, splat<N>(-k)), b), den);
#pragma unroll
  for (int i = 0; i < N; ++i)
    num[i] = fabsf(b[i]) < kSmall ? near[i] : __uint_as_float(__float_as_uint(far[i]) | (~__float_as_uint(b[i]) & 0x80000000u));
}
// sigmoid(x) and tanh(y) from a = -log2(e) x and b = -2 log2(e) y with one reciprocal for both, and what their slopes take, 1 - sigmoid(x) and
// 1 - tanh(y)^2 = 4 e / (1 + e)^2, not by subtraction, which would lose the digits of a saturated gate's. The bound keeps the
// product of the denominators in range; past it the sigmoid is 2^-120.
template <int N>
__device__ __forceinline__ void sigmoid_tanh(const Vec<N>& a, const Vec<N>& b, Vec<N>& s, Vec<N>& rest, Vec<N>& t, Vec<N>& slope) {
  Vec<N> e, num, den;
  tanh_(b, e, num, den);
  const Vec<N> ea = exp2_(min_(a, 120.0f)), da = add_(splat<N>(1.0f), ea), r = rcp_(mul_(da, den)), inv = mul_(da, r);
  s = mul_(den, r);
  rest = mul_(ea, s);
  t = mul_(num, inv);
  slope = mul_(mul_(e, splat<N>(4.0f)), mul_(inv, inv));
}
template <int N>
__device__ __forceinline__ Vec<N> sigmoid_times_tanh(const Vec<N>& a, const Vec<N>& b) {
  Vec<N> e, num, den;
  tanh_(b, e, num, den);
  return mul_(num, rcp_(mul_(add_(splat<N>(1.0f), exp2_(min_(a, 120.0f))), den)));
}

// f = sigmoid(x) and u = 1 - f as one number, from log2(e) x: the smaller of the two, f itself or -u, so that neither loses its digits where
// the other is next to one. With p = 1 where it is -u and 0 where it is f: f = p + m, a step is c -> p c + (m c + v), and f u = |m| - m^2.
// The least subnormal, added where it would round to zero, keeps its sign; a step that is to leave the state alone has m = 0, v = 0.
template <int N>
__device__ __forceinline__ Vec<N> decay_(const Vec<N>& x) {
  Vec<N> q, m;
#pragma unroll
  for (int i = 0; i < N; ++i) q[i] = exp2_fast(-fabsf(x[i]));
  m = fma_(q, rcp_(add_(splat<N>(1.0f), q)), splat<N>(__uint_as_float(1u)));
#pragma unroll
  for (int i = 0; i < N; ++i) m[i] = __uint_as_float(__float_as_uint(m[i]) | (~__float_as_uint(x[i]) & 0x80000000u));
  return m;
}
template <int N>
__device__ __forceinline__ Vec<N> side_(const Vec<N>& m) {  // p
  Vec<N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) asm("set.le.f32.f32 %0, %1, 0f00000000;" : "=f"(r.v[i]) : "f"(m.v[i]));
  return r;
}
// The same, made anew: in a later pass over the steps a register to hold it costs more than the instruction (the leaky backward tile in bf16
// spills 268 bytes without this, none with it).
template <int N>
__device__ __forceinline__ Vec<N> side_again(const Vec<N>& m) {
  Vec<N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("set.le.f32.f32 %0, %1, 0f00000000;" : "=f"(r.v[i]) : "f"(m.v[i]));
  return r;
}
template <int N>
__device__ __forceinline__ Vec<N> pick_(const Vec<N>& m, const Vec<N>& open, const Vec<N>& shut) {  // by p
  Vec<N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r[i] = m[i] <= 0.0f ? open[i] : shut[i];
  return r;
}
template <int N>
__device__ __forceinline__ Vec<N> minus_(const Vec<N>& a, const Vec<N>& b) { return fma_(b, splat<N>(-1.0f), a); }
template <int N>
__device__ __forceinline__ Vec<N> minus_u(const Vec<N>& m, const Vec<N>& p) { return add_(m, add_(p, splat<N>(-1.0f))); }
template <int N>
__device__ __forceinline__ Vec<N> minus_fu(const Vec<N>& m) {
  Vec<N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r[i] = -fabsf(m[i]);
  return fma_(m, m, r);
}
// f x with one rounding; where p is at hand for other things too, and where it is not.
template <int N>
__device__ __forceinline__ Vec<N> times_f(const Vec<N>& m, const Vec<N>& p, const Vec<N>& x) { return fma_(m, x, mul_(p, x)); }
template <int N>
__device__ __forceinline__ Vec<N> times_f(const Vec<N>& m, const Vec<N>& x) { return fma_(m, x, pick_(m, x, splat<N>(0.0f))); }

// Gates arrive as scale(g) (Wx + b): the factor that the exponentials want goes into one fused multiply-add with the bias. What a
// step does is kept as m and w; `step` takes a state through it, `first` the state zero. The leaky cell's w is z: with d = c - z its step
// is c - u d or z + f d, c + m d or z + m d. The LSTM's is v.
// kTile: steps of a tile. The LSTM's backward pass holds five values per step and channel: 64 steps leave room for two CTAs.
template <int CELL> struct LinCell;
template <> struct LinCell<FRNN_LINEAR_LEAKY> {
  static constexpr int G = 2, kTile = 128;
  static __device__ __forceinline__ constexpr float scale(int g) { return g == 0 ? kLog2e : 1.0f; }
  template <int N>
  static __device__ __forceinline__ void gates(const Vec<N>* x, Vec<N>& m, Vec<N>& w) {
    m = decay_(x[0]);
    w = x[1];
  }
  template <int N>
  static __device__ __forceinline__ Vec<N> step(const Vec<N>& m, const Vec<N>& w, const Vec<N>& c) { return fma_(m, minus_(c, w), pick_(m, c, w)); }
  template <int N>
  static __device__ __forceinline__ Vec<N> first(const Vec<N>& m, const Vec<N>& w) { return step(m, w, splat<N>(0.0f)); }
};
template <> struct LinCell<FRNN_LINEAR_LSTM> {
  static constexpr int G = 4, kTile = 64;
  static __device__ __forceinline__ constexpr float scale(int g) { return g == 1 ? kLog2e : (g == 2 ? -2.0f * kLog2e : -kLog2e); }
  template <int N>
  static __device__ __forceinline__ void gates(const Vec<N>* x, Vec<N>& m, Vec<N>& w) {
    m = decay_(x[1]);
    w = sigmoid_times_tanh(x[0], x[2]);
  }
  template <int N>
  static __device__ __forceinline__ Vec<N> step(const Vec<N>& m, const Vec<N>& w, const Vec<N>& c) { return fma_(side_(m), c, fma_(m, c, w)); }
  template <int N>
  static __device__ __forceinline__ Vec<N> first(const Vec<N>&, const Vec<N>& w) { return w; }
};

template <int VEC>
struct Lanes {
  static constexpr int kRow = VEC == 1 ? 32 : 64 / VEC;  // lanes that share a step
  static constexpr int kChannels = kRow * VEC;           // of a tile
  static constexpr int kSpans = 32 / kRow;               // spans of L steps in a warp
};

// A tile: place in time, row of channel blocks, b, channel block, the sequence's length.
struct TileId { int k, row, b, cg, len, mute; };
// The words that tiles of one (batch row, channel block) exchange: maps [tile][channel] (A, H), states [group][channel].
struct Exchange {
  uint8_t *maps, *states;
  int* counter;
  __device__ __forceinline__ Exchange(const LinParams& p, int row, int channels) {
    const long long rows = static_cast<long long>(p.B) * p.n_cg;
    const int groups = (p.n_tiles + kGroup - 1) / kGroup;
    counter = reinterpret_cast<int*>(p.exchange);
    maps = p.exchange + 128 + static_cast<long long>(row) * p.n_tiles * channels * 8;
    states = p.exchange + 128 + rows * p.n_tiles * channels * 8 + static_cast<long long>(row) * groups * channels * 4;
  }
};

__device__ __forceinline__ uint32_t ld_relaxed_gpu_u32(const void* p) {
  uint32_t v;
  asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void st_relaxed_gpu_v2(void* p, uint32_t x, uint32_t y) {
  asm volatile("st.relaxed.gpu.global.v2.u32 [%0], {%1, %2};" ::"l"(p), "r"(x), "r"(y) : "memory");
}

// Polls until `ready()`; false once the limit has run out or another CTA has given up.
template <typename F>
__device__ __forceinline__ bool lin_poll(const LinParams& p, F ready) {
  for (int fast = 0; fast < 32; ++fast)
    if (ready()) return true;
  const uint64_t t0 = global_timer_ns();
  for (uint32_t spins = 1;; ++spins) {
    if (ready()) return true;
    if ((spins & 63u) == 0u) {
      if (*static_cast<volatile int*>(p.err) != 0) return false;
      if (global_timer_ns() - t0 > p.wait_limit_ns) {
        if (atomicCAS(p.err, 0, kErrWaitPart) == 0) p.err[2] = static_cast<int>(blockIdx.x);
        return false;
      }
    }
  }
}

// Joining the tiles of a row, k = this tile in the order of the scan. Every tile but the last of its group hands out its map ...
__device__ __forceinline__ void lin_publish(const LinParams& p, const Exchange& x, int k, int channel, int channels, float a, float h) {
  if (k + 1 < p.n_tiles && k % kGroup != kGroup - 1)
    st_relaxed_gpu_v2(x.maps + (static_cast<long long>(k) * channels + channel) * 8, xg_clean(__float_as_uint(a)),
                      xg_clean(__float_as_uint(h)));
}
// ... the warps fetch those of the group's tiles in front of this one, asked for before the tile's own work and again where one had
// not been there ...
template <int CW, int NW>
struct Fetched {
  static constexpr int kTiles = (kGroup - 1 + NW - 1) / NW, kWords = CW / 32;
  uint2 map[kTiles][kWords];
  const uint8_t* from;
  int n_channels, count;  // count: tiles of the group in front of this one
  // Of this thread's channel, what its group starts from: a state, in a row's first group `first` [B][ND] (null: zeros; an ordinary load: with one
  // tile the same thread may write its last state there). Asked for here, not
  // behind the barrier where it is needed: 4 % of a forward pass.
  uint32_t start;
  __device__ __forceinline__ void ask(const LinParams& p, const TileId& id, int k, const float* first) {
    const int c0 = id.cg * CW, channels = min(CW, p.ND - c0);
    const Exchange x(p, id.row, CW);
    start = 0u;
    if (static_cast<int>(threadIdx.x) < channels) {
      if (k >= kGroup) start = ld_relaxed_gpu_u32(x.states + (static_cast<long long>(k / kGroup) * CW + threadIdx.x) * 4);
      else if (first != nullptr) start = __float_as_uint(first[static_cast<long long>(id.b) * p.ND + c0 + threadIdx.x]);
    }
    if (p.n_tiles == 1) return;
    from = x.maps + static_cast<long long>(k / kGroup * kGroup) * CW * 8;
    n_channels = channels;
    count = k % kGroup;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
#pragma unroll
      for (int j = 0; j < kWords; ++j) {
        const int q = (threadIdx.x >> 5) + i * NW, c = (threadIdx.x & 31) + 32 * j;
        if (q < count && c < n_channels) map[i][j] = ld_relaxed_gpu_v2(from + (q * CW + c) * 8);
      }
    }
  }
  __device__ __forceinline__ void put(const LinParams& p, float2 (*s_prev)[CW]) {
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
#pragma unroll
      for (int j = 0; j < kWords; ++j) {
        const int q = (threadIdx.x >> 5) + i * NW, c = (threadIdx.x & 31) + 32 * j;
        if (q >= count || c >= n_channels) continue;
        uint2 v = map[i][j];
        if (v.x == kXgFill || v.y == kXgFill) {
          const uint8_t* at = from + (q * CW + c) * 8;
          lin_poll(p, [&]() {
            v = ld_relaxed_gpu_v2(at);
            return v.x != kXgFill && v.y != kXgFill;
          });
        }
        s_prev[q][c] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
      }
    }
  }
};
// ... and they are composed in order with the state at the start of the group, which the last tile of the group before hands out.
template <int CW>
__device__ __forceinline__ float lin_carry(const LinParams& p, const Exchange& x, int k, bool mute, int channel, const float2 (*s_prev)[CW],
                                           uint32_t start, float a, float h) {
  const int group = k / kGroup, at = k % kGroup;
  float ra = 1.0f, rh = 0.0f;
#pragma unroll
  for (int q = 0; q < kGroup - 1; ++q) {
    if (q >= at) break;
    const float2 m = s_prev[q][channel];
    rh = fmaf(m.x, rh, m.y);
    ra *= m.x;
  }
  if (group > 0 && start == kXgFill) {
    lin_poll(p, [&]() {
      start = ld_relaxed_gpu_u32(x.states + (static_cast<long long>(group) * CW + channel) * 4);
      return start != kXgFill;
    });
  }
  const float carry = fmaf(ra, __uint_as_float(start), rh);
  if (k + 1 < p.n_tiles && at == kGroup - 1 && !mute)
    st_relaxed_gpu_u32(x.states + (static_cast<long long>(group + 1) * CW + channel) * 4, xg_clean(__float_as_uint(fmaf(a, carry, h))));
  return carry;
}

// The tile of this CTA, from the counter where tiles wait on one another. One thread divides for
// all (two divisions a thread are 2 % of a tile's time).
__device__ __forceinline__ TileId lin_tile(const LinParams& p, TileId* shared) {
  if (threadIdx.x == 0) {
    int id = static_cast<int>(blockIdx.x);
    TileId t;
    t.mute = 0;
    int from = 0;
    if (p.n_tiles > 1) {
      // test hook: with err[4] set, tiles from err[5] on in the order of the scan hand nothing out
      t.mute = static_cast<volatile int*>(p.err)[4];
      from = static_cast<volatile int*>(p.err)[5];
      id = atomicAdd(reinterpret_cast<int*>(p.exchange), 1) + 1;  // it starts at -1
    }
    const int rows = p.B * p.n_cg;
    t.k = id / rows;
    t.row = id - t.k * rows;
    t.b = t.row / p.n_cg;
    t.cg = t.row - t.b * p.n_cg;
    t.len = p.lengths == nullptr ? p.T : min(max(__ldg(p.lengths + t.b), 0), p.T);
    if (t.k < from) t.mute = 0;
    *shared = t;
  }
  __syncthreads();
  return *shared;
}

// What the CTA's warps share: their maps, the maps of earlier tiles, the values that the warps start from.
template <int CW, int NW>
struct Shared {
  float a[NW][CW], h[NW][CW], start[NW][CW];
  float2 prev[kGroup - 1][CW];
};

// From the maps of the CTA's warps to the value that each of them starts from; warps count backwards in reverse time.
// done(state, channel, carry, end) is called per channel with its place in [B][ND], what the tile starts from and what it ends with. The maps are in place and a barrier is behind them.
template <int CW, int NW, bool REVERSE, typename F>
__device__ __forceinline__ void lin_join(const LinParams& p, const TileId& id, int k, Shared<CW, NW>& s, Fetched<CW, NW>& got, F done) {
  const int nw = blockDim.x >> 5, c0 = id.cg * CW, n_channels = min(CW, p.ND - c0);
  const bool mute = id.mute != 0;
  const Exchange x(p, id.row, CW);
  const int c = threadIdx.x;  // a CTA has as many threads as a tile has channels, or more
  float a = 1.0f, h = 0.0f;
  if (c < n_channels) {
#pragma unroll 4
    for (int i = 0; i < nw; ++i) {
      const int w = REVERSE ? nw - 1 - i : i;
      const float wa = s.a[w][c], wh = s.h[w][c];
      h = fmaf(wa, h, wh);
      a *= wa;
    }
    if (p.n_tiles > 1 && !mute) lin_publish(p, x, k, c, CW, a, h);
  }
  if (p.n_tiles > 1) {
    got.put(p, s.prev);
    __syncthreads();
  }
  if (c < n_channels) {
    const long long state = static_cast<long long>(id.b) * p.ND + c0 + c;
    float carry = __uint_as_float(got.start);
    if (p.n_tiles > 1) carry = lin_carry<CW>(p, x, k, mute, c, s.prev, got.start, a, h);
    done(state, c0 + c, carry, fmaf(a, carry, h));
#pragma unroll 4
    for (int i = 0; i < nw; ++i) {
      const int w = REVERSE ? nw - 1 - i : i;
      s.start[w][c] = carry;
      carry = fmaf(s.a[w][c], carry, s.h[w][c]);
    }
  }
  __syncthreads();
}

// This thread's part of a tile.
template <int VEC, int L, int TILE>
struct Place {
  int k, b, c0, chl, ch, warp, span, t0, len;
  bool ok, whole;  // ok: the channels exist; whole: and so do all steps of the warp
  __device__ __forceinline__ Place(const LinParams& p, const TileId& id, bool reverse) {
    using W = Lanes<VEC>;
    const int lane = threadIdx.x & 31;
    warp = threadIdx.x >> 5;
    k = reverse ? p.n_tiles - 1 - id.k : id.k;
    b = id.b;
    c0 = id.cg * W::kChannels;
    span = lane / W::kRow;
    chl = (lane % W::kRow) * VEC;
    ch = c0 + chl;
    t0 = k * TILE + (warp * W::kSpans + span) * L;
    ok = ch < p.ND;
    len = id.len;
    whole = k * TILE + (warp + 1) * W::kSpans * L <= len && c0 + W::kChannels <= p.ND;
  }
  __device__ __forceinline__ bool valid(int l) const { return ok && t0 + l < len; }
};

// The maps of the warp's spans, one to a lane, become those of what lies in front of each (behind, in reverse time); that of the whole
// warp goes to (a, h) in shared memory.
template <int VEC, bool REVERSE>
__device__ __forceinline__ void join_spans(int span, Vec<VEC>& A, Vec<VEC>& H, float* a, float* h) {
  using W = Lanes<VEC>;
  auto from = [&](const Vec<VEC>& v, int o) {
    Vec<VEC> r;
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      r[i] = REVERSE ? __shfl_down_sync(0xffffffffu, v[i], o * W::kRow) : __shfl_up_sync(0xffffffffu, v[i], o * W::kRow);
    return r;
  };
  const int at = REVERSE ? W::kSpans - 1 - span : span;  // place in the order of the scan
#pragma unroll
  for (int o = 1; o < W::kSpans; o *= 2) {
    const Vec<VEC> pa = from(A, o), ph = from(H, o);
    if (at >= o) {
      H = fma_(A, ph, H);
      A = mul_(A, pa);
    }
  }
  if (at == W::kSpans - 1) {
    st_f32_vec<VEC>(a, A.v);
    st_f32_vec<VEC>(h, H.v);
  }
  if constexpr (W::kSpans > 1) {
    A = from(A, 1);
    H = from(H, 1);
  }
  if (at == 0) {
    A = splat<VEC>(1.0f);
    H = splat<VEC>(0.0f);
  }
}

template <int CELL, int VEC>
__device__ __forceinline__ void load_bias(const LinParams& p, bool ok, int ch, Vec<VEC> (&bias)[LinCell<CELL>::G]) {
#pragma unroll
  for (int g = 0; g < LinCell<CELL>::G; ++g) {
    bias[g] = ok ? load_<VEC>(p.bias + static_cast<long long>(g) * p.ND + ch) : splat<VEC>(0.0f);
    bias[g] = mul_(bias[g], splat<VEC>(LinCell<CELL>::scale(g)));
  }
}
template <int CELL, int VEC, bool BF16>
__device__ __forceinline__ Vec<VEC> scaled(const Pack<VEC, BF16>& raw, const Vec<VEC>& bias, int g) {
  return fma_(raw.get(), splat<VEC>(LinCell<CELL>::scale(g)), bias);
}

template <int CELL, int VEC, int L, int NW, int MIN_CTAS, bool BF16>
__global__ void __launch_bounds__(NW * 32, MIN_CTAS) linear_fwd_kernel(const LinParams p) {
  using W = Lanes<VEC>;
  using Cell = LinCell<CELL>;
  using V = Vec<VEC>;
  constexpr int G = Cell::G, CW = W::kChannels;
  static_assert(NW * W::kSpans * L == Cell::kTile, "a full CTA covers a tile");
  __shared__ __align__(16) Shared<CW, NW> s;
  __shared__ TileId s_tile;
  const Place<VEC, L, Cell::kTile> at(p, lin_tile(p, &s_tile), false);

  const size_t es = BF16 ? 2 : 4, gate = static_cast<size_t>(p.ND) * es;
  const uint8_t* from = static_cast<const uint8_t*>(p.wx) + ((static_cast<size_t>(at.b) * p.T + at.t0) * G * p.ND + at.ch) * es;
  Pack<VEC, BF16> raw[L][G];
  if (at.whole) {
#pragma unroll
    for (int l = 0; l < L; ++l)
#pragma unroll
      for (int g = 0; g < G; ++g) {
        raw[l][g].load(from);
        from += gate;
      }
  } else {
#pragma unroll
    for (int l = 0; l < L; ++l)
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if (at.valid(l)) raw[l][g].load(from + (l * G + g) * gate);
        else raw[l][g].clear();
      }
  }
  Fetched<CW, NW> got;
  got.ask(p, s_tile, at.k, p.initial);
  V bias[G];
  load_bias<CELL, VEC>(p, at.ok, at.ch, bias);

  // The LSTM keeps the maps of this thread's steps up to each of them, the leaky cell only the decay of each step: its z's as they came in
  // and a third CTA per SM cost less than twice the registers (8 x 2048 x 4096: 120 us; with two CTAs 135, with the gates made twice 135).
  constexpr int MAPS = CELL == FRNN_LINEAR_LSTM ? L : 1, DECAYS = CELL == FRNN_LINEAR_LEAKY ? L : 1;
  V A[MAPS], H[MAPS], decay[DECAYS], a, h;
  auto gates = [&](int l, V& m, V& w) {
    V x[G];
#pragma unroll
    for (int g = 0; g < G; ++g) x[g] = scaled<CELL>(raw[l][g], bias[g], g);
    Cell::gates(x, m, w);
    if (!at.whole && !at.valid(l)) m = w = splat<VEC>(0.0f);  // a step behind the end of a sequence leaves its state alone
  };
#pragma unroll
  for (int l = 0; l < L; ++l) {
    V m, w;
    gates(l, m, w);
    if (l == 0) {
      a = times_f(m, splat<VEC>(1.0f));
      h = Cell::first(m, w);
    } else {
      h = Cell::step(m, w, h);
      a = times_f(m, a);
    }
    if constexpr (MAPS > 1) { A[l] = a; H[l] = h; }
    else decay[l] = m;
  }
  join_spans<VEC, false>(at.span, a, h, &s.a[at.warp][at.chl], &s.h[at.warp][at.chl]);
  __syncthreads();
  lin_join<CW, NW, false>(p, s_tile, at.k, s, got, [&](long long state, int channel, float carry, float end) {
    if (p.starts != nullptr && at.k > 0) p.starts[(static_cast<long long>(at.b) * (p.n_tiles - 1) + at.k - 1) * p.ND + channel] = carry;
    if (at.k == p.n_tiles - 1) p.last[state] = end;
  });
  if (!at.ok) return;
  V c = fma_(a, load_<VEC>(&s.start[at.warp][at.chl]), h);
  uint8_t* to = static_cast<uint8_t*>(p.hidden) + ((static_cast<size_t>(at.b) * p.T + at.t0) * p.ND + at.ch) * es;
#pragma unroll
  for (int l = 0; l < L; ++l) {
    V out;
    if constexpr (MAPS > 1) {
      out = fma_(A[l], c, H[l]);
      out = sigmoid_times_tanh(scaled<CELL>(raw[l][G - 1], bias[G - 1], G - 1), mul_(out, splat<VEC>(-2.0f * kLog2e)));
    } else {
      out = c = Cell::step(decay[l], scaled<CELL>(raw[l][1], bias[1], 1), c);
    }
    if (!at.whole) {
      if (at.t0 + l >= p.T) continue;
      if (!at.valid(l)) out = splat<VEC>(0.0f);
    }
    Pack<VEC, BF16> w;
    w.set(out);
    w.store(to);
    to += gate;
  }
}

template <int CELL, int VEC, int L, int NW, int MIN_CTAS, bool BF16>
__global__ void __launch_bounds__(NW * 32, MIN_CTAS) linear_bwd_kernel(const LinParams p) {
  using W = Lanes<VEC>;
  using Cell = LinCell<CELL>;
  using V = Vec<VEC>;
  constexpr bool LSTM = CELL == FRNN_LINEAR_LSTM;
  constexpr int G = Cell::G, CW = W::kChannels;
  static_assert(NW * W::kSpans * L == Cell::kTile, "a full CTA covers a tile");
  __shared__ __align__(16) Shared<CW, NW> s;
  __shared__ __align__(16) float s_db[NW][G][CW];  // first the maps of the recomputed states
  __shared__ TileId s_tile;
  static_assert(G >= 2, "room for the maps");
  float(*f_a)[CW] = reinterpret_cast<float(*)[CW]>(&s_db[0][0][0]);  // [NW][CW]
  float(*f_h)[CW] = f_a + NW;
  const int tid = threadIdx.x, nw = blockDim.x >> 5;
  const Place<VEC, L, Cell::kTile> at(p, lin_tile(p, &s_tile), true);
  const int kr = p.n_tiles - 1 - at.k;  // in the order of the scan

  const size_t es = BF16 ? 2 : 4, row_bytes = static_cast<size_t>(p.ND) * es, first = static_cast<size_t>(at.b) * p.T + at.t0;
  const uint8_t* from = static_cast<const uint8_t*>(p.wx) + (first * G * p.ND + at.ch) * es;
  const uint8_t* from_dh = static_cast<const uint8_t*>(p.d_hidden) + (first * p.ND + at.ch) * es;
  uint8_t* to = static_cast<uint8_t*>(p.d_wx) + (first * G * p.ND + at.ch) * es;
  Pack<VEC, BF16> raw[L][G], raw_dh[L];
  if (at.whole) {
#pragma unroll
    for (int l = 0; l < L; ++l) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        raw[l][g].load(from);
        from += row_bytes;
      }
      raw_dh[l].load(from_dh);
      from_dh += row_bytes;
    }
  } else {
#pragma unroll
    for (int l = 0; l < L; ++l) {
      if (at.valid(l)) {
#pragma unroll
        for (int g = 0; g < G; ++g) raw[l][g].load(from + (l * G + g) * row_bytes);
        raw_dh[l].load(from_dh + l * row_bytes);
      } else {
#pragma unroll
        for (int g = 0; g < G; ++g) raw[l][g].clear();
        raw_dh[l].clear();
      }
    }
  }
  Fetched<CW, NW> got;
  got.ask(p, s_tile, kr, p.d_last);
  // the state in front of the tile, channels as in lin_join
  const bool mine = tid < min(CW, p.ND - at.c0);
  float before = 0.0f;
  if (mine) {
    if (at.k > 0) before = __ldg(p.starts + (static_cast<long long>(at.b) * (p.n_tiles - 1) + at.k - 1) * p.ND + at.c0 + tid);
    else if (p.initial != nullptr) before = __ldg(p.initial + static_cast<long long>(at.b) * p.ND + at.c0 + tid);
  }
  V bias[G];
  load_bias<CELL, VEC>(p, at.ok, at.ch, bias);

  // the decays; the state in front of each step (leaky: less its z); the slopes of the LSTM's v by i and z
  V m[L], prev[L], by_i[LSTM ? L : 1], by_z[LSTM ? L : 1];
#pragma unroll
  for (int l = 0; l < L; ++l) {
    V x[G];
#pragma unroll
    for (int g = 0; g < G; ++g) x[g] = scaled<CELL>(raw[l][g], bias[g], g);
    if constexpr (LSTM) {
      m[l] = decay_(x[1]);
      V i, rest, z, slope;
      sigmoid_tanh(x[0], x[2], i, rest, z, slope);
      prev[l] = mul_(i, z);
      by_i[l] = mul_(prev[l], rest);
      by_z[l] = mul_(i, slope);
    } else {
      Cell::gates(x, m[l], prev[l]);  // w, until the states are known
    }
  }
  if (!at.whole) {
#pragma unroll
    for (int l = 0; l < L; ++l)
      if (!at.valid(l)) m[l] = prev[l] = splat<VEC>(0.0f);
  }
  V A = add_(side_(m[0]), m[0]), H = Cell::first(m[0], prev[0]);
#pragma unroll
  for (int l = 1; l < L; ++l) {
    H = Cell::step(m[l], prev[l], H);
    A = times_f(m[l], side_(m[l]), A);
  }
  join_spans<VEC, false>(at.span, A, H, &f_a[at.warp][at.chl], &f_h[at.warp][at.chl]);
  __syncthreads();
  if (mine) {
#pragma unroll 4
    for (int w = 0; w < nw; ++w) {
      s.start[w][tid] = before;
      before = fmaf(f_a[w][tid], before, f_h[w][tid]);
    }
  }
  __syncthreads();
  V c = at.ok ? load_<VEC>(&s.start[at.warp][at.chl]) : splat<VEC>(0.0f), db[G];
#pragma unroll
  for (int g = 0; g < G; ++g) db[g] = splat<VEC>(0.0f);
  c = fma_(A, c, H);
  // the gradient of each state through its hidden state; the output gate's is done with
  V dc[LSTM ? L : 1] = {};
  auto d_state = [&](int l) {
    if constexpr (LSTM) return dc[l];
    else return raw_dh[l].get();
  };
#pragma unroll
  for (int l = 0; l < L; ++l) {
    const V w = prev[l];
    prev[l] = LSTM ? c : minus_(c, w);
    c = Cell::step(m[l], w, c);
    if constexpr (LSTM) {
      V o, rest, tc, slope;
      sigmoid_tanh(scaled<CELL>(raw[l][3], bias[3], 3), mul_(c, splat<VEC>(-2.0f * kLog2e)), o, rest, tc, slope);
      const V dh_o = mul_(raw_dh[l].get(), o);
      dc[l] = mul_(dh_o, slope);
      V d_o = mul_(mul_(dh_o, tc), rest);
      if (!at.whole && !at.valid(l)) dc[l] = d_o = splat<VEC>(0.0f);
      db[3] = add_(db[3], d_o);
      if (at.whole || (at.ok && at.t0 + l < p.T)) {
        Pack<VEC, BF16> w;
        w.set(d_o);
        w.store(to + (l * G + 3) * row_bytes);
      }
    }
  }
  // what leaves this thread's steps towards earlier ones
  A = add_(side_again(m[L - 1]), m[L - 1]);
  V E = mul_(A, d_state(L - 1));
#pragma unroll
  for (int l = L - 2; l >= 0; --l) {
    const V g = add_(d_state(l), E), side = side_again(m[l]);
    E = times_f(m[l], side, g);
    A = times_f(m[l], side, A);
  }
  join_spans<VEC, true>(at.span, A, E, &s.a[at.warp][at.chl], &s.h[at.warp][at.chl]);
  __syncthreads();
  lin_join<CW, NW, true>(p, s_tile, kr, s, got, [&](long long state, int, float, float end) {
    if (at.k == 0 && p.d_initial != nullptr) p.d_initial[state] = end;
  });
  E = fma_(A, at.ok ? load_<VEC>(&s.start[at.warp][at.chl]) : splat<VEC>(0.0f), E);
  to += (L - 1) * G * row_bytes;
#pragma unroll
  for (int l = L - 1; l >= 0; --l) {
    constexpr int kHere = LSTM ? 3 : G;  // gates whose gradients are stored here
    V d[kHere];
    const V g = add_(d_state(l), E), minus = splat<VEC>(-1.0f), side = side_again(m[l]), q = minus_fu(m[l]);
    E = times_f(m[l], side, g);
    if constexpr (LSTM) {
      d[0] = mul_(g, by_i[l]);
      d[1] = mul_(mul_(g, prev[l]), mul_(q, minus));
      d[2] = mul_(g, by_z[l]);
    } else {
      const V mg = mul_(g, minus);
      d[0] = mul_(mul_(mg, q), prev[l]);
      d[1] = mul_(mg, minus_u(m[l], side));
    }
    if (!at.whole && !at.valid(l)) {
#pragma unroll
      for (int j = 0; j < kHere; ++j) d[j] = splat<VEC>(0.0f);
    }
#pragma unroll
    for (int j = 0; j < kHere; ++j) db[j] = add_(db[j], d[j]);
    if (at.whole || (at.ok && at.t0 + l < p.T)) {
#pragma unroll
      for (int j = 0; j < kHere; ++j) {
        Pack<VEC, BF16> w;
        w.set(d[j]);
        w.store(to + j * row_bytes);
      }
    }
    to -= G * row_bytes;
  }
#pragma unroll
  for (int o = W::kRow; o < 32; o *= 2) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      V other;
#pragma unroll
      for (int i = 0; i < VEC; ++i) other[i] = __shfl_xor_sync(0xffffffffu, db[g][i], o);
      db[g] = add_(db[g], other);
    }
  }
  if (at.span == 0) {
#pragma unroll
    for (int g = 0; g < G; ++g) st_f32_vec<VEC>(&s_db[at.warp][g][at.chl], db[g].v);
  }
  __syncthreads();
  for (int j = tid; j < G * CW; j += blockDim.x) {
    const int g = j / CW, cc = j % CW;
    if (at.c0 + cc >= p.ND) continue;
    float sum = 0.0f;
    for (int w = 0; w < nw; ++w) sum += s_db[w][g][cc];
    p.db_part[((static_cast<long long>(at.b) * p.n_tiles + at.k) * G + g) * p.ND + at.c0 + cc] = sum;
  }
}

// Many channels: there is no need to cut time. A thread walks its two channels (one, where ND is odd) through the whole sequence, the
// next steps' loads in flight while it computes; no exchange, a third of the instructions of a tile. The states it keeps for the
// backward pass are kWalkSteps apart: what the backward walk recomputes between two of them stays in registers.
// A step takes about 110 ns forward (LSTM 240) however many threads there are, until the memory is full, so it depends on the channels B N D who
// is faster; walk against tile, forward + backward, us: leaky bf16 65536 x T2048 234 + 378, 235 + 403; 81920 271 + 438, 296 + 504; 131072 331 + 533,
// 482 + 796; fp32 65536 363 + 488, 291 + 461; 131072 627 + 1003, 572 + 906. LSTM bf16 65536 x T1024 248 + 458, 207 + 413; 98304 430 + 700,
// 310 + 618; 131072 489 + 833, 414 + 814; 196608 727 + 1245, 623 + 1221; fp32 98304 436 + 794, 481 + 730; 131072 505 + 930, 646 + 968. The border does
// not know the type: walks win in the leaky cell's bf16 and the LSTM's fp32, tiles in the other two, by up to 25 % forward.
// Channels that are no multiple of four have slower tiles: 48960 x T512 55 + 91, 68 + 121 (LSTM 110 + 198, 125 + 242; fp32 112 + 268, 131 + 246). Up
// to 16 steps there is nothing to cut: 4 x 1 x 768 2.5 us, 4.9 in a tile.
constexpr int kWalkSteps = 8, kWalkThreads = 64;
constexpr long long kWalkChannels = 65536, kWalkLstmChannels = 131072, kWalkOddChannels = 32768;

template <int CELL, int VEC, bool BF16>
struct Walk {
  static constexpr int G = LinCell<CELL>::G, S = kWalkSteps;
  using V = Vec<VEC>;
  using P = Pack<VEC, BF16>;
  int b, ch, len;
  size_t gate;  // bytes from one gate (or hidden state) to the next
  bool ok;
  __device__ __forceinline__ Walk(const LinParams& p) {
    const int per_row = (p.ND + VEC - 1) / VEC;
    const long long id = static_cast<long long>(blockIdx.x) * kWalkThreads + threadIdx.x;
    b = static_cast<int>(id / per_row);
    ch = static_cast<int>(id - static_cast<long long>(b) * per_row) * VEC;
    ok = b < p.B;
    gate = static_cast<size_t>(p.ND) * (BF16 ? 2 : 4);
    len = !ok ? 0 : p.lengths == nullptr ? p.T : min(max(__ldg(p.lengths + b), 0), p.T);
  }
  // `per` values of S steps from step t, those in front of the end of the sequence
  template <int PER>
  __device__ __forceinline__ void load(P (&r)[S][PER], const void* base, int T, int t) const {
    const uint8_t* from = static_cast<const uint8_t*>(base) + (static_cast<size_t>(b) * T + t) * PER * gate + static_cast<size_t>(ch) * (BF16 ? 2 : 4);
    if (t >= 0 && t <= len - S) {
#pragma unroll
      for (int l = 0; l < S; ++l)
#pragma unroll
        for (int g = 0; g < PER; ++g) r[l][g].load(from + (l * PER + g) * gate);
    } else {
#pragma unroll
      for (int l = 0; l < S; ++l)
#pragma unroll
        for (int g = 0; g < PER; ++g)
          if (t >= 0 && t < len - l) r[l][g].load(from + (l * PER + g) * gate);
          else r[l][g].clear();
    }
  }
};

// The LSTM's with one channel a thread is held to six CTAs per SM; left alone it has registers for five (64 x 512 x 765: 162 us, so 110).
template <int CELL, int VEC, bool BF16>
__global__ void __launch_bounds__(kWalkThreads, CELL != FRNN_LINEAR_LSTM ? 7 : VEC == 1 ? 6 : 1) linear_fwd_walk_kernel(const LinParams p) {
  using W = Walk<CELL, VEC, BF16>;
  using Cell = LinCell<CELL>;
  using V = Vec<VEC>;
  constexpr int G = W::G, S = W::S;
  const W w(p);
  if (!w.ok) return;
  V bias[G];
  load_bias<CELL, VEC>(p, true, w.ch, bias);
  const size_t state = static_cast<size_t>(w.b) * p.ND + w.ch;
  V c = p.initial != nullptr ? load_<VEC>(p.initial + state) : splat<VEC>(0.0f);
  const int last_kept = (p.T - 1) / S;  // states 1 .. last_kept are kept, each in front of its step
  auto steps = [&](const Pack<VEC, BF16> (&raw)[S][G], int t) {
    if (t > 0 && p.starts != nullptr) st_f32_vec<VEC>(p.starts + (static_cast<size_t>(w.b) * last_kept + t / S - 1) * p.ND + w.ch, c.v);
    uint8_t* to = static_cast<uint8_t*>(p.hidden) + (static_cast<size_t>(w.b) * p.T + t) * w.gate + static_cast<size_t>(w.ch) * (BF16 ? 2 : 4);
#pragma unroll
    for (int l = 0; l < S; ++l) {
      V x[G], m, in;
#pragma unroll
      for (int g = 0; g < G; ++g) x[g] = scaled<CELL>(raw[l][g], bias[g], g);
      Cell::gates(x, m, in);
      if (t + l < w.len) {
        c = Cell::step(m, in, c);
        V out = c;
        if constexpr (CELL == FRNN_LINEAR_LSTM)
          out = sigmoid_times_tanh(scaled<CELL>(raw[l][G - 1], bias[G - 1], G - 1), mul_(c, splat<VEC>(-2.0f * kLog2e)));
        Pack<VEC, BF16> o;
        o.set(out);
        o.store(to + l * w.gate);
      }
    }
  };
  // groups of steps on their way: two of the leaky cell, one of the LSTM, whose four gates leave no room for more
  constexpr int AHEAD = CELL == FRNN_LINEAR_LSTM ? 1 : 2, R = AHEAD + 1;
  Pack<VEC, BF16> ring[R][S][G];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) w.load(ring[i], p.wx, p.T, i * S);
  for (int t = 0; t < w.len; t += R * S) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (i > 0 && t + i * S >= w.len) break;
      w.load(ring[(i + AHEAD) % R], p.wx, p.T, t + (i + AHEAD) * S);
      steps(ring[i], t + i * S);
    }
  }
  st_f32_vec<VEC>(p.last + state, c.v);
  Pack<VEC, BF16> zero;
  zero.clear();
  for (int q = w.len; q < p.T; ++q)
    zero.store(static_cast<uint8_t*>(p.hidden) + (static_cast<size_t>(w.b) * p.T + q) * w.gate + static_cast<size_t>(w.ch) * (BF16 ? 2 : 4));
}

template <int CELL, int VEC, bool BF16>
__global__ void __launch_bounds__(kWalkThreads, 7) linear_bwd_walk_kernel(const LinParams p) {
  using W = Walk<CELL, VEC, BF16>;
  using Cell = LinCell<CELL>;
  using V = Vec<VEC>;
  constexpr bool LSTM = CELL == FRNN_LINEAR_LSTM;
  constexpr int G = W::G, S = W::S;
  const W w(p);
  if (!w.ok) return;
  V bias[G], db[G];
  load_bias<CELL, VEC>(p, true, w.ch, bias);
#pragma unroll
  for (int g = 0; g < G; ++g) db[g] = splat<VEC>(0.0f);
  const size_t state = static_cast<size_t>(w.b) * p.ND + w.ch;
  const int last_kept = (p.T - 1) / S;
  uint8_t* const to = static_cast<uint8_t*>(p.d_wx) + static_cast<size_t>(w.b) * p.T * G * w.gate + static_cast<size_t>(w.ch) * (BF16 ? 2 : 4);
  Pack<VEC, BF16> zero;
  zero.clear();
  for (int q = w.len; q < p.T; ++q)
#pragma unroll
    for (int g = 0; g < G; ++g) zero.store(to + (static_cast<size_t>(q) * G + g) * w.gate);
  auto start = [&](int t) {
    if (t < 0) return splat<VEC>(0.0f);
    if (t > 0) return load_<VEC>(p.starts + (static_cast<size_t>(w.b) * last_kept + t / S - 1) * p.ND + w.ch);
    return p.initial != nullptr ? load_<VEC>(p.initial + state) : splat<VEC>(0.0f);
  };
  V E = p.d_last != nullptr ? load_<VEC>(p.d_last + state) : splat<VEC>(0.0f);
  const V minus = splat<VEC>(-1.0f);
  auto steps = [&](const Pack<VEC, BF16> (&raw)[S][G], const Pack<VEC, BF16> (&dh)[S][1], V c, int t) {
    V m[S], prev[S], by_i[LSTM ? S : 1], by_z[LSTM ? S : 1], sum[G];
#pragma unroll
    for (int g = 0; g < G; ++g) sum[g] = splat<VEC>(0.0f);
#pragma unroll
    for (int l = 0; l < S; ++l) {
      V x[G], in;
#pragma unroll
      for (int g = 0; g < G; ++g) x[g] = scaled<CELL>(raw[l][g], bias[g], g);
      if constexpr (LSTM) {
        m[l] = decay_(x[1]);
        V i, rest, z, slope;
        sigmoid_tanh(x[0], x[2], i, rest, z, slope);
        in = mul_(i, z);
        by_i[l] = mul_(in, rest);
        by_z[l] = mul_(i, slope);
      } else {
        Cell::gates(x, m[l], in);
      }
      prev[l] = LSTM ? c : minus_(c, in);
      c = Cell::step(m[l], in, c);
    }
#pragma unroll
    for (int l = S - 1; l >= 0; --l) {
      if (t + l < w.len) {
        V d[G], g = dh[l][0].get();
        const V side = side_again(m[l]), q = minus_fu(m[l]);
        if constexpr (LSTM) {
          V o, rest, tc, slope;
          const V c_l = l == S - 1 ? c : prev[l == S - 1 ? l : l + 1];
          sigmoid_tanh(scaled<CELL>(raw[l][3], bias[3], 3), mul_(c_l, splat<VEC>(-2.0f * kLog2e)), o, rest, tc, slope);
          const V dh_o = mul_(g, o);
          d[3] = mul_(mul_(dh_o, tc), rest);
          g = fma_(dh_o, slope, E);
          d[0] = mul_(g, by_i[l]);
          d[1] = mul_(mul_(g, prev[l]), mul_(q, minus));
          d[2] = mul_(g, by_z[l]);
        } else {
          g = add_(g, E);
          const V mg = mul_(g, minus);
          d[0] = mul_(mul_(mg, q), prev[l]);
          d[1] = mul_(mg, minus_u(m[l], side));
        }
        E = times_f(m[l], side, g);
#pragma unroll
        for (int j = 0; j < G; ++j) {
          sum[j] = add_(sum[j], d[j]);
          Pack<VEC, BF16> o;
          o.set(d[j]);
          o.store(to + (static_cast<size_t>(t + l) * G + j) * w.gate);
        }
      }
    }
#pragma unroll
    for (int g = 0; g < G; ++g) db[g] = add_(db[g], sum[g]);
  };
  Pack<VEC, BF16> raw[2][S][G], dh[2][S][1];
  V c[2];
  int t = (w.len - 1) / S * S;
  if (w.len > 0) {
    w.load(raw[0], p.wx, p.T, t);
    w.load(dh[0], p.d_hidden, p.T, t);
    c[0] = start(t);
  }
  for (; t >= 0 && w.len > 0; t -= 2 * S) {
    w.load(raw[1], p.wx, p.T, t - S);
    w.load(dh[1], p.d_hidden, p.T, t - S);
    c[1] = start(t - S);
    steps(raw[0], dh[0], c[0], t);
    if (t - S < 0) break;
    w.load(raw[0], p.wx, p.T, t - 2 * S);
    w.load(dh[0], p.d_hidden, p.T, t - 2 * S);
    c[0] = start(t - 2 * S);
    steps(raw[1], dh[1], c[1], t - S);
  }
  if (p.d_initial != nullptr) st_f32_vec<VEC>(p.d_initial + state, E.v);
#pragma unroll
  for (int g = 0; g < G; ++g) st_f32_vec<VEC>(p.db_part + (static_cast<size_t>(w.b) * G + g) * p.ND + w.ch, db[g].v);
}

int lin_vec(int ND) { return ND % 4 == 0 ? 4 : 1; }
int lin_channels(int ND) { return lin_vec(ND) == 1 ? 32 : 64; }
// Enough channels for every SM to keep its loads in flight without cutting time, or next to no time to cut.
bool lin_walk(int function, long long B, int T, long long ND) {
  const long long many = ND % 4 != 0 ? kWalkOddChannels : (function == FRNN_LINEAR_LSTM ? kWalkLstmChannels : kWalkChannels);
  return T <= 2 * kWalkSteps || B * ND >= many;
}

template <int CELL, int VEC, bool BF16, bool BACKWARD>
int launch_walk(const LinParams& p, cudaStream_t s) {
  const long long threads = static_cast<long long>(p.B) * ((p.ND + VEC - 1) / VEC), blocks = (threads + kWalkThreads - 1) / kWalkThreads;
  if (blocks > 0x7fffffffLL) return -2;
  if constexpr (BACKWARD) linear_bwd_walk_kernel<CELL, VEC, BF16><<<static_cast<unsigned>(blocks), kWalkThreads, 0, s>>>(p);
  else linear_fwd_walk_kernel<CELL, VEC, BF16><<<static_cast<unsigned>(blocks), kWalkThreads, 0, s>>>(p);
  return static_cast<int>(cudaGetLastError());
}

template <int CELL, int VEC, int LF, int LB, bool BF16>
int launch_one(const LinParams& p, bool backward, cudaStream_t s) {
  constexpr int kSpans = Lanes<VEC>::kSpans, kTile = LinCell<CELL>::kTile, kNWF = kTile / (kSpans * LF), kNWB = kTile / (kSpans * LB);
  const long long tiles = static_cast<long long>(p.B) * p.n_cg * p.n_tiles;
  if (tiles > 0x7fffffffLL) return -2;
  const int l = backward ? LB : LF;
  int warps = backward ? kNWB : kNWF;
  static_assert((2 * kWalkSteps + kSpans * LF) / (kSpans * LF) * 32 >= Lanes<VEC>::kChannels, "a thread for every channel of the shortest tile");
  static_assert((2 * kWalkSteps + kSpans * LB) / (kSpans * LB) * 32 >= Lanes<VEC>::kChannels, "a thread for every channel of the shortest tile");
  if (p.n_tiles == 1) warps = (p.T + kSpans * l - 1) / (kSpans * l);
  constexpr int kCtas = CELL == FRNN_LINEAR_LEAKY && BF16 ? 3 : 512 / (kNWF * 32);
  if (!backward) linear_fwd_kernel<CELL, VEC, LF, kNWF, kCtas, BF16><<<static_cast<unsigned>(tiles), warps * 32, 0, s>>>(p);
  else linear_bwd_kernel<CELL, VEC, LB, kNWB, 512 / (kNWB * 32), BF16><<<static_cast<unsigned>(tiles), warps * 32, 0, s>>>(p);
  return static_cast<int>(cudaGetLastError());
}

// L, the steps of a thread: 32 values of a thread of the leaky cell, 32 and 16 of the LSTM's.
template <int CELL, bool BF16>
int launch_vec(const LinParams& p, bool backward, cudaStream_t s) {
  constexpr bool kLstm = CELL == FRNN_LINEAR_LSTM;
  if (lin_walk(CELL, p.B, p.T, p.ND)) {
    constexpr int kBack = kLstm ? 1 : 2;  // two channels of the LSTM's backward walk do not fit the registers
    if (backward) return p.ND % 2 == 0 ? launch_walk<CELL, kBack, BF16, true>(p, s) : launch_walk<CELL, 1, BF16, true>(p, s);
    return p.ND % 2 == 0 ? launch_walk<CELL, 2, BF16, false>(p, s) : launch_walk<CELL, 1, BF16, false>(p, s);
  }
  if (lin_vec(p.ND) == 4) return launch_one<CELL, 4, 8, kLstm ? 4 : 8, BF16>(p, backward, s);
  return launch_one<CELL, 1, 16, kLstm ? 8 : 16, BF16>(p, backward, s);
}

int launch(int function, int wx_bf16, const LinParams& p, bool backward, cudaStream_t s) {
  if (function == FRNN_LINEAR_LEAKY)
    return wx_bf16 ? launch_vec<FRNN_LINEAR_LEAKY, true>(p, backward, s) : launch_vec<FRNN_LINEAR_LEAKY, false>(p, backward, s);
  return wx_bf16 ? launch_vec<FRNN_LINEAR_LSTM, true>(p, backward, s) : launch_vec<FRNN_LINEAR_LSTM, false>(p, backward, s);
}

bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

// Common to both directions: sizes, exchange scratch.
int prepare(LinParams* p, const frnn_b200_linear_plan_t& plan, int B, int T, int N, int D, void* exchange, int wait_limit_ms, int* err,
            cudaStream_t s) {
  if (plan.exchange_bytes > 0 && (exchange == nullptr || err == nullptr || misaligned(exchange) || wait_limit_ms < 0)) return -5;
  p->B = B; p->T = T; p->ND = N * D; p->n_cg = (N * D + plan.tile_channels - 1) / plan.tile_channels; p->n_tiles = plan.tiles;
  p->err = err;
  p->exchange = static_cast<uint8_t*>(exchange);
  p->wait_limit_ns = wait_limit_ms > 0 ? static_cast<unsigned long long>(wait_limit_ms) * 1000000ull : kDefaultWaitNs;
  if (plan.exchange_bytes == 0) return 0;
  return static_cast<int>(cudaMemsetAsync(exchange, 0xFF, static_cast<size_t>(plan.exchange_bytes), s));
}

}  // namespace

}  // namespace frnn

extern "C" int frnn_b200_linear_plan(int function, int B, int T, int N, int D, frnn_b200_linear_plan_t* out) {
  using namespace frnn;
  if (out == nullptr) return -5;
  if (function != FRNN_LINEAR_LEAKY && function != FRNN_LINEAR_LSTM) return -1;
  if (B < 1 || T < 1 || N < 1 || D < 1) return -5;
  const long long nd = static_cast<long long>(N) * D;
  const int gates = function == FRNN_LINEAR_LEAKY ? 2 : 4;
  // the sum of db counts its columns past the end by up to 31, steps are counted so by less than two tiles
  if (nd * gates > 0x7fffffe0LL || T > 0x7fffff00) return -2;
  const int channels = lin_channels(static_cast<int>(nd));
  const int steps = function == FRNN_LINEAR_LEAKY ? LinCell<FRNN_LINEAR_LEAKY>::kTile : LinCell<FRNN_LINEAR_LSTM>::kTile;
  const long long blocks = B * ((nd + channels - 1) / channels), tiles = (static_cast<long long>(T) + steps - 1) / steps;
  if (blocks * tiles > 0x7fffffffLL) return -2;
  *out = {};
  out->gates = gates;
  if (lin_walk(function, B, T, nd)) {
    out->tile_steps = kWalkSteps;
    out->tile_channels = nd % 2 == 0 ? 2 : 1;
    out->tiles = 1;
    out->starts_bytes = 4LL * B * ((T - 1) / kWalkSteps) * nd;
    if (B > 1) out->dbpart_bytes = 4LL * B * gates * nd;
    return 0;
  }
  out->tile_steps = steps;
  out->tile_channels = channels;
  out->tiles = static_cast<int>(tiles);
  if (tiles > 1) {
    const long long groups = (tiles + kGroup - 1) / kGroup;
    out->exchange_bytes = 128 + blocks * channels * (tiles * 8 + groups * 4);
    out->starts_bytes = 4LL * B * (tiles - 1) * nd;
  }
  if (B * tiles > 1) out->dbpart_bytes = 4LL * B * tiles * gates * nd;
  return 0;
}

extern "C" int frnn_b200_linear_forward(int function, const void* wx, int wx_bf16, const float* bias, const float* initial, const int* lengths,
                                        void* hidden, float* last, float* starts, void* exchange, int B, int T, int N, int D,
                                        int wait_limit_ms, int* err, void* stream) {
  using namespace frnn;
  if (!wx || !bias || !hidden || !last || misaligned(wx) || misaligned(bias) || misaligned(initial) || misaligned(hidden) || misaligned(last) ||
      misaligned(starts))
    return -5;
  LinParams p{};
  p.wx = wx; p.bias = bias; p.initial = initial; p.lengths = lengths; p.hidden = hidden; p.last = last; p.starts = starts;
  frnn_b200_linear_plan_t plan;
  int rc = frnn_b200_linear_plan(function, B, T, N, D, &plan);
  if (rc == 0) rc = prepare(&p, plan, B, T, N, D, exchange, wait_limit_ms, err, static_cast<cudaStream_t>(stream));
  return rc != 0 ? rc : launch(function, wx_bf16, p, false, static_cast<cudaStream_t>(stream));
}

extern "C" int frnn_b200_linear_backward(int function, const void* wx, int wx_bf16, const float* bias, const float* initial, const int* lengths,
                                         const float* starts, const void* d_hidden, const float* d_last, void* dwx, float* db,
                                         float* d_initial, float* db_part, void* exchange, int B, int T, int N, int D, int wait_limit_ms,
                                         int* err, void* stream) {
  using namespace frnn;
  if (!wx || !bias || !d_hidden || !dwx || !db || misaligned(wx) || misaligned(bias) || misaligned(initial) || misaligned(starts) ||
      misaligned(d_hidden) || misaligned(d_last) || misaligned(dwx) || misaligned(db) || misaligned(d_initial) || misaligned(db_part))
    return -5;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  LinParams p{};
  p.wx = wx; p.bias = bias; p.initial = initial; p.lengths = lengths; p.starts = const_cast<float*>(starts);
  p.d_hidden = d_hidden; p.d_last = d_last; p.d_wx = dwx; p.d_initial = d_initial;
  frnn_b200_linear_plan_t plan;
  int rc = frnn_b200_linear_plan(function, B, T, N, D, &plan);
  if (rc != 0) return rc;
  if ((plan.starts_bytes > 0 && starts == nullptr) || (plan.dbpart_bytes > 0 && db_part == nullptr)) return -5;
  rc = prepare(&p, plan, B, T, N, D, exchange, wait_limit_ms, err, s);
  if (rc != 0) return rc;
  const long long rows = static_cast<long long>(B) * p.n_tiles;
  p.db_part = rows > 1 ? db_part : db;
  rc = launch(function, wx_bf16, p, true, s);
  if (rc != 0 || rows == 1) return rc;
  const int cols = (function == FRNN_LINEAR_LEAKY ? 2 : 4) * p.ND;
  return static_cast<int>(column_sum(db_part, db, rows, cols, s));
}
