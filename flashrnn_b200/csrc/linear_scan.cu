// Gated linear recurrence: per channel (head, unit) of a batch row
//   c_t = f_t c_{t-1} + v_t,   f_t = 1 - u_t,   u_t = sigmoid(-(x_f + b_f))
//   leaky (f, z):       v = u z,                      hidden = c
//   lstm  (i, f, z, o): v = sigmoid(i) tanh(z),       hidden = sigmoid(o) tanh(c)
// with x the gate pre-activations Wx[B,T,G,N,D]. There is no recurrent matrix, so a span of steps is the map
// c -> A c + H with A = prod f, and spans compose: (A2, H2) o (A1, H1) = (A2 A1, A2 H1 + H2). Written with u instead of f the
// step c + v - u c keeps full precision where f is next to one, which is where errors would add up over the most steps.
//
// Backward: with dc_t the gradient that reaches c_t through hidden_t, g_t = dc_t + f_{t+1} g_{t+1}; the same scan in reverse
// time over e_t = f_t (dc_t + e_{t+1}). The gates' gradients need c_{t-1}: it is recomputed from Wx, which has to be read
// anyway, and from the state at the start of every tile, which the forward pass keeps (1/128 of a history).
//
// One CTA takes a tile of 128 (64) steps x 64 channels of a batch row, read once into registers: a thread has L steps of VEC
// neighbouring channels, scans them, the tile's spans are joined by shuffles and through shared memory, and the second walk over
// the registers starts from the right state. Tiles of a row are joined through global memory: a tile publishes its (A, H), in
// groups of 16 tiles every tile composes the maps of those in front of it, in order, with the state at the start of its group,
// and the last tile of a group publishes the state at the start of the next. The order of the sums does not depend on timing, so
// two calls give the same bits. CTAs take their tiles from a counter, earlier steps first: whoever is waited for has started.
#include "../../include/flashrnn_b200.h"

#include "frnn_common.cuh"

namespace frnn {

namespace {

constexpr int kGroup = 16;   // tiles of a group
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

// VEC neighbouring values of a row, as they lie in memory.
template <int VEC, bool BF16>
struct Pack {
  static constexpr int kBytes = VEC * (BF16 ? 2 : 4);
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
  __device__ __forceinline__ float get(int i) const {
    if constexpr (BF16) return __uint_as_float((i & 1) ? (w[i >> 1] & 0xffff0000u) : (w[i >> 1] << 16));
    else return __uint_as_float(w[i]);
  }
  // one rounding, to the type of Wx, of a value computed in fp32
  __device__ __forceinline__ void set(const float* v) {
    if constexpr (!BF16) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) w[i] = __float_as_uint(v[i]);
    } else if constexpr (VEC == 1) {
      w[0] = __bfloat16_as_ushort(__float2bfloat16_rn(v[0]));
    } else {
#pragma unroll
      for (int i = 0; i < VEC; i += 2) w[i / 2] = pack_bf16x2(v[i], v[i + 1]);
    }
  }
  __device__ __forceinline__ void store(uint8_t* p) const {
    if constexpr (kBytes == 2) *reinterpret_cast<unsigned short*>(p) = static_cast<unsigned short>(w[0]);
    else if constexpr (kBytes == 4) *reinterpret_cast<unsigned*>(p) = w[0];
    else if constexpr (kBytes == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// min that keeps a NaN
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;
// sigmoid(x) and tanh(y) from a = -log2(e) x and b = -2 log2(e) y with one reciprocal for both: 1 / (1 + 2^a) and
// (1 - 2^b) / (1 + 2^b). The bounds keep the product of the denominators in range; past them the results are 0 and -1 anyway.
__device__ __forceinline__ void sigmoid_tanh(float a, float b, float& s, float& t) {
  const float ea = exp2_fast(min_nan(a, 80.0f)), eb = exp2_fast(min_nan(b, 43.0f)), da = 1.0f + ea, db = 1.0f + eb, r = rcp_fast(da * db);
  s = db * r;
  t = (1.0f - eb) * (da * r);
}
__device__ __forceinline__ float sigmoid_times_tanh(float a, float b) {
  const float ea = exp2_fast(min_nan(a, 80.0f)), eb = exp2_fast(min_nan(b, 43.0f));
  return (1.0f - eb) * rcp_fast((1.0f + ea) * (1.0f + eb));
}

// Gates arrive as scale(g) (Wx + b): the factor that the exponentials want goes into one fused multiply-add with the bias.
// kTile: steps of a tile. The LSTM's backward pass holds five values per step and channel: 64 steps leave room for two CTAs.
template <int CELL> struct LinCell;
template <> struct LinCell<FRNN_LINEAR_LEAKY> {
  static constexpr int G = 2, kTile = 128;
  static __device__ __forceinline__ constexpr float scale(int g) { return g == 0 ? kLog2e : 1.0f; }
  static __device__ __forceinline__ void gates(const float* x, float& u, float& v) {
    u = rcp_fast(1.0f + exp2_fast(x[0]));
    v = u * x[1];
  }
  static __device__ __forceinline__ float hidden(float, float c) { return c; }
};
template <> struct LinCell<FRNN_LINEAR_LSTM> {
  static constexpr int G = 4, kTile = 64;
  static __device__ __forceinline__ constexpr float scale(int g) { return g == 1 ? kLog2e : (g == 2 ? -2.0f * kLog2e : -kLog2e); }
  static __device__ __forceinline__ void gates(const float* x, float& u, float& v) {
    u = rcp_fast(1.0f + exp2_fast(x[1]));
    v = sigmoid_times_tanh(x[0], x[2]);
  }
  static __device__ __forceinline__ float hidden(float o, float c) { return sigmoid_times_tanh(o, -2.0f * kLog2e * c); }
};

// c -> f c + v
__device__ __forceinline__ float lin_step(float u, float v, float c) { return fmaf(-u, c, c + v); }

template <int VEC>
struct Lanes {
  static constexpr int kRow = VEC == 1 ? 32 : 64 / VEC;  // lanes that share a step
  static constexpr int kChannels = kRow * VEC;           // of a tile
  static constexpr int kSpans = 32 / kRow;               // spans of L steps in a warp
};

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
  __device__ __forceinline__ void ask(const LinParams& p, const Exchange& x, int k, int channels) {
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
__device__ __forceinline__ float lin_carry(const LinParams& p, const Exchange& x, int k, int channel, const float2 (*s_prev)[CW], float first,
                                           float a, float h) {
  const int group = k / kGroup, at = k % kGroup;
  float ra = 1.0f, rh = 0.0f;
  for (int q = 0; q < at; ++q) {
    const float2 m = s_prev[q][channel];
    rh = fmaf(m.x, rh, m.y);
    ra *= m.x;
  }
  if (group > 0) {
    uint32_t v = kXgFill;
    lin_poll(p, [&]() {
      v = ld_relaxed_gpu_u32(x.states + (static_cast<long long>(group) * CW + channel) * 4);
      return v != kXgFill;
    });
    first = __uint_as_float(v);
  }
  const float carry = fmaf(ra, first, rh);
  if (k + 1 < p.n_tiles && at == kGroup - 1)
    st_relaxed_gpu_u32(x.states + (static_cast<long long>(group + 1) * CW + channel) * 4, xg_clean(__float_as_uint(fmaf(a, carry, h))));
  return carry;
}

// The tile of this CTA: from the counter where tiles wait on one another.
__device__ __forceinline__ int lin_tile(const LinParams& p, int* shared) {
  if (p.n_tiles == 1) return static_cast<int>(blockIdx.x);
  if (threadIdx.x == 0) *shared = atomicAdd(reinterpret_cast<int*>(p.exchange), 1) + 1;  // it starts at -1
  __syncthreads();
  return *shared;
}

// What the CTA's warps share: their maps, the maps of earlier tiles, the values that the warps start from.
template <int CW, int NW>
struct Shared {
  float a[NW][CW], h[NW][CW], start[NW][CW];
  float2 prev[kGroup - 1][CW];
};

template <int VEC>
__device__ __forceinline__ void ld_vec(const float* p, float (&v)[VEC]) { ld_f32_vec<VEC>(p, v); }
template <int VEC>
__device__ __forceinline__ void st_vec(float* p, const float (&v)[VEC]) { st_f32_vec<VEC>(p, v); }

// From the maps of the CTA's warps to the value that each of them starts from; warps count backwards in reverse time. `first` [B][ND]
// (null: zeros) is what the row starts from; done(state, channel, carry, end) is called per channel with its place in [B][ND], what
// the tile starts from and what it ends with. The maps are in place and a barrier is behind them.
template <int CW, int NW, bool REVERSE, typename F>
__device__ __forceinline__ void lin_join(const LinParams& p, int row, int k, const float* first, Shared<CW, NW>& s, const Fetched<CW, NW>& got,
                                         F done) {
  const int nw = blockDim.x >> 5, b = row / p.n_cg, c0 = (row % p.n_cg) * CW, n_channels = min(CW, p.ND - c0);
  const Exchange x(p, row, CW);
  float a[CW / 32], h[CW / 32];
#pragma unroll
  for (int r = 0; r < CW / 32; ++r) {  // a second round only in a CTA of one warp
    const int c = threadIdx.x + r * blockDim.x;
    a[r] = 1.0f; h[r] = 0.0f;
    if (c >= n_channels) continue;
#pragma unroll 4
    for (int i = 0; i < nw; ++i) {
      const int w = REVERSE ? nw - 1 - i : i;
      const float wa = s.a[w][c], wh = s.h[w][c];
      h[r] = fmaf(wa, h[r], wh);
      a[r] *= wa;
    }
    if (p.n_tiles > 1) lin_publish(p, x, k, c, CW, a[r], h[r]);
  }
  if (p.n_tiles > 1) {
    const_cast<Fetched<CW, NW>&>(got).put(p, s.prev);
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < CW / 32; ++r) {
    const int c = threadIdx.x + r * blockDim.x;
    if (c >= n_channels) continue;
    const long long state = static_cast<long long>(b) * p.ND + c0 + c;
    float carry = first != nullptr && k < kGroup ? __ldg(first + state) : 0.0f;
    if (p.n_tiles > 1) carry = lin_carry<CW>(p, x, k, c, s.prev, carry, a[r], h[r]);
    done(state, c0 + c, carry, fmaf(a[r], carry, h[r]));
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
  int k, row, b, c0, chl, ch, warp, span, t0, len;
  bool ok, whole;  // ok: the channels exist; whole: and so do all steps of the warp
  __device__ __forceinline__ Place(const LinParams& p, int id, bool reverse) {
    using W = Lanes<VEC>;
    const int lane = threadIdx.x & 31, rows = p.B * p.n_cg;
    warp = threadIdx.x >> 5;
    k = id / rows;
    row = id - k * rows;
    if (reverse) k = p.n_tiles - 1 - k;
    b = row / p.n_cg;
    c0 = (row - b * p.n_cg) * W::kChannels;
    span = lane / W::kRow;
    chl = (lane % W::kRow) * VEC;
    ch = c0 + chl;
    t0 = k * TILE + (warp * W::kSpans + span) * L;
    ok = ch < p.ND;
    len = p.lengths == nullptr ? p.T : min(max(__ldg(p.lengths + b), 0), p.T);
    whole = k * TILE + (warp + 1) * W::kSpans * L <= len && c0 + W::kChannels <= p.ND;
  }
  __device__ __forceinline__ bool valid(int l) const { return ok && t0 + l < len; }
};

// The maps of the warp's spans, one to a lane, become those of what lies in front of each (behind, in reverse time); that of the whole
// warp goes to (a, h) in shared memory.
template <int VEC, bool REVERSE>
__device__ __forceinline__ void join_spans(int span, float (&A)[VEC], float (&H)[VEC], float* a, float* h) {
  using W = Lanes<VEC>;
  auto from = [&](float v, int o) {
    return REVERSE ? __shfl_down_sync(0xffffffffu, v, o * W::kRow) : __shfl_up_sync(0xffffffffu, v, o * W::kRow);
  };
  const int at = REVERSE ? W::kSpans - 1 - span : span;  // place in the order of the scan
#pragma unroll
  for (int o = 1; o < W::kSpans; o *= 2) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float pa = from(A[i], o), ph = from(H[i], o);
      if (at >= o) {
        H[i] = fmaf(A[i], ph, H[i]);
        A[i] *= pa;
      }
    }
  }
  if (at == W::kSpans - 1) {
    st_vec<VEC>(a, A);
    st_vec<VEC>(h, H);
  }
  if constexpr (W::kSpans > 1) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      A[i] = from(A[i], 1);
      H[i] = from(H[i], 1);
    }
  }
  if (at == 0) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) { A[i] = 1.0f; H[i] = 0.0f; }
  }
}

template <int CELL, int VEC>
__device__ __forceinline__ void load_bias(const LinParams& p, bool ok, int ch, float (&bias)[LinCell<CELL>::G][VEC]) {
#pragma unroll
  for (int g = 0; g < LinCell<CELL>::G; ++g) {
    if (ok) {
      ld_vec<VEC>(p.bias + static_cast<long long>(g) * p.ND + ch, bias[g]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) bias[g][i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) bias[g][i] *= LinCell<CELL>::scale(g);
  }
}

template <int CELL, int VEC, int L, int NW, int MIN_CTAS, bool BF16>
__global__ void __launch_bounds__(NW * 32, MIN_CTAS) linear_fwd_kernel(const LinParams p) {
  using W = Lanes<VEC>;
  using Cell = LinCell<CELL>;
  constexpr int G = Cell::G, CW = W::kChannels;
  static_assert(NW * W::kSpans * L == Cell::kTile, "a full CTA covers a tile");
  __shared__ __align__(16) Shared<CW, NW> s;
  __shared__ int s_tile;
  const int id = lin_tile(p, &s_tile);
  const Place<VEC, L, Cell::kTile> at(p, id, false);

  const size_t es = BF16 ? 2 : 4, gate = static_cast<size_t>(p.ND) * es;
  const uint8_t* from = static_cast<const uint8_t*>(p.wx) + ((static_cast<size_t>(at.b) * p.T + at.t0) * G * p.ND + at.ch) * es;
  Pack<VEC, BF16> raw[L][G];
  if (at.whole) {
#pragma unroll
    for (int l = 0; l < L; ++l)
#pragma unroll
      for (int g = 0; g < G; ++g) raw[l][g].load(from + (l * G + g) * gate);
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
  if (p.n_tiles > 1) got.ask(p, Exchange(p, at.row, CW), at.k, min(CW, p.ND - at.c0));
  float bias[G][VEC];
  load_bias<CELL, VEC>(p, at.ok, at.ch, bias);

  // the maps of this thread's steps up to each of them
  float A[L][VEC], H[L][VEC], a[VEC], h[VEC];
#pragma unroll
  for (int l = 0; l < L; ++l) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float x[G];
#pragma unroll
      for (int g = 0; g < G; ++g) x[g] = fmaf(raw[l][g].get(i), Cell::scale(g), bias[g][i]);
      Cell::gates(x, A[l][i], H[l][i]);  // u and v
    }
  }
  if (!at.whole) {  // a step behind the end of a sequence leaves its state alone
#pragma unroll
    for (int l = 0; l < L; ++l)
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (!at.valid(l)) A[l][i] = H[l][i] = 0.0f;
  }
#pragma unroll
  for (int l = 0; l < L; ++l) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float u = A[l][i], v = H[l][i];
      if (l == 0) {
        A[0][i] = 1.0f - u;
      } else {
        H[l][i] = lin_step(u, v, H[l - 1][i]);
        A[l][i] = fmaf(-u, A[l - 1][i], A[l - 1][i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) { a[i] = A[L - 1][i]; h[i] = H[L - 1][i]; }
  join_spans<VEC, false>(at.span, a, h, &s.a[at.warp][at.chl], &s.h[at.warp][at.chl]);
  __syncthreads();
  lin_join<CW, NW, false>(p, at.row, at.k, p.initial, s, got, [&](long long state, int channel, float carry, float end) {
    if (p.starts != nullptr && at.k > 0) p.starts[(static_cast<long long>(at.b) * (p.n_tiles - 1) + at.k - 1) * p.ND + channel] = carry;
    if (at.k == p.n_tiles - 1) p.last[state] = end;
  });
  if (!at.ok) return;
  float c[VEC];
  ld_vec<VEC>(&s.start[at.warp][at.chl], c);
#pragma unroll
  for (int i = 0; i < VEC; ++i) c[i] = fmaf(a[i], c[i], h[i]);
  const size_t step = static_cast<size_t>(p.ND) * es;
  uint8_t* to = static_cast<uint8_t*>(p.hidden) + ((static_cast<size_t>(at.b) * p.T + at.t0) * p.ND + at.ch) * es;
#pragma unroll
  for (int l = 0; l < L; ++l) {
    float out[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float o = G == 4 ? fmaf(raw[l][G - 1].get(i), Cell::scale(G - 1), bias[G - 1][i]) : 0.0f;
      out[i] = Cell::hidden(o, fmaf(A[l][i], c[i], H[l][i]));
    }
    if (!at.whole) {
      if (at.t0 + l >= p.T) continue;
#pragma unroll
      for (int i = 0; i < VEC; ++i) out[i] = at.valid(l) ? out[i] : 0.0f;
    }
    Pack<VEC, BF16> w;
    w.set(out);
    w.store(to + l * step);
  }
}

template <int CELL, int VEC, int L, int NW, int MIN_CTAS, bool BF16>
__global__ void __launch_bounds__(NW * 32, MIN_CTAS) linear_bwd_kernel(const LinParams p) {
  using W = Lanes<VEC>;
  using Cell = LinCell<CELL>;
  constexpr int G = Cell::G, CW = W::kChannels;
  static_assert(NW * W::kSpans * L == Cell::kTile, "a full CTA covers a tile");
  __shared__ __align__(16) Shared<CW, NW> s;
  __shared__ __align__(16) float s_db[NW][G][CW];  // first the maps of the recomputed states and what their warps start from
  __shared__ int s_tile;
  static_assert(G >= 2, "room for the maps");
  float(*f_a)[CW] = reinterpret_cast<float(*)[CW]>(&s_db[0][0][0]);  // [NW][CW]
  float(*f_h)[CW] = f_a + NW;
  const int tid = threadIdx.x, nw = blockDim.x >> 5;
  const int id = lin_tile(p, &s_tile);
  const Place<VEC, L, Cell::kTile> at(p, id, true);
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
      for (int g = 0; g < G; ++g) raw[l][g].load(from + (l * G + g) * row_bytes);
      raw_dh[l].load(from_dh + l * row_bytes);
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
  if (p.n_tiles > 1) got.ask(p, Exchange(p, at.row, CW), kr, min(CW, p.ND - at.c0));
  // the state in front of the tile, channels as in lin_join
  float before[CW / 32];
#pragma unroll
  for (int r = 0; r < CW / 32; ++r) {
    const int c = tid + r * blockDim.x;
    before[r] = 0.0f;
    if (c >= min(CW, p.ND - at.c0)) continue;
    if (at.k > 0) before[r] = __ldg(p.starts + (static_cast<long long>(at.b) * (p.n_tiles - 1) + at.k - 1) * p.ND + at.c0 + c);
    else if (p.initial != nullptr) before[r] = __ldg(p.initial + static_cast<long long>(at.b) * p.ND + at.c0 + c);
  }
  float bias[G][VEC];
  load_bias<CELL, VEC>(p, at.ok, at.ch, bias);

  // u; the state in front of each step; the LSTM's i and z
  float u[L][VEC], prev[L][VEC], si[G == 4 ? L : 1][VEC], tz[G == 4 ? L : 1][VEC], A[VEC], H[VEC];
#pragma unroll
  for (int l = 0; l < L; ++l) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float x[G];
#pragma unroll
      for (int g = 0; g < G; ++g) x[g] = fmaf(raw[l][g].get(i), Cell::scale(g), bias[g][i]);
      if constexpr (G == 4) {
        u[l][i] = rcp_fast(1.0f + exp2_fast(x[1]));
        sigmoid_tanh(x[0], x[2], si[l][i], tz[l][i]);
        prev[l][i] = si[l][i] * tz[l][i];
      } else {
        Cell::gates(x, u[l][i], prev[l][i]);  // v, until the states are known
      }
    }
  }
  if (!at.whole) {
#pragma unroll
    for (int l = 0; l < L; ++l)
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (!at.valid(l)) u[l][i] = prev[l][i] = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    A[i] = 1.0f - u[0][i];
    H[i] = prev[0][i];
#pragma unroll
    for (int l = 1; l < L; ++l) {
      H[i] = lin_step(u[l][i], prev[l][i], H[i]);
      A[i] = fmaf(-u[l][i], A[i], A[i]);
    }
  }
  join_spans<VEC, false>(at.span, A, H, &f_a[at.warp][at.chl], &f_h[at.warp][at.chl]);
  __syncthreads();
#pragma unroll
  for (int r = 0; r < CW / 32; ++r) {
    const int c = tid + r * blockDim.x;
    if (c >= min(CW, p.ND - at.c0)) continue;
    float v = before[r];
#pragma unroll 4
    for (int w = 0; w < nw; ++w) {
      s.start[w][c] = v;
      v = fmaf(f_a[w][c], v, f_h[w][c]);
    }
  }
  __syncthreads();
  float c[VEC], db[G][VEC];
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int i = 0; i < VEC; ++i) db[g][i] = 0.0f;
  if (at.ok) {
    ld_vec<VEC>(&s.start[at.warp][at.chl], c);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) c[i] = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) c[i] = fmaf(A[i], c[i], H[i]);
  // the gradient of each state through its hidden state; the output gate's is done with
  float dc[G == 4 ? L : 1][VEC];
  auto d_state = [&](int l, int i) {
    if constexpr (G == 4) return dc[l][i];
    else return raw_dh[l].get(i);
  };
#pragma unroll
  for (int l = 0; l < L; ++l) {
    float d_o[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float v = prev[l][i];
      prev[l][i] = c[i];
      c[i] = lin_step(u[l][i], v, c[i]);
      if constexpr (G == 4) {
        float o, tc;
        sigmoid_tanh(fmaf(raw[l][3].get(i), Cell::scale(3), bias[3][i]), -2.0f * kLog2e * c[i], o, tc);
        const float dh_o = raw_dh[l].get(i) * o;
        dc[l][i] = dh_o * fmaf(-tc, tc, 1.0f);
        d_o[i] = dh_o * tc * (1.0f - o);
        if (!at.whole && !at.valid(l)) dc[l][i] = d_o[i] = 0.0f;
        db[3][i] += d_o[i];
      }
    }
    if constexpr (G == 4) {
      if (at.whole || (at.ok && at.t0 + l < p.T)) {
        Pack<VEC, BF16> w;
        w.set(d_o);
        w.store(to + (l * G + 3) * row_bytes);
      }
    }
  }
  // what leaves this thread's steps towards earlier ones
  float E[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const float g0 = d_state(L - 1, i);
    E[i] = fmaf(-u[L - 1][i], g0, g0);
    A[i] = 1.0f - u[L - 1][i];
#pragma unroll
    for (int l = L - 2; l >= 0; --l) {
      const float g = d_state(l, i) + E[i];
      E[i] = fmaf(-u[l][i], g, g);
      A[i] = fmaf(-u[l][i], A[i], A[i]);
    }
  }
  join_spans<VEC, true>(at.span, A, E, &s.a[at.warp][at.chl], &s.h[at.warp][at.chl]);
  __syncthreads();
  lin_join<CW, NW, true>(p, at.row, kr, p.d_last, s, got, [&](long long state, int, float, float end) {
    if (at.k == 0 && p.d_initial != nullptr) p.d_initial[state] = end;
  });
  float e[VEC];
  if (at.ok) {
    ld_vec<VEC>(&s.start[at.warp][at.chl], e);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) e[i] = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) E[i] = fmaf(A[i], e[i], E[i]);
#pragma unroll
  for (int l = L - 1; l >= 0; --l) {
    constexpr int kHere = G == 4 ? 3 : G;  // gates whose gradients are stored here
    float d[kHere][VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float g = d_state(l, i) + E[i], q = fmaf(-u[l][i], u[l][i], u[l][i]);  // u (1 - u)
      E[i] = fmaf(-u[l][i], g, g);
      if constexpr (G == 4) {
        const float gi = g * si[l][i];
        d[0][i] = gi * tz[l][i] * (1.0f - si[l][i]);
        d[1][i] = g * prev[l][i] * q;
        d[2][i] = gi * fmaf(-tz[l][i], tz[l][i], 1.0f);
      } else {
        d[0][i] = g * (prev[l][i] - (raw[l][1].get(i) + bias[1][i])) * q;
        d[1][i] = g * u[l][i];
      }
    }
    if (!at.whole) {
#pragma unroll
      for (int g = 0; g < kHere; ++g)
#pragma unroll
        for (int i = 0; i < VEC; ++i) d[g][i] = at.valid(l) ? d[g][i] : 0.0f;
    }
#pragma unroll
    for (int g = 0; g < kHere; ++g)
#pragma unroll
      for (int i = 0; i < VEC; ++i) db[g][i] += d[g][i];
    if (at.whole || (at.ok && at.t0 + l < p.T)) {
#pragma unroll
      for (int g = 0; g < kHere; ++g) {
        Pack<VEC, BF16> w;
        w.set(d[g]);
        w.store(to + (l * G + g) * row_bytes);
      }
    }
  }
#pragma unroll
  for (int o = W::kRow; o < 32; o *= 2) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < VEC; ++i) db[g][i] += __shfl_xor_sync(0xffffffffu, db[g][i], o);
  }
  if (at.span == 0) {
#pragma unroll
    for (int g = 0; g < G; ++g) st_vec<VEC>(&s_db[at.warp][g][at.chl], db[g]);
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

// out[j] = sum over rows of part[row][j], in a fixed order: 32 columns to a block, its 32 warps take rows in turn.
__global__ void __launch_bounds__(1024) linear_db_kernel(const float* __restrict__ part, float* __restrict__ out, long long rows, int cols) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = blockIdx.x * 32 + lane;
  float sum = 0.0f;
  if (j < cols)
    for (long long r = warp; r < rows; r += 32) sum += part[r * cols + j];
  s[warp][lane] = sum;
  __syncthreads();
  float v = s[lane][warp];  // column `warp` of this block
#pragma unroll
  for (int o = 16; o > 0; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (lane == 0 && blockIdx.x * 32 + warp < cols) out[blockIdx.x * 32 + warp] = v;
}

int lin_vec(int ND) { return ND % 4 == 0 ? 4 : 1; }
int lin_channels(int ND) { return lin_vec(ND) == 1 ? 32 : 64; }

template <int CELL, int VEC, int LF, int LB, bool BF16>
int launch_one(const LinParams& p, bool backward, cudaStream_t s) {
  constexpr int kSpans = Lanes<VEC>::kSpans, kTile = LinCell<CELL>::kTile, kNWF = kTile / (kSpans * LF), kNWB = kTile / (kSpans * LB);
  const long long tiles = static_cast<long long>(p.B) * p.n_cg * p.n_tiles;
  if (tiles > 0x7fffffffLL) return -2;
  const int l = backward ? LB : LF;
  int warps = backward ? kNWB : kNWF;
  if (p.n_tiles == 1) warps = (p.T + kSpans * l - 1) / (kSpans * l);
  if (!backward) linear_fwd_kernel<CELL, VEC, LF, kNWF, 512 / (kNWF * 32), BF16><<<static_cast<unsigned>(tiles), warps * 32, 0, s>>>(p);
  else linear_bwd_kernel<CELL, VEC, LB, kNWB, 512 / (kNWB * 32), BF16><<<static_cast<unsigned>(tiles), warps * 32, 0, s>>>(p);
  return static_cast<int>(cudaGetLastError());
}

// L, the steps of a thread: 32 values of a thread of the leaky cell, 32 and 16 of the LSTM's.
template <int CELL, bool BF16>
int launch_vec(const LinParams& p, bool backward, cudaStream_t s) {
  constexpr bool kLstm = CELL == FRNN_LINEAR_LSTM;
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
  if (nd * gates > 0x7fffffffLL) return -2;
  const int channels = lin_channels(static_cast<int>(nd));
  const int steps = function == FRNN_LINEAR_LEAKY ? LinCell<FRNN_LINEAR_LEAKY>::kTile : LinCell<FRNN_LINEAR_LSTM>::kTile;
  const long long blocks = B * ((nd + channels - 1) / channels), tiles = (static_cast<long long>(T) + steps - 1) / steps;
  if (blocks * tiles > 0x7fffffffLL) return -2;
  *out = {};
  out->gates = gates;
  out->tile_steps = steps;
  out->tile_channels = channels;
  out->tiles = static_cast<int>(tiles);
  if (tiles > 1) {
    const long long groups = (tiles + kGroup - 1) / kGroup;
    out->exchange_bytes = 128 + blocks * channels * (tiles * 8 + groups * 4);
    out->starts_bytes = 4 * B * (tiles - 1) * nd;
  }
  if (B * tiles > 1) out->dbpart_bytes = 4 * B * tiles * gates * nd;
  return 0;
}

extern "C" int frnn_b200_linear_forward(int function, const void* wx, int wx_bf16, const float* bias, const float* initial, const int* lengths,
                                        void* hidden, float* last, float* starts, void* exchange, int B, int T, int N, int D,
                                        int wait_limit_ms, int* err, void* stream) {
  using namespace frnn;
  if (!wx || !bias || !hidden || !last || misaligned(wx) || misaligned(hidden)) return -5;
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
  if (!wx || !bias || !d_hidden || !dwx || !db || misaligned(wx) || misaligned(d_hidden) || misaligned(dwx)) return -5;
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
  linear_db_kernel<<<(cols + 31) / 32, 1024, 0, s>>>(db_part, db, rows, cols);
  return static_cast<int>(cudaGetLastError());
}
