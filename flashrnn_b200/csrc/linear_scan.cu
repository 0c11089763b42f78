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
// One CTA takes a tile of 128 steps x 64 channels of a batch row, read once into registers: a thread has L steps of VEC
// neighbouring channels, scans them, the tile's spans are joined by shuffles and through shared memory, and the second walk over
// the registers starts from the right state. Tiles of a row are joined through global memory: a tile publishes its (A, H), in
// groups of 16 tiles every tile composes the maps of those in front of it, in order, with the state at the start of its group,
// and the last tile of a group publishes the state at the start of the next. The order of the sums does not depend on timing, so
// two calls give the same bits. CTAs take their tiles from a counter, earlier steps first: whoever is waited for has started.
#include "../../include/flashrnn_b200.h"

#include "frnn_common.cuh"

namespace frnn {

namespace {

constexpr int kTile = 128;   // steps of a tile
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
  __device__ __forceinline__ void load(const void* base, long long elem) {
    const uint8_t* p = static_cast<const uint8_t*>(base) + elem * (BF16 ? 2 : 4);
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
  __device__ __forceinline__ void store(void* base, long long elem) const {
    uint8_t* p = static_cast<uint8_t*>(base) + elem * (BF16 ? 2 : 4);
    if constexpr (kBytes == 2) *reinterpret_cast<unsigned short*>(p) = static_cast<unsigned short>(w[0]);
    else if constexpr (kBytes == 4) *reinterpret_cast<unsigned*>(p) = w[0];
    else if constexpr (kBytes == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};

template <int CELL> struct LinCell;
template <> struct LinCell<FRNN_LINEAR_LEAKY> {
  static constexpr int G = 2;
  static __device__ __forceinline__ void gates(const float* x, float& u, float& v) {
    u = sigmoid_p(-x[0]);
    v = u * x[1];
  }
  static __device__ __forceinline__ float hidden(const float*, float c) { return c; }
  // gradient of c through hidden
  static __device__ __forceinline__ float d_state(const float*, float, float dh) { return dh; }
  // g: the whole gradient of c_t
  static __device__ __forceinline__ void d_gates(const float* x, float u, float prev, float, float g, float, float* d) {
    d[0] = g * (prev - x[1]) * (u * (1.0f - u));
    d[1] = g * u;
  }
};
template <> struct LinCell<FRNN_LINEAR_LSTM> {
  static constexpr int G = 4;
  static __device__ __forceinline__ void gates(const float* x, float& u, float& v) {
    u = sigmoid_p(-x[1]);
    v = sigmoid_p(x[0]) * tanh_p(x[2]);
  }
  static __device__ __forceinline__ float hidden(const float* x, float c) { return sigmoid_p(x[3]) * tanh_p(c); }
  static __device__ __forceinline__ float d_state(const float* x, float c, float dh) {
    const float tc = tanh_p(c);
    return dh * sigmoid_p(x[3]) * (1.0f - tc * tc);
  }
  static __device__ __forceinline__ void d_gates(const float* x, float u, float prev, float c, float g, float dh, float* d) {
    const float i = sigmoid_p(x[0]), z = tanh_p(x[2]), o = sigmoid_p(x[3]), tc = tanh_p(c);
    d[0] = g * z * (i * (1.0f - i));
    d[1] = g * prev * (u * (1.0f - u));
    d[2] = g * i * (1.0f - z * z);
    d[3] = dh * tc * (o * (1.0f - o));
  }
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
// ... every warp fetches that of one tile of the group in front of this one ...
template <int CW>
__device__ __forceinline__ void lin_fetch(const LinParams& p, const Exchange& x, int k, int n_channels, float2 (*s_prev)[CW]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp >= k % kGroup) return;
  const uint8_t* from = x.maps + static_cast<long long>(k / kGroup * kGroup + warp) * CW * 8;
  for (int c = lane; c < n_channels; c += 32) {
    uint2 v = make_uint2(kXgFill, kXgFill);
    lin_poll(p, [&]() {
      v = ld_relaxed_gpu_v2(from + c * 8);
      return v.x != kXgFill && v.y != kXgFill;
    });
    s_prev[warp][c] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
  }
}
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

// From the maps of the CTA's warps in s_map to the value that each of them starts from, in s_start; warps count backwards in reverse
// time. `first` [B][ND] (null: zeros) is what the row starts from; done(state, carry, end) is called per channel with its place in
// [B][ND], what the tile starts from and what it ends with.
template <int CW, bool REVERSE, typename F>
__device__ __forceinline__ void lin_join(const LinParams& p, int row, int k, const float* first, float2 (*s_map)[CW], float2 (*s_prev)[CW],
                                         float (*s_start)[CW], F done) {
  const int nw = blockDim.x >> 5, b = row / p.n_cg, c0 = (row % p.n_cg) * CW, n_channels = min(CW, p.ND - c0);
  const Exchange x(p, row, CW);
  float a[CW / 32], h[CW / 32];
#pragma unroll
  for (int r = 0; r < CW / 32; ++r) {  // a second round only in a CTA of one warp
    const int c = threadIdx.x + r * blockDim.x;
    a[r] = 1.0f; h[r] = 0.0f;
    if (c >= n_channels) continue;
    for (int i = 0; i < nw; ++i) {
      const int w = REVERSE ? nw - 1 - i : i;
      const float2 m = s_map[w][c];
      s_map[w][c] = make_float2(a[r], h[r]);
      h[r] = fmaf(m.x, h[r], m.y);
      a[r] *= m.x;
    }
    if (p.n_tiles > 1) lin_publish(p, x, k, c, CW, a[r], h[r]);
  }
  if (p.n_tiles > 1) {
    lin_fetch<CW>(p, x, k, n_channels, s_prev);
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < CW / 32; ++r) {
    const int c = threadIdx.x + r * blockDim.x;
    if (c >= n_channels) continue;
    const long long state = static_cast<long long>(b) * p.ND + c0 + c;
    float carry = first != nullptr && k < kGroup ? __ldg(first + state) : 0.0f;
    if (p.n_tiles > 1) carry = lin_carry<CW>(p, x, k, c, s_prev, carry, a[r], h[r]);
    done(state, c0 + c, carry, fmaf(a[r], carry, h[r]));
    for (int w = 0; w < nw; ++w) s_start[w][c] = fmaf(s_map[w][c].x, carry, s_map[w][c].y);
  }
  __syncthreads();
}

template <int CELL, int VEC, int L, int NW, bool BF16>
__global__ void __launch_bounds__(NW * 32, 2) linear_fwd_kernel(const LinParams p) {
  using W = Lanes<VEC>;
  using Cell = LinCell<CELL>;
  constexpr int G = Cell::G, CW = W::kChannels;
  static_assert(NW * W::kSpans * L == kTile && NW >= kGroup - 1, "a full CTA covers a tile");
  __shared__ float2 s_map[NW][CW], s_prev[kGroup - 1][CW];
  __shared__ float s_start[NW][CW];
  __shared__ int s_tile;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int id = lin_tile(p, &s_tile);
  const int rows = p.B * p.n_cg, k = id / rows, row = id % rows, b = row / p.n_cg, c0 = (row % p.n_cg) * CW;
  const int span = lane / W::kRow, chl = (lane % W::kRow) * VEC, ch = c0 + chl;
  const int t0 = k * kTile + (warp * W::kSpans + span) * L;
  const bool ok = ch < p.ND;
  const int len = p.lengths == nullptr ? p.T : min(max(__ldg(p.lengths + b), 0), p.T);
  const int len_here = ok ? len : 0;  // channels past the last are no steps at all

  Pack<VEC, BF16> raw[L][G];
#pragma unroll
  for (int l = 0; l < L; ++l) {
    const long long at = ((static_cast<long long>(b) * p.T + t0 + l) * G) * p.ND + ch;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (t0 + l < len_here) raw[l][g].load(p.wx, at + static_cast<long long>(g) * p.ND);
      else raw[l][g].clear();
    }
  }
  float bias[G][VEC];
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int i = 0; i < VEC; ++i) bias[g][i] = ok ? __ldg(p.bias + static_cast<long long>(g) * p.ND + ch + i) : 0.0f;

  float u[L][VEC], v[L][VEC], A[VEC], H[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) { A[i] = 1.0f; H[i] = 0.0f; }
#pragma unroll
  for (int l = 0; l < L; ++l) {
    const bool valid = t0 + l < len_here;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float x[G];
#pragma unroll
      for (int g = 0; g < G; ++g) x[g] = raw[l][g].get(i) + bias[g][i];
      Cell::gates(x, u[l][i], v[l][i]);
      if (!valid) u[l][i] = v[l][i] = 0.0f;  // a step behind the end of a sequence leaves its state alone
      H[i] = lin_step(u[l][i], v[l][i], H[i]);
      A[i] = fmaf(-u[l][i], A[i], A[i]);
    }
  }
  // spans of the warp in front of this one
#pragma unroll
  for (int o = 1; o < W::kSpans; o *= 2) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float pa = __shfl_up_sync(0xffffffffu, A[i], o * W::kRow), ph = __shfl_up_sync(0xffffffffu, H[i], o * W::kRow);
      if (span >= o) {
        H[i] = fmaf(A[i], ph, H[i]);
        A[i] *= pa;
      }
    }
  }
  if (span == W::kSpans - 1) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) s_map[warp][chl + i] = make_float2(A[i], H[i]);
  }
  if constexpr (W::kSpans > 1) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      A[i] = __shfl_up_sync(0xffffffffu, A[i], W::kRow);
      H[i] = __shfl_up_sync(0xffffffffu, H[i], W::kRow);
    }
  }
  if (span == 0) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) { A[i] = 1.0f; H[i] = 0.0f; }
  }
  __syncthreads();
  lin_join<CW, false>(p, row, k, p.initial, s_map, s_prev, s_start, [&](long long state, int channel, float carry, float end) {
    if (p.starts != nullptr && k > 0) p.starts[(static_cast<long long>(b) * (p.n_tiles - 1) + k - 1) * p.ND + channel] = carry;
    if (k == p.n_tiles - 1) p.last[state] = end;
  });
  if (!ok) return;
  float c[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) c[i] = fmaf(A[i], s_start[warp][chl + i], H[i]);
#pragma unroll
  for (int l = 0; l < L; ++l) {
    if (t0 + l < p.T) {
      float out[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        float x[G];
#pragma unroll
        for (int g = 0; g < G; ++g) x[g] = raw[l][g].get(i) + bias[g][i];
        c[i] = lin_step(u[l][i], v[l][i], c[i]);
        out[i] = t0 + l < len ? Cell::hidden(x, c[i]) : 0.0f;
      }
      Pack<VEC, BF16> w;
      w.set(out);
      w.store(p.hidden, (static_cast<long long>(b) * p.T + t0 + l) * p.ND + ch);
    }
  }
}

template <int CELL, int VEC, int L, int NW, bool BF16>
__global__ void __launch_bounds__(NW * 32, CELL == FRNN_LINEAR_LEAKY ? 2 : 1) linear_bwd_kernel(const LinParams p) {
  using W = Lanes<VEC>;
  using Cell = LinCell<CELL>;
  constexpr int G = Cell::G, CW = W::kChannels;
  static_assert(NW * W::kSpans * L == kTile && NW >= kGroup - 1, "a full CTA covers a tile");
  // maps and starts of the recomputed states and of the gradients in reverse time; then the parts of db
  __shared__ float2 s_map[2][NW][CW], s_prev[kGroup - 1][CW];
  __shared__ float s_start[2][NW][CW];
  __shared__ int s_tile;
  static_assert(sizeof(s_map) >= sizeof(float) * NW * G * CW, "parts of db take the room of the maps");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nw = blockDim.x >> 5;
  const int id = lin_tile(p, &s_tile);
  const int rows = p.B * p.n_cg, kr = id / rows, k = p.n_tiles - 1 - kr;  // kr: in the order of the scan
  const int row = id % rows, b = row / p.n_cg, c0 = (row % p.n_cg) * CW;
  const int span = lane / W::kRow, chl = (lane % W::kRow) * VEC, ch = c0 + chl;
  const int t0 = k * kTile + (warp * W::kSpans + span) * L;
  const bool ok = ch < p.ND;
  const int len = p.lengths == nullptr ? p.T : min(max(__ldg(p.lengths + b), 0), p.T);
  const int len_here = ok ? len : 0;

  Pack<VEC, BF16> raw[L][G], raw_dh[L];
#pragma unroll
  for (int l = 0; l < L; ++l) {
    const long long step = static_cast<long long>(b) * p.T + t0 + l;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (t0 + l < len_here) raw[l][g].load(p.wx, (step * G + g) * p.ND + ch);
      else raw[l][g].clear();
    }
    if (t0 + l < len_here) raw_dh[l].load(p.d_hidden, step * p.ND + ch);
    else raw_dh[l].clear();
  }
  float bias[G][VEC];
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int i = 0; i < VEC; ++i) bias[g][i] = ok ? __ldg(p.bias + static_cast<long long>(g) * p.ND + ch + i) : 0.0f;

  // the states, as in the forward kernel
  float u[L][VEC], prev[L][VEC], A[VEC], H[VEC], total[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) { A[i] = 1.0f; H[i] = 0.0f; }
#pragma unroll
  for (int l = 0; l < L; ++l) {
    const bool valid = t0 + l < len_here;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float x[G], v;
#pragma unroll
      for (int g = 0; g < G; ++g) x[g] = raw[l][g].get(i) + bias[g][i];
      Cell::gates(x, u[l][i], v);
      if (!valid) u[l][i] = v = 0.0f;
      prev[l][i] = v;  // until the states are known
      H[i] = lin_step(u[l][i], v, H[i]);
      A[i] = fmaf(-u[l][i], A[i], A[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) total[i] = A[i];  // the decay over this thread's steps
#pragma unroll
  for (int o = 1; o < W::kSpans; o *= 2) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float pa = __shfl_up_sync(0xffffffffu, A[i], o * W::kRow), ph = __shfl_up_sync(0xffffffffu, H[i], o * W::kRow);
      if (span >= o) {
        H[i] = fmaf(A[i], ph, H[i]);
        A[i] *= pa;
      }
    }
  }
  if (span == W::kSpans - 1) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) s_map[0][warp][chl + i] = make_float2(A[i], H[i]);
  }
  if constexpr (W::kSpans > 1) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      A[i] = __shfl_up_sync(0xffffffffu, A[i], W::kRow);
      H[i] = __shfl_up_sync(0xffffffffu, H[i], W::kRow);
    }
  }
  if (span == 0) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) { A[i] = 1.0f; H[i] = 0.0f; }
  }
  __syncthreads();
  for (int c = tid; c < CW; c += blockDim.x) {
    if (c0 + c >= p.ND) continue;
    float h = 0.0f;
    if (k > 0) h = __ldg(p.starts + (static_cast<long long>(b) * (p.n_tiles - 1) + k - 1) * p.ND + c0 + c);
    else if (p.initial != nullptr) h = __ldg(p.initial + static_cast<long long>(b) * p.ND + c0 + c);
    for (int w = 0; w < nw; ++w) {
      s_start[0][w][c] = h;
      h = fmaf(s_map[0][w][c].x, h, s_map[0][w][c].y);
    }
  }
  __syncthreads();
  float c[VEC], dc[L][VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) c[i] = ok ? fmaf(A[i], s_start[0][warp][chl + i], H[i]) : 0.0f;
#pragma unroll
  for (int l = 0; l < L; ++l) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float x[G];
#pragma unroll
      for (int g = 0; g < G; ++g) x[g] = raw[l][g].get(i) + bias[g][i];
      const float v = prev[l][i];
      prev[l][i] = c[i];
      c[i] = lin_step(u[l][i], v, c[i]);
      dc[l][i] = t0 + l < len_here ? Cell::d_state(x, c[i], raw_dh[l].get(i)) : 0.0f;
    }
  }
  // the gradients that leave every span towards earlier steps
  float E[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) { A[i] = total[i]; E[i] = 0.0f; }
#pragma unroll
  for (int l = L - 1; l >= 0; --l) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float g = dc[l][i] + E[i];
      E[i] = fmaf(-u[l][i], g, g);
    }
  }
#pragma unroll
  for (int o = 1; o < W::kSpans; o *= 2) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float pa = __shfl_down_sync(0xffffffffu, A[i], o * W::kRow), pe = __shfl_down_sync(0xffffffffu, E[i], o * W::kRow);
      if (span + o < W::kSpans) {
        E[i] = fmaf(A[i], pe, E[i]);
        A[i] *= pa;
      }
    }
  }
  if (span == 0) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) s_map[1][warp][chl + i] = make_float2(A[i], E[i]);
  }
  if constexpr (W::kSpans > 1) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      A[i] = __shfl_down_sync(0xffffffffu, A[i], W::kRow);
      E[i] = __shfl_down_sync(0xffffffffu, E[i], W::kRow);
    }
  }
  if (span == W::kSpans - 1) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) { A[i] = 1.0f; E[i] = 0.0f; }
  }
  __syncthreads();
  lin_join<CW, true>(p, row, kr, p.d_last, s_map[1], s_prev, s_start[1], [&](long long state, int, float, float end) {
    if (k == 0 && p.d_initial != nullptr) p.d_initial[state] = end;
  });
  float db[G][VEC];
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int i = 0; i < VEC; ++i) db[g][i] = 0.0f;
#pragma unroll
  for (int i = 0; i < VEC; ++i) E[i] = ok ? fmaf(A[i], s_start[1][warp][chl + i], E[i]) : 0.0f;
#pragma unroll
  for (int l = L - 1; l >= 0; --l) {
    const bool valid = t0 + l < len_here;
    float d[G][VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float x[G], dg[G];
#pragma unroll
      for (int g = 0; g < G; ++g) x[g] = raw[l][g].get(i) + bias[g][i];
      const float g_c = dc[l][i] + E[i];
      E[i] = fmaf(-u[l][i], g_c, g_c);
      Cell::d_gates(x, u[l][i], prev[l][i], c[i], g_c, raw_dh[l].get(i), dg);
      c[i] = prev[l][i];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        d[g][i] = valid ? dg[g] : 0.0f;
        db[g][i] += d[g][i];
      }
    }
    if (ok && t0 + l < p.T) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        Pack<VEC, BF16> w;
        w.set(d[g]);
        w.store(p.d_wx, ((static_cast<long long>(b) * p.T + t0 + l) * G + g) * p.ND + ch);
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
  float* s_db = reinterpret_cast<float*>(&s_map[0][0][0]);  // [nw][G][CW]; the maps were last read in front of the last barrier
  if (span == 0) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < VEC; ++i) s_db[(warp * G + g) * CW + chl + i] = db[g][i];
  }
  __syncthreads();
  for (int j = tid; j < G * CW; j += blockDim.x) {
    const int g = j / CW, cc = j % CW;
    if (c0 + cc >= p.ND) continue;
    float sum = 0.0f;
    for (int w = 0; w < nw; ++w) sum += s_db[(w * G + g) * CW + cc];
    p.db_part[((static_cast<long long>(b) * p.n_tiles + k) * G + g) * p.ND + c0 + cc] = sum;
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

template <int CELL, int VEC, int L, int NW, bool BF16>
int launch_one(LinParams p, bool backward, cudaStream_t s) {
  const long long tiles = static_cast<long long>(p.B) * p.n_cg * p.n_tiles;
  if (tiles > 0x7fffffffLL) return -2;
  int warps = NW;
  if (p.n_tiles == 1) warps = (p.T + Lanes<VEC>::kSpans * L - 1) / (Lanes<VEC>::kSpans * L);
  if (!backward) linear_fwd_kernel<CELL, VEC, L, NW, BF16><<<static_cast<unsigned>(tiles), warps * 32, 0, s>>>(p);
  else linear_bwd_kernel<CELL, VEC, L, NW, BF16><<<static_cast<unsigned>(tiles), warps * 32, 0, s>>>(p);
  return static_cast<int>(cudaGetLastError());
}

template <int CELL, bool BF16>
int launch_vec(const LinParams& p, bool backward, cudaStream_t s) {
  if (lin_vec(p.ND) == 4) return launch_one<CELL, 4, 4, 16, BF16>(p, backward, s);
  return launch_one<CELL, 1, 8, 16, BF16>(p, backward, s);
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
  const long long blocks = B * ((nd + channels - 1) / channels), tiles = (static_cast<long long>(T) + kTile - 1) / kTile;
  if (blocks * tiles > 0x7fffffffLL) return -2;
  *out = {};
  out->gates = gates;
  out->tile_steps = kTile;
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
