// Matrix product with an epilogue, y = act(x W^T + bias) + residual, and its gradients. bf16 operands, fp32 accumulation in tensor
// memory, one rounding where a result is stored.
//
//   forward  y  [rows][outputs] : x  [rows][inputs]  (K-major)  . W  [outputs][inputs] (K-major),  K = inputs
//            z = x W^T + bias is kept for the backward pass where the activation's slope needs it: as fp16, which has 11
//            significant bits of it (the slope then is off by a few 2^-12; the gradients that it scales are rounded to the 8 bits of
//            bf16) and takes half the room of fp32; values past 65504, where slopes are 0 or 1, are held at 65504
//   dz = dy act'(z), rounded to bf16 for the tensor cores; dbias sums it before that rounding
//   dx [rows][inputs]           : dz [rows][outputs] (K-major)  . W                    (MN-major), K = outputs
//   dW [outputs][inputs]        : dz                 (MN-major) . x                    (MN-major), K = rows
//
// product_kernel: persistent, one CTA pair (cluster of two, cta_group::2) per two SMs, each pair walking 256 x NP output tiles.
// A CTA stages its 128 rows of A and half of the NP rows of B, so that a pair moves 32 KB per CTA and 64 k's where two
// single CTAs with 128 x 256 tiles move 48. One warp feeds the ring by TMA (128-byte swizzle), one thread of the even CTA issues
// the MMAs of both, 16 warps of each CTA take the accumulator out of tensor memory: two accumulators, so the epilogue of a tile
// runs under the contraction of the next. Rows and columns past the edges are read as zeros and not stored.
// Tiles that do not fill another round of all pairs are cut along K, so that their parts do: these go out in fp32 and are summed in
// order by product_join_kernel, which then has the epilogue. Few rows take product_rows_kernel.
//
// Bound: the tensor pipe where K is long. 64 k's of a 256 x 256 tile take 0.40 us (a library product's 0.37): five stages are
// enough (8192^3: three 1163 us, four 927, five 873, six 872; library 812). Short sums are bound by the epilogue's latency, hence its sixteen
// warps and the bias from a register: a tile of 768 k's takes 4.8 us (8192 x 768 x 2048 with bias, gelu and z 30.9 us, without an epilogue
// 24.7, library 23.2). Start and end of the kernel are 4.6 us.
#include "../../include/flashrnn_b200.h"

#include "column_sum.cuh"
#include "frnn_common.cuh"

namespace frnn {

namespace {

constexpr int kEpiWarps = 16;                     // four to each quarter of the tensor memory's lanes
constexpr int kThreads = (kEpiWarps + 2) * 32;    // then TMA, MMA
constexpr int kKC = 64;          // k's per stage: 128 bytes of bf16, one swizzle row
constexpr int kBufBytes = 2048;  // staging of a warp: two buffers of 32 rows x 64 bytes, a piece of 32 columns
// All of an SM's shared memory, whatever a tile needs of it: no CTA of another kernel shares the SM, so that none holds tensor memory there
// that this one's allocation, or its own peer on another SM, would have to wait for.
constexpr int kSmem = 227 * 1024 - 512;
// Stages of the ring: as many as fit beside the staging buffers. B along N comes in boxes of 64 columns, whole ones.
__host__ __device__ constexpr int stage_bytes_of(int np, bool b_mn) { return 16384 + (b_mn ? (np / 2 + 63) / 64 * 8192 : np / 2 * 128); }
__host__ __device__ constexpr int stages_of(int np, bool b_mn) { return (kSmem - 1024 - kEpiWarps * 2 * kBufBytes) / stage_bytes_of(np, b_mn); }
constexpr uint64_t kLimit = 2000000000ull;

struct ProductParams {
  const void* bias;  // [N] or null
  int* err;
  int bias_bf16, act, has_residual, has_z;
  int M, N, K;       // of the contraction
  int n_nt, chunks;
  // units of work: `whole` tiles, then the others in `parts` of chunks_per_part chunks of K each
  int parts, chunks_per_part;
  long long whole, n_units;
};

__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const void* tmap, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const void* tmap, uint32_t bar, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(c0), "r"(c1)
               : "memory");
}
// Both CTAs of the pair take part in these, one warp each.
__device__ __forceinline__ void tmem_alloc_pair(uint32_t dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(ncols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// D (256 x N over both CTAs' tensor memory) (+)= A (128 rows from each CTA) B (N / 2 rows from each); one thread of the even CTA.
__device__ __forceinline__ void umma_bf16_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      " .reg .pred p;\n"
      " setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrive on the barrier at this offset in both CTAs once every MMA issued so far has completed.
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
               "h"(static_cast<uint16_t>(3))
               : "memory");
}
__device__ __forceinline__ void umma_commit_pair_here(uint32_t bar) {  // ... of this CTA only
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
// Behind a wait that ran out or was called off: copies in flight land before their buffer is used again or the CTA leaves. From this GPU's
// memory they take a few microseconds.
__device__ __forceinline__ void settle() {
  const uint64_t t0 = global_timer_ns();
  while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void ld_shared_v4(uint32_t a, uint32_t (&v)[4]) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void st_shared_v4(uint32_t a, const uint32_t (&v)[4]) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// Two fp16 values; what is past their range becomes the largest one, a NaN stays one.
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  uint32_t r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
// Two fp32 operations in one instruction.
__device__ __forceinline__ void add2(float& a, float& b, float c, float d) {
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%0, %1};\n mov.b64 y, {%2, %3};\n add.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}" : "+f"(a), "+f"(b) : "f"(c), "f"(d));
}
__device__ __forceinline__ void mul2(float& a, float& b, float c, float d) {
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%0, %1};\n mov.b64 y, {%2, %3};\n mul.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}" : "+f"(a), "+f"(b) : "f"(c), "f"(d));
}
// (a, b) <- (a, b) * (c, d) + (e, f)
__device__ __forceinline__ void fma2(float& a, float& b, float c, float d, float e, float f) {
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%0, %1};\n mov.b64 y, {%2, %3};\n mov.b64 z, {%4, %5};\n fma.rn.f32x2 x, x, y, z;\n mov.b64 {%0, %1}, x;\n}"
      : "+f"(a), "+f"(b) : "f"(c), "f"(d), "f"(e), "f"(f));
}

// silu and the tanh form of gelu are both z sigmoid(w(z)): w = z and sqrt(8 / pi) (z + 0.044715 z^3).
constexpr float kGelu = 1.5957691216057308f, kGeluCube = 0.044715f, kLog2e = 1.4426950408889634f;
template <int ACT>
__device__ __forceinline__ void act_pair(float& a, float& b) {
  if constexpr (ACT == FRNN_ACT_RELU) {
    a = a < 0.0f ? 0.0f : a;  // a NaN stays one
    b = b < 0.0f ? 0.0f : b;
  }
  if constexpr (ACT == FRNN_ACT_SILU || ACT == FRNN_ACT_GELU_TANH) {
    float ea = a, eb = b;  // -log2(e) w
    if constexpr (ACT == FRNN_ACT_SILU) {
      mul2(ea, eb, -kLog2e, -kLog2e);
    } else {
      mul2(ea, eb, a, b);
      fma2(ea, eb, -kLog2e * kGelu * kGeluCube, -kLog2e * kGelu * kGeluCube, -kLog2e * kGelu, -kLog2e * kGelu);
      mul2(ea, eb, a, b);
    }
    ea = exp2_fast(ea);
    eb = exp2_fast(eb);
    add2(ea, eb, 1.0f, 1.0f);
    mul2(a, b, rcp_fast(ea), rcp_fast(eb));
  }
}
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == FRNN_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  if constexpr (ACT == FRNN_ACT_SILU) {
    const float s = sigmoid_p(z);
    return fmaf(z * s, 1.0f - s, s);
  }
  if constexpr (ACT == FRNN_ACT_GELU_TANH) {
    const float s = sigmoid_p(kGelu * z * fmaf(kGeluCube * z, z, 1.0f));
    return fmaf(z * s * (1.0f - s), kGelu * fmaf(3.0f * kGeluCube * z, z, 1.0f), s);
  }
  return 1.0f;
}

template <int ACT, int N>
__device__ __forceinline__ void act_row(float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) act_pair<ACT>(v[i], v[i + 1]);
}
// What the slope is taken at, eight columns as fp16. Of a relu the side of zero alone counts, which a small z could lose in 16 bits.
template <int ACT>
__device__ __forceinline__ void keep_slope(const float* v, uint32_t (&w)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = v[2 * i], b = v[2 * i + 1];
    if constexpr (ACT == FRNN_ACT_RELU) w[i] = (a > 0.0f ? 0x3c00u : 0u) | (b > 0.0f ? 0x3c000000u : 0u);
    else w[i] = pack_half2(a, b);
  }
}
__device__ __forceinline__ float load_bias(const ProductParams& p, int j) {
  return p.bias_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[j]) : __ldg(static_cast<const float*>(p.bias) + j);
}
// v[i] += bias[j + i], eight columns of a row of N (a multiple of eight)
__device__ __forceinline__ void add_bias(const ProductParams& p, int j, float* v) {
  if (j >= p.N) return;
  if (p.bias_bf16) {
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.bias) + j));
    add2(v[0], v[1], bf16_lo(w.x), bf16_hi(w.x));
    add2(v[2], v[3], bf16_lo(w.y), bf16_hi(w.y));
    add2(v[4], v[5], bf16_lo(w.z), bf16_hi(w.z));
    add2(v[6], v[7], bf16_lo(w.w), bf16_hi(w.w));
  } else {
    const float4 a = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p.bias) + j));
    const float4 b = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p.bias) + j + 4));
    add2(v[0], v[1], a.x, a.y);
    add2(v[2], v[3], a.z, a.w);
    add2(v[4], v[5], b.x, b.y);
    add2(v[6], v[7], b.z, b.w);
  }
}
__device__ __forceinline__ void add_bf16(const uint32_t (&w)[4], float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) add2(v[2 * i], v[2 * i + 1], bf16_lo(w[i]), bf16_hi(w[i]));
}

// A_MN / B_MN: the operand's rows in memory run along M / N instead of K.
template <bool A_MN, bool B_MN, int NP, int ACT>
__global__ void __launch_bounds__(kThreads, 1) __cluster_dims__(2, 1, 1)
product_kernel(const ProductParams p, const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map,
               const __grid_constant__ CUtensorMap out_map, const __grid_constant__ CUtensorMap res_map,
               const __grid_constant__ CUtensorMap z_map, const __grid_constant__ CUtensorMap work_map) {
  extern __shared__ uint8_t smem_raw[];
  constexpr int kStages = stages_of(NP, B_MN);
  __shared__ __align__(8) uint64_t s_full[kStages], s_empty[kStages], s_acc_full[2], s_acc_empty[2], s_done;
  __shared__ __align__(8) uint64_t s_res[kEpiWarps][2];
  __shared__ uint32_t s_tmem_base;
  constexpr int NH = NP / 2;  // rows of B in each CTA
  constexpr uint32_t kStageBytes = stage_bytes_of(NP, B_MN), kCols = NP > 128 ? 512u : 2u * NP;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = static_cast<int>(cluster_rank());  // 0: the one that issues
  const long long pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;  // the same offset in both CTAs
  const uint32_t staging = base + kStages * kStageBytes;
  const volatile int* abort_flag = p.err;

  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&s_full[s]), 1);
      mbar_init(smem_u32(&s_empty[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&s_acc_full[a]), 1);
      mbar_init(smem_u32(&s_acc_empty[a]), 2 * kEpiWarps);  // the epilogue warps of both CTAs, in the even one
    }
    for (int w = 0; w < kEpiWarps; ++w)
      for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&s_res[w][i]), 1);
    mbar_init(smem_u32(&s_done), 1);
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&a_map);
    tma_prefetch_desc(&b_map);
    tma_prefetch_desc(&out_map);
    if (p.has_residual) tma_prefetch_desc(&res_map);
    if (p.has_z) tma_prefetch_desc(&z_map);
  }
  int mute = 0;  // test hook, read while the CTAs meet: with err[4] set no MMA is issued, so the waits for the accumulators run out
  if (warp == kEpiWarps + 1) mute = p.err[4];
  if (warp == kEpiWarps + 1) tmem_alloc_pair(smem_u32(&s_tmem_base), kCols);
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after_sync();
  const uint32_t tbase = s_tmem_base;

  // rows, columns, part of K of a unit; row0: of a part, where its sums go
  struct Tile { int m0, n0, row0, c_begin, c_end; };
  auto tile_at = [&](long long t) {
    Tile r;
    r.row0 = -1;
    r.c_begin = 0;
    r.c_end = p.chunks;
    if (t >= p.whole) {
      const int u = static_cast<int>(t - p.whole), part = u % p.parts;
      r.row0 = u * 256;
      r.c_begin = part * p.chunks_per_part;
      r.c_end = min(r.c_begin + p.chunks_per_part, p.chunks);
      t = p.whole + u / p.parts;
    }
    r.n0 = static_cast<int>(t % p.n_nt) * NP;
    r.m0 = static_cast<int>(t / p.n_nt) * 256;
    return r;
  };

  if (warp == kEpiWarps) {
    if (lane == 0) {
      uint32_t s = 0, round = 0;
      bool dead = false;
      for (long long t = pair; t < p.n_units && !dead; t += pairs) {
        const Tile tile = tile_at(t);
        const int ma = tile.m0 + 128 * cta, nb = tile.n0 + NH * cta;
        for (int i = tile.c_begin; i < tile.c_end; ++i) {
          if (round > 0 && !mbar_wait_bounded<false, true>(smem_u32(&s_empty[s]), (round - 1) & 1, kLimit, abort_flag)) {
            atomicCAS(p.err, 0, kErrWaitEmpty);
            dead = true;
            break;
          }
          const uint32_t bar = map_to_cta(smem_u32(&s_full[s]), 0);
          const uint32_t sa = base + s * kStageBytes, sb = sa + 16384u;
          if (cta == 0) mbar_arrive_expect_tx(smem_u32(&s_full[s]), 2 * kStageBytes);  // what both CTAs stage
          const int k0 = i * kKC;
          if constexpr (A_MN) {
            tma_load_2d_pair(sa, &a_map, bar, ma, k0);
            tma_load_2d_pair(sa + 8192u, &a_map, bar, ma + 64, k0);
          } else {
            tma_load_2d_pair(sa, &a_map, bar, k0, ma);
          }
          if constexpr (B_MN) {
            for (int j = 0; j < (NH + 63) / 64; ++j) tma_load_2d_pair(sb + j * 8192u, &b_map, bar, nb + 64 * j, k0);
          } else {
            tma_load_2d_pair(sb, &b_map, bar, k0, nb);
          }
          if (++s == kStages) { s = 0; ++round; }
        }
      }
      // the last arrivals on this CTA's barriers are in before it leaves
      for (uint32_t left = round > 0 ? kStages : s; left > 0 && !dead; --left) {
        const uint32_t r = s > 0 ? round : round - 1;
        s = s > 0 ? s - 1 : kStages - 1;
        round = r;
        dead = !mbar_wait_bounded<false, true>(smem_u32(&s_empty[s]), r & 1, kLimit, abort_flag);
        if (dead) atomicCAS(p.err, 0, kErrWaitEmpty);
      }
      if (dead) settle();
    }
  } else if (warp == kEpiWarps + 1) {
    if (lane == 0 && cta == 0) {
      const uint32_t idesc = umma_idesc_bf16(256, NP, A_MN, B_MN);
      uint32_t s = 0, round = 0, li = 0;
      bool dead = false;
      for (long long t = pair; t < p.n_units && !dead && mute == 0; t += pairs, ++li) {
        const Tile tile = tile_at(t);
        const uint32_t a = li & 1u;
        if (li >= 2 && !mbar_wait_bounded<true, true>(smem_u32(&s_acc_empty[a]), ((li >> 1) - 1) & 1, kLimit, abort_flag)) {
          atomicCAS(p.err, 0, kErrWaitEpi);
          break;
        }
        tc_fence_after_sync();
        const uint32_t d = tbase + a * NP;
        for (int i = tile.c_begin; i < tile.c_end; ++i) {
          if (!mbar_wait_bounded<false, true>(smem_u32(&s_full[s]), round & 1, kLimit, abort_flag)) {
            atomicCAS(p.err, 0, kErrWaitWx);
            dead = true;
            break;
          }
          tc_fence_after_sync();
          const uint32_t sa = base + s * kStageBytes, sb = sa + 16384u;
          // 16 k's further: 32 bytes inside the swizzled row, or 16 rows of 128 bytes
          uint64_t ad = A_MN ? umma_smem_desc_mn_sw128(sa, 8192u) : umma_smem_desc_k_sw128(sa);
          uint64_t bd = B_MN ? umma_smem_desc_mn_sw128(sb, 8192u) : umma_smem_desc_k_sw128(sb);
#pragma unroll
          for (int kk = 0; kk < kKC / 16; ++kk) {
            umma_bf16_pair(d, ad, bd, idesc, (i > tile.c_begin || kk > 0) ? 1u : 0u);
            ad += A_MN ? 128 : 2;
            bd += B_MN ? 128 : 2;
          }
          umma_commit_pair(smem_u32(&s_empty[s]));
          if (++s == kStages) { s = 0; ++round; }
        }
        if (!dead) umma_commit_pair(smem_u32(&s_acc_full[a]));
      }
      // covers every MMA issued so far, also after a failed wait: tensor and shared memory stay until they are done
      umma_commit_pair_here(smem_u32(&s_done));
      mbar_wait_bounded<false, true>(smem_u32(&s_done), 0, kLimit, nullptr);
    }
  } else {
    const int q = warp & 3, first = warp >> 2;  // quarter of the tensor memory's lanes that this warp may read; its first piece
    constexpr int CW = 32;             // columns of a piece
    constexpr int kPieces = NP / CW;   // of the tile, in turn to the four warps of a quarter: one or two for each
    constexpr int kTurn = kEpiWarps / 4;
    const uint32_t buf0 = staging + static_cast<uint32_t>(warp) * 2u * kBufBytes;
    const uint32_t my_row = static_cast<uint32_t>(lane) * 64u, sw = static_cast<uint32_t>((lane >> 1) & 3);  // TMA's 64-byte swizzle
    // Without z the pieces take the two buffers in turn; with it z has the first and y the second. The residual's piece is loaded into
    // the buffer that y leaves from. What takes time here is latency, not arithmetic: hence four warps to a scheduler, and everything
    // that does not need the accumulator is asked for before it is waited for.
    const bool z_too = ACT != FRNN_ACT_NONE && p.has_z;
    uint32_t li = 0, used = 0, res_phase = 0;  // used: pieces staged so far; res_phase: a bit per buffer
    auto y_slot = [&](uint32_t n) { return z_too ? 1u : n & 1u; };
    auto ask_residual = [&](uint32_t slot, int j, int m) {
      const uint32_t bar = smem_u32(&s_res[warp][slot]);
      mbar_arrive_expect_tx(bar, kBufBytes);
      tma_load_2d(buf0 + slot * kBufBytes, &res_map, bar, j, m);
    };
    for (long long t = pair; t < p.n_units; t += pairs, ++li) {
      const Tile tile = tile_at(t);
      const uint32_t a = li & 1u;
      const int mw = tile.m0 + 128 * cta + 32 * q, j0 = tile.n0;
      const bool any = mw < p.M, part = tile.row0 >= 0;  // warp-uniform
      if (p.has_residual && any && !part && lane == 0) {   // while the tensor cores work: as many pieces as there are buffers
        tma_store_wait_read<0>();
        const int ahead = z_too ? 1 : 2;
        for (int n = 0; n < ahead; ++n) {
          const int piece = first + kTurn * n;
          if (piece < kPieces && j0 + piece * CW < p.N) ask_residual(y_slot(used + n), j0 + piece * CW, mw);
        }
      }
      float bias[(kPieces + kTurn - 1) / kTurn];  // of this lane's column of each piece
#pragma unroll
      for (int n = 0; n < (kPieces + kTurn - 1) / kTurn; ++n) {
        const int j = j0 + (first + kTurn * n) * CW + lane;
        bias[n] = p.bias != nullptr && !part && j < p.N ? load_bias(p, j) : 0.0f;
      }
      // parked, not polled: sixteen polling warps take issue slots and power from a long sum's tensor cores
      const bool have = __all_sync(0xffffffffu, mbar_wait_bounded<false, false>(smem_u32(&s_acc_full[a]), (li >> 1) & 1, kLimit, abort_flag));
      if (!have) {
        if (lane == 0) {
          atomicCAS(p.err, 0, kErrWaitMma);
          settle();  // a residual may be on its way
        }
        break;
      }
      tc_fence_after_sync();
      auto release = [&]() {  // the accumulator is in registers: the next unit but one may have it
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&s_acc_empty[a]), 0));
      };
      if (part) {
#pragma unroll 1
        for (int i = first; i < kPieces; i += kTurn) {  // 32 columns of fp32 take both buffers
          uint32_t v[32];
          tmem_ld_x32(tmem_addr(tbase, 32 * q, a * NP + i * CW), v);
          tmem_ld_wait();
          if (i + kTurn >= kPieces) release();
          const uint32_t buf = buf0 + static_cast<uint32_t>(lane) * 128u;
          if (lane == 0) tma_store_wait_read<0>();
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint32_t w[4] = {v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]};
            st_shared_v4(buf + ((k ^ (lane & 7)) << 4), w);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&work_map, buf, i * CW, tile.row0 + 128 * cta + 32 * q);
            tma_store_commit();
          }
        }
        continue;
      }
#pragma unroll
      for (int n = 0; n < (kPieces + kTurn - 1) / kTurn; ++n) {
        const int i = first + kTurn * n, j = j0 + i * CW;
        if (i >= kPieces) break;
        float v[CW];
        tmem_ld_x32(tmem_addr(tbase, 32 * q, a * NP + i * CW), *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
        tmem_ld_wait();
        if (i + kTurn >= kPieces) release();
        if (!any || j >= p.N) continue;
        const uint32_t slot = y_slot(used), y_at = buf0 + slot * kBufBytes, z_at = buf0;
        ++used;
        if (p.bias != nullptr) {
#pragma unroll
          for (int k = 0; k < CW; k += 2) add2(v[k], v[k + 1], __shfl_sync(0xffffffffu, bias[n], k), __shfl_sync(0xffffffffu, bias[n], k + 1));
        }
        if (lane == 0) {  // the stores that read these buffers; with a residual and no z: before it was asked for
          if (z_too) tma_store_wait_read<0>();
          else if (!p.has_residual) tma_store_wait_read<1>();
        }
        __syncwarp();
        if (z_too && p.has_residual && n > 0 && lane == 0) ask_residual(slot, j, mw);
        if (z_too) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t w[4];
            keep_slope<ACT>(&v[8 * k], w);
            st_shared_v4(z_at + my_row + ((k ^ sw) << 4), w);
          }
        }
        act_row<ACT>(v);
        if (p.has_residual) {
          if (!mbar_wait_warp<false>(smem_u32(&s_res[warp][slot]), (res_phase >> slot) & 1u, kLimit, abort_flag)) {
            if (lane == 0) {
              atomicCAS(p.err, 0, kErrWaitWx);
              settle();
            }
            __syncwarp();
          }
          res_phase ^= 1u << slot;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t w[4];
            ld_shared_v4(y_at + my_row + ((k ^ sw) << 4), w);
            add_bf16(w, &v[8 * k]);
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float* f = &v[8 * k];
          const uint32_t w[4] = {pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
          st_shared_v4(y_at + my_row + ((k ^ sw) << 4), w);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&out_map, y_at, j, mw);
          if (z_too) tma_store_2d(&z_map, z_at, j, mw);
          tma_store_commit();
        }
      }
    }
    if (lane == 0) tma_store_wait_read<0>();  // the staging buffers are read; the end of the kernel completes the writes
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // the other CTA's operands, barriers and tensor memory are in use until here
  if (warp == kEpiWarps + 1) tmem_dealloc_pair(tbase, kCols);
}

// out = epilogue(sum over the parts of a tile), eight columns of a row to a thread; work [tile][part][256][np].
template <int ACT>
__global__ void __launch_bounds__(256) product_join_kernel(const ProductParams p, const float* __restrict__ work, int np,
                                                           const __nv_bfloat16* __restrict__ residual, __nv_bfloat16* __restrict__ out,
                                                           uint4* __restrict__ z) {
  const int per_row = np / 8, blocks = per_row, tile = blockIdx.x / blocks, at = (blockIdx.x % blocks) * 256 + threadIdx.x;  // 256 rows
  const int row = at / per_row, col = at % per_row * 8;
  const long long t = p.whole + tile;
  const int m = static_cast<int>(t / p.n_nt) * 256 + row, j = static_cast<int>(t % p.n_nt) * np + col;
  if (m >= p.M || j >= p.N) return;
  const float* from = work + (static_cast<long long>(tile) * p.parts * 256 + row) * np + col;
  float v[8];
  ld_f32_vec<8>(from, v);
#pragma unroll 4
  for (int s = 1; s < p.parts; ++s) {
    float w[8];
    ld_f32_vec<8>(from + static_cast<long long>(s) * 256 * np, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += w[e];
  }
  if (p.bias != nullptr) add_bias(p, j, v);
  const long long i = static_cast<long long>(m) * p.N + j;
  if (z != nullptr) {
    uint32_t w[4];
    keep_slope<ACT>(v, w);
    z[i / 8] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  act_row<ACT>(v);
  if (residual != nullptr) {
    const uint4 r = __ldg(reinterpret_cast<const uint4*>(residual + i));
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
    add_bf16(w, v);
  }
  *reinterpret_cast<uint4*>(out + i) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

// Few rows: W goes from where it lies into the registers of mma.sync (16 outputs x 16 k's), the rows of x are the other operand,
// eight to an instruction, 32 to a CTA. The tensor pipe's rate does not matter here, the time to get W does: a warp has an eighth (a
// sixteenth) of K and its loads in flight together. 1 x 4096 x 4096 takes 10.3 us (3.3 TB/s; a library product 12.9). The order of k's inside a product is free as long as both operands have the same: a lane takes 16 bytes, eight
// neighbouring k's, which are two instructions' fragments.
template <int ACT, int NB, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) product_rows_kernel(const ProductParams p, const __nv_bfloat16* __restrict__ x,
                                                                     const __nv_bfloat16* __restrict__ w,
                                                                     const __nv_bfloat16* __restrict__ residual,
                                                                     __nv_bfloat16* __restrict__ out, __half* __restrict__ z) {
  __shared__ float s_sum[WARPS][NB * 8][17];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3, j0 = blockIdx.x * 16, m0 = blockIdx.y * NB * 8;
  float d[NB][4];
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) d[n][e] = 0.0f;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  const bool lo = j0 + g < p.N, hi = j0 + g + 8 < p.N;
  const __nv_bfloat16 *w0 = w + static_cast<size_t>(j0 + g) * p.K, *w1 = w0 + static_cast<size_t>(8) * p.K;
#pragma unroll 4
  for (int kb = warp * 32; kb < p.K; kb += WARPS * 32) {
    const int k = kb + q * 8;
    const bool in = k < p.K;
    const uint4 a = lo && in ? __ldg(reinterpret_cast<const uint4*>(w0 + k)) : zero, c = hi && in ? __ldg(reinterpret_cast<const uint4*>(w1 + k)) : zero;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int m = m0 + n * 8 + g;
      const uint4 b = in && m < p.M ? __ldg(reinterpret_cast<const uint4*>(x + static_cast<size_t>(m) * p.K + k)) : zero;
      const uint32_t a0[4] = {a.x, c.x, a.y, c.y}, a1[4] = {a.z, c.z, a.w, c.w};
      mma_bf16_16816(d[n], a0, b.x, b.y);
      mma_bf16_16816(d[n], a1, b.z, b.w);
    }
  }
#pragma unroll
  for (int n = 0; n < NB; ++n) {  // rows g, g + 8 of the outputs, columns 2 q, 2 q + 1 of x's rows
    s_sum[warp][n * 8 + 2 * q][g] = d[n][0];
    s_sum[warp][n * 8 + 2 * q + 1][g] = d[n][1];
    s_sum[warp][n * 8 + 2 * q][g + 8] = d[n][2];
    s_sum[warp][n * 8 + 2 * q + 1][g + 8] = d[n][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < NB * 8 * 8; i += WARPS * 32) {  // two neighbouring outputs of a row
    const int ml = i >> 3, m = m0 + ml, jl = (i & 7) * 2, j = j0 + jl;
    if (m >= p.M || j >= p.N) continue;
    float v[2] = {0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < WARPS; ++u) { v[0] += s_sum[u][ml][jl]; v[1] += s_sum[u][ml][jl + 1]; }
    if (p.bias != nullptr) {
      if (p.bias_bf16) {
        const uint32_t b = __ldg(reinterpret_cast<const unsigned*>(static_cast<const __nv_bfloat16*>(p.bias) + j));
        v[0] += bf16_lo(b); v[1] += bf16_hi(b);
      } else {
        v[0] += __ldg(static_cast<const float*>(p.bias) + j); v[1] += __ldg(static_cast<const float*>(p.bias) + j + 1);
      }
    }
    const size_t at = static_cast<size_t>(m) * p.N + j;
    if (z != nullptr)
      *reinterpret_cast<uint32_t*>(z + at) = ACT == FRNN_ACT_RELU ? (v[0] > 0.0f ? 0x3c00u : 0u) | (v[1] > 0.0f ? 0x3c000000u : 0u) : pack_half2(v[0], v[1]);
    act_pair<ACT>(v[0], v[1]);
    if (residual != nullptr) {
      const uint32_t r = __ldg(reinterpret_cast<const unsigned*>(residual + at));
      v[0] += bf16_lo(r); v[1] += bf16_hi(r);
    }
    *reinterpret_cast<uint32_t*>(out + at) = pack_bf16x2(v[0], v[1]);
  }
}

// dz = dy act'(z) (not stored where the activation is none: dz = dy), and the columns' sums of a block's rows for dbias.
constexpr int kSlopeRows = 64, kGridY = 65535;
template <int ACT>
__global__ void __launch_bounds__(256) product_slope_kernel(const __nv_bfloat16* __restrict__ dy, const __half* __restrict__ z,
                                                            __nv_bfloat16* __restrict__ dz, float* __restrict__ part, int M, int N) {
  constexpr int kBatch = 4;  // rows of a warp whose loads are in flight together
  __shared__ float s_sum[8][32][9];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long j0 = (static_cast<long long>(blockIdx.z) * kGridY + blockIdx.y) * 256, j = j0 + lane * 8;  // 256 columns to a block
  const long long m0 = static_cast<long long>(blockIdx.x) * kSlopeRows + warp;
  float sum[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[e] = 0.0f;
  if (j < N) {
#pragma unroll
    for (int r = 0; r < kSlopeRows / 8; r += kBatch) {
      uint4 g[kBatch], h[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const long long m = m0 + (r + i) * 8;
        g[i] = h[i] = make_uint4(0u, 0u, 0u, 0u);
        if (m < M) {
          g[i] = __ldg(reinterpret_cast<const uint4*>(dy + m * N + j));
          if constexpr (ACT != FRNN_ACT_NONE) h[i] = __ldg(reinterpret_cast<const uint4*>(z + m * N + j));
        }
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const long long m = m0 + (r + i) * 8;
        if (m >= M) break;
        float v[8] = {bf16_lo(g[i].x), bf16_hi(g[i].x), bf16_lo(g[i].y), bf16_hi(g[i].y), bf16_lo(g[i].z), bf16_hi(g[i].z), bf16_lo(g[i].w), bf16_hi(g[i].w)};
        if constexpr (ACT != FRNN_ACT_NONE) {
          const uint32_t w[4] = {h[i].x, h[i].y, h[i].z, h[i].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
            v[2 * e] *= act_slope<ACT>(f.x);
            v[2 * e + 1] *= act_slope<ACT>(f.y);
          }
          *reinterpret_cast<uint4*>(dz + m * N + j) =
              make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += v[e];
      }
    }
  }
  if (part == nullptr) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) s_sum[warp][lane][e] = sum[e];
  __syncthreads();
  const int l = threadIdx.x >> 3, e = threadIdx.x & 7;
  const long long col = j0 + threadIdx.x;
  if (col < N) {
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) v += s_sum[w][l][e];
    part[static_cast<long long>(blockIdx.x) * N + col] = v;
  }
}

// How an M x N x K product is cut: columns of a tile; tiles done whole, the rest in parts of K.
struct Cut { int np, parts, chunks_per_part; long long whole, rest; };
Cut choose_cut(long long M, long long N, long long K) {
  const long long pairs = sm_count() / 2 > 0 ? sm_count() / 2 : 1, mt = (M + 255) / 256, chunks = (K + kKC - 1) / kKC;
  Cut best{};
  double best_us = 0;
  for (int np = 256; np >= 128; np -= 64) {
    // Measured: 64 k's of a tile of 256, 192, 128 columns take 0.40, 0.39, 0.36 us (what a stage takes to arrive, not the tensor
    // cores, sets the narrow ones'), the pass over the parts' sums 2.5 us and their bytes, written and read, at 4 TB/s.
    const double chunk_us = np == 256 ? 0.40 : (np == 192 ? 0.39 : 0.36);
    const long long tiles = mt * ((N + np - 1) / np), whole = tiles / pairs * pairs, rest = tiles - whole;
    for (long long parts = 1; parts <= 16 && parts <= chunks; ++parts) {
      const long long cpp = (chunks + parts - 1) / parts;
      if ((chunks + cpp - 1) / cpp != parts) continue;
      double us = static_cast<double>(whole / pairs) * chunks * chunk_us + static_cast<double>((rest * parts + pairs - 1) / pairs) * cpp * chunk_us;
      if (parts > 1) us += 2.5 + static_cast<double>(rest) * parts * 256 * np * 8 / 4e6;
      if (best.np == 0 || us < best_us) {
        best = parts > 1 ? Cut{np, static_cast<int>(parts), static_cast<int>(cpp), whole, rest} : Cut{np, 1, static_cast<int>(chunks), tiles, 0};
        best_us = us;
      }
      if (rest == 0) break;
    }
  }
  return best;
}
long long work_bytes(long long M, long long N, long long K) {
  const Cut c = choose_cut(M, N, K);
  return 4 * c.rest * c.parts * 256 * c.np;
}

// Rows of `cols` values, boxes whose rows fill the span of the swizzle (64 or 128 bytes).
int map_2d(CUtensorMap* map, const void* base, int elem, long long cols, long long rows, uint32_t box_cols, uint32_t box_rows) {
  const uint64_t dims[2] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows)}, strides[1] = {static_cast<uint64_t>(cols) * elem};
  const uint32_t box[2] = {box_cols, box_rows};
  return make_tensor_map_strided(map, base, elem, 2, dims, strides, box, static_cast<int>(box_cols) * elem);
}

template <bool A_MN, bool B_MN, int NP, int ACT>
int launch_kernel(const ProductParams& p, const CUtensorMap (&maps)[6], cudaStream_t s) {
  const void* kern = reinterpret_cast<const void*>(product_kernel<A_MN, B_MN, NP, ACT>);
  cudaError_t e = raise_limits(kern, kSmem, false);
  if (e != cudaSuccess) return static_cast<int>(e);
  const long long pairs = sm_count() / 2;
  const unsigned grid = 2u * static_cast<unsigned>(p.n_units < pairs ? p.n_units : pairs);
  product_kernel<A_MN, B_MN, NP, ACT><<<grid, kThreads, kSmem, s>>>(p, maps[0], maps[1], maps[2], maps[3], maps[4], maps[5]);
  return static_cast<int>(cudaGetLastError());
}
// The gradients' products have no epilogue.
template <bool A_MN, bool B_MN, int NP>
int launch_act(const ProductParams& p, const CUtensorMap (&maps)[6], cudaStream_t s) {
  if constexpr (!A_MN && !B_MN) {
    if (p.act == FRNN_ACT_RELU) return launch_kernel<false, false, NP, FRNN_ACT_RELU>(p, maps, s);
    if (p.act == FRNN_ACT_SILU) return launch_kernel<false, false, NP, FRNN_ACT_SILU>(p, maps, s);
    if (p.act == FRNN_ACT_GELU_TANH) return launch_kernel<false, false, NP, FRNN_ACT_GELU_TANH>(p, maps, s);
  }
  return launch_kernel<A_MN, B_MN, NP, FRNN_ACT_NONE>(p, maps, s);
}

// C [M][N] = A . B with the epilogue of `p` (bias, act); A [M][K] or, A_MN, [K][M]; B [N][K] or, B_MN, [K][N].
template <bool A_MN, bool B_MN>
int product_launch(ProductParams p, const void* A, const void* B, long long M, long long N, long long K, const void* residual, void* out,
                   void* z, float* work, cudaStream_t s) {
  const Cut cut = choose_cut(M, N, K);
  p.M = static_cast<int>(M); p.N = static_cast<int>(N); p.K = static_cast<int>(K);
  p.n_nt = static_cast<int>((N + cut.np - 1) / cut.np);
  p.chunks = static_cast<int>((K + kKC - 1) / kKC);
  p.parts = cut.parts; p.chunks_per_part = cut.chunks_per_part;
  p.whole = cut.whole; p.n_units = cut.whole + cut.rest * cut.parts;
  p.has_residual = residual != nullptr; p.has_z = z != nullptr;
  if (cut.rest > 0 && work == nullptr) return -5;
  CUtensorMap maps[6];
  const uint32_t half = static_cast<uint32_t>(cut.np / 2);
  int rc = A_MN ? map_2d(&maps[0], A, 2, M, K, 64, kKC) : map_2d(&maps[0], A, 2, K, M, kKC, 128);
  if (rc == 0) rc = B_MN ? map_2d(&maps[1], B, 2, N, K, 64, kKC) : map_2d(&maps[1], B, 2, K, N, kKC, half);
  if (rc == 0) rc = map_2d(&maps[2], out, 2, N, M, 32, 32);
  if (rc == 0 && residual != nullptr) rc = map_2d(&maps[3], residual, 2, N, M, 32, 32);
  if (rc == 0 && z != nullptr) rc = map_2d(&maps[4], z, 2, N, M, 32, 32);
  if (rc == 0 && cut.rest > 0) rc = map_2d(&maps[5], work, 4, cut.np, cut.rest * cut.parts * 256, 32, 32);
  if (rc != 0) return rc;
  if (residual == nullptr) maps[3] = maps[2];
  if (z == nullptr) maps[4] = maps[2];
  if (cut.rest == 0) maps[5] = maps[2];
  rc = cut.np == 256   ? launch_act<A_MN, B_MN, 256>(p, maps, s)
       : cut.np == 192 ? launch_act<A_MN, B_MN, 192>(p, maps, s)
                       : launch_act<A_MN, B_MN, 128>(p, maps, s);
  if (rc != 0 || cut.rest == 0) return rc;
  const unsigned blocks = static_cast<unsigned>(cut.rest * (cut.np / 8));
  const auto* r = static_cast<const __nv_bfloat16*>(residual);
  auto* o = static_cast<__nv_bfloat16*>(out);
  auto* keep = static_cast<uint4*>(z);
  if (p.act == FRNN_ACT_RELU) product_join_kernel<FRNN_ACT_RELU><<<blocks, 256, 0, s>>>(p, work, cut.np, r, o, keep);
  else if (p.act == FRNN_ACT_SILU) product_join_kernel<FRNN_ACT_SILU><<<blocks, 256, 0, s>>>(p, work, cut.np, r, o, keep);
  else if (p.act == FRNN_ACT_GELU_TANH) product_join_kernel<FRNN_ACT_GELU_TANH><<<blocks, 256, 0, s>>>(p, work, cut.np, r, o, keep);
  else product_join_kernel<FRNN_ACT_NONE><<<blocks, 256, 0, s>>>(p, work, cut.np, r, o, keep);
  return static_cast<int>(cudaGetLastError());
}

// Which products the kernel of few rows takes. Every 32 rows read W again, so its time grows with all three sizes, while a tile's start and
// end alone are 6 us. us, against tiles and, in brackets, a library product without an epilogue: rows x inputs x outputs 8 x 768 x 1536
// 2.5, 9.3 (3.5), 16 x 4096 x 4096 13.8, 17.5 (10.1), 32 x 1024 x 4096 6.1, 11.0 (3.6), 256 x 768 x 768 6.2, 9.9 (3.5); behind
// the border 256 x 768 x 1536 10.7, 9.9, 32 x 4096 x 4096 23.6, 17.6.
bool few_rows(long long M, long long N, long long K) { return M <= 16 || (M <= 256 && M * N <= (1 << 28) / K); }

template <int ACT, int NB>
int rows_warps(const ProductParams& p, const void* x, const void* w, const void* residual, void* y, void* z, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>((p.N + 15) / 16), static_cast<unsigned>((p.M + NB * 8 - 1) / (NB * 8)));
  const auto *a = static_cast<const __nv_bfloat16*>(x), *b = static_cast<const __nv_bfloat16*>(w), *r = static_cast<const __nv_bfloat16*>(residual);
  auto* o = static_cast<__nv_bfloat16*>(y);
  auto* h = static_cast<__half*>(z);
  if (p.K <= 1024) product_rows_kernel<ACT, NB, 8><<<grid, 256, 0, s>>>(p, a, b, r, o, h);
  else product_rows_kernel<ACT, NB, 16><<<grid, 512, 0, s>>>(p, a, b, r, o, h);
  return static_cast<int>(cudaGetLastError());
}
template <int ACT>
int rows_act(const ProductParams& p, const void* x, const void* w, const void* residual, void* y, void* z, cudaStream_t s) {
  if (p.M <= 8) return rows_warps<ACT, 1>(p, x, w, residual, y, z, s);
  if (p.M <= 16) return rows_warps<ACT, 2>(p, x, w, residual, y, z, s);
  return rows_warps<ACT, 4>(p, x, w, residual, y, z, s);
}
int rows_launch(const ProductParams& p, const void* x, const void* w, const void* residual, void* y, void* z, cudaStream_t s) {
  if (p.act == FRNN_ACT_RELU) return rows_act<FRNN_ACT_RELU>(p, x, w, residual, y, z, s);
  if (p.act == FRNN_ACT_SILU) return rows_act<FRNN_ACT_SILU>(p, x, w, residual, y, z, s);
  if (p.act == FRNN_ACT_GELU_TANH) return rows_act<FRNN_ACT_GELU_TANH>(p, x, w, residual, y, z, s);
  return rows_act<FRNN_ACT_NONE>(p, x, w, residual, y, z, s);
}

bool bad_sizes(int64_t rows, int outputs, int inputs) { return rows < 1 || outputs < 1 || inputs < 1; }
bool unsupported(int64_t rows, int outputs, int inputs) {
  // coordinates and tile counts are 32-bit, and the k's of product_rows_kernel are counted past the end by up to 511; 16-byte rows
  return rows > 0x7fffff00LL || outputs > 0x7fffff00 || inputs > 0x7ffffe00 || outputs % 8 != 0 || inputs % 8 != 0 ||
         rows * outputs / 8 > 0x7fffffffLL * 256 || static_cast<long long>(inputs) * outputs / 8 > 0x7fffffffLL * 256;
}
bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }
bool bad_act(int a) { return a != FRNN_ACT_NONE && a != FRNN_ACT_RELU && a != FRNN_ACT_SILU && a != FRNN_ACT_GELU_TANH; }

}  // namespace

}  // namespace frnn

extern "C" int frnn_b200_product_plan(int64_t rows, int outputs, int inputs, frnn_b200_product_plan_t* out) {
  using namespace frnn;
  if (out == nullptr || bad_sizes(rows, outputs, inputs)) return -5;
  if (unsupported(rows, outputs, inputs)) return -2;
  *out = {};
  out->forward_waits = !few_rows(rows, outputs, inputs);
  if (out->forward_waits) out->forward_work_bytes = work_bytes(rows, outputs, inputs);
  const long long dx = work_bytes(rows, inputs, outputs), dw = work_bytes(outputs, inputs, rows);
  out->backward_work_bytes = dx > dw ? dx : dw;
  out->dbpart_bytes = 4 * ((rows + kSlopeRows - 1) / kSlopeRows) * outputs;
  return 0;
}

extern "C" int frnn_b200_product_forward(const void* x, const void* w, const void* bias, int bias_bf16, const void* residual, int activation,
                                         void* y, void* z, int64_t rows, int outputs, int inputs, float* work, int* err, void* stream) {
  using namespace frnn;
  if (!x || !w || !y || bad_sizes(rows, outputs, inputs) || bad_act(activation) ) return -5;
  if (misaligned(x) || misaligned(w) || misaligned(y) || misaligned(bias) || misaligned(residual) || misaligned(z) || misaligned(work)) return -5;
  if (unsupported(rows, outputs, inputs)) return -2;
  if (!err && !few_rows(rows, outputs, inputs)) return -5;
  ProductParams p{};
  p.bias = bias; p.bias_bf16 = bias_bf16; p.act = activation; p.err = err;
  if (few_rows(rows, outputs, inputs)) {
    p.M = static_cast<int>(rows); p.N = outputs; p.K = inputs;
    return rows_launch(p, x, w, residual, y, z, static_cast<cudaStream_t>(stream));
  }
  return product_launch<false, false>(p, x, w, rows, outputs, inputs, residual, y, z, work, static_cast<cudaStream_t>(stream));
}

extern "C" int frnn_b200_product_backward(const void* dy, const void* z, const void* x, const void* w, int activation, void* dz, void* dx,
                                          void* dw, void* dbias, int dbias_bf16, float* db_part, int64_t rows, int outputs, int inputs,
                                          float* work, int* err, void* stream) {
  using namespace frnn;
  const bool slopes = activation != FRNN_ACT_NONE;
  if (!dy || !err || bad_sizes(rows, outputs, inputs) || bad_act(activation)) return -5;
  if ((slopes && (!z || !dz)) || (dx && !w) || (dw && !x) || (dbias && !db_part)) return -5;
  if (misaligned(dy) || misaligned(z) || misaligned(x) || misaligned(w) || misaligned(dz) || misaligned(dx) || misaligned(dw) ||
      misaligned(work))
    return -5;
  if (unsupported(rows, outputs, inputs)) return -2;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (slopes || dbias != nullptr) {
    const int blocks = static_cast<int>((rows + kSlopeRows - 1) / kSlopeRows), cols = (outputs / 8 + 31) / 32;
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(cols < kGridY ? cols : kGridY), static_cast<unsigned>((cols + kGridY - 1) / kGridY));
    const auto* g = static_cast<const __nv_bfloat16*>(dy);
    const auto* h = static_cast<const __half*>(z);
    auto* d = static_cast<__nv_bfloat16*>(dz);
    float* part = dbias != nullptr ? db_part : nullptr;
    const int M = static_cast<int>(rows);
    if (activation == FRNN_ACT_RELU) product_slope_kernel<FRNN_ACT_RELU><<<grid, 256, 0, s>>>(g, h, d, part, M, outputs);
    else if (activation == FRNN_ACT_SILU) product_slope_kernel<FRNN_ACT_SILU><<<grid, 256, 0, s>>>(g, h, d, part, M, outputs);
    else if (activation == FRNN_ACT_GELU_TANH) product_slope_kernel<FRNN_ACT_GELU_TANH><<<grid, 256, 0, s>>>(g, h, d, part, M, outputs);
    else product_slope_kernel<FRNN_ACT_NONE><<<grid, 256, 0, s>>>(g, h, d, part, M, outputs);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess && dbias != nullptr) {
      e = dbias_bf16 ? column_sum(db_part, static_cast<__nv_bfloat16*>(dbias), blocks, outputs, s)
                     : column_sum(db_part, static_cast<float*>(dbias), blocks, outputs, s);
    }
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  ProductParams p{};
  p.err = err;
  const void* g = slopes ? dz : dy;
  int rc = 0;
  if (dx != nullptr) rc = product_launch<false, true>(p, g, w, rows, inputs, outputs, nullptr, dx, nullptr, work, s);
  if (rc == 0 && dw != nullptr) rc = product_launch<true, true>(p, g, x, outputs, inputs, rows, nullptr, dw, nullptr, work, s);
  return rc;
}
