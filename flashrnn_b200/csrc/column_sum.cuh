// Sums over the rows of a matrix of partial sums: what the backward passes' CTAs leave of a bias's gradient.
#pragma once

#include "frnn_common.cuh"

namespace frnn {

constexpr int kColumnSplits = 8;
// out[j] = sum over rows of part[row][j], in a fixed order: 32 columns to a CTA, its 32 warps take rows in turn, the CTAs of a cluster
// (gridDim.y of them) each a part of the rows.
template <typename Out>
__global__ void __launch_bounds__(1024) column_sum_kernel(const float* __restrict__ part, Out* __restrict__ out, long long rows, int cols) {
  __shared__ float s[32][33], s_part[kColumnSplits][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = blockIdx.x * 32 + lane;
  if (gridDim.y > 1) cluster_arrive();  // another CTA's shared memory may be written once that CTA has started
  const long long per = (rows + gridDim.y - 1) / gridDim.y, first = per * blockIdx.y, end = first + per < rows ? first + per : rows;
  float sum = 0.0f;
  if (j < cols) {
#pragma unroll 8
    for (long long r = first + warp; r < end; r += 32) sum += __ldg(part + r * cols + j);
  }
  s[warp][lane] = sum;
  __syncthreads();
  float v = s[lane][warp];  // column `warp` of this CTA
#pragma unroll
  for (int o = 16; o > 0; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (gridDim.y > 1) {  // all of it at the cluster's first CTA
    cluster_wait();
    if (lane == 0)
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(map_to_cta(smem_u32(&s_part[blockIdx.y][warp]), 0)), "f"(v) : "memory");
    cluster_sync_all();
    if (blockIdx.y != 0) return;
    v = 0.0f;
    for (unsigned i = 0; i < gridDim.y; ++i) v += s_part[i][warp];
  }
  const int col = blockIdx.x * 32 + warp;
  if (lane != 0 || col >= cols) return;
  if constexpr (sizeof(Out) == 2) out[col] = __float2bfloat16_rn(v);
  else out[col] = v;
}

// Waits for loads until there are CTAs enough to fill the memory's pipe. us, one CTA for 32 columns against eight: 1024 rows x 32 columns 3.2,
// 3.2; 2048 x 32 4.0, 2.8; 2048 x 1024 4.3, 3.7; 2048 x 2048 (512 CTAs of 1024 threads, two rounds of them) 4.4, 6.6; 16384 x 256 18.0, 5.2;
// 65536 x 32 58.5, 11.4.
template <typename Out>
cudaError_t column_sum(const float* part, Out* out, long long rows, int cols, cudaStream_t s) {
  const unsigned blocks = static_cast<unsigned>((cols + 31) / 32);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(blocks, rows >= 2048 && blocks <= 32 ? kColumnSplits : 1);
  cfg.blockDim = dim3(1024);
  cfg.stream = s;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = cfg.gridDim.y;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cfg.gridDim.y > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, column_sum_kernel<Out>, part, out, rows, cols);
}

}  // namespace frnn
