#include "column_sums.cuh"

#include "overlap.cuh"

namespace jla {
namespace {

// A block adds up 32 columns: lane = column (128 contiguous bytes of a partial row), warp w takes the rows w, w + 32, ...
// and the 32 warps' sums are joined by a tree over shared memory.
__global__ void __launch_bounds__(1024) column_sums_kernel(const float* partial, int parts, int cols, float* out) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float sum = 0.f;
  start_next();
  wait_for_previous();
  if (c < cols) {
    for (int p = warp; p < parts; p += 32) sum += partial[(size_t)p * cols + c];
  }
  red[warp][lane] = sum;
  __syncthreads();
  float t = red[lane][warp];  // column `warp` of the block, part `lane`
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) t += __shfl_xor_sync(0xffffffffu, t, off);
  const int mine = blockIdx.x * 32 + warp;
  if (lane == 0 && mine < cols) out[mine] = t;
}

}  // namespace

int column_sums(const float* partial, int parts, int cols, float* out, cudaStream_t stream) {
  if (cols <= 0) return JLA_OK;
  JLA_CUDA_OK(launch_overlapped(column_sums_kernel, dim3((cols + 31) / 32), dim3(1024), 0, stream, 0, partial, parts, cols, out));
  return JLA_OK;
}

}  // namespace jla
