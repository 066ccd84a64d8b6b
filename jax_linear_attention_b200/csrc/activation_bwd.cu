// Gradients through the activations of the projections and of the gated feed-forward block (jla_activation_bwd,
// jla_gated_activation_bwd): what the gradient products then read.
//
//   linear:  dz = dy act'(z), dbias = sum over rows of dz         gated:  dg = dh u act'(g),  du = dh act(g)
//
// Bound by HBM: z (or g and u) is read in float32, dy and the results are 16-bit. The forward pass keeps z in float32, not
// in 16 bits, because its rounding would come on top of the one of dz, which the tensor cores cannot do without; a 16-bit
// z makes dx half as far again from the exact gradient for 2 bytes an element fewer. What the rounding of dz, dg and du costs: dx and
// dW are 2.9e-4 instead of 2.1e-4 off in f16 (4096 x 2048 x 2048 with sigmoid), 2.3e-3 instead of 1.7e-3 in bf16 (gated 16384 x
// 2048 x 5632), as torch's own gradients of these types are; two 16-bit halves of each would keep it at twice the products.
//
// Measured on a B200: gated 16384 x 5632 bf16 188 us (6.7 TB/s); 4096 x 2048 f16 with dbias 12 + 3 us.
//
// A thread owns eight adjacent columns and walks rows, so that dbias is summed in registers, over the block's eight row
// lanes in shared memory, and over the blocks by column_sums(): the same order every time.
#include "column_sums.cuh"
#include "overlap.cuh"
#include "product.cuh"
#include "profile.cuh"

namespace jla {
namespace {

constexpr int kColLanes = 32, kRowLanes = 8;

struct ActParams {
  long rows;
  int cols, act;
  const float *z, *u;
  const void* dy;
  void *dz, *du;
  float* partial;  // [gridDim.y][cols]
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
  const uint4 q = *(reinterpret_cast<const uint4*>(p));
  const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = to_f32(e[i]);
}
__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
  const float4 a = *(reinterpret_cast<const float4*>(p)), b = *(reinterpret_cast<const float4*>(p) + 1);
  f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  uint4 q;
  T* e = reinterpret_cast<T*>(&q);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(f[i]);
  *reinterpret_cast<uint4*>(p) = q;
}

template <typename T, bool GATED>
__global__ void __launch_bounds__(kColLanes * kRowLanes) activation_bwd_kernel(ActParams p) {
  const int ct = threadIdx.x % kColLanes, lr = threadIdx.x / kColLanes;
  const int col = (blockIdx.x * kColLanes + ct) * 8;
  const bool on = col < p.cols;
  float sum[8] = {};
  start_next();
  wait_for_previous();
  for (long r = (long)blockIdx.y * kRowLanes + lr; r < p.rows; r += (long)gridDim.y * kRowLanes) {
    if (!on) break;
    const size_t at = (size_t)r * p.cols + col;
    float dy[8], z[8];
    load8(static_cast<const T*>(p.dy) + at, dy);
    if constexpr (GATED) {
      float u[8], du[8];
      load8(p.z + at, z);
      load8(p.u + at, u);
      with_activation(p.act, [&](auto act) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          du[i] = dy[i] * activate<act()>(z[i]);
          dy[i] *= u[i] * activation_slope<act()>(z[i]);
        }
      });
      store8(static_cast<T*>(p.du) + at, du);
      store8(static_cast<T*>(p.dz) + at, dy);
    } else {
      if (p.z) {
        load8(p.z + at, z);
        with_activation(p.act, [&](auto act) {
#pragma unroll
          for (int i = 0; i < 8; ++i) dy[i] *= activation_slope<act()>(z[i]);
        });
        store8(static_cast<T*>(p.dz) + at, dy);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] += dy[i];
    }
  }
  if constexpr (!GATED) {
    if (!p.partial) return;
    __shared__ float fold[kRowLanes][kColLanes * 8];
#pragma unroll
    for (int i = 0; i < 8; ++i) fold[lr][ct * 8 + i] = sum[i];
    __syncthreads();
    const int c = blockIdx.x * kColLanes * 8 + threadIdx.x;  // 256 columns, 256 threads
    if (c < p.cols) {
      float t = 0.f;
#pragma unroll
      for (int l = 0; l < kRowLanes; ++l) t += fold[l][threadIdx.x];
      p.partial[(size_t)blockIdx.y * p.cols + c] = t;
    }
  }
}

dim3 grid_of(long rows, int cols) {
  const int x = (cols + kColLanes * 8 - 1) / (kColLanes * 8);
  const long groups = (rows + kRowLanes - 1) / kRowLanes;
  long y = 8 * 148 / x;  // eight blocks of 256 threads an SM
  y = y < 1 ? 1 : (y > kMaxParts ? kMaxParts : y);
  return dim3(x, (unsigned)(groups < y ? groups : y));
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

const char* problem(int dtype, long rows, int cols, int act) {
  if (dtype != JLA_DTYPE_BF16 && dtype != JLA_DTYPE_F16) return "activation gradient: bf16 and f16 only";
  if (rows < 0 || rows > (1L << 31) - 1 || cols < 8 || cols % 8) return "activation gradient: columns must be a multiple of 8";
  if (act < JLA_ACT_NONE || act > JLA_ACT_SIGMOID) return "unknown activation";
  return nullptr;
}

}  // namespace
}  // namespace jla

using namespace jla;

extern "C" {

size_t jla_activation_bwd_scratch_bytes(int64_t rows, int out) {
  if (rows <= 0 || out < 8) return 0;
  return (size_t)grid_of(rows, out).y * out * sizeof(float);
}

int jla_activation_bwd(int dtype, int64_t rows, int out, int act, const float* z, const void* dy, void* dz, float* dbias,
                       void* scratch, size_t scratch_bytes, jla_stream_t stream) {
  if (const char* why = problem(dtype, rows, out, act)) {
    set_error("%s", why);
    return JLA_ERR_BAD_ARGUMENT;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    if (dbias) JLA_CUDA_OK(cudaMemsetAsync(dbias, 0, sizeof(float) * out, s));
    return JLA_OK;
  }
  if (!dy || (z && !dz) || (!z && !dbias) || (!z && act != JLA_ACT_NONE) || !aligned16(dy) || !aligned16(z) || !aligned16(dz)) {
    set_error("activation gradient: null or unaligned pointer");
    return JLA_ERR_BAD_ARGUMENT;
  }
  if (dbias && (!scratch || scratch_bytes < jla_activation_bwd_scratch_bytes(rows, out))) {
    set_error("activation gradient: %zu bytes of scratch, %zu needed", scratch_bytes, jla_activation_bwd_scratch_bytes(rows, out));
    return JLA_ERR_WORKSPACE;
  }
  ActParams p{};
  p.rows = rows, p.cols = out, p.act = act, p.z = z, p.dy = dy, p.dz = dz;
  p.partial = dbias ? static_cast<float*>(scratch) : nullptr;
  const dim3 grid = grid_of(rows, out);
  {
    ProfScope scope(kProfActBwd, s);
    auto* kern = dtype == JLA_DTYPE_BF16 ? activation_bwd_kernel<__nv_bfloat16, false> : activation_bwd_kernel<__half, false>;
    JLA_CUDA_OK(launch_overlapped(kern, grid, dim3(kColLanes * kRowLanes), 0, s, 0, p));
  }
  return dbias ? column_sums(p.partial, grid.y, out, dbias, s) : JLA_OK;
}

int jla_gated_activation_bwd(int dtype, int64_t rows, int out, int act, const float* g, const float* u, const void* dh,
                             void* dg, void* du, jla_stream_t stream) {
  if (const char* why = problem(dtype, rows, out, act)) {
    set_error("%s", why);
    return JLA_ERR_BAD_ARGUMENT;
  }
  if (rows == 0) return JLA_OK;
  if (!g || !u || !dh || !dg || !du || !aligned16(g) || !aligned16(u) || !aligned16(dh) || !aligned16(dg) || !aligned16(du)) {
    set_error("activation gradient: null or unaligned pointer");
    return JLA_ERR_BAD_ARGUMENT;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ActParams p{};
  p.rows = rows, p.cols = out, p.act = act, p.z = g, p.u = u, p.dy = dh, p.dz = dg, p.du = du;
  const dim3 grid = grid_of(rows, out);
  {
    ProfScope scope(kProfActBwd, s);
    auto* kern = dtype == JLA_DTYPE_BF16 ? activation_bwd_kernel<__nv_bfloat16, true> : activation_bwd_kernel<__half, true>;
    JLA_CUDA_OK(launch_overlapped(kern, grid, dim3(kColLanes * kRowLanes), 0, s, 0, p));
  }
  return JLA_OK;
}

}  // extern "C"
