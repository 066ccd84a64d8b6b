// RMS norm of the residual stream in front of a mixer or a feed-forward block, with the residual's addition and, for
// 8-bit projections, its output in e4m3 with one scale a row; forward and backward in one pass over the rows each.
//
//   t = x + residual                      x, residual, y, stream [rows, dim] dtype; weight [dim] f32
//   stream = round(t)
//   rstd = rsqrt(mean(t^2) + eps),  y = t * rstd * weight
//   e4m3: scale = max |y| / 448 a row (1 where that is no positive normal number), q = e4m3(y / scale)
//
//   backward, with n = t * rstd:
//   dx = dstream + rstd (dy weight - n mean(dy weight n)),  dweight = sum over rows of dy n
//
// Bound by HBM. The row lies in registers between its two uses (the norm, then the values), so every tensor is read and
// written once. A row belongs to a group of threads, a power of two, each with VPT vectors of VEC adjacent channels: 8
// channels in 16-byte loads where the width and the addresses allow it, else single channels (neighbouring threads still
// read neighbouring channels). Sums are held in float32. The norm is taken of the unrounded t, and the backward pass adds x
// and the residual up again: the rounded stream, half the bytes to read, would leave the float32 weight gradient with an
// error of 2e-3 instead of 2e-7.
//
// The weight gradient is summed in registers over the rows that a thread walks, over the block in shared memory, and
// over the blocks by column_sums(), always in the same order.
#include <cuda_fp8.h>

#include "column_sums.cuh"
#include "profile.cuh"

namespace jla {
namespace {

constexpr int kMaxDim = 16384;
constexpr float kE4m3Max = 448.f;

struct RmsParams {
  long rows;
  int dim;
  const void *x, *residual;
  const float* w;
  float eps;
  void *y, *stream;
  float *rstd, *scale;
  // backward
  const void *dy, *dstream;
  void* dx;
  float* partial;  // [gridDim.x][dim], or NULL where no weight gradient is wanted
};

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    f[0] = to_f32(*p);
  } else if constexpr (sizeof(T) == 2) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = to_f32(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const float4 u = *reinterpret_cast<const float4*>(p + i);
      f[i] = u.x, f[i + 1] = u.y, f[i + 2] = u.z, f[i + 3] = u.w;
    }
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    *p = from_f32<T>(f[0]);
  } else if constexpr (sizeof(T) == 2) {
    uint4 u;
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < VEC; ++i) e[i] = from_f32<T>(f[i]);
    *reinterpret_cast<uint4*>(p) = u;
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
  }
}

__device__ __forceinline__ float max_nan(float a, float b) {  // a NaN wins: the scale of a row that holds one is NaN
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Sum (or maximum) over the blockDim.x threads of a row. Up to 32 threads: a butterfly inside the warp. More: a warp's
// value through `red` ([blockDim.y][blockDim.x / 32], 32 floats at most), every thread of the block has to call it.
// `red` may be used again after another __syncthreads of the block.
template <bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* red) {
  const int tpr = blockDim.x, lanes = tpr < 32 ? tpr : 32;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const float o = __shfl_xor_sync(0xffffffffu, v, off);
    if (off < lanes) v = MAX ? max_nan(v, o) : v + o;
  }
  if (tpr <= 32) return v;
  const int wpr = tpr >> 5;
  float* mine = red + threadIdx.y * wpr;
  if ((threadIdx.x & 31) == 0) mine[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = mine[0];
  for (int w = 1; w < wpr; ++w) t = MAX ? max_nan(t, mine[w]) : t + mine[w];
  return t;
}

template <typename T, int VEC, int VPT, bool E4M3>
__global__ void __launch_bounds__(1024) rms_norm_fwd_kernel(RmsParams p) {
  __shared__ float red[2][32];
  const long row = (long)blockIdx.x * blockDim.y + threadIdx.y;
  const bool live = row < p.rows;
  const size_t base = (size_t)(live ? row : 0) * p.dim;
  const int tpr = blockDim.x;
  const T* x = static_cast<const T*>(p.x);
  const T* res = static_cast<const T*>(p.residual);
  float f[VPT][VEC];
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int c = (j * tpr + threadIdx.x) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[j][i] = 0.f;
    if (live && c < p.dim) load_vec<T, VEC>(x + base + c, f[j]);
  }
  if (res) {
    T* stream = static_cast<T*>(p.stream);
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int c = (j * tpr + threadIdx.x) * VEC;
      if (live && c < p.dim) {
        float r[VEC];
        load_vec<T, VEC>(res + base + c, r);
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[j][i] += r[i];
        store_vec<T, VEC>(stream + base + c, f[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) ss += f[j][i] * f[j][i];
  }
  const float rstd = rsqrtf(row_reduce<false>(ss, red[0]) / (float)p.dim + p.eps);
  if (p.rstd && live && threadIdx.x == 0) p.rstd[row] = rstd;
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int c = (j * tpr + threadIdx.x) * VEC;
    if (c < p.dim) {
      float w[VEC];
      load_vec<float, VEC>(p.w + c, w);
#pragma unroll
      for (int i = 0; i < VEC; ++i) f[j][i] = f[j][i] * rstd * w[i];
      if constexpr (E4M3) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) top = max_nan(top, fabsf(f[j][i]));
      } else if (live) {
        store_vec<T, VEC>(static_cast<T*>(p.y) + base + c, f[j]);
      }
    }
  }
  if constexpr (E4M3) {
    float scale = row_reduce<true>(top, red[1]) / kE4m3Max;
    if (scale < 1.17549435e-38f) scale = 1.f;  // a row of zeros (or of subnormal numbers, which e4m3 then holds as zeros)
    if (live && threadIdx.x == 0) p.scale[row] = scale;
    unsigned char* q = static_cast<unsigned char*>(p.y);
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int c = (j * tpr + threadIdx.x) * VEC;
      if (live && c < p.dim) {
        if constexpr (VEC == 8) {
          __nv_fp8x2_storage_t e[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            e[i] = __nv_cvt_float2_to_fp8x2(make_float2(f[j][2 * i] / scale, f[j][2 * i + 1] / scale), __NV_SATFINITE,
                                            __NV_E4M3);
          }
          *reinterpret_cast<uint2*>(q + base + c) =
              make_uint2((uint32_t)e[0] | ((uint32_t)e[1] << 16), (uint32_t)e[2] | ((uint32_t)e[3] << 16));
        } else {
          q[base + c] = __nv_cvt_float_to_fp8(f[j][0] / scale, __NV_SATFINITE, __NV_E4M3);
        }
      }
    }
  }
}

// Blocks walk the rows blockIdx.x * blockDim.y + threadIdx.y, + gridDim.x * blockDim.y, ... (the same number of steps for
// all threads of a block: row_reduce may synchronise it).
template <typename T, int VEC, int VPT, int MAXT>
__global__ void __launch_bounds__(MAXT) rms_norm_bwd_kernel(RmsParams p) {
  __shared__ float red[2][32];
  extern __shared__ float fold[];  // [blockDim.y][dim] of the weight gradient, where a block has several rows
  const int tpr = blockDim.x;
  const T* x = static_cast<const T*>(p.x);
  const T* res = static_cast<const T*>(p.residual);
  const T* dy = static_cast<const T*>(p.dy);
  const T* ds = static_cast<const T*>(p.dstream);
  const float inv_dim = 1.f / (float)p.dim;
  float dw[VPT][VEC];
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[j][i] = 0.f;
  }
  int turn = 0;
  for (long r0 = (long)blockIdx.x * blockDim.y; r0 < p.rows; r0 += (long)gridDim.x * blockDim.y, turn ^= 1) {
    const long row = r0 + threadIdx.y;
    const bool live = row < p.rows;
    const size_t base = (size_t)(live ? row : 0) * p.dim;
    float n[VPT][VEC], d[VPT][VEC], s[VPT][VEC];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int c = (j * tpr + threadIdx.x) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) n[j][i] = d[j][i] = s[j][i] = 0.f;
      if (live && c < p.dim) {
        load_vec<T, VEC>(x + base + c, n[j]);
        load_vec<T, VEC>(dy + base + c, d[j]);
        if (ds) load_vec<T, VEC>(ds + base + c, s[j]);
        if (res) {
          float r[VEC];
          load_vec<T, VEC>(res + base + c, r);
#pragma unroll
          for (int i = 0; i < VEC; ++i) n[j][i] += r[i];
        }
      }
    }
    const float rstd = live ? p.rstd[row] : 0.f;
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int c = (j * tpr + threadIdx.x) * VEC;
      if (c < p.dim) {
        float w[VEC];
        load_vec<float, VEC>(p.w + c, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          n[j][i] *= rstd;
          dw[j][i] += d[j][i] * n[j][i];
          d[j][i] *= w[i];
          dot += d[j][i] * n[j][i];
        }
      }
    }
    const float mean = row_reduce<false>(dot, red[turn]) * inv_dim;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int c = (j * tpr + threadIdx.x) * VEC;
      if (live && c < p.dim) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) s[j][i] += rstd * (d[j][i] - n[j][i] * mean);
        store_vec<T, VEC>(static_cast<T*>(p.dx) + base + c, s[j]);
      }
    }
  }
  if (!p.partial) return;
  float* out = p.partial + (size_t)blockIdx.x * p.dim;
  if (blockDim.y > 1) {
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int c = (j * tpr + threadIdx.x) * VEC;
      if (c < p.dim) store_vec<float, VEC>(fold + (size_t)threadIdx.y * p.dim + c, dw[j]);
    }
    __syncthreads();
    for (int c = threadIdx.y * tpr + threadIdx.x; c < p.dim; c += tpr * blockDim.y) {
      float t = 0.f;
      for (int y = 0; y < (int)blockDim.y; ++y) t += fold[(size_t)y * p.dim + c];
      out[c] = t;
    }
  } else {
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int c = (j * tpr + threadIdx.x) * VEC;
      if (c < p.dim) store_vec<float, VEC>(out + c, dw[j]);
    }
  }
}

int ceil_pow2(int x) {
  int p = 1;
  while (p < x) p *= 2;
  return p;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

const char* problem(int dtype, long rows, int dim) {
  if (dtype < JLA_DTYPE_BF16 || dtype > JLA_DTYPE_F32) return "rms norm: unknown dtype";
  if (rows < 0) return "rms norm: negative number of rows";
  if (dim < 1 || dim > kMaxDim) return "rms norm: the width must be 1 .. 16384";
  if (rows > (1L << 31) - 1) return "rms norm: more than 2^31 - 1 rows";
  return nullptr;
}

template <typename T, bool E4M3>
void launch_fwd(const RmsParams& p, bool vec, cudaStream_t s) {
  // Threads of a row, and vectors of a thread. Few rows: one vector a thread, so that a row's loads all leave at once
  // (a decoding step is latency). Many rows: four vectors, fewer threads meet in the reduction and more rows are in flight.
  const int vectors = vec ? p.dim / 8 : p.dim;
  int vpt = vec ? (vectors <= 1024 && p.rows <= 148 ? 1 : 4) : (vectors <= 4096 ? 4 : 16);
  int tpr = ceil_pow2((vectors + vpt - 1) / vpt);
  if (tpr < 8) tpr = 8;
  const int rpb = tpr >= 256 ? 1 : 256 / tpr;
  const dim3 block(tpr, rpb), grid((unsigned)((p.rows + rpb - 1) / rpb));
  if (vec) {
    if (vpt == 1) rms_norm_fwd_kernel<T, 8, 1, E4M3><<<grid, block, 0, s>>>(p);
    else rms_norm_fwd_kernel<T, 8, 4, E4M3><<<grid, block, 0, s>>>(p);
  } else {
    if (vpt == 4) rms_norm_fwd_kernel<T, 1, 4, E4M3><<<grid, block, 0, s>>>(p);
    else rms_norm_fwd_kernel<T, 1, 16, E4M3><<<grid, block, 0, s>>>(p);
  }
}

struct BwdShape {
  int tpr, rpb, vpt, blocks;
};
BwdShape bwd_shape(long rows, int dim, bool vec) {
  BwdShape b;
  const int vectors = vec ? dim / 8 : dim;
  b.vpt = vec ? 2 : (vectors <= 4096 ? 4 : 16);
  b.tpr = ceil_pow2((vectors + b.vpt - 1) / b.vpt);
  if (b.tpr < 8) b.tpr = 8;
  b.rpb = b.tpr >= 256 ? 1 : 256 / b.tpr;
  const long groups = (rows + b.rpb - 1) / b.rpb;
  const long most = b.tpr > 512 ? 148 : (b.tpr > 256 ? 296 : kMaxParts);
  b.blocks = (int)(groups < most ? groups : most);
  return b;
}

template <typename T>
cudaError_t launch_bwd(const RmsParams& p, const BwdShape& b, bool vec, cudaStream_t s) {
  const dim3 block(b.tpr, b.rpb);
  const size_t smem = b.rpb > 1 && p.partial ? (size_t)b.rpb * p.dim * sizeof(float) : 0;  // at most 16 KB
  const bool wide = b.tpr > 256;
  if (vec) {
    if (wide) rms_norm_bwd_kernel<T, 8, 2, 1024><<<b.blocks, block, smem, s>>>(p);
    else rms_norm_bwd_kernel<T, 8, 2, 256><<<b.blocks, block, smem, s>>>(p);
  } else if (b.vpt == 4) {
    if (wide) rms_norm_bwd_kernel<T, 1, 4, 1024><<<b.blocks, block, smem, s>>>(p);
    else rms_norm_bwd_kernel<T, 1, 4, 256><<<b.blocks, block, smem, s>>>(p);
  } else {
    rms_norm_bwd_kernel<T, 1, 16, 1024><<<b.blocks, block, smem, s>>>(p);
  }
  return cudaSuccess;
}

}  // namespace
}  // namespace jla

using namespace jla;

extern "C" {

int jla_rms_norm_fwd(int dtype, int64_t rows, int dim, const void* x, const void* residual, const float* weight, float eps,
                     int out_e4m3, void* y, void* stream_out, float* rstd, float* scale, jla_stream_t stream) {
  if (const char* why = problem(dtype, rows, dim)) {
    set_error("%s", why);
    return JLA_ERR_BAD_ARGUMENT;
  }
  if (rows == 0) return JLA_OK;
  if (!x || !weight || !y || (residual && !stream_out) || (out_e4m3 && !scale)) {
    set_error("rms norm: null pointer");
    return JLA_ERR_BAD_ARGUMENT;
  }
  RmsParams p{};
  p.rows = rows, p.dim = dim, p.x = x, p.residual = residual, p.w = weight, p.eps = eps, p.y = y, p.stream = stream_out;
  p.rstd = rstd, p.scale = scale;
  const bool vec = dim % 8 == 0 && aligned16(x) && aligned16(residual) && aligned16(weight) && aligned16(y) &&
                   aligned16(stream_out);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  {
    ProfScope scope(kProfRmsNorm, s);
    switch (dtype) {
      case JLA_DTYPE_BF16: out_e4m3 ? launch_fwd<__nv_bfloat16, true>(p, vec, s) : launch_fwd<__nv_bfloat16, false>(p, vec, s); break;
      case JLA_DTYPE_F16: out_e4m3 ? launch_fwd<__half, true>(p, vec, s) : launch_fwd<__half, false>(p, vec, s); break;
      default: out_e4m3 ? launch_fwd<float, true>(p, vec, s) : launch_fwd<float, false>(p, vec, s); break;
    }
  }
  JLA_LAUNCH_OK();
  return JLA_OK;
}

size_t jla_rms_norm_bwd_scratch_bytes(int64_t rows, int dim) {
  if (problem(JLA_DTYPE_F32, rows, dim) || rows == 0) return 0;
  const int a = bwd_shape(rows, dim, false).blocks, b = dim % 8 == 0 ? bwd_shape(rows, dim, true).blocks : 0;
  return (size_t)(a > b ? a : b) * dim * sizeof(float);
}

int jla_rms_norm_bwd(int dtype, int64_t rows, int dim, const void* x, const void* residual, const float* rstd,
                     const float* weight, const void* dy, const void* dstream, void* dx, float* dweight, void* scratch, size_t scratch_bytes,
                     jla_stream_t stream) {
  if (const char* why = problem(dtype, rows, dim)) {
    set_error("%s", why);
    return JLA_ERR_BAD_ARGUMENT;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    if (dweight) JLA_CUDA_OK(cudaMemsetAsync(dweight, 0, sizeof(float) * dim, s));
    return JLA_OK;
  }
  if (!x || !rstd || !weight || !dy || !dx) {
    set_error("rms norm: null pointer");
    return JLA_ERR_BAD_ARGUMENT;
  }
  if (dweight && (!scratch || scratch_bytes < jla_rms_norm_bwd_scratch_bytes(rows, dim))) {
    set_error("rms norm: %zu bytes of scratch, %zu needed", scratch_bytes, jla_rms_norm_bwd_scratch_bytes(rows, dim));
    return JLA_ERR_WORKSPACE;
  }
  RmsParams p{};
  p.rows = rows, p.dim = dim, p.x = x, p.residual = residual, p.rstd = const_cast<float*>(rstd), p.w = weight, p.dy = dy;
  p.dstream = dstream;
  p.dx = dx, p.partial = dweight ? static_cast<float*>(scratch) : nullptr;
  const bool vec = dim % 8 == 0 && aligned16(x) && aligned16(residual) && aligned16(weight) && aligned16(dy) &&
                   aligned16(dstream) && aligned16(dx) && aligned16(scratch);
  const BwdShape b = bwd_shape(rows, dim, vec);
  {
    ProfScope scope(kProfRmsNormBwd, s);
    switch (dtype) {
      case JLA_DTYPE_BF16: JLA_CUDA_OK(launch_bwd<__nv_bfloat16>(p, b, vec, s)); break;
      case JLA_DTYPE_F16: JLA_CUDA_OK(launch_bwd<__half>(p, b, vec, s)); break;
      default: JLA_CUDA_OK(launch_bwd<float>(p, b, vec, s)); break;
    }
  }
  JLA_LAUNCH_OK();
  return dweight ? column_sums(p.partial, b.blocks, dim, dweight, s) : JLA_OK;
}

}  // extern "C"
