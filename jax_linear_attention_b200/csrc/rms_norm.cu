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
// written once. A row belongs to a group of threads, a power of two, each with VPT vectors of VEC adjacent channels: 16
// bytes where the width and the addresses allow it, else single channels (neighbouring threads still read neighbouring
// channels). Sums are held in float32. The norm is taken of the unrounded t, and the backward pass adds x
// and the residual up again: the rounded stream, half the bytes to read, would leave the float32 weight gradient with an
// error of 2e-3 instead of 2e-7.
//
// Measured on a B200, inputs from HBM: 16384 x 2048 bf16 with residual 44 us forward (6.0 TB/s), 60 us backward (5.6 TB/s);
// 5003 x 4096 f16 with residual to e4m3 29 us (5.0 TB/s); one row 2.2 us.
//
// The weight gradient is summed in registers over the rows that a thread walks, over the block in shared memory, and
// over the blocks by column_sums(), always in the same order.
#include <cuda_fp8.h>

#include <type_traits>

#include "column_sums.cuh"
#include "overlap.cuh"
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

// VEC adjacent elements of T as they lie in memory (16 bytes, or one element), and as floats in pairs.
template <typename T, int VEC> struct Raw {
  typedef typename std::conditional<VEC == 1, T, uint4>::type Bits;
  static_assert(VEC == 1 || VEC * sizeof(T) == 16, "a vector is 16 bytes");
  Bits bits;
  __device__ __forceinline__ void load(const T* p) { bits = *reinterpret_cast<const Bits*>(p); }
  __device__ __forceinline__ void zero() {
    if constexpr (VEC == 1) bits = from_f32<T>(0.f);
    else bits = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void get(float (&f)[VEC]) const {
    if constexpr (VEC == 1) {
      f[0] = to_f32(bits);
    } else {
      const uint32_t w[4] = {bits.x, bits.y, bits.z, bits.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, float>::value) {
          f[i] = __uint_as_float(w[i]);
        } else if constexpr (std::is_same<T, __half>::value) {
          const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
          f[2 * i] = v.x, f[2 * i + 1] = v.y;
        } else {
          f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
      }
    }
  }
  static __device__ __forceinline__ void store(T* p, const float (&f)[VEC]) {
    if constexpr (VEC == 1) {
      *p = from_f32<T>(f[0]);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, float>::value) {
          w[i] = __float_as_uint(f[i]);
        } else if constexpr (std::is_same<T, __half>::value) {
          const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&v);
        } else {
          const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
      }
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
};

template <int VEC>
__device__ __forceinline__ void load_weight(const float* p, float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    f[0] = *(p);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const float4 u = *(reinterpret_cast<const float4*>(p + i));
      f[i] = u.x, f[i + 1] = u.y, f[i + 2] = u.z, f[i + 3] = u.w;
    }
  }
}

// Products and sums of VEC floats, two an instruction where there are two.
template <int VEC>
__device__ __forceinline__ void add_to(float (&a)[VEC], const float (&b)[VEC]) {
  if constexpr (VEC == 1) {
    a[0] += b[0];
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const float2 v = unpack2f(add2(pack2f(a[i], a[i + 1]), pack2f(b[i], b[i + 1])));
      a[i] = v.x, a[i + 1] = v.y;
    }
  }
}
template <int VEC>
__device__ __forceinline__ void scale_by(float (&a)[VEC], float s) {
  if constexpr (VEC == 1) {
    a[0] *= s;
  } else {
    const f32x2 ss = pack2f(s, s);
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const float2 v = unpack2f(mul2(pack2f(a[i], a[i + 1]), ss));
      a[i] = v.x, a[i + 1] = v.y;
    }
  }
}
template <int VEC>
__device__ __forceinline__ void multiply_by(float (&a)[VEC], const float (&b)[VEC]) {
  if constexpr (VEC == 1) {
    a[0] *= b[0];
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const float2 v = unpack2f(mul2(pack2f(a[i], a[i + 1]), pack2f(b[i], b[i + 1])));
      a[i] = v.x, a[i + 1] = v.y;
    }
  }
}
// acc += a b, element by element
template <int VEC>
__device__ __forceinline__ void fma_to(float (&acc)[VEC], const float (&a)[VEC], const float (&b)[VEC]) {
  if constexpr (VEC == 1) {
    acc[0] += a[0] * b[0];
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const float2 v = unpack2f(fma2(pack2f(a[i], a[i + 1]), pack2f(b[i], b[i + 1]), pack2f(acc[i], acc[i + 1])));
      acc[i] = v.x, acc[i + 1] = v.y;
    }
  }
}
template <int VEC>
__device__ __forceinline__ float sum_of(const float (&a)[VEC]) {
  if constexpr (VEC == 1) return a[0];
  else if constexpr (VEC == 4) return (a[0] + a[1]) + (a[2] + a[3]);
  else return ((a[0] + a[1]) + (a[2] + a[3])) + ((a[4] + a[5]) + (a[6] + a[7]));
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
  typedef Raw<T, VEC> R;
  const long row = (long)blockIdx.x * blockDim.y + threadIdx.y;
  const bool live = row < p.rows;
  const size_t base = (size_t)(live ? row : 0) * p.dim;
  const int tpr = blockDim.x;
  const T* x = static_cast<const T*>(p.x);
  const T* res = static_cast<const T*>(p.residual);
  R xr[VPT], rr[VPT];
  start_next();
  wait_for_previous();
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int c = (j * tpr + threadIdx.x) * VEC;
    const bool on = live && c < p.dim;
    xr[j].zero(), rr[j].zero();
    if (on) xr[j].load(x + base + c);
    if (on && res) rr[j].load(res + base + c);
  }
  float f[VPT][VEC], sq[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) sq[i] = 0.f;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    xr[j].get(f[j]);
    if (res) {
      float r[VEC];
      rr[j].get(r);
      add_to<VEC>(f[j], r);
    }
    if (p.stream) {
      const int c = (j * tpr + threadIdx.x) * VEC;
      if (live && c < p.dim) R::store(static_cast<T*>(p.stream) + base + c, f[j]);
    }
    fma_to<VEC>(sq, f[j], f[j]);
  }
  const float rstd = rsqrtf(row_reduce<false>(sum_of<VEC>(sq), red[0]) / (float)p.dim + p.eps);
  if (p.rstd && live && threadIdx.x == 0) p.rstd[row] = rstd;
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int c = (j * tpr + threadIdx.x) * VEC;
    if (c < p.dim) {
      float w[VEC];
      load_weight<VEC>(p.w + c, w);
      scale_by<VEC>(f[j], rstd);
      multiply_by<VEC>(f[j], w);
      if constexpr (E4M3) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) top = max_nan(top, fabsf(f[j][i]));
      } else if (live) {
        R::store(static_cast<T*>(p.y) + base + c, f[j]);
      }
    }
  }
  if constexpr (E4M3) {
    float scale = row_reduce<true>(top, red[1]) / kE4m3Max;
    if (scale < 1.17549435e-38f) scale = 1.f;  // a row of zeros (or of subnormal numbers, which e4m3 then holds as zeros)
    if (live && threadIdx.x == 0) p.scale[row] = scale;
    const float inv = 1.f / scale;  // (one division a row: a value within 2^-23 of the middle of two codes may take either)
    unsigned char* q = static_cast<unsigned char*>(p.y);
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int c = (j * tpr + threadIdx.x) * VEC;
      if (live && c < p.dim) {
        scale_by<VEC>(f[j], inv);
        if constexpr (VEC == 1) {
          q[base + c] = __nv_cvt_float_to_fp8(f[j][0], __NV_SATFINITE, __NV_E4M3);
        } else {
          uint32_t e[VEC / 4];
#pragma unroll
          for (int i = 0; i < VEC / 4; ++i) {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[j][4 * i], f[j][4 * i + 1]), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[j][4 * i + 2], f[j][4 * i + 3]), __NV_SATFINITE, __NV_E4M3);
            e[i] = lo | (hi << 16);
          }
          if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(q + base + c) = e[0];
          else *reinterpret_cast<uint2*>(q + base + c) = make_uint2(e[0], e[1]);
        }
      }
    }
  }
}

// Blocks walk the rows blockIdx.x * blockDim.y + threadIdx.y, + gridDim.x * blockDim.y, ... (the same number of steps for
// all threads of a block: row_reduce may synchronise it). The next row's loads leave before a row is worked on: with four
// tensors to read, the loads of one row in flight at a time left HBM at 4.1 TB/s.
// (Blocks of 1024 threads have no registers for that.)
template <typename T, int VEC, int VPT, int MAXT>
__global__ void __launch_bounds__(MAXT) rms_norm_bwd_kernel(RmsParams p) {
  constexpr bool kAhead = MAXT < 1024;
  __shared__ float red[2][32];
  extern __shared__ float fold[];  // [blockDim.y][dim] of the weight gradient, where a block has several rows
  typedef Raw<T, VEC> R;
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
  R xr[VPT], rr[VPT], dr[VPT], sr[VPT];
  float rstd_next = 0.f;
  auto request = [&](long r0) {
    const long row = r0 + threadIdx.y;
    const bool live = row < p.rows;
    const size_t base = (size_t)(live ? row : 0) * p.dim;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int c = (j * tpr + threadIdx.x) * VEC;
      const bool on = live && c < p.dim;
      xr[j].zero(), rr[j].zero(), dr[j].zero(), sr[j].zero();
      if (on) {
        xr[j].load(x + base + c);
        dr[j].load(dy + base + c);
        if (res) rr[j].load(res + base + c);
        if (ds) sr[j].load(ds + base + c);
      }
    }
    rstd_next = live ? p.rstd[row] : 0.f;
  };
  start_next();
  wait_for_previous();
  const long first = (long)blockIdx.x * blockDim.y, step = (long)gridDim.x * blockDim.y;
  if (kAhead && first < p.rows) request(first);
  int turn = 0;
  for (long r0 = first; r0 < p.rows; r0 += step, turn ^= 1) {
    const long row = r0 + threadIdx.y;
    const bool live = row < p.rows;
    const size_t base = (size_t)(live ? row : 0) * p.dim;
    if (!kAhead) request(r0);
    const float rstd = rstd_next;
    float n[VPT][VEC], d[VPT][VEC], s[VPT][VEC], dot[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) dot[i] = 0.f;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      xr[j].get(n[j]), dr[j].get(d[j]), sr[j].get(s[j]);
      if (res) {
        float r[VEC];
        rr[j].get(r);
        add_to<VEC>(n[j], r);
      }
    }
    if (kAhead && r0 + step < p.rows) request(r0 + step);
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int c = (j * tpr + threadIdx.x) * VEC;
      if (c < p.dim) {
        float w[VEC];
        load_weight<VEC>(p.w + c, w);
        scale_by<VEC>(n[j], rstd);
        fma_to<VEC>(dw[j], d[j], n[j]);
        multiply_by<VEC>(d[j], w);
        fma_to<VEC>(dot, d[j], n[j]);
      }
    }
    const float mean = row_reduce<false>(sum_of<VEC>(dot), red[turn]) * inv_dim;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int c = (j * tpr + threadIdx.x) * VEC;
      if (live && c < p.dim) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) s[j][i] += rstd * (d[j][i] - n[j][i] * mean);
        R::store(static_cast<T*>(p.dx) + base + c, s[j]);
      }
    }
  }
  if (!p.partial) return;
  float* out = p.partial + (size_t)blockIdx.x * p.dim;
  if (blockDim.y > 1) {
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int c = (j * tpr + threadIdx.x) * VEC;
      if (c < p.dim) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) fold[(size_t)threadIdx.y * p.dim + c + i] = dw[j][i];
      }
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
      if (c < p.dim) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[c + i] = dw[j][i];
      }
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

// Threads of a row (a power of two), its vectors a thread, and rows a block.
struct RowShape {
  int tpr, vpt, rpb;
};
RowShape row_shape(int vectors, int vpt) {
  int tpr = ceil_pow2((vectors + vpt - 1) / vpt);
  if (tpr < 8) tpr = 8;
  return {tpr, vpt, tpr >= 256 ? 1 : 256 / tpr};
}

template <typename T, bool E4M3>
cudaError_t launch_fwd(const RmsParams& p, bool vec, cudaStream_t s) {
  cudaError_t err = cudaSuccess;
  // Few rows: one vector a thread, so that a row's loads all leave at once (a decoding step is latency). Many rows: four
  // vectors, fewer threads meet in the reduction and more rows are in flight.
  constexpr int VEC = 16 / sizeof(T);
  const int vectors = vec ? p.dim / VEC : p.dim;
  const RowShape b = row_shape(vectors, vec ? (vectors <= 1024 && p.rows <= 148 ? 1 : 4) : (vectors <= 4096 ? 4 : 16));
  const dim3 block(b.tpr, b.rpb), grid((unsigned)((p.rows + b.rpb - 1) / b.rpb));
  if (vec) {
    if (b.vpt == 1) err = launch_overlapped(rms_norm_fwd_kernel<T, VEC, 1, E4M3>, grid, block, 0, s, 0, p);
    else err = launch_overlapped(rms_norm_fwd_kernel<T, VEC, 4, E4M3>, grid, block, 0, s, 0, p);
  } else {
    if (b.vpt == 4) err = launch_overlapped(rms_norm_fwd_kernel<T, 1, 4, E4M3>, grid, block, 0, s, 0, p);
    else err = launch_overlapped(rms_norm_fwd_kernel<T, 1, 16, E4M3>, grid, block, 0, s, 0, p);
  }
  return err;
}

// Backward: two vectors a thread (registers), four where a block would not have the threads.
RowShape bwd_shape(int dim, int vec) {
  const int vectors = dim / vec;
  return row_shape(vectors, vec > 1 ? (vectors <= 2048 ? 2 : 4) : (vectors <= 4096 ? 4 : 16));
}
// Blocks that walk the rows: two of 256 threads an SM are there at one time (by their registers), one of 512 or 1024.
int bwd_blocks(long rows, const RowShape& b) {
  const long groups = (rows + b.rpb - 1) / b.rpb, most = b.tpr > 256 ? 148 : 296;
  return (int)(groups < most ? groups : most);
}

template <typename T>
cudaError_t launch_bwd(const RmsParams& p, const RowShape& b, int blocks, bool vec, cudaStream_t s) {
  cudaError_t err = cudaSuccess;
  constexpr int VEC = 16 / sizeof(T);
  const dim3 block(b.tpr, b.rpb);
  const size_t smem = b.rpb > 1 && p.partial ? (size_t)b.rpb * p.dim * sizeof(float) : 0;  // at most 16 KB
  if (vec && b.vpt == 2) {
    if (b.tpr > 512) err = launch_overlapped(rms_norm_bwd_kernel<T, VEC, 2, 1024>, dim3(blocks), block, smem, s, 0, p);
    else if (b.tpr > 256) err = launch_overlapped(rms_norm_bwd_kernel<T, VEC, 2, 512>, dim3(blocks), block, smem, s, 0, p);
    else err = launch_overlapped(rms_norm_bwd_kernel<T, VEC, 2, 256>, dim3(blocks), block, smem, s, 0, p);
  } else if (vec) {
    if constexpr (VEC == 4) err = launch_overlapped(rms_norm_bwd_kernel<T, VEC, 4, 1024>, dim3(blocks), block, smem, s, 0, p);
  } else if (b.vpt == 4) {
    if (b.tpr > 512) err = launch_overlapped(rms_norm_bwd_kernel<T, 1, 4, 1024>, dim3(blocks), block, smem, s, 0, p);
    else if (b.tpr > 256) err = launch_overlapped(rms_norm_bwd_kernel<T, 1, 4, 512>, dim3(blocks), block, smem, s, 0, p);
    else err = launch_overlapped(rms_norm_bwd_kernel<T, 1, 4, 256>, dim3(blocks), block, smem, s, 0, p);
  } else {
    err = launch_overlapped(rms_norm_bwd_kernel<T, 1, 16, 1024>, dim3(blocks), block, smem, s, 0, p);
  }
  return err;
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
  const bool vec = dim % (dtype == JLA_DTYPE_F32 ? 4 : 8) == 0 && aligned16(x) && aligned16(residual) && aligned16(weight) &&
                   aligned16(y) && aligned16(stream_out);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t err = cudaSuccess;
  {
    ProfScope scope(kProfRmsNorm, s);
    switch (dtype) {
      case JLA_DTYPE_BF16: err = out_e4m3 ? launch_fwd<__nv_bfloat16, true>(p, vec, s) : launch_fwd<__nv_bfloat16, false>(p, vec, s); break;
      case JLA_DTYPE_F16: err = out_e4m3 ? launch_fwd<__half, true>(p, vec, s) : launch_fwd<__half, false>(p, vec, s); break;
      default: err = out_e4m3 ? launch_fwd<float, true>(p, vec, s) : launch_fwd<float, false>(p, vec, s); break;
    }
  }
  JLA_CUDA_OK(err);
  return JLA_OK;
}

size_t jla_rms_norm_bwd_scratch_bytes(int64_t rows, int dim) {
  if (problem(JLA_DTYPE_F32, rows, dim) || rows == 0) return 0;
  int most = bwd_blocks(rows, bwd_shape(dim, 1));
  for (int vec = 4; vec <= 8; vec += 4) {
    const int n = dim % vec == 0 ? bwd_blocks(rows, bwd_shape(dim, vec)) : 0;
    most = n > most ? n : most;
  }
  return (size_t)most * dim * sizeof(float);
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
  const int width = dtype == JLA_DTYPE_F32 ? 4 : 8;
  const bool vec = dim % width == 0 && aligned16(x) && aligned16(residual) && aligned16(weight) && aligned16(dy) &&
                   aligned16(dstream) && aligned16(dx);
  const RowShape b = bwd_shape(dim, vec ? width : 1);
  const int blocks = bwd_blocks(rows, b);
  cudaError_t err = cudaSuccess;
  {
    ProfScope scope(kProfRmsNormBwd, s);
    switch (dtype) {
      case JLA_DTYPE_BF16: err = launch_bwd<__nv_bfloat16>(p, b, blocks, vec, s); break;
      case JLA_DTYPE_F16: err = launch_bwd<__half>(p, b, blocks, vec, s); break;
      default: err = launch_bwd<float>(p, b, blocks, vec, s); break;
    }
  }
  JLA_CUDA_OK(err);
  return dweight ? column_sums(p.partial, blocks, dim, dweight, s) : JLA_OK;
}

}  // extern "C"
