// What the matrix-product kernels share: the activations of their epilogues, their parameters, and their launchers.
//
//   linear:  z = (x W^T) xs ws + bias,  y = act(z) + residual          gated:  h = act(x Wg^T xs gs) * (x Wu^T xs us)
#pragma once

#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "tma.cuh"

namespace jla {

enum { kActNone = JLA_ACT_NONE, kActSilu = JLA_ACT_SILU, kActGelu = JLA_ACT_GELU, kActSigmoid = JLA_ACT_SIGMOID };

constexpr int kStatusProduct = 4, kStatusFewTokens = 5;  // codes of the device status word

__device__ __forceinline__ float sigmoid_f32(float z) { return fast_rcp(1.f + fast_exp(-z)); }

// gelu in its tanh form: 0.5 z (1 + tanh(t)) = z sigmoid(2 t), t = sqrt(2 / pi) (z + 0.044715 z^3)
constexpr float kGelu2C = 1.5957691216057308f, kGeluA = 0.044715f;

template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == kActNone) return z;
  const float s = sigmoid_f32(ACT == kActGelu ? kGelu2C * (z + kGeluA * z * z * z) : z);
  return ACT == kActSigmoid ? s : z * s;
}
// f(std::integral_constant) with the activation as a compile-time constant: one branch for many values
template <typename F>
__device__ __forceinline__ void with_activation(int act, F&& f) {
  switch (act) {
    case kActSilu: f(std::integral_constant<int, kActSilu>{}); break;
    case kActGelu: f(std::integral_constant<int, kActGelu>{}); break;
    case kActSigmoid: f(std::integral_constant<int, kActSigmoid>{}); break;
    default: f(std::integral_constant<int, kActNone>{}); break;
  }
}
// act'(z)
template <int ACT>
__device__ __forceinline__ float activation_slope(float z) {
  if constexpr (ACT == kActNone) return 1.f;
  if constexpr (ACT == kActGelu) {
    z = fabsf(z) > 32.f ? copysignf(32.f, z) : z;  // the slope is 0 or 1 from far below that on; z^2 must not overflow (NaN stays)
    const float s = sigmoid_f32(kGelu2C * (z + kGeluA * z * z * z));
    return s + z * s * (1.f - s) * kGelu2C * (1.f + 3.f * kGeluA * z * z);
  }
  const float s = sigmoid_f32(z);
  return ACT == kActSigmoid ? s * (1.f - s) : s * (1.f + z * (1.f - s));
}

// f(std::true_type) for float16 outputs, f(std::false_type) for bfloat16
template <typename F>
__device__ __forceinline__ void with_half(bool half, F&& f) {
  if (half) f(std::true_type{});
  else f(std::false_type{});
}

// Two float32 values rounded to bf16 or f16 (HALF) in one register.
template <bool HALF>
__device__ __forceinline__ uint32_t pack_out(float lo, float hi) {
  if constexpr (HALF) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <bool HALF>
__device__ __forceinline__ float2 unpack_out(uint32_t x) {
  if constexpr (HALF) return __half22float2(*reinterpret_cast<const __half2*>(&x));
  else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
}

// Steps of the contraction (128 bytes of a row each: four instructions) that are summed in one accumulator. An instruction cuts
// the sum off to float32's 24 bits where an addition would round it: up to 2^-23 of the sum each time, always to the same
// side. 1024 of them are off by 2^-13 at most, a quarter of half a step of float16 (measured: 2e-5 of the result with random signs,
// 6.5e-5 where all terms are positive; twice as many: 4e-5 and 1.5e-4, so that the gradient of a weight over 400k tokens would be off
// by more than half a step). Longer contractions are summed in parts, and the parts joined with rounding. It also bounds what a
// wait for a finished accumulator waits for: 256 steps are about 75 us, its limit is kSpinLimit polls, over 40 ms.
constexpr int kPartSteps = 256;

// One product (host view). "tokens" are the rows of y, "features" its columns; the contraction runs over `depth`, and over
// the second pair of operands after the first where there is one (dx = dg Wg + du Wu).
struct Product {
  int dtype = 0;      // of the operands: JLA_DTYPE_BF16, _F16 or _E4M3
  int out_dtype = 0;  // of y and the residual: JLA_DTYPE_BF16 or _F16
  int64_t rows = 0;
  int features = 0, depth = 0;
  bool gated = false;    // two weights, two accumulators a column
  bool pair = false;     // a second pair of operands in the contraction
  bool group = false;    // a second product with operands x[1] and w[0], written to y[1]
  bool x_mn = false, w_mn = false;  // operand stored with the contraction along its rows ([depth][tokens], [depth][features])
  const void* x[2] = {};
  int64_t x_stride = 0;  // elements between the rows of x in memory
  const void* w[2] = {};
  int64_t w_stride = 0;
  const float* x_scale = nullptr;
  const float* w_scale[2] = {};
  const float* bias = nullptr;
  int act = 0;
  const void* residual = nullptr;
  void* y[2] = {};
  float* save[2] = {};   // z, or g and u, in float32 for a later backward pass
};

int product_pairs(const Product& p, int device, int sms, cudaStream_t stream);       // product_tc.cu: any number of tokens
int product_few_tokens(const Product& p, int device, cudaStream_t stream);  // few_tokens.cu: where few_tokens_applies
bool few_tokens_applies(const Product& p, int sms);

int* tc_status_ptr();  // status.cu

// The current device and its number of SMs; a jla_status.
int current_device(int* device, int* sms);  // product_api.cu

// Allows `kern` its dynamic shared memory, once on each device: `done` (one bit a device) belongs to this kernel alone.
template <typename K>
inline cudaError_t allow_smem(K* kern, int bytes, int device, std::atomic<uint64_t>& done) {
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

}  // namespace jla
