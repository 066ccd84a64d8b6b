// C entry points of the matrix products (declared in include/jla_b200.h): argument checks and the choice of kernel.
#include <stdio.h>

#include "product.cuh"

namespace jla {

int current_device(int* device, int* sms) {
  static std::atomic<int> known[64];  // a device's SMs, 0 while nobody has asked
  JLA_CUDA_OK(cudaGetDevice(device));
  const bool kept = *device >= 0 && *device < 64;
  *sms = kept ? known[*device].load(std::memory_order_relaxed) : 0;
  if (*sms == 0) {
    JLA_CUDA_OK(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, *device));
    if (kept) known[*device].store(*sms, std::memory_order_relaxed);
  }
  return JLA_OK;
}

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int refuse(const char* why) {
  set_error("%s", why);
  return JLA_ERR_BAD_ARGUMENT;
}

const char* sizes_problem(int64_t rows, int in, int out, int in_step) {
  static thread_local char buf[160];
  if (rows < 0 || rows > (1L << 31) - 512) return "linear: rows must be 0 .. 2^31 - 512";
  if (in < in_step || in % in_step || out < 8 || out % 8 || in > (1 << 24) || out > (1 << 24)) {
    snprintf(buf, sizeof(buf), "linear: in features (%d) must be a multiple of %d, out features (%d) of 8, both at most 2^24", in,
             in_step, out);
    return buf;
  }
  return nullptr;
}

const char* fwd_problem(int dtype, int out_dtype, int64_t rows, int in, int out, int64_t x_stride, const float* x_scale,
                        const float* w_scale, const float* w_scale2, int act) {
  const bool e4m3 = dtype == JLA_DTYPE_E4M3;
  if (!e4m3 && dtype != JLA_DTYPE_BF16 && dtype != JLA_DTYPE_F16) return "linear: operands must be bf16, f16 or e4m3";
  if (out_dtype != JLA_DTYPE_BF16 && out_dtype != JLA_DTYPE_F16) return "linear: the output must be bf16 or f16";
  if (!e4m3 && out_dtype != dtype) return "linear: the output has the operands' type unless they are e4m3";
  if (rows != 0 && (e4m3 != (x_scale != nullptr) || e4m3 != (w_scale != nullptr) || e4m3 != (w_scale2 != nullptr))) {
    return "linear: scales go with e4m3 operands";  // (those of no rows may be a null pointer)
  }
  if (act < JLA_ACT_NONE || act > JLA_ACT_SIGMOID) return "linear: unknown activation";
  if (const char* why = sizes_problem(rows, in, out, e4m3 ? 16 : 8)) return why;
  if (x_stride < in || x_stride % (e4m3 ? 16 : 8)) return "linear: rows of x must start on multiples of 16 bytes";
  return nullptr;
}

int run(const Product& p, cudaStream_t s) {
  for (const void* q : {p.x[0], p.x[1], p.w[0], p.w[1], static_cast<const void*>(p.x_scale),
                        static_cast<const void*>(p.w_scale[0]), static_cast<const void*>(p.w_scale[1]),
                        static_cast<const void*>(p.bias), p.residual, static_cast<const void*>(p.y[0]),
                        static_cast<const void*>(p.y[1]), static_cast<const void*>(p.save[0]),
                        static_cast<const void*>(p.save[1])}) {
    if (!aligned16(q)) return refuse("linear: pointers must be 16-byte aligned");
  }
  int device = 0, sms = 0;
  if (const int rc = current_device(&device, &sms)) return rc;
  return few_tokens_applies(p, sms) ? product_few_tokens(p, device, s) : product_pairs(p, device, sms, s);
}

}  // namespace
}  // namespace jla

using namespace jla;

extern "C" {

int jla_linear_fwd(int dtype, int out_dtype, int64_t rows, int in, int out, const void* x, int64_t x_stride, const void* w,
                   const float* x_scale, const float* w_scale, const float* bias, int act, const void* residual, void* y,
                   float* z, jla_stream_t stream) {
  if (const char* why = fwd_problem(dtype, out_dtype, rows, in, out, x_stride, x_scale, w_scale, w_scale, act)) return refuse(why);
  if (rows == 0) return JLA_OK;
  if (!x || !w || !y) return refuse("linear: null pointer");
  Product p;
  p.dtype = dtype, p.out_dtype = out_dtype, p.rows = rows, p.features = out, p.depth = in;
  p.x[0] = x, p.x_stride = x_stride, p.w[0] = w, p.w_stride = in, p.x_scale = x_scale, p.w_scale[0] = w_scale;
  p.bias = bias, p.act = act, p.residual = residual, p.y[0] = y, p.save[0] = z;
  return run(p, static_cast<cudaStream_t>(stream));
}

int jla_gated_linear_fwd(int dtype, int out_dtype, int64_t rows, int in, int out, const void* x, int64_t x_stride,
                         const void* w_gate, const void* w_up, const float* x_scale, const float* gate_scale,
                         const float* up_scale, int act, void* h, float* g, float* u, jla_stream_t stream) {
  if (const char* why = fwd_problem(dtype, out_dtype, rows, in, out, x_stride, x_scale, gate_scale, up_scale, act)) {
    return refuse(why);
  }
  if (rows == 0) return JLA_OK;
  if (!x || !w_gate || !w_up || !h || (g != nullptr) != (u != nullptr)) return refuse("gated linear: null pointer");
  Product p;
  p.dtype = dtype, p.out_dtype = out_dtype, p.rows = rows, p.features = out, p.depth = in, p.gated = true;
  p.x[0] = x, p.x_stride = x_stride, p.w[0] = w_gate, p.w[1] = w_up, p.w_stride = in, p.x_scale = x_scale;
  p.w_scale[0] = gate_scale, p.w_scale[1] = up_scale, p.act = act, p.y[0] = h, p.save[0] = g, p.save[1] = u;
  return run(p, static_cast<cudaStream_t>(stream));
}

int jla_linear_bwd_input(int dtype, int64_t rows, int in, int out, const void* dz, const void* w, const void* dz2,
                         const void* w2, void* dx, jla_stream_t stream) {
  if (dtype != JLA_DTYPE_BF16 && dtype != JLA_DTYPE_F16) return refuse("linear gradient: bf16 and f16 only");
  if (const char* why = sizes_problem(rows, in, out, 8)) return refuse(why);
  if (rows == 0) return JLA_OK;
  if (!dz || !w || !dx || (dz2 != nullptr) != (w2 != nullptr)) return refuse("linear gradient: null pointer");
  Product p;
  p.dtype = p.out_dtype = dtype, p.rows = rows, p.features = in, p.depth = out, p.pair = dz2 != nullptr, p.w_mn = true;
  p.x[0] = dz, p.x[1] = dz2, p.x_stride = out, p.w[0] = w, p.w[1] = w2, p.w_stride = in, p.y[0] = dx;
  return run(p, static_cast<cudaStream_t>(stream));
}

int jla_linear_bwd_weight(int dtype, int64_t rows, int in, int out, const void* dz, const void* dz2, const void* x,
                          int64_t x_stride, void* dw, void* dw2, jla_stream_t stream) {
  if (dtype != JLA_DTYPE_BF16 && dtype != JLA_DTYPE_F16) return refuse("linear gradient: bf16 and f16 only");
  if (const char* why = sizes_problem(rows, in, out, 8)) return refuse(why);
  if (x_stride < in || x_stride % 8) return refuse("linear gradient: rows of x must start on multiples of 16 bytes");
  if (!dw) return refuse("linear gradient: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    JLA_CUDA_OK(cudaMemsetAsync(dw, 0, (size_t)in * out * 2, s));
    if (dw2) JLA_CUDA_OK(cudaMemsetAsync(dw2, 0, (size_t)in * out * 2, s));
    return JLA_OK;
  }
  if (!dz || !x || (dz2 != nullptr) != (dw2 != nullptr)) return refuse("linear gradient: null pointer");
  Product p;
  p.dtype = p.out_dtype = dtype, p.rows = out, p.features = in, p.depth = (int)rows, p.group = dz2 != nullptr;
  p.x_mn = p.w_mn = true, p.x[0] = dz, p.x[1] = dz2, p.x_stride = out, p.w[0] = x, p.w_stride = x_stride;
  p.y[0] = dw, p.y[1] = dw2;
  return run(p, s);
}

}  // extern "C"
