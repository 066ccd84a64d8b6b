// Matrix products of few tokens (a decoding step, a short prompt) or few features with the epilogue fused: what
// product_tc.cu computes, for calls whose time is that of reading the weights.
//
// Bound by HBM, so the weights have to stream through as many SMs as there are. The roles of the operands are swapped: 128
// features (rows of W) fill the 128 TMEM lanes, BN tokens are the accumulator's columns, so that few tokens waste
// neither tensor-core rows nor shared memory. The contraction is cut into up to eight parts, one for each CTA of a
// cluster; the cluster's CTAs share out the tokens among themselves, push each other their partial sums over distributed
// shared memory, and add the parts up in the order of the parts, every time the same. A CTA with more than kPartSteps steps of
// its own sums those in runs of as many, one after the other in the same accumulator, and joins them in a second one.
//
// Measured on a B200, weights from HBM, one pass among others (a kernel starts under the end of the one before; by itself it takes
// about 4 us more): one token, 2048 -> 8512 bf16 9.3 us (35 MB; 5.3 at HBM's rate); 33 tokens, 4096 -> 2048 e4m3 6.6 us; gated, four
// tokens, 2048 -> 5632 bf16 10.9 us (46 MB; 7.1). Of that about 0.8 us are set-up, 1.5 to 2.5 us the way of the first bytes, 1.5 to
// 2 us the sums and results.
//
// Every wait is bounded, as in product_tc.cu (kStatusFewTokens).
#include "overlap.cuh"
#include "product.cuh"
#include "profile.cuh"
#include "umma_pair.cuh"

namespace jla {
namespace {

using umma::smem_addr;

constexpr int kWarps = 8, kThreads = 32 * kWarps;  // warps 0 .. 3 accumulators, 4 loads, 5 products; all of them the last sums
constexpr int kMaxSplit = 8;

struct Maps {
  CUtensorMap x[2], w[2];
};

struct Params {
  int rows, features;
  int kt0, kt;
  uint32_t idesc;
  int act, half;
  const float *x_scale, *w_scale[2], *bias;
  const void* residual;
  void* y;
  float* save[2];
  int* status;
};

template <int BN, bool GATED> struct Shape {
  static constexpr int kWeights = GATED ? 2 : 1;
  static constexpr int kWeightBytes = 128 * 128;
  static constexpr int kStageBytes = kWeights * kWeightBytes + BN * 128;
  // Partial sums that arrive: whole rounds of up to eight parts, [weight][part][token][128 features].
  static constexpr int kPartRows = BN + kMaxSplit, kPartBytes = kWeights * kPartRows * 512;
  // The ring of operand tiles; afterwards this CTA's own partial sums, [weight][token][128 features]. Half an SM's memory where
  // one weight's sums leave enough of it for the ring: the next kernel's CTAs are set up beside this one's, and two CTAs of a wide
  // product have room. (A pass among others, with all of the memory in brackets: one token, 2048 -> 32768 22.5 us (26.7),
  // 4096 -> 2048 6.6 (6.9), 2048 -> 8512 9.2 (9.3; 9.1 where torch allocates between the passes); but 32 tokens, 2048 -> 8512 10.6 (10.0),
  // and 20 tokens, 8192 -> 8192 27.3 (24.9).)
  static constexpr int kCtas = !GATED && BN <= 32 ? 2 : 1;
  static constexpr int kRoom = (kCtas == 2 ? 110 : 224) * 1024 - 1024 - kPartBytes;
  static constexpr int kFit = kRoom / kStageBytes;
  static constexpr int kStages = kFit < 12 ? kFit : 12;
  static constexpr int kRing = kStages * kStageBytes;
  static_assert(kStages >= 2 && kRing >= kWeights * BN * 512, "the ring has to hold the partial sums");
  static constexpr int kSmem = kRing + kPartBytes + 1024;
  // TMEM columns: a load takes 32 from the start of an accumulator, also where the accumulator has 16
  static constexpr int kNeed = (GATED ? BN : 0) + (BN < 32 ? 32 : BN);
  static_assert(kNeed <= 128, "twice as many where a CTA sums several runs of steps");
  static constexpr int kCols = kNeed <= 32 ? 32 : kNeed <= 64 ? 64 : 128;
};

struct Quad {
  float v[4];
};
__device__ __forceinline__ Quad quad(const float* p) {
  if (!p) return Quad{};
  const float4 f = *(reinterpret_cast<const float4*>(p));
  return Quad{{f.x, f.y, f.z, f.w}};
}

// What is left of four neighbouring features at one token after the products: scales, bias, activation, residual, store.
template <int ACT, bool FP8, bool GATED>
__device__ __forceinline__ void finish(const Params& p, int token, int f, Quad v, Quad u, const Quad& ws0, const Quad& ws1,
                                       const Quad& bias, float xs, uint2 res) {
  const size_t at = (size_t)token * p.features + f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (FP8) v.v[i] *= xs * ws0.v[i];
    if constexpr (FP8 && GATED) u.v[i] *= xs * ws1.v[i];
    if constexpr (!GATED) v.v[i] += bias.v[i];
  }
  if (p.save[0]) *reinterpret_cast<float4*>(p.save[0] + at) = make_float4(v.v[0], v.v[1], v.v[2], v.v[3]);
  if (GATED && p.save[1]) *reinterpret_cast<float4*>(p.save[1] + at) = make_float4(u.v[0], u.v[1], u.v[2], u.v[3]);
#pragma unroll
  for (int i = 0; i < 4; ++i) v.v[i] = activate<ACT>(v.v[i]) * (GATED ? u.v[i] : 1.f);
  if (!GATED && p.residual) {
    with_half(p.half, [&](auto is_half) {
      const float2 lo = unpack_out<is_half()>(res.x), hi = unpack_out<is_half()>(res.y);
      v.v[0] += lo.x, v.v[1] += lo.y, v.v[2] += hi.x, v.v[3] += hi.y;
    });
  }
  with_half(p.half, [&](auto is_half) {
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.y) + at) =
        make_uint2(pack_out<is_half()>(v.v[0], v.v[1]), pack_out<is_half()>(v.v[2], v.v[3]));
  });
}

// RUNS: some CTA has more than kPartSteps steps. (A kernel of its own: the tests for it cost one token, 2048 -> 8512, 0.6 us of 9.4.)
template <int BN, bool W_MN, bool FP8, bool GATED, bool RUNS>
__global__ void __launch_bounds__(kThreads, (Shape<BN, GATED>::kCtas)) few_tokens_kernel(const __grid_constant__ Maps maps,
                                                                 const __grid_constant__ Params p, int split) {
  using S = Shape<BN, GATED>;
  constexpr int ST = S::kStages, NW = GATED ? 2 : 1;
  extern __shared__ unsigned char smem_dyn[];
  __shared__ __align__(8) uint64_t full[ST], empty[ST], done, freed, drain, arrived;
  __shared__ uint32_t tmem_slot;
  const uint32_t base = (smem_addr(smem_dyn) + 1023) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = split > 1 ? (int)umma::cluster_rank() : 0;
  const int f0 = (int)(blockIdx.x / split) * 128, m0 = (int)blockIdx.y * BN;
  const int tokens = p.rows - m0 < BN ? p.rows - m0 : BN, per = (tokens + split - 1) / split;
  auto per_of = [&](int r) { return min(max(tokens - r * per, 0), per); };  // tokens that CTA r finishes
  const int k_lo = (int)((long)p.kt * part / split), k_hi = (int)((long)p.kt * (part + 1) / split);

  // Step `it` of this part's contraction into its stage of the ring.
  auto load = [&](int it, int s) {
    const int kt = k_lo + it;
    tma::expect_tx(full + s, S::kStageBytes);
    const uint32_t bar = smem_addr(full + s);
    const bool second = kt >= p.kt0;
    const int k0 = (second ? kt - p.kt0 : kt) * (FP8 ? 128 : 64);
    const uint32_t ws = base + s * S::kStageBytes, xs = ws + NW * S::kWeightBytes;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      const CUtensorMap* mw = &maps.w[GATED ? i : (second ? 1 : 0)];
      if constexpr (W_MN) {
        tma::load_2d(ws + i * S::kWeightBytes, mw, f0, k0, bar);
        tma::load_2d(ws + i * S::kWeightBytes + 8192, mw, f0 + 64, k0, bar);
      } else {
        tma::load_2d(ws + i * S::kWeightBytes, mw, k0, f0, bar);
      }
    }
    tma::load_2d(xs, &maps.x[second ? 1 : 0], k0, m0, bar);
  };
  const int steps = k_hi - k_lo;
  constexpr uint32_t kCols = RUNS ? 2 * S::kCols : S::kCols;
  int asked = steps < ST ? steps : ST;
  if (warp == 4) {
    if (umma::elect_one()) {
      for (int i = 0; i < ST; ++i) {
        umma::mbar_init(full + i, 1);
        umma::mbar_init(empty + i, 1);
      }
      umma::mbar_init(&done, 1);
      if constexpr (RUNS) umma::mbar_init(&freed, 4);
      umma::mbar_init(&drain, 1);
      umma::mbar_init(&arrived, 1);
      umma::mbar_init_fence();
      umma::fence_async_smem();
      tma::expect_tx(&arrived, NW * split * per_of(part) * 512);
    }
    __syncwarp();
  }
  if (warp == 5) umma::tmem_alloc(&tmem_slot, kCols);
  umma::fence_before_sync();
  umma::cluster_arrive();  // (waited for before the first partial sums leave for another CTA)
  if (warp == 4) {  // the first copies wait for nobody
    asm volatile("bar.arrive 1, %0;\n" ::"n"(kThreads) : "memory");
    wait_for_previous();
    if (umma::elect_one()) {
      for (int it = 0; it < asked; ++it) load(it, it);
    }
    __syncwarp();
  } else {
    asm volatile("bar.sync 1, %0;\n" ::"n"(kThreads) : "memory");
    start_next();
    wait_for_previous();
  }
  umma::fence_after_sync();
  const uint32_t tmem = tmem_slot;
  bool ok = true;

  if (warp == 4) {
    int s = 0;
    uint32_t phase = 0;
    for (int it = ST; it < steps; ++it) {
      ok = umma::mbar_wait_warp(smem_addr(empty) + 8 * s, phase);
      if (!ok) break;
      if (umma::elect_one()) load(it, s);
      __syncwarp();
      asked = it + 1;
      if (++s == ST) s = 0, phase ^= 1;
    }
    if (!ok) {
      for (int j = asked > ST ? asked - ST : 0; j < asked; ++j) umma::mbar_wait_warp(smem_addr(full) + 8 * (j % ST), (j / ST) & 1);
    }
  } else if (warp == 5) {
    const uint64_t w0 = umma::smem_desc(base, W_MN ? 8192 : 16, 1024);
    const uint64_t x0 = umma::smem_desc(base + NW * S::kWeightBytes, 16, 1024);
    int s = 0;
    uint32_t phase = 0;
    for (int it = 0; it < steps; ++it) {
      const int in_run = RUNS ? it % kPartSteps : it;
      if (RUNS && in_run == 0 && it > 0) {  // the run before has been taken over
        ok = umma::mbar_wait_warp(smem_addr(&freed), (it / kPartSteps - 1) & 1);
        if (!ok) break;
      }
      ok = umma::mbar_wait_warp(smem_addr(full) + 8 * s, phase);
      if (!ok) break;
      umma::fence_after_sync();
      if (umma::elect_one()) {
        const uint32_t off = (uint32_t)(s * S::kStageBytes) >> 4;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            umma::mma_any<FP8>(tmem + i * BN, w0 + off + i * (S::kWeightBytes >> 4) + (W_MN ? ks * 128 : ks * 2),
                               x0 + off + ks * 2, p.idesc, in_run > 0 || ks > 0);
          }
        }
        umma::commit(empty + s);
        if ((RUNS && in_run == kPartSteps - 1) || it == steps - 1) umma::commit(&done);
      }
      __syncwarp();
      if (++s == ST) s = 0, phase ^= 1;
    }
    if (!ok) {
      if (umma::elect_one()) umma::commit(&drain);
      __syncwarp();
      umma::mbar_wait_warp(smem_addr(&drain), 0);
    }
  }
  const int f4 = f0 + lane * 4;
  Quad ws0{}, ws1{}, bias{};
  if (f4 < p.features) {
    if constexpr (FP8) ws0 = quad(p.w_scale[0] + f4);
    if constexpr (FP8 && GATED) ws1 = quad(p.w_scale[1] + f4);
    if (!GATED && p.bias) bias = quad(p.bias + f4);
  }
  const uint32_t sums = tmem + (RUNS ? S::kCols : 0) + ((uint32_t)(32 * (warp & 3)) << 16);
  if (warp < 4) {
    ok = umma::mbar_wait(&done, 0);
    umma::fence_after_sync();
  }
  if (RUNS && warp < 4) {
    for (int it = 0, run = 0; it < steps; it += kPartSteps, ++run) {
      if (run > 0) ok = umma::mbar_wait(&done, run & 1);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      umma::fence_after_sync();
#pragma unroll 1
      for (int c = 0; c < NW * BN; c += 16) umma::join_x16(sums + c, sums - S::kCols + c, run == 0);
      umma::wait_st();
      umma::fence_before_sync();
      __syncwarp();
      if (lane == 0) umma::arrive_cluster(smem_addr(&freed));
    }
  }
  // This part's sums, [weight][token][128 features], over the ring, which is idle now. Column c of the accumulator is a token.
  if (warp < 4 && __all_sync(0xffffffffu, ok)) {
    constexpr int CH = BN < 32 ? BN : 32;  // (of a load of 32 columns where there are 16, the last 16 are not looked at)
#pragma unroll 1
    for (int c = 0; c < tokens; c += CH) {
      float v[NW][32];
#pragma unroll
      for (int i = 0; i < NW; ++i) umma::ld_32x32b_x32(v[i], sums + i * BN + c);
      umma::wait_ld();
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        const uint32_t to = base + ((i * BN + c) * 128 + threadIdx.x) * 4;
#pragma unroll
        for (int j = 0; j < CH; ++j) asm volatile("st.shared.f32 [%0], %1;\n" ::"r"(to + j * 512), "f"(v[i][j]) : "memory");
      }
    }
  }
  // CTA r of the cluster finishes the tokens per * r .. per * (r + 1) - 1. Everybody copies it its part of them, one copy a
  // weight and CTA, which count on its barrier; nobody waits for an answer from afar.
  const uint32_t parts_at = base + S::kRing;
  umma::cluster_wait();
  if (split > 1) {
    umma::fence_async_smem();
    __syncthreads();
    if (warp == 4 && lane < split) {
      const int to = part + lane < split ? part + lane : part + lane - split;  // everybody begins with another CTA
      const int n = per_of(to);
      if (n > 0) {
#pragma unroll
        for (int i = 0; i < NW; ++i) {
          umma::copy_cluster(umma::map_rank(parts_at + (i * S::kPartRows + part * per) * 512, to),
                             base + (i * BN + to * per) * 512, n * 512, umma::map_rank(smem_addr(&arrived), to));
        }
      }
    }
    ok = umma::mbar_wait_warp(smem_addr(&arrived), 0) && ok;
  } else {
    __syncthreads();
  }
  // A thread adds up four features of one token in the order of the parts; a warp has up to four tokens on their way.
  const uint32_t from = (split > 1 ? parts_at : base) + lane * 16;
  const int weight_rows = split > 1 ? S::kPartRows : BN, mine = per_of(part);
  if (f4 < p.features) {
    with_activation(p.act, [&](auto act) {
      constexpr int kBatch = 4;
#pragma unroll 1
      for (int c0 = warp; c0 < mine; c0 += kWarps * kBatch) {
        float xs[kBatch];
        uint2 res[kBatch];
        Quad sum[kBatch][NW];
        uint32_t at[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {  // (a token too many is the last one again, and not stored)
          const int c = min(c0 + b * kWarps, mine - 1), token = m0 + part * per + c;
          at[b] = from + c * 512;
          xs[b] = 1.f, res[b] = make_uint2(0, 0);
          if constexpr (FP8) xs[b] = *(p.x_scale + token);
          if (!GATED && p.residual) {
            res[b] = *(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.residual) + (size_t)token * p.features + f4));
          }
#pragma unroll
          for (int i = 0; i < NW; ++i) sum[b][i] = Quad{};
        }
#pragma unroll 1
        for (int r = 0; r < split; ++r) {
#pragma unroll
          for (int b = 0; b < kBatch; ++b) {
#pragma unroll
            for (int i = 0; i < NW; ++i) {
              float v[4];
              asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];\n" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
                           : "r"(at[b] + i * weight_rows * 512) : "memory");
#pragma unroll
              for (int j = 0; j < 4; ++j) sum[b][i].v[j] += v[j];
            }
            at[b] += per * 512;
          }
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          const int c = c0 + b * kWarps;
          if (c < mine) {
            finish<act(), FP8, GATED>(p, m0 + part * per + c, f4, sum[b][0], sum[b][NW - 1], ws0, ws1, bias, xs[b], res[b]);
          }
        }
      }
    });
  }
  if (!ok) atomicExch(p.status, kStatusFewTokens);
  umma::fence_before_sync();
  if (split > 1) umma::cluster_sync();  // the others' copies of this CTA's sums have arrived
  else __syncthreads();
  if (warp == 5) umma::tmem_dealloc(tmem, kCols);
}

template <int BN, bool W_MN, bool FP8, bool GATED>
int launch(const Product& p, int device, cudaStream_t s) {
  using S = Shape<BN, GATED>;
  Maps maps;
  Params q{};
  const int esz = FP8 ? 1 : 2, kb = FP8 ? 128 : 64;
  bool ok = true;
  for (int i = 0; i < 2 && ok; ++i) {
    ok = (!p.x[i] || tma::encode_2d(&maps.x[i], p.x[i], esz, p.depth, p.rows, p.x_stride, BN)) &&
         (!p.w[i] || (W_MN ? tma::encode_2d(&maps.w[i], p.w[i], esz, p.features, p.depth, p.w_stride, 64)
                           : tma::encode_2d(&maps.w[i], p.w[i], esz, p.depth, p.features, p.w_stride, 128)));
  }
  if (!ok) return JLA_ERR_CUDA;
  q.rows = (int)p.rows, q.features = p.features;
  q.kt0 = (p.depth + kb - 1) / kb;
  q.kt = q.kt0 * (p.pair ? 2 : 1);
  q.idesc = FP8 ? umma::instr_desc_e4m3(128, BN) : umma::instr_desc(128, BN, p.dtype == JLA_DTYPE_BF16, W_MN, 0);
  q.act = p.act, q.half = p.out_dtype == JLA_DTYPE_F16;
  q.x_scale = p.x_scale, q.w_scale[0] = p.w_scale[0], q.w_scale[1] = p.w_scale[1], q.bias = p.bias, q.residual = p.residual;
  q.y = p.y[0], q.save[0] = p.save[0], q.save[1] = p.save[1];
  q.status = tc_status_ptr();
  if (!q.status) {
    set_error("the status word of the current device could not be located");
    return JLA_ERR_CUDA;
  }
  const int tiles_f = (p.features + 127) / 128, tiles_m = (int)((p.rows + BN - 1) / BN);
  auto* kern = few_tokens_kernel<BN, W_MN, FP8, GATED, false>;
  static std::atomic<uint64_t> allowed{0}, allowed_runs{0};
  JLA_CUDA_OK(allow_smem(kern, S::kSmem, device, allowed));
  // Parts of the contraction: as many as there is room for at one time, each of at least two steps. (A cluster lies within
  // one of the GPU's groups of SMs, so fewer large clusters fit than their CTAs' number says; one that had to wait for
  // another to finish would double the time.)
  static std::atomic<int> room[64][kMaxSplit + 1];  // clusters of a size at one time, by device
  int split = 1;
  for (int c = kMaxSplit; c > 1; --c) {
    if (c * 2 > q.kt || device >= 64) continue;
    int fit = room[device][c].load(std::memory_order_relaxed);
    if (fit == 0) {
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(c), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = S::kSmem, cfg.stream = s;
      cudaLaunchAttribute attr{};
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = c, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
      cfg.attrs = &attr, cfg.numAttrs = 1;
      JLA_CUDA_OK(cudaOccupancyMaxActiveClusters(&fit, kern, &cfg));
      room[device][c].store(fit > 0 ? fit : -1, std::memory_order_relaxed);
    }
    if (tiles_f * tiles_m <= fit) {
      split = c;
      break;
    }
  }
  if ((q.kt + split - 1) / split > kPartSteps) {
    kern = few_tokens_kernel<BN, W_MN, FP8, GATED, true>;
    JLA_CUDA_OK(allow_smem(kern, S::kSmem, device, allowed_runs));
  }
  ProfScope scope(kProfFewTokens, s);
  JLA_CUDA_OK(launch_overlapped(kern, dim3(tiles_f * split, tiles_m), dim3(kThreads), S::kSmem, s, split, maps, q, split));
  return JLA_OK;
}

template <bool W_MN, bool FP8, bool GATED>
int pick(const Product& p, int dev, cudaStream_t s) {
  if (p.rows <= 16) return launch<16, W_MN, FP8, GATED>(p, dev, s);
  if (p.rows <= 32) return launch<32, W_MN, FP8, GATED>(p, dev, s);
  if (p.rows <= 64) return launch<64, W_MN, FP8, GATED>(p, dev, s);
  if constexpr (GATED) return launch<64, W_MN, FP8, GATED>(p, dev, s);  // (two weights' sums of 128 tokens fit no SM)
  else return launch<128, W_MN, FP8, GATED>(p, dev, s);
}

}  // namespace

// Up to 64 tokens always; up to 8192 where this kernel is expected to be the faster one. Fitted, in hundredths of a us with
// inputs from HBM, to times of both in bf16 and f16 from 33 to 1500 tokens, depths of 64 to 4096 and widths of 256 to 6144:
//   this kernel: 200 + waves (390 + 36 a step of the longest CTA), 110 more where the contraction is split (gated 360, 48, 160)
//   pairs: 720 + 20 a step of the busiest pair; an activation or bias shows with 290 (here 30), a residual with 200 (here 100)
// Some of the times, in us, this kernel against pairs of CTAs: 4096 -> 256, 512 tokens: 10.7, 18.7; 4096 -> 2048, 256: 14.5,
// 20.2; 512 -> 512, 256: 7.9, 9.6, with silu and a residual 8.4, 15.2; 2048 -> 6144, 256: 18.6, 14.8; gated 2048 -> 6144, 256:
// 40.9, 21.3; gated 64 -> 256, 1500: 5.5, 7.6.
// Beyond what it was fitted to (546 calls of 65 to 8192 tokens, depths of 64 to 16384, widths of 64 to 8192, e4m3, dx and gated
// among them) it takes the kernel that is slower by more than 15 % in 18 cases: e4m3 with 64 features (13 us, 10 with pairs),
// and sums over 8192 and more at 4000 tokens and 256 features (74 us with pairs, 64 here).
bool few_tokens_applies(const Product& p, int sms) {
  if (p.x_mn || p.group || p.rows > 8192) return false;
  if (p.rows <= 64) return true;
  const int kb = p.dtype == JLA_DTYPE_E4M3 ? 128 : 64, kt = (p.depth + kb - 1) / kb * (p.pair ? 2 : 1);
  const int bn = p.gated ? 64 : 128, tiles = (p.features + 127) / 128 * (int)((p.rows + bn - 1) / bn);
  int split = sms / tiles < kMaxSplit ? sms / tiles : kMaxSplit;
  split = split > kt / 2 ? kt / 2 : split;
  split = split < 1 ? 1 : split;
  const int steps = (kt + split - 1) / split, waves = (tiles * split + sms - 1) / sms;
  const int cols = p.features * (p.gated ? 2 : 1);
  const int pair_tiles = (int)((p.rows + 255) / 256) * ((cols + 255) / 256), rest = pair_tiles % (sms / 2);
  const int64_t pair_rounds = pair_tiles / (sms / 2) * 100 + (rest == 0 ? 0 : 2 * rest <= sms / 2 ? 69 : 100);  // hundredths
  const bool busy = !p.gated && (p.act != kActNone || p.bias);
  const int64_t here = 200 + (int64_t)waves * (p.gated ? 360 + 48 * steps : 390 + 36 * steps) + (split > 1 ? (p.gated ? 160 : 110) : 0) +
                       (busy ? 30 : 0) + (p.residual ? 100 : 0);
  const int64_t pairs = 720 + 20 * pair_rounds * kt / 100 + (busy ? 290 : 0) + (p.residual ? 200 : 0);
  return here < pairs;
}

int product_few_tokens(const Product& p, int dev, cudaStream_t s) {
  if (p.dtype == JLA_DTYPE_E4M3) return p.gated ? pick<false, true, true>(p, dev, s) : pick<false, true, false>(p, dev, s);
  if (p.w_mn) return pick<true, false, false>(p, dev, s);
  return p.gated ? pick<false, false, true>(p, dev, s) : pick<false, false, false>(p, dev, s);
}

}  // namespace jla
