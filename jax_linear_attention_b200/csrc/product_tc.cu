// Matrix products of any number of tokens on pairs of CTAs (tcgen05.mma.cta_group::2), with the epilogue fused:
//
//   linear   y = act((x W^T) xs ws + bias) + residual      (z before the activation in float32 for a backward pass)
//   gated    h = act(g) u,  g = x Wg^T,  u = x Wu^T          (g and u in float32 for a backward pass)
//   dx       = dz W, or dg Wg + du Wu                        (W read with the contraction along its rows)
//   dW       = dz^T x, or two of them in one launch          (both operands with the contraction along their rows)
//
// Bound by the tensor cores. A persistent pair of CTAs takes tiles of 256 rows and BN columns (BN / 2 columns of each
// weight where gated): a warp fetches operand tiles of 128 bytes of contraction by TMA into a ring of 6 or 8 stages, one
// thread of the leading CTA issues the products, eight warps of each CTA take finished accumulators out of TMEM (32 rows a
// warp, a row a thread) through shared memory and TMA stores. Two sets of accumulators: the epilogue of one tile
// runs under the products of the next. (Contractions of more than kPartSteps steps are summed in parts: one set is the running
// part's, the other holds the sum of the parts.) A pair reads an operand byte from L2 half as often as two CTAs of 128 x BN would.
// Tiles of a last round that would leave more than half of the pairs idle are taken in halves (1003 x 2048 x 6144 f16, 96
// tiles on 74 pairs: 31 -> 27 us with silu; 700 x 2048 x 2048, 24 tiles: 19.5 -> 15.7 us).
//
// Measured on a B200, inputs from HBM, each launch by itself: 16384 x 4096 x 2048 bf16 163 us forward, 165 us dx, 177 us dW (128 tiles on 74 pairs; cuBLAS
// 178, 169, 168); gated 16384 x 2048 x 5632 bf16 460 us, 532 us with g and u kept; gated 5003 x 2048 x 5632 e4m3 81 us. In a row of
// steps the power limit adds up to a third. The tensor pipe is active 73 to 95 % of the time. A step of the contraction takes 512 cycles of the tensor core and as much of what an SM
// can read from L2 (64 bytes a cycle), so that neither waits for the other by much.
//
// Where the operands end inside a tile TMA reads zeros and its stores leave out what lies beyond. No load is multicast.
// Every wait is bounded: one that runs out records kStatusProduct, and the kernel lets its copies and products in flight
// finish, frees its TMEM and returns.
#include "overlap.cuh"
#include "product.cuh"
#include "profile.cuh"
#include "umma_pair.cuh"

namespace jla {
namespace {

using umma::smem_addr;

constexpr int kThreads = 384;  // warps: 0 loads, 1 products, 2 TMEM, 3 none, 4 .. 11 epilogue
constexpr int kEpilogueWarps = 8;
constexpr int kStagingWarp = 4096;  // a box of 32 rows x 128 bytes for each epilogue warp

struct Maps {
  CUtensorMap x[2], w[2], y[2], save[2];
  CUtensorMap w_half[2];  // the weights in boxes of half a tile's rows (K-major)
};

struct Params {
  int rows, features;           // of y
  int tiles_n, tiles_mn;        // tiles in a row of tiles, in one product
  int whole, pieces;            // tiles taken whole, and pieces in all: those and the halves of the others
  int kt0, kt;                  // steps of the contraction with the first pair of operands, and in all
  int part;                     // steps that are summed in one accumulator (kt where they are few enough)
  uint32_t idesc, idesc_half;
  int act, half, saves;
  const float *x_scale, *w_scale[2], *bias;
  const void* residual;
  int* status;
};

template <int BN> struct Shape {
  static constexpr int kStageBytes = 128 * 128 + BN / 2 * 128;  // a CTA's part of both operands
  static constexpr int kStages = BN == 256 ? 6 : 8;
  static constexpr int kSmem = kStages * kStageBytes + kEpilogueWarps * kStagingWarp + 1024;
};

// Tile `t` of one product: bands of 8 columns of tiles, row after row inside a band, so that the tiles in work at one time
// form a block whose operands stay in L2.
__device__ __forceinline__ void locate(const Params& p, int t, int& tm, int& tn) {
  constexpr int kBand = 8;
  const int tiles_m = p.tiles_mn / p.tiles_n;
  const int band = t / (kBand * tiles_m);
  const int left = p.tiles_n - band * kBand, width = left < kBand ? left : kBand;
  const int in = t - band * kBand * tiles_m;
  tm = in / width;
  tn = band * kBand + in % width;
}

// What a pair works on at a time: a whole tile, or the left or right half of one (in a last round of tiles that would leave
// more than half of the pairs idle; a step of half a tile takes 0.69 of the time of one of a whole tile).
struct Piece {
  int product, tm, tn, part;
  bool whole;
  template <int BN> __device__ __forceinline__ static Piece at(const Params& p, int i) {
    Piece q;
    q.whole = BN != 256 || i < p.whole;
    const int t = q.whole ? i : p.whole + (i - p.whole) / 2;
    q.part = q.whole ? 0 : (i - p.whole) % 2;
    q.product = t / p.tiles_mn;
    locate(p, t - q.product * p.tiles_mn, q.tm, q.tn);
    return q;
  }
};

// A warp's staging box: 32 rows of 128 bytes, 128-byte swizzle (16-byte chunk j of row r lies at chunk j ^ (r % 8)).
struct Staging {
  uint32_t base;
  __device__ __forceinline__ uint32_t acquire(int lane) {
    if (lane == 0) tma::store_wait_read<0>();
    __syncwarp();
    return base;
  }
  static __device__ __forceinline__ void put(uint32_t box, int lane, int chunk, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(box + lane * 128 + ((chunk ^ (lane & 7)) << 4)), "r"(a),
                 "r"(b), "r"(c), "r"(d)
                 : "memory");
  }
  static __device__ __forceinline__ void release(uint32_t box, int lane, const CUtensorMap* map, int col, int row, int cols,
                                                 int rows) {
    umma::fence_async_smem();
    __syncwarp();
    if (lane == 0) {
      if (col < cols && row < rows) tma::store_2d(map, box, col, row);
      tma::store_commit();
    }
  }
  __device__ __forceinline__ void save32(const float (&v)[32], int lane, const CUtensorMap* map, int col, int row, int cols,
                                         int rows) {
    const uint32_t box = acquire(lane);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      put(box, lane, j, __float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]), __float_as_uint(v[4 * j + 2]),
          __float_as_uint(v[4 * j + 3]));
    }
    release(box, lane, map, col, row, cols, rows);
  }
  __device__ __forceinline__ void store64(const uint32_t (&v)[32], int lane, const CUtensorMap* map, int col, int row,
                                          int cols, int rows) {
    const uint32_t box = acquire(lane);
#pragma unroll
    for (int j = 0; j < 8; ++j) put(box, lane, j, v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
    release(box, lane, map, col, row, cols, rows);
  }
};

// A float for each of 64 columns from `col` on, two a lane (columns lane and 32 + lane): read before they are needed, handed
// to all lanes by shuffles. (Every lane reading all columns' values when it needs them left the epilogue waiting on them
// for three quarters of a tile's time.)
struct Columns {
  float v[2];
  __device__ __forceinline__ void read(const float* p, int col, int lane, int cols) {
#pragma unroll
    for (int h = 0; h < 2; ++h) v[h] = p && col + 32 * h + lane < cols ? *(p + col + 32 * h + lane) : 0.f;
  }
  __device__ __forceinline__ float at(int h, int i) const { return __shfl_sync(0xffffffffu, v[h], i); }
};

template <int BN, bool X_MN, bool W_MN, bool FP8, bool GATED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
product_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
  using S = Shape<BN>;
  constexpr int ST = S::kStages;
  extern __shared__ unsigned char smem_dyn[];
  __shared__ __align__(8) uint64_t full[ST], empty[ST], acc_full[2], acc_empty[2], drain;
  __shared__ uint32_t tmem_slot;
  const uint32_t base = (smem_addr(smem_dyn) + 1023) & ~1023u;
  const uint32_t staging = base + ST * S::kStageBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = umma::cluster_rank();
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      umma::mbar_init(full + i, 1);
      umma::mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      umma::mbar_init(acc_full + i, 1);
      umma::mbar_init(acc_empty + i, 2 * kEpilogueWarps);  // the epilogue warps of both CTAs
    }
    umma::mbar_init(&drain, 1);
    umma::mbar_init_fence();
  }
  if (warp == 2) umma::tmem_alloc_pair(&tmem_slot, 2 * BN);
  umma::fence_before_sync();
  umma::cluster_sync();
  umma::fence_after_sync();
  const uint32_t tmem = tmem_slot;
  bool ok = true;
  start_next();
  wait_for_previous();

  if (warp == 0) {
    // ---- loads: this CTA's 128 rows of x and its half of the weight's; the bytes count on the leader's barrier
    if (lane == 0) {
      tma::prefetch_map(&maps.x[0]);
      tma::prefetch_map(&maps.w[GATED ? rank : 0]);
    }
    const uint32_t bars = umma::map_rank(smem_addr(full), 0), mine = smem_addr(full), freed = smem_addr(empty);
    int s = 0, issued = 0;
    uint32_t phase = 1;  // (a fresh barrier's phase before the first counts as complete)
    for (int i = first; i < p.pieces && ok; i += step) {
      const Piece q = Piece::at<BN>(p, i);
      const int m0 = q.tm * 256 + (int)rank * 128;
      const int wide = q.whole ? BN / 2 : BN / 4;  // this CTA's rows of the weight (of one of them where gated)
      const int n0 = q.tn * (GATED ? BN / 2 : BN) + (GATED ? q.part : 2 * q.part + (int)rank) * wide;
      const CUtensorMap* mx = &maps.x[q.product];
      const CUtensorMap* ws_of = q.whole || W_MN ? maps.w : maps.w_half;
      const CUtensorMap* mw = ws_of + (GATED ? rank : 0);
      int k0 = 0;
      for (int kt = 0; kt < p.kt; ++kt, k0 += FP8 ? 128 : 64) {
        if (kt == p.kt0) mx = &maps.x[1], mw = ws_of + 1, k0 = 0;  // the second pair of operands
        ok = umma::mbar_wait_warp(freed + 8 * s, phase);
        if (!ok) break;
        if (umma::elect_one()) {
          if (rank == 0) tma::expect_tx(mine + 8 * s, 2 * (128 * 128 + wide * 128));
          const uint32_t bar = bars + 8 * s, xs = base + s * S::kStageBytes, ws = xs + 128 * 128;
          if constexpr (X_MN) {
            tma::load_2d_pair(xs, mx, m0, k0, bar);
            tma::load_2d_pair(xs + 8192, mx, m0 + 64, k0, bar);
          } else {
            tma::load_2d_pair(xs, mx, k0, m0, bar);
          }
          if constexpr (W_MN) {
#pragma unroll
            for (int b = 0; b < BN / 128; ++b) {
              if (b * 64 < wide) tma::load_2d_pair(ws + b * 8192, mw, n0 + b * 64, k0, bar);
            }
          } else {
            tma::load_2d_pair(ws, mw, k0, n0, bar);
          }
        }
        __syncwarp();
        ++issued;
        if (++s == ST) s = 0, phase ^= 1;
      }
    }
    if (!ok && rank == 0) {  // let what was asked for land before the block's memory is given up
      for (int j = issued > ST ? issued - ST : 0; j < issued; ++j) umma::mbar_wait_warp(mine + 8 * (j % ST), (j / ST) & 1);
    }
  } else if (warp == 1 && rank == 0) {
    // ---- products
    const uint64_t x0 = umma::smem_desc(base, X_MN ? 8192 : 16, 1024);
    const uint64_t w0 = umma::smem_desc(base + 128 * 128, W_MN ? 8192 : 16, 1024);
    const uint32_t filled = smem_addr(full), acc_freed = smem_addr(acc_empty);
    const bool parts = p.part < p.kt;
    int s = 0, n = 0;
    uint32_t phase = 0;
    for (int i = first, k0 = 0; i < p.pieces && ok; ++n) {  // (a piece, or one part of its contraction)
      const int a = parts ? 0 : n & 1, k1 = k0 + p.part < p.kt ? k0 + p.part : p.kt;
      const uint32_t idesc = BN != 256 || i < p.whole ? p.idesc : p.idesc_half;
      ok = umma::mbar_wait_warp(acc_freed + 8 * a, ((parts ? n : n >> 1) & 1) ^ 1);
      umma::fence_after_sync();
      for (int kt = k0; kt < k1 && ok; ++kt) {
        ok = umma::mbar_wait_warp(filled + 8 * s, phase);
        if (!ok) break;
        umma::fence_after_sync();
        if (umma::elect_one()) {
          const uint32_t off = (uint32_t)(s * S::kStageBytes) >> 4;
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            umma::mma_pair<FP8>(tmem + a * BN, x0 + off + (X_MN ? ks * 128 : ks * 2), w0 + off + (W_MN ? ks * 128 : ks * 2),
                                idesc, kt > k0 || ks > 0);
          }
          umma::commit_pair(empty + s);
          if (kt == k1 - 1) umma::commit_pair(acc_full + a);
        }
        __syncwarp();
        if (++s == ST) s = 0, phase ^= 1;
      }
      k0 = k1;
      if (k1 == p.kt) k0 = 0, i += step;
    }
    if (!ok) {  // products in flight read both CTAs' shared memory: wait for them
      if (umma::elect_one()) umma::commit_pair(&drain);
      __syncwarp();
      umma::mbar_wait_warp(smem_addr(&drain), 0);
    }
  } else if (warp >= 4) {
    // ---- epilogue: a warp has the TMEM lanes (rows) 32 w .. 32 w + 31 of its CTA, and every other 64 columns. (Four warps
    // with all columns and two boxes each: 39 -> 49 us for 8192 x 512 x 2048 bf16 with silu and a residual.)
    const int w = warp & 3, odd = warp >= 8;
    Staging stage{staging + (uint32_t)(warp - 4) * kStagingWarp};
    const bool half = p.half;
    auto release_accumulator = [&](int a) {
      umma::fence_before_sync();
      __syncwarp();
      if (lane == 0) umma::arrive_cluster(umma::map_rank(smem_addr(acc_empty + a), 0));
    };
    // A long contraction: its parts come one after the other in the first accumulator, their sum is kept in the second, each
    // column by the warp that needs it in the end. (The products stand still while a part is taken over, which does not show: dW
    // of 65536 x 2048 x 2048 345 us with and without.)
    int joined = 0;
    auto join = [&](int cols, uint32_t sum) {
      for (int k0 = 0; k0 < p.kt; k0 += p.part, ++joined) {
        const bool here = umma::mbar_wait(acc_full, joined & 1);
        if (!__all_sync(0xffffffffu, here)) return false;
        umma::fence_after_sync();
#pragma unroll 1
        for (int c = odd * 64; c < cols; c += 128) {
#pragma unroll 1
          for (int h = 0; h < (GATED ? 8 : 4); ++h) {
            const uint32_t at = sum + c + 16 * (h & 3) + (h > 3 ? cols : 0);
            umma::join_x16(at, at - BN, k0 == 0);
          }
        }
        umma::wait_st();
        release_accumulator(0);
      }
      return true;
    };
    const bool parts = p.part < p.kt;
    int n = 0;
    for (int i = first; i < p.pieces; i += step, ++n) {
      const int a = parts ? 1 : n & 1;
      const Piece q = Piece::at<BN>(p, i);
      const int row0 = q.tm * 256 + (int)rank * 128 + w * 32, row = row0 + lane;
      const bool live = row < p.rows;
      const uint32_t acc = tmem + a * BN + ((uint32_t)(32 * w) << 16);
      const int cols = (GATED ? BN / 2 : BN) / (q.whole ? 1 : 2);  // of y in this piece, from column col0 on
      const int col0 = q.tn * (GATED ? BN / 2 : BN) + q.part * cols;
      if (parts && !join(cols, acc)) {
        ok = false;
        break;
      }
      Columns bias, scale0, scale1;
      auto read_columns = [&](int col) {
        if constexpr (!GATED) bias.read(p.bias, col, lane, p.features);
        if constexpr (FP8) scale0.read(p.w_scale[0], col, lane, p.features);
        if constexpr (FP8 && GATED) scale1.read(p.w_scale[1], col, lane, p.features);
      };
      read_columns(odd * 64 < cols ? col0 + odd * 64 : p.features);
      uint4 res[GATED ? 1 : 8];
      auto read_residual = [&](int col) {
        if constexpr (!GATED) {
          const uint4* r = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.residual) + (size_t)row * p.features + col);
#pragma unroll
          for (int j = 0; j < 8; ++j) res[j] = live && col + 8 * j < p.features ? *(r + j) : make_uint4(0, 0, 0, 0);
        }
      };
      if (!GATED && p.residual && odd * 64 < cols) read_residual(col0 + odd * 64);
      float xs = 1.f;
      if constexpr (FP8) xs = live ? *(p.x_scale + row) : 0.f;
      if (!parts) ok = umma::mbar_wait(acc_full + a, (n >> 1) & 1);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      umma::fence_after_sync();
#pragma unroll 1
      for (int c = odd * 64; c < cols; c += 128) {
        const int col = col0 + c;
        if (col >= p.features || row0 >= p.rows) break;
        const Columns b = bias, s0 = scale0, s1 = scale1;
        read_columns(c + 128 < cols ? col + 128 : p.features);
        uint32_t out[32];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int hc = col + 32 * h;
          float v[32];
          umma::ld_32x32b_x32(v, acc + c + 32 * h);
          if constexpr (GATED) {
            float u[32];
            umma::ld_32x32b_x32(u, acc + cols + c + 32 * h);
            umma::wait_ld();
            if constexpr (FP8) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] *= xs * s0.at(h, i), u[i] *= xs * s1.at(h, i);
            }
            if (p.saves) {
              stage.save32(v, lane, &maps.save[0], hc, row0, p.features, p.rows);
              stage.save32(u, lane, &maps.save[1], hc, row0, p.features, p.rows);
            }
            with_activation(p.act, [&](auto act) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = activate<act()>(v[i]) * u[i];
            });
          } else {
            umma::wait_ld();
            if constexpr (FP8) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] *= xs * s0.at(h, i);
            }
            if (p.bias) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] += b.at(h, i);
            }
            if (p.saves) stage.save32(v, lane, &maps.save[0], hc, row0, p.features, p.rows);
            with_activation(p.act, [&](auto act) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = activate<act()>(v[i]);
            });
            if (p.residual) {
              with_half(half, [&](auto is_half) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const uint4 q = res[4 * h + j];
                  const uint32_t e[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    const float2 f = unpack_out<is_half()>(e[i]);
                    v[8 * j + 2 * i] += f.x, v[8 * j + 2 * i + 1] += f.y;
                  }
                }
              });
            }
          }
          with_half(half, [&](auto is_half) {
#pragma unroll
            for (int i = 0; i < 16; ++i) out[16 * h + i] = pack_out<is_half()>(v[2 * i], v[2 * i + 1]);
          });
        }
        if (!GATED && p.residual && c + 128 < cols) read_residual(col + 128);
        stage.store64(out, lane, &maps.y[q.product], col, row0, p.features, p.rows);
      }
      if (!parts) release_accumulator(a);
    }
    if (lane == 0) tma::store_wait<0>();
  }
  if (!ok) atomicExch(p.status, kStatusProduct);
  __syncthreads();
  umma::fence_before_sync();
  umma::cluster_sync();  // no product or arrival of the other CTA may still be on its way here
  umma::fence_after_sync();
  if (warp == 2) umma::tmem_dealloc_pair(tmem, 2 * BN);
}

template <int BN, bool X_MN, bool W_MN, bool FP8, bool GATED>
int launch(const Product& p, int device, int sms, cudaStream_t s) {
  using S = Shape<BN>;
  Maps maps;
  Params q{};
  const int esz = FP8 ? 1 : 2, kb = FP8 ? 128 : 64;
  const int xr = X_MN ? 64 : 128, wr = W_MN ? 64 : BN / 2;
  constexpr int COLS = GATED ? BN / 2 : BN;
  q.rows = (int)p.rows, q.features = p.features;
  q.tiles_n = (p.features + COLS - 1) / COLS;
  q.tiles_mn = (int)((p.rows + 255) / 256) * q.tiles_n;
  const int tiles = q.tiles_mn * (p.group ? 2 : 1), rest = tiles % (sms / 2);
  const bool halves = BN == 256 && rest > 0 && 2 * rest <= sms / 2;
  q.whole = halves ? tiles - rest : tiles;
  q.pieces = halves ? tiles + rest : tiles;
  bool ok = true;
  for (int i = 0; i < 2 && ok; ++i) {  // (a second operand or output that is not there is not asked for either)
    ok = (!p.x[i] || (X_MN ? tma::encode_2d(&maps.x[i], p.x[i], esz, p.rows, p.depth, p.x_stride, xr)
                           : tma::encode_2d(&maps.x[i], p.x[i], esz, p.depth, p.rows, p.x_stride, xr))) &&
         (!p.w[i] || (W_MN ? tma::encode_2d(&maps.w[i], p.w[i], esz, p.features, p.depth, p.w_stride, wr)
                           : tma::encode_2d(&maps.w[i], p.w[i], esz, p.depth, p.features, p.w_stride, wr))) &&
         (!p.w[i] || W_MN || !halves || tma::encode_2d(&maps.w_half[i], p.w[i], esz, p.depth, p.features, p.w_stride, BN / 4)) &&
         (!p.y[i] || tma::encode_2d(&maps.y[i], p.y[i], 2, p.features, p.rows, p.features, 32)) &&
         (!p.save[i] || tma::encode_2d(&maps.save[i], p.save[i], 4, p.features, p.rows, p.features, 32));
  }
  if (!ok) return JLA_ERR_CUDA;
  q.kt0 = (p.depth + kb - 1) / kb;
  q.kt = q.kt0 * (p.pair ? 2 : 1);
  const int parts = (q.kt + kPartSteps - 1) / kPartSteps;
  q.part = (q.kt + parts - 1) / parts;  // (equal ones, but for the last)
  q.idesc = FP8 ? umma::instr_desc_e4m3(256, BN) : umma::instr_desc(256, BN, p.dtype == JLA_DTYPE_BF16, X_MN, W_MN);
  q.idesc_half = FP8 ? umma::instr_desc_e4m3(256, BN / 2)
                     : umma::instr_desc(256, BN / 2, p.dtype == JLA_DTYPE_BF16, X_MN, W_MN);
  q.act = p.act, q.half = p.out_dtype == JLA_DTYPE_F16, q.saves = p.save[0] != nullptr;
  q.x_scale = p.x_scale, q.w_scale[0] = p.w_scale[0], q.w_scale[1] = p.w_scale[1], q.bias = p.bias, q.residual = p.residual;
  q.status = tc_status_ptr();
  if (!q.status) {
    set_error("the status word of the current device could not be located");
    return JLA_ERR_CUDA;
  }
  auto* kern = product_kernel<BN, X_MN, W_MN, FP8, GATED>;
  static std::atomic<uint64_t> allowed{0};
  JLA_CUDA_OK(allow_smem(kern, S::kSmem, device, allowed));
  const int pairs = sms / 2 < q.pieces ? sms / 2 : q.pieces;
  ProfScope scope(kProfProduct, s);
  JLA_CUDA_OK(launch_overlapped(kern, dim3(2 * pairs), dim3(kThreads), S::kSmem, s, 0, maps, q));  // (the kernel has its cluster size)
  return JLA_OK;
}

// A step of a tile of 128 columns takes two thirds of the time of one of 256 (4096 x 2048 x 2048 bf16: 38 us against 29): the
// narrow tiles are for products of up to 128 columns.
bool narrow(const Product& p) { return p.features * (p.gated ? 2 : 1) <= 128; }

template <bool X_MN, bool W_MN, bool FP8, bool GATED>
int pick(const Product& p, int dev, int sms, cudaStream_t s) {
  return narrow(p) ? launch<128, X_MN, W_MN, FP8, GATED>(p, dev, sms, s)
                   : launch<256, X_MN, W_MN, FP8, GATED>(p, dev, sms, s);
}

}  // namespace

int product_pairs(const Product& p, int dev, int sms, cudaStream_t s) {
  if (p.dtype == JLA_DTYPE_E4M3) return p.gated ? pick<false, false, true, true>(p, dev, sms, s) : pick<false, false, true, false>(p, dev, sms, s);
  if (p.x_mn) return pick<true, true, false, false>(p, dev, sms, s);
  if (p.w_mn) return pick<false, true, false, false>(p, dev, sms, s);
  return p.gated ? pick<false, false, false, true>(p, dev, sms, s) : pick<false, false, false, false>(p, dev, sms, s);
}

}  // namespace jla
