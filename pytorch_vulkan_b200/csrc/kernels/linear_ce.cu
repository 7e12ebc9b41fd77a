// Softmax cross entropy of a linear layer over a large vocabulary, z = x w^T + b,
// and its gradients.
//
//   lse_i = log sum_j exp z_ij      loss_i = lse_i - (1 - s) z_i,t(i) - s / V sum_j z_ij
//   G_ij  = g_i (exp(z_ij - lse_i) - (1 - s) [j = t(i)] - s / V)
//   dx = G w     dw = G^T x     db = sum_i G_i
//
// Forward: one matrix product whose epilogue keeps, per row and 64
// columns, the largest logit, the sum of exp(z - largest) and the target's
// logit; a second launch joins them.  For a backward pass it also writes what
// that needs of the first `kept` entries: the exponentials as 16-bit codes, for
// fp32 operands the logits themselves (as the caller has memory for them).
// Backward: per piece of the vocabulary, G in 16 bits (piece x tokens, sized to
// stay near the L2 cache), from what was kept or from logits that are formed
// again; two products make dx += G w and the piece's rows of dw = G^T x.  Going
// by pieces of the vocabulary finishes dw in one go and adds dx up in fp32: 6 N
// V D operations in all from what was kept, 8 without it, when nothing of the
// size N x V exists.
//
// Operands are 16-bit (tcgen05 kind::f16, fp32 accumulators).  fp32 operands
// are split into two fp16 numbers each, x = x0 + x1 (11 bits apiece), of which
// three products are formed: x0 w0, x0 w1 and x1 w0.  What is left out is, in
// the mean, 2^-24 of |x||w| (3 2^-22 at most), as much as rounding the product
// to fp32 would cost; three bf16 parts, which need no scaling, took six
// products for the same (1.88 ms a step of N 2048, D 768, V 32768, where these
// took 1.34 then and 1.08 now).  fp16's range is met by a power of two for each
// tensor that brings its largest finite magnitude to 2^14 .. 2^15; parts below
// 2^-39 of that are lost.
//
// G is rounded to what the products take: bf16 or fp16 for such operands, which
// puts a gradient 2.3e-3 (bf16, N 4095, D 1000, V 49999) from its value where
// rounding it alone makes 1.7e-3, and saves half of both products against two
// parts; two fp16 parts for fp32 operands.  db is summed from the same numbers.
// G is formed without the factor that all rows share and, in fp16, times 2^15
// (steps of 2^-39 are the least); both are undone on the fp32 results.  Where
// each row has a gradient g_i of its own, dx multiplies its rows by g_i at the
// end, so that a row's errors are relative to itself, and what is not finite in
// one reaches no other; dw and db, sums over rows, take a second G, of g_i /
// max|g| (8192 x 4096 -> 32768 bf16: 5.4 ms as with one G from what was kept,
// 8.5 and 7.0 ms with nothing kept; 4095 x 1000 -> 49999: 1.46 and 1.27, 1.90 and
// 1.59).
#include <algorithm>
#include "tc_common.cuh"
#include "types.cuh"

namespace pvb2 {

constexpr int kLBM = 256;  // rows of a tile: 128 for each CTA of a pair
constexpr int kLBK = 64;
// Warps: three issue loads, one the products, the others run the epilogue.  12
// or 20 in all: an SM's four schedulers hold 16384 registers each, and one more
// warp would cost the others a quarter of theirs.
constexpr int kLProducers = 3, kLMmaWarp = 3;

// A slot of the ring holds a K block of one plane of each operand: this CTA's
// 128 rows of A and BN / 2 columns of B.  An epilogue warp takes 32 rows and 64
// columns: 16 of them for 256 columns (with 8, two for each scheduler, an
// epilogue of exponentials took twice as long as the products of a K of 1000).
template <int P, int BN>
struct LceSmem {
  static constexpr int EPI_WARPS = BN / 16;
  static constexpr int THREADS = (kLProducers + 1 + EPI_WARPS) * 32;
  static constexpr int COLS = 64;
  static constexpr int A_BYTES = 128 * kLBK * 2;
  static constexpr int B_BYTES = BN / 2 * kLBK * 2;
  static constexpr int SLOT_BYTES = A_BYTES + B_BYTES;
  static constexpr int SLOTS = (224 * 1024 - EPI_WARPS * 4096) / SLOT_BYTES;
  static constexpr int EPI_OFF = SLOTS * SLOT_BYTES;  // one 4 KB store box per epilogue warp
  static constexpr int BAR_OFF = EPI_OFF + EPI_WARPS * 4096;
  static constexpr int TOTAL = BAR_OFF + (2 * SLOTS + 4) * 8 + 16;
};

// Kept exponentials, in [0, 1] relative to the largest of 64 columns, as 16-bit
// numbers of their own: no sign, 4 bits of exponent (bias 15), 12 of mantissa.
// Half a step is 2^-13 of the value down to 2^-14, and 2^-27 below; fp16 would
// spend a bit on the sign and one on exponents that are not needed, and its
// 2^-11 would add to the gradients' own rounding.  The bits are a float's with
// the exponent shifted by 112.
__device__ __forceinline__ uint32_t keep_code(float e) {
  const uint32_t b = __float_as_uint(e * 1.925929944387235853055977942584927e-34f);  // 2^-112
  return (b + 0x3ffu + ((b >> 11) & 1u)) >> 11;
}
// the number times 2^-112
__device__ __forceinline__ float keep_bits(uint32_t code) { return __uint_as_float(code << 11); }
constexpr float k2p112 = 5192296858534827628530496329220096.f;

enum { kEpiStats = 0, kEpiGrad = 1, kEpiAcc = 2, kEpiOut = 3 };

// what a gradient's fp32 sums are multiplied by, on the device: a power of two
// (fp16's scales), and one number for each row (own) or for all (common)
struct LceScale {
  const float *unit, *common, *own;
};

struct LceGemm {
  int M, N, K;
  int b_row0;             // where B's rows (K-major) or K rows (MN-major) begin in its map
  int n_fast, group;      // tile order: columns (else rows) fastest, `group` of them at a time
  int splits, kb_per;     // kEpiAcc: split s takes k blocks [s kb_per, (s + 1) kb_per) into slab s
  // epilogues of logits: column n is vocabulary entry v0 + n
  int v0;
  const void* bias;
  int bias_dtype;
  const int64_t* target;
  int64_t V, ignore;
  float smoothing;
  float2* part;           // kEpiStats: [64-column groups][part_ld]
  float* zsum;            // kEpiStats with smoothing: sums of z, laid out as part
  float* ztarget;
  int64_t part_ld;
  int keep;               // kEpiStats: entries (of the whole vocabulary) below this one are kept
  float* keep_max;        // what their exponentials are relative to: [64-column groups][keep_ld]
  int64_t keep_ld;
  const float* lse;       // kEpiGrad
  const float* grow;      // kEpiGrad: the rows' factors (0 for rows without a loss)
  const float* zscale;    // two factors of the logits, on the device, for split operands
  float gscale;
  // kEpiAcc / kEpiOut
  int accumulate;         // kEpiAcc: add to the slab
  void* out;              // kEpiOut without a tensor map
  int64_t out_ld;
  int out_dtype, out_tma;
  LceScale out_scale;     // kEpiOut
};

// the bias of 64 columns added to a row's logits: each lane fetches two, all
// lanes take them in turn
__device__ __forceinline__ void lce_add_bias(const LceGemm& p, int n0, int lane, float* v) {
  const float b0 = n0 + lane < p.N ? load_as<float>(p.bias, p.v0 + n0 + lane, p.bias_dtype) : 0.f;
  const float b1 = n0 + 32 + lane < p.N ? load_as<float>(p.bias, p.v0 + n0 + 32 + lane, p.bias_dtype) : 0.f;
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    v[j] += __shfl_sync(0xffffffffu, b0, j);
    v[32 + j] += __shfl_sync(0xffffffffu, b1, j);
  }
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// exp(x) for x <= 0: 2 ulp of expf where the operands are fp32, the exponent
// unit's own 2^-22 where they have 16 bits
template <bool PRECISE>
__device__ __forceinline__ float lce_exp(float x) {
  return PRECISE ? expf(x) : ex2(x * 1.4426950408889634f);
}

__device__ __forceinline__ bool lce_scored(int64_t t, int64_t V, int64_t ignore) {
  return t != ignore && t >= 0 && t < V;
}

// 64 columns of a row as 16-bit numbers into the warp's box (32 rows x 128 B,
// 128-byte swizzle)
template <typename T>
__device__ __forceinline__ void box16(uint8_t* box, int lane, const float* v) {
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    union {
      uint4 u;
      T e[8];
    } w;
    w.u = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int k = 0; k < 8; ++k) w.e[k] = from_f32<T>(v[8 * q + k]);
    *reinterpret_cast<uint4*>(box + lane * 128 + ((q ^ (lane & 7)) * 16)) = w.u;
  }
}

__device__ __forceinline__ void box_codes(uint8_t* box, int lane, const float* v) {
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = keep_code(v[8 * q + 2 * k]) | keep_code(v[8 * q + 2 * k + 1]) << 16;
    *reinterpret_cast<uint4*>(box + lane * 128 + ((q ^ (lane & 7)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

__device__ __forceinline__ void box32(uint8_t* box, int lane, const float* v) {
#pragma unroll
  for (int q = 0; q < 8; ++q)
    *reinterpret_cast<float4*>(box + lane * 128 + ((q ^ (lane & 7)) * 16)) =
        make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
}

template <typename F>
__device__ __forceinline__ void store_box(uint8_t* box, int lane, F fill_and_store) {
  if (lane == 0) bulk_wait_read<0>();  // the box's last store has read it
  __syncwarp();
  fill_and_store(0);
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    fill_and_store(1);
    bulk_commit();
  }
}

// the two factors that undo the scales of x and w on a logit: their product and
// 1, unless that is beyond fp32
__device__ __forceinline__ float2 lce_unscale(const float* scales) {
  if (!scales) return make_float2(1.f, 1.f);
  const float a = scales[0], b = scales[1], both = a * b;
  return both >= 1e-37f && both <= 1e37f ? make_float2(both, 1.f) : make_float2(a, b);
}

// the same for a row of a gradient.  Where the product of the two is beyond
// fp32's normal numbers, the one that keeps the sum in the middle comes first:
// the larger where the product is too small, the smaller where it is too large.
__device__ __forceinline__ float2 lce_row_scale(const LceScale& p, int64_t row) {
  const float a = *p.unit, b = p.own ? p.own[row] : *p.common, both = a * b, size = fabsf(both);
  if (size >= 1e-37f && size <= 1e37f) return make_float2(both, 1.f);
  const bool a_first = size < 1e-37f ? a >= fabsf(b) : a <= fabsf(b);
  return a_first ? make_float2(a, b) : make_float2(b, a);
}

// One tile: C[256 x BN] by a pair of CTAs, in two accumulators in turn.  With
// CHUNK = 0 an accumulator takes the whole of K.  With CHUNK > 0 it takes CHUNK
// blocks of K and the epilogue adds the chunks in registers: the tensor core
// cuts rather than rounds when it adds to an accumulator, so that a sum over
// thousands of products drifts by 2^-24 of itself for every 16 of them.  Of
// split operands each K block's lesser products come first, so that in a
// chunk's first block only the main one's additions are cut at its size.
template <int EPI, typename T, int P, int BN, int CHUNK>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__((LceSmem<P, BN>::THREADS), 1)
    lce_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmC, const __grid_constant__ LceGemm p, int a_mn, int b_mn) {
  using L = LceSmem<P, BN>;
  constexpr bool kPrecise = P > 1;
  constexpr int kCols = L::COLS;            // columns of an epilogue warp
  constexpr int kSlots = L::SLOTS;
  static_assert(CHUNK || P == 1, "split operands are summed in chunks");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = (uint64_t*)(smem + L::BAR_OFF);  // waited on in the even CTA
  uint64_t* empty = full + kSlots;
  uint64_t* acc_full = empty + kSlots;
  uint64_t* acc_empty = acc_full + 2;               // waited on in the even CTA
  uint32_t* tmem_slot = (uint32_t*)(acc_empty + 2);
  volatile int* abort = (volatile int*)(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank();
  const int tiles_m = (p.M + kLBM - 1) / kLBM, tiles_n = (p.N + BN - 1) / BN;
  const int base_tiles = tiles_m * tiles_n, total_tiles = base_tiles * p.splits;
  const int kblocks = (p.K + kLBK - 1) / kLBK;
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * L::EPI_WARPS);
    }
    *abort = 0;
    fence_barrier_init();
  }
  if (warp == kLMmaWarp) tmem_alloc_pair(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers exist before either is signalled
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // tile -> block row, block column, first and last block of K
  auto place = [&](int tile, int& mb, int& nb, int& sp, int& kb0, int& kb1) {
    sp = tile / base_tiles;
    const int t = tile % base_tiles;
    const int fast = p.n_fast ? tiles_n : tiles_m, slow = p.n_fast ? tiles_m : tiles_n;
    const int first = t / (p.group * slow) * p.group, wide = min(p.group, fast - first);
    const int r = t - first * slow, f = first + r % wide, q = r / wide;
    mb = p.n_fast ? q : f;
    nb = p.n_fast ? f : q;
    kb0 = sp * p.kb_per;
    kb1 = min(kblocks, kb0 + p.kb_per);
  };

  if (warp < kLProducers) {
    // ------------------------------------------------- loads: slot s by warp s % kLProducers
    if (lane == 0) {
      tma_prefetch(&tmA);
      tma_prefetch(&tmB);
      uint32_t it = 0;
      for (int tile = pair; tile < total_tiles && !*abort; tile += pairs) {
        int mb, nb, sp, kb0, kb1;
        place(tile, mb, nb, sp, kb0, kb1);
        const int am = mb * kLBM + rank * 128, bn = nb * BN + rank * (BN / 2);
        for (int kb = kb0; kb < kb1; ++kb) {
#pragma unroll
          for (int z = 0; z < P; ++z, ++it) {
            const int s = it % kSlots;
            if (s % kLProducers != warp) continue;
            if (!mbar_wait(&empty[s], ((it / kSlots) & 1) ^ 1, abort)) break;
            uint8_t* sa = smem + s * L::SLOT_BYTES;
            uint8_t* sb = sa + L::A_BYTES;
            const uint32_t bar = even_cta_addr(&full[s]);
            if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * L::SLOT_BYTES);
            if (!a_mn) {
              tma_load_3d_pair(sa, &tmA, bar, kb * kLBK, am, z);
            } else {
#pragma unroll
              for (int q = 0; q < 2; ++q)
                tma_load_3d_pair(sa + q * 8192, &tmA, bar, am + 64 * q, kb * kLBK, z);
            }
            if (!b_mn) {
              tma_load_3d_pair(sb, &tmB, bar, kb * kLBK, p.b_row0 + bn, z);
            } else {
#pragma unroll
              for (int q = 0; q < BN / 128; ++q)
                tma_load_3d_pair(sb + q * 8192, &tmB, bar, bn + 64 * q, p.b_row0 + kb * kLBK, z);
            }
          }
        }
      }
    }
  } else if (warp == kLMmaWarp) {
    // ------------------------------------------------- products, by the even CTA for both
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = idesc_f16(kLBM, BN, !std::is_same<T, __half>::value, a_mn, b_mn);
      // One thread issues everything in order, so that what it computes between
      // two MMAs holds up the tensor core: the descriptors are formed once, and
      // a step along K or a slot is an addition to their address
      // (16-byte units, below 2^14).  Formed anew for each MMA they took it
      // longer than the MMA.
      const uint32_t smem0 = smem_u32(smem);
      const uint64_t a0 = a_mn ? desc_mnmajor16(smem0, 0, 8192) : desc_kmajor(smem0, 0);
      const uint64_t b0 = b_mn ? desc_mnmajor16(smem0 + L::A_BYTES, 0, 8192) : desc_kmajor(smem0 + L::A_BYTES, 0);
      const uint32_t a_step = a_mn ? 128u : 2u, b_step = b_mn ? 128u : 2u;
      uint32_t it = 0, chunk = 0;
      for (int tile = pair; tile < total_tiles && !*abort; tile += pairs) {
        int mb, nb, sp, kb0, kb1;
        place(tile, mb, nb, sp, kb0, kb1);
        for (int c0 = kb0; c0 < kb1; ++chunk) {
          const int c1 = CHUNK ? min(kb1, c0 + CHUNK) : kb1;
          const int buf = chunk & 1;
          if (!mbar_wait(&acc_empty[buf], ((chunk >> 1) & 1) ^ 1, abort)) break;
          tc_fence_after();
          const uint32_t d = tmem_base + buf * BN;
          // the product of plane slots sa (of A) and sb (of B); `fresh`: into an empty accumulator
          auto product = [&](int sa, int sb, bool fresh) {
            uint64_t ad = a0 + (uint32_t)(sa * (L::SLOT_BYTES / 16)), bd = b0 + (uint32_t)(sb * (L::SLOT_BYTES / 16));
#pragma unroll
            for (int kk = 0; kk < kLBK / 16; ++kk) {
              mma_f16_pair(d, ad, bd, idesc, fresh && kk == 0 ? 0u : 1u);
              ad += a_step;
              bd += b_step;
            }
          };
          bool ok = true;
          auto arrived = [&](uint32_t n) {
            ok = ok && mbar_wait(&full[n % kSlots], (n / kSlots) & 1, abort);
            tc_fence_after();
          };
          for (int kb = c0; kb < c1 && ok; ++kb, it += P) {
            // the lesser products first; a slot is released after its last one
            const int s0 = it % kSlots;
            arrived(it);
            if (P == 2) {
              const int s1 = (it + 1) % kSlots;
              arrived(it + 1);
              product(s1, s0, kb == c0);
              product(s0, s1, false);
              mma_commit_pair(&empty[s1]);
            }
            product(s0, s0, P == 1 && kb == c0);
            mma_commit_pair(&empty[s0]);
          }
          if (!ok) break;
          mma_commit_pair(&acc_full[buf]);
          c0 = c1;
        }
      }
    }
  } else if (warp > kLMmaWarp) {
    // ------------------------------------------------- epilogue: TMEM lane quarter warp % 4, 64 columns (warp - 4) / 4
    const int quarter = warp & 3, group = (warp - kLMmaWarp - 1) >> 2;
    uint8_t* box = smem + L::EPI_OFF + (warp - kLMmaWarp - 1) * 4096;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    uint32_t chunk = 0;
    for (int tile = pair; tile < total_tiles && !*abort; tile += pairs) {
      int mb, nb, sp, kb0, kb1;
      place(tile, mb, nb, sp, kb0, kb1);
      const int m0 = mb * kLBM + rank * 128 + quarter * 32, m = m0 + lane;
      const bool mrow = m < p.M;
      const int nh = nb * BN + group * kCols;  // first column of this warp
      int t = INT32_MIN;  // column of the row's target
      float row_lse = 0.f, row_g = 0.f;
      if (EPI == kEpiStats || EPI == kEpiGrad) {
        if (mrow) {
          const int64_t tt = p.target[m];
          if (lce_scored(tt, p.V, p.ignore)) t = (int)tt - p.v0;
          if (EPI == kEpiGrad) {
            row_lse = p.lse[m];
            row_g = p.grow[m];
          }
        }
      }
      const float2 unscale = lce_unscale(P == 2 ? p.zscale : nullptr);
      const float flat = EPI == kEpiGrad ? p.smoothing / (float)p.V : 0.f;
      const float2 oscale = EPI == kEpiOut && mrow ? lce_row_scale(p.out_scale, m) : make_float2(0.f, 0.f);
      float mx = -INFINITY, sum = 0.f, zs = 0.f;
      float v[64];
      bool ok = true;
      if (CHUNK > 0) {
#pragma unroll
        for (int j = 0; j < 64; ++j) v[j] = 0.f;
#pragma unroll 1
        for (int c0 = kb0; c0 < kb1 && ok; c0 += CHUNK, ++chunk) {
          const int buf = chunk & 1;
          ok = mbar_wait(&acc_full[buf], (chunk >> 1) & 1, abort);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            float u[16];
            tmem_ld16(tmem_base + lanes + buf * BN + group * kCols + 16 * h, u);
#pragma unroll
            for (int j = 0; j < 16; ++j) v[16 * h + j] += u[j];
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(even_cta_addr(&acc_empty[buf]));
        }
      } else {
        ok = mbar_wait(&acc_full[chunk & 1], (chunk >> 1) & 1, abort);
        tc_fence_after();
      }
      if (!ok) break;
      const int n0 = nh;
      if (n0 < p.N) {
        if (CHUNK == 0) {
          const uint32_t ta = tmem_base + lanes + (chunk & 1) * BN + group * kCols;
          tmem_ld32(ta, v);
          tmem_ld32(ta + 32, v + 32);
          // the accumulator is free: the values are in registers
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(even_cta_addr(&acc_empty[chunk & 1]));
        }
        if ((EPI == kEpiStats || EPI == kEpiGrad) && P == 2) {
#pragma unroll
          for (int j = 0; j < 64; ++j) v[j] = v[j] * unscale.x * unscale.y;
        }
        // whether any of the warp's targets is among these columns
        const bool has_target = (EPI == kEpiStats || EPI == kEpiGrad) &&
                                __any_sync(0xffffffffu, t >= n0 && t < n0 + 64);
        if ((EPI == kEpiStats || EPI == kEpiGrad) && p.bias) lce_add_bias(p, n0, lane, v);
        if (EPI == kEpiStats) {
          if (n0 + 64 > p.N) {
#pragma unroll
            for (int j = 0; j < 64; ++j) {
              if (p.zsum && n0 + j < p.N) zs += v[j];
              if (n0 + j >= p.N) v[j] = -INFINITY;
            }
          } else if (p.zsum) {
#pragma unroll
            for (int j = 0; j < 64; ++j) zs += v[j];
          }
          if (has_target) {
            float zt = 0.f;
#pragma unroll
            for (int j = 0; j < 64; ++j) zt = t == n0 + j ? v[j] : zt;
            if (t >= n0 && t < n0 + 64) p.ztarget[m] = zt;
          }
          const bool keep = p.v0 + n0 < p.keep;
          if (kPrecise && keep && m0 < p.M) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (p.v0 + n0 + 32 * h < p.keep)
                store_box(box, lane, [&](int phase) {
                  if (phase == 0) box32(box, lane, v + 32 * h);
                  else tma_store_3d(&tmC, box, p.v0 + n0 + 32 * h, m0, 0);
                });
          }
          mx = v[0];
#pragma unroll
          for (int j = 1; j < 64; ++j) mx = fmaxf(mx, v[j]);  // a NaN logit makes the sum NaN instead
          const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll
          for (int j = 0; j < 64; ++j) {
            v[j] = lce_exp<kPrecise>(v[j] - base);
            sum += v[j];
          }
          if (!kPrecise && keep && m0 < p.M) {
            // -inf where all 64 are masked, whose codes are 0: any finite number there could make the factor that the
            // backward pass forms of it, exp(maximum - lse), infinite
            if (mrow) p.keep_max[(int64_t)((p.v0 + n0) >> 6) * p.keep_ld + m] = mx;
            store_box(box, lane, [&](int phase) {
              if (phase == 0) box_codes(box, lane, v);
              else tma_store_3d(&tmC, box, p.v0 + n0, m0, 0);
            });
          }
        } else if (EPI == kEpiGrad) {
          const float scale = row_g * p.gscale;
#pragma unroll
          for (int j = 0; j < 64; ++j) v[j] = lce_exp<kPrecise>(v[j] - row_lse) - flat;
          if (has_target) {
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] -= t == n0 + j ? 1.f - p.smoothing : 0.f;
          }
#pragma unroll
          for (int j = 0; j < 64; ++j) v[j] *= scale;
          if (__any_sync(0xffffffffu, row_g == 0.f)) {
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] = row_g == 0.f ? 0.f : v[j];
          }
          if (m0 < p.M) {
            for (int z = 0; z < P; ++z) {
              store_box(box, lane, [&](int phase) {
                if (phase == 0) box16<T>(box, lane, v);
                else tma_store_3d(&tmC, box, n0, m0, z);
              });
              if (z + 1 < P) {
#pragma unroll
                for (int j = 0; j < 64; ++j) v[j] -= to_f32(from_f32<T>(v[j]));
              }
            }
          }
        } else if (EPI == kEpiAcc) {
          if (m0 < p.M) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (n0 + 32 * h < p.N)
                store_box(box, lane, [&](int phase) {
                  if (phase == 0) box32(box, lane, v + 32 * h);
                  else if (p.accumulate) tma_reduce_add_3d(&tmC, box, n0 + 32 * h, m0, sp);
                  else tma_store_3d(&tmC, box, n0 + 32 * h, m0, sp);
                });
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < 64; ++j) v[j] = v[j] * oscale.x * oscale.y;
          if (!p.out_tma) {
            // through the box, rotated by the row: lanes then write along rows
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float* f = reinterpret_cast<float*>(box);
#pragma unroll
              for (int j = 0; j < 32; ++j) f[lane * 32 + ((j + lane) & 31)] = v[32 * h + j];
              __syncwarp();
              const int n = n0 + 32 * h + lane;
              if (n < p.N)
                for (int r = 0; r < 32 && m0 + r < p.M; ++r)
                  store_as<float>(p.out, (int64_t)(m0 + r) * p.out_ld + n, p.out_dtype, f[r * 32 + ((lane + r) & 31)]);
              __syncwarp();
            }
          } else if (m0 < p.M) {
            if (p.out_dtype == PVB2_F32) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                if (n0 + 32 * h < p.N)
                  store_box(box, lane, [&](int phase) {
                    if (phase == 0) box32(box, lane, v + 32 * h);
                    else tma_store_3d(&tmC, box, n0 + 32 * h, m0, 0);
                  });
              }
            } else {
              store_box(box, lane, [&](int phase) {
                if (phase == 0) box16<T>(box, lane, v);
                else tma_store_3d(&tmC, box, n0, m0, 0);
              });
            }
          }
        }
      }
      if (EPI == kEpiStats && mrow && nh < p.N) {
        const int64_t at = (int64_t)(p.v0 / kCols + nh / kCols) * p.part_ld + m;
        p.part[at] = make_float2(mx, sum);
        if (p.zsum) p.zsum[at] = zs;
      }
      if (CHUNK == 0) {
        if (n0 >= p.N) {
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(even_cta_addr(&acc_empty[chunk & 1]));
        }
        ++chunk;
      }
    }
    if (lane == 0) bulk_wait_all();
  }
  // ------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  if (warp == kLMmaWarp && *abort) {
    // let any MMA still in flight finish before the columns are released
    const uint64_t t0 = globaltimer();
    while (globaltimer() - t0 < 10000000ull) {
    }
  }
  cluster_sync();  // neither CTA's shared memory goes while the other may signal it
  if (warp == kLMmaWarp) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ------------------------------------------------------------ small kernels
// src [rows][cols] (row stride ld) -> planes [P][rows][ldp] of T, columns
// from cols to ldp zero; rows without a loss become zeros when `target` is
// given (what they hold, NaN among it, then has no part in a product)
template <typename S>
struct LcePackJob {
  const S* src;
  int64_t rows, ld;
  uint16_t* dst;
  const int64_t* target;  // or NULL
  int vec;
};

// Scales of split operands.  One block's largest finite magnitudes of x (rows
// that have a loss) come first in `part`, then those of w; each block of a
// later launch reduces them anew.
constexpr int kLScaleBlocks = 296;  // of x's and w's together: two blocks of 1024 threads for each SM
struct LceScaleJob {
  const float* part;      // or NULL
  int nx, nw;
  float* scales;          // 1 / s_x and 1 / s_w, written by the first block
  const float* given;     // these two from the forward pass, or NULL
};

// 2^k that brings m to [2^14, 2^15) (k in [-113, 120]), 1 for 0
__device__ __forceinline__ float lce_pow2(float m) {
  const int e = (int)(__float_as_uint(m) >> 23) - 127;
  return m == 0.f ? 1.f : __uint_as_float((uint32_t)(127 + min(120, 14 - e)) << 23);
}

__global__ void __launch_bounds__(1024, 2)
    lce_absmax_kernel(const float* __restrict__ x, int64_t rows_x, int64_t ldx, const float* __restrict__ w,
                      int64_t rows_w, int64_t ldw, int64_t cols, const int64_t* __restrict__ target, int64_t V,
                      int64_t ignore, int nx, float* __restrict__ part) {
  const bool is_x = (int)blockIdx.x < nx;
  const float* src = is_x ? x : w;
  const int64_t rows = is_x ? rows_x : rows_w, ld = is_x ? ldx : ldw;
  const int64_t block = is_x ? blockIdx.x : blockIdx.x - nx, blocks = is_x ? nx : gridDim.x - nx;
  const bool vec = ((uintptr_t)src & 15) == 0 && ld % 4 == 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float m = 0.f;
  auto take = [&](float v) {
    v = fabsf(v);
    m = v <= 3.402823466e38f ? fmaxf(m, v) : m;  // neither infinity nor NaN
  };
  // a warp takes 512 columns of a row at a time
  const int64_t segs = (cols + 511) / 512;
  for (int64_t i = block * 32 + warp; i < rows * segs; i += blocks * 32) {
    const int64_t r = i <= INT32_MAX ? (int64_t)((uint32_t)i / (uint32_t)segs) : i / segs, c0 = (i - r * segs) * 512;
    if (is_x && !lce_scored(target[r], V, ignore)) continue;
    const float* row = src + r * ld;
    if (vec && c0 + 512 <= cols) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 v = *reinterpret_cast<const float4*>(row + c0 + q * 128 + lane * 4);
        take(v.x);
        take(v.y);
        take(v.z);
        take(v.w);
      }
    } else {
#pragma unroll 4
      for (int64_t c = c0 + lane; c < min(cols, c0 + 512); c += 32) take(row[c]);
    }
  }
  __shared__ float s[32];
  m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));
  if (lane == 0) s[warp] = m;
  __syncthreads();
  if (warp == 0) {
    m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(s[lane])));
    if (lane == 0) part[blockIdx.x] = m;
  }
}

// what each row's gradient is multiplied by, where that is one number for all
// rows (mean and sum): row[i] is 1, and own[i] that number, or both 0 where row i
// has no loss, whose dx is 0 under a gradient that is not finite too
struct LceRowsJob {
  float *row, *own;       // NULL: nothing to do
  float* factor;          // powers of two of db, dx (w's scale is in it) and dw (x's), and the number for all rows
  const float *grad_out, *count;
  const int64_t* target;
  int64_t N;
  int mean;
  float inv_gscale;
};

template <typename S, typename T>
__device__ __forceinline__ void lce_pack_one(const LcePackJob<S>& j, int64_t e, int per_row, int64_t cols, int64_t ldp,
                                             int planes, int64_t V, int64_t ignore, float scale) {
  const int64_t r = e <= INT32_MAX ? (int64_t)((int)e / per_row) : e / per_row;
  const int64_t c = (e - r * per_row) * 8, plane = j.rows * ldp;
  float v[8];
  if (j.vec && c + 8 <= cols) {
    load_vec<8>(j.src + r * j.ld + c, v);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = c + k < cols ? to_f32(j.src[r * j.ld + c + k]) : 0.f;
  }
  if (j.target && !lce_scored(j.target[r], V, ignore)) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = 0.f;
  }
  T* dst = reinterpret_cast<T*>(j.dst) + r * ldp + c;
  if (planes > 1) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] *= scale;
  }
  for (int z = 0; z < planes; ++z) {
    store_vec<8>(dst + z * plane, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      // infinity is its first part alone
      const float h = to_f32(from_f32<T>(v[k]));
      v[k] = isinf(h) ? 0.f : v[k] - h;
    }
  }
}

// one or two operands of the same row length (eight columns a thread), and
// the rows' factors with them
template <typename S, typename T>
__global__ void __launch_bounds__(256)
    lce_pack_kernel(LcePackJob<S> a, LcePackJob<S> b, LceRowsJob rj, LceScaleJob sj, int64_t cols, int64_t ldp,
                    int planes, int64_t V, int64_t ignore) {
  float sx = 1.f, sw = 1.f;  // of a and of b
  if (sj.given) {
    sx = 1.f / sj.given[0];  // powers of two
    sw = 1.f / sj.given[1];
  } else if (sj.part) {
    __shared__ float smax[2][8];
    float mx = 0.f, mw = 0.f;
    for (int q = threadIdx.x; q < sj.nx + sj.nw; q += 256) {
      const float m = sj.part[q];
      if (q < sj.nx) mx = fmaxf(mx, m);
      else mw = fmaxf(mw, m);
    }
    mx = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mx)));
    mw = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mw)));
    if ((threadIdx.x & 31) == 0) {
      smax[0][threadIdx.x >> 5] = mx;
      smax[1][threadIdx.x >> 5] = mw;
    }
    __syncthreads();
    for (int q = 0; q < 8; ++q) {
      mx = fmaxf(mx, smax[0][q]);
      mw = fmaxf(mw, smax[1][q]);
    }
    sx = lce_pow2(mx);
    sw = lce_pow2(mw);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      sj.scales[0] = 1.f / sx;
      sj.scales[1] = 1.f / sw;
    }
  }
  const int per_row = (int)(ldp / 8);
  const int64_t na = a.rows * per_row, total = na + b.rows * per_row;
  const int64_t first = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t e = first; e < total; e += step) {
    if (e < na) lce_pack_one<S, T>(a, e, per_row, cols, ldp, planes, V, ignore, sx);
    else lce_pack_one<S, T>(b, e - na, per_row, cols, ldp, planes, V, ignore, sw);
  }
  if (rj.row) {
    const float n = *rj.count, f = n > 0.f ? (rj.mean ? *rj.grad_out / n : *rj.grad_out) : 0.f;
    for (int64_t i = first; i < rj.N; i += step) {
      const bool scored = lce_scored(rj.target[i], V, ignore);
      rj.row[i] = scored ? 1.f : 0.f;
      rj.own[i] = scored ? f : 0.f;
    }
    if (first == 0) {
      rj.factor[0] = rj.inv_gscale;
      rj.factor[1] = rj.inv_gscale / sw;
      rj.factor[2] = rj.inv_gscale / sx;
      rj.factor[3] = f;
    }
  }
}

// joins the parts of each row: lse and loss (0 for rows without one).  32
// rows a block, 32 threads a row.
__global__ void __launch_bounds__(1024)
    lce_rows_kernel(const float2* __restrict__ part, const float* __restrict__ zsum, int64_t part_ld, int parts,
                    const float* __restrict__ ztarget, const int64_t* __restrict__ target, int64_t N, int64_t V,
                    int64_t ignore, float smoothing, float* __restrict__ lse, float* __restrict__ loss) {
  __shared__ float sm[32][33], ss[32][33], sz[32][33];
  const int r = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t i = (int64_t)blockIdx.x * 32 + r;
  float mx = -INFINITY, sum = 0.f, zs = 0.f;
  if (i < N) {
#pragma unroll 4
    for (int q = g; q < parts; q += 32) {
      const float2 v = part[q * part_ld + i];
      const float nm = fmaxf(mx, v.x), base = nm == -INFINITY ? 0.f : nm;
      sum = sum * expf(mx - base) + v.y * expf(v.x - base);
      mx = nm;
      if (zsum) zs += zsum[q * part_ld + i];
    }
  }
  sm[g][r] = mx;
  ss[g][r] = sum;
  sz[g][r] = zs;
  __syncthreads();
  // warp g takes row g, its lanes the 32 threads' shares
  mx = sm[r][g];
  sum = ss[r][g];
  zs = sz[r][g];
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, mx, o), os = __shfl_xor_sync(0xffffffffu, sum, o);
    const float nm = fmaxf(mx, om), base = nm == -INFINITY ? 0.f : nm;
    sum = sum * expf(mx - base) + os * expf(om - base);
    mx = nm;
    zs += __shfl_xor_sync(0xffffffffu, zs, o);
  }
  const int64_t row = (int64_t)blockIdx.x * 32 + g;
  if (r == 0 && row < N) {
    const float l = (mx == -INFINITY ? 0.f : mx) + logf(sum);
    lse[row] = l;
    float v = 0.f;
    if (lce_scored(target[row], V, ignore)) {
      v = l - ztarget[row];
      if (smoothing != 0.f) v = (1.f - smoothing) * v + smoothing * (l - zs / (float)V);
    }
    loss[row] = v;
  }
}

// the same for at most 8 rows, a warp each, with their total: the parts of a
// row are all on their way at once
__global__ void __launch_bounds__(256)
    lce_few_join_kernel(const float2* __restrict__ part, const float* __restrict__ zsum, int parts,
                        const float* __restrict__ ztarget, const int64_t* __restrict__ target, int N, int64_t V,
                        int64_t ignore, float smoothing, int reduction, float* __restrict__ lse,
                        float* __restrict__ loss, float* __restrict__ out, float* __restrict__ count) {
  __shared__ float sl[8];
  const int i = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (i < N) {
    float mx = -INFINITY, sum = 0.f, zs = 0.f;
    for (int q0 = 0; q0 < parts; q0 += 32 * 10) {
      float2 v[10];
#pragma unroll
      for (int k = 0; k < 10; ++k) {
        const int q = q0 + k * 32 + lane;
        v[k] = q < parts ? part[q * N + i] : make_float2(-INFINITY, 0.f);
        if (zsum && q < parts) zs += zsum[q * N + i];
      }
      float nm = mx;
#pragma unroll
      for (int k = 0; k < 10; ++k) nm = fmaxf(nm, v[k].x);
      const float base = nm == -INFINITY ? 0.f : nm;
      sum *= expf(mx - base);
#pragma unroll
      for (int k = 0; k < 10; ++k) sum += v[k].y * expf(v[k].x - base);
      mx = nm;
    }
    for (int o = 16; o > 0; o >>= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, mx, o), os = __shfl_xor_sync(0xffffffffu, sum, o);
      const float nm = fmaxf(mx, om), base = nm == -INFINITY ? 0.f : nm;
      sum = sum * expf(mx - base) + os * expf(om - base);
      mx = nm;
      zs += __shfl_xor_sync(0xffffffffu, zs, o);
    }
    if (lane == 0) {
      const float l = (mx == -INFINITY ? 0.f : mx) + logf(sum);
      lse[i] = l;
      float v = 0.f;
      if (lce_scored(target[i], V, ignore)) {
        v = l - ztarget[i];
        if (smoothing != 0.f) v = (1.f - smoothing) * v + smoothing * (l - zs / (float)V);
      }
      loss[i] = v;
      sl[i] = v;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double all = 0.0;
    int n = 0;
    for (int q = 0; q < N; ++q) {
      all += (double)sl[q];
      n += lce_scored(target[q], V, ignore) ? 1 : 0;
    }
    *count = (float)n;
    if (reduction != PVB2_LOSS_NONE) *out = (float)(reduction == PVB2_LOSS_MEAN ? all / (double)n : all);
  }
}

// the same from logits that lie in S partial sums [S][rows][ld]: one block a
// row
__device__ __forceinline__ float lce_slab_logit(const float* __restrict__ slab, int S, int64_t size, int64_t at,
                                                const void* bias, int64_t n, int bias_dtype, float2 zscale) {
  float z = slab[at];
  for (int s = 1; s < S; ++s) z += slab[s * size + at];
  z = z * zscale.x * zscale.y;
  return bias ? z + load_as<float>(bias, n, bias_dtype) : z;
}

__global__ void __launch_bounds__(512)
    lce_slab_rows_kernel(const float* __restrict__ slab, int S, int64_t rows, int64_t ld, const void* __restrict__ bias,
                         int bias_dtype, const int64_t* __restrict__ target, int64_t V, int64_t ignore, float smoothing,
                         float* __restrict__ lse, float* __restrict__ loss, float* __restrict__ kept, int64_t keep,
                         int64_t keep_ld, float* __restrict__ ztarget, const float* __restrict__ zscale) {
  __shared__ float sm[16], ss[16], sz[16], zt;
  const float2 unscale = lce_unscale(zscale);
  const int64_t i = blockIdx.x, t = target[i];
  const bool scored = lce_scored(t, V, ignore);
  float mx = -INFINITY, sum = 0.f, zs = 0.f;
  for (int64_t n = threadIdx.x; n < V; n += blockDim.x) {
    const float z = lce_slab_logit(slab, S, rows * ld, i * ld + n, bias, n, bias_dtype, unscale);
    if (n < keep) kept[i * keep_ld + n] = z;
    if (scored && n == t) zt = z;
    const float nm = fmaxf(mx, z), base = nm == -INFINITY ? 0.f : nm;
    sum = sum * expf(mx - base) + expf(z - base);
    mx = nm;
    zs += z;
  }
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, mx, o), os = __shfl_xor_sync(0xffffffffu, sum, o);
    const float nm = fmaxf(mx, om), base = nm == -INFINITY ? 0.f : nm;
    sum = sum * expf(mx - base) + os * expf(om - base);
    mx = nm;
    zs += __shfl_xor_sync(0xffffffffu, zs, o);
  }
  if ((threadIdx.x & 31) == 0) {
    sm[threadIdx.x >> 5] = mx;
    ss[threadIdx.x >> 5] = sum;
    sz[threadIdx.x >> 5] = zs;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int q = 1; q < (int)blockDim.x / 32; ++q) {
      const float nm = fmaxf(mx, sm[q]), base = nm == -INFINITY ? 0.f : nm;
      sum = sum * expf(mx - base) + ss[q] * expf(sm[q] - base);
      mx = nm;
      zs += sz[q];
    }
    const float l = (mx == -INFINITY ? 0.f : mx) + logf(sum);
    lse[i] = l;
    float v = 0.f;
    if (scored) {
      v = l - zt;
      if (smoothing != 0.f) v = (1.f - smoothing) * v + smoothing * (l - zs / (float)V);
      if (ztarget) ztarget[i] = zt;
    }
    loss[i] = v;
  }
}

// Few rows (a token or some while serving): a product with so few rows is a
// pass over w, bound by HBM, which 256-row tiles read at half the rate (their
// loads take 128 bytes of each of w's rows at a time, and as many of x's).
// Here a warp reads R of w's rows at once, each lane 16 bytes of each, and
// multiplies them by the NT rows of x from shared memory in fp32; its lanes
// then keep the running maximum and sum of their row of x.  One V = 32768, D =
// 2048 fp16 row: 30 us and 4 for the join, against 54 on tiles.  R fills the
// registers: four rows of w for one row of x in fp32 (V 32768, D 2048: 55 us, 75
// with eight), four for eight (87 us, 101 with two, where x's reads from shared
// memory bound it).
template <int L>
__device__ __forceinline__ float sum_spread(float (&a)[L], int lane) {
  // sums of L values over the warp, value i in the lanes i * 32 / L ..
  int o = 16;
#pragma unroll
  for (int n = L; n > 1; n /= 2, o /= 2) {
    const bool upper = lane & o;
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const float send = upper ? a[i] : a[i + n / 2];
      a[i] = (upper ? a[i + n / 2] : a[i]) + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  float s = a[0];
  for (; o > 0; o /= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

template <typename S, int NT, int R, bool VEC>
__global__ void __launch_bounds__(256, 2)
    lce_few_rows_kernel(const S* __restrict__ x, int64_t ldx, const S* __restrict__ w, int64_t ldw,
                        const S* __restrict__ bias, const int64_t* __restrict__ target, int N, int D, int V,
                        int64_t ignore, int smooth, float2* __restrict__ part, float* __restrict__ zsum,
                        float* __restrict__ ztarget, float* __restrict__ kept, int keep, int64_t keep_ld) {
  constexpr int L = R * NT;          // logits of a pass over R rows of w
  constexpr int kSpan = 32 / L;      // lanes that hold each
  extern __shared__ __align__(16) uint8_t few_smem[];
  S* xs = reinterpret_cast<S*>(few_smem);  // [NT][dp], zeros behind D and N
  __shared__ float sm[8][L], ss[8][L], sz[8][L];
  const int dp = (D + 7) / 8 * 8;
  for (int e = threadIdx.x; e < NT * dp; e += 256) {
    const int t = e / dp, c = e - t * dp;
    xs[e] = t < N && c < D ? x[t * ldx + c] : from_f32<S>(0.f);
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int my_r = lane / kSpan / NT, my_t = lane / kSpan % NT;  // the logit that this lane ends up with
  const int64_t goal = my_t < N ? target[my_t] : -1;
  const int t_col = my_t < N && lce_scored(goal, V, ignore) ? (int)goal : -1;
  float mx = -INFINITY, sum = 0.f, zs = 0.f;
  const int groups = (V + R - 1) / R;
  for (int q = blockIdx.x * 8 + warp; q < groups; q += gridDim.x * 8) {
    const int v0 = q * R;
    const S* rows[R];
#pragma unroll
    for (int r = 0; r < R; ++r) rows[r] = w + (int64_t)min(v0 + r, V - 1) * ldw;  // behind the last: read, not used
    float acc[L];
#pragma unroll
    for (int k = 0; k < L; ++k) acc[k] = 0.f;
    auto multiply = [&](const float (&wv)[8], int r, int c) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float xv[8];
        load_vec<8>(xs + t * dp + c, xv);
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[r * NT + t] = fmaf(wv[k], xv[k], acc[r * NT + t]);
      }
    };
    int c = lane * 8;
    if (VEC) {
      // the loads of the next 256 columns are on their way while these are multiplied
      RawVec<8 * sizeof(S)> now[R], next[R];
      const int whole = D / 8 * 8;
      if (c < whole) {
#pragma unroll
        for (int r = 0; r < R; ++r) now[r] = *reinterpret_cast<const RawVec<8 * sizeof(S)>*>(rows[r] + c);
      }
      for (; c < whole; c += 256) {
        if (c + 256 < whole) {
#pragma unroll
          for (int r = 0; r < R; ++r) next[r] = *reinterpret_cast<const RawVec<8 * sizeof(S)>*>(rows[r] + c + 256);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float wv[8];
          unpack_vec<8, S>(now[r], wv);
          multiply(wv, r, c);
          now[r] = next[r];
        }
      }
    }
    for (; c < D; c += 256) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float wv[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) wv[k] = c + k < D ? to_f32(rows[r][c + k]) : 0.f;
        multiply(wv, r, c);
      }
    }
    float z = sum_spread<L>(acc, lane);
    const int v = v0 + my_r;
    if (v < V && my_t < N && lane % kSpan == 0) {
      if (bias) z += to_f32(bias[v]);
      if (v == t_col) ztarget[my_t] = z;
      if (v < keep) kept[my_t * keep_ld + v] = z;
      const float nm = fmaxf(mx, z), base = nm == -INFINITY ? 0.f : nm;
      sum = sum * expf(mx - base) + expf(z - base);
      mx = nm;
      zs += z;
    }
  }
  if (lane % kSpan == 0) {
    sm[warp][lane / kSpan] = mx;
    ss[warp][lane / kSpan] = sum;
    sz[warp][lane / kSpan] = zs;
  }
  __syncthreads();
  if (threadIdx.x < N) {
    mx = -INFINITY;
    sum = zs = 0.f;
    for (int g = 0; g < 8; ++g)
      for (int r = 0; r < R; ++r) {
        const int at = r * NT + threadIdx.x;
        const float om = sm[g][at], nm = fmaxf(mx, om), base = nm == -INFINITY ? 0.f : nm;
        sum = sum * expf(mx - base) + ss[g][at] * expf(om - base);
        mx = nm;
        zs += sz[g][at];
      }
    part[blockIdx.x * N + threadIdx.x] = make_float2(mx, sum);
    if (smooth) zsum[blockIdx.x * N + threadIdx.x] = zs;
  }
}

// G [planes][rows][ldg] of the vocabulary's entries v0 .. v0 + width from such
// logits
template <typename T>
__global__ void __launch_bounds__(256)
    lce_slab_grad_kernel(const float* __restrict__ slab, int S, int64_t rows, int64_t ld, const void* __restrict__ bias,
                         int bias_dtype, const int64_t* __restrict__ target, int64_t v0, int64_t width, int64_t V,
                         int64_t ignore, float smoothing, const float* __restrict__ lse, const float* __restrict__ grow,
                         float gscale, T* __restrict__ G, int64_t ldg, int planes, const float* __restrict__ zscale) {
  const float2 unscale = lce_unscale(zscale);
  const int64_t i = blockIdx.x, tt = target[i];
  const int64_t t = lce_scored(tt, V, ignore) ? tt - v0 : -1;
  const float l = lse[i], g = grow[i], flat = smoothing / (float)V;
  for (int64_t n = threadIdx.x; n < width; n += 256) {
    float e = expf(lce_slab_logit(slab, S, rows * ld, i * ld + n, bias, v0 + n, bias_dtype, unscale) - l) - flat;
    if (n == t) e -= 1.f - smoothing;
    e = g == 0.f ? 0.f : e * g * gscale;
    for (int z = 0; z < planes; ++z) {
      const T h = from_f32<T>(e);
      G[(z * rows + i) * ldg + n] = h;
      e -= to_f32(h);
    }
  }
}

// the same from what the forward pass kept of the entries [v0, v0 + width),
// eight columns a thread: logits in fp32 (FP32), or their exponentials as
// 16-bit codes relative to a maximum per row and 64 columns.  The target's own comes from
// its logit in fp32, since 1 - p may be far smaller than p's rounding.
template <typename T, bool FP32>
__global__ void __launch_bounds__(256)
    lce_kept_grad_kernel(const void* __restrict__ kept, int64_t keep_ld, const float* __restrict__ keep_max,
                         const float* __restrict__ ztarget, int64_t rows, const int64_t* __restrict__ target,
                         int64_t v0, int64_t width, int64_t V, int64_t ignore, float smoothing,
                         const float* __restrict__ lse, const float* __restrict__ grow, float gscale,
                         T* __restrict__ G, int64_t ldg, int planes) {
  constexpr int U = FP32 ? 2 : 4;  // vectors of a thread, 2048 columns apart
  const int64_t i = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
  if (i >= rows) return;
  const float flat = smoothing / (float)V, l = lse[i], g = grow[i], scale = g * gscale;
  const int64_t tt = target[i], t = lce_scored(tt, V, ignore) ? tt - v0 : -1;
  const int64_t n0 = ((int64_t)blockIdx.x * U * 256 + threadIdx.x) * 8;
  float v[U][8];
  if (FP32) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (n0 + u * 2048 < ldg) load_vec<8>((const float*)kept + i * keep_ld + v0 + n0 + u * 2048, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < 8; ++k) v[u][k] = expf(v[u][k] - l);
  } else {
    uint4 c[U];
    float f[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t col = v0 + n0 + u * 2048;
      c[u] = make_uint4(0u, 0u, 0u, 0u);
      f[u] = 0.f;
      if (n0 + u * 2048 < ldg) {
        c[u] = *reinterpret_cast<const uint4*>((const uint16_t*)kept + i * keep_ld + col);
        f[u] = keep_max[(col >> 6) * rows + i];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float e = expf(f[u] - l) * k2p112;  // the codes' power of two with it: at most 2^112
      const uint32_t w[4] = {c[u].x, c[u].y, c[u].z, c[u].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[u][2 * k] = keep_bits(w[k] & 0xffffu) * e;
        v[u][2 * k + 1] = keep_bits(w[k] >> 16) * e;
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t n = n0 + u * 2048;
    if (n >= ldg) break;
    if (t >= n && t < n + 8) {
      const float p = expf(ztarget[i] - l) - (1.f - smoothing);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (n + k == t) v[u][k] = p;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) v[u][k] = g == 0.f ? 0.f : (v[u][k] - flat) * scale;
    for (int z = 0; z < planes; ++z) {
      store_vec<8>(G + (z * rows + i) * ldg + n, v[u]);
      if (z + 1 < planes) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[u][k] -= to_f32(from_f32<T>(v[u][k]));
      }
    }
  }
}

// sum of the losses in a fixed order (fp64), and how many rows have one
__global__ void __launch_bounds__(1024)
    lce_total_kernel(const float* __restrict__ loss, const int64_t* __restrict__ target, int64_t N, int64_t V,
                     int64_t ignore, int reduction, float* __restrict__ out, float* __restrict__ count) {
  __shared__ double s_sum[32];
  __shared__ long long s_n[32];
  double sum = 0.0;
  long long n = 0;
  for (int64_t i = threadIdx.x; i < N; i += 1024) {
    sum += (double)loss[i];
    n += lce_scored(target[i], V, ignore) ? 1 : 0;
  }
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    n += __shfl_xor_sync(0xffffffffu, n, o);
  }
  if ((threadIdx.x & 31) == 0) {
    s_sum[threadIdx.x >> 5] = sum;
    s_n[threadIdx.x >> 5] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 32; ++w) {
      sum += s_sum[w];
      n += s_n[w];
    }
    *count = (float)n;
    if (reduction != PVB2_LOSS_NONE) *out = (float)(reduction == PVB2_LOSS_MEAN ? sum / (double)n : sum);
  }
}

// the rows' factors where each has a gradient of its own: whether it has a loss
// (one) and g_i (own; 0 without a loss) for dx, and for the sums over rows
// g_i / max |g| (row) with that maximum as the number for all
__global__ void __launch_bounds__(1024)
    lce_grad_rows_kernel(const float* __restrict__ grad_out, const int64_t* __restrict__ target, int64_t N, int64_t V,
                         int64_t ignore, float inv_gscale, const float* __restrict__ scales, float* __restrict__ row,
                         float* __restrict__ one, float* __restrict__ own, float* __restrict__ factor) {
  __shared__ float s_max[32];
  float mx = 0.f;
  for (int64_t i = threadIdx.x; i < N; i += 1024)
    if (lce_scored(target[i], V, ignore)) {
      const float a = fabsf(grad_out[i]);
      mx = (a > mx || a != a) ? a : mx;
    }
  for (int o = 16; o > 0; o >>= 1) {
    const float a = __shfl_xor_sync(0xffffffffu, mx, o);
    mx = (a > mx || a != a) ? a : mx;
  }
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = mx;
  __syncthreads();
  mx = s_max[0];
  for (int w = 1; w < 32; ++w) mx = (s_max[w] > mx || s_max[w] != s_max[w]) ? s_max[w] : mx;
  for (int64_t i = threadIdx.x; i < N; i += 1024) {
    const bool scored = lce_scored(target[i], V, ignore);
    const float g = grad_out[i];
    row[i] = scored && mx != 0.f ? g / mx : 0.f;
    one[i] = scored ? 1.f : 0.f;
    own[i] = scored ? g : 0.f;
  }
  if (threadIdx.x == 0) {
    factor[0] = inv_gscale;
    factor[1] = scales ? inv_gscale * scales[1] : inv_gscale;
    factor[2] = scales ? inv_gscale * scales[0] : inv_gscale;
    factor[3] = mx;
  }
}

// out [rows][cols] = scale * sum of S slabs [rows][ld], four columns a thread
template <typename T>
__global__ void lce_join_kernel(const float* __restrict__ slab, int S, int64_t rows, int64_t cols, int64_t ld,
                                LceScale scale, T* __restrict__ out, int vec) {
  const int per_row = (int)(ld / 4);
  const int64_t total = rows * per_row, size = rows * ld;
  for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < total; e += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = total <= INT32_MAX ? (int64_t)((int)e / per_row) : e / per_row;
    const int64_t c = (e - r * per_row) * 4;
    float v[4];
    load_vec<4>(slab + r * ld + c, v);
    for (int s = 1; s < S; ++s) {
      float u[4];
      load_vec<4>(slab + s * size + r * ld + c, u);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] += u[k];
    }
    const float2 f = lce_row_scale(scale, r);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = v[k] * f.x * f.y;
    if (vec) {
      store_vec<4>(out + r * cols + c, v);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (c + k < cols) out[r * cols + c + k] = from_f32<T>(v[k]);
    }
  }
}

// column sums of G (planes added): 32 columns and 32 rows at a time, partial
// sums per part of the rows first, then in order
template <typename T, typename O>
__global__ void __launch_bounds__(1024) lce_colsum_kernel(const T* __restrict__ G, int64_t rows, int64_t cols, int64_t ld,
                                                         int planes, int64_t rows_per, float* __restrict__ part,
                                                         const float* __restrict__ factor, O* __restrict__ out) {
  __shared__ float s[32][33];
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t col = (int64_t)blockIdx.x * 32 + c;
  const int64_t r0 = blockIdx.y * rows_per, r1 = min(rows, r0 + rows_per);
  float sum = 0.f;
  if (col < cols)
    for (int64_t r = r0 + g; r < r1; r += 32) {
      float v = 0.f;
      for (int z = planes - 1; z >= 0; --z) v += to_f32(G[(z * rows + r) * ld + col]);
      sum += v;
    }
  s[g][c] = sum;
  __syncthreads();
  if (g == 0 && col < cols) {
    for (int q = 1; q < 32; ++q) sum += s[q][c];
    if (gridDim.y == 1) out[col] = from_f32<O>(sum * factor[0] * factor[3]);  // there is one part
    else part[blockIdx.y * cols + col] = sum;
  }
}

template <typename T>
__global__ void lce_dbias_kernel(const float* __restrict__ part, int parts, int64_t cols,
                                 const float* __restrict__ factor, T* __restrict__ out) {
  const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= cols) return;
  double s = 0.0;
  for (int q = 0; q < parts; ++q) s += (double)part[q * cols + c];
  out[c] = from_f32<T>((float)(s * (double)factor[0] * (double)factor[3]));
}

// --------------------------------------------------------------- host side
static int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }
static int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

static int lce_pairs_on_device() { return std::max(1, num_sms() / 2); }

// How a product M x N x K is cut: tiles of 256 x bn, K in `splits` parts of
// kb_per blocks (each part a slab of partial sums, joined by a launch of its
// own).
struct LceTiling {
  int bn, splits, kb_per;
  double cycles;
};

// The cut with the least modelled time.  Cycles of a K block of a tile, for each
// product: 520 for 256 x 256 (512 is both the MMAs' rate and that of 16-bit
// operands' loads from L2), 400 for 256 x 128, where 16-bit operands wait for
// their loads (384) and split ones' MMA reads share 128 bytes of shared memory a
// cycle with the loads' writes.  A tile costs about 2500 more (its last loads and
// its epilogue), joining slabs their traffic and a launch.
static LceTiling lce_tiling(int64_t M, int64_t N, int64_t K, int P, int64_t read_bytes, bool cut = true) {
  const int64_t kb = cdiv(K, kLBK), pairs = lce_pairs_on_device();
  const double read = read_bytes / 3200.0;  // cycles at 6.1 TB/s and 1.9 GHz
  LceTiling best{0, 1, 0, 0};
  for (int bn = 256; bn >= 128; bn /= 2) {
    const double products = P == 2 ? 3 : 1;
    const double block = products * (bn == 256 ? 520 : 400);
    const int64_t tiles = cdiv(M, kLBM) * cdiv(N, bn);
    const int64_t most = cut && tiles < pairs ? std::min<int64_t>(16, std::max<int64_t>(1, kb / 2)) : 1;
    for (int64_t S = 1; S <= most; ++S) {
      const int64_t per = cdiv(kb, S);
      if (cdiv(kb, per) != S) continue;
      double c = cdiv(tiles * S, pairs) * (per * block + 2500);
      c = std::max(c, read);
      if (S > 1) c += 6000 + (double)S * M * N * 8 / 3200.0;
      if (!best.bn || c < best.cycles) best = LceTiling{bn, (int)S, (int)per, c};
    }
  }
  return best;
}

struct LcePlan {
  bool few;          // forward: few rows, no tiles
  int P;             // planes of an operand
  bool half;         // fp16 planes (bf16 otherwise)
  int64_t ldp;       // row length of packed operands
  bool pack_w;       // w is packed piece by piece
  bool pack_x;       // forward: x is packed (the backward pass always does)
  int64_t piece;     // vocabulary entries of a piece
  int pieces;
  LceTiling z, dx, dw;
  int colsum_parts;
  int64_t rows_per;
};

// rows that lce_few_rows_kernel takes, and their bytes in shared memory
constexpr int kLFewRows = 8, kLFewBytes = 64 * 1024;

constexpr int64_t kLRowsFwd = 16384;  // rows whose parts are held at a time

// 16-bit operands whose rows begin on 16-byte boundaries are read as they lie
static bool lce_direct(const pvb2_linear_ce_desc* d, int64_t ld) { return d->dtype != PVB2_F32 && ld % 8 == 0; }

// with one row the stride says nothing
static pvb2_linear_ce_desc lce_normal(const pvb2_linear_ce_desc* d) {
  pvb2_linear_ce_desc n = *d;
  if (n.N <= 1) n.ldx = up(n.D, 8);
  if (n.V <= 1) n.ldw = up(n.D, 8);
  return n;
}

// Five to eight 16-bit rows go there while w is below 64 MB (768 x 8000: 17 us
// against 21 on tiles); beyond, the products in fp32 cost more than w's slower
// reads (2048 x 32768: 64 and 55 us, 4096 x 50000: 150 and 117).  fp32 tiles need
// three products and w's parts (768 x 32768: 45 us for eight rows, 115 for nine).
static bool lce_few_rows(const pvb2_linear_ce_desc* d, int64_t ldp) {
  const int64_t most = d->dtype == PVB2_F32 || d->V * d->D < (1 << 25) ? kLFewRows : 4;
  return d->N <= most && kLFewRows * ldp * (d->dtype == PVB2_F32 ? 4 : 2) <= kLFewBytes;
}

static LcePlan lce_make_plan(const pvb2_linear_ce_desc* d, bool backward) {
  LcePlan p;
  p.half = d->dtype != PVB2_BF16;
  p.P = d->dtype == PVB2_F32 ? 2 : 1;
  // packed rows begin on 128-byte lines, unless that would be mostly padding
  p.ldp = up(d->D, d->D >= 256 ? 64 : 8);
  // Rows of w that straddle lines take two reads from L2 for each 128 bytes.  A
  // copy costs the same for any number of tokens and pays from about 3500 on
  // (D 1000, V 49999, forward: 397 us as it lies and 376 us with the copy at
  // 4095 tokens, 196 and 244 us at 2048; between the two, where a line through
  // the differences is 0).
  p.pack_w = !lce_direct(d, d->ldw) || (d->ldw % 64 != 0 && d->D >= 256 && d->N >= 3500);
  p.pack_x = !lce_direct(d, d->ldx) || (d->ldx % 64 != 0 && d->D >= 256 && d->V >= 2048);
  p.few = !backward && lce_few_rows(d, p.ldp);
  const int64_t rows = backward ? d->N : std::min(d->N, kLRowsFwd);
  const int64_t esize = 2 * p.P;
  // most entries of a piece: a packed piece of w in 256 MB, G in 128 MB, at
  // least 1024 entries
  int64_t most = up(d->V, 256);
  if (p.pack_w) most = std::min<int64_t>(most, ((int64_t)256 << 20) / (p.ldp * esize));
  if (backward) most = std::min<int64_t>(most, ((int64_t)128 << 20) / (rows * esize));
  most = std::max<int64_t>(std::min<int64_t>(1024, up(d->V, 256)), most / 256 * 256);
  auto cost = [&](int64_t width) {
    double c = lce_tiling(rows, width, d->D, p.P, width * d->D * 2).cycles + 4000;
    if (backward)
      c += lce_tiling(rows, d->D, width, p.P, 0).cycles + lce_tiling(width, d->D, rows, p.P, 0).cycles + 8000;
    return c;
  };
  p.piece = most;
  if (backward && most < d->V) {
    // widths from half of the most on: the one whose tiles fill the SMs best
    double least = 0;
    for (int64_t w = most; w >= std::max<int64_t>(1024, most / 2); w -= 256) {
      const double c = d->V / w * cost(w) + (d->V % w ? cost(d->V % w) : 0);
      if (least == 0 || c < 0.995 * least) {
        least = c;
        p.piece = w;
      }
    }
  }
  p.pieces = (int)cdiv(d->V, p.piece);
  const int64_t width = std::min(p.piece, d->V);
  // the forward pass joins the slabs of a whole row
  p.z = lce_tiling(rows, width, d->D, p.P, width * d->D * 2, backward || p.pieces == 1);
  // slabs of dx are laid down by the first piece, which has to be the widest
  p.dx = lce_tiling(d->N, d->D, width, p.P, 0, d->kept == 0 || d->kept == d->V);
  p.dw = lce_tiling(width, d->D, d->N, p.P, 0);
  p.colsum_parts = (int)std::min<int64_t>(64, cdiv(d->N, 512));
  p.rows_per = p.colsum_parts ? up(cdiv(d->N, p.colsum_parts), 8) : 0;
  return p;
}

// The plan of a call is asked for several times over (memory to keep,
// workspace, launch): the last ones of this thread, by all that they depend
// on.
static LcePlan lce_plan(const pvb2_linear_ce_desc* d, bool backward) {
  struct Made {
    int64_t N = -1, D, V, ldx, ldw, kept;
    int32_t dtype, sms;
    bool backward;
    LcePlan plan;
  };
  static thread_local Made made[4];
  static thread_local int next = 0;
  const int sms = num_sms();
  for (const Made& m : made)
    if (m.N == d->N && m.D == d->D && m.V == d->V && m.ldx == d->ldx && m.ldw == d->ldw && m.kept == d->kept && m.dtype == d->dtype &&
        m.sms == sms && m.backward == backward)
      return m.plan;
  Made& m = made[next];
  next = (next + 1) % 4;
  m.N = d->N;
  m.D = d->D;
  m.V = d->V;
  m.ldx = d->ldx;
  m.ldw = d->ldw;
  m.kept = d->kept;
  m.dtype = d->dtype;
  m.sms = sms;
  m.backward = backward;
  m.plan = lce_make_plan(d, backward);
  return m.plan;
}

// places in the workspace, 1024-byte aligned
struct Arena {
  uint8_t* base;
  size_t at = 0;
  template <typename T>
  T* take(size_t n) {
    T* r = (T*)(base + at);
    at += (n * sizeof(T) + 1023) / 1024 * 1024;
    return r;
  }
};

// What a forward pass keeps for the backward one, of the first d->kept
// entries: logits in fp32 (fp32 operands, and logits that were formed in
// slabs), else 16-bit codes of their exponentials with the maxima per 64
// columns; and every row's target logit.
struct LceKept {
  bool fp32;
  int64_t ld;
  void* data;
  float *max, *ztarget;
};

static size_t lce_kept_space(const pvb2_linear_ce_desc* d, bool fp32, const void* base, LceKept* k) {
  Arena a{(uint8_t*)base};
  k->fp32 = fp32;
  k->ld = up(d->kept, 64);
  k->data = a.take<uint8_t>(d->N * k->ld * (fp32 ? 4 : 2));
  k->max = a.take<float>(fp32 ? 0 : k->ld / 64 * d->N);
  k->ztarget = a.take<float>(d->N);
  return a.at;
}

struct LceFwdSpace {
  uint16_t *x, *w;
  float* absmax;
  float* slab;
  float2* part;
  float *zsum, *ztarget, *loss;
};

static bool lce_slabs(const LcePlan& p) { return !p.few && p.z.splits > 1; }

// blocks of lce_few_rows_kernel: two for every SM
static int lce_few_blocks(const pvb2_linear_ce_desc* d) {
  return (int)std::min<int64_t>(2 * num_sms(), cdiv(d->V, 16));
}

static bool lce_kept_fp32(const pvb2_linear_ce_desc* d) {
  const LcePlan p = lce_plan(d, false);
  return d->dtype == PVB2_F32 || p.few || lce_slabs(p);
}

static size_t lce_fwd_space(const pvb2_linear_ce_desc* d, const LcePlan& p, void* base, LceFwdSpace* s) {
  Arena a{(uint8_t*)base};
  const int64_t rows = std::min(d->N, kLRowsFwd);
  const int64_t parts = p.few ? lce_few_blocks(d) : up(d->V, 256) / 64;
  const bool slabs = lce_slabs(p);
  s->x = a.take<uint16_t>(!p.few && p.pack_x ? rows * p.ldp * p.P : 0);
  s->w = a.take<uint16_t>(!p.few && p.pack_w ? p.piece * p.ldp * p.P : 0);
  s->absmax = a.take<float>(!p.few && p.P == 2 ? kLScaleBlocks : 0);
  s->slab = a.take<float>(slabs ? p.z.splits * rows * up(d->V, 4) : 0);
  s->part = a.take<float2>(slabs ? 0 : rows * parts);
  s->zsum = a.take<float>(!slabs && d->label_smoothing != 0 ? rows * parts : 0);
  s->ztarget = a.take<float>(slabs ? 0 : rows);
  s->loss = a.take<float>(d->N);
  return a.at;
}

struct LceBwdSpace {
  uint16_t *x, *w, *G;
  float *absmax, *scales;
  float *slab, *row, *factor, *dx, *dw, *colsum;  // factor: see LceRowsJob
  float *own, *one;                               // see LceRowsJob; one: see lce_grad_rows_kernel
};

static size_t lce_bwd_space(const pvb2_linear_ce_desc* d, const LcePlan& p, void* base, LceBwdSpace* s) {
  Arena a{(uint8_t*)base};
  const int64_t ld32 = up(d->D, 4), width = std::min(p.piece, d->V);
  s->x = a.take<uint16_t>(d->N * p.ldp * p.P);
  s->w = a.take<uint16_t>(p.pack_w ? p.piece * p.ldp * p.P : 0);
  s->G = a.take<uint16_t>(d->N * up(width, 64) * p.P);
  s->slab = a.take<float>(lce_slabs(p) ? p.z.splits * d->N * up(width, 4) : 0);
  s->row = a.take<float>(d->N);
  s->own = a.take<float>(d->N);
  s->one = a.take<float>(d->reduction == PVB2_LOSS_NONE ? d->N : 0);
  const bool scales = p.P == 2 && lce_few_rows(d, p.ldp);
  s->absmax = a.take<float>(scales ? kLScaleBlocks : 0);
  s->scales = a.take<float>(scales ? 2 : 0);
  s->factor = a.take<float>(4);
  s->dx = a.take<float>(p.pieces > 1 || (d->kept > 0 && d->kept < d->V) || p.dx.splits > 1 ? p.dx.splits * d->N * ld32 : 0);
  s->dw = a.take<float>(p.dw.splits > 1 ? p.dw.splits * width * ld32 : 0);
  s->colsum = a.take<float>(p.colsum_parts * width);
  return a.at;
}

static int lce_check(const pvb2_linear_ce_desc* d) {
  PVB2_CHECK_ARG(d, "linear cross entropy: no descriptor");
  PVB2_CHECK_ARG(d->dtype == PVB2_F32 || d->dtype == PVB2_F16 || d->dtype == PVB2_BF16,
                 "linear cross entropy: fp32, fp16 or bf16 expected (got dtype %d)", d->dtype);
  PVB2_CHECK_ARG(d->reduction >= PVB2_LOSS_NONE && d->reduction <= PVB2_LOSS_SUM,
                 "linear cross entropy: unknown reduction %d", d->reduction);
  PVB2_CHECK_ARG(d->N >= 0 && d->V >= 1 && d->D >= 1 && d->N < (1 << 24) && d->V < (1 << 24) && d->D < (1 << 20),
                 "linear cross entropy: sizes N=%lld D=%lld V=%lld out of range", (long long)d->N, (long long)d->D,
                 (long long)d->V);
  PVB2_CHECK_ARG((d->N <= 1 || d->ldx >= d->D) && (d->V <= 1 || d->ldw >= d->D),
                 "linear cross entropy: row strides below the row length");
  PVB2_CHECK_ARG(d->kept >= 0 && d->kept <= d->V && (d->kept == d->V || d->kept % 256 == 0),
                 "linear cross entropy: all entries or a multiple of 256 are kept (got %lld)", (long long)d->kept);
  PVB2_CHECK_ARG(d->label_smoothing >= 0.0 && d->label_smoothing <= 1.0,
                 "linear cross entropy: label smoothing in [0, 1] expected");
  return PVB2_OK;
}

static int lce_aligned(const void* p, bool direct) {
  PVB2_CHECK_ARG(!direct || ((uintptr_t)p & 15) == 0,
                 "linear cross entropy: 16-bit operands with row strides of 16 bytes begin on 16-byte boundaries");
  return PVB2_OK;
}

// a [planes][rows][ld] operand of 16-bit numbers; box: 64 columns x `rows_box` rows
static int lce_map(CUtensorMap* m, const void* base, int64_t cols, int64_t rows, int64_t ld, int planes, int rows_box,
                   bool half) {
  uint64_t dims[3] = {(uint64_t)cols, (uint64_t)rows, (uint64_t)planes};
  uint64_t str[2] = {(uint64_t)ld * 2, (uint64_t)ld * 2 * rows};
  uint32_t box[3] = {64, (uint32_t)rows_box, 1};
  return encode_tiled(m, 3, base, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      nullptr, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
}

static int lce_map32(CUtensorMap* m, const void* base, int64_t cols, int64_t rows, int64_t ld, int slabs) {
  uint64_t dims[3] = {(uint64_t)cols, (uint64_t)rows, (uint64_t)slabs};
  uint64_t str[2] = {(uint64_t)ld * 4, (uint64_t)ld * 4 * rows};
  uint32_t box[3] = {32, 32, 1};
  return encode_tiled(m, 3, base, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// K-major operands: 128 rows of A, bn / 2 of B
static int lce_map_a(CUtensorMap* m, const void* base, int64_t cols, int64_t rows, int64_t ld, const LcePlan& p) {
  return lce_map(m, base, cols, rows, ld, p.P, 128, p.half);
}
static int lce_map_b(CUtensorMap* m, const void* base, int64_t cols, int64_t rows, int64_t ld, const LcePlan& p, int bn) {
  return lce_map(m, base, cols, rows, ld, p.P, bn / 2, p.half);
}
// MN-major operands, and G as it is stored: 64 columns x 64 (32) rows
static int lce_map_mn(CUtensorMap* m, const void* base, int64_t cols, int64_t rows, int64_t ld, const LcePlan& p) {
  return lce_map(m, base, cols, rows, ld, p.P, 64, p.half);
}

template <int EPI, typename T, int P, int BN, int CHUNK>
static int lce_launch(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& c, const LceGemm& g, bool a_mn,
                      bool b_mn, cudaStream_t s) {
  constexpr int smem = LceSmem<P, BN>::TOTAL + 1024;
  auto kernel = lce_gemm_kernel<EPI, T, P, BN, CHUNK>;
  static DeviceOnce once;
  PVB2_TRY(allow_smem(kernel, smem, once));
  const int64_t tiles = cdiv(g.M, kLBM) * cdiv(g.N, BN) * g.splits;
  PVB2_CHECK_ARG(tiles < INT32_MAX / 2, "linear cross entropy: too many tiles");
  const int grid = 2 * (int)std::min<int64_t>(tiles, lce_pairs_on_device());
  // as many blocks of the fast side as stay in L2 (32 MB of its 126) while the
  // other side goes by: without it (8192 x 16384 x 4096) the whole fast side
  // came from HBM again for every two columns of tiles, 1.55 GB where 0.6 do
  LceGemm h = g;
  const int64_t block = (int64_t)(g.n_fast ? BN : kLBM) * g.K * 2 * P;
  const int64_t fast = g.n_fast ? cdiv(g.N, BN) : cdiv(g.M, kLBM);
  h.group = (int)std::min<int64_t>(fast, std::max<int64_t>(8, ((int64_t)32 << 20) / block));
  kernel<<<grid, LceSmem<P, BN>::THREADS, smem, s>>>(a, b, c, h, a_mn ? 1 : 0, b_mn ? 1 : 0);
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

// Chunks: split operands (results to fp32) every two blocks (N 2048, D 768, V
// 16384, mean error of losses and gradients: 6e-8 and 3.4e-7, where a product in
// fp32 has 6e-8 and 6 to 8e-7; every block 5e-8 and 2e-7, but a step of V 32768
// takes 1.21 ms instead of 1.00; every three 5e-7 and 0.98 ms); 16-bit ones every 8 on 256 x 128 tiles, which wait for their
// loads anyway, and every 16 where the result is fp32 (the losses: up to 2e-6
// off without, 3e-7 with, for 3% of the forward product's time).
template <int EPI>
static int lce_gemm(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& c, const LceGemm& g, bool a_mn,
                    bool b_mn, const LcePlan& p, int bn, cudaStream_t s) {
  if (p.P == 2 && bn == 256) return lce_launch<EPI, __half, 2, 256, 2>(a, b, c, g, a_mn, b_mn, s);
  if (p.P == 2) return lce_launch<EPI, __half, 2, 128, 2>(a, b, c, g, a_mn, b_mn, s);
  if (p.half) {
    if (bn == 256) return lce_launch<EPI, __half, 1, 256, EPI == kEpiStats ? 16 : 0>(a, b, c, g, a_mn, b_mn, s);
    return lce_launch<EPI, __half, 1, 128, 8>(a, b, c, g, a_mn, b_mn, s);
  }
  if (bn == 256) return lce_launch<EPI, __nv_bfloat16, 1, 256, EPI == kEpiStats ? 16 : 0>(a, b, c, g, a_mn, b_mn, s);
  return lce_launch<EPI, __nv_bfloat16, 1, 128, 8>(a, b, c, g, a_mn, b_mn, s);
}

struct LceOperand {  // to be packed
  const void* src = nullptr;
  int64_t row0 = 0, rows = 0, ld = 0;
  uint16_t* dst = nullptr;
  const int64_t* target = nullptr;
};

template <typename S, typename T>
static int lce_pack_as(const pvb2_linear_ce_desc* d, const LcePlan& p, const LceOperand& a, const LceOperand& b,
                       const LceRowsJob& rows, const LceScaleJob& scale, cudaStream_t s) {
  auto job = [](const LceOperand& o) {
    const S* src = (const S*)o.src + o.row0 * o.ld;
    return LcePackJob<S>{src, o.rows, o.ld, o.dst, o.target, ((uintptr_t)src & 15) == 0 && o.ld * sizeof(S) % 16 == 0};
  };
  const int64_t total = std::max((a.rows + b.rows) * (p.ldp / 8), rows.row ? rows.N : 0);
  if (total == 0) return PVB2_OK;
  lce_pack_kernel<S, T><<<grid_for(total, 256), 256, 0, s>>>(job(a), job(b), rows, scale, d->D, p.ldp, p.P, d->V,
                                                             d->ignore_index);
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

static int lce_pack(const pvb2_linear_ce_desc* d, const LcePlan& p, const LceOperand& a, const LceOperand& b,
                    const LceRowsJob& rows, const LceScaleJob& scale, cudaStream_t s) {
  if (d->dtype == PVB2_F32) return lce_pack_as<float, __half>(d, p, a, b, rows, scale, s);
  if (p.half) return lce_pack_as<__half, __half>(d, p, a, b, rows, scale, s);
  return lce_pack_as<__nv_bfloat16, __nv_bfloat16>(d, p, a, b, rows, scale, s);
}

// the scales of split operands: their magnitudes, for the launches that pack
static int lce_scales(const pvb2_linear_ce_desc* d, const LcePlan& p, const void* x, const void* w,
                      const int64_t* target, float* absmax, float* scales, LceScaleJob* job, cudaStream_t s) {
  if (p.P == 1) return PVB2_OK;
  job->part = absmax;
  const int64_t blocks = std::min<int64_t>(kLScaleBlocks, std::max<int64_t>(2, cdiv((d->N + d->V) * d->D, 16384)));
  job->nx = (int)std::min(blocks - 1, std::max<int64_t>(1, blocks * d->N / (d->N + d->V)));
  job->nw = (int)blocks - job->nx;
  job->scales = scales;
  lce_absmax_kernel<<<job->nx + job->nw, 1024, 0, s>>>((const float*)x, d->N, d->ldx, (const float*)w, d->V, d->ldw, d->D,
                                                      target, d->V, d->ignore_index, job->nx, absmax);
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

static LceRowsJob lce_no_rows() {
  LceRowsJob r;
  memset(&r, 0, sizeof(r));
  return r;
}

// out = scale * (sum of slabs), as the operands' type
static int lce_join(const pvb2_linear_ce_desc* d, const float* slab, int S, int64_t rows, const LceScale& scale,
                    void* out, cudaStream_t s) {
  const int64_t ld = up(d->D, 4);
  const int grid = grid_for(rows * (ld / 4), 256), vec = d->D % 4 == 0 && ((uintptr_t)out & 15) == 0;
  if (d->dtype == PVB2_F32) lce_join_kernel<<<grid, 256, 0, s>>>(slab, S, rows, d->D, ld, scale, (float*)out, vec);
  else if (d->dtype == PVB2_F16) lce_join_kernel<<<grid, 256, 0, s>>>(slab, S, rows, d->D, ld, scale, (__half*)out, vec);
  else lce_join_kernel<<<grid, 256, 0, s>>>(slab, S, rows, d->D, ld, scale, (__nv_bfloat16*)out, vec);
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

static LceGemm lce_logits(const pvb2_linear_ce_desc* d, const void* bias, int64_t rows, int64_t v0, int64_t width,
                          int w_row0, const int64_t* target) {
  LceGemm g;
  memset(&g, 0, sizeof(g));
  g.M = (int)rows;
  g.N = (int)width;
  g.K = (int)d->D;
  g.v0 = (int)v0;
  g.b_row0 = w_row0;
  g.splits = 1;
  g.kb_per = INT32_MAX / 2;
  g.bias = bias;
  g.bias_dtype = d->dtype;
  g.target = target;
  g.V = d->V;
  g.ignore = d->ignore_index;
  g.smoothing = (float)d->label_smoothing;
  return g;
}

static LceGemm lce_product(int64_t M, int64_t N, int64_t K, int b_row0, const LceTiling& t) {
  LceGemm g;
  memset(&g, 0, sizeof(g));
  g.M = (int)M;
  g.N = (int)N;
  g.K = (int)K;
  g.b_row0 = b_row0;
  g.n_fast = 1;
  g.splits = t.splits;
  g.kb_per = t.splits > 1 ? t.kb_per : INT32_MAX / 2;
  return g;
}

// a map that no kernel reads, where an epilogue has none
static CUtensorMap no_map() {
  CUtensorMap m;
  memset(&m, 0, sizeof(m));
  return m;
}

// the product A B (K not cut) into `out`, rows x D
static int lce_out(const pvb2_linear_ce_desc* d, const LcePlan& p, const CUtensorMap& a, const CUtensorMap& b, LceGemm g,
                   bool a_mn, int64_t rows, void* out, const LceScale& scale, int bn, cudaStream_t s) {
  const int size = d->dtype == PVB2_F32 ? 4 : 2;
  CUtensorMap c = no_map();
  g.out = out;
  g.out_ld = d->D;
  g.out_dtype = d->dtype;
  g.out_scale = scale;
  g.out_tma = ((uintptr_t)out & 15) == 0 && d->D * size % 16 == 0;
  if (g.out_tma) {
    if (size == 4) PVB2_TRY(lce_map32(&c, out, d->D, rows, d->D, 1));
    else PVB2_TRY(lce_map(&c, out, d->D, rows, d->D, 1, 32, p.half));
  }
  return lce_gemm<kEpiOut>(a, b, c, g, a_mn, true, p, bn, s);
}

template <typename S, int NT, int R>
static int lce_few_launch(const pvb2_linear_ce_desc* d, const void* x, const void* w, const void* bias,
                          const int64_t* target, const LceFwdSpace& sp, const LceKept& k, cudaStream_t s) {
  const bool vec = ((uintptr_t)w & 15) == 0 && d->ldw * sizeof(S) % 16 == 0;
  auto kernel = vec ? lce_few_rows_kernel<S, NT, R, true> : lce_few_rows_kernel<S, NT, R, false>;
  static DeviceOnce once[2];
  PVB2_TRY(allow_smem(kernel, kLFewBytes, once[vec]));
  const size_t smem = (size_t)NT * up(d->D, 8) * sizeof(S);
  kernel<<<lce_few_blocks(d), 256, smem, s>>>((const S*)x, d->ldx, (const S*)w, d->ldw, (const S*)bias, target,
                                              (int)d->N, (int)d->D, (int)d->V, d->ignore_index,
                                              d->label_smoothing != 0, sp.part, sp.zsum,
                                              d->kept ? k.ztarget : sp.ztarget, (float*)k.data, (int)d->kept, k.ld);
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

template <typename S>
static int lce_few(const pvb2_linear_ce_desc* d, const void* x, const void* w, const void* bias, const int64_t* target,
                   const LceFwdSpace& sp, const LceKept& k, cudaStream_t s) {
  if (d->N == 1) return lce_few_launch<S, 1, sizeof(S) == 4 ? 4 : 8>(d, x, w, bias, target, sp, k, s);
  if (d->N == 2) return lce_few_launch<S, 2, 4>(d, x, w, bias, target, sp, k, s);
  if (d->N <= 4) return lce_few_launch<S, 4, 4>(d, x, w, bias, target, sp, k, s);
  return lce_few_launch<S, 8, 4>(d, x, w, bias, target, sp, k, s);
}

// logits of `rows` rows as partial sums
static int lce_slab_logits(const pvb2_linear_ce_desc* d, const LcePlan& p, const CUtensorMap& x, const CUtensorMap& w,
                           LceGemm g, float* slab, cudaStream_t s) {
  CUtensorMap c;
  g.splits = p.z.splits;
  g.kb_per = p.z.kb_per;
  PVB2_TRY(lce_map32(&c, slab, g.N, g.M, up(g.N, 4), p.z.splits));
  return lce_gemm<kEpiAcc>(x, w, c, g, false, false, p, p.z.bn, s);
}

template <typename T>
static int lce_kept_grad(const pvb2_linear_ce_desc* d, const LcePlan& p, const LceBwdSpace& sp, const LceKept& k,
                         const int64_t* target, const float* lse, const float* grow, int64_t v0, int64_t width,
                         int64_t ldg, float gscale, cudaStream_t s) {
  const unsigned rows = (unsigned)std::min<int64_t>(d->N, 32768);
  const dim3 grid((unsigned)cdiv(ldg, k.fp32 ? 4096 : 8192), rows, (unsigned)cdiv(d->N, rows));
  const float smoothing = (float)d->label_smoothing;
  if (k.fp32)
    lce_kept_grad_kernel<T, true><<<grid, 256, 0, s>>>(k.data, k.ld, k.max, k.ztarget, d->N, target, v0, width, d->V,
                                                       d->ignore_index, smoothing, lse, grow, gscale, (T*)sp.G, ldg,
                                                       p.P);
  else
    lce_kept_grad_kernel<T, false><<<grid, 256, 0, s>>>(k.data, k.ld, k.max, k.ztarget, d->N, target, v0, width, d->V,
                                                        d->ignore_index, smoothing, lse, grow, gscale, (T*)sp.G, ldg,
                                                        p.P);
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

template <typename T>
static int lce_slab_grad(const pvb2_linear_ce_desc* d, const LcePlan& p, const LceBwdSpace& sp, const void* bias,
                         const int64_t* target, const float* lse, const float* grow, int64_t v0, int64_t width,
                         int64_t ldg, float gscale, const float* zscale, cudaStream_t s) {
  lce_slab_grad_kernel<<<(int)d->N, 256, 0, s>>>(sp.slab, p.z.splits, d->N, up(width, 4), bias, d->dtype, target, v0,
                                                 width, d->V, d->ignore_index, (float)d->label_smoothing, lse, grow,
                                                 gscale, (T*)sp.G, ldg, p.P, zscale);
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

template <typename T, typename O>
static int lce_bias_grad_as(const pvb2_linear_ce_desc* d, const LcePlan& p, const LceBwdSpace& sp, int64_t width,
                            int64_t ldg, O* out, cudaStream_t s) {
  const dim3 grid((unsigned)cdiv(width, 32), (unsigned)p.colsum_parts);
  lce_colsum_kernel<<<grid, 1024, 0, s>>>((const T*)sp.G, d->N, width, ldg, p.P, p.rows_per, sp.colsum, sp.factor, out);
  PVB2_LAUNCH_CHECK();
  if (p.colsum_parts == 1) return PVB2_OK;
  lce_dbias_kernel<<<(int)cdiv(width, 256), 256, 0, s>>>(sp.colsum, p.colsum_parts, width, sp.factor, out);
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

static int lce_bias_grad(const pvb2_linear_ce_desc* d, const LcePlan& p, const LceBwdSpace& sp, int64_t width,
                         int64_t ldg, void* out, cudaStream_t s) {
  if (d->dtype == PVB2_F32) return lce_bias_grad_as<__half, float>(d, p, sp, width, ldg, (float*)out, s);
  if (p.half) return lce_bias_grad_as<__half, __half>(d, p, sp, width, ldg, (__half*)out, s);
  return lce_bias_grad_as<__nv_bfloat16, __nv_bfloat16>(d, p, sp, width, ldg, (__nv_bfloat16*)out, s);
}

}  // namespace pvb2

using namespace pvb2;

extern "C" {

size_t pvb2_linear_ce_fwd_workspace_size(const pvb2_linear_ce_desc* desc) {
  if (lce_check(desc) != PVB2_OK || desc->N == 0) return 0;
  const pvb2_linear_ce_desc normal = lce_normal(desc), *d = &normal;
  LceFwdSpace s;
  return lce_fwd_space(d, lce_plan(d, false), nullptr, &s) + 1024;
}

int pvb2_linear_ce_fwd(const pvb2_linear_ce_desc* desc, const void* x, const void* w, const void* bias,
                       const int64_t* target, float* out, float* lse, float* count, void* kept, void* workspace,
                       size_t workspace_bytes, pvb2_stream stream) {
  PVB2_TRY(lce_check(desc));
  const pvb2_linear_ce_desc normal = lce_normal(desc), *d = &normal;
  PVB2_CHECK_ARG(w && count && (d->N == 0 || (x && target && lse && out)), "linear cross entropy: null pointer");
  cudaStream_t s = as_stream(stream);
  float* loss = out;
  if (d->N > 0) {
    const LcePlan p = lce_plan(d, false);
    LceFwdSpace sp;
    const size_t need = lce_fwd_space(d, p, (void*)(((uintptr_t)workspace + 1023) & ~(uintptr_t)1023), &sp) + 1024;
    PVB2_CHECK_ARG(workspace && workspace_bytes >= need, "linear cross entropy: workspace of %zu bytes needed", need);
    if (d->reduction != PVB2_LOSS_NONE) loss = sp.loss;
    const bool direct_x = !p.pack_x, slabs = lce_slabs(p);
    PVB2_TRY(lce_aligned(x, direct_x && !p.few));
    PVB2_TRY(lce_aligned(w, !p.pack_w && !p.few));
    const int parts = p.few ? lce_few_blocks(d) : (int)cdiv(d->V, 64), esize = d->dtype == PVB2_F32 ? 4 : 2;
    const float smoothing = (float)d->label_smoothing;
    PVB2_CHECK_ARG(d->kept == 0 || (kept && ((uintptr_t)kept & 15) == 0),
                   "linear cross entropy: 16-byte aligned memory for what is kept needed");
    LceKept k;
    lce_kept_space(d, d->dtype == PVB2_F32 || p.few || slabs, kept, &k);
    LceScaleJob scale{};
    if (!p.few) PVB2_TRY(lce_scales(d, p, x, w, target, sp.absmax, count + 1, &scale, s));
    const float* zscale = p.P == 2 ? count + 1 : nullptr;
    for (int64_t r0 = 0; r0 < d->N; r0 += kLRowsFwd) {
      const int64_t rows = std::min(kLRowsFwd, d->N - r0);
      CUtensorMap ma, mb;
      if (p.few) {
        if (d->dtype == PVB2_F32) PVB2_TRY(lce_few<float>(d, x, w, bias, target, sp, k, s));
        else if (p.half) PVB2_TRY(lce_few<__half>(d, x, w, bias, target, sp, k, s));
        else PVB2_TRY(lce_few<__nv_bfloat16>(d, x, w, bias, target, sp, k, s));
        lce_few_join_kernel<<<1, 256, 0, s>>>(sp.part, smoothing != 0.f ? sp.zsum : nullptr, parts,
                                              d->kept ? k.ztarget : sp.ztarget, target, (int)d->N, d->V,
                                              d->ignore_index, smoothing, d->reduction, lse, loss, out, count);
        PVB2_LAUNCH_CHECK();
        return PVB2_OK;
      }
      if (direct_x) {
        PVB2_TRY(lce_map_a(&ma, (const uint8_t*)x + r0 * d->ldx * esize, d->D, rows, d->ldx, p));
      } else {
        PVB2_TRY(lce_map_a(&ma, sp.x, d->D, rows, p.ldp, p));
      }
      for (int64_t v0 = 0; v0 < d->V; v0 += p.piece) {
        const int64_t width = std::min(p.piece, d->V - v0);
        // x goes with the first piece of w
        LceOperand px, pw;
        if (!direct_x && v0 == 0) px = LceOperand{x, r0, rows, d->ldx, sp.x, target + r0};
        if (p.pack_w) pw = LceOperand{w, v0, width, d->ldw, sp.w, nullptr};
        PVB2_TRY(lce_pack(d, p, px, pw, lce_no_rows(), scale, s));
        if (!p.pack_w) PVB2_TRY(lce_map_b(&mb, w, d->D, d->V, d->ldw, p, p.z.bn));
        else PVB2_TRY(lce_map_b(&mb, sp.w, d->D, width, p.ldp, p, p.z.bn));
        LceGemm g = lce_logits(d, bias, rows, v0, width, p.pack_w ? 0 : (int)v0, target + r0);
        if (slabs) {
          PVB2_TRY(lce_slab_logits(d, p, ma, mb, g, sp.slab, s));
        } else {
          g.zscale = zscale;
          g.part = sp.part;
          g.zsum = smoothing != 0.f ? sp.zsum : nullptr;
          g.ztarget = d->kept ? k.ztarget + r0 : sp.ztarget;
          g.part_ld = rows;
          CUtensorMap mk = no_map();
          if (d->kept) {
            g.keep = (int)d->kept;
            g.keep_max = k.max + r0;
            g.keep_ld = d->N;
            if (k.fp32) PVB2_TRY(lce_map32(&mk, (float*)k.data + r0 * k.ld, d->kept, rows, k.ld, 1));
            else PVB2_TRY(lce_map(&mk, (uint16_t*)k.data + r0 * k.ld, d->kept, rows, k.ld, 1, 32, true));
          }
          PVB2_TRY(lce_gemm<kEpiStats>(ma, mb, mk, g, false, false, p, p.z.bn, s));
        }
      }
      if (slabs) {
        // two logits a thread (7663 rows of 24: 117 us with 512 threads, 10 with 32)
        int threads = 32;
        while (threads < 512 && 2 * threads < d->V) threads *= 2;
        lce_slab_rows_kernel<<<(int)rows, threads, 0, s>>>(
            sp.slab, p.z.splits, rows, up(d->V, 4), bias, d->dtype, target + r0, d->V, d->ignore_index, smoothing,
            lse + r0, loss + r0, (float*)k.data + r0 * k.ld, d->kept, k.ld, d->kept ? k.ztarget + r0 : nullptr,
            zscale);
      } else {
        lce_rows_kernel<<<(int)cdiv(rows, 32), 1024, 0, s>>>(
            sp.part, smoothing != 0.f ? sp.zsum : nullptr, rows, parts, d->kept ? k.ztarget + r0 : sp.ztarget,
            target + r0, rows, d->V, d->ignore_index, smoothing, lse + r0, loss + r0);
      }
      PVB2_LAUNCH_CHECK();
    }
  }
  lce_total_kernel<<<1, 1024, 0, s>>>(loss, target, d->N, d->V, d->ignore_index, d->reduction, out, count);
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

size_t pvb2_linear_ce_keep(pvb2_linear_ce_desc* desc, size_t budget) {
  if (!desc) return 0;
  desc->kept = 0;
  if (lce_check(desc) != PVB2_OK || desc->N == 0) return 0;
  const pvb2_linear_ce_desc normal = lce_normal(desc);
  const bool fp32 = lce_kept_fp32(&normal);
  // an entry takes its number for each row, and its share of the maxima
  const double entry = (double)desc->N * (fp32 ? 4 : 2 + 4.0 / 64);
  const int64_t fit = (int64_t)std::min<double>((double)desc->V, (double)budget / entry);
  desc->kept = fit >= desc->V ? desc->V : fit / 256 * 256;
  if (desc->kept < std::min<int64_t>(desc->V, 1024)) desc->kept = 0;
  if (desc->kept == 0) return 0;
  LceKept k;
  return lce_kept_space(desc, fp32, nullptr, &k);
}

size_t pvb2_linear_ce_bwd_workspace_size(const pvb2_linear_ce_desc* desc) {
  if (lce_check(desc) != PVB2_OK || desc->N == 0) return 0;
  const pvb2_linear_ce_desc normal = lce_normal(desc), *d = &normal;
  LceBwdSpace s;
  return lce_bwd_space(d, lce_plan(d, true), nullptr, &s) + 1024;
}

int pvb2_linear_ce_bwd(const pvb2_linear_ce_desc* desc, const void* x, const void* w, const void* bias,
                       const int64_t* target, const float* lse, const float* count, const void* kept,
                       const float* grad_out, void* dx, void* dw, void* dbias, void* workspace, size_t workspace_bytes, pvb2_stream stream) {
  PVB2_TRY(lce_check(desc));
  const pvb2_linear_ce_desc normal = lce_normal(desc), *d = &normal;
  cudaStream_t s = as_stream(stream);
  const int size = d->dtype == PVB2_F32 ? 4 : 2;
  if (d->N == 0) {
    if (dw) PVB2_CUDA_TRY(cudaMemsetAsync(dw, 0, (size_t)d->V * d->D * size, s));
    if (dbias) PVB2_CUDA_TRY(cudaMemsetAsync(dbias, 0, (size_t)d->V * size, s));
    return PVB2_OK;
  }
  PVB2_CHECK_ARG(x && w && target && lse && count && grad_out, "linear cross entropy backward: null pointer");
  PVB2_CHECK_ARG(d->kept == 0 || (kept && ((uintptr_t)kept & 15) == 0),
                 "linear cross entropy backward: what the forward pass kept is missing");
  if (!dx && !dw && !dbias) return PVB2_OK;
  const LcePlan p = lce_plan(d, true);
  LceBwdSpace sp;
  const size_t need = lce_bwd_space(d, p, (void*)(((uintptr_t)workspace + 1023) & ~(uintptr_t)1023), &sp) + 1024;
  PVB2_CHECK_ARG(workspace && workspace_bytes >= need, "linear cross entropy backward: workspace of %zu bytes needed",
                 need);
  const bool direct_w = !p.pack_w, slabs = lce_slabs(p);
  PVB2_TRY(lce_aligned(w, direct_w));
  const float gscale = p.half ? 32768.f : 1.f;
  // the forward pass found the scales, unless its rows were few
  LceScaleJob scale{};
  const bool given = p.P == 2 && !lce_few_rows(d, p.ldp);
  if (given) scale.given = count + 1;
  else PVB2_TRY(lce_scales(d, p, x, w, target, sp.absmax, sp.scales, &scale, s));
  const float* zscale = given ? count + 1 : p.P == 2 ? sp.scales : nullptr;
  LceRowsJob rows = lce_no_rows();
  if (d->reduction != PVB2_LOSS_NONE)
    rows = LceRowsJob{sp.row, sp.own, sp.factor, grad_out, count, target, d->N, d->reduction == PVB2_LOSS_MEAN,
                      1.f / gscale};
  const bool own = d->reduction == PVB2_LOSS_NONE;  // each row has its own gradient
  bool row_factors = !own;                          // or still to be formed, after the scales
  const LceScale dx_scale{sp.factor + 1, nullptr, sp.own};
  const LceScale dw_scale{sp.factor + 2, sp.factor + 3, nullptr};
  LceOperand px{x, 0, d->N, d->ldx, sp.x, target};
  CUtensorMap x_k, x_mn, w_k, w_mn, g_store, g_k, g_mn, acc;
  PVB2_TRY(lce_map_a(&x_k, sp.x, d->D, d->N, p.ldp, p));
  PVB2_TRY(lce_map_mn(&x_mn, sp.x, d->D, d->N, p.ldp, p));
  LceKept k;
  if (d->kept) lce_kept_space(d, lce_kept_fp32(d), kept, &k);
  const int64_t ld32 = up(d->D, 4);
  // a piece ends where the kept entries do
  const bool dx_slabs = p.piece < d->V || (d->kept > 0 && d->kept < d->V) || p.dx.splits > 1;
  for (int64_t v0 = 0, end; v0 < d->V; v0 = end) {
    end = std::min(d->V, v0 + p.piece);
    if (v0 < d->kept && end > d->kept) end = d->kept;
    const int64_t width = end - v0, ldg = up(width, 64);
    const bool from_kept = v0 < d->kept;
    const int row0 = direct_w ? (int)v0 : 0;
    if (direct_w) {
      PVB2_TRY(lce_map_b(&w_k, w, d->D, d->V, d->ldw, p, p.z.bn));
      PVB2_TRY(lce_map_mn(&w_mn, w, d->D, d->V, d->ldw, p));
    } else if (dx || !from_kept) {
      PVB2_TRY(lce_pack(d, p, px, LceOperand{w, v0, width, d->ldw, sp.w, nullptr}, rows, scale, s));
      px = LceOperand();
      rows = lce_no_rows();
      PVB2_TRY(lce_map_b(&w_k, sp.w, d->D, width, p.ldp, p, p.z.bn));
      PVB2_TRY(lce_map_mn(&w_mn, sp.w, d->D, width, p.ldp, p));
    }
    // x and the rows' factors, unless they went with w
    PVB2_TRY(lce_pack(d, p, px, LceOperand(), rows, scale, s));
    px = LceOperand();
    rows = lce_no_rows();
    if (!row_factors) {
      lce_grad_rows_kernel<<<1, 1024, 0, s>>>(grad_out, target, d->N, d->V, d->ignore_index, 1.f / gscale,
                                              zscale, sp.row, sp.one, sp.own, sp.factor);
      PVB2_LAUNCH_CHECK();
      row_factors = true;
    }
    PVB2_TRY(lce_map_a(&g_k, sp.G, width, d->N, ldg, p));
    PVB2_TRY(lce_map_mn(&g_mn, sp.G, width, d->N, ldg, p));
    // G of this piece, for one kind of row factors
    bool logits = false;  // those of the slabs are there
    auto form = [&](const float* grow) {
      if (from_kept) {
        if (p.half) return lce_kept_grad<__half>(d, p, sp, k, target, lse, grow, v0, width, ldg, gscale, s);
        return lce_kept_grad<__nv_bfloat16>(d, p, sp, k, target, lse, grow, v0, width, ldg, gscale, s);
      }
      LceGemm g = lce_logits(d, bias, d->N, v0, width, row0, target);
      if (slabs) {
        if (!logits) PVB2_TRY(lce_slab_logits(d, p, x_k, w_k, g, sp.slab, s));
        logits = true;
        if (p.half)
          return lce_slab_grad<__half>(d, p, sp, bias, target, lse, grow, v0, width, ldg, gscale, zscale, s);
        return lce_slab_grad<__nv_bfloat16>(d, p, sp, bias, target, lse, grow, v0, width, ldg, gscale, zscale, s);
      }
      g.lse = lse;
      g.grow = grow;
      g.zscale = zscale;
      g.gscale = gscale;
      PVB2_TRY(lce_map(&g_store, sp.G, width, d->N, ldg, p.P, 32, p.half));
      return lce_gemm<kEpiGrad>(x_k, w_k, g_store, g, false, false, p, p.z.bn, s);
    };
    PVB2_TRY(form(dx && own ? sp.one : sp.row));
    if (dx) {
      LceGemm h = lce_product(d->N, d->D, width, row0, p.dx);
      if (dx_slabs) {
        // the first piece is the widest; a shorter one leaves the far slabs alone
        if (p.dx.splits > 1) h.splits = (int)std::min<int64_t>(h.splits, cdiv(cdiv(width, kLBK), h.kb_per));
        h.accumulate = v0 > 0;
        PVB2_TRY(lce_map32(&acc, sp.dx, d->D, d->N, ld32, p.dx.splits));
        PVB2_TRY(lce_gemm<kEpiAcc>(g_k, w_mn, acc, h, false, true, p, p.dx.bn, s));
      } else {
        PVB2_TRY(lce_out(d, p, g_k, w_mn, h, false, d->N, dx, dx_scale, p.dx.bn, s));
      }
      if (own && (dw || dbias)) PVB2_TRY(form(sp.row));
    }
    if (dw) {
      LceGemm h = lce_product(width, d->D, d->N, 0, p.dw);
      void* out = (uint8_t*)dw + v0 * d->D * size;
      if (p.dw.splits > 1) {
        PVB2_TRY(lce_map32(&acc, sp.dw, d->D, width, ld32, p.dw.splits));
        PVB2_TRY(lce_gemm<kEpiAcc>(g_mn, x_mn, acc, h, true, true, p, p.dw.bn, s));
        PVB2_TRY(lce_join(d, sp.dw, p.dw.splits, width, dw_scale, out, s));
      } else {
        PVB2_TRY(lce_out(d, p, g_mn, x_mn, h, true, width, out, dw_scale, p.dw.bn, s));
      }
    }
    if (dbias) {
      void* out = (uint8_t*)dbias + v0 * size;
      PVB2_TRY(lce_bias_grad(d, p, sp, width, ldg, out, s));
    }
  }
  if (dx && dx_slabs) PVB2_TRY(lce_join(d, sp.dx, p.dx.splits, d->N, dx_scale, dx, s));
  return PVB2_OK;
}

int pvb2_linear_ce_status(int* timed_out, int reset) { return tc_timeout_flag_local(timed_out, reset); }

}  // extern "C"
