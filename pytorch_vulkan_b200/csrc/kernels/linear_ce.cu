// Softmax cross entropy of a linear layer over a large vocabulary, z = x w^T + b,
// and its gradients, without keeping z.
//
//   lse_i = log sum_j exp z_ij      loss_i = lse_i - (1 - s) z_i,t(i) - s / V sum_j z_ij
//   G_ij  = g_i (exp(z_ij - lse_i) - (1 - s) [j = t(i)] - s / V)
//   dx = G w     dw = G^T x     db = sum_i G_i
//
// Forward: one matrix product whose epilogue keeps, per row and half tile of
// 128 columns, the largest logit, the sum of exp(z - largest) and the target's
// logit; a second launch joins them.  The logits never leave the chip.
// Backward: per piece of the vocabulary, the logits are formed again and their
// epilogue writes G in 16 bits (piece x tokens, sized to stay near the L2
// cache); two products make dx += G w and the piece's rows of dw = G^T x.
// Going by pieces of the vocabulary finishes dw in one go and adds dx up in
// fp32: 8 N V D operations instead of the 6 that a stored z would take.
//
// Operands are 16-bit (tcgen05 kind::f16, fp32 accumulators).  fp32 operands
// are split into P bf16 numbers each, x = x0 + x1 + x2 (8 bits apiece), and
// the product is the sum of the pairs whose sizes matter: 6 of 9 for P = 3
// (what is left out is below 2^-24 of |x||w|), 3 of 4 for P = 2.  The loop
// over K simply runs over the pairs as well, smallest first.
//
// fp16 keeps G in range by scaling: G is formed for |g_i| / max|g| and times
// 2^15, undone on the fp32 results.
#include <algorithm>
#include <atomic>
#include "tc_common.cuh"
#include "types.cuh"

namespace pvb2 {

constexpr int kLBM = 128, kLBN = 256, kLBK = 64;
constexpr int kLProducers = 4, kLMmaWarp = 4, kLEpiWarps = 8;
constexpr int kLThreads = (kLProducers + 1 + kLEpiWarps) * 32;

struct LceSmem {
  static constexpr int A_BYTES = kLBM * kLBK * 2;
  static constexpr int B_BYTES = kLBN * kLBK * 2;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = 4;
  static constexpr int EPI_OFF = STAGES * STAGE_BYTES;  // one 4 KB store box per epilogue warp
  static constexpr int BAR_OFF = EPI_OFF + kLEpiWarps * 4096;
  static constexpr int TOTAL = BAR_OFF + (2 * STAGES + 4) * 8 + 16;
};

enum { kEpiStats = 0, kEpiGrad = 1, kEpiAcc = 2, kEpiOut = 3 };

struct LceGemm {
  int M, N, K;
  int a_row0, b_row0;     // where the operands' rows (K-major) or K rows (MN-major) begin in their maps
  int nseg;               // pairs of operand planes
  int8_t pa[6], pb[6];
  int n_fast;             // tile order: columns fastest
  int splits, kb_per;     // kEpiAcc: split s takes k blocks [s kb_per, (s + 1) kb_per) into slab s
  // epilogues of logits: column n is vocabulary entry v0 + n
  int v0;
  const void* bias;
  int bias_dtype;
  const int64_t* target;
  int64_t V, ignore;
  float smoothing;
  float2* part;           // kEpiStats: [2 column tiles][part_ld]
  float* zsum;            // kEpiStats with smoothing: sums of z, laid out as part
  float* ztarget;
  int64_t part_ld;
  const float* lse;       // kEpiGrad
  const float* grow;      // kEpiGrad: g_i / max|g| (0 for rows without a loss)
  int planes;             // kEpiGrad: planes of G
  float gscale;
  // kEpiAcc / kEpiOut
  int accumulate;         // kEpiAcc: add to the slab
  void* out;              // kEpiOut without a tensor map
  int64_t out_ld;
  int out_dtype, out_tma;
  const float* out_scale; // kEpiOut: factor on the device
};

__device__ __forceinline__ float lce_bias(const LceGemm& p, int n) {
  if (!p.bias) return 0.f;
  return load_as<float>(p.bias, p.v0 + n, p.bias_dtype);
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

template <int EPI, typename T, bool PRECISE>
__global__ void __launch_bounds__(kLThreads, 1)
    lce_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmC, const __grid_constant__ LceGemm p, int a_mn, int b_mn) {
  using L = LceSmem;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  constexpr int kStages = L::STAGES;
  uint64_t* full = (uint64_t*)(smem + L::BAR_OFF);
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = (uint32_t*)(acc_empty + 2);
  volatile int* abort = (volatile int*)(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles_m = (p.M + kLBM - 1) / kLBM, tiles_n = (p.N + kLBN - 1) / kLBN;
  const int base_tiles = tiles_m * tiles_n, total_tiles = base_tiles * p.splits;
  const int kblocks = (p.K + kLBK - 1) / kLBK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], kLEpiWarps);
    }
    *abort = 0;
    fence_barrier_init();
  }
  if (warp == kLMmaWarp) tmem_alloc(tmem_slot, 2 * kLBN);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // tile -> block row, block column, split
  auto place = [&](int tile, int& mb, int& nb, int& sp) {
    sp = tile / base_tiles;
    const int t = tile % base_tiles;
    mb = p.n_fast ? t / tiles_n : t % tiles_m;
    nb = p.n_fast ? t % tiles_n : t / tiles_m;
  };

  if (warp < kLProducers) {
    if (lane == 0) {
      tma_prefetch(&tmA);
      tma_prefetch(&tmB);
      uint32_t it = 0;
      for (int tile = blockIdx.x; tile < total_tiles && !*abort; tile += gridDim.x) {
        int mb, nb, sp;
        place(tile, mb, nb, sp);
        const int kb0 = sp * p.kb_per, kb1 = min(kblocks, kb0 + p.kb_per);
        for (int seg = 0; seg < p.nseg; ++seg) {
          const int za = p.pa[seg], zb = p.pb[seg];
          for (int kb = kb0; kb < kb1; ++kb, ++it) {
            const int s = it % kStages;
            const uint32_t ph = (it / kStages) & 1;
            if ((int)(it % kLProducers) != warp) continue;
            if (!mbar_wait(&empty[s], ph ^ 1, abort)) break;
            uint8_t* sa = smem + s * L::STAGE_BYTES;
            uint8_t* sb = sa + L::A_BYTES;
            mbar_arrive_expect_tx(&full[s], L::STAGE_BYTES);
            if (!a_mn) {
              tma_load_3d(sa, &tmA, &full[s], kb * kLBK, p.a_row0 + mb * kLBM, za);
            } else {
#pragma unroll
              for (int j = 0; j < kLBM / 64; ++j)
                tma_load_3d(sa + j * 8192, &tmA, &full[s], mb * kLBM + 64 * j, p.a_row0 + kb * kLBK, za);
            }
            if (!b_mn) {
              tma_load_3d(sb, &tmB, &full[s], kb * kLBK, p.b_row0 + nb * kLBN, zb);
            } else {
#pragma unroll
              for (int j = 0; j < kLBN / 64; ++j)
                tma_load_3d(sb + j * 8192, &tmB, &full[s], nb * kLBN + 64 * j, p.b_row0 + kb * kLBK, zb);
            }
          }
        }
      }
    }
  } else if (warp == kLMmaWarp) {
    if (lane == 0) {
      const uint32_t idesc = idesc_f16(kLBM, kLBN, sizeof(T) == 2 && !std::is_same<T, __half>::value, a_mn, b_mn);
      uint32_t it = 0;
      int local = 0;
      for (int tile = blockIdx.x; tile < total_tiles && !*abort; tile += gridDim.x, ++local) {
        int mb, nb, sp;
        place(tile, mb, nb, sp);
        const int buf = local & 1;
        if (!mbar_wait(&acc_empty[buf], ((local >> 1) & 1) ^ 1, abort)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * kLBN;
        const int kb0 = sp * p.kb_per, kb1 = min(kblocks, kb0 + p.kb_per);
        const int iters = (kb1 - kb0) * p.nseg;
        for (int k = 0; k < iters; ++k, ++it) {
          const int s = it % kStages;
          if (!mbar_wait(&full[s], (it / kStages) & 1, abort)) break;
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + s * L::STAGE_BYTES);
          const uint32_t sb = sa + L::A_BYTES;
#pragma unroll
          for (int kk = 0; kk < kLBK / 16; ++kk) {
            const uint64_t ad = a_mn ? desc_mnmajor16(sa, kk, 8192) : desc_kmajor(sa, kk);
            const uint64_t bd = b_mn ? desc_mnmajor16(sb, kk, 8192) : desc_kmajor(sb, kk);
            mma_f16(d_tmem, ad, bd, idesc, (k > 0 || kk > 0) ? 1u : 0u);
          }
          mma_commit(&empty[s]);
        }
        mma_commit(&acc_full[buf]);
      }
    }
  } else {
    // epilogue warps: TMEM lane quarter warp % 4, column half (warp - 5) / 4
    const int quarter = warp & 3, half = (warp - kLMmaWarp - 1) >> 2;
    uint8_t* box = smem + L::EPI_OFF + (warp - kLMmaWarp - 1) * 4096;
    int local = 0;
    for (int tile = blockIdx.x; tile < total_tiles && !*abort; tile += gridDim.x, ++local) {
      int mb, nb, sp;
      place(tile, mb, nb, sp);
      const int buf = local & 1;
      const int m0 = mb * kLBM + quarter * 32, m = m0 + lane;
      const bool mrow = m < p.M;
      const int nh = nb * kLBN + half * 128;  // first column of this warp
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
      const float oscale = EPI == kEpiOut && p.out_scale ? *p.out_scale : 1.f;
      if (!mbar_wait(&acc_full[buf], (local >> 1) & 1, abort)) break;
      tc_fence_after();
      float mx = -INFINITY, sum = 0.f, zs = 0.f;
#pragma unroll 1
      for (int c = 0; c < 2; ++c) {  // 64 columns at a time
        const int n0 = nh + c * 64;
        if (n0 >= p.N) break;
        float v[64];
        const uint32_t ta = tmem_base + ((uint32_t)(quarter * 32) << 16) + buf * kLBN + half * 128 + c * 64;
        tmem_ld32(ta, v);
        tmem_ld32(ta + 32, v + 32);
        if (EPI == kEpiStats) {
          float cm = -INFINITY;
#pragma unroll
          for (int j = 0; j < 64; ++j) {
            const bool in = n0 + j < p.N;
            if (p.bias && in) v[j] += lce_bias(p, n0 + j);
            if (p.zsum && in) zs += v[j];
            if (t == n0 + j) p.ztarget[m] = v[j];
            if (!in) v[j] = -INFINITY;
            // a NaN logit makes the row's sum NaN by exp below
            cm = fmaxf(cm, v[j]);
          }
          const float nm = fmaxf(mx, cm);
          const float base = nm == -INFINITY ? 0.f : nm;
          sum *= lce_exp<PRECISE>(mx - base);
#pragma unroll
          for (int j = 0; j < 64; ++j) sum += lce_exp<PRECISE>(v[j] - base);
          mx = nm;
        } else if (EPI == kEpiGrad) {
          const float flat = p.smoothing / (float)p.V;
#pragma unroll
          for (int j = 0; j < 64; ++j) {
            const float z = v[j] + (p.bias && n0 + j < p.N ? lce_bias(p, n0 + j) : 0.f);
            float e = lce_exp<PRECISE>(z - row_lse) - flat;
            if (t == n0 + j) e -= 1.f - p.smoothing;
            v[j] = row_g == 0.f ? 0.f : e * row_g * p.gscale;
          }
          if (m0 < p.M) {
            for (int z = 0; z < p.planes; ++z) {
              store_box(box, lane, [&](int phase) {
                if (phase == 0) box16<T>(box, lane, v);
                else tma_store_3d(&tmC, box, n0, m0, z);
              });
              if (z + 1 < p.planes) {
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
          for (int j = 0; j < 64; ++j) v[j] *= oscale;
          if (!p.out_tma) {
            if (mrow) {
              const int64_t row = (int64_t)m * p.out_ld;
              for (int j = 0; j < 64; ++j)
                if (n0 + j < p.N) store_as<float>(p.out, row + n0 + j, p.out_dtype, v[j]);
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
        const int64_t at = (int64_t)(p.v0 / 128 + nh / 128) * p.part_ld + m;
        p.part[at] = make_float2(mx, sum);
        if (p.zsum) p.zsum[at] = zs;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[buf]);
    }
    if (lane == 0) bulk_wait_all();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kLMmaWarp) {
    if (*abort) {
      // let any MMA still in flight finish before the columns are released
      if (lane == 0) mma_commit(&acc_full[0]);
      __syncwarp();
      const uint64_t t0 = globaltimer();
      while (globaltimer() - t0 < 10000000ull) {
      }
    }
    tc_fence_after();
    tmem_dealloc(tmem_base, 2 * kLBN);
  }
}

// ------------------------------------------------------------ small kernels
// src [rows][cols] (row stride ld) -> planes [P][rows][ldp] of T, columns
// from cols to ldp zero; rows without a loss become zeros when `target` is
// given (what they hold, NaN among it, then has no part in a product)
template <typename S, typename T>
__global__ void lce_pack_kernel(const S* __restrict__ src, int64_t rows, int64_t cols, int64_t ld, T* __restrict__ dst,
                                int64_t ldp, int planes, const int64_t* __restrict__ target, int64_t V,
                                int64_t ignore) {
  const int64_t total = rows * ldp, plane = rows * ldp;
  for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < total; e += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = e / ldp, c = e % ldp;
    float v = c < cols ? to_f32(src[r * ld + c]) : 0.f;
    if (target && !lce_scored(target[r], V, ignore)) v = 0.f;
    for (int z = 0; z < planes; ++z) {
      const T h = from_f32<T>(v);
      dst[z * plane + e] = h;
      // infinity is its first part alone
      v = isinf(to_f32(h)) ? 0.f : v - to_f32(h);
    }
  }
}

// joins the parts of each row: lse and loss (0 for rows without one).  32
// rows a block, 8 threads a row.
__global__ void __launch_bounds__(256)
    lce_rows_kernel(const float2* __restrict__ part, const float* __restrict__ zsum, int64_t part_ld, int parts,
                    const float* __restrict__ ztarget, const int64_t* __restrict__ target, int64_t N, int64_t V,
                    int64_t ignore, float smoothing, float* __restrict__ lse, float* __restrict__ loss) {
  __shared__ float sm[8][32], ss[8][32], sz[8][32];
  const int r = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t i = (int64_t)blockIdx.x * 32 + r;
  float mx = -INFINITY, sum = 0.f, zs = 0.f;
  if (i < N) {
    for (int q = g; q < parts; q += 8) {
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
  if (g == 0 && i < N) {
    for (int q = 1; q < 8; ++q) {
      const float nm = fmaxf(mx, sm[q][r]), base = nm == -INFINITY ? 0.f : nm;
      sum = sum * expf(mx - base) + ss[q][r] * expf(sm[q][r] - base);
      mx = nm;
      zs += sz[q][r];
    }
    const float l = (mx == -INFINITY ? 0.f : mx) + logf(sum);
    lse[i] = l;
    float v = 0.f;
    if (lce_scored(target[i], V, ignore)) {
      v = l - ztarget[i];
      if (smoothing != 0.f) v = (1.f - smoothing) * v + smoothing * (l - zs / (float)V);
    }
    loss[i] = v;
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

// what each row's gradient is multiplied by: row[i] in [-1, 1] and one factor
// for all results
__global__ void __launch_bounds__(1024)
    lce_grad_rows_kernel(const float* __restrict__ grad_out, const float* __restrict__ count,
                         const int64_t* __restrict__ target, int64_t N, int64_t V, int64_t ignore, int reduction,
                         float inv_gscale, float* __restrict__ row, float* __restrict__ factor) {
  __shared__ float s_max[32];
  float scale;
  if (reduction == PVB2_LOSS_NONE) {
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
    scale = mx;
  } else {
    scale = *grad_out;
    if (reduction == PVB2_LOSS_MEAN) scale = *count > 0.f ? scale / *count : 0.f;
  }
  for (int64_t i = threadIdx.x; i < N; i += 1024) {
    float g = 0.f;
    if (lce_scored(target[i], V, ignore)) g = reduction == PVB2_LOSS_NONE ? (scale != 0.f ? grad_out[i] / scale : 0.f) : 1.f;
    row[i] = g;
  }
  if (threadIdx.x == 0) *factor = scale * inv_gscale;
}

// out [rows][cols] = factor * sum of S slabs [rows][ld]
template <typename T>
__global__ void lce_join_kernel(const float* __restrict__ slab, int S, int64_t rows, int64_t cols, int64_t ld,
                                const float* __restrict__ factor, T* __restrict__ out) {
  const float f = *factor;
  const int64_t total = rows * cols, size = rows * ld;
  for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < total; e += (int64_t)gridDim.x * blockDim.x) {
    const int64_t at = e / cols * ld + e % cols;
    float v = slab[at];
    for (int s = 1; s < S; ++s) v += slab[s * size + at];
    out[e] = from_f32<T>(v * f);
  }
}

// column sums of G (planes added), 64 rows a thread row: partial sums first,
// then in order
template <typename T>
__global__ void __launch_bounds__(256) lce_colsum_kernel(const T* __restrict__ G, int64_t rows, int64_t cols, int64_t ld,
                                                         int planes, int64_t rows_per, float* __restrict__ part) {
  __shared__ float s[8][33];
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t col = (int64_t)blockIdx.x * 32 + c;
  const int64_t r0 = blockIdx.y * rows_per, r1 = min(rows, r0 + rows_per);
  float sum = 0.f;
  if (col < cols)
    for (int64_t r = r0 + g; r < r1; r += 8) {
      float v = 0.f;
      for (int z = planes - 1; z >= 0; --z) v += to_f32(G[(z * rows + r) * ld + col]);
      sum += v;
    }
  s[g][c] = sum;
  __syncthreads();
  if (g == 0 && col < cols) {
    for (int q = 1; q < 8; ++q) sum += s[q][c];
    part[blockIdx.y * cols + col] = sum;
  }
}

template <typename T>
__global__ void lce_dbias_kernel(const float* __restrict__ part, int parts, int64_t cols,
                                 const float* __restrict__ factor, T* __restrict__ out) {
  const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= cols) return;
  double s = 0.0;
  for (int q = 0; q < parts; ++q) s += (double)part[q * cols + c];
  out[c] = from_f32<T>((float)(s * (double)*factor));
}

// --------------------------------------------------------------- host side
static int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

struct LcePlan {
  int P;             // planes of an operand
  int nseg;
  bool half;         // fp16 operands (bf16 otherwise)
  int64_t ldp;       // row length of packed operands
  bool pack_w;       // w is packed piece by piece
  int64_t piece;     // vocabulary entries of a piece (backward; forward where w is packed)
  int pieces;
  // backward
  int dx_splits, dx_kb;
  int dw_splits, dw_kb;
  int colsum_parts;
  int64_t rows_per;
};



// 16-bit operands whose rows begin on 16-byte boundaries are read as they lie
static bool lce_direct(const pvb2_linear_ce_desc* d, int64_t ld) { return d->dtype != PVB2_F32 && ld % 8 == 0; }

// with one row the stride says nothing
static pvb2_linear_ce_desc lce_normal(const pvb2_linear_ce_desc* d) {
  pvb2_linear_ce_desc n = *d;
  if (n.N <= 1) n.ldx = up(n.D, 8);
  if (n.V <= 1) n.ldw = up(n.D, 8);
  return n;
}

// K of a product with few tiles is cut so that every SM has one: at least 8
// blocks of K each
static void lce_split(int64_t M, int64_t N, int64_t K, int* splits, int* kb_per) {
  const int64_t tiles = up(M, kLBM) / kLBM * (up(N, kLBN) / kLBN), kb = up(K, kLBK) / kLBK;
  int64_t s = std::max<int64_t>(1, std::min<int64_t>(num_sms() / tiles, kb / 8));
  *kb_per = (int)((kb + s - 1) / s);
  *splits = (int)((kb + *kb_per - 1) / *kb_per);
}

static LcePlan lce_plan(const pvb2_linear_ce_desc* d, bool backward) {
  LcePlan p;
  p.half = d->dtype == PVB2_F16;
  p.P = d->dtype != PVB2_F32 ? 1 : d->math == PVB2_MATH_FP32 ? 3 : 2;
  p.nseg = p.P == 1 ? 1 : p.P == 2 ? 3 : 6;
  p.ldp = up(d->D, 8);
  p.pack_w = !lce_direct(d, d->ldw);
  // G of a piece in about 128 MB, the packed piece of w in about 256 MB, at
  // least 1024 entries
  int64_t piece = backward ? ((int64_t)128 << 20) / (std::max<int64_t>(d->N, 1) * 2 * p.P) : d->V;
  if (p.pack_w) piece = std::min<int64_t>(piece, ((int64_t)256 << 20) / (p.ldp * 2 * p.P));
  piece = std::max<int64_t>(1024, piece / kLBN * kLBN);
  p.piece = std::min<int64_t>(piece, up(d->V, kLBN));
  p.pieces = (int)((d->V + p.piece - 1) / p.piece);
  const int64_t width = std::min(p.piece, d->V);
  lce_split(d->N, d->D, width, &p.dx_splits, &p.dx_kb);
  lce_split(width, d->D, d->N, &p.dw_splits, &p.dw_kb);
  p.colsum_parts = (int)std::min<int64_t>(64, (d->N + 255) / 256);
  p.rows_per = p.colsum_parts ? up((d->N + p.colsum_parts - 1) / p.colsum_parts, 8) : 0;
  return p;
}

constexpr int64_t kLRowsFwd = 16384;  // rows whose parts are held at a time

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

struct LceFwdSpace {
  uint16_t *x, *w;
  float2* part;
  float *zsum, *ztarget, *loss;
};

static size_t lce_fwd_space(const pvb2_linear_ce_desc* d, const LcePlan& p, void* base, LceFwdSpace* s) {
  Arena a{(uint8_t*)base};
  const int64_t rows = std::min(d->N, kLRowsFwd), parts = up(d->V, kLBN) / 128;
  s->x = a.take<uint16_t>(lce_direct(d, d->ldx) ? 0 : rows * p.ldp * p.P);
  s->w = a.take<uint16_t>(p.pack_w ? p.piece * p.ldp * p.P : 0);
  s->part = a.take<float2>(rows * parts);
  s->zsum = a.take<float>(d->label_smoothing != 0 ? rows * parts : 0);
  s->ztarget = a.take<float>(rows);
  s->loss = a.take<float>(d->N);
  return a.at;
}

struct LceBwdSpace {
  uint16_t *x, *w, *G;
  float *row, *factor, *dx, *dw, *colsum;
};

static size_t lce_bwd_space(const pvb2_linear_ce_desc* d, const LcePlan& p, void* base, LceBwdSpace* s) {
  Arena a{(uint8_t*)base};
  const int64_t ld32 = up(d->D, 4);
  s->x = a.take<uint16_t>(d->N * p.ldp * p.P);
  s->w = a.take<uint16_t>(p.pack_w ? p.piece * p.ldp * p.P : 0);
  s->G = a.take<uint16_t>(d->N * p.piece * p.P);
  s->row = a.take<float>(d->N);
  s->factor = a.take<float>(1);
  s->dx = a.take<float>(p.pieces > 1 || p.dx_splits > 1 ? p.dx_splits * d->N * ld32 : 0);
  s->dw = a.take<float>(p.dw_splits > 1 ? p.dw_splits * p.piece * ld32 : 0);
  s->colsum = a.take<float>(p.colsum_parts * p.piece);
  return a.at;
}

static int lce_check(const pvb2_linear_ce_desc* d) {
  PVB2_CHECK_ARG(d, "linear cross entropy: no descriptor");
  PVB2_CHECK_ARG(d->dtype == PVB2_F32 || d->dtype == PVB2_F16 || d->dtype == PVB2_BF16,
                 "linear cross entropy: fp32, fp16 or bf16 expected (got dtype %d)", d->dtype);
  PVB2_CHECK_ARG(d->reduction >= PVB2_LOSS_NONE && d->reduction <= PVB2_LOSS_SUM,
                 "linear cross entropy: unknown reduction %d", d->reduction);
  PVB2_CHECK_ARG(d->math == PVB2_MATH_FP32 || d->math == PVB2_MATH_TF32, "linear cross entropy: unknown math mode %d",
                 d->math);
  PVB2_CHECK_ARG(d->N >= 0 && d->V >= 1 && d->D >= 1 && d->N < (1 << 24) && d->V < (1 << 24) && d->D < (1 << 20),
                 "linear cross entropy: sizes N=%lld D=%lld V=%lld out of range", (long long)d->N, (long long)d->D,
                 (long long)d->V);
  PVB2_CHECK_ARG((d->N <= 1 || d->ldx >= d->D) && (d->V <= 1 || d->ldw >= d->D),
                 "linear cross entropy: row strides below the row length");
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

static void lce_segments(LceGemm* g, const LcePlan& p) {
  static const int8_t a3[6] = {2, 0, 1, 1, 0, 0}, b3[6] = {0, 2, 1, 0, 1, 0};
  static const int8_t a2[3] = {1, 0, 0}, b2[3] = {0, 1, 0};
  g->nseg = p.nseg;
  for (int i = 0; i < p.nseg; ++i) {
    g->pa[i] = p.P == 3 ? a3[i] : p.P == 2 ? a2[i] : 0;
    g->pb[i] = p.P == 3 ? b3[i] : p.P == 2 ? b2[i] : 0;
  }
}

template <int EPI, typename T, bool PRECISE>
static int lce_launch(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& c, const LceGemm& g, bool a_mn,
                      bool b_mn, cudaStream_t s) {
  constexpr int smem = LceSmem::TOTAL + 1024;
  static std::atomic<uint64_t> attr_done{0};
  if (first_on_device(attr_done))
    PVB2_CUDA_TRY(cudaFuncSetAttribute(lce_gemm_kernel<EPI, T, PRECISE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       smem));
  const int64_t tiles = up(g.M, kLBM) / kLBM * (up(g.N, kLBN) / kLBN) * g.splits;
  PVB2_CHECK_ARG(tiles < INT32_MAX / 2, "linear cross entropy: too many tiles");
  const int grid = (int)std::min<int64_t>(tiles, num_sms());
  lce_gemm_kernel<EPI, T, PRECISE><<<grid, kLThreads, smem, s>>>(a, b, c, g, a_mn ? 1 : 0, b_mn ? 1 : 0);
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

template <int EPI>
static int lce_gemm(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& c, const LceGemm& g, bool a_mn,
                    bool b_mn, const LcePlan& p, cudaStream_t s) {
  if (p.half) return lce_launch<EPI, __half, false>(a, b, c, g, a_mn, b_mn, s);
  if ((EPI == kEpiStats || EPI == kEpiGrad) && p.P > 1)
    return lce_launch<EPI, __nv_bfloat16, true>(a, b, c, g, a_mn, b_mn, s);
  return lce_launch<EPI, __nv_bfloat16, false>(a, b, c, g, a_mn, b_mn, s);
}

static int lce_pack(const pvb2_linear_ce_desc* d, const LcePlan& p, const void* src, int64_t row0, int64_t rows,
                    int64_t ld, uint16_t* dst, const int64_t* target, cudaStream_t s) {
  const int64_t total = rows * p.ldp;
  if (total == 0) return PVB2_OK;
  const int grid = grid_for(total, 256);
  if (d->dtype == PVB2_F32)
    lce_pack_kernel<<<grid, 256, 0, s>>>((const float*)src + row0 * ld, rows, d->D, ld, (__nv_bfloat16*)dst, p.ldp, p.P,
                                         target, d->V, d->ignore_index);
  else if (p.half)
    lce_pack_kernel<<<grid, 256, 0, s>>>((const __half*)src + row0 * ld, rows, d->D, ld, (__half*)dst, p.ldp, 1, target,
                                         d->V, d->ignore_index);
  else
    lce_pack_kernel<<<grid, 256, 0, s>>>((const __nv_bfloat16*)src + row0 * ld, rows, d->D, ld, (__nv_bfloat16*)dst,
                                         p.ldp, 1, target, d->V, d->ignore_index);
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

// out = factor * (sum of slabs), as the operands' type
static int lce_join(const pvb2_linear_ce_desc* d, const float* slab, int S, int64_t rows, const float* factor, void* out,
                    cudaStream_t s) {
  const int64_t ld = up(d->D, 4), total = rows * d->D;
  const int grid = grid_for(total, 256);
  if (d->dtype == PVB2_F32) lce_join_kernel<<<grid, 256, 0, s>>>(slab, S, rows, d->D, ld, factor, (float*)out);
  else if (d->dtype == PVB2_F16) lce_join_kernel<<<grid, 256, 0, s>>>(slab, S, rows, d->D, ld, factor, (__half*)out);
  else lce_join_kernel<<<grid, 256, 0, s>>>(slab, S, rows, d->D, ld, factor, (__nv_bfloat16*)out);
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

static void lce_logits(LceGemm* g, const pvb2_linear_ce_desc* d, const LcePlan& p, const void* bias) {
  memset(g, 0, sizeof(*g));
  lce_segments(g, p);
  g->K = (int)d->D;
  g->splits = 1;
  g->kb_per = INT32_MAX / 2;
  g->bias = bias;
  g->bias_dtype = d->dtype;
  g->V = d->V;
  g->ignore = d->ignore_index;
  g->smoothing = (float)d->label_smoothing;
}

// a map that no kernel reads, where an epilogue has none
static CUtensorMap no_map() {
  CUtensorMap m;
  memset(&m, 0, sizeof(m));
  return m;
}

// the product A B into `out` (rows x D), through slabs where K is cut
static int lce_out(const pvb2_linear_ce_desc* d, const LcePlan& p, const CUtensorMap& a, const CUtensorMap& b, LceGemm g,
                   bool a_mn, int64_t rows, void* out, const float* factor, cudaStream_t s) {
  const int size = d->dtype == PVB2_F32 ? 4 : 2;
  CUtensorMap c = no_map();
  g.out = out;
  g.out_ld = d->D;
  g.out_dtype = d->dtype;
  g.out_scale = factor;
  g.out_tma = ((uintptr_t)out & 15) == 0 && d->D * size % 16 == 0;
  if (g.out_tma) {
    if (size == 4) PVB2_TRY(lce_map32(&c, out, d->D, rows, d->D, 1));
    else PVB2_TRY(lce_map(&c, out, d->D, rows, d->D, 1, 32, p.half));
  }
  return lce_gemm<kEpiOut>(a, b, c, g, a_mn, true, p, s);
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
                       const int64_t* target, float* out, float* lse, float* count, void* workspace,
                       size_t workspace_bytes, pvb2_stream stream) {
  PVB2_TRY(lce_check(desc));
  const pvb2_linear_ce_desc normal = lce_normal(desc), *d = &normal;
  PVB2_CHECK_ARG(w && count && (d->N == 0 || (x && target && lse && out)), "linear cross entropy: null pointer");
  cudaStream_t s = as_stream(stream);
  float* loss = out;
  if (d->N > 0) {
    PVB2_CHECK_ARG(workspace && workspace_bytes >= pvb2_linear_ce_fwd_workspace_size(d),
                   "linear cross entropy: workspace of %zu bytes needed", pvb2_linear_ce_fwd_workspace_size(d));
    const LcePlan p = lce_plan(d, false);
    LceFwdSpace sp;
    lce_fwd_space(d, p, (void*)(((uintptr_t)workspace + 1023) & ~(uintptr_t)1023), &sp);
    if (d->reduction != PVB2_LOSS_NONE) loss = sp.loss;
    const bool direct_x = lce_direct(d, d->ldx), direct_w = !p.pack_w;
    PVB2_TRY(lce_aligned(x, direct_x));
    PVB2_TRY(lce_aligned(w, direct_w));
    const int64_t piece = direct_w ? up(d->V, kLBN) : p.piece;
    const int parts = (int)(up(d->V, 128) / 128);
    const int esize = d->dtype == PVB2_F32 ? 4 : 2;
    for (int64_t r0 = 0; r0 < d->N; r0 += kLRowsFwd) {
      const int64_t rows = std::min(kLRowsFwd, d->N - r0);
      CUtensorMap ma, mb;
      if (direct_x) {
        PVB2_TRY(lce_map(&ma, (const uint8_t*)x + r0 * d->ldx * esize, d->D, rows, d->ldx, 1, kLBM, p.half));
      } else {
        PVB2_TRY(lce_pack(d, p, x, r0, rows, d->ldx, sp.x, nullptr, s));
        PVB2_TRY(lce_map(&ma, sp.x, d->D, rows, p.ldp, p.P, kLBM, p.half));
      }
      for (int64_t v0 = 0; v0 < d->V; v0 += piece) {
        const int64_t width = std::min(piece, d->V - v0);
        LceGemm g;
        lce_logits(&g, d, p, bias);
        if (direct_w) {
          PVB2_TRY(lce_map(&mb, w, d->D, d->V, d->ldw, 1, kLBN, p.half));
          g.b_row0 = (int)v0;
        } else {
          PVB2_TRY(lce_pack(d, p, w, v0, width, d->ldw, sp.w, nullptr, s));
          PVB2_TRY(lce_map(&mb, sp.w, d->D, width, p.ldp, p.P, kLBN, p.half));
        }
        g.M = (int)rows;
        g.N = (int)width;
        g.v0 = (int)v0;
        g.target = target + r0;
        g.part = sp.part;
        g.zsum = d->label_smoothing != 0 ? sp.zsum : nullptr;
        g.ztarget = sp.ztarget;
        g.part_ld = rows;
        PVB2_TRY(lce_gemm<kEpiStats>(ma, mb, no_map(), g, false, false, p, s));
      }
      lce_rows_kernel<<<(int)((rows + 31) / 32), 256, 0, s>>>(
          sp.part, d->label_smoothing != 0 ? sp.zsum : nullptr, rows, parts, sp.ztarget, target + r0, rows, d->V,
          d->ignore_index, (float)d->label_smoothing, lse + r0, loss + r0);
      PVB2_LAUNCH_CHECK();
    }
  }
  lce_total_kernel<<<1, 1024, 0, s>>>(loss, target, d->N, d->V, d->ignore_index, d->reduction, out, count);
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

size_t pvb2_linear_ce_bwd_workspace_size(const pvb2_linear_ce_desc* desc) {
  if (lce_check(desc) != PVB2_OK || desc->N == 0) return 0;
  const pvb2_linear_ce_desc normal = lce_normal(desc), *d = &normal;
  LceBwdSpace s;
  return lce_bwd_space(d, lce_plan(d, true), nullptr, &s) + 1024;
}

int pvb2_linear_ce_bwd(const pvb2_linear_ce_desc* desc, const void* x, const void* w, const void* bias,
                       const int64_t* target, const float* lse, const float* count, const float* grad_out, void* dx,
                       void* dw, void* dbias, void* workspace, size_t workspace_bytes, pvb2_stream stream) {
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
  if (!dx && !dw && !dbias) return PVB2_OK;
  PVB2_CHECK_ARG(workspace && workspace_bytes >= pvb2_linear_ce_bwd_workspace_size(d),
                 "linear cross entropy backward: workspace of %zu bytes needed", pvb2_linear_ce_bwd_workspace_size(d));
  const LcePlan p = lce_plan(d, true);
  LceBwdSpace sp;
  lce_bwd_space(d, p, (void*)(((uintptr_t)workspace + 1023) & ~(uintptr_t)1023), &sp);
  const bool direct_w = !p.pack_w;
  PVB2_TRY(lce_aligned(w, direct_w));
  const float gscale = p.half ? 32768.f : 1.f;
  lce_grad_rows_kernel<<<1, 1024, 0, s>>>(grad_out, count, target, d->N, d->V, d->ignore_index, d->reduction,
                                          1.f / gscale, sp.row, sp.factor);
  PVB2_LAUNCH_CHECK();
  PVB2_TRY(lce_pack(d, p, x, 0, d->N, d->ldx, sp.x, target, s));
  CUtensorMap x_k, x_mn, w_k, w_mn, g_store, g_k, g_mn, acc;
  PVB2_TRY(lce_map(&x_k, sp.x, d->D, d->N, p.ldp, p.P, kLBM, p.half));
  PVB2_TRY(lce_map(&x_mn, sp.x, d->D, d->N, p.ldp, p.P, 64, p.half));
  const bool dx_slabs = p.pieces > 1 || p.dx_splits > 1;
  const int64_t ld32 = up(d->D, 4);
  for (int q = 0; q < p.pieces; ++q) {
    const int64_t v0 = q * p.piece, width = std::min(p.piece, d->V - v0), ldg = up(width, 8);
    const int row0 = direct_w ? (int)v0 : 0;
    if (direct_w) {
      PVB2_TRY(lce_map(&w_k, w, d->D, d->V, d->ldw, 1, kLBN, p.half));
      PVB2_TRY(lce_map(&w_mn, w, d->D, d->V, d->ldw, 1, 64, p.half));
    } else {
      PVB2_TRY(lce_pack(d, p, w, v0, width, d->ldw, sp.w, nullptr, s));
      PVB2_TRY(lce_map(&w_k, sp.w, d->D, width, p.ldp, p.P, kLBN, p.half));
      PVB2_TRY(lce_map(&w_mn, sp.w, d->D, width, p.ldp, p.P, 64, p.half));
    }
    PVB2_TRY(lce_map(&g_store, sp.G, width, d->N, ldg, p.P, 32, p.half));
    PVB2_TRY(lce_map(&g_k, sp.G, width, d->N, ldg, p.P, kLBM, p.half));
    PVB2_TRY(lce_map(&g_mn, sp.G, width, d->N, ldg, p.P, 64, p.half));
    // G of this piece
    LceGemm g;
    lce_logits(&g, d, p, bias);
    g.M = (int)d->N;
    g.N = (int)width;
    g.v0 = (int)v0;
    g.b_row0 = row0;
    g.target = target;
    g.lse = lse;
    g.grow = sp.row;
    g.planes = p.P;
    g.gscale = gscale;
    PVB2_TRY(lce_gemm<kEpiGrad>(x_k, w_k, g_store, g, false, false, p, s));
    if (dx) {
      LceGemm h;
      memset(&h, 0, sizeof(h));
      lce_segments(&h, p);
      h.M = (int)d->N;
      h.N = (int)d->D;
      h.K = (int)width;
      h.b_row0 = row0;
      h.n_fast = 1;
      if (dx_slabs) {
        h.splits = p.dx_splits;
        h.kb_per = p.dx_kb;
        // a last piece that is shorter leaves the far slabs alone
        const int kb = (int)(up(width, kLBK) / kLBK);
        if (q > 0) h.splits = std::min(h.splits, (kb + h.kb_per - 1) / h.kb_per);
        h.accumulate = q > 0;
        PVB2_TRY(lce_map32(&acc, sp.dx, d->D, d->N, ld32, p.dx_splits));
        PVB2_TRY(lce_gemm<kEpiAcc>(g_k, w_mn, acc, h, false, true, p, s));
      } else {
        h.splits = 1;
        h.kb_per = INT32_MAX / 2;
        PVB2_TRY(lce_out(d, p, g_k, w_mn, h, false, d->N, dx, sp.factor, s));
      }
    }
    if (dw) {
      LceGemm h;
      memset(&h, 0, sizeof(h));
      lce_segments(&h, p);
      h.M = (int)width;
      h.N = (int)d->D;
      h.K = (int)d->N;
      h.n_fast = 1;
      void* out = (uint8_t*)dw + v0 * d->D * size;
      if (p.dw_splits > 1) {
        h.splits = p.dw_splits;
        h.kb_per = p.dw_kb;
        PVB2_TRY(lce_map32(&acc, sp.dw, d->D, width, ld32, p.dw_splits));
        PVB2_TRY(lce_gemm<kEpiAcc>(g_mn, x_mn, acc, h, true, true, p, s));
        PVB2_TRY(lce_join(d, sp.dw, p.dw_splits, width, sp.factor, out, s));
      } else {
        h.splits = 1;
        h.kb_per = INT32_MAX / 2;
        PVB2_TRY(lce_out(d, p, g_mn, x_mn, h, true, width, out, sp.factor, s));
      }
    }
    if (dbias) {
      const dim3 grid((unsigned)((width + 31) / 32), (unsigned)p.colsum_parts);
      void* out = (uint8_t*)dbias + v0 * size;
      const int blocks = (int)((width + 255) / 256);
      if (p.half) {
        lce_colsum_kernel<<<grid, 256, 0, s>>>((const __half*)sp.G, d->N, width, ldg, p.P, p.rows_per, sp.colsum);
        PVB2_LAUNCH_CHECK();
        lce_dbias_kernel<<<blocks, 256, 0, s>>>(sp.colsum, p.colsum_parts, width, sp.factor, (__half*)out);
      } else {
        lce_colsum_kernel<<<grid, 256, 0, s>>>((const __nv_bfloat16*)sp.G, d->N, width, ldg, p.P, p.rows_per, sp.colsum);
        PVB2_LAUNCH_CHECK();
        if (d->dtype == PVB2_F32)
          lce_dbias_kernel<<<blocks, 256, 0, s>>>(sp.colsum, p.colsum_parts, width, sp.factor, (float*)out);
        else
          lce_dbias_kernel<<<blocks, 256, 0, s>>>(sp.colsum, p.colsum_parts, width, sp.factor, (__nv_bfloat16*)out);
      }
      PVB2_LAUNCH_CHECK();
    }
  }
  if (dx && dx_slabs) PVB2_TRY(lce_join(d, sp.dx, p.dx_splits, d->N, sp.factor, dx, s));
  return PVB2_OK;
}

int pvb2_linear_ce_status(int* timed_out, int reset) { return tc_timeout_flag_local(timed_out, reset); }

}  // extern "C"
