// A linear layer in 8-bit floating point: e4m3 codes with one fp32 scale for
// every 128 inputs of a row of x and for every 128 x 128 of the weight,
//
//   y[m][n] = sum over b of xs[m][b] ws[n / 128][b] sum_{k in block b} xc[m][k] wc[n][k]  + bias[n]
//
// The inner sums are the tensor cores' (tcgen05.mma kind::f8f6f4, four steps of
// 32 along K, fp32 in TMEM); the outer one is formed in registers, since the
// scales change with the block.  A block's products go to one of two accumulators
// (of up to eight, few rows); while the epilogue's warps read one, multiply it by its
// scales and add it to their sums, the tensor core fills another.  Products of codes
// are exact, a block's 128 of them lose bits below 2^-24 of their largest, and
// what the epilogue adds rounds as fp32 does.
//
// Two kernels:
//   * many rows: CTA pairs (cta_group::2) on tiles of 256 rows x 256 outputs,
//     persistent, loads by TMA into a ring of five K blocks, stores by TMA.  A
//     block's products take the tensor core 512 clocks and a block as a whole 1040
//     (8192^3: 896 one after the other in 596 us, at the 1.57 GHz that the board's
//     power leaves; 514 in a burst): bound by the epilogue, whose four rounds of
//     load, wait and multiply-add stand in line, with no load behind the arithmetic.
//   * few rows: tiles of 128 outputs x 16 to 128 rows, the weight in the
//     place of the left operand, so that one row costs little; K is split over
//     the CTAs of a cluster where the tiles are few, whose sums join through
//     shared memory in a fixed order.  Bound by the weight's bytes.
#include <algorithm>
#include <cfloat>
#include <type_traits>
#include "overlap.cuh"
#include "quant8.cuh"
#include "tc_common.cuh"

namespace pvb2 {

constexpr int kL8BK = kGroup8;  // a K block: one scale, and a 128-byte row of a swizzled tile

struct L8Args {
  const float* xs;   // [M][blocks]
  const float* ws;   // [ceil(N / 128)][blocks]
  const void* bias;  // of the output's type, or null
  void* y;           // [M][N]
  const uint8_t* x;  // the codes, for blocks whose scales' product is odd
  const uint8_t* w;
  int64_t ldx, ldw;
  int M, N, K, blocks;
  int tma_store;     // many rows: y's rows lie on 16-byte boundaries
  int vector_store;  // few rows: and four outputs on theirs
  int group;         // blocks of rows whose tiles lie together
};

__host__ __device__ constexpr uint32_t idesc_e4m3(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void mma_e4m3(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_e4m3_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                              uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// tells the even CTA that an accumulator has been read.  What it guards is in
// TMEM, and has arrived in registers (tcgen05.wait::ld) ahead of the fence for
// tcgen05 that every caller has made: nothing in memory has to be ordered, and
// releasing it for the cluster cost more than the epilogue's arithmetic
__device__ __forceinline__ void arrive_even_cta(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// two fp32 numbers in a register pair; a = b s + a, each rounded once
__device__ __forceinline__ uint64_t pair_of(float x, float y) {
  uint64_t p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(x), "f"(y));
  return p;
}
__device__ __forceinline__ void fma2(uint64_t& a, uint64_t b, uint64_t s) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(a) : "l"(b), "l"(s));
}
__device__ __forceinline__ float2 numbers(uint64_t p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
  return f;
}

// The scales' product x w where it leaves fp32's normal numbers ("odd"): a block's
// sum is 0 or has 2^-18 to 2^25, so that its multiple may be a number all the same.
// The sum is then multiplied by 2^100 or 2^-100 first, which is exact, and by what
// is left of the product afterwards.  (Beyond 2^228 that is cut to fp32's largest:
// the multiple of any sum but 0 is infinite, and that of 0 is 0.  Scales that are
// 0, infinite or NaN are multiplied as they are.)
__device__ __forceinline__ bool normal(float f) { return abs_bits(f) - 0x00800000u < 0x7f000000u; }
__device__ __forceinline__ bool odd_product(float x, float w, float product) {
  return !normal(product) && x != 0.f && w != 0.f && fabsf(x) <= FLT_MAX && fabsf(w) <= FLT_MAX;
}
// No product is odd of an x of 2^-62 to 2^66 and a w of 2^-62 to 2^61.  Of any
// number of them, `or`ed: the top bit says whether one lies beyond.  (It does where
// the exponent is not among the 128 from 65 on, for w also not among those from 60.)
__device__ __forceinline__ uint32_t beyond_x(float x) { return 2 * __float_as_uint(x) - (65u << 24); }
__device__ __forceinline__ uint32_t beyond_w(float w) { return beyond_x(w) | (2 * __float_as_uint(w) - (60u << 24)); }
__device__ __forceinline__ bool unusual(uint32_t beyond) { return (int32_t)beyond < 0; }
// the two parts
__device__ __forceinline__ float odd_first(float x, float w) {
  const float product = x * w;
  return odd_product(x, w, product) ? (fabsf(product) > 1.f ? 0x1p100f : 0x1p-100f) : 1.f;
}
__device__ __forceinline__ float odd_rest(float x, float w, float first) {
  if (first == 1.f) return x * w;
  const float rest = (first > 1.f ? x * 0x1p-100f : x * 0x1p100f) * w;
  return fminf(fmaxf(rest, -FLT_MAX), FLT_MAX);
}

// 16 columns of this warp's 32 lanes, as pairs.  The wait is part of the
// statement: apart from it, each value was copied before its use
__device__ __forceinline__ void tmem_ld16_pairs(uint32_t taddr, uint64_t* u) {
  asm volatile(
      "{\n\t.reg .b32 r<16>;\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{r0,r1,r2,r3,r4,r5,r6,r7,r8,r9,r10,r11,r12,r13,r14,r15}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;\n\t"
      "mov.b64 %0, {r0, r1};\n\t"
      "mov.b64 %1, {r2, r3};\n\t"
      "mov.b64 %2, {r4, r5};\n\t"
      "mov.b64 %3, {r6, r7};\n\t"
      "mov.b64 %4, {r8, r9};\n\t"
      "mov.b64 %5, {r10, r11};\n\t"
      "mov.b64 %6, {r12, r13};\n\t"
      "mov.b64 %7, {r14, r15};\n\t"
      "}"
      : "=l"(u[0]), "=l"(u[1]), "=l"(u[2]), "=l"(u[3]), "=l"(u[4]), "=l"(u[5]), "=l"(u[6]), "=l"(u[7])
      : "r"(taddr)
      : "memory");
}

// The issuing warp stays whole: its loop runs in all lanes, on values that the
// compiler knows to be the same in each (a warp's number by a shuffle, a wait's
// result by a vote, TMEM's base by a reduction), and one lane is elected for the
// instructions alone.  Descriptors are then in uniform registers; from within
// a branch of lane 0 each MMA took 75 clocks to issue, a block of four, with
// its waits and commits, 700, where the tensor core needs 512.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ int warp_number() { return __shfl_sync(~0u, (int)(threadIdx.x >> 5), 0); }

// ---------------------------------------------------------------- many rows
constexpr int kL8M = 256, kL8N = 256;
// Warps: two issue loads, one prepares the scales, one issues the products, 16
// run the epilogue, 32 rows and 64 columns each: five for each of the SM's four
// schedulers.  The epilogue's 96 registers hold 64 sums and 16 columns on their
// way from TMEM; scales loaded by its own threads did not fit beside them, and
// what spilled had left L1 (the ring takes it) by the time it was needed.
constexpr int kL8Producers = 2, kL8ScaleWarp = 2, kL8MmaWarp = 3, kL8EpiWarps = 16;
struct L8Smem {
  static constexpr int THREADS = (kL8MmaWarp + 1 + kL8EpiWarps) * 32;
  static constexpr int A_BYTES = 128 * kL8BK;          // this CTA's rows of x
  static constexpr int B_BYTES = kL8N / 2 * kL8BK;     // and its half of the outputs
  static constexpr int SLOT_BYTES = A_BYTES + B_BYTES;
  static constexpr int SLOTS = 5;
  static constexpr int BOX = 2048;                     // of an epilogue warp: 32 rows of 64 bytes
  static constexpr int EPI_OFF = SLOTS * SLOT_BYTES;
  static constexpr int SCALE_BYTES = 4 * 2 * 128 * 4;  // [block of four][half of the outputs][row]
  static constexpr int SCALE_OFF = EPI_OFF + kL8EpiWarps * BOX;
  static constexpr int BAR_OFF = SCALE_OFF + 2 * SCALE_BYTES;
  static constexpr int TOTAL = BAR_OFF + (2 * SLOTS + 8) * 8 + 16;
};

// `group` blocks of rows go past all outputs before the next ones do
__device__ __forceinline__ void l8_place(int group, int tiles_m, int tiles_n, int tile, int& mb, int& nb) {
  const int first = tile / (group * tiles_n) * group, wide = min(group, tiles_m - first);
  const int r = tile - first * tiles_n;
  mb = first + r % wide;
  nb = r / wide;
}

// The rows of this CTA's tiles in which a product of scales is odd, formed again
// from the codes in memory, with such products in two parts.  That is slow (4096^3,
// all rows: 30 ms against 76 us), for operands that next to nothing has: the
// epilogue has no register for a second way through its loop (with one, or with
// the loop once more in the same kernel, all calls took a tenth longer).
template <typename T>
__device__ __forceinline__ void form_odd_rows(const L8Args& p) {
  const int tiles_m = (p.M + kL8M - 1) / kL8M, tiles_n = (p.N + kL8N - 1) / kL8N;
#pragma unroll 1
  for (int tile = blockIdx.x >> 1; tile < tiles_m * tiles_n; tile += gridDim.x >> 1) {
    int mb, nb;
    l8_place(p.group, tiles_m, tiles_n, tile, mb, nb);
    const int m0 = mb * kL8M + (blockIdx.x & 1) * 128, m1 = min(m0 + 128, p.M);
    // a warp to a row and the 128 outputs of one scale, 32 at a time
#pragma unroll 1
    for (int job = threadIdx.x >> 5; job < 256; job += L8Smem::THREADS / 32) {
      const int m = m0 + (job >> 1), n0 = nb * kL8N + (job & 1) * kGroup8;
      if (m >= m1 || n0 >= p.N) continue;
      const float* xs = p.xs + (int64_t)m * p.blocks;
      const float* ws = p.ws + (int64_t)(n0 / kGroup8) * p.blocks;
      bool odd = false;
      for (int kb = threadIdx.x & 31; kb < p.blocks; kb += 32) odd |= odd_product(xs[kb], ws[kb], xs[kb] * ws[kb]);
      if (!__any_sync(~0u, odd)) continue;
      const uint8_t* xc = p.x + (int64_t)m * p.ldx;
#pragma unroll 1
      for (int n = n0 + (threadIdx.x & 31); n < min(n0 + kGroup8, p.N); n += 32) {
        const uint8_t* wc = p.w + (int64_t)n * p.ldw;
        float sum = 0.f;
#pragma unroll 1
        for (int kb = 0; kb < p.blocks; ++kb) {
          const int k1 = min((kb + 1) * kL8BK, p.K);
          float u = 0.f;
          int k = kb * kL8BK;
          for (; k + 16 <= k1; k += 16) {  // (rows begin on 16-byte boundaries)
            const uint4 a = *(const uint4*)(xc + k), b = *(const uint4*)(wc + k);
            const uint32_t as[4] = {a.x, a.y, a.z, a.w}, bs[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float2 av = values2(as[i / 2] >> (16 * (i & 1))), bv = values2(bs[i / 2] >> (16 * (i & 1)));
              u = fmaf(av.y, bv.y, fmaf(av.x, bv.x, u));
            }
          }
          for (; k < k1; ++k) u = fmaf(values2(xc[k]).x, values2(wc[k]).x, u);
          const float first = odd_first(xs[kb], ws[kb]);
          sum = fmaf(u * first, odd_rest(xs[kb], ws[kb], first), sum);
        }
        if (p.bias) sum += to_f32(((const T*)p.bias)[n]);
        ((T*)p.y)[(int64_t)m * p.N + n] = from_f32<T>(sum);
      }
    }
  }
}

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(L8Smem::THREADS, 1)
    linear8_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                   const __grid_constant__ CUtensorMap tmY, const __grid_constant__ L8Args p) {
  using L = L8Smem;
  constexpr int kSlots = L::SLOTS;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = (uint64_t*)(smem + L::BAR_OFF);  // waited on in the even CTA
  uint64_t* empty = full + kSlots;
  uint64_t* acc_full = empty + kSlots;
  uint64_t* acc_empty = acc_full + 2;               // waited on in the even CTA
  uint64_t* scales_full = acc_empty + 2;
  uint64_t* scales_empty = scales_full + 2;
  uint32_t* tmem_slot = (uint32_t*)(scales_empty + 2);
  volatile int* abort = (volatile int*)(tmem_slot + 1);
  int* odd_met = (int*)(tmem_slot + 2);             // whether a product of scales was odd

  const int warp = warp_number(), lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank();
  const int tiles_m = (p.M + kL8M - 1) / kL8M, tiles_n = (p.N + kL8N - 1) / kL8N;
  const int tiles = tiles_m * tiles_n;
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * kL8EpiWarps);
      mbar_init(&scales_full[b], 1);
      mbar_init(&scales_empty[b], kL8EpiWarps);
    }
    *abort = *odd_met = 0;
    fence_barrier_init();
  }
  if (warp == kL8MmaWarp) tmem_alloc_pair(tmem_slot, 512);
  wait_for_last();
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers exist before either is signalled
  tc_fence_after();
  let_next_come();
  const uint32_t tmem_base = *tmem_slot;

  auto place = [&](int tile, int& mb, int& nb) { l8_place(p.group, tiles_m, tiles_n, tile, mb, nb); };

  if (warp < kL8Producers) {
    // ------------------------------------------------- loads: slot s by warp s % kL8Producers
    if (lane == 0) {
      tma_prefetch(&tmX);
      tma_prefetch(&tmW);
      uint32_t it = 0;
      for (int tile = pair; tile < tiles && !*abort; tile += pairs) {
        int mb, nb;
        place(tile, mb, nb);
        const int am = mb * kL8M + rank * 128, bn = nb * kL8N + rank * (kL8N / 2);
        for (int kb = 0; kb < p.blocks; ++kb, ++it) {
          const int s = it % kSlots;
          if (s % kL8Producers != warp) continue;
          if (!mbar_wait(&empty[s], ((it / kSlots) & 1) ^ 1, abort)) break;
          uint8_t* sa = smem + s * L::SLOT_BYTES;
          const uint32_t bar = even_cta_addr(&full[s]);
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * L::SLOT_BYTES);
          tma_load_3d_pair(sa, &tmX, bar, kb * kL8BK, am, 0);
          tma_load_3d_pair(sa + L::A_BYTES, &tmW, bar, kb * kL8BK, bn, 0);
        }
      }
    }
  } else if (warp == kL8ScaleWarp) {
    // ------------------------------------------------- the scales of four blocks at a time: x's times the weight's
    uint32_t group = 0;
    for (int tile = pair; tile < tiles && !*abort; tile += pairs) {
      int mb, nb;
      place(tile, mb, nb);
      const int m0 = mb * kL8M + rank * 128 + lane;
      // (rows and outputs past the end: some scale, of codes that are 0)
      const float* ws0 = p.ws + (int64_t)(nb * (kL8N / kGroup8)) * p.blocks;
      const float* ws1 = p.ws + (int64_t)min(nb * (kL8N / kGroup8) + 1, (p.N - 1) / kGroup8) * p.blocks;
      float x[4][4], w[2][4];
      auto fetch = [&](int kb) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = min(kb + i, p.blocks - 1);
#pragma unroll
          for (int r = 0; r < 4; ++r) x[r][i] = p.xs[(int64_t)min(m0 + 32 * r, p.M - 1) * p.blocks + k];
          w[0][i] = ws0[k];
          w[1][i] = ws1[k];
        }
      };
      fetch(0);
      for (int kb = 0; kb < p.blocks; kb += 4, ++group) {
        const int slot = group & 1;
        if (!mbar_wait(&scales_empty[slot], ((group >> 1) & 1) ^ 1, abort)) break;
        float* to = (float*)(smem + L::SCALE_OFF + slot * L::SCALE_BYTES) + lane;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) to[(i * 2 + h) * 128 + 32 * r] = x[r][i] * w[h][i];
        // Whether a product is odd.  (As little as can be, and no detail in registers:
        // it is issued beside the epilogue, and took a tenth of its time when the
        // products were looked at one by one in a straight line.)
        uint32_t out = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int h = 0; h < 2; ++h) out |= beyond_w(w[h][i]);
#pragma unroll
          for (int r = 0; r < 4; ++r) out |= beyond_x(x[r][i]);
        }
        if (unusual(out)) {
          out = 0;  // zeros are as usual as others
#pragma unroll
          for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int h = 0; h < 2; ++h) out |= w[h][i] != 0.f ? beyond_w(w[h][i]) : 0;
#pragma unroll
            for (int r = 0; r < 4; ++r) out |= x[r][i] != 0.f ? beyond_x(x[r][i]) : 0;
          }
          if (unusual(out)) {  // (blocks of 1e-16 and less are: 29 us in place of 22.5 for 1024 rows, 4096 of 4096)
#pragma unroll 8
            for (int j = 0; j < 32; ++j) {
              const float product = to[(j >> 2) * 128 + 32 * (j & 3)];
              if (normal(product)) continue;
              const int k = min(kb + (j >> 3), p.blocks - 1);
              if (odd_product(p.xs[(int64_t)min(m0 + 32 * (j & 3), p.M - 1) * p.blocks + k], (j & 4 ? ws1 : ws0)[k], product)) *odd_met = 1;
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&scales_full[slot]);
        if (kb + 4 < p.blocks) fetch(kb + 4);
      }
    }
  } else if (warp == kL8MmaWarp) {
    // ------------------------------------------------- products, by the even CTA for both
    if (rank == 0) {
      constexpr uint32_t idesc = idesc_e4m3(kL8M, kL8N);
      const uint32_t base = __reduce_or_sync(~0u, tmem_base);
      const uint64_t a0 = desc_kmajor(smem_u32(smem), 0), b0 = desc_kmajor(smem_u32(smem) + L::A_BYTES, 0);
      uint32_t it = 0;
      bool ok = true;
      for (int tile = pair; tile < tiles && ok; tile += pairs) {
        for (int kb = 0; kb < p.blocks; ++kb, ++it) {
          const int buf = it & 1, s = it % kSlots;
          ok = __all_sync(~0u, mbar_wait(&acc_empty[buf], ((it >> 1) & 1) ^ 1, abort) &&
                                   mbar_wait(&full[s], (it / kSlots) & 1, abort));
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t ad = a0 + (uint32_t)(s * (L::SLOT_BYTES / 16)), bd = b0 + (uint32_t)(s * (L::SLOT_BYTES / 16));
#pragma unroll
            for (int kk = 0; kk < kL8BK / 32; ++kk)
              mma_e4m3_pair(base + buf * kL8N, ad + 2 * kk, bd + 2 * kk, idesc, kk ? 1u : 0u);
            mma_commit_pair(&empty[s]);
            mma_commit_pair(&acc_full[buf]);
          }
          __syncwarp();
        }
      }
    }
  } else {
    // ------------------------------------------------- epilogue: TMEM lane quarter warp % 4, 64 columns (warp - 4) / 4
    const int quarter = warp & 3, part = (warp - kL8MmaWarp - 1) >> 2;
    uint8_t* box = smem + L::EPI_OFF + (warp - kL8MmaWarp - 1) * L::BOX;
    const uint32_t acc = tmem_base + ((uint32_t)(quarter * 32) << 16) + part * 64;
    const float* scales = (const float*)(smem + L::SCALE_OFF) + (part >> 1) * 128 + quarter * 32 + lane;
    const uint32_t even_empty = even_cta_addr(acc_empty);
    uint32_t it = 0, group = 0;
    for (int tile = pair; tile < tiles && !*abort; tile += pairs) {
      uint64_t sums[32];  // of two columns each
#pragma unroll
      for (int j = 0; j < 32; ++j) sums[j] = 0;
      bool ok = true;
#pragma unroll 1
      for (int kb = 0; kb < p.blocks; ++kb, ++it) {
        const int buf = it & 1, slot = group & 1;
        if ((kb & 3) == 0) ok = mbar_wait(&scales_full[slot], (group >> 1) & 1, abort);
        const float scale = scales[slot * (L::SCALE_BYTES / 4) + (kb & 3) * 256];
        const uint64_t ss = pair_of(scale, scale);
        ok = ok && mbar_wait(&acc_full[buf], (it >> 1) & 1, abort);
        if (!ok) break;
        tc_fence_after();
        const bool last = (kb & 3) == 3 || kb + 1 == p.blocks;  // of the scales' slot
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          if (h) __syncwarp();  // (the next columns stay behind these sums: 626 -> 615 us for 8192^3)
          uint64_t u[8];
          tmem_ld16_pairs(acc + buf * kL8N + 16 * h, u);
          if (h == 3) {  // all of it is in registers
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              arrive_even_cta(even_empty + buf * 8);
              if (last) mbar_arrive(&scales_empty[slot]);
            }
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) fma2(sums[8 * h + j], u[j], ss);
        }
        group += last;
      }
      if (!ok) break;
      int mb, nb;
      place(tile, mb, nb);
      const int m0 = mb * kL8M + rank * 128 + quarter * 32, n0 = nb * kL8N + part * 64;
      if (n0 >= p.N || m0 >= p.M) continue;
      float v[64];
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const float2 f = numbers(sums[j]);
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
      }
      if (p.bias) {
#pragma unroll
        for (int j = 0; j < 64; ++j) v[j] += to_f32(((const T*)p.bias)[min(n0 + j, p.N - 1)]);
      }
      // through the box: 32 rows of 64 bytes, 16-byte pieces swizzled by bits 1 and 2 of the row
      constexpr int kWide = 64 / (int)sizeof(T), E = 16 / (int)sizeof(T);
#pragma unroll
      for (int h = 0; h < 64 / kWide; ++h) {
        if (p.tma_store) {
          if (lane == 0) bulk_wait_read<0>();
          __syncwarp();
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
          store_vec<E>((T*)(box + lane * 64 + ((q ^ ((lane >> 1) & 3)) * 16)), v + h * kWide + q * E);
        const int nn = n0 + h * kWide;
        if (p.tma_store) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && nn < p.N) {
            tma_store_3d(&tmY, box, nn, m0, 0);
            bulk_commit();
          }
        } else {
          __syncwarp();
          // 32 / kWide rows at a time
#pragma unroll 4
          for (int r = lane / kWide; r < 32; r += 32 / std::min(32, kWide)) {
            const int j = lane % kWide;
            if (m0 + r < p.M && nn + j < p.N)
              ((T*)p.y)[(int64_t)(m0 + r) * p.N + nn + j] =
                  *(const T*)(box + r * 64 + (((j / E) ^ ((r >> 1) & 3)) * 16) + (j % E) * sizeof(T));
          }
          __syncwarp();
        }
      }
    }
    if (lane == 0) bulk_wait_all();
  }
  __syncthreads();
  if (warp == kL8MmaWarp && *abort) {
    // let any MMA still in flight finish before the columns are released
    const uint64_t t0 = globaltimer();
    while (globaltimer() - t0 < 10000000ull) {
    }
  }
  cluster_sync();  // neither CTA's shared memory goes while the other may signal it
  if (warp == kL8MmaWarp) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
  if (*odd_met) form_odd_rows<T>(p);
}

// ----------------------------------------------------------------- few rows
// Warps: one issues loads, one the products, eight run the epilogue, 32
// outputs and half the rows each (four of them took half as long again for
// short K: alone on its scheduler, a warp waits for each of its instructions).
// As many accumulators as TMEM holds, eight at most: a block of 16 rows is
// multiplied faster than its accumulator goes to the epilogue and back.
constexpr int kL8FewEpi = 8;
template <int NT>
struct L8Few {
  static constexpr int THREADS = (2 + kL8FewEpi) * 32;
  static constexpr int W_BYTES = 128 * kL8BK;
  static constexpr int SLOT_BYTES = W_BYTES + NT * kL8BK;
  static constexpr int BUFS = std::min(8, 512 / NT);
  static constexpr int COLUMNS = BUFS * NT;             // of TMEM
  static constexpr int RUN = 32;                        // blocks whose scales are at hand
  static constexpr int PITCH = NT + 4;                  // of a block's scales
  static constexpr int SLOTS = std::min(11, (224 * 1024 - RUN * PITCH * 4) / SLOT_BYTES);
  static constexpr int SCALE_OFF = SLOTS * SLOT_BYTES;  // [block][row]: x's times the weight's
  static constexpr int BAR_OFF = SCALE_OFF + RUN * PITCH * 4;
  static constexpr int TOTAL = BAR_OFF + (2 * SLOTS + 2 * BUFS) * 8 + 16;
  static_assert(SLOTS * SLOT_BYTES >= 128 * NT * 4, "the sums go where the ring was");
};

__device__ __forceinline__ void epilogue_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kL8FewEpi * 32) : "memory"); }
// and whether any of its threads says so
__device__ __forceinline__ bool epilogue_any(bool mine) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"((uint32_t)mine), "n"(kL8FewEpi * 32)
      : "memory");
  return any != 0;
}
// four floats of another CTA of the cluster
__device__ __forceinline__ float4 load_cluster(const float* p, int rank) {
  uint32_t at;
  float4 f;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(at) : "memory");
  return f;
}
// COLS columns of this warp's 32 lanes
template <int COLS>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float* v) {
  if constexpr (COLS == 32) {
    tmem_ld32(taddr, v);
  } else if constexpr (COLS == 16) {
    tmem_ld16(taddr, v);
  } else {
    static_assert(COLS == 8, "8, 16 or 32 columns");
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
        : "r"(taddr)
        : "memory");
  }
}

// The scales of the blocks [kb, kb + count) for the tile's rows, x's times the
// weight's, by the epilogue's threads; whether one of this thread's is odd.
template <int NT>
__device__ __forceinline__ bool load_scales(const L8Args& p, const float* ws, int m0, int kb, int count, float* run, int warp,
                                            int lane) {
  constexpr int kPitch = L8Few<NT>::PITCH;
  bool odd = false;
  if (NT >= 64) {
    // some threads to a row, eight blocks at a time each
    constexpr int kPer = NT >= 64 ? kL8FewEpi * 32 / NT : 1;
    const int t = (warp - 2) * 32 + lane, j = t % NT;
    const float* row = p.xs + (int64_t)min(m0 + j, p.M - 1) * p.blocks + kb;
#pragma unroll 1
    for (int k0 = t / NT * 8; k0 < count; k0 += 8 * kPer) {
      float x[8], w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = row[min(k0 + i, count - 1)];
        w[i] = ws[kb + min(k0 + i, count - 1)];
      }
      uint32_t out = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        out |= beyond_x(x[i]) | beyond_w(w[i]);
        if (k0 + i < count) run[(k0 + i) * kPitch + j] = x[i] * w[i];
      }
      if (unusual(out)) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (k0 + i < count && odd_product(x[i], w[i], x[i] * w[i])) {
            odd = true;
            run[(k0 + i) * kPitch + j] = odd_rest(x[i], w[i], odd_first(x[i], w[i]));
          }
      }
    }
  } else {
    // a warp to a row, a lane to a block
    constexpr int kRows = NT / kL8FewEpi;
    const int k = min(lane, count - 1);
    const float w = ws[kb + k];
    float x[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      x[i] = p.xs[(int64_t)min(m0 + warp - 2 + kL8FewEpi * i, p.M - 1) * p.blocks + kb + k];
    uint32_t out = beyond_w(w);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      out |= beyond_x(x[i]);
      if (lane < count) run[lane * kPitch + warp - 2 + kL8FewEpi * i] = x[i] * w;
    }
    if (unusual(out)) {
#pragma unroll
      for (int i = 0; i < kRows; ++i)
        if (lane < count && odd_product(x[i], w, x[i] * w)) {
          odd = true;
          run[lane * kPitch + warp - 2 + kL8FewEpi * i] = odd_rest(x[i], w, odd_first(x[i], w));
        }
    }
  }
  return odd;
}

template <typename T, int NT>
__global__ void __launch_bounds__(L8Few<NT>::THREADS, 1)
    linear8_few_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                       const __grid_constant__ L8Args p, int splits) {
  using L = L8Few<NT>;
  constexpr int kSlots = L::SLOTS, kBufs = L::BUFS;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = (uint64_t*)(smem + L::BAR_OFF);
  uint64_t* empty = full + kSlots;
  uint64_t* acc_full = empty + kSlots;
  uint64_t* acc_empty = acc_full + kBufs;
  uint32_t* tmem_slot = (uint32_t*)(acc_empty + kBufs);
  volatile int* abort = (volatile int*)(tmem_slot + 1);

  const int warp = warp_number(), lane = threadIdx.x & 31;
  const int rank = blockIdx.x % splits, tile = blockIdx.x / splits;
  // tiles of the same outputs lie together: their weight is read once
  const int tiles_m = (p.M + NT - 1) / NT;
  const int m0 = tile % tiles_m * NT, nb = tile / tiles_m, n0 = nb * 128;
  const int kb0 = (int)((int64_t)p.blocks * rank / splits), kb1 = (int)((int64_t)p.blocks * (rank + 1) / splits);

  const float* ws = p.ws + (int64_t)nb * p.blocks;
  float* run = (float*)(smem + L::SCALE_OFF);
  bool odd = false;  // whether one of the run's scales is
  if (warp == 0) {
#pragma unroll
    for (int i = lane; i < 2 * kSlots + 2 * kBufs; i += 32) mbar_init(&full[i], i < 2 * kSlots + kBufs ? 1 : kL8FewEpi);
    fence_barrier_init();
    __syncwarp();
    wait_for_last();
    if (lane == 0) {
      *abort = 0;
      // the first loads need nothing of the others
      for (int it = 0; it < min(kSlots, kb1 - kb0); ++it) {
        uint8_t* sw = smem + it * L::SLOT_BYTES;
        mbar_arrive_expect_tx(&full[it], L::SLOT_BYTES);
        tma_load_3d(sw, &tmW, &full[it], (kb0 + it) * kL8BK, n0, 0);
        tma_load_3d(sw + L::W_BYTES, &tmX, &full[it], (kb0 + it) * kL8BK, m0, 0);
      }
    }
  } else if (warp == 1) {
    tmem_alloc(tmem_slot, L::COLUMNS);
  } else {
    wait_for_last();
    odd = load_scales<NT>(p, ws, m0, kb0, min(L::RUN, kb1 - kb0), run, warp, lane);
  }
  tc_fence_before();
  odd = __syncthreads_or(odd);
  tc_fence_after();
  let_next_come();
  const uint32_t tmem_base = *tmem_slot;

  constexpr int kHalf = NT / 2, kWide = kHalf < 32 ? kHalf : 32;
  const int first = warp < 6 ? 0 : kHalf;  // an epilogue warp's first row of the tile
  float v[kHalf];
  if (warp == 0) {
    if (lane == 0) {
      for (int kb = kb0 + kSlots, it = kSlots; kb < kb1; ++kb, ++it) {
        const int s = it % kSlots;
        if (!mbar_wait(&empty[s], ((it / kSlots) & 1) ^ 1, abort)) break;
        uint8_t* sw = smem + s * L::SLOT_BYTES;
        mbar_arrive_expect_tx(&full[s], L::SLOT_BYTES);
        tma_load_3d(sw, &tmW, &full[s], kb * kL8BK, n0, 0);
        tma_load_3d(sw + L::W_BYTES, &tmX, &full[s], kb * kL8BK, m0, 0);
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = idesc_e4m3(128, NT);
    const uint32_t base = __reduce_or_sync(~0u, tmem_base);
    const uint64_t a0 = desc_kmajor(smem_u32(smem), 0), b0 = desc_kmajor(smem_u32(smem) + L::W_BYTES, 0);
    for (int kb = kb0, it = 0; kb < kb1; ++kb, ++it) {
      const int buf = it % kBufs, s = it % kSlots;
      if (!__all_sync(~0u, mbar_wait(&acc_empty[buf], ((it / kBufs) & 1) ^ 1, abort) &&
                               mbar_wait(&full[s], (it / kSlots) & 1, abort)))
        break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t ad = a0 + (uint32_t)(s * (L::SLOT_BYTES / 16)), bd = b0 + (uint32_t)(s * (L::SLOT_BYTES / 16));
#pragma unroll
        for (int kk = 0; kk < kL8BK / 32; ++kk) mma_e4m3(base + buf * NT, ad + 2 * kk, bd + 2 * kk, idesc, kk ? 1u : 0u);
        mma_commit(&empty[s]);
        mma_commit(&acc_full[buf]);
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------------- epilogue: lane = output, register = row of x
    const uint32_t acc = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + first;
#pragma unroll
    for (int j = 0; j < kHalf; ++j) v[j] = 0.f;
    bool ok = true;  // where a wait gave up, the others still meet at the barriers
    // the blocks of a run, whose scales are at hand; with odd ones in narrow loads, for the registers
    auto add = [&](int first_block, int count, auto any_scales) {
      constexpr bool kAny = decltype(any_scales)::value;
      constexpr int kCols = kAny ? 8 : kWide;
#pragma unroll 1
      for (int i = 0; i < count; ++i) {
        const int it = first_block + i, buf = it % kBufs;
        int row = m0 + first;
        if constexpr (kAny) asm volatile("" : "+r"(row));  // (places of 64 scales are not worth registers)
        ok = ok && mbar_wait(&acc_full[buf], (it / kBufs) & 1, abort);
        if (!ok) return;
        tc_fence_after();
#pragma unroll
        for (int h = 0; h < kHalf / kCols; ++h) {
          float u[kCols];
          tmem_ld<kCols>(acc + buf * NT + kCols * h, u);
          if constexpr (kAny) {
            const int kb = kb0 + it;
#pragma unroll
            for (int j = 0; j < kCols; ++j)
              u[j] *= odd_first(p.xs[(int64_t)min(row + kCols * h + j, p.M - 1) * p.blocks + kb], ws[kb]);
          }
#pragma unroll
          for (int j = 0; j < kCols; j += 4) {
            const float4 s = *reinterpret_cast<const float4*>(run + i * L::PITCH + first + kCols * h + j);
            float* a = v + kCols * h + j;
            a[0] = fmaf(u[j], s.x, a[0]);
            a[1] = fmaf(u[j + 1], s.y, a[1]);
            a[2] = fmaf(u[j + 2], s.z, a[2]);
            a[3] = fmaf(u[j + 3], s.w, a[3]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[buf]);
      }
    };
#pragma unroll 1
    for (int kb = kb0; kb < kb1; kb += L::RUN) {
      const int count = min(L::RUN, kb1 - kb);
      if (kb > kb0) {
        epilogue_sync();  // the last run's have been read
        odd = epilogue_any(load_scales<NT>(p, ws, m0, kb, count, run, warp, lane));
      }
      if (!odd) add(kb - kb0, count, std::false_type());
      else add(kb - kb0, count, std::true_type());
    }
  }

  // ---------------------------------------------------- the splits' sums, and y
  // By way of shared memory and in loops that stay loops: a straight line with a
  // store per register took longer than all the rest of a short K.  Several
  // rows are read before the first is stored, since the compiler cannot know
  // that y is not in shared memory.
  float* sums = (float*)smem;  // [NT][128]: every load has landed and every product been formed
  const bool epi = warp >= 2, gave_up = *abort;
  if (epi && !gave_up) {
    const int out = (warp & 3) * 32 + lane;
#pragma unroll
    for (int j = 0; j < kHalf; ++j) sums[(first + j) * 128 + out] = v[j];
  }
  const int rows = min(NT, p.M - m0);
  T* y = (T*)p.y + (int64_t)m0 * p.N + n0;
  // four outputs of a row for each lane, next to each other or 32 apart
  const int step = p.vector_store || splits > 1 ? 1 : 32, o = step == 1 ? lane * 4 : lane;
  float b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = epi && p.bias && n0 + o + i * step < p.N ? to_f32(((const T*)p.bias)[n0 + o + i * step]) : 0.f;
  if (splits == 1) {
    if (epi) {
      epilogue_sync();
      if (!gave_up && p.vector_store) {
        constexpr int R = 8;
#pragma unroll 1
        for (int j0 = warp - 2; j0 < rows; j0 += kL8FewEpi * R) {
          float4 x[R];
#pragma unroll
          for (int r = 0; r < R; ++r) x[r] = *reinterpret_cast<const float4*>(sums + min(j0 + kL8FewEpi * r, NT - 1) * 128 + o);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float all[4] = {x[r].x + b[0], x[r].y + b[1], x[r].z + b[2], x[r].w + b[3]};
            if (j0 + kL8FewEpi * r < rows && n0 + o < p.N) store_vec<4>(y + (int64_t)(j0 + kL8FewEpi * r) * p.N + o, all);
          }
        }
      } else if (!gave_up) {
        constexpr int R = 4;
#pragma unroll 1
        for (int j0 = warp - 2; j0 < rows; j0 += kL8FewEpi * R) {
          float x[R][4];
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[r][i] = sums[min(j0 + kL8FewEpi * r, NT - 1) * 128 + i * 32 + lane] + b[i];
#pragma unroll
          for (int r = 0; r < R; ++r) {
            T* row = y + (int64_t)(j0 + kL8FewEpi * r) * p.N + lane;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (j0 + kL8FewEpi * r < rows && n0 + i * 32 + lane < p.N) row[i * 32] = from_f32<T>(x[r][i]);
          }
        }
      }
    }
  } else {
    cluster_sync();
    if (epi && !gave_up) {
      constexpr int R = 2;
#pragma unroll 1
      for (int j0 = rank + (warp - 2) * splits; j0 < rows; j0 += kL8FewEpi * R * splits) {
        float4 part[R][8];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k < splits) part[r][k] = load_cluster(sums + min(j0 + kL8FewEpi * r * splits, NT - 1) * 128 + o, k);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float all[4] = {b[0], b[1], b[2], b[3]};
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k < splits) {
              all[0] += part[r][k].x;
              all[1] += part[r][k].y;
              all[2] += part[r][k].z;
              all[3] += part[r][k].w;
            }
          const int j = j0 + kL8FewEpi * r * splits;
          if (j >= rows) break;
          T* row = y + (int64_t)j * p.N + o;
          if (p.vector_store) {
            if (n0 + o < p.N) store_vec<4>(row, all);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (n0 + o + i < p.N) row[i] = from_f32<T>(all[i]);
          }
        }
      }
    }
    cluster_sync();  // no block leaves while its sums are read
  }
  __syncthreads();
  if (warp == 1) {
    if (*abort) {
      const uint64_t t0 = globaltimer();
      while (globaltimer() - t0 < 10000000ull) {
      }
    }
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, L::COLUMNS);
  }
}

// --------------------------------------------------------------- host side
static int64_t l8_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

static int l8_map(CUtensorMap* m, const void* base, int64_t cols, int64_t rows, int64_t ld_bytes, int box_cols, int box_rows,
                  CUtensorMapDataType type, CUtensorMapSwizzle swizzle) {
  uint64_t dims[3] = {(uint64_t)cols, (uint64_t)rows, 1};
  uint64_t str[2] = {(uint64_t)ld_bytes, (uint64_t)ld_bytes * rows};
  uint32_t box[3] = {(uint32_t)box_cols, (uint32_t)box_rows, 1};
  return encode_tiled(m, 3, base, dims, str, box, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, nullptr, type);
}
static int l8_codes(CUtensorMap* m, const void* base, int64_t K, int64_t rows, int64_t ld, int box_rows) {
  // (one row: its stride counts for nothing, but has to be one)
  return l8_map(m, base, K, rows, rows == 1 ? l8_div(K, 16) * 16 : ld, kL8BK, box_rows,
                CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <typename T>
static int l8_many(const pvb2_linear8_desc* d, const void* x, const void* w, L8Args p, cudaStream_t s) {
  constexpr int smem = L8Smem::TOTAL + 1024;
  static DeviceOnce once;
  PVB2_TRY(allow_smem(linear8_kernel<T>, smem, once));
  CUtensorMap mx, mw, my;
  PVB2_TRY(l8_codes(&mx, x, d->K, d->M, d->ldx, 128));
  PVB2_TRY(l8_codes(&mw, w, d->K, d->N, d->ldw, kL8N / 2));
  p.tma_store = ((uintptr_t)p.y & 15) == 0 && d->N * (int64_t)sizeof(T) % 16 == 0;
  memset(&my, 0, sizeof(my));
  if (p.tma_store)
    PVB2_TRY(l8_map(&my, p.y, d->N, d->M, d->N * sizeof(T), 64 / (int)sizeof(T), 32,
                    sizeof(T) == 4                              ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                    : std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                    CU_TENSOR_MAP_SWIZZLE_64B));
  const int64_t tiles = l8_div(d->M, kL8M) * l8_div(d->N, kL8N);
  // blocks of rows that stay in L2 (32 MB of its 126) while the outputs go by
  p.group = (int)std::max<int64_t>(8, std::min<int64_t>(l8_div(d->M, kL8M), ((int64_t)32 << 20) / (kL8M * d->K)));
  const int grid = 2 * (int)std::min<int64_t>(tiles, std::max(1, num_sms() / 2));
  PVB2_CUDA_TRY(launch_over(linear8_kernel<T>, grid, L8Smem::THREADS, smem, s, 0, mx, mw, my, p));
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

template <typename T, int NT>
static int l8_few(const pvb2_linear8_desc* d, const void* x, const void* w, const L8Args& p, int splits, cudaStream_t s) {
  constexpr int smem = L8Few<NT>::TOTAL + 1024;
  static DeviceOnce once;
  PVB2_TRY(allow_smem(linear8_few_kernel<T, NT>, smem, once));
  CUtensorMap mx, mw;
  PVB2_TRY(l8_codes(&mx, x, d->K, d->M, d->ldx, NT));
  PVB2_TRY(l8_codes(&mw, w, d->K, d->N, d->ldw, 128));
  PVB2_CUDA_TRY(launch_over(linear8_few_kernel<T, NT>, (unsigned)(l8_div(d->N, 128) * l8_div(d->M, NT) * splits),
                            L8Few<NT>::THREADS, smem, s, (unsigned)splits, mx, mw, p, splits));
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

// CTAs of a cluster that share K: as many as have an SM, and eight K blocks
// before each halving (joining the sums takes as long as four blocks do; one
// launch after the other, without overlap: 512
// outputs of 512 inputs, 128 rows: 7.3 us whole, 8.3 in two; 4096 of 4096: 20.7
// whole, 15.0 in two, 11.4 in four)
static int l8_splits(int64_t tiles, int64_t blocks) {
  int splits = 1;
  while (splits < 8 && tiles * splits * 2 <= num_sms() && blocks >= 8 * splits) splits *= 2;
  return splits;
}

template <typename T>
static int l8_run(const pvb2_linear8_desc* d, const void* x, const void* w, const L8Args& p, cudaStream_t s) {
  const int nt = d->M <= 16 ? 16 : d->M <= 32 ? 32 : d->M <= 64 ? 64 : 128;
  const int64_t few = l8_div(d->N, 128) * l8_div(d->M, nt);
  // Tiles of 128 x 128 as long as each has an SM of its own, then pairs' of 256 x
  // 256 (us without overlap, the former and the latter: 512 rows, 4096 outputs of 4096 inputs
  // 21.5 and 21.9, 1024 rows 41 and 23; 300 rows, 5001 of 1008 9.9 and 13.0, 512
  // rows 17.6 and 13.4; 1024 rows, 1024 of 8192 23.5 and 37); few rows are bound
  // by the weight, whatever its tiles.
  if (d->M > 64 && few > num_sms()) return l8_many<T>(d, x, w, p, s);
  const int splits = l8_splits(few, p.blocks);
  if (nt == 16) return l8_few<T, 16>(d, x, w, p, splits, s);
  if (nt == 32) return l8_few<T, 32>(d, x, w, p, splits, s);
  if (nt == 64) return l8_few<T, 64>(d, x, w, p, splits, s);
  return l8_few<T, 128>(d, x, w, p, splits, s);
}

}  // namespace pvb2

using namespace pvb2;

extern "C" {

int pvb2_linear8(const pvb2_linear8_desc* d, const uint8_t* x, const float* x_scales, const uint8_t* w,
                 const float* w_scales, const void* bias, void* y, pvb2_stream stream) {
  PVB2_CHECK_ARG(d, "linear_8bit: no descriptor");
  PVB2_CHECK_ARG(d->dtype == PVB2_F32 || d->dtype == PVB2_F16 || d->dtype == PVB2_BF16,
                 "linear_8bit: an output in fp32, fp16 or bf16 expected (got dtype %d)", d->dtype);
  const int64_t most = (int64_t)1 << 30;
  PVB2_CHECK_ARG(d->M >= 0 && d->M < most && d->N >= 0 && d->N < most && d->K >= 1 && d->K < most,
                 "linear_8bit: %lld rows, %lld outputs of %lld inputs out of range", (long long)d->M, (long long)d->N,
                 (long long)d->K);
  PVB2_CHECK_ARG(l8_div(d->M, 16) * l8_div(d->N, 128) < ((int64_t)1 << 27), "linear_8bit: more outputs than one launch has tiles for");
  if (d->M == 0 || d->N == 0) return PVB2_OK;
  PVB2_CHECK_ARG(x && x_scales && w && w_scales && y, "linear_8bit: null pointer");
  PVB2_CHECK_ARG((d->M == 1 || d->ldx >= d->K) && (d->N == 1 || d->ldw >= d->K), "linear_8bit: row strides below the inputs");
  PVB2_CHECK_ARG(((uintptr_t)x & 15) == 0 && ((uintptr_t)w & 15) == 0 && (d->M == 1 || d->ldx % 16 == 0) &&
                     (d->N == 1 || d->ldw % 16 == 0),
                 "linear_8bit: rows of codes have to begin on 16-byte boundaries");
  L8Args p = {};
  p.xs = x_scales;
  p.ws = w_scales;
  p.bias = bias;
  p.y = y;
  p.x = x;
  p.w = w;
  p.ldx = d->ldx;
  p.ldw = d->ldw;
  p.K = (int)d->K;
  p.M = (int)d->M;
  p.N = (int)d->N;
  p.blocks = (int)l8_div(d->K, kL8BK);
  p.vector_store = d->N % 4 == 0 && ((uintptr_t)y & 15) == 0;
  cudaStream_t s = as_stream(stream);
  if (d->dtype == PVB2_F32) return l8_run<float>(d, x, w, p, s);
  if (d->dtype == PVB2_BF16) return l8_run<__nv_bfloat16>(d, x, w, p, s);
  return l8_run<__half>(d, x, w, p, s);
}

int pvb2_linear8_status(int* timed_out, int reset) { return tc_timeout_flag_local(timed_out, reset); }

}  // extern "C"
