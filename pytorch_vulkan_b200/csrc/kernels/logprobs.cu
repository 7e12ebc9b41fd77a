// Log probabilities of given tokens, the entropy and the best alternatives of
// rows of logits, and their gradient.
//
//   m = max z,  s = sum e^(z - m),  u = sum e^(z - m) (z - m)
//   log p_t = (z_t - m) - log s,    H = log s - u / s
//   dz_j = p_j (-g - k (log p_j + H)) + g [j = t]      (g of log p_t, k of H)
//
// The forward pass reads the logits once, the backward pass reads them once
// more and writes as much: both are bound by HBM, the forward pass over 16-bit
// logits by its instructions too (one exponential and seven others for two
// bytes).  m is the running maximum of each thread, s and u are rescaled where
// it grows.  Rows of few are split over the blocks of a cluster, which join
// their numbers through shared memory: one launch, no workspace.
//
// The best ones.  Each thread's running maximum m is the best of its share of
// the row.  Of the k best, none is in a share whose maximum is below the k-th
// best maximum of the block's 512 threads, and so few more than k shares are
// read a second time (out of L2), each by a whole warp.  A warp keeps a sorted
// list of 32 with one entry per lane; an entry is a 64-bit number, the logit's
// bits in an order in which integers compare as numbers do, and below them the
// complement of its place, so that of equal logits the lower place is better.
// Lists are merged by bitonic networks.  The main loop does nothing for it.
//
// Rows begin on any element: whole 16-byte chunks are read wherever they lie,
// the ones at the ends element by element.
#include <cooperative_groups.h>
#include <algorithm>
#include <cfloat>
#include "types.cuh"

namespace pvb2 {
namespace cg = cooperative_groups;

constexpr int kLpThreads = 512;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpTop = 32;
constexpr int kLpCluster = 8;

struct LpArgs {
  const void* z;
  const int64_t* token;
  float* logp;
  float* entropy;
  float* stats;      // [N][3]: m, log s, H; or null
  float* top_logp;   // [N][top]
  int64_t* top_at;
  int64_t N, V, ldz;
  int top;
};

struct LpBwdArgs {
  const void* z;
  const int64_t* token;
  const float* stats;
  const float* g_logp;     // or null; `one_*`: one number for all rows
  const float* g_entropy;  // or null
  void* dz;
  int64_t N, V, ldz;
  int one_logp, one_entropy;
};

constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float exp_of(float d) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(d * kLog2e));
  return e;
}

struct Running {
  float m, s, u;
};
// m of no element: finite, so that nothing is subtracted from itself in infinity
__device__ __forceinline__ Running nothing() { return {-FLT_MAX, 0.f, 0.f}; }

__device__ __forceinline__ void move_max(Running& r, float m) {
  const float d = r.m - m, c = exp_of(d);
  // (c is 0 where d is far below; 0 times an infinity is none)
  r.u = c > 0.f || r.s != r.s ? c * fmaf(r.s, d, r.u) : 0.f;
  r.s *= c;
  r.m = m;
}

__device__ __forceinline__ Running join(Running a, Running b) {
  const float m = fmaxf(a.m, b.m);
  if (a.m != m) move_max(a, m);
  if (b.m != m) move_max(b, m);
  return {m, a.s + b.s, a.u + b.u};
}

// E logits more
template <int E>
__device__ __forceinline__ void take(Running& r, const float* z, float most) {
  if (most > r.m) move_max(r, most);
  float s = 0.f, u = 0.f;
#pragma unroll
  for (int k = 0; k < E; ++k) {
    const float d = z[k] - r.m, e = exp_of(d);
    s += e;
    u = fmaf(e, d, u);
  }
  if (u != u) {  // e is 0 and d -inf somewhere (or something is NaN, which s is too)
    u = 0.f;
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const float d = z[k] - r.m;
      u = fmaf(exp_of(d), fmaxf(d, -200.f), u);
    }
  }
  r.s += s;
  r.u += u;
}

// ------------------------------------------------------------ best entries
__device__ __forceinline__ uint64_t entry(float z, uint32_t place) {
  const uint32_t b = __float_as_uint(z + 0.f);  // -0 is 0
  const uint32_t o = (int32_t)b < 0 ? ~b : b | 0x80000000u;
  return (uint64_t)o << 32 | (uint32_t)~place;
}
__device__ __forceinline__ float entry_value(uint64_t e) {
  const uint32_t o = (uint32_t)(e >> 32);
  return __uint_as_float((int32_t)o < 0 ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint32_t entry_place(uint64_t e) { return ~(uint32_t)e; }

// the 32 lanes' entries, which rise and fall or fall and rise once, in falling order
__device__ __forceinline__ uint64_t sort_bitonic(uint64_t v, int lane) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const uint64_t w = __shfl_xor_sync(~0u, v, o);
    v = ((lane & o) == 0) == (v > w) ? v : w;
  }
  return v;
}
__device__ __forceinline__ uint64_t sort32(uint64_t v, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int o = size / 2; o; o >>= 1) {
      const uint64_t w = __shfl_xor_sync(~0u, v, o);
      const bool falling = (lane & size) == 0 || size == 32;
      v = (((lane & o) == 0) == falling) == (v > w) ? v : w;
    }
  return v;
}
// the best 32 of two lists in falling order
__device__ __forceinline__ uint64_t merge32(uint64_t a, uint64_t b, int lane) {
  const uint64_t r = __shfl_sync(~0u, b, 31 - lane);
  return sort_bitonic(a > r ? a : r, lane);
}

// merges the best of this warp's E x 32 logits into the list; `first`: this
// lane's first place (places outside [0, V) are none)
template <int E>
__device__ __forceinline__ void take_best(uint64_t& list, const float* z, int64_t first, int64_t V, int top, int lane) {
  uint64_t offered = ~0ull, worst = __shfl_sync(~0u, list, top - 1);
  while (true) {
    uint64_t mine = 0;  // the best that is better than the worst that counts
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const int64_t at = first + k;
      if (at >= 0 && at < V) {
        const uint64_t e = entry(z[k], (uint32_t)at);
        if (e > worst && e < offered && e > mine) mine = e;
      }
    }
    if (!__any_sync(~0u, mine != 0)) return;
    if (mine) offered = mine;
    list = merge32(list, sort32(mine, lane), lane);
    worst = __shfl_sync(~0u, list, top - 1);
  }
}

// the warps' lists into the first one's
__device__ __forceinline__ uint64_t join_lists(uint64_t list, uint64_t (*lists)[32], int warp, int lane) {
  lists[warp][lane] = list;
  __syncthreads();
#pragma unroll
  for (int n = kLpWarps / 2; n; n >>= 1) {
    if (warp < n) {
      list = merge32(list, lists[warp + n][lane], lane);
      lists[warp][lane] = list;
    }
    __syncthreads();
  }
  return list;
}

// ----------------------------------------------------------------- forward
template <typename T>
struct LpChunk {
  static constexpr int E = 16 / (int)sizeof(T);
};

// E logits of the row from place `at` on; -inf for places outside it
template <typename T>
__device__ __forceinline__ RawVec<16> load_chunk(const T* z, int64_t at, int64_t V) {
  constexpr int E = LpChunk<T>::E;
  if (at >= 0 && at + E <= V) return *reinterpret_cast<const RawVec<16>*>(z + at);
  union U {
    RawVec<16> raw;
    T e[E];
    __device__ U() {}
  } u;
#pragma unroll
  for (int k = 0; k < E; ++k) u.e[k] = at + k >= 0 && at + k < V ? z[at + k] : from_f32<T>(-INFINITY);
  return u.raw;
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kLpThreads, 2) logp_kernel(LpArgs a, int cluster) {
  constexpr int E = LpChunk<T>::E, U = 4;
  __shared__ Running warps[kLpWarps];
  __shared__ uint64_t lists[kLpWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x / cluster;
  const int rank = blockIdx.x % cluster;
  const T* z = (const T*)a.z + row * a.ldz;
  // chunk c holds places [c E - off, c E - off + E), on a 16-byte boundary
  const int off = (int)(((uintptr_t)z & 15) / sizeof(T));
  const int64_t chunks = (a.V + off + E - 1) / E;
  const int64_t share = (chunks + cluster - 1) / cluster;
  const int64_t from = min(chunks, rank * share), to = min(chunks, from + share);

  Running r = nothing();
  // a warp's chunks lie together; whole warps go round
  for (int64_t c0 = from + warp * 32; c0 < to; c0 += U * kLpThreads) {
    RawVec<16> raw[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t c = c0 + i * kLpThreads + lane;
      raw[i] = load_chunk<T>(z, c < to ? c * E - off : a.V, a.V);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (c0 + i * kLpThreads >= to) break;
      float v[E];
      unpack_vec<E, T>(raw[i], v);
      float most = v[0];
#pragma unroll
      for (int k = 1; k < E; ++k) most = fmaxf(most, v[k]);
      take<E>(r, v, most);
    }
  }

  uint64_t best = 0;
  if (TOP) {
    // (a share of infinities below has the maximum of none, which is no less)
    const int64_t c0 = from + warp * 32;
    const bool some = c0 + lane < to;
    join_lists(sort32(some ? entry(r.m, threadIdx.x) : 0, lane), lists, warp, lane);
    const uint64_t kth = lists[0][a.top - 1];
    const float least = kth ? entry_value(kth) : -INFINITY;
    __syncthreads();
    for (uint32_t left = __ballot_sync(~0u, some && r.m >= least); left; left &= left - 1) {
      for (int64_t c = c0 + __ffs(left) - 1 + (int64_t)lane * kLpThreads; __any_sync(~0u, c < to); c += 32 * kLpThreads) {
        const int64_t at = c < to ? c * E - off : a.V;
        float v[E];
        unpack_vec<E, T>(load_chunk<T>(z, at, a.V), v);
        take_best<E>(best, v, at, a.V, a.top, lane);
      }
    }
    best = join_lists(best, lists, warp, lane);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1)
    r = join(r, {__shfl_xor_sync(~0u, r.m, o), __shfl_xor_sync(~0u, r.s, o), __shfl_xor_sync(~0u, r.u, o)});
  if (lane == 0) warps[warp] = r;
  __syncthreads();
  if (warp == 0) {
    r = lane < kLpWarps ? warps[lane] : nothing();
#pragma unroll
    for (int o = kLpWarps / 2; o; o >>= 1)
      r = join(r, {__shfl_xor_sync(~0u, r.m, o), __shfl_xor_sync(~0u, r.s, o), __shfl_xor_sync(~0u, r.u, o)});
    if (lane == 0) warps[0] = r;
  }
  if (cluster > 1) {
    cg::cluster_group group = cg::this_cluster();
    group.sync();
    if (rank == 0 && warp == 0) {
      for (int other = 1; other < cluster; ++other) {
        r = join(r, *group.map_shared_rank(&warps[0], other));
        if (TOP) best = merge32(best, group.map_shared_rank(&lists[0][0], other)[lane], lane);
      }
    }
    group.sync();  // no block leaves while its memory is read
  }
  if (rank != 0 || warp != 0) return;
  // (all lanes have it: lane 0's, so that there is one)
  r = {__shfl_sync(~0u, r.m, 0), __shfl_sync(~0u, r.s, 0), __shfl_sync(~0u, r.u, 0)};
  // a row without any probability: log p is -inf, H is 0
  const bool empty = r.s == 0.f;
  const float logs = empty ? 0.f : logf(r.s);
  const float m = empty ? INFINITY : r.m;
  if (lane == 0) {
    const int64_t t = a.token[row];
    const float h = empty ? 0.f : logs - r.u / r.s;
    const bool given = t >= 0 && t < a.V;
    a.logp[row] = given ? (empty ? -INFINITY : (to_f32(z[t]) - m) - logs) : 0.f;
    a.entropy[row] = h;
    if (a.stats) {
      a.stats[3 * row] = m;
      a.stats[3 * row + 1] = logs;
      a.stats[3 * row + 2] = h;
    }
  }
  if (TOP && lane < a.top) {
    a.top_logp[row * a.top + lane] = empty ? -INFINITY : (entry_value(best) - m) - logs;
    a.top_at[row * a.top + lane] = entry_place(best);
  }
}

// ---------------------------------------------------------------- backward
// blockIdx.x: row, blockIdx.y: part of it
template <typename T>
__global__ void __launch_bounds__(256) logp_bwd_kernel(LpBwdArgs a, int64_t share, int same) {
  constexpr int E = LpChunk<T>::E, U = 4;
  const int64_t row = blockIdx.x;
  const T* z = (const T*)a.z + row * a.ldz;
  T* dz = (T*)a.dz + row * a.V;
  const int64_t t = a.token[row];
  const float m = a.stats[3 * row], logs = a.stats[3 * row + 1], h = a.stats[3 * row + 2];
  const bool given = t >= 0 && t < a.V;
  const float g = given && a.g_logp ? a.g_logp[a.one_logp ? 0 : row] : 0.f;
  const float k = a.g_entropy ? a.g_entropy[a.one_entropy ? 0 : row] : 0.f;
  const bool empty = m == INFINITY && logs == 0.f && h == 0.f;
  auto one = [&](float zz, int64_t at) {
    const float lp = (zz - m) - logs, p = exp_of(lp);
    // (p is 0 below -88)
    float d = p * -fmaf(k, fmaxf(lp, -200.f) + h, g);
    d = empty ? 0.f : d;
    return at == t ? (empty ? 0.f : d + g) : d;
  };
  const int off = (int)(((uintptr_t)dz & 15) / sizeof(T));
  const int64_t chunks = (a.V + off + E - 1) / E;
  const int64_t to = min(chunks, (blockIdx.y + 1) * share);
  for (int64_t c0 = blockIdx.y * share + threadIdx.x; c0 < to; c0 += U * 256) {
    RawVec<16> raw[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t at = (c0 + i * 256) * E - off;
      if (same && c0 + i * 256 < to && at >= 0 && at + E <= a.V) raw[i] = *reinterpret_cast<const RawVec<16>*>(z + at);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (c0 + i * 256 >= to) break;
      const int64_t at = (c0 + i * 256) * E - off;
      if (same && at >= 0 && at + E <= a.V) {
        float v[E];
        unpack_vec<E, T>(raw[i], v);
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = one(v[j], at + j);
        store_vec<E>(dz + at, v);
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (at + j >= 0 && at + j < a.V) dz[at + j] = from_f32<T>(one(to_f32(z[at + j]), at + j));
      }
    }
  }
}

// --------------------------------------------------------------- host side
static int lp_check(const pvb2_token_logp_desc* d) {
  PVB2_CHECK_ARG(d, "token_log_probs: no descriptor");
  PVB2_CHECK_ARG(d->dtype == PVB2_F32 || d->dtype == PVB2_F16 || d->dtype == PVB2_BF16,
                 "token_log_probs: fp32, fp16 or bf16 logits expected (got dtype %d)", d->dtype);
  PVB2_CHECK_ARG(d->N >= 0 && d->N < (1 << 27) && d->V >= 1 && d->V < ((int64_t)1 << 31),
                 "token_log_probs: %lld rows of %lld logits out of range", (long long)d->N, (long long)d->V);
  PVB2_CHECK_ARG(d->top >= 0 && d->top <= kLpTop && d->top <= d->V, "token_log_probs: top is 0 to %d and at most the logits",
                 kLpTop);
  PVB2_CHECK_ARG(d->N <= 1 || d->ldz >= d->V, "token_log_probs: row stride below the rows' length");
  return PVB2_OK;
}

template <typename T, bool TOP>
static int launch_lp(const LpArgs& a, cudaStream_t s) {
  // a row over as many blocks as leave each 16 KB, while there are SMs without one
  int cluster = 1;
  while (cluster < kLpCluster && a.N * cluster < num_sms() && a.V * (int64_t)sizeof(T) / (2 * cluster) >= 16384) cluster *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.N * cluster));
  cfg.blockDim = dim3(kLpThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  PVB2_CUDA_TRY(cudaLaunchKernelEx(&cfg, logp_kernel<T, TOP>, a, cluster));
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

template <typename T>
static int launch_lp_bwd(const LpBwdArgs& a, cudaStream_t s) {
  constexpr int E = LpChunk<T>::E;
  // parts of 8 rounds of a block, fewer where the rows alone do not fill the SMs
  const int64_t chunks = (a.V + 2 * E - 2) / E;
  int64_t share = 8 * 4 * 256;
  while (share > 256 && a.N * ((chunks + share - 1) / share) < 4 * (int64_t)num_sms()) share /= 2;
  share = std::max(share, (chunks + 65534) / 65535);
  const int same = ((uintptr_t)a.z & 15) == ((uintptr_t)a.dz & 15) && (a.N <= 1 || (a.ldz - a.V) * (int64_t)sizeof(T) % 16 == 0);
  logp_bwd_kernel<T><<<dim3((unsigned)a.N, (unsigned)((chunks + share - 1) / share)), 256, 0, s>>>(a, share, same);
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

}  // namespace pvb2

using namespace pvb2;

extern "C" {

int pvb2_token_logp_fwd(const pvb2_token_logp_desc* d, const void* logits, const int64_t* tokens, float* logp,
                        float* entropy, float* stats, float* top_logp, int64_t* top_index, pvb2_stream stream) {
  PVB2_TRY(lp_check(d));
  if (d->N == 0) return PVB2_OK;
  PVB2_CHECK_ARG(logits && tokens && logp && entropy && (!d->top || (top_logp && top_index)), "token_log_probs: null pointer");
  const LpArgs a = {logits, tokens, logp, entropy, stats, top_logp, top_index, d->N, d->V, d->ldz, d->top};
  cudaStream_t s = as_stream(stream);
  if (d->dtype == PVB2_F32) return d->top ? launch_lp<float, true>(a, s) : launch_lp<float, false>(a, s);
  if (d->dtype == PVB2_BF16) return d->top ? launch_lp<__nv_bfloat16, true>(a, s) : launch_lp<__nv_bfloat16, false>(a, s);
  return d->top ? launch_lp<__half, true>(a, s) : launch_lp<__half, false>(a, s);
}

int pvb2_token_logp_bwd(const pvb2_token_logp_desc* d, const void* logits, const int64_t* tokens, const float* stats,
                        const float* g_logp, int one_logp, const float* g_entropy, int one_entropy, void* dlogits,
                        pvb2_stream stream) {
  PVB2_TRY(lp_check(d));
  if (d->N == 0) return PVB2_OK;
  PVB2_CHECK_ARG(logits && tokens && stats && dlogits, "token_log_probs: null pointer");
  const LpBwdArgs a = {logits, tokens, stats, g_logp, g_entropy, dlogits, d->N, d->V, d->ldz, one_logp, one_entropy};
  cudaStream_t s = as_stream(stream);
  if (d->dtype == PVB2_F32) return launch_lp_bwd<float>(a, s);
  if (d->dtype == PVB2_BF16) return launch_lp_bwd<__nv_bfloat16>(a, s);
  return launch_lp_bwd<__half>(a, s);
}

}  // extern "C"
