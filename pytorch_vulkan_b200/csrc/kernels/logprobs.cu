// Log probabilities of given tokens, the entropy and the best alternatives of
// rows of logits, and their gradient.
//
//   m = max z,  s = sum e^(z - m),  u = sum e^(z - m) (z - m)
//   log p_t = (z_t - m) - log s,    H = log s - u / s
//   dz_j = p_j (-g - k (log p_j + H)) + g [j = t]      (g of log p_t, k of H)
//
// The forward pass reads the logits once, the backward pass reads them once
// more and writes as much: both are bound by HBM.  16-bit logits come at a rate
// at which the forward pass has ten instructions for each: exponentials are 2^x
// with x = z log2(e) - M, one multiply-add, M being the thread's running maximum
// times log2(e), rounded.  A thread's s and u hold relative to M exactly as it
// is, and are moved to m itself at the end, so that M's rounding does not count
// however large the logits are.  Where M is beyond fp32 (logits of 2e38, or
// nothing but the type's lowest number) a thread that has summed nothing reads
// its share again and subtracts before it multiplies.
//
// Each thread copies its chunks of 16 bytes into a ring of its own in shared
// memory, eight ahead, without barriers: registers for as many loads in flight
// would halve the threads.  A row is a warp's, a block's of 128 or 512, or, where
// rows are few, a cluster's, whose blocks join through shared memory: one
// launch, no workspace.
//
// The best ones.  A thread's maximum is the best of its share of the row.  Of
// the k best, none is in a share whose maximum is below the k-th best maximum
// of all threads, and so few more than k shares are read a second time (out of
// L2), by all threads together, and what is not below that goes to a list that
// one warp sorts.  An entry is a 64-bit number, the logit's bits in an order in
// which integers compare as numbers do, and below them the complement of its
// place, so that of equal logits the lower place is better.  Where equal logits
// overflow the list, each warp keeps its best 32, one entry a lane, and they are
// merged by bitonic networks.  The main loop does nothing for any of this.
//
// Rows begin on any element: whole 16-byte chunks are read wherever they lie,
// the ones at the ends element by element.
#include <cooperative_groups.h>
#include <algorithm>
#include <cfloat>
#include <type_traits>
#include "types.cuh"

namespace pvb2 {
namespace cg = cooperative_groups;

constexpr int kLpTop = 32;
constexpr int kLpCluster = 8;
constexpr int kLpRing = 8;  // chunks of a thread on their way

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

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
__device__ __forceinline__ float exp2_of(float x) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x));
  return e;
}

struct Running {
  float m, s, u;  // m: -inf before any logit above that
};

// relative to m, no less than r.m
__device__ __forceinline__ void move_max(Running& r, float m) {
  if (!(m > r.m)) return;
  const float d = r.m - m, c = exp2_of(d * kLog2e);
  // (c is 0 where d is far below; 0 times an infinity is none)
  r.u = c > 0.f || r.s != r.s ? c * fmaf(r.s, d, r.u) : 0.f;
  r.s *= c;
  r.m = m;
}

__device__ __forceinline__ Running join(Running a, Running b) {
  const float m = fmaxf(a.m, b.m);
  move_max(a, m);
  move_max(b, m);
  return {m, a.s + b.s, a.u + b.u};
}

// E logits more, by differences: for any of them
template <int E>
__device__ __forceinline__ void take_slowly(Running& r, const float* z) {
  float most = z[0];
#pragma unroll
  for (int k = 1; k < E; ++k) most = fmaxf(most, z[k]);
  move_max(r, most);
#pragma unroll
  for (int k = 0; k < E; ++k) {
    // below -200 an exponential is 0 (and -inf times it is none); without a maximum there are but -inf and NaN
    const float d = r.m == -INFINITY ? (z[k] != z[k] ? z[k] : -INFINITY) : z[k] - r.m, e = exp2_of(d * kLog2e);
    r.s += e;
    r.u = fmaf(e, fmaxf(d, -200.f), r.u);
  }
}

// the same in powers of two, relative to `ref`
struct Running2 {
  float m, ref, s, u;
};
template <int E>
__device__ __forceinline__ void take(Running2& r, const float* z, float most) {
  if (most > r.m) {
    // (logits of 2e38 make it infinite and those of -2e38 clamp it: nothing is summed)
    const float ref = fmaxf(most * kLog2e, -FLT_MAX);
    if (r.s != 0.f) {
      const float d = r.ref - ref, c = exp2_of(d);
      r.u = c > 0.f || r.s != r.s ? c * fmaf(r.s, d, r.u) : 0.f;
      r.s *= c;
    }
    r.m = most;
    r.ref = ref;
  }
  float s = 0.f, u = 0.f;
#pragma unroll
  for (int k = 0; k < E; ++k) {
    const float d = fmaf(z[k], kLog2e, -r.ref), e = exp2_of(d);
    s += e;
    u = fmaf(e, d, u);
  }
  if (u != u) {  // e is 0 and d -inf somewhere (or something is NaN, which s is too)
    u = 0.f;
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const float d = fmaf(z[k], kLog2e, -r.ref);
      u = fmaf(exp2_of(d), fmaxf(d, -200.f), u);
    }
  }
  r.s += s;
  r.u += u;
}

// relative to m, in powers of e
__device__ __forceinline__ Running moved(const Running2& r) {
  if (r.s == 0.f) return {r.m, 0.f, 0.f};
  // sum 2^(z l - ref) = 2^c sum 2^((z - m) l)
  const float c = fmaf(r.m, kLog2e, -r.ref), back = exp2_of(-c), s = r.s * back;
  return {r.m, s, kLn2 * fmaf(-c, s, r.u * back)};
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

// the same of maxima alone
__device__ __forceinline__ float sort32(float v, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int o = size / 2; o; o >>= 1) {
      const float w = __shfl_xor_sync(~0u, v, o);
      v = ((lane & o) == 0) == ((lane & size) == 0 || size == 32) ? fmaxf(v, w) : fminf(v, w);
    }
  return v;
}
__device__ __forceinline__ float merge32(float a, float b, int lane) {
  float v = fmaxf(a, __shfl_sync(~0u, b, 31 - lane));
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float w = __shfl_xor_sync(~0u, v, o);
    v = (lane & o) == 0 ? fmaxf(v, w) : fminf(v, w);
  }
  return v;
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

// G threads to a row: a warp (of blocks of four), or a block
template <int G>
struct LpRow {
  static constexpr int THREADS = G < 128 ? 128 : G, ROWS = THREADS / G, WARPS = G / 32;
  static constexpr int LIST = G < 128 ? 64 : 256;  // candidates that fit
  // of a row
  Running parts[WARPS];
  float maxima[WARPS][32];
  uint64_t lists[WARPS][32];
  uint64_t found[LIST];
  int shares[G];
  int n_shares, n_found;
};
template <int G>
__device__ __forceinline__ void row_sync() {
  if (G == 32) __syncwarp();
  else __syncthreads();
}

// the lists of the first n warps of a row into the first one's
template <typename V>
__device__ __forceinline__ V join_lists(V list, V (*lists)[32], int n, int warp, int lane) {
  if (n == 1) return list;
  if (warp < n) lists[warp][lane] = list;
  __syncthreads();
  for (n /= 2; n; n /= 2) {
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

template <typename T>
__device__ __forceinline__ float most_of(const RawVec<16>& raw, const float* v) {
  if constexpr (sizeof(T) == 2) {
    using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
    union U {
      RawVec<16> raw;
      T2 e[4];
      __device__ U() {}
    } u;
    u.raw = raw;
    const T2 m = __hmax2(__hmax2(u.e[0], u.e[1]), __hmax2(u.e[2], u.e[3]));
    return fmaxf(to_f32(m.x), to_f32(m.y));  // (a NaN loses, as it does below)
  } else {
    return fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
  }
}

__device__ __forceinline__ void copy16_async(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}

template <typename T, bool TOP, int G>
__global__ void __launch_bounds__(LpRow<G>::THREADS, G == 512 ? 2 : 8) logp_kernel(LpArgs a, int cluster) {
  constexpr int E = LpChunk<T>::E, R = kLpRing;
  using Row = LpRow<G>;
  extern __shared__ __align__(16) uint8_t ring[];  // [R][threads][16]
  __shared__ Row rows[Row::ROWS];
  const int t = threadIdx.x % G, lane = threadIdx.x & 31, warp = t >> 5;
  Row& mine = rows[threadIdx.x / G];
  const int64_t row = (int64_t)(blockIdx.x / cluster) * Row::ROWS + threadIdx.x / G;
  const int rank = blockIdx.x % cluster;
  if (row >= a.N) return;  // whole warps, of blocks whose warps do not meet
  const T* z = (const T*)a.z + row * a.ldz;
  // chunk c holds places [c E - off, c E - off + E), on a 16-byte boundary; of
  // the whole ones this block has [from, to), the others are the first and the
  // last block's
  const int off = (int)(((uintptr_t)z & 15) / sizeof(T));
  const int64_t lo = off ? 1 : 0, hi = max(lo, (a.V + off) / E);
  const int64_t share = (hi - lo + cluster - 1) / cluster;
  const int64_t from = min(hi, lo + rank * share), to = min(hi, from + share);
  // the places that thread `th` has beside them: none (V) or those of an end
  auto end_of = [&](int th) {
    if (th == 0 && off && rank == 0) return (int64_t)-off;
    if (th == 1 && rank == cluster - 1 && hi * E - off < a.V) return hi * E - off;
    return a.V;
  };

  // this thread's chunks: from + t, and every G-th from there
  const int n = (int)max((int64_t)0, (to - from - t + G - 1) / G);
  const T* next = z + ((from + t) * E - off);
  uint32_t slot0;
  slot0 = (uint32_t)__cvta_generic_to_shared(ring) + threadIdx.x * 16;
  constexpr int kSlot = Row::THREADS * 16;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (i < n) {
      copy16_async(slot0 + i * kSlot, next);
      next += G * E;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  Running2 r = {-INFINITY, 0.f, 0.f, 0.f};
  {
    const int64_t at = end_of(t);
    if (at < a.V) {
      const RawVec<16> raw = load_chunk<T>(z, at, a.V);
      float v[E];
      unpack_vec<E, T>(raw, v);
      take<E>(r, v, most_of<T>(raw, v));
    }
  }
  for (int i0 = 0; i0 < n; i0 += R) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (i0 + i >= n) break;
      asm volatile("cp.async.wait_group %0;" ::"n"(R - 1) : "memory");
      RawVec<16> raw;
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(raw.a.x), "=r"(raw.a.y), "=r"(raw.a.z), "=r"(raw.a.w)
                   : "r"(slot0 + i * kSlot)
                   : "memory");
      float v[E];
      unpack_vec<E, T>(raw, v);
      take<E>(r, v, most_of<T>(raw, v));
      // (the slot has been read: its numbers have been used)
      if (i0 + i + R < n) {
        copy16_async(slot0 + i * kSlot, next);
        next += G * E;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  }
  const float most = r.m;
  Running sum = moved(r);
  if (r.s == 0.f && most > -INFINITY) {  // beyond fp32 times log2(e)
    sum = {-INFINITY, 0.f, 0.f};
    float v[E];
    for (int i = 0; i < n; ++i) {
      unpack_vec<E, T>(load_chunk<T>(z, (from + t + (int64_t)i * G) * E - off, a.V), v);
      take_slowly<E>(sum, v);
    }
    unpack_vec<E, T>(load_chunk<T>(z, end_of(t), a.V), v);
    take_slowly<E>(sum, v);
  }

  uint64_t best = 0;
  if (TOP) {
    const bool some = n > 0 || end_of(t) < a.V;
    // NaN: no share (fmax and fmin would take it for the other's)
    const float kth_most = join_lists<float>(sort32(some ? most : -INFINITY, lane), mine.maxima, Row::WARPS, warp, lane);
    if (warp == 0) mine.maxima[0][lane] = kth_most;
    if (t == 0) mine.n_shares = mine.n_found = 0;
    row_sync<G>();
    const float least = mine.maxima[0][a.top - 1];
    if (some && most >= least) mine.shares[atomicAdd(&mine.n_shares, 1)] = t;
    row_sync<G>();
    // the chunks of these shares, and the ends
    const int shares = mine.n_shares, per = (int)((to - from + G - 1) / G) + 1;
    const int pairs = shares * per;
    auto chunk_of = [&](int pair, float* v) {
      int64_t at = a.V;
      if (pair < pairs) {
        const int th = mine.shares[pair / per], i = pair % per;
        const int64_t c = from + th + (int64_t)(i - 1) * G;
        if (i == 0) at = end_of(th);
        else if (c < to) at = c * E - off;
      }
      unpack_vec<E, T>(load_chunk<T>(z, at, a.V), v);
      return at;
    };
    for (int pair = t; pair < pairs; pair += G) {
      float v[E];
      const int64_t at = chunk_of(pair, v);
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (at + k >= 0 && at + k < a.V && !(v[k] < least)) {
          const int i = atomicAdd(&mine.n_found, 1);
          if (i < Row::LIST) mine.found[i] = entry(v[k], (uint32_t)(at + k));
        }
    }
    row_sync<G>();
    const int found = mine.n_found;
    if (found <= Row::LIST) {
      if (warp == 0)
        for (int i = 0; i < found; i += 32) {
          const uint64_t sorted = sort32(i + lane < found ? mine.found[i + lane] : 0, lane);
          best = i ? merge32(best, sorted, lane) : sorted;
        }
    } else {
      for (int pair = warp * 32; pair < pairs; pair += G) {
        float v[E];
        const int64_t at = chunk_of(pair + lane, v);
        take_best<E>(best, v, at, a.V, a.top, lane);
      }
      best = join_lists<uint64_t>(best, mine.lists, Row::WARPS, warp, lane);
    }
    if (G > 32 && warp == 0) mine.lists[0][lane] = best;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1)
    sum = join(sum, {__shfl_xor_sync(~0u, sum.m, o), __shfl_xor_sync(~0u, sum.s, o), __shfl_xor_sync(~0u, sum.u, o)});
  if (G > 32) {
    if (lane == 0) mine.parts[warp] = sum;
    __syncthreads();
    if (warp == 0) {
      sum = lane < Row::WARPS ? mine.parts[lane] : Running{-INFINITY, 0.f, 0.f};
#pragma unroll
      for (int o = Row::WARPS / 2; o; o >>= 1)
        sum = join(sum, {__shfl_xor_sync(~0u, sum.m, o), __shfl_xor_sync(~0u, sum.s, o), __shfl_xor_sync(~0u, sum.u, o)});
      if (lane == 0) mine.parts[0] = sum;
    }
  }
  if (cluster > 1) {
    cg::cluster_group group = cg::this_cluster();
    group.sync();
    if (rank == 0 && warp == 0) {
      Running part[kLpCluster];
      uint64_t list[kLpCluster];
#pragma unroll
      for (int i = 1; i < kLpCluster; ++i)
        if (i < cluster) {
          part[i] = *group.map_shared_rank(&mine.parts[0], i);
          if (TOP) list[i] = group.map_shared_rank(&mine.lists[0][0], i)[lane];
        }
#pragma unroll
      for (int i = 1; i < kLpCluster; ++i)
        if (i < cluster) {
          sum = join(sum, part[i]);
          if (TOP) best = merge32(best, list[i], lane);
        }
    }
    group.sync();  // no block leaves while its memory is read
  }
  if (rank != 0 || warp != 0) return;
  // (all lanes have it: lane 0's, so that there is one)
  sum = {__shfl_sync(~0u, sum.m, 0), __shfl_sync(~0u, sum.s, 0), __shfl_sync(~0u, sum.u, 0)};
  // a row without any probability: log p is -inf, H is 0
  const bool empty = sum.s == 0.f;
  const float logs = empty ? 0.f : logf(sum.s);
  const float m = empty ? INFINITY : sum.m;
  if (lane == 0) {
    const int64_t tok = a.token[row];
    const float h = empty ? 0.f : logs - sum.u / sum.s;
    const bool given = tok >= 0 && tok < a.V;
    a.logp[row] = given ? (empty ? -INFINITY : (to_f32(z[tok]) - m) - logs) : 0.f;
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
  // (a row without any probability has m = inf and no other number)
  const bool empty = m == INFINITY && logs == 0.f && h == 0.f;
  const float logs2 = -logs * kLog2e, slope = -k * kLn2, rest = -fmaf(k, h, g);
  // -p (g + k (log p + H)); p is 0 below 2^-126, where log p may be -inf
  auto one = [&](float zz) {
    const float lp = fmaf(zz - m, kLog2e, logs2), p = exp2_of(lp);
    return p * fmaf(fmaxf(lp, -300.f), slope, rest);
  };
  auto with_token = [&](float d, int64_t at) { return empty ? 0.f : at == t && given ? d + g : d; };
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
        for (int j = 0; j < E; ++j) v[j] = one(v[j]);
        if (empty || (uint64_t)(t - at) < E) {
#pragma unroll
          for (int j = 0; j < E; ++j) v[j] = with_token(v[j], at + j);
        }
        store_vec<E>(dz + at, v);
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (at + j >= 0 && at + j < a.V) dz[at + j] = from_f32<T>(with_token(one(to_f32(z[at + j])), at + j));
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

template <typename T, bool TOP, int G>
static int launch_lp_as(const LpArgs& a, int cluster, cudaStream_t s) {
  using Row = LpRow<G>;
  constexpr int smem = kLpRing * Row::THREADS * 16;
  auto kernel = logp_kernel<T, TOP, G>;
  static DeviceOnce once;
  PVB2_TRY(allow_smem(kernel, smem, once));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.N + Row::ROWS - 1) / Row::ROWS * cluster));
  cfg.blockDim = dim3(Row::THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  PVB2_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a, cluster));
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

template <typename T, bool TOP>
static int launch_lp(const LpArgs& a, cudaStream_t s) {
  const int64_t bytes = a.V * (int64_t)sizeof(T);
  // Rows of up to eight chunks for each of their threads are a warp's, or 128
  // threads'; where they leave SMs without a row, more threads' and, while each
  // block keeps 16 KB, several blocks'.
  if (bytes <= 4096 && (a.N >= num_sms() || bytes <= 1024)) return launch_lp_as<T, TOP, 32>(a, 1, s);
  if (bytes <= 32768 && (a.N >= num_sms() || bytes <= 8192)) return launch_lp_as<T, TOP, 128>(a, 1, s);
  int cluster = 1;
  while (cluster < kLpCluster && a.N * cluster < num_sms() && bytes / (2 * cluster) >= 16384) cluster *= 2;
  return launch_lp_as<T, TOP, 512>(a, cluster, s);
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
