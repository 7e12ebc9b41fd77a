// Log probabilities of given tokens, the entropy and the best alternatives of
// rows of logits, and their gradient.
//
//   m = max z,  s = sum e^(z - m),  u = sum e^(z - m) (z - m)
//   log p_t = (z_t - m) - log s,    H = log s - u / s
//   dz_j = p_j (-g - k (log p_j + H)) + g [j = t]      (g of log p_t, k of H)
//
// The forward pass reads the logits once, the backward pass reads them once
// more and writes as much: both are bound by HBM (8192 x 131072 bf16: 355 us
// forward, 6.0 TB/s, and 650 us backward, 6.6 TB/s; called without a pause the
// forward pass draws all of the board's power and takes 420 at 1.5 GHz).  16-bit
// logits come at a rate at which the forward pass has ten instructions for each;
// it takes 6.6.  Exponentials are 2^x with x = z log2(e) - M, one multiply-add, M
// being the thread's running maximum times log2(e), rounded, or that of an
// earlier maximum at most 2 below.  A thread's s and u hold relative to M exactly
// as it is, and are moved to m itself at the end, so that M's rounding does not
// count however large the logits are.  M is rounded up; where its steps are so
// wide that a thread has summed nothing (logits of 1e10 or more, or nothing but
// -1e10 or less, as a finite mask leaves it), it reads its share again and
// subtracts before it multiplies.
//
// Each thread copies its chunks of 16 bytes into a ring of its own in shared
// memory, eight ahead, without barriers: registers for as many loads in flight
// would halve the threads.  The forward pass takes four at a time (4095 x 49999
// with 5 alternatives: 97 us; in twos 104).  A row is a warp's, a block's of 128
// or 256, or, where rows are few, a cluster's, whose blocks join through shared
// memory: one launch, no workspace.
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
#include "overlap.cuh"
#include "types.cuh"

namespace pvb2 {
namespace cg = cooperative_groups;

constexpr int kLpTop = 32;
constexpr int kLpCluster = 8;
constexpr int kLpRing = 8;  // chunks of a thread on their way
constexpr int kLpGroup = 4;  // that the forward pass takes at a time

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

// two fp32 numbers in a register pair, which one instruction works on
__device__ __forceinline__ uint64_t pair_of(float x, float y) {
  uint64_t p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(x), "f"(y));
  return p;
}
__device__ __forceinline__ float2 numbers(uint64_t p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
  return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// the same in powers of two, relative to `ref`, which serves logits up to `next`
struct Running2 {
  float m, next, ref, s, u;
};
constexpr float kAhead = 2.f;
template <int N>
__device__ __forceinline__ void take(Running2& r, const float* z, float most) {
  r.m = fmaxf(r.m, most);
  // (a maximum that grows by less than kAhead leaves ref where it is: powers up
  // to 8 cost the sums nothing, and some lane of a warp has a new one nearly
  // every time)
  if (most > r.next) {
    // rounded up, so that the maximum's power is no more than 1: where ref's steps
    // are wide (logits of 1e10 either way; 2e38 makes it infinite) nothing is summed
    const float ref = fmaxf(__fmul_ru(most, kLog2e), -FLT_MAX);
    if (r.s != 0.f) {
      const float d = r.ref - ref, c = exp2_of(d);
      r.u = c > 0.f || r.s != r.s ? c * fmaf(r.s, d, r.u) : 0.f;
      r.s *= c;
    }
    r.next = most + kAhead;
    r.ref = ref;
  }
  const uint64_t l = pair_of(kLog2e, kLog2e), ref = pair_of(-r.ref, -r.ref);
  uint64_t s2 = 0, u2 = 0;
#pragma unroll
  for (int k = 0; k < N; k += 2) {
    const uint64_t d2 = fma2(pair_of(z[k], z[k + 1]), l, ref);
    const float2 d = numbers(d2);
    const uint64_t e2 = pair_of(exp2_of(d.x), exp2_of(d.y));
    s2 = k ? add2(s2, e2) : e2;
    u2 = k ? fma2(e2, d2, u2) : mul2(e2, d2);
  }
  const float2 s = numbers(s2), us = numbers(u2);
  float u = us.x + us.y;
  if (u != u) {  // e is 0 and d -inf somewhere (or something is NaN, which s is too)
    u = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float d = fmaf(z[k], kLog2e, -r.ref);
      u = fmaf(exp2_of(d), fmaxf(d, -200.f), u);
    }
  }
  r.s += s.x + s.y;
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
  static constexpr int LIST = G < 128 ? 96 : 256;  // candidates that fit: three times the best at least
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

// (a NaN loses, to the other and to r.m)
template <typename T, int CHUNKS>
__device__ __forceinline__ float most_of(const RawVec<16>* raw) {
  if constexpr (sizeof(T) == 2) {
    using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
    union U {
      RawVec<16> raw[CHUNKS];
      T2 e[4 * CHUNKS];
      __device__ U() {}
    } u;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) u.raw[i] = raw[i];
    T2 m = u.e[0];
#pragma unroll
    for (int i = 1; i < 4 * CHUNKS; ++i) m = __hmax2(m, u.e[i]);
    return fmaxf(to_f32(m.x), to_f32(m.y));
  } else {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      float v[4];
      unpack_vec<4, float>(raw[i], v);
      m = fmaxf(m, fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])));
    }
    return m;
  }
}

// A thread's chunks of 16 bytes, STEP bytes apart, by way of its slots in shared
// memory, GROUP of them at a time.
template <int THREADS, int GROUP>
struct Ring {
  uint32_t slots;
  const char* next;
  int left;  // chunks that have not been asked for
  static constexpr int kSlot = THREADS * 16;

  // chunk `i` from here, if there is one
  template <int STEP>
  __device__ __forceinline__ void ask(int i) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.gt.s32 p, %2, %3;\n\t"
        "@p cp.async.cg.shared.global [%0], [%1], 16;\n\t}" ::"r"(slots + i * kSlot),
        "l"(next + (int64_t)i * STEP), "r"(left), "r"(i)
        : "memory");
  }
  template <int STEP>
  __device__ __forceinline__ void ask_group(int slot) {
#pragma unroll
    for (int i = slot; i < slot + GROUP; ++i) ask<STEP>(i);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  template <int STEP>
  __device__ __forceinline__ void begin(void* smem, const void* first, int n) {
    slots = (uint32_t)__cvta_generic_to_shared(smem) + threadIdx.x * 16;
    next = (const char*)first;
    left = n;
#pragma unroll
    for (int i = 0; i < kLpRing; i += GROUP) ask_group<STEP>(i);
    left -= kLpRing;
    next += (int64_t)kLpRing * STEP;
  }
  __device__ __forceinline__ RawVec<16> get(int slot) const {
    RawVec<16> raw;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(raw.a.x), "=r"(raw.a.y), "=r"(raw.a.z), "=r"(raw.a.w)
                 : "r"(slots + slot * kSlot)
                 : "memory");
    return raw;
  }
  // the n chunks go to `f`, in groups and the last ones singly: the first's number, they, how many
  template <int STEP, typename F>
  __device__ __forceinline__ void walk(int n, F f) {
    int i0 = 0;
    for (; i0 + kLpRing <= n; i0 += kLpRing) {
#pragma unroll
      for (int i = 0; i < kLpRing; i += GROUP) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kLpRing / GROUP - 1) : "memory");
        RawVec<16> raw[GROUP];
#pragma unroll
        for (int k = 0; k < GROUP; ++k) raw[k] = get(i + k);
        f(i0 + i, raw, std::integral_constant<int, GROUP>());
        // (the slots have been read: their numbers have been used)
        ask_group<STEP>(i);
      }
      left -= kLpRing;
      next += (int64_t)kLpRing * STEP;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    int i = 0;
    for (; i0 + i + GROUP <= n; i += GROUP) {
      RawVec<16> raw[GROUP];
#pragma unroll
      for (int k = 0; k < GROUP; ++k) raw[k] = get(i + k);
      f(i0 + i, raw, std::integral_constant<int, GROUP>());
    }
    for (; i0 + i < n; ++i) {
      const RawVec<16> raw[1] = {get(i)};
      f(i0 + i, raw, std::integral_constant<int, 1>());
    }
  }
};

template <typename T, bool TOP, int G>
__global__ void __launch_bounds__(LpRow<G>::THREADS, 1024 / LpRow<G>::THREADS) logp_kernel(LpArgs a, int cluster) {
  let_next_come();
  wait_for_last();
  constexpr int E = LpChunk<T>::E;
  using Row = LpRow<G>;
  extern __shared__ __align__(16) uint8_t ring[];  // [kLpRing][threads][16]
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
  Ring<Row::THREADS, kLpGroup> chunks;
  chunks.template begin<G * 16>(ring, z + ((from + t) * E - off), n);
  Running2 r = {-INFINITY, -INFINITY, 0.f, 0.f, 0.f};
  {
    const int64_t at = end_of(t);
    if (at < a.V) {
      const RawVec<16> raw = load_chunk<T>(z, at, a.V);
      float v[E];
      unpack_vec<E, T>(raw, v);
      take<E>(r, v, most_of<T, 1>(&raw));
    }
  }
  chunks.template walk<G * 16>(n, [&](int, const RawVec<16>* raw, auto count) {
    constexpr int N = decltype(count)::value;
    float v[N * E];
#pragma unroll
    for (int k = 0; k < N; ++k) unpack_vec<E, T>(raw[k], v + k * E);
    take<N * E>(r, v, most_of<T, N>(raw));
  });
  const float most = r.m;
  Running sum = moved(r);
  if (r.s == 0.f && most > -INFINITY) {  // M is further from log2(e) times the maximum than 126
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
    // (a mask that leaves fewer shares than that: what it left, and the first of what it hid)
    const bool masked = least == -INFINITY;
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
      if (*(volatile int*)&mine.n_found > Row::LIST) break;  // (they are counted one at a time)
      float v[E];
      const int64_t at = chunk_of(pair, v);
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (at + k >= 0 && at + k < a.V && !(masked ? v[k] == -INFINITY : v[k] < least)) {
          const int i = atomicAdd(&mine.n_found, 1);
          if (i < Row::LIST) mine.found[i] = entry(v[k], (uint32_t)(at + k));
        }
    }
    row_sync<G>();
    int found = mine.n_found;
    if (masked && found < a.top) {
      // among as many places as there are to find and have been found, enough are hidden
      const int64_t begin = rank == 0 ? 0 : from * E - off, end = rank == cluster - 1 ? a.V : to * E - off;
      row_sync<G>();
      for (int i = t; i < a.top + found; i += G)
        if (begin + i < end && to_f32(z[begin + i]) == -INFINITY)
          mine.found[atomicAdd(&mine.n_found, 1)] = entry(-INFINITY, (uint32_t)(begin + i));
      row_sync<G>();
      found = mine.n_found;
    }
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
  // (s holds the maximum's 1, u nothing above 0: roundings must not make a log
  // probability of more than 0 or an entropy of less; a NaN stays one)
  if (sum.s < 1.f && !empty) sum.s = 1.f;
  if (sum.u > 0.f) sum.u = 0.f;
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
// two numbers, rounded
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

struct LpRowGrad {
  float m, logs2, slope, rest, g;
  int64_t t;  // place of the token, -1: none
  bool empty;
  __device__ __forceinline__ LpRowGrad(const LpBwdArgs& a, int64_t row) {
    m = a.stats[3 * row];
    const float logs = a.stats[3 * row + 1], h = a.stats[3 * row + 2];
    const int64_t token = a.token[row];
    t = token >= 0 && token < a.V ? token : -1;
    g = t >= 0 && a.g_logp ? a.g_logp[a.one_logp ? 0 : row] : 0.f;
    const float k = a.g_entropy ? a.g_entropy[a.one_entropy ? 0 : row] : 0.f;
    logs2 = -logs * kLog2e;
    slope = -k * kLn2;
    rest = -fmaf(k, h, g);
    // (a row without any probability has m = inf and no other number)
    empty = m == INFINITY && logs == 0.f && h == 0.f;
  }
  // -p (g + k (log p + H)); p is 0 below 2^-126, where log p may be -inf
  __device__ __forceinline__ float one(float z) const {
    const float lp = fmaf(z - m, kLog2e, logs2);
    return exp2_of(lp) * fmaf(fmaxf(lp, -300.f), slope, rest);
  }
  __device__ __forceinline__ float with_token(float d, int64_t at) const { return empty ? 0.f : at == t ? d + g : d; }
};

constexpr int kLpBwdThreads = 256;

// blockIdx.x: row, blockIdx.y: part of it, of `share` whole chunks.  SAME: the
// chunks of z and of dz lie on the same boundaries.
template <typename T, bool SAME>
__global__ void __launch_bounds__(kLpBwdThreads, 5) logp_bwd_kernel(LpBwdArgs a, int64_t share) {
  let_next_come();
  wait_for_last();
  constexpr int E = LpChunk<T>::E, G = kLpBwdThreads;
  extern __shared__ __align__(16) uint8_t ring[];  // [kLpRing][threads][16]
  const int64_t row = blockIdx.x;
  const T* z = (const T*)a.z + row * a.ldz;
  T* dz = (T*)a.dz + row * a.V;
  if (!SAME) {  // element by element (8192 rows of 50257 bf16, 50304 apart: 762 us; next to each other 253)
    const LpRowGrad r(a, row);
    const int64_t end = min(a.V, (blockIdx.y + 1) * share * E);
    for (int64_t i = blockIdx.y * share * E + threadIdx.x; i < end; i += G)
      dz[i] = from_f32<T>(r.with_token(r.one(to_f32(z[i])), i));
    return;
  }
  const int off = (int)(((uintptr_t)dz & 15) / sizeof(T));
  const int64_t lo = off ? 1 : 0, hi = max(lo, (a.V + off) / E);
  const int64_t from = min(hi, lo + blockIdx.y * share), to = min(hi, from + share);
  const int n = (int)max((int64_t)0, (to - from - threadIdx.x + G - 1) / G);
  const int64_t first = (from + threadIdx.x) * E - off;
  Ring<G, 2> chunks;
  chunks.template begin<G * 16>(ring, z + first, n);
  const LpRowGrad r(a, row);
  // the chunk with the token, if it is this thread's
  int token_at = -1;
  const int64_t rel = r.t >= 0 ? (r.t + off) / E - from - threadIdx.x : -1;
  if (rel >= 0 && rel % G == 0 && rel / G < n) token_at = (int)(rel / G);
  const uint64_t l = pair_of(kLog2e, kLog2e), m2 = pair_of(-r.m, -r.m), logs2 = pair_of(r.logs2, r.logs2),
                 slope = pair_of(r.slope, r.slope), rest = pair_of(r.rest, r.rest);
  T* out = dz + first;
  chunks.template walk<G * 16>(n, [&](int i, const RawVec<16>* raw, auto count) {
#pragma unroll
    for (int c = 0; c < decltype(count)::value; ++c) {
      float v[E];
      unpack_vec<E, T>(raw[c], v);
#pragma unroll
      for (int j = 0; j < E; j += 2) {
        const float2 lp = numbers(fma2(add2(pair_of(v[j], v[j + 1]), m2), l, logs2));
        const uint64_t w = fma2(pair_of(fmaxf(lp.x, -300.f), fmaxf(lp.y, -300.f)), slope, rest);
        const float2 d = numbers(mul2(pair_of(exp2_of(lp.x), exp2_of(lp.y)), w));
        v[j] = d.x;
        v[j + 1] = d.y;
      }
      T* to = out + (int64_t)(i + c) * (G * E);
      if (r.empty || i + c == token_at) {
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = r.with_token(v[j], (to - dz) + j);
      }
      if constexpr (sizeof(T) == 4) {
        store_vec<4>(to, v);
      } else {
        uint4 q;
        q.x = pack2<T>(v[0], v[1]);
        q.y = pack2<T>(v[2], v[3]);
        q.z = pack2<T>(v[4], v[5]);
        q.w = pack2<T>(v[6], v[7]);
        *reinterpret_cast<uint4*>(to) = q;
      }
    }
  });
  // the ends
  if (threadIdx.x < E) {
    const int64_t head = (int64_t)threadIdx.x - off, tail = hi * E - off + threadIdx.x;
    if (blockIdx.y == 0 && off && head >= 0 && head < a.V) dz[head] = from_f32<T>(r.with_token(r.one(to_f32(z[head])), head));
    if (blockIdx.y == gridDim.y - 1 && tail < a.V) dz[tail] = from_f32<T>(r.with_token(r.one(to_f32(z[tail])), tail));
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
  PVB2_CUDA_TRY(launch_over(kernel, dim3((unsigned)((a.N + Row::ROWS - 1) / Row::ROWS * cluster)), Row::THREADS, smem, s,
                            (unsigned)cluster, a, cluster));
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

template <typename T, bool TOP>
static int launch_lp(const LpArgs& a, cudaStream_t s) {
  const int64_t bytes = a.V * (int64_t)sizeof(T);
  if (a.N < num_sms()) {
    // fewer rows than SMs: more threads to a row, and several blocks, while there
    // are SMs for them and each keeps 16 KB
    if (bytes <= 1024) return launch_lp_as<T, TOP, 32>(a, 1, s);
    if (bytes <= 10240) return launch_lp_as<T, TOP, 128>(a, 1, s);
    int cluster = 1;
    while (cluster < kLpCluster && a.N * cluster * 2 <= num_sms() && bytes / (2 * cluster) >= 16384) cluster *= 2;
    return launch_lp_as<T, TOP, 256>(a, cluster, s);
  }
  // Short rows a warp's, since a block's joins take longer than the row; long ones
  // few threads' all the same, so that many rows begin and end at different
  // times (us for a warp, 128 and 256 threads, bf16: 16384 x 1000 18, 45, 84; 8192 x
  // 10000 35, 45, 68, with 20 alternatives 120, 80, 111; 4096 x 49999 79, 73, 82, with
  // 5 alternatives 165, 91, 104; 2048 x 131072 109, 92, 102, with 5 274, 115, 106).
  if (bytes <= (TOP ? 10240 : 20480)) return launch_lp_as<T, TOP, 32>(a, 1, s);
  if (bytes <= 160 * 1024) return launch_lp_as<T, TOP, 128>(a, 1, s);
  return launch_lp_as<T, TOP, 256>(a, 1, s);
}

template <typename T, bool SAME>
static int launch_lp_bwd_as(const LpBwdArgs& a, int64_t share, int64_t parts, cudaStream_t s) {
  constexpr int smem = kLpRing * kLpBwdThreads * 16;
  static DeviceOnce once;
  PVB2_TRY(allow_smem(logp_bwd_kernel<T, SAME>, smem, once));
  PVB2_CUDA_TRY(launch_over(logp_bwd_kernel<T, SAME>, dim3((unsigned)a.N, (unsigned)parts), kLpBwdThreads, SAME ? smem : 0,
                            s, 0, a, share));
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

template <typename T>
static int launch_lp_bwd(const LpBwdArgs& a, cudaStream_t s) {
  constexpr int E = LpChunk<T>::E;
  // parts of 32 chunks for each thread, fewer where the rows alone do not fill the SMs
  const int64_t chunks = (a.V + E - 1) / E;
  int64_t share = 32 * kLpBwdThreads;
  while (share > kLpBwdThreads && a.N * ((chunks + share - 1) / share) < 5 * (int64_t)num_sms()) share /= 2;
  const int64_t parts = std::min<int64_t>(65535, (chunks + share - 1) / share);
  share = (chunks + parts - 1) / parts;
  if (((uintptr_t)a.z & 15) == ((uintptr_t)a.dz & 15) && (a.N <= 1 || (a.ldz - a.V) * (int64_t)sizeof(T) % 16 == 0))
    return launch_lp_bwd_as<T, true>(a, share, parts, s);
  return launch_lp_bwd_as<T, false>(a, share, parts, s);
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
