// Root-mean-square norm of rows, with the residual's addition before it and
// 8-bit codes with scales after it, its gradients, and the codes of plain rows
// and weights.
//
//   h = x + r, rounded to the type (the residual stream as it goes on)
//   rstd = 1 / sqrt(mean(h^2) + eps);   n = h rstd;   y = n w
//   backward, with a = gy w:  dh = rstd (a - n mean(a n)) + gh;   dw = sum over rows of gy n
//
// One pass over the data: a row's elements stay in the registers of the
// threads that share it (a warp up to 128 chunks, a block beyond) between the sum
// and the output.  Rows of more than 4096 chunks (32768 16-bit elements, 16384 in
// fp32 or in the chunks of four below; backward half as many) are read twice, the
// second time out of L2.  Large forward passes are bound by HBM (8192 x 4096 bf16
// with a residual 6.4 TB/s); the others are by what a block does in turn: load, meet,
// store (codes of 2047 x 5000 19 us for 11 us of bytes, backward 55 for 41).
//
// The mean of squares is summed in 64 bits and rounded once, root and quotient
// are the IEEE ones, and n and y are rounded products: a code of the 8-bit
// output changes where y moves across the border of two codes, so that y must
// not depend on the order of a sum.  (The conversions to 64 bits cost nothing
// beside the loads: a square is converted for 4 to 8 bytes of traffic.)
//
// Elements go to threads in chunks of 16 bytes where rows begin on 16-byte
// boundaries, else in chunks of four that lie 32 elements apart, so that a warp
// still reads consecutive ones and 128 of them, a group of one scale, are a
// warp's.  16-bit rows of 2048 or more elements whose operands all begin alike
// between the boundaries (an odd length) take the chunks of memory, with a
// row's first and last element by element: steps of 4000 x 5001 bf16 100 us
// against 127 with chunks of four, 9760 x 2049 116 against 159, 3001 x 10001 fp16
// 132 against 228; but 13012 x 1537 114 against 114, 19512 x 1025 146 against 126.
#include <algorithm>
#include <atomic>
#include <initializer_list>
#include "overlap.cuh"
#include "quant8.cuh"

namespace pvb2 {

enum { kNorm = 0, kNorm8 = 1, kQuant8 = 2 };

struct NormArgs {
  const void* x;
  const void* r;   // residual, or null
  const void* w;   // or null: ones
  void* y;         // kNorm
  void* sum;       // with a residual
  float* rstd;     // or null
  uint8_t* codes;  // kNorm8, kQuant8
  float* scales;
  int64_t rows, ldx, ldr, ldc;
  int D, groups;
  float eps;
  double per_element;  // 1 / D
};

struct NormBwdArgs {
  const void* h;
  const void* w;
  const float* rstd;
  const void* gy;
  const void* gh;   // or null
  void* dx;         // or null
  float* partial;   // [blocks][D], or null
  int64_t rows, ldh, ldg, ldgh;
  int D;
};

enum { kApart = 0, kWhole = 1, kShifted = 2 };  // chunks: see above

// E elements of a chunk
template <typename T, int VEC>
struct Chunk {
  static constexpr int E = VEC ? 16 / (int)sizeof(T) : 4;
  // first element of chunk c, and the step to the next; `off`: where in its
  // 16 bytes a shifted row begins
  static __device__ __forceinline__ int64_t at(int c, int off) {
    return VEC ? (int64_t)c * E - off : (int64_t)(c >> 5) * 128 + (c & 31);
  }
  static constexpr int kStep = VEC ? 1 : 32;

  T e[E];
  __device__ __forceinline__ void load_each(const T* row, int c, int D, int off) {
    const int64_t i = at(c, off);
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const int64_t j = i + k * kStep;
      e[k] = j < D && (VEC != kShifted || j >= 0) ? row[j] : from_f32<T>(0.f);
    }
  }
  __device__ __forceinline__ void load(const T* row, int c, int D, int off) {
    const int64_t i = at(c, off);
    if (VEC == kWhole) {
      if (i < D) *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(row + i);
      else *reinterpret_cast<uint4*>(e) = make_uint4(0, 0, 0, 0);
    } else if (VEC == kShifted) {
      // (the ends by load_ends, once all other loads are on their way)
      uint4 v = make_uint4(0, 0, 0, 0);
      if (i >= 0 && i + E <= D) v = *reinterpret_cast<const uint4*>(row + i);
      *reinterpret_cast<uint4*>(e) = v;
    } else {
      load_each(row, c, D, off);
    }
  }
  __device__ __forceinline__ void load_ends(const T* row, int c, int D, int off) {
    if (VEC != kShifted) return;
    const int64_t i = at(c, off);
    if (i < D && (i < 0 || i + E > D)) load_each(row, c, D, off);
  }
  __device__ __forceinline__ void store(T* row, int c, int D, int off) const {
    const int64_t i = at(c, off);
    if (VEC == kWhole) {
      if (i < D) *reinterpret_cast<uint4*>(row + i) = *reinterpret_cast<const uint4*>(e);
    } else if (VEC == kShifted && i >= 0 && i + E <= D) {
      *reinterpret_cast<uint4*>(row + i) = *reinterpret_cast<const uint4*>(e);
    } else {
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const int64_t j = i + k * kStep;
        if (j < D && (VEC != kShifted || j >= 0)) row[j] = e[k];
      }
    }
  }
};
template <typename T, int VEC>
__device__ __forceinline__ int shift_of(const T* row) {
  return VEC == kShifted ? (int)(((uintptr_t)row & 15) / sizeof(T)) : 0;
}
// (16-byte accesses to its elements)
template <typename T, int VEC>
struct alignas(16) AChunk : Chunk<T, VEC> {};

// Sum over the threads of a row, a warp or a block, in a fixed order; all of
// them get it.  `line`: one number per warp, that nobody reads any more.
template <bool WARP, typename A>
__device__ __forceinline__ A row_sum(A v, A* line) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  if (!WARP) {
    const int warps = blockDim.x / 32;
    if ((threadIdx.x & 31) == 0) line[threadIdx.x >> 5] = v;
    __syncthreads();
    // (eight loads at once, where a loop would wait for each)
    A part[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) part[i] = i < warps ? line[i] : A(0);
    v = part[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) v += part[i];
    for (int i = 8; i < warps; ++i) v += line[i];
  }
  return v;
}

// SMALL: with an eps that is next to nothing the mean may lie beneath fp32's normal
// numbers; then by way of powers of two.  (Kernels of their own: in the others this
// took registers, 4000 x 5001 fp32 with a residual 55 us in place of 52.)
constexpr float kSmallEps = 0x1p-101f;
template <bool SMALL>
__device__ __forceinline__ float rstd_of(double squares, double per_element, float eps) {
  const double mean = squares * per_element;
  if (SMALL && mean < kSmallEps) return __fdiv_rn(0x1p99f, __fsqrt_rn((float)((mean + eps) * 0x1p198)));
  return __fdiv_rn(1.f, __fsqrt_rn(__fadd_rn((float)mean, eps)));
}

// elements [cE - off, cE - off + E) of what itself begins on a 16-byte boundary:
// the two chunks that hold them, moved together
template <typename T, int VEC>
__device__ __forceinline__ void load_beside(AChunk<T, VEC>& w, const T* p, int c, int D, int off) {
  constexpr int E = Chunk<T, VEC>::E;
  if ((int64_t)(c + 1) * E > D) {
    w.load_each(p, c, D, off);
    return;
  }
  alignas(16) uint32_t v[9] = {};
  if (c > 0) *reinterpret_cast<uint4*>(v) = *(reinterpret_cast<const uint4*>(p) + c - 1);
  *reinterpret_cast<uint4*>(v + 4) = *(reinterpret_cast<const uint4*>(p) + c);
  const int skip = 16 - off * (int)sizeof(T);  // bytes
#pragma unroll
  for (int step = 4; step; step >>= 1)
#pragma unroll
    for (int k = 0; k + step < 9; ++k) v[k] = skip >> 2 & step ? v[k + step] : v[k];
  uint32_t* to = reinterpret_cast<uint32_t*>(w.e);
#pragma unroll
  for (int k = 0; k < 4; ++k) to[k] = __funnelshift_r(v[k], v[k + 1], (skip & 3) * 8);
}
// the weight's numbers, or ones
template <typename T, int VEC>
__device__ __forceinline__ void load_weight(AChunk<T, VEC>& w, const void* p, int c, int D, int off) {
  if (p) {
    if (VEC == kShifted) load_beside(w, (const T*)p, c, D, off);
    else w.load((const T*)p, c, D, off);
  } else {
#pragma unroll
    for (int k = 0; k < Chunk<T, VEC>::E; ++k) w.e[k] = from_f32<T>(1.f);
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void scale_row(const AChunk<T, VEC>& h, const AChunk<T, VEC>& w, float rstd, float* y) {
#pragma unroll
  for (int k = 0; k < Chunk<T, VEC>::E; ++k) y[k] = __fmul_rn(__fmul_rn(to_f32(h.e[k]), rstd), to_f32(w.e[k]));
}

// the group's scale and this chunk's codes
template <typename T, int VEC>
__device__ __forceinline__ void put_codes(const float* y, uint8_t* row, float* scales, int c, int D) {
  static_assert(VEC != kShifted, "groups of a scale count from the row's beginning");
  constexpr int E = Chunk<T, VEC>::E;
  constexpr int kLanes = VEC ? kGroup8 / E : 32;  // that share a group
  const int64_t i = Chunk<T, VEC>::at(c, 0);
  uint32_t most = 0;
#pragma unroll
  for (int k = 0; k < E; ++k) most = max(most, abs_bits(y[k]));
#pragma unroll
  for (int o = kLanes / 2; o; o >>= 1) most = max(most, __shfl_xor_sync(~0u, most, o));
  const Scale8 s = scale8(most);
  const int64_t group = i / kGroup8;
  if ((c & (kLanes - 1)) == 0 && i < D) scales[group] = s.scale;
  float q[E];
#pragma unroll
  for (int k = 0; k < E; ++k) q[k] = __fmul_rn(y[k], s.inv);
  if (VEC) {
    if (i < D) {
      if (E == 8) {
        *reinterpret_cast<uint2*>(row + i) =
            make_uint2(codes4(q[0], q[1], q[2], q[3]), codes4(q[E - 4], q[E - 3], q[E - 2], q[E - 1]));
      } else {
        *reinterpret_cast<uint32_t*>(row + i) = codes4(q[0], q[1], q[2], q[3]);
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < E; ++k)
      if (i + 32 * k < D) row[i + 32 * k] = (uint8_t)codes2(q[k], 0.f);
  }
}

// h of a chunk: x, or x + r, which is stored
template <typename T, int VEC>
__device__ __forceinline__ void form_sum(const NormArgs& a, int64_t row, int c, int off, AChunk<T, VEC>& x,
                                         const AChunk<T, VEC>& r) {
  if (!a.r) return;
#pragma unroll
  for (int k = 0; k < Chunk<T, VEC>::E; ++k) x.e[k] = from_f32<T>(to_f32(x.e[k]) + to_f32(r.e[k]));
  x.store((T*)a.sum + row * a.D, c, a.D, off);
}

// A warp (WARP; blocks of four) or a block shares a row, each thread keeps NV
// chunks of it.
template <typename T, int VEC, bool WARP, int NV, int MODE, bool SMALL = false>
__global__ void __launch_bounds__(WARP ? 128 : 1024) norm_kernel(NormArgs a) {
  let_next_come();
  wait_for_last();
  using C = Chunk<T, VEC>;
  __shared__ double line[32];
  const int G = WARP ? 32 : (int)blockDim.x, t = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int64_t row = WARP ? (int64_t)blockIdx.x * 4 + threadIdx.x / 32 : blockIdx.x;
  if (row >= a.rows) return;  // whole warps: only where a warp has a row of its own
  const int off = shift_of<T, VEC>((const T*)a.x + row * a.ldx);
  AChunk<T, VEC> h[NV];
  {
    AChunk<T, VEC> r[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) h[i].load((const T*)a.x + row * a.ldx, i * G + t, a.D, off);
    if (a.r) {
#pragma unroll
      for (int i = 0; i < NV; ++i) r[i].load((const T*)a.r + row * a.ldr, i * G + t, a.D, off);
    }
    if (VEC == kShifted) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        h[i].load_ends((const T*)a.x + row * a.ldx, i * G + t, a.D, off);
        if (a.r) r[i].load_ends((const T*)a.r + row * a.ldr, i * G + t, a.D, off);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) form_sum(a, row, i * G + t, off, h[i], r[i]);
  }
  float rstd = 1.f;
  if constexpr (MODE != kQuant8) {
    double q = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < C::E; ++k) {
        const double v = to_f32(h[i].e[k]);
        q = fma(v, v, q);
      }
    rstd = rstd_of<SMALL>(row_sum<WARP>(q, line), a.per_element, a.eps);
    if (a.rstd && t == 0) a.rstd[row] = rstd;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = i * G + t;
    float y[C::E];
    if constexpr (MODE == kQuant8) {
#pragma unroll
      for (int k = 0; k < C::E; ++k) y[k] = to_f32(h[i].e[k]);
    } else {
      AChunk<T, VEC> w;
      load_weight(w, a.w, c, a.D, off);
      scale_row(h[i], w, rstd, y);
    }
    if constexpr (MODE == kNorm) {
      AChunk<T, VEC> out;
#pragma unroll
      for (int k = 0; k < C::E; ++k) out.e[k] = from_f32<T>(y[k]);
      out.store((T*)a.y + row * a.D, c, a.D, off);
    } else {
      put_codes<T, VEC>(y, a.codes + row * a.ldc, a.scales + row * a.groups, c, a.D);
    }
  }
}

// rows that outgrow the registers: read again for the output
template <typename T, int VEC, int MODE, bool SMALL = false>
__global__ void __launch_bounds__(1024) norm_long_kernel(NormArgs a) {
  let_next_come();
  wait_for_last();
  using C = Chunk<T, VEC>;
  __shared__ double line[32];
  const int64_t row = blockIdx.x;
  // whole warps stay together: a group's lanes meet
  const int chunks = (a.D + C::E * 32 - 1) / (C::E * 32) * 32;
  float rstd = 1.f;
  if constexpr (MODE != kQuant8) {
    double q = 0;
    for (int c = threadIdx.x; c < chunks; c += 1024) {
      AChunk<T, VEC> h, r;
      h.load((const T*)a.x + row * a.ldx, c, a.D, 0);
      if (a.r) r.load((const T*)a.r + row * a.ldr, c, a.D, 0);
      form_sum(a, row, c, 0, h, r);
#pragma unroll
      for (int k = 0; k < C::E; ++k) {
        const double v = to_f32(h.e[k]);
        q = fma(v, v, q);
      }
    }
    rstd = rstd_of<SMALL>(row_sum<false>(q, line), a.per_element, a.eps);
    if (a.rstd && threadIdx.x == 0) a.rstd[row] = rstd;
  }
  // the sum that this thread wrote, or x
  const T* src = a.r ? (const T*)a.sum + row * a.D : (const T*)a.x + row * a.ldx;
  for (int c = threadIdx.x; c < chunks; c += 1024) {
    AChunk<T, VEC> h;
    h.load(src, c, a.D, 0);
    float y[C::E];
    if constexpr (MODE == kQuant8) {
#pragma unroll
      for (int k = 0; k < C::E; ++k) y[k] = to_f32(h.e[k]);
    } else {
      AChunk<T, VEC> w;
      load_weight(w, a.w, c, a.D, 0);
      scale_row(h, w, rstd, y);
    }
    if constexpr (MODE == kNorm) {
      AChunk<T, VEC> out;
#pragma unroll
      for (int k = 0; k < C::E; ++k) out.e[k] = from_f32<T>(y[k]);
      out.store((T*)a.y + row * a.D, c, a.D, 0);
    } else {
      put_codes<T, VEC>(y, a.codes + row * a.ldc, a.scales + row * a.groups, c, a.D);
    }
  }
}

// ------------------------------------------------------------- backward
// A block walks rows and keeps its share of dw in registers: gy and h are read
// once for both gradients.  The blocks' shares are summed by a second launch,
// in a fixed order.
// MOST: 32 for a warp to a row, else the most threads of a row.
template <typename T, int VEC, int MOST, int NV>
__global__ void __launch_bounds__(MOST < 128 ? 128 : MOST, (sizeof(T) == 4 || MOST == 1024 ? 1024 : 768) /
                                                               (MOST < 128 ? 128 : MOST)) norm_bwd_kernel(NormBwdArgs a) {
  let_next_come();
  wait_for_last();
  using C = Chunk<T, VEC>;
  constexpr int kRows = MOST == 32 ? 4 : 1;  // of a block
  const int G = MOST == 32 ? 32 : blockDim.x;
  __shared__ float line[2][32];
  extern __shared__ float share[];  // kRows > 1: dw of the rows' warps
  const int t = MOST == 32 ? threadIdx.x % 32 : threadIdx.x, mine = MOST == 32 ? threadIdx.x / 32 : 0;
  static_assert(VEC != kShifted || kRows == 1, "a warp's row is too short to be shifted");
  // (all rows of a block begin alike: the host sees to it)
  const int off = shift_of<T, VEC>((const T*)a.h + (int64_t)blockIdx.x * a.ldh);
  AChunk<T, VEC> w[NV];
  float dw[NV][C::E];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    load_weight(w[i], a.w, i * G + t, a.D, off);
#pragma unroll
    for (int k = 0; k < C::E; ++k) dw[i][k] = 0.f;
  }
  int parity = 0;
  for (int64_t row = (int64_t)blockIdx.x * kRows + mine; row < a.rows; row += (int64_t)gridDim.x * kRows, parity ^= 1) {
    AChunk<T, VEC> h[NV], g[NV], gh[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      h[i].load((const T*)a.h + row * a.ldh, i * G + t, a.D, off);
      g[i].load((const T*)a.gy + row * a.ldg, i * G + t, a.D, off);
      if (a.gh) gh[i].load((const T*)a.gh + row * a.ldgh, i * G + t, a.D, off);
    }
    if (VEC == kShifted) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        h[i].load_ends((const T*)a.h + row * a.ldh, i * G + t, a.D, off);
        g[i].load_ends((const T*)a.gy + row * a.ldg, i * G + t, a.D, off);
        if (a.gh) gh[i].load_ends((const T*)a.gh + row * a.ldgh, i * G + t, a.D, off);
      }
    }
    const float rstd = a.rstd[row];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < C::E; ++k) {
        const float n = to_f32(h[i].e[k]) * rstd, gv = to_f32(g[i].e[k]);
        dot = fmaf(gv * to_f32(w[i].e[k]), n, dot);
        dw[i][k] = fmaf(gv, n, dw[i][k]);
      }
    if (!a.dx) continue;
    const float mean = row_sum<MOST == 32>(dot, line[parity]) / (float)a.D;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      AChunk<T, VEC> out;
#pragma unroll
      for (int k = 0; k < C::E; ++k) {
        const float n = to_f32(h[i].e[k]) * rstd;
        float d = fmaf(-n, mean, to_f32(g[i].e[k]) * to_f32(w[i].e[k])) * rstd;
        if (a.gh) d += to_f32(gh[i].e[k]);
        out.e[k] = from_f32<T>(d);
      }
      out.store((T*)a.dx + row * a.D, i * G + t, a.D, off);
    }
  }
  if (!a.partial) return;
  if (kRows > 1) {
    // (NV * 32 * E numbers for each row's warp)
    constexpr int kWide = NV * 32 * C::E;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < C::E; ++k) share[mine * kWide + (int)C::at(i * G + t, off) + k * C::kStep] = dw[i][k];
    __syncthreads();
    for (int j = threadIdx.x; j < a.D; j += 128) {
      float s = share[j];
#pragma unroll
      for (int m = 1; m < kRows; ++m) s += share[m * kWide + j];
      a.partial[(int64_t)blockIdx.x * a.D + j] = s;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < C::E; ++k) {
        const int64_t j = C::at(i * G + t, off) + k * C::kStep;
        if (j >= 0 && j < a.D) a.partial[(int64_t)blockIdx.x * a.D + j] = dw[i][k];
      }
  }
}

// long rows: dh alone, and the shares of dw by columns
template <typename T, int VEC>
__global__ void __launch_bounds__(1024) norm_bwd_long_kernel(NormBwdArgs a) {
  let_next_come();
  wait_for_last();
  using C = Chunk<T, VEC>;
  __shared__ float line[32];
  const int64_t row = blockIdx.x;
  const int chunks = (a.D + C::E * 32 - 1) / (C::E * 32) * 32;
  const float rstd = a.rstd[row];
  float dot = 0.f, mean = 0.f;
  for (int pass = 0; pass < 2; ++pass) {
    for (int c = threadIdx.x; c < chunks; c += 1024) {
      AChunk<T, VEC> h, g, w, gh, out;
      h.load((const T*)a.h + row * a.ldh, c, a.D, 0);
      g.load((const T*)a.gy + row * a.ldg, c, a.D, 0);
      if (a.w) w.load((const T*)a.w, c, a.D, 0);
      if (pass && a.gh) gh.load((const T*)a.gh + row * a.ldgh, c, a.D, 0);
#pragma unroll
      for (int k = 0; k < C::E; ++k) {
        const float n = to_f32(h.e[k]) * rstd, v = to_f32(g.e[k]) * (a.w ? to_f32(w.e[k]) : 1.f);
        if (!pass) {
          dot = fmaf(v, n, dot);
        } else {
          float d = fmaf(-n, mean, v) * rstd;
          if (a.gh) d += to_f32(gh.e[k]);
          out.e[k] = from_f32<T>(d);
        }
      }
      if (pass) out.store((T*)a.dx + row * a.D, c, a.D, 0);
    }
    if (!pass) mean = row_sum<false>(dot, line) / (float)a.D;
  }
}

// rows blockIdx.y, blockIdx.y + gridDim.y, ... of 256 columns
template <typename T>
__global__ void __launch_bounds__(256) norm_dw_columns_kernel(NormBwdArgs a) {
  let_next_come();
  wait_for_last();
  const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (j >= a.D) return;
  float s = 0.f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y)
    s = fmaf(to_f32(((const T*)a.gy)[row * a.ldg + j]), to_f32(((const T*)a.h)[row * a.ldh + j]) * a.rstd[row], s);
  a.partial[(int64_t)blockIdx.y * a.D + j] = s;
}

// dw[j] = sum of the shares, eight columns a block (a sector of each share), in
// a fixed order: a thread every 128th, then the threads of a column
template <typename T>
__global__ void __launch_bounds__(1024) norm_dw_sum_kernel(const float* partial, int count, int D, T* dw) {
  let_next_come();
  wait_for_last();
  __shared__ float part[8][129];
  const int x = threadIdx.x & 7, y = threadIdx.x >> 3;
  const int64_t j = (int64_t)blockIdx.x * 8 + x;
  float s = 0.f;
  if (j < D) {
    int p = y;
    for (; p + 3 * 128 < count; p += 4 * 128) {
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = partial[(int64_t)(p + 128 * i) * D + j];
#pragma unroll
      for (int i = 0; i < 4; ++i) s += v[i];
    }
    for (; p < count; p += 128) s += partial[(int64_t)p * D + j];
  }
  part[x][y] = s;
  __syncthreads();
  if (threadIdx.x >= 256) return;
  const int c = threadIdx.x >> 5, lane = threadIdx.x & 31;
  s = (part[c][lane] + part[c][lane + 32]) + (part[c][lane + 64] + part[c][lane + 96]);
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  const int64_t jj = (int64_t)blockIdx.x * 8 + c;
  if (lane == 0 && jj < D) dw[jj] = from_f32<T>(s);
}

// ------------------------------------------- codes of weights, and values
// 128 x 128 elements with one scale; a warp reads 4 x 32 of a row at a time, an
// element a thread (4096 x 4096 bf16 26 us, 1.9 TB/s: weights, once)
template <typename T>
__global__ void __launch_bounds__(256) quant_tile_kernel(const T* x, int64_t rows, int64_t D, int64_t ldx, uint8_t* codes,
                                                         int64_t ldc, float* scales, int64_t groups) {
  let_next_come();
  wait_for_last();
  __shared__ uint32_t most_of[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t r0 = (int64_t)blockIdx.y * 128, c0 = (int64_t)blockIdx.x * 128;
  float v[16][4];
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t r = r0 + i * 8 + warp, c = c0 + k * 32 + lane;
      v[i][k] = r < rows && c < D ? to_f32(x[r * ldx + c]) : 0.f;
      most = max(most, abs_bits(v[i][k]));
    }
  most = __reduce_max_sync(~0u, most);
  if (lane == 0) most_of[warp] = most;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max(most, most_of[i]);
  const Scale8 s = scale8(most);
  if (threadIdx.x == 0) scales[blockIdx.y * groups + blockIdx.x] = s.scale;
#pragma unroll
  for (int i = 0; i < 16; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t r = r0 + i * 8 + warp, c = c0 + k * 32 + lane;
      if (r < rows && c < D) codes[r * ldc + c] = (uint8_t)codes2(__fmul_rn(v[i][k], s.inv), 0.f);
    }
}

// values of codes: 16 bytes of values a thread (VEC), or one; blockIdx.x: part of
// a row, blockIdx.y: which rows
template <typename T, int VEC>
__global__ void __launch_bounds__(256) dequant_kernel(const uint8_t* codes, const float* scales, T* out, int64_t rows, int D,
                                                      int64_t ldc, int groups, int tall) {
  let_next_come();
  wait_for_last();
  constexpr int E = VEC ? 16 / (int)sizeof(T) : 1;
  const int c = (blockIdx.x * 256 + threadIdx.x) * E;
  if (c >= D) return;
  constexpr int R = 4;  // rows at a time
  for (int64_t row0 = (int64_t)blockIdx.y * R; row0 < rows; row0 += (int64_t)gridDim.y * R) {
    uint2 q[R];
    float s[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = min(row0 + r, rows - 1);
      s[r] = scales[(tall ? row / 128 : row) * groups + c / kGroup8];
      const uint8_t* from = codes + row * ldc + c;
      if (E == 8) q[r] = *reinterpret_cast<const uint2*>(from);
      else if (E == 4) q[r].x = *reinterpret_cast<const uint32_t*>(from);
      else q[r].x = *from;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (row0 + r >= rows) break;
      T* to = out + (row0 + r) * D + c;
      if constexpr (VEC) {
        float v[E];
#pragma unroll
        for (int k = 0; k < E / 2; ++k) {
          const float2 p = values2((k < 2 ? q[r].x : q[r].y) >> (16 * (k & 1)));
          v[2 * k] = p.x * s[r];
          v[2 * k + 1] = p.y * s[r];
        }
        store_vec<E>(to, v);
      } else {
        *to = from_f32<T>(values2(q[r].x).x * s[r]);
      }
    }
  }
}

// --------------------------------------------------------------- host side
static bool on16(const void* p, int64_t ld, int size, int64_t rows) {
  return ((uintptr_t)p & 15) == 0 && (rows <= 1 || ld * size % 16 == 0);
}

constexpr int64_t kNormMostRows = (int64_t)1 << 31;

static int norm_check(const char* op, const pvb2_rms_norm_desc* d) {
  PVB2_CHECK_ARG(d, "%s: no descriptor", op);
  PVB2_CHECK_ARG(d->dtype == PVB2_F32 || d->dtype == PVB2_F16 || d->dtype == PVB2_BF16,
                 "%s: fp32, fp16 or bf16 expected (got dtype %d)", op, d->dtype);
  PVB2_CHECK_ARG(d->rows >= 0 && d->rows < kNormMostRows && d->D >= 0 && d->D <= (1 << 24), "%s: %lld rows of %lld out of range",
                 op, (long long)d->rows, (long long)d->D);
  PVB2_CHECK_ARG(d->eps >= 0 && d->eps <= 3e38, "%s: eps has to be finite and not below 0", op);
  return PVB2_OK;
}

static int norm_strides(const char* op, const pvb2_rms_norm_desc* d, std::initializer_list<int64_t> lds) {
  for (int64_t ld : lds)
    PVB2_CHECK_ARG(d->rows <= 1 || ld >= d->D, "%s: row strides below the rows' length", op);
  return PVB2_OK;
}

// resident blocks of a kernel on an SM, asked for once
template <typename K>
static int resident(K kernel, int threads, int smem, std::atomic<int>& known) {
  int n = known.load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = 1;
    }
    known.store(n, std::memory_order_relaxed);
  }
  return n;
}

// chunks of a row, however it is shifted
static int chunks_of(int64_t D, int E, int vec) { return (int)((D + (vec == kShifted ? E - 1 : 0) + E - 1) / E); }

template <typename T, int VEC, int MODE>
static int launch_norm(const NormArgs& a, cudaStream_t s) {
  const int chunks = chunks_of(a.D, Chunk<T, VEC>::E, VEC);
  const unsigned rows = (unsigned)a.rows, fours = (unsigned)((a.rows + 3) / 4);
  // A warp to a row that its lanes hold in four chunks each, since it needs no
  // barrier; else a block, with four chunks a thread as well: each thread takes a
  // root and a quotient for its row (8192 x 4096 bf16 with a residual: 41 us; in
  // two chunks 47, a warp to the row with 16 chunks a lane 73).  Few rows have
  // more threads, for the first chunk to be the only one.
  const bool few = a.rows < num_sms();
  const unsigned one = (unsigned)((chunks + 31) / 32 * 32), four = (unsigned)((chunks + 127) / 128 * 32);
  constexpr int kLong = VEC == kWhole ? kWhole : kApart;
  if constexpr (MODE != kQuant8) {
    if (a.eps < kSmallEps) {  // (fewer kinds: next to nobody asks for it)
      if (chunks <= 4096) PVB2_CUDA_TRY(launch_over(norm_kernel<T, VEC, false, 4, MODE, true>, rows, four, 0, s, 0, a));
      else PVB2_CUDA_TRY(launch_over(norm_long_kernel<T, kLong, MODE, true>, rows, 1024, 0, s, 0, a));
      PVB2_LAUNCH_CHECK();
      return PVB2_OK;
    }
  }
  if constexpr (VEC != kShifted) {  // (which has 257 or more)
    if (chunks <= 128 && (chunks <= 32 || !few)) {
      if (chunks <= 32) PVB2_CUDA_TRY(launch_over(norm_kernel<T, VEC, true, 1, MODE>, fours, 128, 0, s, 0, a));
      else if (chunks <= 64) PVB2_CUDA_TRY(launch_over(norm_kernel<T, VEC, true, 2, MODE>, fours, 128, 0, s, 0, a));
      else PVB2_CUDA_TRY(launch_over(norm_kernel<T, VEC, true, 4, MODE>, fours, 128, 0, s, 0, a));
      PVB2_LAUNCH_CHECK();
      return PVB2_OK;
    }
  }
  if (chunks <= 1024 && few) PVB2_CUDA_TRY(launch_over(norm_kernel<T, VEC, false, 1, MODE>, rows, one, 0, s, 0, a));
  else if (chunks <= 4096) PVB2_CUDA_TRY(launch_over(norm_kernel<T, VEC, false, 4, MODE>, rows, four, 0, s, 0, a));
  else PVB2_CUDA_TRY(launch_over(norm_long_kernel<T, kLong, MODE>, rows, 1024, 0, s, 0, a));
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

template <typename T, int MODE>
static int run_norm_as(const NormArgs& a, int vec, cudaStream_t s) {
  if (vec == kWhole) return launch_norm<T, kWhole, MODE>(a, s);
  if constexpr (MODE == kNorm)
    if constexpr (sizeof(T) == 2)
      if (vec == kShifted) return launch_norm<T, kShifted, MODE>(a, s);
  return launch_norm<T, kApart, MODE>(a, s);
}
template <int MODE>
static int run_norm(const NormArgs& a, int dtype, int vec, cudaStream_t s) {
  if (dtype == PVB2_F32) return run_norm_as<float, MODE>(a, vec, s);
  if (dtype == PVB2_BF16) return run_norm_as<__nv_bfloat16, MODE>(a, vec, s);
  return run_norm_as<__half, MODE>(a, vec, s);
}

static NormArgs norm_args(const pvb2_rms_norm_desc* d, const void* x, const void* r, const void* w, void* sum) {
  NormArgs a = {};
  a.x = x;
  a.r = r;
  a.w = w;
  a.sum = sum;
  a.rows = d->rows;
  a.ldx = d->ldx;
  a.ldr = d->ldr;
  a.ldc = d->ldc;
  a.D = (int)d->D;
  a.groups = (int)((d->D + kGroup8 - 1) / kGroup8);
  a.eps = (float)d->eps;
  a.per_element = 1.0 / (double)d->D;
  return a;
}

// an operand of the rows: its address and row stride
struct RowsAt {
  const void* p;
  int64_t ld;
};
// how its rows lie: on 16-byte boundaries, or all operands' alike off them, or neither
static int rows_lie(int64_t rows, int64_t D, int size, std::initializer_list<RowsAt> all, const void* weight) {
  const int E = 16 / size;
  bool whole = D % E == 0 && ((uintptr_t)weight & 15) == 0, alike = true;
  const RowsAt* first = nullptr;
  for (const RowsAt& r : all) {
    if (!r.p) continue;
    if (!first) first = &r;
    whole = whole && on16(r.p, r.ld, size, rows);
    alike = alike && ((uintptr_t)r.p & 15) == ((uintptr_t)first->p & 15) && (rows <= 1 || (r.ld - first->ld) % E == 0);
  }
  if (whole) return kWhole;
  return size == 2 && D >= 2048 && alike && ((uintptr_t)weight & 15) == 0 ? kShifted : kApart;
}
static int norm_vec(const NormArgs& a, int dtype) {
  const int size = dtype_size(dtype);
  const int lie = rows_lie(a.rows, a.D, size, {{a.x, a.ldx}, {a.r, a.ldr}, {a.y, a.D}, {a.sum, a.D}}, a.w);
  if (!a.codes) return lie;
  return lie == kWhole && ((uintptr_t)a.codes & 7) == 0 && (a.rows <= 1 || a.ldc % 8 == 0) ? kWhole : kApart;
}

// Blocks of the backward pass, each of which keeps a share of dw: as many as the
// workspace is for, and no more than are resident (a second wave of a few blocks
// would take as long as the first).
// A row has the warps that hold it in two chunks a thread (a step of 4000 x 5000
// bf16 82 us; rounded up to a power of two 92).
struct NormBwdPlan {
  int threads, rows_per_block;  // threads of a row (0: long rows)
  int64_t blocks;
};
static NormBwdPlan bwd_plan(const pvb2_rms_norm_desc* d, int vec) {
  const int size = dtype_size(d->dtype);
  const int chunks = chunks_of(d->D, vec ? 16 / size : 4, vec);
  NormBwdPlan p = {};
  p.threads = chunks <= 64 ? 32 : chunks <= 128 ? (chunks + 31) / 32 * 32 : chunks <= 2048 ? (chunks + 63) / 64 * 32 : 0;
  p.rows_per_block = p.threads == 32 ? 4 : 1;
  const int64_t most = (int64_t)num_sms() * (p.threads == 0 ? 1 : std::min(8, 1024 / p.threads));
  const int64_t want = (d->rows + p.rows_per_block - 1) / p.rows_per_block;
  p.blocks = std::max<int64_t>(1, std::min(want, most));
  return p;
}

template <typename T, int VEC, int MOST, int NV>
static int launch_bwd_as(const NormBwdArgs& a, NormBwdPlan& p, cudaStream_t s) {
  const int threads = MOST == 32 ? 128 : p.threads, smem = MOST == 32 ? 4 * NV * 32 * Chunk<T, VEC>::E * 4 : 0;
  static std::atomic<int> known[33];  // by warps
  auto kernel = norm_bwd_kernel<T, VEC, MOST, NV>;
  p.blocks = std::min<int64_t>(p.blocks, (int64_t)num_sms() * resident(kernel, threads, smem, known[threads / 32]));
  // (the rows of a block begin alike where they lie a multiple of E rows apart)
  constexpr int E = Chunk<T, VEC>::E;
  if (VEC == kShifted && p.blocks < a.rows) p.blocks = p.blocks / E * E;
  PVB2_CUDA_TRY(launch_over(kernel, (unsigned)p.blocks, threads, smem, s, 0, a));
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

template <typename T, int VEC>
static int launch_bwd(const NormBwdArgs& a, NormBwdPlan& p, cudaStream_t s) {
  const int chunks = chunks_of(a.D, Chunk<T, VEC>::E, VEC);
  if constexpr (VEC != kShifted) {  // (which has 257 or more)
    if (chunks <= 32) return launch_bwd_as<T, VEC, 32, 1>(a, p, s);
    if (chunks <= 64) return launch_bwd_as<T, VEC, 32, 2>(a, p, s);
    if (chunks <= 128) return launch_bwd_as<T, VEC, 128, 1>(a, p, s);
    if (chunks <= 256) return launch_bwd_as<T, VEC, 128, 2>(a, p, s);
  }
  if (chunks <= 512) return launch_bwd_as<T, VEC, 256, 2>(a, p, s);
  if (chunks <= 768) return launch_bwd_as<T, VEC, 384, 2>(a, p, s);
  if (chunks <= 1024) return launch_bwd_as<T, VEC, 512, 2>(a, p, s);
  if (chunks <= 2048) return launch_bwd_as<T, VEC, 1024, 2>(a, p, s);
  if (a.dx) {
    constexpr int kVec = VEC == kWhole ? kWhole : kApart;
    PVB2_CUDA_TRY(launch_over(norm_bwd_long_kernel<T, kVec>, (unsigned)a.rows, 1024, 0, s, 0, a));
    PVB2_LAUNCH_CHECK();
  }
  if (!a.partial) return PVB2_OK;
  const dim3 columns((unsigned)((a.D + 255) / 256), (unsigned)p.blocks);
  PVB2_CUDA_TRY(launch_over(norm_dw_columns_kernel<T>, columns, 256, 0, s, 0, a));
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

template <typename T>
static int run_bwd(const NormBwdArgs& a, NormBwdPlan p, int vec, void* dw, cudaStream_t s) {
  if (a.rows) {
    if (vec == kWhole) PVB2_TRY((launch_bwd<T, kWhole>(a, p, s)));
    else if constexpr (sizeof(T) == 2) {
      if (vec == kShifted) PVB2_TRY((launch_bwd<T, kShifted>(a, p, s)));
      else PVB2_TRY((launch_bwd<T, kApart>(a, p, s)));
    } else PVB2_TRY((launch_bwd<T, kApart>(a, p, s)));
  }
  if (!dw) return PVB2_OK;
  PVB2_CUDA_TRY(launch_over(norm_dw_sum_kernel<T>, (unsigned)((a.D + 7) / 8), 1024, 0, s, 0,
                            a.partial, a.rows ? (int)p.blocks : 0, a.D, (T*)dw));
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

}  // namespace pvb2

using namespace pvb2;

extern "C" {

int pvb2_rms_norm_fwd(const pvb2_rms_norm_desc* d, const void* x, const void* residual, const void* weight, void* y,
                      void* sum, float* rstd, pvb2_stream stream) {
  PVB2_TRY(norm_check("rms_norm", d));
  if (d->rows == 0 || d->D == 0) return PVB2_OK;
  PVB2_CHECK_ARG(x && y && (!residual || sum), "rms_norm: null pointer");
  PVB2_TRY(norm_strides("rms_norm", d, {d->ldx, residual ? d->ldr : d->D}));
  NormArgs a = norm_args(d, x, residual, weight, residual ? sum : nullptr);
  a.y = y;
  a.rstd = rstd;
  return run_norm<kNorm>(a, d->dtype, norm_vec(a, d->dtype), as_stream(stream));
}

int pvb2_rms_norm_8bit(const pvb2_rms_norm_desc* d, const void* x, const void* residual, const void* weight,
                       uint8_t* codes, float* scales, void* sum, pvb2_stream stream) {
  PVB2_TRY(norm_check("rms_norm_8bit", d));
  if (d->rows == 0 || d->D == 0) return PVB2_OK;
  PVB2_CHECK_ARG(x && codes && scales && (!residual || sum), "rms_norm_8bit: null pointer");
  PVB2_TRY(norm_strides("rms_norm_8bit", d, {d->ldx, residual ? d->ldr : d->D, d->ldc}));
  NormArgs a = norm_args(d, x, residual, weight, residual ? sum : nullptr);
  a.codes = codes;
  a.scales = scales;
  return run_norm<kNorm8>(a, d->dtype, norm_vec(a, d->dtype), as_stream(stream));
}

size_t pvb2_rms_norm_bwd_workspace_size(const pvb2_rms_norm_desc* d) {
  if (norm_check("rms_norm", d) != PVB2_OK) return 0;
  // (how the rows lie is not known here)
  int64_t blocks = 0;
  for (int vec : {(int)kApart, (int)kWhole, (int)kShifted}) blocks = std::max(blocks, bwd_plan(d, vec).blocks);
  return (size_t)blocks * d->D * 4;
}

int pvb2_rms_norm_bwd(const pvb2_rms_norm_desc* d, const void* h, const void* weight, const float* rstd, const void* gy,
                      const void* gsum, void* dx, void* dw, void* workspace, size_t workspace_bytes, pvb2_stream stream) {
  PVB2_TRY(norm_check("rms_norm_bwd", d));
  if (d->D == 0 || (!dx && !dw) || (d->rows == 0 && !dw)) return PVB2_OK;
  if (d->rows) {
    PVB2_CHECK_ARG(h && rstd && gy, "rms_norm_bwd: null pointer");
    PVB2_TRY(norm_strides("rms_norm_bwd", d, {d->ldx, d->ldg, gsum ? d->ldr : d->D}));
  }
  PVB2_CHECK_ARG(!dw || (workspace && ((uintptr_t)workspace & 3) == 0 &&
                         workspace_bytes >= pvb2_rms_norm_bwd_workspace_size(d)),
                 "rms_norm_bwd: workspace of %zu bytes needed", pvb2_rms_norm_bwd_workspace_size(d));
  NormBwdArgs a = {};
  a.h = h;
  a.w = weight;
  a.rstd = rstd;
  a.gy = gy;
  a.gh = gsum;
  a.dx = dx;
  a.partial = dw ? (float*)workspace : nullptr;
  a.rows = d->rows;
  a.ldh = d->ldx;
  a.ldg = d->ldg;
  a.ldgh = d->ldr;
  a.D = (int)d->D;
  const int vec = rows_lie(a.rows, a.D, dtype_size(d->dtype), {{h, a.ldh}, {gy, a.ldg}, {gsum, a.ldgh}, {dx, a.D}}, weight);
  const NormBwdPlan p = bwd_plan(d, vec);
  cudaStream_t s = as_stream(stream);
  if (d->dtype == PVB2_F32) return run_bwd<float>(a, p, vec, dw, s);
  if (d->dtype == PVB2_BF16) return run_bwd<__nv_bfloat16>(a, p, vec, dw, s);
  return run_bwd<__half>(a, p, vec, dw, s);
}

int pvb2_quantize_8bit(int dtype, int64_t rows, int64_t D, const void* x, int64_t ldx, int tall, uint8_t* codes,
                       int64_t ldc, float* scales, pvb2_stream stream) {
  pvb2_rms_norm_desc d = {};
  d.rows = rows;
  d.D = D;
  d.ldx = ldx;
  d.ldc = ldc;
  d.dtype = dtype;
  PVB2_TRY(norm_check("quantize_8bit", &d));
  if (rows == 0 || D == 0) return PVB2_OK;
  PVB2_CHECK_ARG(x && codes && scales, "quantize_8bit: null pointer");
  PVB2_TRY(norm_strides("quantize_8bit", &d, {ldx, ldc}));
  cudaStream_t s = as_stream(stream);
  if (!tall) {
    NormArgs a = norm_args(&d, x, nullptr, nullptr, nullptr);
    a.codes = codes;
    a.scales = scales;
    return run_norm<kQuant8>(a, dtype, norm_vec(a, dtype), s);
  }
  const int64_t groups = (D + 127) / 128, blocks = (rows + 127) / 128;
  PVB2_CHECK_ARG(blocks <= 65535, "quantize_8bit: more than %d rows in blocks of 128", 65535 * 128);
  const dim3 grid((unsigned)groups, (unsigned)blocks);
  if (dtype == PVB2_F32)
    PVB2_CUDA_TRY(launch_over(quant_tile_kernel<float>, grid, 256, 0, s, 0,
                              (const float*)x, rows, D, ldx, codes, ldc, scales, groups));
  else if (dtype == PVB2_BF16)
    PVB2_CUDA_TRY(launch_over(quant_tile_kernel<__nv_bfloat16>, grid, 256, 0, s, 0,
                              (const __nv_bfloat16*)x, rows, D, ldx, codes, ldc, scales, groups));
  else PVB2_CUDA_TRY(launch_over(quant_tile_kernel<__half>, grid, 256, 0, s, 0,
                                 (const __half*)x, rows, D, ldx, codes, ldc, scales, groups));
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

int pvb2_dequantize_8bit(int64_t rows, int64_t D, const uint8_t* codes, int64_t ldc, const float* scales, int tall,
                         int dtype, void* out, pvb2_stream stream) {
  pvb2_rms_norm_desc d = {};
  d.rows = rows;
  d.D = D;
  d.dtype = dtype;
  PVB2_TRY(norm_check("dequantize_8bit", &d));
  if (rows == 0 || D == 0) return PVB2_OK;
  PVB2_CHECK_ARG(codes && scales && out, "dequantize_8bit: null pointer");
  PVB2_TRY(norm_strides("dequantize_8bit", &d, {ldc}));
  const int groups = (int)((D + 127) / 128), size = dtype_size(dtype);
  const bool vec = D % 8 == 0 && ((uintptr_t)codes & 7) == 0 && (rows <= 1 || ldc % 8 == 0) && ((uintptr_t)out & 15) == 0 &&
                   D * size % 16 == 0;
  cudaStream_t s = as_stream(stream);
  const unsigned wide = (unsigned)((D / (vec ? 16 / size : 1) + 255) / 256);
  const dim3 grid(wide, (unsigned)std::min<int64_t>(65535, (rows + 3) / 4));
  auto go = [&](auto* p) -> int {
    using T = std::remove_pointer_t<decltype(p)>;
    if (vec) PVB2_CUDA_TRY(launch_over(dequant_kernel<T, true>, grid, 256, 0, s, 0,
                                       codes, scales, p, rows, (int)D, ldc, groups, tall));
    else PVB2_CUDA_TRY(launch_over(dequant_kernel<T, false>, grid, 256, 0, s, 0,
                                   codes, scales, p, rows, (int)D, ldc, groups, tall));
    PVB2_LAUNCH_CHECK();
    return PVB2_OK;
  };
  if (dtype == PVB2_F32) return go((float*)out);
  if (dtype == PVB2_BF16) return go((__nv_bfloat16*)out);
  return go((__half*)out);
}

}  // extern "C"
