// Learned relative position bias: a value per head and bucket of the distance
// r = j - i - q_offset, spread over the scores, and its gradient.
//
// A bucket is an interval of r (the buckets grow with the logarithm of the
// distance), so the host hands the kernels each bucket's first and last r and
// no kernel takes a logarithm.  Both directions are bound by HBM: the forward
// pass writes H Lq Lk elements, the backward pass reads as many.
//
// Forward: a block writes R rows x 1024 columns of one head.  All it needs is
// the value of each of the R + 1023 diagonals that it crosses, which it lays
// out in shared memory in 16 / sizeof(T) copies, copy s shifted by s elements:
// whatever the row's shift and the row's alignment in memory, each 16-byte
// store then takes one aligned 16-byte load from the copy that fits.
//
// Backward: a block owns 248 diagonals and walks down the rows of one head; at
// the end it adds those of each bucket in order.  16 bytes of a row begin on a
// boundary, and the row below it is shifted by an element against the
// diagonals; but 8 rows further the boundary is at the same diagonals again,
// whatever the row stride.  So a warp takes every eighth row, 256 elements from
// the boundary before its first diagonal, and its lanes' 16-byte loads meet the
// same 8 diagonals in each: their sums stay in registers, and nothing is staged
// or shifted.  Loads at a row's ends reach into what lies beside it, as far as
// the gradient itself reaches, and the foreign elements are set to 0 (16 x 4096
// x 4096 bf16: 109 us; 158 with slanted strips staged in shared memory, from
// which threads read their diagonals' two bytes; 142 where loads at the ends
// were guarded one by one; 118 with 504 diagonals a block, which meet more ends).
// Sums are fp32 over at most 64 rows and fp64 beyond; nothing is added in an
// order that depends on timing.
#include <math.h>
#include <vector>
#include "types.cuh"

namespace pvb2 {

constexpr int kRelMaxBuckets = 512;
constexpr int kRelCols = 1024;   // columns of a forward block
constexpr int kRelRows = 64;     // most rows of a block
constexpr int kRelDiag = 248;    // diagonals of a block in the backward pass
constexpr int kRelInf = 1 << 30;

struct RelMap {  // bucket b holds r in [lo[b], hi[b]] (empty where lo > hi)
  int nb;
  int lo[kRelMaxBuckets], hi[kRelMaxBuckets];
};

template <typename T>
__global__ void __launch_bounds__(256)
    rel_bias_fwd_kernel(const __grid_constant__ RelMap map, const T* __restrict__ table, T* __restrict__ out, int H,
                        int Lq, int Lk, int q_offset, int R, int row_tiles, int col_tiles) {
  constexpr int V = 16 / sizeof(T);  // elements of a 16-byte store
  constexpr int kLen = (kRelRows + kRelCols + 2 * V - 1) / V * V;
  __shared__ __align__(16) T sv[V][kLen];
  int tile = blockIdx.x;
  const int ct = tile % col_tiles;
  tile /= col_tiles;
  const int rt = tile % row_tiles, h = tile / row_tiles;
  const int i0 = rt * R, j0 = ct * kRelCols;
  const int rows = min(R, Lq - i0), cols = min(kRelCols, Lk - j0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // entry e: the diagonal j - i = first + e; row i, column j of the tile is
  // entry (j - j0) + (rows - 1 - (i - i0))
  const int first = j0 - (i0 + rows - 1), len = rows + cols - 1;
  const int r0 = first - q_offset;
  for (int b = warp; b < map.nb; b += 8) {
    const int lo = max(map.lo[b], r0), hi = min(map.hi[b], r0 + len - 1);
    if (lo > hi) continue;
    const T x = table[(int64_t)b * H + h];
    for (int r = lo + lane; r <= hi; r += 32) {
      const int e = r - r0;
#pragma unroll
      for (int s = 0; s < V; ++s)
        if (e >= s) sv[s][e - s] = x;
    }
  }
  __syncthreads();
  for (int i = warp; i < rows; i += 8) {
    T* row = out + ((int64_t)h * Lq + i0 + i) * Lk + j0;
    const int shift = rows - 1 - i;
    // columns before the first 16-byte boundary of the row
    const int head = min(cols, (int)(((16 - ((uintptr_t)row & 15)) & 15) / sizeof(T)));
    if (lane < head) row[lane] = sv[0][shift + lane];
    const int e0 = shift + head, s = e0 % V;
    const int vecs = (cols - head) / V;
    const uint4* src = reinterpret_cast<const uint4*>(&sv[s][e0 - s]);
    uint4* dst = reinterpret_cast<uint4*>(row + head);
    for (int q = lane; q < vecs; q += 32) dst[q] = src[q];
    const int done = head + vecs * V;
    if (lane < cols - done) row[done + lane] = sv[0][shift + done + lane];
  }
}

// grid: (segments of the rows) x (tiles of diagonals) x (B * H); part:
// [B*H][nb][tiles][segments].  FLAT: unit stride along the keys; `low` is the
// gradient's first element and `high` the last address from which 16 bytes lie
// within it.
template <typename T, bool FLAT>
__global__ void __launch_bounds__(256, 3)
    rel_bias_bwd_kernel(const __grid_constant__ RelMap map, const T* __restrict__ grad, int64_t sb, int64_t sh,
                        int64_t si, int64_t sj, double* __restrict__ part, int H, int Lq, int Lk, int q_offset,
                        int per, const T* low, const T* high) {
  constexpr int V = 16 / sizeof(T);  // elements of a 16-byte load
  constexpr int M = 8 / V;           // loads of a row, 256 elements for a warp
  constexpr int U = 8 / M;           // rows in flight
  __shared__ double sums[FLAT ? 8 : 1][FLAT ? kRelDiag : 1], diag[kRelDiag];
  const int seg = blockIdx.x, tile = blockIdx.y;
  const int64_t z = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int d0 = tile * kRelDiag - (Lq - 1);  // first diagonal j - i
  const int parts = gridDim.y * gridDim.x;
  double* p = part + z * map.nb * parts + tile * gridDim.x + seg;  // of bucket 0
  // of the rows that these diagonals meet `per`
  const int ra = max(0, -(d0 + kRelDiag - 1)), rb = min(Lq, Lk - d0);
  const int i0 = ra + seg * per, i1 = min(rb, i0 + per);
  if (i0 >= i1) {
    for (int b = threadIdx.x; b < map.nb; b += 256) p[(int64_t)b * parts] = 0.0;
    return;
  }
  const T* g = grad + ((int)blockIdx.z / H) * sb + ((int)blockIdx.z % H) * sh;

  if (FLAT) {
    const int first = i0 + warp;
    // elements from the 16-byte boundary to the first diagonal: the same in every eighth row
    const int lead = (int)(((uintptr_t)(g + (int64_t)first * si + d0 + first) & 15) / sizeof(T));
    for (int e = lane; e < kRelDiag; e += 32) sums[warp][e] = 0.0;
    __syncwarp();
    float s[M][V];
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int j = 0; j < V; ++j) s[m][j] = 0.f;
    int held = 0;
    const int64_t step = 8 * (si + 1);
    // only the first and the last rows of all can meet an end
    const bool ends = g + (int64_t)i0 * si < low + V || g + (int64_t)(i1 - 1) * si + Lk > high;
    auto flush = [&]() {
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int e = (m * 32 + lane) * V + j - lead;
          if (e >= 0 && e < kRelDiag) sums[warp][e] += (double)s[m][j];
          s[m][j] = 0.f;
        }
      held = 0;
    };
    for (int i = first; i < i1; i += 8 * U) {
      uint4 v[U][M];
      const int c0 = d0 + i - lead + lane * V;  // column of load m of row u: c0 + 8 u + 32 V m
      const T* at0 = g + (int64_t)i * si + c0;
      held += U;
      if (d0 + i >= lead && d0 + i + 8 * (U - 1) - lead + 32 * V * M <= Lk && i + 8 * (U - 1) < i1) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int m = 0; m < M; ++m) v[u][m] = *reinterpret_cast<const uint4*>(at0 + u * step + 32 * V * m);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int m = 0; m < M; ++m) {
            float x[V];
            unpack_vec<V, T>(RawVec<16>{v[u][m]}, x);
#pragma unroll
            for (int j = 0; j < V; ++j) s[m][j] += x[j];
          }
        if (held == 64) flush();
        continue;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int m = 0; m < M; ++m) {
          const int c = c0 + 8 * u + 32 * V * m;
          const T* at = at0 + u * step + 32 * V * m;
          v[u][m] = make_uint4(0u, 0u, 0u, 0u);
          if (i + 8 * u < i1 && c > -V && c < Lk && at >= low && at <= high) v[u][m] = *reinterpret_cast<const uint4*>(at);
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int m = 0; m < M; ++m) {
          const int c = c0 + 8 * u + 32 * V * m;
          float x[V];
          unpack_vec<V, T>(RawVec<16>{v[u][m]}, x);
          if (c < 0 || c + V > Lk) {  // what lies beside the row
#pragma unroll
            for (int j = 0; j < V; ++j) x[j] = c + j >= 0 && c + j < Lk ? x[j] : 0.f;
          }
#pragma unroll
          for (int j = 0; j < V; ++j) s[m][j] += x[j];
        }
      if (ends) {  // loads that would reach beyond the whole gradient
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int m = 0; m < M; ++m) {
            const int c = c0 + 8 * u + 32 * V * m;
            const T* at = at0 + u * step + 32 * V * m;
            if (i + 8 * u < i1 && c > -V && c < Lk && !(at >= low && at <= high)) {
#pragma unroll
              for (int j = 0; j < V; ++j)
                if (c + j >= 0 && c + j < Lk) s[m][j] += to_f32(at[j]);
            }
          }
      }
      if (held == 64) flush();
    }
    flush();
    __syncthreads();
    for (int e = threadIdx.x; e < kRelDiag; e += 256) {
      double t = 0.0;
#pragma unroll
      for (int w = 0; w < 8; ++w) t += sums[w][e];
      diag[e] = t;
    }
  } else {
    for (int e = threadIdx.x; e < kRelDiag; e += 256) {
      double t = 0.0;
      for (int i = i0; i < i1; i += 64) {
        float s = 0.f;
#pragma unroll 4
        for (int q = i; q < min(i1, i + 64); ++q) {
          const int c = d0 + q + e;
          if (c >= 0 && c < Lk) s += to_f32(g[(int64_t)q * si + (int64_t)c * sj]);
        }
        t += (double)s;
      }
      diag[e] = t;
    }
  }
  __syncthreads();
  const int r0 = d0 - q_offset;
  for (int b = warp; b < map.nb; b += 8) {
    const int lo = max(map.lo[b], r0), hi = min(map.hi[b], r0 + kRelDiag - 1);
    if (lo > hi) {
      if (lane == 0) p[(int64_t)b * parts] = 0.0;
      continue;
    }
    double s = 0.0;
    for (int r = lo + lane; r <= hi; r += 32) s += diag[r - r0];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) p[(int64_t)b * parts] = s;
  }
}

// one warp per (bucket, head)
template <typename T>
__global__ void rel_bias_sum_kernel(const double* __restrict__ part, T* __restrict__ dtable, int nb, int H, int B,
                                    int per_z) {
  const int w = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, lane = threadIdx.x & 31;
  if (w >= nb * H) return;
  const int b = w / H, h = w % H;
  double s = 0.0;
#pragma unroll 8
  for (uint32_t q = lane; q < (uint32_t)(B * per_z); q += 32) {
    const uint32_t at = q / (uint32_t)per_z;  // of the batch
    s += part[((int64_t)(at * H + h) * nb + b) * per_z + (q - at * per_z)];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) dtable[w] = from_f32<T>((float)s);
}

// --------------------------------------------------------------- host side
// the buckets' intervals; a distance on a border (equal to the power that
// begins a bucket) belongs to the bucket that it begins: the slack of 1e-9 is
// far above the error of the logarithms and, up to a distance of 2^20, below
// the step from one distance to the next
static void rel_map(const pvb2_relative_bias_desc* d, RelMap* m) {
  const int n = d->bidirectional ? d->num_buckets / 2 : d->num_buckets, e = n / 2;
  std::vector<int> first(n + 1);  // smallest distance of each of the n buckets of one side
  for (int b = 0; b <= e; ++b) first[b] = b;
  const double span = std::log((double)d->max_distance / e);
  auto step = [&](int64_t x) { return (int64_t)std::floor(std::log((double)x / e) / span * (n - e) + 1e-9); };
  for (int b = e + 1; b < n; ++b) {
    int64_t x = std::max<int64_t>(e, (int64_t)(e * std::exp(span * (b - e) / (n - e))));
    while (x > e && step(x - 1) >= b - e) --x;
    while (step(x) < b - e) ++x;
    first[b] = (int)x;
  }
  first[n] = kRelInf;
  m->nb = d->num_buckets;
  for (int b = 0; b < m->nb; ++b) m->lo[b] = 1, m->hi[b] = 0;
  for (int b = 0; b < n; ++b) {
    const int a = first[b], z = first[b + 1] - 1;
    if (a > z) continue;
    m->lo[b] = -z;
    m->hi[b] = (!d->bidirectional && a == 0) ? kRelInf : -a;
    if (d->bidirectional && z >= 1) {
      m->lo[n + b] = std::max(a, 1);
      m->hi[n + b] = z;
    }
  }
}

static int rel_check(const pvb2_relative_bias_desc* d) {
  PVB2_CHECK_ARG(d, "relative bias: no descriptor");
  PVB2_CHECK_ARG(d->dtype == PVB2_F32 || d->dtype == PVB2_F16 || d->dtype == PVB2_BF16,
                 "relative bias: fp32, fp16 or bf16 expected (got dtype %d)", d->dtype);
  PVB2_CHECK_ARG(d->num_buckets >= 2 && d->num_buckets <= kRelMaxBuckets, "relative bias: 2 to %d buckets (got %d)",
                 kRelMaxBuckets, d->num_buckets);
  PVB2_CHECK_ARG(!d->bidirectional || (d->num_buckets % 2 == 0 && d->num_buckets >= 4),
                 "relative bias: an even number of at least 4 buckets for both directions (got %d)", d->num_buckets);
  const int e = (d->bidirectional ? d->num_buckets / 2 : d->num_buckets) / 2;
  PVB2_CHECK_ARG(d->max_distance > e && d->max_distance <= (1 << 20),
                 "relative bias: max_distance above %d (a quarter or half of the buckets) and at most 2^20 (got %lld)", e,
                 (long long)d->max_distance);
  const int64_t most = 1 << 28;
  PVB2_CHECK_ARG(d->H >= 0 && d->H <= 65535 && d->Lq >= 0 && d->Lk >= 0 && d->Lq < most && d->Lk < most &&
                     d->q_offset > -most && d->q_offset < most,
                 "relative bias: heads, lengths or offset out of range");
  return PVB2_OK;
}

static int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
static int64_t up(int64_t a, int64_t b) { return cdiv(a, b) * b; }

// rows of a block: as many as keep four blocks for every SM (fewer rows, more
// blocks: a block's fixed work, the diagonals, is shared by its rows)
static int rel_rows(int64_t heads, int64_t Lq, int64_t across) {
  int R = kRelRows;
  while (R > 1 && heads * cdiv(Lq, R) * across < 4 * (int64_t)num_sms()) R /= 2;
  return R;
}

struct RelBwdPlan {
  int64_t tiles, segments;
  int per;  // rows of a segment
};

// Rows of a segment: as many as leave five blocks for every SM (16 x 4096 x 4096
// bf16: 118 us with three, 109 with five, 115 with twelve), at least 128 (12 x
// 197 x 4096: 19 us, 22 with 64).  Every row meets as many tiles as its columns
// take, and a tile at most Lk + 247 rows.
static RelBwdPlan rel_bwd_plan(const pvb2_relative_bias_desc* d, int64_t B) {
  RelBwdPlan p;
  p.tiles = cdiv(d->Lq + d->Lk - 1, kRelDiag);
  const double visits = (double)B * d->H * d->Lq * (1.0 + (double)d->Lk / kRelDiag);
  p.per = (int)std::max<int64_t>(128, up((int64_t)std::min<double>(1 << 28, visits / (5.0 * num_sms())), 32));
  p.segments = cdiv(std::min(d->Lq, d->Lk + kRelDiag - 1), p.per);
  return p;
}

template <typename T>
static int rel_fwd(const pvb2_relative_bias_desc* d, const RelMap& m, const void* table, void* out, cudaStream_t s) {
  const int64_t col_tiles = cdiv(d->Lk, kRelCols);
  const int R = rel_rows(d->H, d->Lq, col_tiles);
  const int64_t row_tiles = cdiv(d->Lq, R), blocks = d->H * row_tiles * col_tiles;
  PVB2_CHECK_ARG(blocks < INT32_MAX, "relative bias: too many elements");
  rel_bias_fwd_kernel<T><<<(int)blocks, 256, 0, s>>>(m, (const T*)table, (T*)out, d->H, (int)d->Lq, (int)d->Lk,
                                                     (int)d->q_offset, R, (int)row_tiles, (int)col_tiles);
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

template <typename T>
static int rel_bwd(const pvb2_relative_bias_desc* d, const RelMap& m, const pvb2_tensor* g, void* dtable, double* part,
                   cudaStream_t s) {
  const int64_t B = g->sizes[0];
  const RelBwdPlan p = rel_bwd_plan(d, B);
  int64_t per_z = 0;
  if (B > 0 && d->Lq > 0 && d->Lk > 0) {
    PVB2_CHECK_ARG(B * d->H <= 65535 && p.tiles <= 65535 && B * p.tiles * p.segments <= INT32_MAX,
                   "relative bias: batch x heads or lengths out of range");
    per_z = p.tiles * p.segments;
    int64_t extent = 1;
    for (int k = 0; k < 4; ++k) extent += (g->sizes[k] - 1) * g->strides[k];
    const dim3 grid((unsigned)p.segments, (unsigned)p.tiles, (unsigned)(B * d->H));
    auto kernel = g->strides[3] == 1 || d->Lk == 1 ? rel_bias_bwd_kernel<T, true> : rel_bias_bwd_kernel<T, false>;
    kernel<<<grid, 256, 0, s>>>(m, (const T*)g->data, g->strides[0], g->strides[1], g->strides[2], g->strides[3],
                                   part, d->H, (int)d->Lq, (int)d->Lk, (int)d->q_offset, p.per, (const T*)g->data,
                                 (const T*)g->data + extent - 16 / (int)sizeof(T));
    PVB2_LAUNCH_CHECK();
  }
  const int warps = m.nb * d->H;
  rel_bias_sum_kernel<T><<<(int)cdiv(warps, 8), 256, 0, s>>>(part, (T*)dtable, m.nb, d->H, (int)(per_z ? B : 0),
                                                             (int)std::max<int64_t>(per_z, 1));
  PVB2_LAUNCH_CHECK();
  return PVB2_OK;
}

}  // namespace pvb2

using namespace pvb2;

extern "C" {

int pvb2_relative_bias_fwd(const pvb2_relative_bias_desc* d, const void* table, void* out, pvb2_stream stream) {
  PVB2_TRY(rel_check(d));
  if (d->H == 0 || d->Lq == 0 || d->Lk == 0) return PVB2_OK;
  PVB2_CHECK_ARG(table && out, "relative bias: null pointer");
  RelMap m;
  rel_map(d, &m);
  cudaStream_t s = as_stream(stream);
  if (d->dtype == PVB2_F32) return rel_fwd<float>(d, m, table, out, s);
  if (d->dtype == PVB2_BF16) return rel_fwd<__nv_bfloat16>(d, m, table, out, s);
  return rel_fwd<__half>(d, m, table, out, s);
}

size_t pvb2_relative_bias_bwd_workspace_size(const pvb2_relative_bias_desc* d, int64_t B) {
  if (rel_check(d) != PVB2_OK || B <= 0 || d->Lq == 0 || d->Lk == 0) return 0;
  const RelBwdPlan p = rel_bwd_plan(d, B);
  return (size_t)(B * d->H * p.tiles * p.segments) * d->num_buckets * sizeof(double);
}

int pvb2_relative_bias_bwd(const pvb2_relative_bias_desc* d, const pvb2_tensor* grad, void* dtable, void* workspace,
                           size_t workspace_bytes, pvb2_stream stream) {
  PVB2_TRY(rel_check(d));
  PVB2_CHECK_ARG(grad && grad->ndim == 4 && grad->sizes[1] == d->H && grad->sizes[2] == d->Lq &&
                     grad->sizes[3] == d->Lk && grad->dtype == d->dtype,
                 "relative bias backward: grad [B, H, Lq, Lk] of the table's type expected");
  if (d->H == 0) return PVB2_OK;
  PVB2_CHECK_ARG(dtable && (grad->data || numel(grad) == 0), "relative bias backward: null pointer");
  const size_t need = pvb2_relative_bias_bwd_workspace_size(d, grad->sizes[0]);
  PVB2_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 7) == 0),
                 "relative bias backward: workspace of %zu bytes needed", need);
  RelMap m;
  rel_map(d, &m);
  cudaStream_t s = as_stream(stream);
  if (d->dtype == PVB2_F32) return rel_bwd<float>(d, m, grad, dtable, (double*)workspace, s);
  if (d->dtype == PVB2_BF16) return rel_bwd<__nv_bfloat16>(d, m, grad, dtable, (double*)workspace, s);
  return rel_bwd<__half>(d, m, grad, dtable, (double*)workspace, s);
}

}  // extern "C"
