// The norm of many gradients as one vector, and their scaling to it:
//   norm = (sum |g|^p)^(1/p), p = 1 or 2, or max |g|;   g *= min(1, max_norm / (norm + 1e-6))
//
// Bound by HBM: the gradients are read once for the norm and, where the norm
// is over the maximum, read and written once more.  One launch sums (each
// block a run of chunks, the block's sum to memory), the next adds the blocks'
// sums up, every block by itself and in one order, and scales, each block its
// run from the end.  Four blocks an SM: 353M bf16 gradients take 118 us for the
// norm and 353 us in all, 6.0 TB/s; with eight, whose runs are more streams for
// HBM to serve, 127 and 383.  (Chunks dealt out in turn had each looked up its
// tensor by bisection, which took longer than the chunk's loads: 148 us.)
//
// Sums are of eight squares in 32 bits and of those in 64.  Where eight
// squares leave fp32's normal numbers (magnitudes of 1e19, or of 1e-16 and
// less) they are formed in 64 bits.
#include <algorithm>
#include <vector>
#include "types.cuh"

namespace pvb2 {

constexpr int kClipMax = 512;     // tensors per launch
constexpr int kClipChunk = 8192;  // elements a block takes at a time; a quarter where the chunks are few

struct ClipPack {
  int n, total_chunks, chunk, run;  // run: chunks of a block
  void* g[kClipMax];
  int64_t numel[kClipMax];
  int chunk_prefix[kClipMax + 1];
};

enum { kNormMax = 0, kNorm1 = 1, kNorm2 = 2 };

__device__ __forceinline__ int clip_tensor(const ClipPack& pk, int chunk) {
  int lo = 0, hi = pk.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pk.chunk_prefix[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// a NaN wins
__device__ __forceinline__ double max_nan(double a, double b) { return a > b || a != a ? a : b; }

template <int P>
__device__ __forceinline__ double clip_join(double a, double b) {
  return P == kNormMax ? max_nan(a, b) : a + b;
}

// sum (or maximum) over the block, the same bits in every block that gives
// the same numbers
template <int P, int THREADS>
__device__ __forceinline__ double clip_block(double v) {
  __shared__ double line[THREADS / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) v = clip_join<P>(v, __shfl_xor_sync(~0u, v, o));
  if ((threadIdx.x & 31) == 0) line[threadIdx.x >> 5] = v;
  __syncthreads();
  v = line[0];
#pragma unroll
  for (int i = 1; i < THREADS / 32; ++i) v = clip_join<P>(v, line[i]);
  return v;
}

template <int P, int N>
__device__ __forceinline__ double clip_part(const float* v) {
  if constexpr (P == kNormMax) {
    uint32_t m = 0;  // magnitudes as integers: a NaN is above all
#pragma unroll
    for (int k = 0; k < N; ++k) m = max(m, __float_as_uint(v[k]) & 0x7fffffffu);
    return (double)__uint_as_float(m);
  } else if constexpr (P == kNorm1) {
    double d = 0;
#pragma unroll
    for (int k = 0; k < N; ++k) d += (double)fabsf(v[k]);
    return d;
  } else {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) s = fmaf(v[k], v[k], s);
    if (s >= 0x1p-100f && s <= 3e38f) return (double)s;
    double d = 0;
#pragma unroll
    for (int k = 0; k < N; ++k) d = fma((double)v[k], (double)v[k], d);
    return d;
  }
}

template <typename T, int P>
__global__ void __launch_bounds__(256) clip_sum_kernel(const __grid_constant__ ClipPack pk, double* sums) {
  constexpr int E = 16 / (int)sizeof(T);
  double acc = 0;
  const int c0 = blockIdx.x * pk.run, c1 = min(pk.total_chunks, c0 + pk.run);
  int t = c0 < c1 ? clip_tensor(pk, c0) : 0;
  for (int c = c0; c < c1; ++c) {
    while (c >= pk.chunk_prefix[t + 1]) ++t;
    const int64_t from = (int64_t)(c - pk.chunk_prefix[t]) * pk.chunk;
    const int n = (int)min((int64_t)pk.chunk, pk.numel[t] - from);
    const T* g = (const T*)pk.g[t] + from;
    if (((uintptr_t)g & 15) == 0) {
      const int full = n / E;
      int i = threadIdx.x;
      for (; i + 768 < full; i += 1024) {
        RawVec<16> raw[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) raw[u] = *reinterpret_cast<const RawVec<16>*>(g + (int64_t)(i + u * 256) * E);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float v[E];
          unpack_vec<E, T>(raw[u], v);
          acc = clip_join<P>(acc, clip_part<P, E>(v));
        }
      }
      for (; i < full; i += 256) {
        float v[E];
        load_vec<E>(g + (int64_t)i * E, v);
        acc = clip_join<P>(acc, clip_part<P, E>(v));
      }
      for (i = full * E + threadIdx.x; i < n; i += 256) {
        const float v = to_f32(g[i]);
        acc = clip_join<P>(acc, clip_part<P, 1>(&v));
      }
    } else {
      for (int i = threadIdx.x; i < n; i += 256) {
        const float v = to_f32(g[i]);
        acc = clip_join<P>(acc, clip_part<P, 1>(&v));
      }
    }
  }
  acc = clip_block<P, 256>(acc);
  if (threadIdx.x == 0) sums[blockIdx.x] = acc;
}

// `count` sums of all launches before; *norm is written where asked for
template <typename T, int P>
__global__ void __launch_bounds__(256) clip_scale_kernel(const __grid_constant__ ClipPack pk, const double* sums, int count,
                                                         float max_norm, int scale, float* norm) {
  constexpr int E = 16 / (int)sizeof(T);
  double total = 0;
  for (int i = threadIdx.x; i < count; i += 256) total = clip_join<P>(total, sums[i]);
  total = clip_block<P, 256>(total);
  const float nrm = (float)(P == kNorm2 ? sqrt(total) : total);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = nrm;
  if (!scale) return;
  const float coef = __fdiv_rn(max_norm, __fadd_rn(nrm, 1e-6f));
  if (coef >= 1.f) return;  // (a NaN is not, and goes to every gradient)
  const int c0 = blockIdx.x * pk.run, c1 = min(pk.total_chunks, c0 + pk.run);
  int t = c0 < c1 ? clip_tensor(pk, c1 - 1) : 0;
  for (int c = c1 - 1; c >= c0; --c) {
    while (c < pk.chunk_prefix[t]) --t;
    const int64_t from = (int64_t)(c - pk.chunk_prefix[t]) * pk.chunk;
    const int n = (int)min((int64_t)pk.chunk, pk.numel[t] - from);
    T* g = (T*)pk.g[t] + from;
    if (((uintptr_t)g & 15) == 0) {
      const int full = n / E;
      int i = threadIdx.x;
      for (; i + 768 < full; i += 1024) {
        RawVec<16> raw[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) raw[u] = *reinterpret_cast<const RawVec<16>*>(g + (int64_t)(i + u * 256) * E);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float v[E];
          unpack_vec<E, T>(raw[u], v);
#pragma unroll
          for (int k = 0; k < E; ++k) v[k] *= coef;
          store_vec<E>(g + (int64_t)(i + u * 256) * E, v);
        }
      }
      for (; i < full; i += 256) {
        float v[E];
        load_vec<E>(g + (int64_t)i * E, v);
#pragma unroll
        for (int k = 0; k < E; ++k) v[k] *= coef;
        store_vec<E>(g + (int64_t)i * E, v);
      }
      for (i = full * E + threadIdx.x; i < n; i += 256) g[i] = from_f32<T>(to_f32(g[i]) * coef);
    } else {
      for (int i = threadIdx.x; i < n; i += 256) g[i] = from_f32<T>(to_f32(g[i]) * coef);
    }
  }
}

// --------------------------------------------------------------- host side
static int clip_most_blocks() { return num_sms() * 4; }
static int clip_run_of(int chunks) { return std::max(1, (chunks + clip_most_blocks() - 1) / clip_most_blocks()); }
static int clip_blocks(int chunks) { return std::max(1, (chunks + clip_run_of(chunks) - 1) / clip_run_of(chunks)); }

// the launches' packs, of one type each, in the tensors' order within a type
static int clip_packs(int n, const pvb2_grad* ts, std::vector<ClipPack>& packs, std::vector<int>& dtypes) {
  int64_t total = 0;
  for (int i = 0; i < n; ++i) total += ts[i].numel;
  const int chunk = total / kClipChunk < 4 * (int64_t)num_sms() ? kClipChunk / 4 : kClipChunk;
  for (int dtype : {(int)PVB2_F32, (int)PVB2_BF16, (int)PVB2_F16}) {
    ClipPack* pk = nullptr;
    for (int i = 0; i < n; ++i) {
      if (ts[i].dtype != dtype || ts[i].numel == 0) continue;
      if (!pk || pk->n == kClipMax) {
        packs.emplace_back();
        dtypes.push_back(dtype);
        pk = &packs.back();
        pk->n = 0;
        pk->chunk = chunk;
        pk->chunk_prefix[0] = 0;
      }
      const int64_t end = pk->chunk_prefix[pk->n] + (ts[i].numel + chunk - 1) / chunk;
      PVB2_CHECK_ARG(end <= INT32_MAX / 2, "clip_grad_norm: too many elements in one call");
      pk->g[pk->n] = ts[i].data;
      pk->numel[pk->n] = ts[i].numel;
      pk->chunk_prefix[++pk->n] = (int)end;
      pk->total_chunks = (int)end;
    }
  }
  for (ClipPack& pk : packs) pk.run = clip_run_of(pk.total_chunks);
  return PVB2_OK;
}

static int clip_check(int n, const pvb2_grad* ts) {
  PVB2_CHECK_ARG(n >= 0 && (n == 0 || ts), "clip_grad_norm: no tensors");
  std::vector<std::pair<uintptr_t, uintptr_t>> spans;
  for (int i = 0; i < n; ++i) {
    PVB2_CHECK_ARG(ts[i].dtype == PVB2_F32 || ts[i].dtype == PVB2_F16 || ts[i].dtype == PVB2_BF16,
                   "clip_grad_norm: gradients are fp32, fp16 or bf16 (%d has dtype %d)", i, ts[i].dtype);
    PVB2_CHECK_ARG(ts[i].numel >= 0 && ts[i].numel < ((int64_t)1 << 40), "clip_grad_norm: gradient %d has %lld elements", i,
                   (long long)ts[i].numel);
    if (ts[i].numel == 0) continue;
    PVB2_CHECK_ARG(ts[i].data, "clip_grad_norm: gradient %d has a null pointer", i);
    PVB2_CHECK_ARG((uintptr_t)ts[i].data % dtype_size(ts[i].dtype) == 0, "clip_grad_norm: gradient %d is not aligned", i);
    const uintptr_t at = (uintptr_t)ts[i].data;
    spans.push_back({at, at + (uintptr_t)ts[i].numel * dtype_size(ts[i].dtype)});
  }
  // what two blocks scale at once would be scaled twice or once
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    PVB2_CHECK_ARG(spans[i - 1].second <= spans[i].first, "clip_grad_norm: a gradient is listed twice, or two overlap");
  return PVB2_OK;
}

template <typename T>
static void launch_sum(const ClipPack& pk, int kind, int grid, double* sums, cudaStream_t s) {
  if (kind == kNorm2) clip_sum_kernel<T, kNorm2><<<grid, 256, 0, s>>>(pk, sums);
  else if (kind == kNorm1) clip_sum_kernel<T, kNorm1><<<grid, 256, 0, s>>>(pk, sums);
  else clip_sum_kernel<T, kNormMax><<<grid, 256, 0, s>>>(pk, sums);
}

template <typename T>
static void launch_scale(const ClipPack& pk, int kind, int grid, const double* sums, int count, float most, int scale,
                         float* norm, cudaStream_t s) {
  if (kind == kNorm2) clip_scale_kernel<T, kNorm2><<<grid, 256, 0, s>>>(pk, sums, count, most, scale, norm);
  else if (kind == kNorm1) clip_scale_kernel<T, kNorm1><<<grid, 256, 0, s>>>(pk, sums, count, most, scale, norm);
  else clip_scale_kernel<T, kNormMax><<<grid, 256, 0, s>>>(pk, sums, count, most, scale, norm);
}

static int clip_run(int n, const pvb2_grad* tensors, int norm_type, int scale, double max_norm, float* norm, void* workspace,
                    size_t workspace_bytes, pvb2_stream stream) {
  PVB2_CHECK_ARG(norm_type == kNorm1 || norm_type == kNorm2 || norm_type == kNormMax,
                 "clip_grad_norm: norms are 1, 2 or the maximum (0), got %d", norm_type);
  PVB2_CHECK_ARG(!scale || max_norm >= 0, "clip_grad_norm: max_norm is below 0");
  PVB2_TRY(clip_check(n, tensors));
  PVB2_CHECK_ARG(norm, "clip_grad_norm: null pointer");
  std::vector<ClipPack> packs;
  std::vector<int> dtypes;
  PVB2_TRY(clip_packs(n, tensors, packs, dtypes));
  cudaStream_t s = as_stream(stream);
  if (packs.empty()) {
    PVB2_CUDA_TRY(cudaMemsetAsync(norm, 0, sizeof(float), s));
    return PVB2_OK;
  }
  int count = 0;
  for (const ClipPack& pk : packs) count += clip_blocks(pk.total_chunks);
  PVB2_CHECK_ARG(workspace && ((uintptr_t)workspace & 7) == 0 && workspace_bytes >= count * sizeof(double),
                 "clip_grad_norm: workspace of %zu bytes (8-byte aligned) needed", count * sizeof(double));
  double* sums = (double*)workspace;
  int at = 0;
  for (size_t i = 0; i < packs.size(); ++i) {
    const int grid = clip_blocks(packs[i].total_chunks);
    if (dtypes[i] == PVB2_F32) launch_sum<float>(packs[i], norm_type, grid, sums + at, s);
    else if (dtypes[i] == PVB2_BF16) launch_sum<__nv_bfloat16>(packs[i], norm_type, grid, sums + at, s);
    else launch_sum<__half>(packs[i], norm_type, grid, sums + at, s);
    PVB2_LAUNCH_CHECK();
    at += grid;
  }
  // the first of them writes the norm; where nothing is scaled, one block of it
  for (size_t i = 0; i < (scale ? packs.size() : 1); ++i) {
    const int grid = scale ? clip_blocks(packs[i].total_chunks) : 1;
    float* out = i == 0 ? norm : nullptr;
    const float most = (float)max_norm;
    if (dtypes[i] == PVB2_F32) launch_scale<float>(packs[i], norm_type, grid, sums, count, most, scale, out, s);
    else if (dtypes[i] == PVB2_BF16) launch_scale<__nv_bfloat16>(packs[i], norm_type, grid, sums, count, most, scale, out, s);
    else launch_scale<__half>(packs[i], norm_type, grid, sums, count, most, scale, out, s);
    PVB2_LAUNCH_CHECK();
  }
  return PVB2_OK;
}

}  // namespace pvb2

using namespace pvb2;

extern "C" {

size_t pvb2_clip_grad_norm_workspace_size(int n) {
  // a launch for every kClipMax tensors, and one more for each further type
  return n > 0 ? (size_t)(n / kClipMax + 3) * clip_most_blocks() * sizeof(double) : 0;
}

int pvb2_clip_grad_norm(int n, const pvb2_grad* tensors, int norm_type, int scale, double max_norm, float* norm,
                        void* workspace, size_t workspace_bytes, pvb2_stream stream) {
  try {
    return clip_run(n, tensors, norm_type, scale, max_norm, norm, workspace, workspace_bytes, stream);
  } catch (const std::bad_alloc&) {
    return fail(PVB2_ERR_OOM, "clip_grad_norm: out of host memory");
  }
}

}  // extern "C"
