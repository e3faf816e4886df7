// Global norm of many gradient tensors and their scaling (dance/modules/spatial/spatial_domain/stagate.py: clip_grad_norm_ between
// loss.backward() and optimizer.step()):
//
//   norm = (sum_t sum_i |g_t[i]|^p)^(1/p)  for p = 1, 2;   norm = max |g|  for p = inf (a NaN anywhere makes it NaN)
//   out_t[i] = g_t[i] * min(1, max_norm / (norm + 1e-6))
//
// Bound: HBM.  The scaling cannot start before the norm is known, so a set larger than the caches is read twice and written once: 328 million
// fp32 elements in 32 tensors 246 us (5.3 TB/s) and 518 us (5.1 TB/s).  The launches and their latencies for small ones: 2000 x 512, 512 x 30
// and their biases 9 us, 320 tensors of at most 200 x 64 30 us.
// Layout: the tensors' addresses travel as kernel arguments, 128 per launch (nothing is uploaded, so a captured call replays with the
// addresses it was recorded with); a launch walks its tensors in chunks of 16 KB of fp32, up to GRID workgroups (2 GRID for the scaling) striding over the chunks.
// Sums are double from the first product (the conversions and fp64 FMAs cost 2 of ~16 issue slots that a 16-byte load leaves) and are
// joined in a fixed order: the result does not depend on timing.  Every workgroup of the scaling launch joins the partial sums itself
// (<= 8 KB from the L2) instead of waiting for a launch of its own to do it.
#include "common.h"

namespace {

constexpr int MAX_T = 128;        // tensors per launch: 128 x (8 + 8 + 8 + 4) bytes of kernel arguments stay under 4 KB
constexpr int GRID = 1024;        // workgroups of a norm launch at most = its partial sums
constexpr int THREADS = 256;
constexpr int CHUNK = 4096;       // elements of one workgroup's pass over a chunk: 16 per thread
constexpr int INLINE_PARTIALS = 1024;  // up to here the scaling workgroups join the partial sums themselves

struct Table {
  const void* in[MAX_T];
  void* out[MAX_T];
  int64_t numel[MAX_T];
  uint32_t first[MAX_T];  // first chunk of tensor t among the launch's chunks
  uint32_t n_chunks;
  uint32_t in_bf16[MAX_T / 32], out_bf16[MAX_T / 32];
  int n;
};
static_assert(sizeof(Table) <= 4000, "kernel arguments");

// 16-byte accesses at the element's own alignment: views of a flat buffer start anywhere (global memory takes unaligned accesses)
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x8u __attribute__((ext_vector_type(8), aligned(2)));

__device__ __forceinline__ float bf16_f32(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ uint16_t f32_bf16(float x) {  // nearest even; NaN stays a quiet NaN
  const uint32_t u = __float_as_uint(x);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);
  return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}

__device__ __forceinline__ bool bit(const uint32_t* words, int t) { return (words[t >> 5] >> (t & 31)) & 1u; }

// tensor of chunk c: the last t with first[t] <= c (tensors without elements own no chunk and are never found: the host leaves them out)
__device__ __forceinline__ int tensor_of(const Table& tb, uint32_t c) {
  int lo = 0, hi = tb.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tb.first[mid] <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// sixteen consecutive-by-vector elements of a chunk per thread; count < CHUNK only in a tensor's last chunk
template <bool BF16>
__device__ __forceinline__ void load16(const void* base, int64_t at, int count, float (&v)[16]) {
  const int tid = threadIdx.x;
  if (count == CHUNK) {
    if (BF16) {
      const uint16_t* p = static_cast<const uint16_t*>(base) + at;
      u16x8u r[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) r[q] = *reinterpret_cast<const u16x8u*>(p + (q * THREADS + tid) * 8);
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[q * 8 + e] = bf16_f32(r[q][e]);
    } else {
      const float* p = static_cast<const float*>(base) + at;
      f32x4u r[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) r[q] = *reinterpret_cast<const f32x4u*>(p + (q * THREADS + tid) * 4);
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[q * 4 + e] = r[q][e];
    }
  } else {
#pragma unroll
    for (int q = 0; q < 16; ++q) {
      const int i = q * THREADS + tid, j = min(i, count - 1);  // clamped address instead of a guarded load: sixteen loads in flight
      const float t = BF16 ? bf16_f32(static_cast<const uint16_t*>(base)[at + j]) : static_cast<const float*>(base)[at + j];
      v[q] = i < count ? t : 0.f;
    }
  }
}

template <bool IN_BF16, bool OUT_BF16>
__device__ __forceinline__ void store16(void* base, int64_t at, int count, const float (&v)[16]) {
  const int tid = threadIdx.x;
  if (count == CHUNK) {
    // element of v[q * W + e] = (q * THREADS + tid) * W + e with W the input's vector width
    if (IN_BF16) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int i = (q * THREADS + tid) * 8;
        if (OUT_BF16) {
          u16x8u r;
#pragma unroll
          for (int e = 0; e < 8; ++e) r[e] = f32_bf16(v[q * 8 + e]);
          *reinterpret_cast<u16x8u*>(static_cast<uint16_t*>(base) + at + i) = r;
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            f32x4u r;
#pragma unroll
            for (int e = 0; e < 4; ++e) r[e] = v[q * 8 + h * 4 + e];
            *reinterpret_cast<f32x4u*>(static_cast<float*>(base) + at + i + h * 4) = r;
          }
        }
      }
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int i = (q * THREADS + tid) * 4;
        if (OUT_BF16) {
#pragma unroll
          for (int e = 0; e < 4; ++e) static_cast<uint16_t*>(base)[at + i + e] = f32_bf16(v[q * 4 + e]);
        } else {
          f32x4u r;
#pragma unroll
          for (int e = 0; e < 4; ++e) r[e] = v[q * 4 + e];
          *reinterpret_cast<f32x4u*>(static_cast<float*>(base) + at + i) = r;
        }
      }
    }
  } else {
#pragma unroll
    for (int q = 0; q < 16; ++q) {
      const int i = q * THREADS + tid;
      if (i < count) {
        if (OUT_BF16) static_cast<uint16_t*>(base)[at + i] = f32_bf16(v[q]);
        else static_cast<float*>(base)[at + i] = v[q];
      }
    }
  }
}

enum { P_INF = 0, P_ONE = 1, P_TWO = 2 };

// larger of two values, NaN if either is
__device__ __forceinline__ double max_nan(double a, double b) { return (a != a || a > b) ? a : b; }

template <int P>
__device__ __forceinline__ double join(double a, double b) { return P == P_INF ? max_nan(a, b) : a + b; }

template <int P>
__device__ __forceinline__ double accumulate(double acc, const float (&v)[16]) {
#pragma unroll
  for (int q = 0; q < 16; ++q) {
    if (P == P_TWO) acc = __builtin_fma((double)v[q], (double)v[q], acc);
    else acc = join<P>(fabs((double)v[q]), acc);
  }
  return acc;
}

// the workgroup's value in every thread
template <int P>
__device__ __forceinline__ double block_join(double v) {
  __shared__ double part[THREADS / 64];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = join<P>(v, __shfl_xor(v, o));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) v = join<P>(v, part[w]);
  return v;
}

template <int P>
__global__ __launch_bounds__(THREADS) void norm_partials_kernel(const Table tb, double* __restrict__ partials) {
  double acc = 0.0;
  for (uint32_t c = blockIdx.x; c < tb.n_chunks; c += gridDim.x) {
    const int t = tensor_of(tb, c);
    const int64_t at = (int64_t)(c - tb.first[t]) * CHUNK;
    const int count = (int)min((int64_t)CHUNK, tb.numel[t] - at);
    float v[16];
    if (bit(tb.in_bf16, t)) load16<true>(tb.in[t], at, count, v);
    else load16<false>(tb.in[t], at, count, v);
    acc = accumulate<P>(acc, v);
  }
  acc = block_join<P>(acc);
  if (threadIdx.x == 0) partials[blockIdx.x] = acc;
}

template <int P>
__device__ __forceinline__ double total_of(const double* __restrict__ partials, int n_partials) {
  double acc = 0.0;
  for (int i = threadIdx.x; i < n_partials; i += THREADS) acc = join<P>(acc, partials[i]);
  acc = block_join<P>(acc);
  return P == P_TWO ? sqrt(acc) : acc;
}

template <int P>
__global__ __launch_bounds__(THREADS) void norm_finish_kernel(const double* __restrict__ partials, int n_partials, double* __restrict__ total,
                                                              float* __restrict__ norm_out) {
  const double norm = total_of<P>(partials, n_partials);
  if (threadIdx.x == 0) {
    if (total) *total = norm;
    if (norm_out) *norm_out = (float)norm;
  }
}

// n_partials < 0: partials[0] is the finished norm
template <int P>
__global__ __launch_bounds__(THREADS) void scale_kernel(const Table tb, const double* __restrict__ partials, int n_partials, double max_norm,
                                                        float* __restrict__ norm_out) {
  const double norm = n_partials < 0 ? partials[0] : total_of<P>(partials, n_partials);
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  const double ratio = max_norm / (norm + 1e-6);
  const double factor = ratio > 1.0 ? 1.0 : ratio;  // double: against huge gradients it lies below fp32's normal numbers.  A NaN stays NaN
  // backwards: what the norm pass read last is still in the 256 MB memory-side cache
  for (uint32_t i = blockIdx.x; i < tb.n_chunks; i += gridDim.x) {
    const uint32_t c = tb.n_chunks - 1 - i;
    const int t = tensor_of(tb, c);
    const bool ib = bit(tb.in_bf16, t), ob = bit(tb.out_bf16, t);
    if (factor == 1.0 && tb.in[t] == tb.out[t]) continue;  // g * 1 in place: the same bits
    const int64_t at = (int64_t)(c - tb.first[t]) * CHUNK;
    const int count = (int)min((int64_t)CHUNK, tb.numel[t] - at);
    float v[16];
    if (ib) load16<true>(tb.in[t], at, count, v);
    else load16<false>(tb.in[t], at, count, v);
#pragma unroll
    for (int q = 0; q < 16; ++q) v[q] = (float)((double)v[q] * factor);
    if (ib) {
      if (ob) store16<true, true>(tb.out[t], at, count, v);
      else store16<true, false>(tb.out[t], at, count, v);
    } else {
      if (ob) store16<false, true>(tb.out[t], at, count, v);
      else store16<false, false>(tb.out[t], at, count, v);
    }
  }
}

int fill(Table& tb, int n, int base, const void* const* in, void* const* out, const int64_t* numel, const int32_t* in_dtype,
         const int32_t* out_dtype) {
  tb.n = 0;
  tb.n_chunks = 0;
  for (int w = 0; w < MAX_T / 32; ++w) tb.in_bf16[w] = tb.out_bf16[w] = 0;
  int i = base;
  for (; i < n && tb.n < MAX_T; ++i) {
    if (numel[i] == 0) continue;
    const int64_t chunks = dh::ceil_div(numel[i], CHUNK);
    if ((int64_t)tb.n_chunks + chunks > 0x7fffffff) break;
    const int t = tb.n++;
    tb.in[t] = in[i];
    tb.out[t] = out ? out[i] : nullptr;
    tb.numel[t] = numel[i];
    tb.first[t] = tb.n_chunks;
    tb.n_chunks += (uint32_t)chunks;
    if (in_dtype[i] == DH_DTYPE_BF16) tb.in_bf16[t >> 5] |= 1u << (t & 31);
    if (out && out_dtype[i] == DH_DTYPE_BF16) tb.out_bf16[t >> 5] |= 1u << (t & 31);
  }
  return i;
}

int check(const char* me, int n, const void* const* in, void* const* out, const int64_t* numel, const int32_t* in_dtype, const int32_t* out_dtype,
          int norm_type, const void* ws, size_t ws_bytes, size_t need) {
  if (n < 0) return dh::fail(DH_ERR_INVALID, "%s: negative count", me);
  if (norm_type != P_INF && norm_type != P_ONE && norm_type != P_TWO) return dh::fail(DH_ERR_INVALID, "%s: norm type %d (0 = inf, 1, 2)", me, norm_type);
  if (n > 0 && (!in || !numel || !in_dtype)) return dh::fail(DH_ERR_INVALID, "%s: null table", me);
  for (int i = 0; i < n; ++i) {
    if (numel[i] < 0 || numel[i] > (int64_t)0x7fffffff * CHUNK) return dh::fail(DH_ERR_INVALID, "%s: size of tensor %d", me, i);
    if (numel[i] > 0 && (!in[i] || (out && !out[i]))) return dh::fail(DH_ERR_INVALID, "%s: null tensor %d", me, i);
    if ((in_dtype[i] != DH_DTYPE_F32 && in_dtype[i] != DH_DTYPE_BF16) ||
        (out && out_dtype[i] != DH_DTYPE_F32 && out_dtype[i] != DH_DTYPE_BF16))
      return dh::fail(DH_ERR_INVALID, "%s: dtype of tensor %d", me, i);
    if (out && numel[i] > 0 && in[i] == out[i] && in_dtype[i] != out_dtype[i]) return dh::fail(DH_ERR_INVALID, "%s: tensor %d in place with another dtype", me, i);
  }
  if (!ws || ws_bytes < need) return dh::fail(DH_ERR_WORKSPACE, "%s: workspace of %zu bytes, need %zu", me, ws_bytes, need);
  if (!dh::aligned16(ws)) return dh::fail(DH_ERR_INVALID, "%s: workspace must be 16-byte aligned", me);
  return DH_OK;
}

template <int P>
int run(const char* me, int n, const void* const* in, void* const* out, const int64_t* numel, const int32_t* in_dtype, const int32_t* out_dtype,
        double max_norm, float* norm_out, double* ws, hipStream_t st) {
  Table tb;
  double* partials = ws + 2;  // ws[0]: the finished norm when many launches' partial sums were joined by a launch of their own
  int n_partials = 0;
  for (int base = 0; base < n;) {
    base = fill(tb, n, base, in, out, numel, in_dtype, out_dtype);
    if (tb.n == 0) continue;
    const int grid = (int)(tb.n_chunks < (uint32_t)GRID ? tb.n_chunks : (uint32_t)GRID);
    hipLaunchKernelGGL(norm_partials_kernel<P>, dim3(grid), dim3(THREADS), 0, st, tb, partials + n_partials);
    n_partials += grid;
  }
  if (!out || n_partials == 0 || n_partials > INLINE_PARTIALS) {
    hipLaunchKernelGGL(norm_finish_kernel<P>, dim3(1), dim3(THREADS), 0, st, partials, n_partials, ws, norm_out);
    norm_out = nullptr;
    partials = ws;
    n_partials = -1;
  }
  if (out) {
    for (int base = 0; base < n;) {
      base = fill(tb, n, base, in, out, numel, in_dtype, out_dtype);
      if (tb.n == 0) continue;
      const int grid = (int)(tb.n_chunks < (uint32_t)(2 * GRID) ? tb.n_chunks : (uint32_t)(2 * GRID));
      hipLaunchKernelGGL(scale_kernel<P>, dim3(grid), dim3(THREADS), 0, st, tb, partials, n_partials, max_norm, norm_out);
      norm_out = nullptr;
    }
  }
  return dh::check_launch(me);
}

int dispatch(const char* me, int n, const void* const* in, void* const* out, const int64_t* numel, const int32_t* in_dtype,
             const int32_t* out_dtype, int norm_type, double max_norm, float* norm_out, void* ws, hipStream_t st) {
  double* w = static_cast<double*>(ws);
  switch (norm_type) {
    case P_INF: return run<P_INF>(me, n, in, out, numel, in_dtype, out_dtype, max_norm, norm_out, w, st);
    case P_ONE: return run<P_ONE>(me, n, in, out, numel, in_dtype, out_dtype, max_norm, norm_out, w, st);
    default: return run<P_TWO>(me, n, in, out, numel, in_dtype, out_dtype, max_norm, norm_out, w, st);
  }
}

}  // namespace

// a launch takes up to MAX_T tensors; one that is cut short by the 2^31 chunk limit takes at least one, so n launches bound it
extern "C" size_t dh_grad_norm_workspace_bytes(int n, const int64_t* numel) {
  if (n <= 0 || !numel) return 16;
  size_t partials = 0;
  int t = 0;
  int64_t chunks = 0;
  for (int i = 0; i < n; ++i) {  // the same cuts as fill()
    if (numel[i] <= 0) continue;
    const int64_t c = dh::ceil_div(numel[i], CHUNK);
    if (t == MAX_T || chunks + c > 0x7fffffff) {
      partials += (size_t)(chunks < GRID ? chunks : GRID);
      t = 0;
      chunks = 0;
    }
    ++t;
    chunks += c;
  }
  partials += (size_t)(chunks < GRID ? chunks : GRID);
  return 16 + 8 * partials;
}

extern "C" int dh_grad_norm(int n, const void* const* grads, const int64_t* numel, const int32_t* dtype, int norm_type, float* norm, void* workspace,
                            size_t workspace_bytes, dh_stream_t stream) {
  const char* me = "dh_grad_norm";
  if (!norm) return dh::fail(DH_ERR_INVALID, "%s: null norm", me);
  const int rc = check(me, n, grads, nullptr, numel, dtype, nullptr, norm_type, workspace, workspace_bytes,
                       n < 0 ? 0 : dh_grad_norm_workspace_bytes(n, numel));
  if (rc != DH_OK) return rc;
  return dispatch(me, n, grads, nullptr, numel, dtype, nullptr, norm_type, 0.0, norm, workspace, dh::as_stream(stream));
}

extern "C" int dh_grad_clip(int n, const void* const* grads, void* const* out, const int64_t* numel, const int32_t* dtype, const int32_t* out_dtype,
                            int norm_type, double max_norm, float* norm, void* workspace, size_t workspace_bytes, dh_stream_t stream) {
  const char* me = "dh_grad_clip";
  if (!norm) return dh::fail(DH_ERR_INVALID, "%s: null norm", me);
  if (n > 0 && (!out || !out_dtype)) return dh::fail(DH_ERR_INVALID, "%s: null table", me);
  const int rc = check(me, n, grads, out, numel, dtype, out_dtype, norm_type, workspace, workspace_bytes,
                       n < 0 ? 0 : dh_grad_norm_workspace_bytes(n, numel));
  if (rc != DH_OK) return rc;
  return dispatch(me, n, grads, out, numel, dtype, out_dtype, norm_type, max_norm, norm, workspace, dh::as_stream(stream));
}
