// The norms around a block, its gate and its residual in one pass each way (dance/models/nn/gnn.py:84-96: the `norm` slot of a layer and
// the sum of a node's own and its neighbours' features are the reference's places for it):
//
//   n = post-norm(f)  or f          norm(v) = (v - mean) rstd w + b  (layer)  or  v rstd w + b, rstd = 1 / sqrt(mean(v^2) + eps)  (rms)
//   r = x + scale * act(gate) * n   act = identity or sigmoid; gate per element, per row, per column, one for all, or none
//   h = pre-norm(r)  or nothing     from the unrounded r
//
// Backward, with fhat / rhat the normalised f / r, u = dout w of the norm concerned and <.> the mean over a row:
//   dr~ = dr + rstd2 (u2 - <u2> - rhat <u2 rhat>)      (rms: without <u2>);   dx = dr~
//   dn  = scale act(gate) dr~;   dgate = scale dr~ n act'(gate);   df = rstd1 (u1 - <u1> - fhat <u1 fhat>)
//   dw = sum_rows dout vhat,  db = sum_rows dout
//
// Bound: HBM.  Forward reads f and x and writes r and h; backward reads f, x, dr, dh and writes df, dx: r is recomputed from f, x and the
// gate (the same bytes as reading it back, and unrounded in the bf16 case), only mean and rstd of each row are kept.
// Split: a row lives in the registers of 8 .. 64 lanes of a wave (rows up to 512 columns) or of a workgroup of two to eight waves (up to
// 4096), 4 or 8 elements per lane (16 spill: the backward holds ten arrays of them), 16 bytes per access whatever the rows' alignment
// (global memory takes unaligned accesses); a row length that is no multiple of the access reads its last piece from D - V and shifts it
// down in registers (ODD), so no load is guarded.  The two-pass variance and both reductions of the backward run on registers.  Column
// gradients are summed in registers over the rows a workgroup walks, joined in its LDS, written once per workgroup and added up by a second
// kernel in workgroup order: no atomics, the result does not depend on timing.  All arithmetic is fp32; bf16 rounds once, at the stores.
// Measured, layer norms and channel gate, forward / backward: 200003 x 512 bf16 165 / 282 us (5.0 / 4.4 TB/s), fp32 321 / 446 us (5.1 / 5.5);
// 50001 x 504 bf16 37 / 76 us, x 500 (ODD) 50 / 95, x 501 53 / 101; 50001 x 1000 109 / 184.  The bf16 backward has the arithmetic of twice
// as many elements to a byte and comes near the vector units' limit.
// Wide rows (4097 .. 8192 columns, entries of their own): a workgroup of up to eight waves, sixteen elements a lane.  The backward takes one
// workgroup for every row, without the column gradients, which would spill, and leaves two numbers a row; a second kernel walks the columns
// down the rows and reads f, x, dr and dh again, so a training pass moves 14 row lengths instead of 10.  12001 rows, bf16 / fp32, forward and
// training pass: x 4096 (not wide) 102, 282 / 163, 405 us; x 5000 162, 496 / 236, 772; x 8192 185, 651 / 302, 1124; x 4097 281, 709 / 293, 789
// (rows that start at odd elements).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.h"

namespace {

enum { GATE_NONE = DH_GATE_NONE, GATE_SCALAR = DH_GATE_SCALAR, GATE_CHANNEL = DH_GATE_CHANNEL, GATE_ROW = DH_GATE_ROW, GATE_FULL = DH_GATE_FULL };
constexpr int64_t MAX_D = 4096, WIDE_D = 8192;  // columns of a row; of one in the wide entries
// who holds a row: part of a wave, a wave, a workgroup;  how the row ends: with the lanes' last access, with an access before, inside one
enum { SUB = 0, WAVE = 1, GROUP = 2 };
enum { WHOLE = 0, SHORT = 1, ODD = 2 };
constexpr int BWD_BLOCKS = 1024;  // workgroups of a backward launch at most = partial rows of the column gradients
constexpr int WIDE_CHUNKS = 256;  // row chunks of wide rows' column gradients = partial rows; 3 to 8 workgroups side by side in each

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));

struct Args {
  int64_t M;
  int D, gate_kind, gate_sigmoid, rms, tpr, has_post, has_pre;
  float scale, eps, inv_d;
  const void *f, *x, *gate;
  int64_t ldf, ldx, ldg;
  const float *w1, *b1, *w2, *b2;
  float* stats;  // [M, 4]: mean1, rstd1, mean2, rstd2
  // forward
  void *r, *h;
  int64_t ldr, ldh;
  // backward
  const void *dr, *dh;
  int64_t lddr, lddh;
  void *df, *dx, *dgate;  // dgate: row and full gates
  int64_t lddf, lddx, lddg;
  float* partials;  // [n_arrays][gridDim.x][D]
  int want_w1, want_b1, want_w2, want_b2, want_gate;
  // wide rows
  float2* terms;  // [M]: <u2 rhat>, <u2> of each row, for the kernel of the column gradients; null: nobody asks
  int64_t rows;   // of a workgroup of that kernel
};

__device__ __forceinline__ float bf16_f32(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
// two values rounded to bf16 (v_cvt_pk_bf16_f32: nearest even, a NaN stays one)
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
}

template <class T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int VEC = 4;
  static __device__ __forceinline__ float get(const void* p, int64_t i) { return static_cast<const float*>(p)[i]; }
  static __device__ __forceinline__ void put(void* p, int64_t i, float v) { static_cast<float*>(p)[i] = v; }
  template <int V>
  static __device__ __forceinline__ void store(void* p, int64_t i, const float* v) {
    if (V == 4) {
      f32x4u t;
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] = v[e];
      *reinterpret_cast<f32x4u*>(static_cast<float*>(p) + i) = t;
    } else {
      put(p, i, v[0]);
    }
  }
  // the first n (uniform) of four values
  static __device__ __forceinline__ void store_first(void* p, int64_t i, int n, const float* v) {
    typedef float f32x2u __attribute__((ext_vector_type(2), aligned(4)));
    if (n & 2) *reinterpret_cast<f32x2u*>(static_cast<float*>(p) + i) = f32x2u{v[0], v[1]};
    if (n & 1) {
      const float last = v[2], first = v[0];
      put(p, i + (n & 2), (n & 2) ? last : first);
    }
  }
};
template <>
struct Elem<uint16_t> {
  static constexpr int VEC = 8;
  static __device__ __forceinline__ float get(const void* p, int64_t i) { return bf16_f32(static_cast<const uint16_t*>(p)[i]); }
  static __device__ __forceinline__ void put(void* p, int64_t i, float v) { static_cast<uint16_t*>(p)[i] = (uint16_t)pack_bf16(v, 0.f); }
  template <int V>
  static __device__ __forceinline__ void store(void* p, int64_t i, const float* v) {
    if (V == 8) {
      u32x4u t;
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] = pack_bf16(v[2 * e], v[2 * e + 1]);
      *reinterpret_cast<u32x4u*>(static_cast<uint16_t*>(p) + i) = t;
    } else {
      put(p, i, v[0]);
    }
  }
  // the first n (uniform) of eight values
  static __device__ __forceinline__ void store_first(void* p, int64_t i, int n, const float* v) {
    typedef uint32_t u32x2u __attribute__((ext_vector_type(2), aligned(2)));
    typedef uint32_t u32u __attribute__((aligned(2)));
    uint16_t* to = static_cast<uint16_t*>(p) + i;
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = pack_bf16(v[2 * e], v[2 * e + 1]);
    if (n & 4) {
      *reinterpret_cast<u32x2u*>(to) = u32x2u{w[0], w[1]};
      to += 4;
      w[0] = w[2];
      w[1] = w[3];
    }
    if (n & 2) {
      *reinterpret_cast<u32u*>(to) = w[0];
      to += 2;
      w[0] = w[1];
    }
    if (n & 1) *to = (uint16_t)w[0];
  }
};

// V consecutive fp32 parameters; they carry no alignment promise beyond their own four bytes
template <int V>
__device__ __forceinline__ void load_param(const float* p, int col, float* v) {
  typedef float f32x4p __attribute__((ext_vector_type(4), aligned(4)));
  if (V >= 4) {
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
      const f32x4p t = *reinterpret_cast<const f32x4p*>(p + col + q * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[q * 4 + e] = t[e];
    }
  } else {
    v[0] = p[col];
  }
}

__device__ __forceinline__ float sigmoid(float v) { return 1.f / (1.f + expf(-v)); }

// the sum over a wave in every lane, by DPP adds: 6 instructions where a butterfly through LDS takes 18 and its latencies
__device__ __forceinline__ float wave_sum(float v) {
  auto add = [&](auto ctrl, auto rows) __attribute__((always_inline)) {
    v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
  };
  add(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{});  // row_shr 1, 2, 4, 8: lane 15 of a row of 16 has its sum
  add(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{});
  add(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{});
  add(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{});
  add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});  // row_bcast 15 into rows 1 and 3
  add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});  // row_bcast 31 into rows 2 and 3
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 63));
}

// N sums over the threads of a row, the result in each of them
template <int MODE, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], int tpr, float* lds) {
  if (MODE == SUB) {
    for (int o = tpr >> 1; o > 0; o >>= 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], o);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
  if (MODE == GROUP) {
    const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    __syncthreads();  // the previous reduction's values have been read
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) lds[wave * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.f;
    for (int w = 0; w < waves; ++w) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += lds[w * N + i];
    }
  }
}

// A lane's columns: chunk c covers (c * tpr + t) * V .. + V.  Chunks that end behind D read the last V values of the row instead; with
// ODD their values are shifted down to the columns they belong to.  What lies at columns >= D is some value of the same row.
// (The two values are read before the choice: a choice between array elements themselves becomes an index into the registers, a chain of
// compares each; rows of 500 columns took five times as long as rows of 504.)
template <int V>
__device__ __forceinline__ void shift_down(int by, float* v) {
#pragma unroll
  for (int bit = 1; bit < V; bit *= 2)
#pragma unroll
    for (int e = 0; e + bit < V; ++e) {
      const float far = v[e + bit], near = v[e];
      v[e] = (by & bit) ? far : near;
    }
}
// the same of 16 bytes, PER elements to a word
template <int PER>
__device__ __forceinline__ void shift_words(int by, uint32_t (&w)[4]) {
#pragma unroll
  for (int bit = 1; bit < 4; bit *= 2)
#pragma unroll
    for (int e = 0; e + bit < 4; ++e) {
      const uint32_t far = w[e + bit], near = w[e];
      w[e] = (by & (bit * PER)) ? far : near;
    }
  if (PER == 2) {
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = __builtin_amdgcn_alignbyte(w[e < 3 ? e + 1 : e], w[e], (by & 1) * 2);
  }
}
// A row's pieces as they lie in memory (requested before any of them is used).
template <class T, int V, int CH>
struct RawRow {
  static constexpr int WORDS = V == 1 ? 1 : 4;
  uint32_t w[CH][WORDS];

  __device__ __forceinline__ void load(const void* p, int64_t row_at, int t, int tpr, int D) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const T* from = static_cast<const T*>(p) + row_at + min((c * tpr + t) * V, D - V);
      if constexpr (V == 1) {
        if constexpr (sizeof(T) == 2) w[c][0] = *from;
        else w[c][0] = __float_as_uint(*from);
      } else {
        const u32x4u v = *reinterpret_cast<const u32x4u*>(from);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[c][e] = v[e];
      }
    }
  }
  template <int TAIL>
  __device__ __forceinline__ void unpack(int t, int tpr, int D, float (&v)[V * CH]) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if constexpr (TAIL == ODD) shift_words<V / 4>(max((c * tpr + t) * V - (D - V), 0), w[c]);
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int e = 0; e < WORDS; ++e) {
          v[c * V + (V == 1 ? 0 : 2 * e)] = __uint_as_float(w[c][e] << 16);
          if constexpr (V != 1) v[c * V + 2 * e + 1] = __uint_as_float(w[c][e] & 0xffff0000u);
        }
      } else {
#pragma unroll
        for (int e = 0; e < WORDS; ++e) v[c * V + e] = __uint_as_float(w[c][e]);
      }
    }
  }
};
template <int V, int CH, int TAIL>
__device__ __forceinline__ void zero_tail(int t, int tpr, int D, float (&v)[V * CH]) {
  if (TAIL == WHOLE) return;
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e)
      if ((c * tpr + t) * V + (TAIL == ODD ? e : 0) >= D) v[c * V + e] = 0.f;
}
template <int V, int CH, int TAIL>
__device__ __forceinline__ void load_params(const float* p, float fallback, int t, int tpr, int D, float (&v)[V * CH]) {
  if (p) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      load_param<V>(p, min((c * tpr + t) * V, D - V), v + c * V);
      if (TAIL == ODD) shift_down<V>(max((c * tpr + t) * V - (D - V), 0), v + c * V);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V * CH; ++i) v[i] = fallback;
  }
}
template <class T, int V, int CH, int TAIL>
__device__ __forceinline__ void store_row(void* p, int64_t row_at, int t, int tpr, int D, const float (&v)[V * CH]) {
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int col = (c * tpr + t) * V;
    if (TAIL == WHOLE || (TAIL == ODD ? col + V <= D : col < D)) Elem<T>::template store<V>(p, row_at + col, v + c * V);
    else if (TAIL == ODD && col < D) Elem<T>::store_first(p, row_at + col, D % V, v + c * V);
  }
}

// mean and rstd of a row held in registers (entries beyond D are zero); v becomes v - mean: the subtraction comes first everywhere, so a row
// that is nearly constant keeps the digits its differences have
template <int MODE, int V, int CH, int TAIL>
__device__ __forceinline__ void row_stats(const Args& a, int t, float (&v)[V * CH], float* lds, float& mean, float& rstd) {
  const int tpr = MODE == WAVE ? 64 : a.tpr;
  float s[1] = {0.f};
  mean = 0.f;
  if (!a.rms) {
#pragma unroll
    for (int i = 0; i < V * CH; ++i) s[0] += v[i];
    row_sums<MODE, 1>(s, tpr, lds);
    mean = s[0] * a.inv_d;
#pragma unroll
    for (int i = 0; i < V * CH; ++i) v[i] -= mean;
    zero_tail<V, CH, TAIL>(t, tpr, a.D, v);
    s[0] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < V * CH; ++i) s[0] = __builtin_fmaf(v[i], v[i], s[0]);
  row_sums<MODE, 1>(s, tpr, lds);
  rstd = 1.f / sqrtf(s[0] * a.inv_d + a.eps);
}

// v = v rstd w + b
template <int E>
__device__ __forceinline__ void scale_shift(float (&v)[E], float rstd, const float (&w)[E], const float (&b)[E]) {
#pragma unroll
  for (int i = 0; i < E; ++i) v[i] = __builtin_fmaf(v[i] * rstd, w[i], b[i]);
}

template <class T, int V, int CH, int MODE, bool FULL, int TAIL>
__global__ __launch_bounds__(MODE == GROUP ? 512 : 256) void residual_norm_forward_kernel(const Args a) {
  constexpr int E = V * CH;
  __shared__ float lds[8];
  const int tpr = MODE == WAVE ? 64 : a.tpr, t = MODE == GROUP ? threadIdx.x : threadIdx.x & (tpr - 1);
  const int rows_per_block = MODE == GROUP ? 1 : 256 / tpr;
  // the row within the workgroup's pass; uniform (a scalar, and with it the rows' addresses) where a wave holds one row
  const int sub = MODE == GROUP ? 0 : MODE == WAVE ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : threadIdx.x / tpr;
  float ga[E];
  if (!FULL) {
    if (a.gate_kind == GATE_CHANNEL) load_params<V, CH, TAIL>(static_cast<const float*>(a.gate), 1.f, t, tpr, a.D, ga);
    else {
      const float g = a.gate_kind == GATE_SCALAR ? *static_cast<const float*>(a.gate) : 1.f;
#pragma unroll
      for (int i = 0; i < E; ++i) ga[i] = g;
    }
    if (a.gate_sigmoid && (a.gate_kind == GATE_CHANNEL || a.gate_kind == GATE_SCALAR)) {
#pragma unroll
      for (int i = 0; i < E; ++i) ga[i] = sigmoid(ga[i]);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) ga[i] *= a.scale;
  }
  for (int64_t base = (int64_t)blockIdx.x * rows_per_block; base < a.M; base += (int64_t)gridDim.x * rows_per_block) {
    const int64_t row = min(base + sub, a.M - 1);
    const bool valid = base + sub < a.M;
    float f[E], x[E], gf[E], w[E], b[E], grow = 1.f;
    RawRow<T, V, CH> rf, rx, rg;
    rf.load(a.f, row * a.ldf, t, tpr, a.D);
    if (a.x) rx.load(a.x, row * a.ldx, t, tpr, a.D);
    if (FULL) rg.load(a.gate, row * a.ldg, t, tpr, a.D);
    else if (a.gate_kind == GATE_ROW) grow = Elem<T>::get(a.gate, row * a.ldg);
    rf.template unpack<TAIL>(t, tpr, a.D, f);
    if (a.x) rx.template unpack<TAIL>(t, tpr, a.D, x);
    else {
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = 0.f;
    }
    if (FULL) rg.template unpack<TAIL>(t, tpr, a.D, gf);
    if (!FULL && a.gate_kind == GATE_ROW && a.gate_sigmoid) grow = sigmoid(grow);
    zero_tail<V, CH, TAIL>(t, tpr, a.D, f);
    float m1 = 0.f, s1 = 1.f, m2 = 0.f, s2 = 1.f;
    if (a.has_post) {
      load_params<V, CH, TAIL>(a.w1, 1.f, t, tpr, a.D, w);
      load_params<V, CH, TAIL>(a.b1, 0.f, t, tpr, a.D, b);
      row_stats<MODE, V, CH, TAIL>(a, t, f, lds, m1, s1);
      scale_shift<E>(f, s1, w, b);
    }
    if (FULL) {
      if (a.gate_sigmoid) {
#pragma unroll
        for (int i = 0; i < E; ++i) gf[i] = sigmoid(gf[i]);
      }
#pragma unroll
      for (int i = 0; i < E; ++i) f[i] = __builtin_fmaf(a.scale * gf[i], f[i], x[i]);
    } else if (a.gate_kind == GATE_ROW) {
      const float g = a.scale * grow;
#pragma unroll
      for (int i = 0; i < E; ++i) f[i] = __builtin_fmaf(g, f[i], x[i]);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) f[i] = __builtin_fmaf(ga[i], f[i], x[i]);
    }
    if (valid && a.r) store_row<T, V, CH, TAIL>(a.r, row * a.ldr, t, tpr, a.D, f);
    if (a.has_pre) {
      zero_tail<V, CH, TAIL>(t, tpr, a.D, f);
      load_params<V, CH, TAIL>(a.w2, 1.f, t, tpr, a.D, w);
      load_params<V, CH, TAIL>(a.b2, 0.f, t, tpr, a.D, b);
      row_stats<MODE, V, CH, TAIL>(a, t, f, lds, m2, s2);
      scale_shift<E>(f, s2, w, b);
      if (valid) store_row<T, V, CH, TAIL>(a.h, row * a.ldh, t, tpr, a.D, f);
    }
    if (valid && a.stats && t == 0) *reinterpret_cast<float4*>(a.stats + row * 4) = make_float4(m1, s1, m2, s2);
  }
}

// the workgroup's column sums of one array: joined over its row groups in LDS, written to partials[slot][blockIdx.x]
template <int V, int CH, int MODE>
__device__ __forceinline__ void put_partials(const Args& a, int t, int sub, const float (&acc)[V * CH], int slot, float* lds) {
  const int tpr = MODE == WAVE ? 64 : a.tpr;
  float* out = a.partials + ((int64_t)slot * gridDim.x + blockIdx.x) * a.D;
  if (MODE == GROUP) {
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int col = (c * tpr + t) * V + e;
        if (col < a.D) out[col] = acc[c * V + e];
      }
  } else {
    const int span = tpr * V * CH, groups = 256 / tpr;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) lds[sub * span + (c * tpr + t) * V + e] = acc[c * V + e];
    __syncthreads();
    for (int col = threadIdx.x; col < a.D; col += 256) {
      float s = 0.f;
      for (int g = 0; g < groups; ++g) s += lds[g * span + col];
      out[col] = s;
    }
  }
}

template <class T, int V, int CH, int MODE, bool FULL, int TAIL>
__global__ __launch_bounds__(MODE == GROUP ? 512 : 256) void residual_norm_backward_kernel(const Args a) {
  constexpr int E = V * CH;
  __shared__ float lds[MODE == GROUP ? 32 : 256 * E];
  const int tpr = MODE == WAVE ? 64 : a.tpr, t = MODE == GROUP ? threadIdx.x : threadIdx.x & (tpr - 1);
  const int rows_per_block = MODE == GROUP ? 1 : 256 / tpr;
  // the row within the workgroup's pass; uniform (a scalar, and with it the rows' addresses) where a wave holds one row
  const int sub = MODE == GROUP ? 0 : MODE == WAVE ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : threadIdx.x / tpr;
  constexpr bool COLUMNS = E <= 8;  // column gradients: sixteen elements a lane leave no registers for them (wide_columns_kernel)
  constexpr int A = COLUMNS ? E : 1;
  float acc_w1[A], acc_b1[A], acc_w2[A], acc_b2[A], acc_g[A];
#pragma unroll
  for (int i = 0; i < A; ++i) acc_w1[i] = acc_b1[i] = acc_w2[i] = acc_b2[i] = acc_g[i] = 0.f;
  const bool col_gate = !FULL && (a.gate_kind == GATE_CHANNEL || a.gate_kind == GATE_SCALAR);
  const bool use_x = a.x && a.dh;  // r enters through the second norm only
  // (blockIdx.y: wide rows only)
  for (int64_t base = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * rows_per_block; base < a.M; base += (int64_t)gridDim.x * rows_per_block) {
    const int64_t row = min(base + sub, a.M - 1);
    const bool valid = base + sub < a.M;
    float f[E], x[E], gf[E], dr[E], dh[E], w[E], b[E];
    RawRow<T, V, CH> rf, rx, rr, rh, rg;
    float grow = 1.f;
    rf.load(a.f, row * a.ldf, t, tpr, a.D);
    if (use_x) rx.load(a.x, row * a.ldx, t, tpr, a.D);
    if (a.dr) rr.load(a.dr, row * a.lddr, t, tpr, a.D);
    if (a.dh) rh.load(a.dh, row * a.lddh, t, tpr, a.D);
    if (FULL) rg.load(a.gate, row * a.ldg, t, tpr, a.D);
    else if (a.gate_kind == GATE_ROW) grow = Elem<T>::get(a.gate, row * a.ldg);
    const float4 st = *reinterpret_cast<const float4*>(a.stats + row * 4);
    rf.template unpack<TAIL>(t, tpr, a.D, f);
    if (use_x) rx.template unpack<TAIL>(t, tpr, a.D, x);
    else {
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = 0.f;
    }
    if (a.dr) rr.template unpack<TAIL>(t, tpr, a.D, dr);
    else {
#pragma unroll
      for (int i = 0; i < E; ++i) dr[i] = 0.f;
    }
    if (a.dh) rh.template unpack<TAIL>(t, tpr, a.D, dh);
    if (FULL) rg.template unpack<TAIL>(t, tpr, a.D, gf);
    // the gate and its derivative's factor
    if (!FULL) {
      if (a.gate_kind == GATE_CHANNEL) load_params<V, CH, TAIL>(static_cast<const float*>(a.gate), 1.f, t, tpr, a.D, gf);
      else {
        const float g = a.gate_kind == GATE_SCALAR ? *static_cast<const float*>(a.gate) : a.gate_kind == GATE_ROW ? grow : 1.f;
#pragma unroll
        for (int i = 0; i < E; ++i) gf[i] = g;
      }
    }
    const bool sig = a.gate_sigmoid && a.gate_kind != GATE_NONE;
    if (sig) {
#pragma unroll
      for (int i = 0; i < E; ++i) gf[i] = sigmoid(gf[i]);
    }
    if (a.has_post) {
      load_params<V, CH, TAIL>(a.w1, 1.f, t, tpr, a.D, w);
      load_params<V, CH, TAIL>(a.b1, 0.f, t, tpr, a.D, b);
#pragma unroll
      for (int i = 0; i < E; ++i) f[i] = (f[i] - st.x) * st.y;  // fhat from here on
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) { w[i] = 1.f; b[i] = 0.f; }
    }
    if (a.dh) {
      float w2[E];
      load_params<V, CH, TAIL>(a.w2, 1.f, t, tpr, a.D, w2);
      zero_tail<V, CH, TAIL>(t, tpr, a.D, dh);
      float s[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float n = __builtin_fmaf(f[i], w[i], b[i]);
        x[i] = (__builtin_fmaf(a.scale * gf[i], n, x[i]) - st.z) * st.w;  // rhat
      }
      // behind the end of a bf16 row of odd length the features stand beside other columns' gate and parameters: a product that no column
      // has, and that may be infinite where all of theirs are finite
      if constexpr (TAIL == ODD && sizeof(T) == 2) zero_tail<V, CH, TAIL>(t, tpr, a.D, x);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if constexpr (COLUMNS) {
          if (valid) {
            acc_w2[i] = __builtin_fmaf(dh[i], x[i], acc_w2[i]);
            acc_b2[i] += dh[i];
          }
        }
        dh[i] *= w2[i];
        s[0] = __builtin_fmaf(dh[i], x[i], s[0]);
        s[1] += dh[i];
      }
      row_sums<MODE, 2>(s, tpr, lds);
      const float c1 = s[0] * a.inv_d, c0 = a.rms ? 0.f : s[1] * a.inv_d;
      if constexpr (!COLUMNS) {
        if (a.terms && t == 0) a.terms[row] = make_float2(c1, c0);
      }
#pragma unroll
      for (int i = 0; i < E; ++i) dr[i] = __builtin_fmaf(st.w, __builtin_fmaf(-x[i], c1, dh[i] - c0), dr[i]);
    }
    if (valid && a.dx) store_row<T, V, CH, TAIL>(a.dx, row * a.lddx, t, tpr, a.D, dr);
    zero_tail<V, CH, TAIL>(t, tpr, a.D, dr);
    float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float n = __builtin_fmaf(f[i], w[i], b[i]), sd = a.scale * dr[i];
      float dg = sd * n;
      if (sig) dg *= gf[i] * (1.f - gf[i]);
      const float dn = sd * gf[i];
      if constexpr (COLUMNS) {
        if (valid) {
          acc_w1[i] = __builtin_fmaf(dn, f[i], acc_w1[i]);
          acc_b1[i] += dn;
          if (col_gate) acc_g[i] += dg;
        }
      }
      const float u = dn * w[i];
      s[0] = __builtin_fmaf(u, f[i], s[0]);
      s[1] += u;
      gf[i] = dg;
      dr[i] = u;
    }
    if (FULL && valid && a.dgate) store_row<T, V, CH, TAIL>(a.dgate, row * a.lddg, t, tpr, a.D, gf);
    if (a.gate_kind == GATE_ROW && a.dgate) {  // (behind the row's end lies a product of zero with some value of the row, which may be infinite)
      zero_tail<V, CH, TAIL>(t, tpr, a.D, gf);
#pragma unroll
      for (int i = 0; i < E; ++i) s[2] += gf[i];
    }
    if (a.has_post || (a.gate_kind == GATE_ROW && a.dgate)) row_sums<MODE, 3>(s, tpr, lds);
    if (a.gate_kind == GATE_ROW && a.dgate && valid && t == 0) Elem<T>::put(a.dgate, row * a.lddg, s[2]);
    if (a.df && valid) {
      if (a.has_post) {
        const float c1 = s[0] * a.inv_d, c0 = a.rms ? 0.f : s[1] * a.inv_d;
#pragma unroll
        for (int i = 0; i < E; ++i) dr[i] = st.y * __builtin_fmaf(-f[i], c1, dr[i] - c0);
      }
      store_row<T, V, CH, TAIL>(a.df, row * a.lddf, t, tpr, a.D, dr);
    }
    if constexpr (!COLUMNS) break;  // one workgroup for every row: no parameters to keep in registers from row to row
  }
  if constexpr (COLUMNS) {
    int slot = 0;
    if (a.want_w1) put_partials<V, CH, MODE>(a, t, sub, acc_w1, slot++, lds);
    if (a.want_b1) put_partials<V, CH, MODE>(a, t, sub, acc_b1, slot++, lds);
    if (a.want_w2) put_partials<V, CH, MODE>(a, t, sub, acc_w2, slot++, lds);
    if (a.want_b2) put_partials<V, CH, MODE>(a, t, sub, acc_b2, slot++, lds);
    if (a.want_gate) put_partials<V, CH, MODE>(a, t, sub, acc_g, slot++, lds);
  }
}

// The column gradients of wide rows: a thread walks V columns down the rows of its workgroup, with the row's four statistics and the two
// means of the second norm's gradient that the row kernel left.  f, x, dr and dh are read a second time for it.
template <class T, int V, bool FULL, int TAIL>
__global__ __launch_bounds__(256) void wide_columns_kernel(const Args a) {
  const int t = blockIdx.x * 256 + threadIdx.x;  // the piece of the row
  if (t * V >= a.D) return;
  float w1[V], b1[V], w2[V], gc[V], acc_w1[V], acc_b1[V], acc_w2[V], acc_b2[V], acc_g[V];
  load_params<V, 1, TAIL>(a.has_post ? a.w1 : nullptr, 1.f, t, 0, a.D, w1);
  load_params<V, 1, TAIL>(a.has_post ? a.b1 : nullptr, 0.f, t, 0, a.D, b1);
  load_params<V, 1, TAIL>(a.has_pre ? a.w2 : nullptr, 1.f, t, 0, a.D, w2);
  load_params<V, 1, TAIL>(a.gate_kind == GATE_CHANNEL ? static_cast<const float*>(a.gate) : nullptr,
                          a.gate_kind == GATE_SCALAR ? *static_cast<const float*>(a.gate) : 1.f, t, 0, a.D, gc);
#pragma unroll
  for (int e = 0; e < V; ++e) acc_w1[e] = acc_b1[e] = acc_w2[e] = acc_b2[e] = acc_g[e] = 0.f;
  const bool sig = a.gate_sigmoid && a.gate_kind != GATE_NONE;
  const int64_t first = (int64_t)blockIdx.y * a.rows, last = min(first + a.rows, a.M);
  for (int64_t row = first; row < last; ++row) {
    RawRow<T, V, 1> rf, rx, rr, rh, rg;
    float f[V], x[V], dr[V], dh[V], gf[V];
    rf.load(a.f, row * a.ldf, t, 0, a.D);
    if (a.x && a.dh) rx.load(a.x, row * a.ldx, t, 0, a.D);
    if (a.dr) rr.load(a.dr, row * a.lddr, t, 0, a.D);
    if (a.dh) rh.load(a.dh, row * a.lddh, t, 0, a.D);
    if (FULL) rg.load(a.gate, row * a.ldg, t, 0, a.D);
    const float grow = !FULL && a.gate_kind == GATE_ROW ? Elem<T>::get(a.gate, row * a.ldg) : 0.f;
    const float4 st = *reinterpret_cast<const float4*>(a.stats + row * 4);
    const float2 c = a.dh ? a.terms[row] : make_float2(0.f, 0.f);
    rf.template unpack<TAIL>(t, 0, a.D, f);
    if (a.x && a.dh) rx.template unpack<TAIL>(t, 0, a.D, x);
    if (a.dr) rr.template unpack<TAIL>(t, 0, a.D, dr);
    if (a.dh) rh.template unpack<TAIL>(t, 0, a.D, dh);
    if (FULL) rg.template unpack<TAIL>(t, 0, a.D, gf);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (!FULL) gf[e] = a.gate_kind == GATE_ROW ? grow : gc[e];
      if (sig) gf[e] = sigmoid(gf[e]);
      const float fhat = a.has_post ? (f[e] - st.x) * st.y : f[e], n = __builtin_fmaf(fhat, w1[e], b1[e]);
      float d = a.dr ? dr[e] : 0.f;
      if (a.dh) {
        const float rhat = (__builtin_fmaf(a.scale * gf[e], n, a.x ? x[e] : 0.f) - st.z) * st.w;
        acc_w2[e] = __builtin_fmaf(dh[e], rhat, acc_w2[e]);
        acc_b2[e] += dh[e];
        d = __builtin_fmaf(st.w, __builtin_fmaf(-rhat, c.x, dh[e] * w2[e] - c.y), d);
      }
      const float sd = a.scale * d, dn = sd * gf[e];
      acc_w1[e] = __builtin_fmaf(dn, fhat, acc_w1[e]);
      acc_b1[e] += dn;
      float dg = sd * n;
      if (sig) dg *= gf[e] * (1.f - gf[e]);
      acc_g[e] += dg;
    }
  }
  int slot = 0;
  auto put = [&](const float (&acc)[V]) __attribute__((always_inline)) {
    float* out = a.partials + ((int64_t)slot++ * gridDim.y + blockIdx.y) * a.D;
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (t * V + e < a.D) out[t * V + e] = acc[e];
  };
  if (a.want_w1) put(acc_w1);
  if (a.want_b1) put(acc_b1);
  if (a.want_w2) put(acc_w2);
  if (a.want_b2) put(acc_b2);
  if (a.want_gate) put(acc_g);
}

struct ReduceArgs {
  const float* partials;
  float* out[5];
  int n_blocks, D;
};

// out[slot][col] = sum over workgroups, 64 columns x 16 row splits per workgroup, joined in split order
__global__ __launch_bounds__(1024) void column_reduce_kernel(const ReduceArgs a) {
  __shared__ float part[16][64];
  const int col = blockIdx.x * 64 + (threadIdx.x & 63), split = threadIdx.x >> 6, slot = blockIdx.y;
  const float* p = a.partials + (int64_t)slot * a.n_blocks * a.D + min(col, a.D - 1);
  float s = 0.f;
  int b = split;
  for (; b + 7 * 16 < a.n_blocks; b += 8 * 16) {
    float v[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = p[(int64_t)(b + q * 16) * a.D];
#pragma unroll
    for (int q = 0; q < 8; ++q) s += v[q];
  }
  for (; b < a.n_blocks; b += 16) s += p[(int64_t)b * a.D];
  part[split][threadIdx.x & 63] = s;
  __syncthreads();
  if (split == 0 && col < a.D) {
    s = part[0][threadIdx.x];
#pragma unroll
    for (int w = 1; w < 16; ++w) s += part[w][threadIdx.x];
    a.out[slot][col] = s;
  }
}

// one value: the sum of v[0 .. n) (the gate that is one for all columns)
__global__ __launch_bounds__(256) void sum_kernel(const float* __restrict__ v, int n, float* __restrict__ out) {
  __shared__ float part[4];
  float s = 0.f;
  for (int i = threadIdx.x; i < n; i += 256) s += v[i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) *out = ((part[0] + part[1]) + part[2]) + part[3];
}

// How a row is split: V elements per access (16 bytes; rows shorter than that: 1), CH accesses per lane, tpr lanes per row.  As many
// lanes as the row has accesses up to a wave, then up to 8 elements per lane, then a workgroup of as many waves as that takes (50001 x 1000
// bf16 on two waves 107 / 185 us forward / backward, on four 157 / 245).
struct Split {
  int v, ch, tpr;
  int mode, tail;
};

Split split_of(int64_t D, int vec_width) {
  Split s;
  s.v = D >= vec_width ? vec_width : 1;
  const int64_t n = dh::ceil_div(D, s.v);
  const int64_t eight = 8 / s.v;  // accesses that hold eight elements
  if (n > 64 * eight) {
    s.mode = GROUP;
    s.tpr = 64 * (int)dh::ceil_div(n, 64 * (D > MAX_D ? 2 * eight : eight));  // wide rows: sixteen elements per lane
  } else {
    s.tpr = 8;
    while (s.tpr < 64 && s.tpr < n) s.tpr *= 2;
    s.mode = s.tpr == 64 ? WAVE : SUB;
  }
  s.ch = 1;
  while ((int64_t)s.ch * s.tpr < n) s.ch *= 2;
  s.tail = D % s.v != 0 ? ODD : (int64_t)s.tpr * s.ch == n ? WHOLE : SHORT;
  return s;
}

int64_t rows_per_block(const Split& s) { return s.mode == GROUP ? 1 : 256 / s.tpr; }

// Workgroups of a launch: what the chip holds at a time, so that no second, partly filled round follows (backward, 200003 x 512 bf16: 1024
// workgroups where 768 fit took 398 us instead of 312), and the rows shared out evenly among them.
int64_t even_grid(int64_t M, int64_t per_block, int64_t resident) {
  const int64_t need = dh::ceil_div(M, per_block);
  return need <= resident ? need : dh::ceil_div(need, dh::ceil_div(need, resident));
}

template <class T, int V, int CH, int MODE, bool FULL, int TAIL>
int64_t launch(bool backward, const Args& a, const Split& s, hipStream_t st) {
  const dim3 b(MODE == GROUP ? a.tpr : 256);
  const void* kernel = backward ? reinterpret_cast<const void*>(residual_norm_backward_kernel<T, V, CH, MODE, FULL, TAIL>)
                                : reinterpret_cast<const void*>(residual_norm_forward_kernel<T, V, CH, MODE, FULL, TAIL>);
  static std::atomic<int> per_cu[2][9];  // by direction and waves of a workgroup
  int fit = per_cu[backward][b.x / 64].load(std::memory_order_relaxed);
  if (fit == 0) {
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kernel, (int)b.x, 0) != hipSuccess || fit < 1) {
      (void)hipGetLastError();
      fit = 2;
    }
    per_cu[backward][b.x / 64].store(fit, std::memory_order_relaxed);
  }
  // the forward runs no faster with more than 20 waves on a CU, wide bf16 rows slower (200003 x 512: 174 us with 24, 166 with 20, 185 with 12)
  if (!backward) fit = std::min(fit, 20 / ((int)b.x / 64));
  int64_t resident = (int64_t)256 * fit;
  if (backward && resident > BWD_BLOCKS) resident = BWD_BLOCKS;
  const bool every_row = backward && V * CH > 8;  // wide rows, in two dimensions: one holds less than 2^32 threads
  const int64_t grid = every_row ? std::min<int64_t>(a.M, 1 << 20) : even_grid(a.M, rows_per_block(s), resident);
  const dim3 g((unsigned)grid, every_row ? (unsigned)dh::ceil_div(a.M, grid) : 1u);
  if (backward) hipLaunchKernelGGL((residual_norm_backward_kernel<T, V, CH, MODE, FULL, TAIL>), g, b, 0, st, a);
  else hipLaunchKernelGGL((residual_norm_forward_kernel<T, V, CH, MODE, FULL, TAIL>), g, b, 0, st, a);
  return grid;
}

template <class T, int V, int CH, int MODE, int TAIL>
int64_t launch_gate(bool backward, const Args& a, const Split& s, hipStream_t st) {
  return a.gate_kind == GATE_FULL ? launch<T, V, CH, MODE, true, TAIL>(backward, a, s, st) : launch<T, V, CH, MODE, false, TAIL>(backward, a, s, st);
}
template <class T, int V, int CH, int MODE>
int64_t launch_tail(bool backward, const Args& a, const Split& s, hipStream_t st) {
  if constexpr (V > 1) {
    if (s.tail == ODD) return launch_gate<T, V, CH, MODE, ODD>(backward, a, s, st);
    if (s.tail == WHOLE) return launch_gate<T, V, CH, MODE, WHOLE>(backward, a, s, st);
  }
  return launch_gate<T, V, CH, MODE, SHORT>(backward, a, s, st);
}

// returns the number of workgroups
template <class T>
int64_t launch_t(bool backward, const Args& a, const Split& s, hipStream_t st) {
  constexpr int V = Elem<T>::VEC, EIGHT = 8 / V;
  if (s.v == 1) return launch_tail<T, 1, 1, SUB>(backward, a, s, st);
  if (s.mode == GROUP) return s.ch > EIGHT ? launch_tail<T, V, 2 * EIGHT, GROUP>(backward, a, s, st) : launch_tail<T, V, EIGHT, GROUP>(backward, a, s, st);
  if (s.mode == SUB) return launch_tail<T, V, 1, SUB>(backward, a, s, st);
  if constexpr (EIGHT == 2) {
    if (s.ch == 2) return launch_tail<T, V, 2, WAVE>(backward, a, s, st);
  }
  return launch_tail<T, V, 1, WAVE>(backward, a, s, st);
}

int check_common(const char* me, bool wide, int64_t M, int64_t D, int dtype, const void* f, const void* x, int64_t ldf, int64_t ldx, const void* gate,
                 int64_t ldg, int gate_kind, int gate_sigmoid, int kind, float eps, int has_post, int has_pre) {
  const int64_t least = wide ? MAX_D + 1 : 1, most = wide ? WIDE_D : MAX_D;
  if (M < 0 || D < least || D > most)
    return dh::fail(DH_ERR_INVALID, "%s: %lld rows of %lld columns (%lld .. %lld)", me, (long long)M, (long long)D, (long long)least, (long long)most);
  if (wide && (M > 0x7fffffff || (!has_post && !has_pre))) return dh::fail(DH_ERR_INVALID, "%s: wide rows without a norm, or too many of them", me);
  if (dtype != DH_DTYPE_F32 && dtype != DH_DTYPE_BF16) return dh::fail(DH_ERR_INVALID, "%s: dtype %d", me, dtype);
  if (kind != DH_NORM_LAYER && kind != DH_NORM_RMS) return dh::fail(DH_ERR_INVALID, "%s: norm kind %d", me, kind);
  if (gate_kind < GATE_NONE || gate_kind > GATE_FULL) return dh::fail(DH_ERR_INVALID, "%s: gate kind %d", me, gate_kind);
  if (gate_sigmoid != 0 && gate_sigmoid != 1) return dh::fail(DH_ERR_INVALID, "%s: gate activation %d", me, gate_sigmoid);
  if (!(eps >= 0.f)) return dh::fail(DH_ERR_INVALID, "%s: eps must not be negative", me);
  if (M == 0) return DH_OK;
  if (!f || (gate_kind != GATE_NONE && !gate)) return dh::fail(DH_ERR_INVALID, "%s: null tensor", me);
  if (ldf < D || (x && ldx < D) || (gate_kind == GATE_FULL && ldg < D) || (gate_kind == GATE_ROW && ldg < 1))
    return dh::fail(DH_ERR_INVALID, "%s: leading dimension below the row length", me);
  return DH_OK;
}

int forward(const char* me, bool wide, int64_t M, int64_t D, int dtype, const void* f, int64_t ldf, const void* x, int64_t ldx, const void* gate, int64_t ldg,
            int gate_kind, int gate_sigmoid, float scale, int kind, float eps, int has_post, const float* w1, const float* b1, int has_pre,
            const float* w2, const float* b2, void* r, int64_t ldr, void* h, int64_t ldh, float* stats, dh_stream_t stream) {
  const int rc = check_common(me, wide, M, D, dtype, f, x, ldf, ldx, gate, ldg, gate_kind, gate_sigmoid, kind, eps, has_post, has_pre);
  if (rc != DH_OK) return rc;
  if (M == 0) return DH_OK;
  if ((!r && !has_pre) || (has_pre && !h)) return dh::fail(DH_ERR_INVALID, "%s: null output", me);
  if ((r && ldr < D) || (has_pre && ldh < D)) return dh::fail(DH_ERR_INVALID, "%s: leading dimension below the row length", me);
  if (stats && !dh::aligned16(stats)) return dh::fail(DH_ERR_INVALID, "%s: stats must be 16-byte aligned", me);
  Args a{};
  a.M = M; a.D = (int)D; a.gate_kind = gate_kind; a.gate_sigmoid = gate_sigmoid; a.rms = kind == DH_NORM_RMS;
  a.has_post = has_post != 0; a.has_pre = has_pre != 0; a.scale = scale; a.eps = eps; a.inv_d = 1.f / (float)D;
  a.f = f; a.x = x; a.gate = gate; a.ldf = ldf; a.ldx = ldx; a.ldg = ldg;
  a.w1 = w1; a.b1 = b1; a.w2 = w2; a.b2 = b2; a.stats = stats; a.r = r; a.h = h; a.ldr = ldr; a.ldh = ldh;
  const int vw = dtype == DH_DTYPE_BF16 ? 8 : 4;
  const Split s = split_of(D, vw);
  a.tpr = s.tpr;
  if (dtype == DH_DTYPE_BF16) launch_t<uint16_t>(false, a, s, dh::as_stream(stream));
  else launch_t<float>(false, a, s, dh::as_stream(stream));
  return dh::check_launch(me);
}

// five arrays of one partial row per workgroup, and the per-column sums of a scalar gate
size_t partials_bytes(int64_t M, int64_t D) { return (size_t)(5 * std::min<int64_t>(M, BWD_BLOCKS) + 1) * (size_t)D * 4; }
// and, for wide rows, two numbers of each row behind them
size_t workspace_bytes_of(int64_t M, int64_t D) {
  if (M <= 0 || D <= 0) return 16;
  return D > MAX_D ? (partials_bytes(M, D) + 15) / 16 * 16 + (size_t)M * 8 : partials_bytes(M, D);
}

template <class T>
void launch_columns(const Args& a, int64_t chunks, hipStream_t st) {
  constexpr int V = Elem<T>::VEC;
  const dim3 g((unsigned)dh::ceil_div(dh::ceil_div(a.D, V), 256), (unsigned)chunks), b(256);
  const bool odd = a.D % V != 0, full = a.gate_kind == GATE_FULL;
  if (full && odd) hipLaunchKernelGGL((wide_columns_kernel<T, V, true, ODD>), g, b, 0, st, a);
  else if (full) hipLaunchKernelGGL((wide_columns_kernel<T, V, true, WHOLE>), g, b, 0, st, a);
  else if (odd) hipLaunchKernelGGL((wide_columns_kernel<T, V, false, ODD>), g, b, 0, st, a);
  else hipLaunchKernelGGL((wide_columns_kernel<T, V, false, WHOLE>), g, b, 0, st, a);
}

int backward(const char* me, bool wide, int64_t M, int64_t D, int dtype, const void* f, int64_t ldf, const void* x, int64_t ldx, const void* gate, int64_t ldg,
             int gate_kind, int gate_sigmoid, float scale, int kind, int has_post, const float* w1, const float* b1, int has_pre, const float* w2,
             const float* stats, const void* dr, int64_t lddr, const void* dhh, int64_t lddh, void* df, int64_t lddf, void* dx, int64_t lddx, void* dgate,
             int64_t lddg, float* dw1, float* db1, float* dw2, float* db2, void* workspace, size_t workspace_bytes, dh_stream_t stream) {
  const int rc = check_common(me, wide, M, D, dtype, f, x, ldf, ldx, gate, ldg, gate_kind, gate_sigmoid, kind, 0.f, has_post, has_pre);
  if (rc != DH_OK) return rc;
  if ((!has_post && (dw1 || db1)) || (!has_pre && (dw2 || db2)) || (gate_kind == GATE_NONE && dgate))
    return dh::fail(DH_ERR_INVALID, "%s: the gradient of a parameter that is not there", me);
  hipStream_t st = dh::as_stream(stream);
  const bool col_gate = gate_kind == GATE_CHANNEL || gate_kind == GATE_SCALAR;
  if (M == 0) {  // no rows: the column gradients are empty sums
    for (float* p : {dw1, db1, dw2, db2})
      if (p && dh::zero_async(p, (size_t)D * 4, st) != hipSuccess) return dh::fail(DH_ERR_LAUNCH, "%s: zero fill", me);
    if (col_gate && dgate && dh::zero_async(dgate, (gate_kind == GATE_SCALAR ? 1 : (size_t)D) * 4, st) != hipSuccess)
      return dh::fail(DH_ERR_LAUNCH, "%s: zero fill", me);
    return DH_OK;
  }
  if (!stats) return dh::fail(DH_ERR_INVALID, "%s: null stats", me);
  if (!dh::aligned16(stats)) return dh::fail(DH_ERR_INVALID, "%s: stats must be 16-byte aligned", me);
  if (dhh && !has_pre) return dh::fail(DH_ERR_INVALID, "%s: dh without a second norm", me);
  if (!dr && !dhh) return dh::fail(DH_ERR_INVALID, "%s: no upstream gradient", me);
  if ((dr && lddr < D) || (dhh && lddh < D) || (df && lddf < D) || (dx && lddx < D) || (gate_kind == GATE_FULL && dgate && lddg < D) ||
      (gate_kind == GATE_ROW && dgate && lddg < 1))
    return dh::fail(DH_ERR_INVALID, "%s: leading dimension below the row length", me);
  const size_t need = workspace_bytes_of(M, D);
  if (!workspace || workspace_bytes < need) return dh::fail(DH_ERR_WORKSPACE, "%s: workspace of %zu bytes, need %zu", me, workspace_bytes, need);
  if (wide && !dh::aligned16(workspace)) return dh::fail(DH_ERR_INVALID, "%s: workspace must be 16-byte aligned", me);
  Args a{};
  a.M = M; a.D = (int)D; a.gate_kind = gate_kind; a.gate_sigmoid = gate_sigmoid; a.rms = kind == DH_NORM_RMS;
  a.has_post = has_post != 0; a.has_pre = has_pre != 0; a.scale = scale; a.inv_d = 1.f / (float)D;
  a.f = f; a.x = x; a.gate = gate; a.ldf = ldf; a.ldx = ldx; a.ldg = ldg; a.w1 = w1; a.b1 = b1; a.w2 = w2;
  a.stats = const_cast<float*>(stats); a.dr = dr; a.dh = dhh; a.lddr = lddr; a.lddh = lddh;
  a.df = df; a.dx = dx; a.lddf = lddf; a.lddx = lddx; a.lddg = lddg;
  a.dgate = col_gate ? nullptr : dgate;
  a.partials = static_cast<float*>(workspace);
  a.want_w1 = dw1 != nullptr; a.want_b1 = db1 != nullptr; a.want_w2 = dw2 != nullptr; a.want_b2 = db2 != nullptr;
  a.want_gate = col_gate && dgate;
  const int vw = dtype == DH_DTYPE_BF16 ? 8 : 4;
  const Split s = split_of(D, vw);
  a.tpr = s.tpr;
  const bool columns = a.want_w1 || a.want_b1 || a.want_w2 || a.want_b2 || a.want_gate;
  if (wide && columns) a.terms = reinterpret_cast<float2*>(static_cast<char*>(workspace) + (partials_bytes(M, D) + 15) / 16 * 16);
  int64_t grid = dtype == DH_DTYPE_BF16 ? launch_t<uint16_t>(true, a, s, st) : launch_t<float>(true, a, s, st);
  if (wide && columns) {
    a.rows = dh::ceil_div(M, WIDE_CHUNKS);
    grid = dh::ceil_div(M, a.rows);
    if (dtype == DH_DTYPE_BF16) launch_columns<uint16_t>(a, grid, st);
    else launch_columns<float>(a, grid, st);
  }
  ReduceArgs ra{};
  ra.partials = a.partials; ra.n_blocks = (int)grid; ra.D = (int)D;
  int slots = 0;
  if (a.want_w1) ra.out[slots++] = dw1;
  if (a.want_b1) ra.out[slots++] = db1;
  if (a.want_w2) ra.out[slots++] = dw2;
  if (a.want_b2) ra.out[slots++] = db2;
  float* gate_cols = a.partials + 5 * std::min<int64_t>(M, BWD_BLOCKS) * D;
  if (a.want_gate) ra.out[slots++] = gate_kind == GATE_SCALAR ? gate_cols : static_cast<float*>(dgate);
  if (slots > 0) hipLaunchKernelGGL(column_reduce_kernel, dim3((unsigned)dh::ceil_div(D, 64), (unsigned)slots), dim3(1024), 0, st, ra);
  if (a.want_gate && gate_kind == GATE_SCALAR)
    hipLaunchKernelGGL(sum_kernel, dim3(1), dim3(256), 0, st, gate_cols, (int)D, static_cast<float*>(dgate));
  return dh::check_launch(me);
}

}  // namespace

#define FORWARD_PARAMS                                                                                                                                       \
  int64_t M, int64_t D, int dtype, const void *f, int64_t ldf, const void *x, int64_t ldx, const void *gate, int64_t ldg, int gate_kind, int gate_sigmoid,   \
      float scale, int kind, float eps, int has_post, const float *w1, const float *b1, int has_pre, const float *w2, const float *b2, void *r, int64_t ldr, \
      void *h, int64_t ldh, float *stats, dh_stream_t stream
#define FORWARD_ARGS M, D, dtype, f, ldf, x, ldx, gate, ldg, gate_kind, gate_sigmoid, scale, kind, eps, has_post, w1, b1, has_pre, w2, b2, r, ldr, h, ldh, stats, stream
#define BACKWARD_PARAMS                                                                                                                                      \
  int64_t M, int64_t D, int dtype, const void *f, int64_t ldf, const void *x, int64_t ldx, const void *gate, int64_t ldg, int gate_kind, int gate_sigmoid,   \
      float scale, int kind, int has_post, const float *w1, const float *b1, int has_pre, const float *w2, const float *stats, const void *dr, int64_t lddr, \
      const void *dhh, int64_t lddh, void *df, int64_t lddf, void *dx, int64_t lddx, void *dgate, int64_t lddg, float *dw1, float *db1, float *dw2,          \
      float *db2, void *workspace, size_t workspace_bytes, dh_stream_t stream
#define BACKWARD_ARGS                                                                                                                                        \
  M, D, dtype, f, ldf, x, ldx, gate, ldg, gate_kind, gate_sigmoid, scale, kind, has_post, w1, b1, has_pre, w2, stats, dr, lddr, dhh, lddh, df, lddf, dx,     \
      lddx, dgate, lddg, dw1, db1, dw2, db2, workspace, workspace_bytes, stream

extern "C" int dh_residual_norm_forward(FORWARD_PARAMS) { return forward("dh_residual_norm_forward", false, FORWARD_ARGS); }
extern "C" int dh_residual_norm_wide_forward(FORWARD_PARAMS) { return forward("dh_residual_norm_wide_forward", true, FORWARD_ARGS); }
extern "C" size_t dh_residual_norm_backward_workspace_bytes(int64_t M, int64_t D) { return workspace_bytes_of(M, D); }
extern "C" int dh_residual_norm_backward(BACKWARD_PARAMS) { return backward("dh_residual_norm_backward", false, BACKWARD_ARGS); }
extern "C" int dh_residual_norm_wide_backward(BACKWARD_PARAMS) { return backward("dh_residual_norm_wide_backward", true, BACKWARD_ARGS); }
