// Products grouped by row type with ragged group sizes: one weight per type (tissue, donor, node type), rows sorted by type.
//
//   forward     Y[i] = act(X[i] op(W_g) + b_g)            op(W_g) = W_g^T (W [G][N][K], torch.nn.Linear's layout) or W_g (W [G][K][N])
//   gradient    dX   = the same product with the other op;   dW_g = sum_i dY[i]^T X[i],  db_g = sum_i dY[i]
//   for the rows ptr[g] <= i < ptr[g + 1] of group g.
//
// The bounds ptr stay on the device: no launch depends on their values.  A launch covers every possible raggedness with a closed form of
// them: group g owns the row slots [floor(ptr[g] / R) + g, floor(ptr[g + 1] / R) + g + 1), R rows each, always enough for its
// ceil(len / R) tiles and monotone in g, so a workgroup finds its group with one 64-wide search per 64 groups instead of a prefix sum;
// at most one slot per group and none of the work is wasted on it.
//
// Bound: the matrix cores, and what they wait for at a tile's start and end, for many rows (200003 rows of 9 types, 2000 -> 512 bf16: Y 501 us, dX 616, dW
// and db 476 + 31: 820 / 665 / 860 TFLOP/s, the cores busy 38 / 30 / 40 % of the cycles;
// fp32 100003 rows: 125 / 122 / 134 TFLOP/s), latency for few (16 rows of 8 types, 400 -> 200: 7.3 us; 500 rows of 17 types, forward and all
// gradients: 33 us in four launches).  Four kernels: a tile filled by LDS DMA for aligned operands, one staged through registers for the
// others and for few columns (60000 x 401 -> 203 bf16 169 us for the three products, 97 at 400 -> 200), one of 32 x 32 with K split over the
// waves for few rows, and the weight gradient's, which cuts the rows into chunks of equal work whatever the groups.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.h"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned int u32x4u __attribute__((ext_vector_type(4), aligned(2)));  // 16 bytes at an element's own alignment

__device__ __forceinline__ float bf16_f32(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
// two values rounded to bf16 (v_cvt_pk_bf16_f32: nearest even, a NaN stays one); the rounding in integer arithmetic, eight instructions a
// value, cost a third of a tile's time at K = 512
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
}

// ---- groups --------------------------------------------------------------------------------------------------------------------------
// The bounds with a group of "no weight" in front (rows before ptr[0]) and behind (rows from ptr[G] on): edge(0) = 0, edge(i) = ptr[i - 1],
// edge(G + 2) = M.  Values outside [0, M] are clamped, so a wrong table can cost wrong rows but no access out of bounds.
struct Groups {
  const int32_t* ptr;
  int64_t M;
  int G;
  __device__ __forceinline__ int64_t edge(int i) const {
    if (i <= 0) return 0;
    if (i >= G + 2) return M;
    const int64_t v = ptr[i - 1];
    return v < 0 ? 0 : v > M ? M : v;
  }
  // of an index that all lanes share: a scalar
  __device__ __forceinline__ int64_t shared_edge(int i) const {
    if (i <= 0) return 0;
    if (i >= G + 2) return M;
    const int64_t v = __builtin_amdgcn_readfirstlane(ptr[i - 1]);
    return v < 0 ? 0 : v > M ? M : v;
  }
};

// the last i in [0, n) with key(i) <= s, key non-decreasing and key(0) <= s: 64 probes at a time
template <class Key>
__device__ __forceinline__ int search(int n, int64_t s, Key key) {
  const int lane = threadIdx.x & 63;
  int lo = 0, len = n;
  while (len > 1) {
    const int step = (len + 63) / 64, i = lo + lane * step;
    const bool le = i < lo + len && key(i) <= s;
    const unsigned long long mask = __ballot(le);
    const int last = mask ? 63 - __builtin_clzll(mask) : 0;
    const int next = lo + last * step;
    len = min(step, lo + len - next);
    lo = next;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

struct Slot {
  int group;       // -1: rows that belong to no group
  int64_t begin, end;  // the slot's rows
  bool live;
};

// slot s of R rows (R a power of two: shift)
__device__ __forceinline__ Slot find_slot(const Groups& gr, int64_t s, int shift) {
  const int n = gr.G + 2;
  const int i = search(n, s, [&](int j) { return (gr.edge(j) >> shift) + j; });
  const int64_t a = gr.shared_edge(i), b = gr.shared_edge(i + 1);
  const int64_t first = (a >> shift) + i;
  Slot r;
  r.group = i == 0 || i == n - 1 ? -1 : i - 1;
  r.begin = a + ((s - first) << shift);
  r.end = min(b, r.begin + ((int64_t)1 << shift));
  r.live = s >= first && r.begin < b;
  return r;
}

// the logical number of a workgroup: the dispatcher deals workgroups round robin to the 8 XCDs; handing each XCD a contiguous run keeps
// the tiles that share an operand panel on one L2
__device__ __forceinline__ int xcd_run(int bid, int n) {
  const int q = n / 8, r = n % 8, xcd = bid % 8;
  return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + bid / 8;
}

// ---- operand tiles -------------------------------------------------------------------------------------------------------------------
template <class T>
struct Geo;
template <>
struct Geo<uint16_t> {
  static constexpr int VEC = 8, BK = 64, LD_MK = 72;  // 144-byte rows: the 16-byte fragment reads of 32 rows fall on distinct banks
};
template <>
struct Geo<float> {
  static constexpr int VEC = 4, BK = 32, LD_MK = 36;
};

// The value again, unknown to the compiler: what is computed from it is not kept in registers across the loop over tiles (hoisted, the
// lane-dependent addresses of all phases together spilled 180 registers).
__device__ __forceinline__ int anew(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// R rows (m or n) x BK of an operand.  KM = false: memory is [row][k]; true: [k][row].  Both stay as they lie in memory in LDS too:
// a [k][row] image is read back transposed (bf16: ds_read_b64_tr_b16) or by single elements (fp32).
template <class T, bool KM, int R, int THREADS>
struct Operand {
  static constexpr int VEC = Geo<T>::VEC, BK = Geo<T>::BK;
  // [k][row] images: bf16 rows of R + 32 elements, or 32 (an odd number of 64 bytes: the four k rows that one transposing read takes from
  // lie on distinct banks); fp32 rows of R + 8 (the two half waves read rows 4 apart: 32 banks apart)
  static constexpr int LD = KM ? (sizeof(T) == 2 ? (R == 32 ? R : R + 32) : R + 8) : Geo<T>::LD_MK;
  static constexpr int ELEMS = KM ? BK * LD : R * LD;
  static constexpr int CPR = KM ? R / VEC : 8;                        // 16-byte pieces per image row
  static constexpr int PIECES = (KM ? BK : R) * CPR / THREADS;        // per thread
  static constexpr int ROWS_PER_PASS = THREADS / CPR;
  static_assert(PIECES >= 1 && PIECES * THREADS == (KM ? BK : R) * CPR, "tile does not divide among the threads");

  u32x4 reg[2][PIECES];  // two steps in flight
  const T* p[KM ? 1 : PIECES];  // the lane's pieces of the next step; [k][row] images: the first, the others lie whole rows behind it
  int valid;                    // [k][row] images: values of the pieces below rlim, negative behind it
  bool wide;                    // the memory rows hold a whole piece

  // rows [r0, rlim) of the operand from k0 on, up to k_end.  Rows beyond rlim read some row below it (their products are never stored).
  __device__ __forceinline__ void start(const T* base, int64_t ld, int64_t r0, int64_t rlim, int64_t k0, int64_t k_end) {
    const int tid = threadIdx.x;
    wide = (KM ? rlim : k_end) >= VEC;
    const int ir = tid / CPR, ic = (tid % CPR) * VEC;
    if constexpr (KM) {
      p[0] = base + (k0 + ir) * ld + r0 + ic;
      valid = (int)min((int64_t)VEC, rlim - r0 - ic);
    } else {
#pragma unroll
      for (int q = 0; q < PIECES; ++q) p[q] = base + min(r0 + ir + q * ROWS_PER_PASS, rlim - 1) * ld + k0 + ic;
    }
  }
  // values of the lane's pieces within their memory rows, of a step that has `left` k
  __device__ __forceinline__ int inside(int left) const { return KM ? valid : min(VEC, left - (int)(threadIdx.x % CPR) * VEC); }

  // The next BK of k, of which `left` exist.  FULL: all of them (and for KM all R rows).  Otherwise nothing here is guarded, which would
  // cost a round trip per guard: k rows that do not exist repeat the last one, a piece that passes its memory row's end is fetched from
  // where it just does not, and finish() moves and clears, when the values have arrived.
  template <bool FULL, int U>
  __device__ __forceinline__ void load(int64_t ld, int left) {
    const int tid = anew(threadIdx.x);
#pragma unroll
    for (int q = 0; q < PIECES; ++q) {
      const T* from = KM ? p[0] + q * ROWS_PER_PASS * ld : p[KM ? 0 : q];
      if (!FULL) {
        const int in = inside(left);
        if (KM) from -= max(0, tid / CPR + q * ROWS_PER_PASS - (left - 1)) * ld;
        if (wide) {
          from += min(0, in - VEC);
        } else {  // a memory row shorter than a piece: its values one by one
          T e[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) e[i] = from[min(i, in - 1)];
          __builtin_memcpy(&reg[U][q], e, 16);
        }
      }
      if (FULL || wide) reg[U][q] = *reinterpret_cast<const u32x4u*>(from);
      if (!KM) p[KM ? 0 : q] += BK;
    }
    if (KM) p[0] += BK * ld;
  }
  // the pieces of a step that was not FULL: into place, zeros behind the memory row's end and in k rows that do not exist
  template <int U>
  __device__ __forceinline__ void finish(int left) {
    constexpr int PER = 4 / sizeof(T);  // values of a word
#pragma unroll
    for (int q = 0; q < PIECES; ++q) {
      const int tid = anew(threadIdx.x), in = inside(left), by = wide ? VEC - in : 0;
      const int n = !KM || (int)(tid / CPR) + q * ROWS_PER_PASS < left ? in : 0;
      uint32_t w[4] = {reg[U][q][0], reg[U][q][1], reg[U][q][2], reg[U][q][3]};
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
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t keep = n > e * PER ? 0xffffffffu : 0u;
        if (PER == 2) keep &= n > e * 2 + 1 ? 0xffffffffu : 0xffffu;
        reg[U][q][e] = w[e] & keep;
      }
    }
  }
  template <int U>
  __device__ __forceinline__ void store(T* img) const {
    const int tid = anew(threadIdx.x);
#pragma unroll
    for (int q = 0; q < PIECES; ++q) {
      const int ir = tid / CPR + q * ROWS_PER_PASS, ic = (tid % CPR) * VEC;
      *reinterpret_cast<u32x4*>(img + ir * LD + ic) = reg[U][q];
    }
  }
  // bf16: the 32x32x16 fragment of rows [row, row + 32), k [kk, kk + 16): lane l holds row l & 31, k (l >> 5) * 8 .. + 8
  static __device__ __forceinline__ bf16x8 frag_bf16(const uint16_t* img, int row, int kk) {
    const int lane = threadIdx.x & 63;
    if (!KM) return *reinterpret_cast<const bf16x8*>(img + (row + (lane & 31)) * LD + kk + (lane >> 5) * 8);
    // ds_read_b64_tr_b16: 16 lanes fetch a 4 (k) x 16 (row) block, lane 4 r + c the four elements c of row r, and each receives one column of it
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef s16x4 __attribute__((address_space(3))) * lds_s16x4;
    const int b = lane >> 4, i = lane & 15;
    const uint16_t* p = img + (kk + (b >> 1) * 8 + (i >> 2)) * LD + row + (b & 1) * 16 + (i & 3) * 4;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)p);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(p + 4 * LD));
    bf16x8 f;
    __builtin_memcpy(&f, &lo, 8);
    __builtin_memcpy(reinterpret_cast<char*>(&f) + 8, &hi, 8);
    return f;
  }
  // fp32: k = kk + 4 (lane >> 5) + s for the four 32x32x2 steps s (the same permutation of k on both operands)
  static __device__ __forceinline__ f32x4 frag_f32(const float* img, int row, int kk) {
    const int lane = threadIdx.x & 63, r = row + (lane & 31), k = kk + 4 * (lane >> 5);
    if (!KM) return *reinterpret_cast<const f32x4*>(img + r * LD + k);
    f32x4 f;
#pragma unroll
    for (int s = 0; s < 4; ++s) f[s] = img[(k + s) * LD + r];
    return f;
  }
};

// f(m, n, values) for the elements of a workgroup's accumulators, four consecutive n of a row at a time: the B rows are given as the
// instruction's first operand, so a lane's 32x32 results are row m = lane & 31, n = (r & 3) + 8 (r >> 2) + 4 (lane >> 5), r = 0 .. 15
// (with A first a lane holds 16 rows of one column: four times as many, two-byte, stores)
template <int MI, int NI, int WC, class F>
__device__ __forceinline__ void each4(const f32x16 (&acc)[MI][NI], int64_t m0, int64_t mlim, int64_t n0, int64_t nlim, F&& f) {
  const int tid = anew(threadIdx.x), lane = tid & 63, wave = tid >> 6;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int64_t m = m0 + (wave / WC) * MI * 32 + i * 32 + (lane & 31);
    if (m >= mlim) continue;
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t n = n0 + (wave % WC) * NI * 32 + j * 32 + 8 * q + 4 * (lane >> 5);
        if (n < nlim) f(m, n, f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]});
      }
  }
}

// ---- the tile ------------------------------------------------------------------------------------------------------------------------
// BM x BN of C = A B^T over k: WR x WC waves of MI x NI 32 x 32 accumulators.  Two LDS stages and two register buffers: while the products
// of one step run, the next one's pieces are written and those of the step two behind it are requested.
template <class T, bool A_KM, bool B_KM, int MI, int NI, int WR, int WC>
struct Tile {
  static constexpr int BM = MI * WR * 32, BN = NI * WC * 32, THREADS = WR * WC * 64, BK = Geo<T>::BK;
  typedef Operand<T, A_KM, BM, THREADS> OpA;
  typedef Operand<T, B_KM, BN, THREADS> OpB;
  static constexpr int STAGE = OpA::ELEMS + OpB::ELEMS, LDS_BYTES = 2 * STAGE * (int)sizeof(T);

  f32x16 acc[MI][NI];

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  }
  __device__ __forceinline__ void products(const T* st) {
    const int wave = threadIdx.x >> 6, wm = (wave / WC) * MI * 32, wn = (wave % WC) * NI * 32;
    const T *ia = st, *ib = st + OpA::ELEMS;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int kk = 0; kk < BK; kk += 16) {
        bf16x8 a[MI], b[NI];
#pragma unroll
        for (int i = 0; i < MI; ++i) a[i] = OpA::frag_bf16(ia, wm + i * 32, kk);
#pragma unroll
        for (int j = 0; j < NI; ++j) b[j] = OpB::frag_bf16(ib, wn + j * 32, kk);
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NI; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(b[j], a[i], acc[i][j], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int kk = 0; kk < BK; kk += 8) {
        f32x4 a[MI], b[NI];
#pragma unroll
        for (int i = 0; i < MI; ++i) a[i] = OpA::frag_f32(ia, wm + i * 32, kk);
#pragma unroll
        for (int j = 0; j < NI; ++j) b[j] = OpB::frag_f32(ib, wn + j * 32, kk);
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(b[j][s], a[i][s], acc[i][j], 0, 0, 0);
      }
    }
  }
  // seen(pieces): called with the A operand's pieces of every step (the bias gradient's column sums)
  template <class Seen>
  __device__ __forceinline__ void run(const T* A, int64_t lda, int64_t m0, int64_t mlim, const T* B, int64_t ldb, int64_t n0, int64_t nlim,
                                      int64_t k_begin, int64_t k_end, T* lds, Seen&& seen) {
    zero();
    if (k_end <= k_begin) return;
    const bool whole = (!A_KM || m0 + BM <= mlim) && (!B_KM || n0 + BN <= nlim);
    OpA a;
    OpB b;
    a.start(A, lda, m0, mlim, k_begin, k_end);
    b.start(B, ldb, n0, nlim, k_begin, k_end);
    auto left = [&](int64_t t) { return (int)min((int64_t)BK, k_end - k_begin - t * BK); };
    auto fetch = [&](int64_t t, auto buf) __attribute__((always_inline)) {
      constexpr int U = decltype(buf)::value;
      if (whole && left(t) == BK) {
        a.template load<true, U>(lda, BK);
        b.template load<true, U>(ldb, BK);
      } else {
        a.template load<false, U>(lda, left(t));
        b.template load<false, U>(ldb, left(t));
      }
    };
    auto put = [&](int64_t t, auto buf) __attribute__((always_inline)) {  // the buffer's step t into the stage of the same parity
      constexpr int U = decltype(buf)::value;
      if (!whole || left(t) < BK) {
        a.template finish<U>(left(t));
        b.template finish<U>(left(t));
      }
      a.template store<U>(lds + U * STAGE);
      b.template store<U>(lds + U * STAGE + OpA::ELEMS);
      seen(a.reg[U]);
    };
    typedef std::integral_constant<int, 0> Even;
    typedef std::integral_constant<int, 1> Odd;
    const int64_t steps = (k_end - k_begin + BK - 1) / BK;
    fetch(0, Even{});
    if (steps > 1) fetch(1, Odd{});
    put(0, Even{});
    if (steps > 2) fetch(2, Even{});
    __syncthreads();
    auto step = [&](int64_t t, auto mine, auto other) __attribute__((always_inline)) {
      if (t + 1 < steps) {
        put(t + 1, other);
        if (t + 3 < steps) fetch(t + 3, other);
      }
      products(lds + decltype(mine)::value * STAGE);
      __syncthreads();
    };
    for (int64_t t = 0; t < steps; t += 2) {
      step(t, Even{}, Odd{});
      if (t + 1 < steps) step(t + 1, Odd{}, Even{});
    }
  }
  template <class F>
  __device__ __forceinline__ void each(int64_t m0, int64_t mlim, int64_t n0, int64_t nlim, F&& f) const {
    each4<MI, NI, WC>(acc, m0, mlim, n0, nlim, f);
  }
};

// four consecutive values of a row; n + 4 may pass the row's end
template <bool BF16>
__device__ __forceinline__ void put4(void* row, int64_t n, int64_t nlim, f32x4 v) {
  typedef unsigned int u32x2u __attribute__((ext_vector_type(2), aligned(2)));
  if (BF16) {
    uint16_t* p = static_cast<uint16_t*>(row) + n;
    const u32x2 h = {pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
    if (n + 4 <= nlim) {
      *reinterpret_cast<u32x2u*>(p) = h;
    } else {
      for (int e = 0; e < 3; ++e)
        if (n + e < nlim) p[e] = (uint16_t)(h[e >> 1] >> (16 * (e & 1)));
    }
  } else {
    float* p = static_cast<float*>(row) + n;
    if (n + 4 <= nlim) {
      *reinterpret_cast<f32x4u*>(p) = v;
    } else {
      for (int e = 0; e < 3; ++e)
        if (n + e < nlim) p[e] = v[e];
    }
  }
}

// ---- the tile filled by LDS DMA --------------------------------------------------------------------------------------------------------
// The same product with the operands going from memory to LDS without passing registers (global_load_lds, 16 bytes a lane): what the big
// products run on.  The DMA writes a wave's 64 pieces to 1 KB of LDS in lane order, so images cannot be padded; bank conflicts are avoided by
// choosing WHICH piece a lane fetches: piece c of an image row lies at position c ^ x,
//   [row][k] images (128-byte rows):  x = (row >> 1) & 7: the 16 rows that a 16-byte fragment read takes at a time cover all 16 slots of 256
//                                     bytes;
//   [k][row] images, bf16:            x = (k & 3) << 2: the four k rows that a transposing read takes from lie 64 bytes apart;
//   [k][row] images, fp32:            x = ((k >> 2) & 1) << 3: the half waves read rows 4 apart, in opposite halves of 256 bytes.
// Needs 16-byte aligned rows (address and stride), k counts that are whole pieces where k is contiguous, and for a [k][row] operand whole
// pieces of rows.  In the last, partial step of k the lanes whose pieces lie behind the end fetch a piece of zeros instead.
typedef const __attribute__((address_space(1))) void* global_ptr;
typedef __attribute__((address_space(3))) void* lds_ptr;

__device__ __attribute__((aligned(16))) const uint32_t zero_piece[4] = {0, 0, 0, 0};

// a lane's share of a 32-row fragment: 16 bytes, 8 bf16 or 4 fp32 of k
template <class T>
struct Fragment;
template <>
struct Fragment<uint16_t> {
  typedef bf16x8 Type;
};
template <>
struct Fragment<float> {
  typedef f32x4 Type;
};

template <class T, bool KM, int R, int THREADS>
struct DmaOperand {
  static constexpr int VEC = 16 / sizeof(T), BK = 128 / sizeof(T);  // a step of k is 128 bytes of a [row][k] operand
  static constexpr int CPR = KM ? R / VEC : 8, PIECES = R * 8 / THREADS, ELEMS = R * BK;
  static_assert(PIECES * THREADS == R * 8 && (!KM || R >= (sizeof(T) == 2 ? 128 : 64)), "tile does not divide among the threads");
  typedef typename Fragment<T>::Type Frag;

  const char* base;         // uniform: advances with k
  uint32_t offset[PIECES];  // the lane's pieces, in bytes (a tile spans less than 4 GB: dma_rows)

  static __device__ __forceinline__ int image_row(int q, int tid) { return (q * THREADS + tid) / CPR; }
  static __device__ __forceinline__ int piece(int q, int tid) {
    const int row = image_row(q, tid), c = (q * THREADS + tid) % CPR;
    return c ^ (!KM ? (row >> 1) & 7 : sizeof(T) == 2 ? (row & 3) << 2 : ((row >> 2) & 1) << 3);
  }
  __device__ __forceinline__ void start(const T* op, int64_t ld, int64_t r0, int64_t rlim, int64_t k0) {
    const int tid = anew(threadIdx.x), most = (int)min(rlim - r0, (int64_t)R);
    base = reinterpret_cast<const char*>(op + (KM ? k0 * ld + r0 : r0 * ld + k0));
#pragma unroll
    for (int q = 0; q < PIECES; ++q) {
      if (KM) offset[q] = ((uint32_t)image_row(q, tid) * (uint32_t)ld + (uint32_t)min(piece(q, tid) * VEC, most - VEC)) * (uint32_t)sizeof(T);
      else offset[q] = ((uint32_t)min(image_row(q, tid), most - 1) * (uint32_t)ld + (uint32_t)(piece(q, tid) * VEC)) * (uint32_t)sizeof(T);
    }
  }
  // the next BK of k into an image
  __device__ __forceinline__ void issue(T* img, int64_t ld) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int q = 0; q < PIECES; ++q)
      __builtin_amdgcn_global_load_lds((global_ptr)(base + offset[q]), (lds_ptr)(img + (q * THREADS + wave * 64) * VEC), 16, 0, 0);
    base += (KM ? BK * ld : BK) * (int64_t)sizeof(T);
  }
  // the last `left` < BK of k, zeros behind them
  __device__ __forceinline__ void issue_last(T* img, int left) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), tid = anew(threadIdx.x);
#pragma unroll
    for (int q = 0; q < PIECES; ++q) {
      const int k = KM ? image_row(q, tid) : piece(q, tid) * VEC;
      const void* from = k < left ? static_cast<const void*>(base + offset[q]) : static_cast<const void*>(zero_piece);
      __builtin_amdgcn_global_load_lds((global_ptr)from, (lds_ptr)(img + (q * THREADS + wave * 64) * VEC), 16, 0, 0);
    }
  }
  // the fragment of rows [32 tile, 32 tile + 32), k group g (16 bf16 or 8 fp32): lane l holds row l & 31, the half l >> 5 of the group's k
  static __device__ __forceinline__ Frag frag(const T* img, int tile, int g, int lane) {
    if constexpr (!KM) {
      return *reinterpret_cast<const Frag*>(img + (tile * 32 + (lane & 31)) * BK + (((2 * g + (lane >> 5)) ^ ((lane >> 1) & 7)) * VEC));
    } else if constexpr (sizeof(T) == 2) {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef s16x4 __attribute__((address_space(3))) * lds_s16x4;
      const int b = lane >> 4, i = lane & 15, x = i >> 2;  // x = k & 3 of the lane's row
      const T* at = img + (g * 16 + (b >> 1) * 8 + x) * R + (tile ^ x) * 32 + (b & 1) * 16 + (i & 3) * 4;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)at);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at + 4 * R));
      Frag f;
      __builtin_memcpy(&f, &lo, 8);
      __builtin_memcpy(reinterpret_cast<char*>(&f) + 8, &hi, 8);
      return f;
    } else {
      const int h = lane >> 5;
      const T* at = img + (g * 8 + 4 * h) * R + (tile ^ h) * 32 + (lane & 31);
      return Frag{at[0], at[R], at[2 * R], at[3 * R]};
    }
  }
};

// Every wave's DMA but its last LATER instructions has landed and its image reads are done: the barrier by itself waits for neither.
template <int LATER>
__device__ __forceinline__ void images_ready() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LATER) : "memory");
}

// Between LDS writes of a wave and reads of what its other lanes wrote: the hardware keeps a wave's LDS accesses in order, the compiler is told to.
__device__ __forceinline__ void lanes_exchange() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Schedule of a step: its first fragments are in registers when it begins; the fragments of k group kk + 1 are read while the products of
// group kk run, the barrier that hands over the next image stands in front of the LAST group, and behind it the next step's first fragments
// are read and the image just emptied is requested again, STAGES steps ahead: a wave never waits for LDS with nothing to multiply.
// begin() requests a tile's first steps, main() multiplies, store() writes the result out of an LDS region of its own, so that the next
// tile's begin() runs before this one's store(): with one workgroup on a CU nothing else would fill these gaps (measured in cycles at
// 200003 rows, 2000 -> 512, per tile: first request to first product 8500, 32 steps 107000, stores 16000 before they went out as whole row pieces; dX
// there, 24.7 tiles a CU of eight steps each, takes 1.33 M cycles, of which its steps at that pace are about half).
template <class T, bool A_KM, bool B_KM, int MI, int NI, int WR, int WC>
struct DmaTile {
  static constexpr int STAGES = 2, BM = MI * WR * 32, BN = NI * WC * 32, THREADS = WR * WC * 64, BK = 128 / sizeof(T);
  static constexpr int GROUPS = 4, GK = BK / GROUPS, STEPS_PER_GROUP = sizeof(T) == 2 ? 1 : 4;  // matrix instructions per fragment pair
  typedef DmaOperand<T, A_KM, BM, THREADS> OpA;
  typedef DmaOperand<T, B_KM, BN, THREADS> OpB;
  static constexpr int STAGE = OpA::ELEMS + OpB::ELEMS, OUT = 4096, LDS_BYTES = STAGES * STAGE * (int)sizeof(T) + WR * WC * OUT;
  static constexpr int INSTRS = OpA::PIECES + OpB::PIECES;  // DMA instructions of a wave per step
  static_assert((STAGES - 1) * INSTRS < 64 && GROUPS % 2 == 0, "");
  typedef T Elem;

  struct Source {  // a tile's operands: rows [m0, mlim) of A and [n0, nlim) of B, k in [k_begin, k_end)
    const T *A, *B;
    int64_t lda, ldb, m0, mlim, n0, nlim, k_begin, k_end;
  };

  OpA a;
  OpB b;
  T* lds;
  int64_t lda, ldb, full, steps;
  int left;
  f32x16 acc[MI][NI];
  float row_sum[MI];  // with SUMS: sum over k of the A rows, over the k that this lane's fragments hold

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      row_sum[i] = 0.f;
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    }
  }
  struct Frags {
    typename Fragment<T>::Type a[MI], b[NI];
    __device__ __forceinline__ void read(const T* st, int g, int lane) {
      const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), tm = (wave / WC) * MI, tn = (wave % WC) * NI;
#pragma unroll
      for (int i = 0; i < MI; ++i) a[i] = OpA::frag(st, tm + i, g, lane);
#pragma unroll
      for (int j = 0; j < NI; ++j) b[j] = OpB::frag(st + OpA::ELEMS, tn + j, g, lane);
    }
  };
  template <bool SUMS>
  __device__ __forceinline__ void multiply(const Frags& f) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.b[j], f.a[i], acc[i][j], 0, 0, 0);
    } else {
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NI; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(f.b[j][s], f.a[i][s], acc[i][j], 0, 0, 0);
    }
    if (SUMS) {
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        u32x4 v;
        __builtin_memcpy(&v, &f.a[i], 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (sizeof(T) == 2) row_sum[i] += __uint_as_float(v[e] << 16) + __uint_as_float(v[e] & 0xffff0000u);
          else row_sum[i] += __uint_as_float(v[e]);
        }
      }
    }
  }
  // the LDS reads of one fragment set spread behind the products of a group
  static constexpr int KM_READS = sizeof(T) == 2 ? 2 : 4, READS = (A_KM ? KM_READS : 1) * MI + (B_KM ? KM_READS : 1) * NI;
  static constexpr int PRODUCTS = MI * NI * STEPS_PER_GROUP, PER = (READS + PRODUCTS - 1) / PRODUCTS;
  static __device__ __forceinline__ void interleave() {
#pragma unroll
    for (int i = 0; i < PRODUCTS; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
    }
  }
  __device__ __forceinline__ void issue(int64_t t, T* image) {
    if (t < full) {
      a.issue(image, lda);
      b.issue(image + OpA::ELEMS, ldb);
    } else {
      a.issue_last(image, left);
      b.issue_last(image + OpA::ELEMS, left);
    }
  }
  __device__ __forceinline__ void begin(const Source& s) {
    const int64_t k = s.k_end > s.k_begin ? s.k_end - s.k_begin : 0;
    full = k / BK;
    left = (int)(k % BK);
    steps = full + (left > 0);
    lda = s.lda;
    ldb = s.ldb;
    if (steps == 0) return;
    a.start(s.A, lda, s.m0, s.mlim, s.k_begin);
    b.start(s.B, ldb, s.n0, s.nlim, s.k_begin);
#pragma unroll
    for (int t = 0; t < STAGES; ++t)
      if (t < steps) issue(t, lds + t * STAGE);
  }
  template <bool SUMS>
  __device__ __forceinline__ void main() {
    zero();
    if (steps == 0) return;
    const int lane = anew(threadIdx.x & 63);
    Frags f[2];
    T* image = lds;
    // (whatever was issued after begin() only makes this wait longer)
    if (steps >= STAGES) images_ready<(STAGES - 1) * INSTRS>();
    else images_ready<0>();
    f[0].read(image, 0, lane);
    int64_t t = 0;
    for (; t + 1 < steps; ++t) {
      T* next = image == lds + (STAGES - 1) * STAGE ? lds : image + STAGE;
#pragma unroll
      for (int g = 0; g + 1 < GROUPS; ++g) {
        f[(g + 1) & 1].read(image, g + 1, lane);
        multiply<SUMS>(f[g & 1]);
        interleave();
      }
      // step t + 1 has landed when only the STAGES - 2 steps behind it are outstanding; near the end fewer were requested: wait for all
      if (t + STAGES - 1 < steps) images_ready<(STAGES - 2) * INSTRS>();
      else images_ready<0>();
      if (t + STAGES < steps) issue(t + STAGES, image);
      f[0].read(next, 0, lane);
      multiply<SUMS>(f[1]);
      interleave();
      image = next;
    }
    const int groups = left > 0 ? (left + GK - 1) / GK : GROUPS;
    for (int g = 0; g < groups; ++g) {
      if (g + 1 < groups) f[1].read(image, g + 1, lane);
      multiply<SUMS>(f[0]);
      f[0] = f[1];
    }
    images_ready<0>();  // nobody reads the images any more: the next begin() may overwrite them
  }
  // The tile to memory: base[m * ld + n] = act(accumulator + bias[n]) for m < mlim, n < nlim.  A lane holds four-runs of one row each 8
  // columns apart; written like that, every store instruction scatters 16-byte bits over 32 rows.  Each wave turns 32 rows x 128 bytes at
  // a time in its own 4 KB of LDS (16-byte piece c of row r at c ^ (r >> 1) & 7, as in the images) and stores whole 128-byte row pieces.
  template <bool BF16>
  __device__ __forceinline__ void store(void* base, int64_t ld, int64_t m0, int64_t mlim, int64_t n0, int64_t nlim, const float* bias, bool relu) const {
    constexpr int SIZE = BF16 ? 2 : 4, PER = BF16 && NI > 1 ? 2 : 1;  // accumulator tiles of a 128-byte (one bf16 tile: 64-byte) row piece
    static_assert(NI % PER == 0, "a wave's columns do not divide into row pieces");
    const int lane = anew(threadIdx.x & 63), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    unsigned char* out = reinterpret_cast<unsigned char*>(lds + STAGES * STAGE) + wave * OUT;
    const int r = lane & 31, x = (r >> 1) & 7, h = lane >> 5;
    const int64_t wm = m0 + (wave / WC) * MI * 32, wn = n0 + (wave % WC) * NI * 32;
    const int rows = (int)min((int64_t)(MI * 32), mlim - wm), cols = (int)min((int64_t)(NI * 32), nlim - wn);  // of the wave's part; <= 0: none
    unsigned char* const origin = static_cast<unsigned char*>(base) + (wm * ld + wn) * SIZE;
    if (rows <= 0 || cols <= 0) return;
#pragma unroll
    for (int jj = 0; jj < NI; jj += PER) {
      if (jj * 32 >= cols) continue;
      f32x4 add[PER][4];
      if (bias) {
#pragma unroll
        for (int j = 0; j < PER; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int n = (jj + j) * 32 + 8 * q + 4 * h;
#pragma unroll
            for (int e = 0; e < 4; ++e) add[j][q][e] = bias[wn + min(n + e, cols - 1)];
          }
      }
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        if (i * 32 >= rows) continue;
#pragma unroll
        for (int j = 0; j < PER; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            f32x4 v = {acc[i][jj + j][4 * q], acc[i][jj + j][4 * q + 1], acc[i][jj + j][4 * q + 2], acc[i][jj + j][4 * q + 3]};
            if (bias) v += add[j][q];
            if (relu) {
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] = v[e] < 0.f ? 0.f : v[e];  // (a NaN passes)
            }
            const int col = j * 32 + 8 * q + 4 * h;
            if (BF16) *reinterpret_cast<u32x2*>(out + r * 128 + (((col >> 3) ^ x) << 4) + (col & 4) * 2) = u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
            else *reinterpret_cast<f32x4*>(out + r * 128 + (((col >> 2) ^ x) << 4)) = v;
          }
        lanes_exchange();
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          const int row = it * 8 + (lane >> 3), c = lane & 7, m = i * 32 + row, n = jj * 32 + c * (16 / SIZE);
          const u32x4 v = *reinterpret_cast<const u32x4*>(out + row * 128 + ((c ^ ((row >> 1) & 7)) << 4));
          if (m < rows && n < cols) {
            unsigned char* to = origin + (int64_t)m * ld * SIZE + n * SIZE;
            if (n + 16 / SIZE <= cols) {
              *reinterpret_cast<u32x4u*>(to) = v;
            } else {
              for (int e = 0; e < 16 / SIZE - 1; ++e) {
                if (n + e >= cols) break;
                if (BF16) reinterpret_cast<uint16_t*>(to)[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
                else reinterpret_cast<uint32_t*>(to)[e] = v[e];
              }
            }
          }
        }
        lanes_exchange();  // the next rows are written over these
      }
    }
  }
  // put(row of the tile, its sum): the waves of the first tile column hold every row, the two half waves half of its k each
  template <class Put>
  __device__ __forceinline__ void row_sums(Put&& put) const {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const float v = row_sum[i] + __shfl_xor(row_sum[i], 32);
      if (wave % WC == 0 && lane < 32) put((wave / WC) * MI * 32 + i * 32 + lane, v);
    }
  }
};

// ---- forward (and dX) ----------------------------------------------------------------------------------------------------------------
struct FwdArgs {
  Groups gr;
  int64_t N, K;
  const void *X, *W;
  int64_t ldx, ldw, stride_w;
  const float* bias;  // [G][N]
  int64_t ld_bias;
  void* Y;
  int64_t ldy;
  int act, y_bf16, zero_outside;
};

// tile `id` of the launch: its row slot and first column; false where there is nothing to write
template <class TileT>
__device__ __forceinline__ bool forward_tile(const FwdArgs& a, int id, int tiles_n, Slot& s, int64_t& n0) {
  const int slot = __builtin_amdgcn_readfirstlane(id / tiles_n);
  s = find_slot(a.gr, slot, __builtin_ctz(TileT::BM));
  n0 = (int64_t)(id - slot * tiles_n) * TileT::BN;
  return s.live && (s.group >= 0 || a.zero_outside);
}

template <class T, class TileT>
__global__ __launch_bounds__(TileT::THREADS, 2) void grouped_forward_kernel(const FwdArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char raw_lds[];
  const int tiles_n = (int)((a.N + TileT::BN - 1) / TileT::BN);
  Slot s;
  int64_t n0;
  if (!forward_tile<TileT>(a, xcd_run(blockIdx.x, gridDim.x), tiles_n, s, n0)) return;
  TileT t;
  const float* bias = nullptr;
  if (s.group < 0) {
    t.zero();
  } else {
    t.run(static_cast<const T*>(a.X), a.ldx, s.begin, s.end, static_cast<const T*>(a.W) + s.group * a.stride_w, a.ldw, n0, a.N, 0, a.K,
          reinterpret_cast<T*>(raw_lds), [](const auto&) {});
    if (a.bias) bias = a.bias + s.group * a.ld_bias;
  }
  const bool relu = s.group >= 0 && a.act == DH_ACT_RELU;
  t.each(s.begin, s.end, n0, a.N, [&](int64_t m, int64_t n, f32x4 v) __attribute__((always_inline)) {
    if (bias) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += bias[min(n + e, a.N - 1)];
    }
    if (relu) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = v[e] < 0.f ? 0.f : v[e];  // (a NaN passes)
    }
    if (a.y_bf16) put4<true>(static_cast<uint16_t*>(a.Y) + m * a.ldy, n, a.N, v);
    else put4<false>(static_cast<float*>(a.Y) + m * a.ldy, n, a.N, v);
  });
}

// As many workgroups as the chip holds; each walks the tiles l, l + L, l + 2 L ... of its XCD's contiguous run, L workgroups on that XCD.
template <class TileT>
__global__ __launch_bounds__(TileT::THREADS, 2) void grouped_forward_dma_kernel(const FwdArgs a, int n_tiles) {
  typedef typename TileT::Elem T;
  extern __shared__ __attribute__((aligned(16))) unsigned char raw_lds[];
  const int tiles_n = (int)((a.N + TileT::BN - 1) / TileT::BN);
  const int xcd = blockIdx.x % 8, q = n_tiles / 8, rest = n_tiles % 8;
  const int run = xcd < rest ? xcd * (q + 1) : rest * (q + 1) + (xcd - rest) * q, stop = run + (xcd < rest ? q + 1 : q), step = (gridDim.x + 7 - xcd) / 8;
  int id = run + blockIdx.x / 8;
  TileT t;
  t.lds = reinterpret_cast<T*>(raw_lds);
  auto advance = [&](Slot& s, int64_t& n0) __attribute__((always_inline)) {  // the next tile with something to write
    for (; id < stop; id += step)
      if (forward_tile<TileT>(a, id, tiles_n, s, n0)) {
        id += step;
        return true;
      }
    return false;
  };
  auto begin = [&](const Slot& s, int64_t n0) __attribute__((always_inline)) {
    t.begin({static_cast<const T*>(a.X), static_cast<const T*>(a.W) + (s.group < 0 ? 0 : s.group * a.stride_w), a.ldx, a.ldw, s.begin,
             s.end, n0, a.N, 0, s.group < 0 ? 0 : a.K});
  };
  Slot s, ns;
  int64_t n0, nn0 = 0;
  if (!advance(s, n0)) return;
  begin(s, n0);
  bool more = advance(ns, nn0);
  while (true) {
    t.template main<false>();
    if (more) begin(ns, nn0);
    const float* bias = a.bias && s.group >= 0 ? a.bias + s.group * a.ld_bias : nullptr;
    const bool relu = s.group >= 0 && a.act == DH_ACT_RELU;
    if (a.y_bf16) t.template store<true>(a.Y, a.ldy, s.begin, s.end, n0, a.N, bias, relu);
    else t.template store<false>(a.Y, a.ldy, s.begin, s.end, n0, a.N, bias, relu);
    if (!more) return;
    s = ns;
    n0 = nn0;
    more = advance(ns, nn0);
  }
}

// ---- few rows: K split over the waves -------------------------------------------------------------------------------------------------
// A 32 x 32 tile per workgroup, its K cut into one contiguous piece per wave: every wave requests the fragments of up to BATCH k groups
// straight into registers before it multiplies the first, so a whole product of K <= 8 waves x BATCH groups costs one round trip to memory
// where the staged tile pays one per step (16 rows of 8 types, 400 -> 200 fp32: 14.7 us staged).  The waves' partial tiles are added in LDS
// in wave order.  Bound: latency, then the L1 (every 2 KB of fragments feeds one or four matrix instructions).
template <class T, bool W_KM>
struct SmallFrags {
  static constexpr int KG = sizeof(T) == 2 ? 16 : 8, PER = KG / 2, BATCH = 4;  // k per group, per lane, groups in flight
  T a[BATCH][PER], b[BATCH][PER];

  static __device__ __forceinline__ void vec(T (&to)[PER], const T* p) {
    const u32x4 v = *reinterpret_cast<const u32x4u*>(p);
    __builtin_memcpy(to, &v, 16);
  }
  // groups [g, g + BATCH) below g_end; xr: the lane's row of X, w: its row (or, W_KM, column) of W
  __device__ __forceinline__ void load(const T* xr, const T* w, int64_t ldw, int g, int g_end, int64_t K, int half) {
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int64_t k = (int64_t)min(g + u, g_end - 1) * KG + half * PER;
      const int64_t whole = (int64_t)min(g + u, g_end - 1) * KG + KG;
      if (whole <= K) {  // uniform
        vec(a[u], xr + k);
        if (!W_KM) vec(b[u], w + k);
        else {
#pragma unroll
          for (int e = 0; e < PER; ++e) b[u][e] = w[(k + e) * ldw];
        }
      } else {
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          const int64_t c = min(k + e, K - 1);
          const T av = xr[c], bv = W_KM ? w[c * ldw] : w[c];
          a[u][e] = k + e < K ? av : T(0);
          b[u][e] = k + e < K ? bv : T(0);
        }
      }
    }
  }
  __device__ __forceinline__ void multiply(f32x16& acc, int g, int g_end) const {
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      if (g + u >= g_end) continue;  // uniform
      if constexpr (sizeof(T) == 2) {
        bf16x8 fa, fb;
        __builtin_memcpy(&fa, a[u], 16);
        __builtin_memcpy(&fb, b[u], 16);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fb, fa, acc, 0, 0, 0);
      } else {
#pragma unroll
        for (int e = 0; e < PER; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(b[u][e], a[u][e], acc, 0, 0, 0);
      }
    }
  }
};

template <class T, bool W_KM>
__global__ __launch_bounds__(512) void grouped_small_kernel(const FwdArgs a) {
  typedef SmallFrags<T, W_KM> Frags;
  __shared__ __attribute__((aligned(16))) float part[8][32][36];
  const int tiles_n = (int)((a.N + 31) / 32), id = xcd_run(blockIdx.x, gridDim.x), slot = __builtin_amdgcn_readfirstlane(id / tiles_n);
  const Slot s = find_slot(a.gr, slot, 5);
  const int64_t n0 = (int64_t)(id - slot * tiles_n) * 32;
  if (!s.live || (s.group < 0 && !a.zero_outside)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, half = lane >> 5;
  f32x16 acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.f;
  if (s.group >= 0 && a.K > 0) {
    const int groups = (int)((a.K + Frags::KG - 1) / Frags::KG), per = (groups + waves - 1) / waves, g_end = min(groups, (wave + 1) * per);
    const T* xr = static_cast<const T*>(a.X) + min(s.begin + (lane & 31), s.end - 1) * a.ldx;
    const int64_t n = min(n0 + (lane & 31), a.N - 1);
    const T* w = static_cast<const T*>(a.W) + s.group * a.stride_w + (W_KM ? n : n * a.ldw);
    int g = wave * per;
    if (g < g_end) {
      Frags f[2];
      f[0].load(xr, w, a.ldw, g, g_end, a.K, half);
      for (; g < g_end; g += 2 * Frags::BATCH) {  // two batches in flight
        if (g + Frags::BATCH < g_end) f[1].load(xr, w, a.ldw, g + Frags::BATCH, g_end, a.K, half);
        f[0].multiply(acc, g, g_end);
        if (g + 2 * Frags::BATCH < g_end) f[0].load(xr, w, a.ldw, g + 2 * Frags::BATCH, g_end, a.K, half);
        if (g + Frags::BATCH < g_end) f[1].multiply(acc, g + Frags::BATCH, g_end);
      }
    }
  }
#pragma unroll
  for (int q = 0; q < 4; ++q)  // the lane's row, columns 8 q + 4 half .. + 4
    *reinterpret_cast<f32x4*>(&part[wave][lane & 31][8 * q + 4 * half]) = f32x4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
  __syncthreads();
  const float* bias = a.bias && s.group >= 0 ? a.bias + s.group * a.ld_bias : nullptr;
  const bool relu = s.group >= 0 && a.act == DH_ACT_RELU;
  for (int i = threadIdx.x; i < 32 * 8; i += blockDim.x) {
    const int64_t m = s.begin + (i >> 3), n = n0 + (i & 7) * 4;
    if (m >= s.end || n >= a.N) continue;
    f32x4 v = *reinterpret_cast<const f32x4*>(&part[0][i >> 3][(i & 7) * 4]);
    for (int w = 1; w < waves; ++w) v += *reinterpret_cast<const f32x4*>(&part[w][i >> 3][(i & 7) * 4]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (bias) v[e] += bias[min(n + e, a.N - 1)];
      if (relu) v[e] = v[e] < 0.f ? 0.f : v[e];  // (a NaN passes)
    }
    if (a.y_bf16) put4<true>(static_cast<uint16_t*>(a.Y) + m * a.ldy, n, a.N, v);
    else put4<false>(static_cast<float*>(a.Y) + m * a.ldy, n, a.N, v);
  }
}

// ---- dW, db --------------------------------------------------------------------------------------------------------------------------
// dW_g [N][K] = sum over the group's rows of dY[i, n] X[i, k]: both operands [k][row] images with the rows as the contraction.  The rows are
// cut into chunks of equal work whatever the groups: a workgroup takes one tile of dW through one chunk, group by group.  A group costs its
// rows and, for the start and the end of its tile, about as much as GROUP_ROWS rows: row r of group g lies at position r + g GROUP_ROWS of a
// line that is cut into equal pieces, a closed form of the bounds again (27630 rows of 476 types, 560 -> 16 bf16: 107 us with pieces of equal
// rows, 40 so; 52 with 32 positions for a group, 46 with 128).  A group that lies inside a chunk is finished in place; of one that spans
// several, chunk c holds either its beginning (partial slot 2 c) or a later part that starts with the chunk (slot 2 c + 1; never two of a
// kind), which wgrad_join_kernel adds in chunk order (no atomics).  The zeros of empty groups are written by workgroups of their own, the
// first `zeroers` of the launch.
constexpr int GROUP_ROWS = 64;

struct WgradArgs {
  Groups gr;
  int64_t N, K;
  const void *dY, *X;
  int64_t ldy, ldx;
  void* dW;
  int64_t ldw, stride_w;
  int dw_bf16;
  float* db;  // [G][N] or null
  int64_t ld_db;
  float* part_w;  // [2 chunks][N][K]
  float* part_b;  // [2 chunks][N]
  int64_t chunk, chunks;  // positions of a chunk
  int tiles_k, tiles;
  int zeroers;  // a multiple of the XCDs: the other workgroups keep their places
  int slices;
};

struct WgradTile {
  int chunk, n, k;
};
__device__ __forceinline__ WgradTile wgrad_tile(const WgradArgs& a) {  // of this workgroup, scalars
  const int id = xcd_run(blockIdx.x - a.zeroers, gridDim.x - a.zeroers), chunk = __builtin_amdgcn_readfirstlane(id / a.tiles), tile = id - chunk * a.tiles;
  const int n = __builtin_amdgcn_readfirstlane(tile / a.tiles_k);
  return {chunk, n, tile - n * a.tiles_k};
}

// where a group (of those with the two groups of no weight) begins on the line; the group at position s; the first row at s or behind it
__device__ __forceinline__ int64_t place_of(int i, int64_t start) { return start + (int64_t)max(i - 1, 0) * GROUP_ROWS; }
__device__ __forceinline__ int group_at(const Groups& gr, int64_t s) {
  return search(gr.G + 2, s, [&](int j) { return place_of(j, gr.edge(j)); });
}
__device__ __forceinline__ int64_t row_at(const Groups& gr, int64_t s) {
  const int i = group_at(gr, s);
  const int64_t start = gr.shared_edge(i);
  return min(start + max((int64_t)0, s - place_of(i, start)), gr.shared_edge(i + 1));
}

struct Segment {  // the rows [begin, end) of a group inside a chunk
  int group;
  int64_t begin, end;
  int64_t slot;  // partial slot, -1: the whole group
};

// Walks the groups of chunk c, from row to row: empty ones cost nothing.
struct Segments {
  const WgradArgs& a;
  int64_t c, first, last;  // rows [first, last)
  int64_t at;              // the next row

  __device__ __forceinline__ Segments(const WgradArgs& args, int64_t chunk_id) : a(args), c(chunk_id) {
    first = at = row_at(a.gr, c * a.chunk);
    last = row_at(a.gr, (c + 1) * a.chunk);
  }
  __device__ __forceinline__ bool next(Segment& s) {
    while (at < last) {
      const int64_t from = at;
      const int i = search(a.gr.G + 2, from, [&](int j) { return a.gr.edge(j); });  // holds row `from`
      const int64_t b = a.gr.shared_edge(i), e = a.gr.shared_edge(i + 1);
      if (e <= from) return false;  // (bounds that decrease)
      at = min(e, last);
      if (i == 0) continue;  // rows before the first group
      if (i == a.gr.G + 1) return false;
      s = {i - 1, from, at, b >= first && e <= last ? -1 : b >= first ? 2 * c : 2 * c + 1};
      return true;
    }
    return false;
  }
};

// dW, db of the empty groups: every group cut into `slices` runs of rows, run u of group g written by workgroup (g slices + u) mod zeroers
__device__ void write_empty_groups(const WgradArgs& a, int part) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t units = (int64_t)a.gr.G * a.slices;
  for (int64_t base = part; base < units; base += (int64_t)a.zeroers * 64) {
    const int64_t unit = base + (int64_t)lane * a.zeroers;
    const int g = (int)(min(unit, units - 1) / a.slices);
    for (unsigned long long empty = __ballot(unit < units && a.gr.edge(g + 2) <= a.gr.edge(g + 1)); empty; empty &= empty - 1) {
      const int64_t mine = base + (int64_t)__builtin_ctzll(empty) * a.zeroers, group = mine / a.slices, u = mine - group * a.slices;
      char* to = static_cast<char*>(a.dW) + group * a.stride_w * (a.dw_bf16 ? 2 : 4);
      const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
      const int pieces = (int)min((a.K + 3) / 4, (int64_t)blockDim.x), rows = blockDim.x / pieces, r = tid / pieces, c = tid % pieces;
      const int64_t end = (u + 1) * a.N / a.slices;
      for (int64_t n = u * a.N / a.slices + r; r < rows && n < end; n += rows)
        for (int64_t k = (int64_t)c * 4; k < a.K; k += (int64_t)blockDim.x * 4) {
          if (a.dw_bf16) put4<true>(reinterpret_cast<uint16_t*>(to) + n * a.ldw, k, a.K, zero);
          else put4<false>(reinterpret_cast<float*>(to) + n * a.ldw, k, a.K, zero);
        }
      if (a.db && u == 0)
        for (int64_t n = tid; n < a.N; n += blockDim.x) a.db[group * a.ld_db + n] = 0.f;
    }
  }
}

// where a segment's result goes
struct WgradOut {
  void* to;
  int64_t ld;
  float* sums;
  bool bf16;
};
__device__ __forceinline__ WgradOut wgrad_out(const WgradArgs& a, const Segment& s) {
  if (s.slot >= 0) return {a.part_w + s.slot * a.N * a.K, a.K, a.part_b + s.slot * a.N, false};
  return {static_cast<char*>(a.dW) + s.group * a.stride_w * (a.dw_bf16 ? 2 : 4), a.ldw, a.db ? a.db + s.group * a.ld_db : nullptr, a.dw_bf16 != 0};
}

template <class T, class TileT>
__global__ __launch_bounds__(TileT::THREADS, 2) void grouped_wgrad_kernel(const WgradArgs a) {
  typedef typename TileT::OpA OpA;
  extern __shared__ __attribute__((aligned(16))) unsigned char raw_lds[];
  if ((int)blockIdx.x < a.zeroers) return write_empty_groups(a, blockIdx.x);
  const WgradTile w = wgrad_tile(a);
  const int64_t n0 = (int64_t)w.n * TileT::BM, k0 = (int64_t)w.k * TileT::BN;
  const bool sums = a.db && k0 == 0;
  constexpr int VEC = Geo<T>::VEC;
  Segments walk(a, w.chunk);
  Segment s;
  while (walk.next(s)) {
    TileT t;
    float cs[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) cs[e] = 0.f;
    t.run(static_cast<const T*>(a.dY), a.ldy, n0, a.N, static_cast<const T*>(a.X), a.ldx, k0, a.K, s.begin, s.end, reinterpret_cast<T*>(raw_lds),
          [&](const u32x4(&reg)[OpA::PIECES]) __attribute__((always_inline)) {
            if (!sums) return;
#pragma unroll
            for (int q = 0; q < OpA::PIECES; ++q) {
              T e[VEC];
              __builtin_memcpy(e, &reg[q], 16);
#pragma unroll
              for (int i = 0; i < VEC; ++i) {
                if constexpr (sizeof(T) == 2) cs[i] += bf16_f32(e[i]);
                else cs[i] += e[i];
              }
            }
          });
    const WgradOut o = wgrad_out(a, s);
    t.each(n0, a.N, k0, a.K, [&](int64_t n, int64_t k, f32x4 v) __attribute__((always_inline)) {
      if (o.bf16) put4<true>(static_cast<uint16_t*>(o.to) + n * o.ld, k, a.K, v);
      else put4<false>(static_cast<float*>(o.to) + n * o.ld, k, a.K, v);
    });
    if (sums) {  // thread t summed columns (t % CPR) * VEC of the rows it staged
      float* lds = reinterpret_cast<float*>(raw_lds);
      __syncthreads();
      constexpr int LD = TileT::BM + 4;
      const int rg = threadIdx.x / OpA::CPR, c = (threadIdx.x % OpA::CPR) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) lds[rg * LD + c + e] = cs[e];
      __syncthreads();
      for (int i = threadIdx.x; i < TileT::BM; i += TileT::THREADS) {
        float v = 0.f;
        for (int r = 0; r < OpA::ROWS_PER_PASS; ++r) v += lds[r * LD + i];
        if (n0 + i < a.N) o.sums[n0 + i] = v;
      }
    }
    __syncthreads();  // the next segment's images
  }
}

template <class TileT, bool SUMS>
__device__ __forceinline__ void wgrad_dma(const WgradArgs& a, int64_t c, int64_t n0, int64_t k0, typename TileT::Elem* lds) {
  typedef typename TileT::Elem T;
  TileT t;
  t.lds = lds;
  auto begin = [&](const Segment& s) __attribute__((always_inline)) {
    t.begin({static_cast<const T*>(a.dY), static_cast<const T*>(a.X), a.ldy, a.ldx, n0, a.N, k0, a.K, s.begin, s.end});
  };
  Segments walk(a, c);
  Segment s, ns;
  if (!walk.next(s)) return;
  begin(s);
  bool more = walk.next(ns);
  while (true) {
    t.template main<SUMS>();
    if (more) begin(ns);
    const WgradOut o = wgrad_out(a, s);
    if (o.bf16) t.template store<true>(o.to, o.ld, n0, a.N, k0, a.K, nullptr, false);
    else t.template store<false>(o.to, o.ld, n0, a.N, k0, a.K, nullptr, false);
    if (SUMS)
      t.row_sums([&](int i, float v) __attribute__((always_inline)) {
        if (n0 + i < a.N) o.sums[n0 + i] = v;
      });
    if (!more) return;
    s = ns;
    more = walk.next(ns);
  }
}

template <class TileT>
__global__ __launch_bounds__(TileT::THREADS, 2) void grouped_wgrad_dma_kernel(const WgradArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char raw_lds[];
  if ((int)blockIdx.x < a.zeroers) return write_empty_groups(a, blockIdx.x);
  const WgradTile w = wgrad_tile(a);
  const int64_t n0 = (int64_t)w.n * TileT::BM, k0 = (int64_t)w.k * TileT::BN;
  if (a.db && w.k == 0) wgrad_dma<TileT, true>(a, w.chunk, n0, k0, reinterpret_cast<typename TileT::Elem*>(raw_lds));
  else wgrad_dma<TileT, false>(a, w.chunk, n0, k0, reinterpret_cast<typename TileT::Elem*>(raw_lds));
}

// The parts of every group that spans chunks.  blockIdx.y = c: the group that begins in chunk c and reaches beyond it, if there is one, lies
// at the chunk's last position.
__global__ __launch_bounds__(256) void wgrad_join_kernel(const WgradArgs a) {
  const int64_t c0 = blockIdx.y, next = (c0 + 1) * a.chunk;
  const int i = group_at(a.gr, next - 1);
  const int64_t start = a.gr.shared_edge(i), end = a.gr.shared_edge(i + 1), place = place_of(i, start);
  if (i == 0 || i == a.gr.G + 1 || place < c0 * a.chunk || place > next - 1 || end - start <= next - place) return;
  const int group = i - 1, parts = (int)((place + end - 1 - start) / a.chunk - c0);  // later ones
  const int64_t nk = a.N * a.K, at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  // four consecutive values of the parts' sum; part c > 0: slot 2 (c0 + c) + 1; eight in flight, past the last one it is read again and not added
  auto joined = [&](const float* p, int64_t step, int64_t count) __attribute__((always_inline)) {
    p += 2 * c0 * step;
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = p[min((int64_t)e, count - 1)];
    for (int c = 1; c <= parts; c += 8) {
      f32x4 t[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float* from = p + (2 * (int64_t)min(c + u, parts) + 1) * step;
        if (count >= 4) {
          t[u] = *reinterpret_cast<const f32x4u*>(from);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) t[u][e] = from[min((int64_t)e, count - 1)];
        }
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (c + u <= parts) v += t[u];
    }
    return v;
  };
  if (at < nk) {
    const f32x4 v = joined(a.part_w + at, nk, nk - at);
    void* to = static_cast<char*>(a.dW) + group * a.stride_w * (a.dw_bf16 ? 2 : 4);
    int64_t n = nk <= 0xffffffffll ? (int64_t)((uint32_t)at / (uint32_t)a.K) : at / a.K, k = at - n * a.K;
    if (k + 4 <= a.K || n + 1 == a.N) {
      if (a.dw_bf16) put4<true>(static_cast<uint16_t*>(to) + n * a.ldw, k, a.K, v);
      else put4<false>(static_cast<float*>(to) + n * a.ldw, k, a.K, v);
    } else {  // the four pass the end of a row
      for (int e = 0; e < 4 && n < a.N; ++e) {
        if (a.dw_bf16) static_cast<uint16_t*>(to)[n * a.ldw + k] = (uint16_t)pack_bf16(v[e], 0.f);
        else static_cast<float*>(to)[n * a.ldw + k] = v[e];
        if (++k == a.K) {
          k = 0;
          ++n;
        }
      }
    }
  }
  if (a.db && at < a.N) put4<false>(a.db + group * a.ld_db, at, a.N, joined(a.part_b + at, a.N, a.N - at));
}

// ---- host ----------------------------------------------------------------------------------------------------------------------------
constexpr int64_t MAX_GRID = 0x7fffffff;

constexpr int CUS = 256;
// Few columns: tiles 32 wide.  Forward, 60833 rows of 172 types 937 -> 12: bf16 31 us against 62 of the 128-wide tile, fp32 78 against 267; 60000 of
// 9 types 400 -> 32, aligned: 14.1 / 14.9 and 32 / 38; two of them for 64 columns: 24.3 / 15.6 and 60 / 38.  Weight gradient, staged: the first 49
// / 67 and 125 / 182; against the DMA tile, 400 -> 32: 21.5 / 19.4 and 43 / 39, so only where that cannot be used.
constexpr int NARROW = 32;

// Raises a kernel's dynamic LDS limit, once per device: `done` is the kernel's own mask of devices.
int allow_lds(const char* me, const void* kernel, int bytes, std::atomic<uint64_t>& done) {
  int device = 0;
  if (hipGetDevice(&device) != hipSuccess) return dh::fail(DH_ERR_NO_DEVICE, "%s: no device", me);
  const uint64_t bit = 1ull << (device & 63);
  if (done.load(std::memory_order_relaxed) & bit) return DH_OK;
  const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) return dh::fail(DH_ERR_LAUNCH, "%s: %d bytes of LDS: %s", me, bytes, hipGetErrorString(e));
  done.fetch_or(bit, std::memory_order_relaxed);
  return DH_OK;
}

template <class T, class TileT>
int forward_launch(const char* me, const FwdArgs& a, hipStream_t st) {
  const int64_t grid = (a.gr.M / TileT::BM + a.gr.G + 2) * dh::ceil_div(a.N, TileT::BN);
  if (grid > MAX_GRID) return dh::fail(DH_ERR_INVALID, "%s: %lld tiles in one launch", me, (long long)grid);
  static std::atomic<uint64_t> done{0};
  const int allowed = allow_lds(me, reinterpret_cast<const void*>(grouped_forward_kernel<T, TileT>), TileT::LDS_BYTES, done);
  if (allowed != DH_OK) return allowed;
  hipLaunchKernelGGL((grouped_forward_kernel<T, TileT>), dim3((unsigned)grid), dim3(TileT::THREADS), TileT::LDS_BYTES, st, a);
  return dh::check_launch(me);
}

template <class TileT>
int forward_dma_launch(const char* me, const FwdArgs& a, hipStream_t st) {
  const int64_t tiles = (a.gr.M / TileT::BM + a.gr.G + 2) * dh::ceil_div(a.N, TileT::BN);
  const int64_t resident = (int64_t)CUS * (160 * 1024 / TileT::LDS_BYTES);
  if (tiles > MAX_GRID - resident) return dh::fail(DH_ERR_INVALID, "%s: %lld tiles in one launch", me, (long long)tiles);
  static std::atomic<uint64_t> done{0};
  const int allowed = allow_lds(me, reinterpret_cast<const void*>(grouped_forward_dma_kernel<TileT>), TileT::LDS_BYTES, done);
  if (allowed != DH_OK) return allowed;
  hipLaunchKernelGGL((grouped_forward_dma_kernel<TileT>), dim3((unsigned)(tiles < resident ? tiles : resident)), dim3(TileT::THREADS), TileT::LDS_BYTES, st,
                     a, (int)tiles);
  return dh::check_launch(me);
}

// whole 16-byte pieces: address, row stride; and a tile (256 rows) within the 32-bit byte offsets of its lanes
bool dma_rows(const void* p, int64_t ld, int vec) { return dh::aligned16(p) && ld % vec == 0 && ld < (1 << 21); }

template <class T, bool W_KM>
int small_launch(const char* me, const FwdArgs& a, hipStream_t st) {
  const int64_t grid = (a.gr.M / 32 + a.gr.G + 2) * dh::ceil_div(a.N, 32);
  if (grid > MAX_GRID) return dh::fail(DH_ERR_INVALID, "%s: %lld tiles in one launch", me, (long long)grid);
  const int64_t groups = dh::ceil_div(a.K, SmallFrags<T, W_KM>::KG), waves = dh::ceil_div(groups, SmallFrags<T, W_KM>::BATCH);
  hipLaunchKernelGGL((grouped_small_kernel<T, W_KM>), dim3((unsigned)grid), dim3(64 * (unsigned)(waves < 1 ? 1 : waves > 8 ? 8 : waves)), 0, st, a);
  return dh::check_launch(me);
}

template <class T, bool W_KM>
int forward_pick(const char* me, const FwdArgs& a, hipStream_t st) {
  constexpr int VEC = 16 / sizeof(T);
  constexpr bool BF16 = sizeof(T) == 2;
  const bool dma = dma_rows(a.X, a.ldx, VEC) && dma_rows(a.W, a.ldw, VEC) && a.stride_w % VEC == 0 && a.K % VEC == 0 && (!W_KM || a.N % VEC == 0);
  // Few 32 x 32 tiles, in us, small against DMA tile: bf16 500 rows of 9 types 400 -> 200 (168 tiles) 5.2 / 10.8, 1500 of 30 types (532) 8.5 /
  // 10.7, 3000 of 3 types 512 -> 256 (768) 15.8 / 12.3; fp32 the first 8.2 / 14.0, 500 of 17 types 200 -> 400 (416) 7.5 / 8.8, 1500 of 30
  // types 15.5 / 13.3.  Against the staged tile: bf16 1500 of 30 types 401 -> 203 (532) 14.7 / 16.3, 203 -> 401 (988) 14.6 / 12.7; fp32 2000
  // rows 511 -> 510 (1008) 36 / 46, 3000 of 3 types 255 -> 510 (1536) 28 / 29.  Against the narrow tile: bf16 10000 of 5 types 400 -> 16 (317) 6.1 /
  // 8.4, 15913 of 30 types 872 -> 32 (527) 19.5 / 16.7; fp32 the latter 34 / 43, 30000 of 5 types 100 -> 16 (942) 10.5 / 8.9.
  const int64_t small_tiles = (a.gr.M / 32 + a.gr.G) * dh::ceil_div(a.N, 32);
  const int64_t few = a.N <= NARROW ? (BF16 ? 400 : 700) : BF16 ? 640 : dma ? 420 : 1536;
  if (small_tiles <= few) return small_launch<T, W_KM>(me, a, st);
  // Few rows per group: fp32 4000 rows of 100 types, 2000 -> 512: 302 us against 383.  (bf16 the same: 148 against 107: there the DMA tile
  // stays ahead.  Measured at that K; with K = 200 and 6 rows a group, 700 groups -> 64, it takes 13.5 us, and 32-row tiles took 12.2.)
  if (a.gr.M <= (int64_t)48 * a.gr.G && !(BF16 && dma)) return small_launch<T, W_KM>(me, a, st);
  if (a.N <= NARROW) return forward_launch<T, Tile<T, false, W_KM, 1, 1, 4, 1>>(me, a, st);
  if (dma) {
    if constexpr (sizeof(T) == 2) {
      // 256 x 256 with rows enough to fill such tiles (27630 rows of 476 types, 16 -> 560: 42 us against 34) and three rounds of them: 200003 x
      // 400 -> 200 (791 tiles) 90 us against 96 of the 128 x 128 one, which has two workgroups on a CU to fill each other's gaps and half the
      // waste at ragged ends: 50000 x 1000 -> 304 (402 tiles) 70 against 64, 8000 x 2000 -> 512 53 against 37
      if (a.N > 128 && a.gr.M >= 256 * (int64_t)a.gr.G && (a.gr.M / 256 + a.gr.G) * dh::ceil_div(a.N, 256) >= 3 * CUS)
        return forward_dma_launch<DmaTile<T, false, W_KM, 4, 2, 2, 4>>(me, a, st);
    } else {
      // fp32 with less than a round of workgroups: 64 x 64 (20011 x 512 -> 256, 336 tiles of 128: 68 / 67 us against 78 / 65; 60000 x 400 ->
      // 200, 996 tiles: 141 against 128)
      if ((a.gr.M / 128 + a.gr.G) * dh::ceil_div(a.N, 128) < 2 * CUS) return forward_dma_launch<DmaTile<T, false, W_KM, 1, 1, 2, 2>>(me, a, st);
    }
    return forward_dma_launch<DmaTile<T, false, W_KM, 2, 2, 2, 2>>(me, a, st);
  }
  return forward_launch<T, Tile<T, false, W_KM, 2, 2, 2, 2>>(me, a, st);
}

// The tile of the weight gradient and its chunks: as many chunks x tiles as workgroups run at a time, so that all end together; no chunk below
// 64 positions.  The large tile reads its operands least often; where it would leave a chunk short (few rows, or a small dW) the smaller
// one has more workgroups to share the groups among.
struct WgradPlan {
  int edge;  // rows and columns of the tile; NARROW: 32 of the narrow side x 128
  int64_t chunk;
};
int64_t wgrad_positions(int64_t M, int64_t G) { return M + (G > 1 ? G - 1 : 0) * GROUP_ROWS; }
WgradPlan wgrad_plan(int64_t M, int64_t N, int64_t K, int64_t G, int dtype) {
  const int large = dtype == DH_DTYPE_BF16 ? 256 : 128;
  WgradPlan p{};
  const int64_t positions = wgrad_positions(M, G);
  const int vec = dtype == DH_DTYPE_BF16 ? 8 : 4;
  const bool narrow = (N <= NARROW || K <= NARROW) && (N % vec != 0 || K % vec != 0);
  for (int edge : {large, large / 2}) {
    if (narrow) edge = NARROW;
    const int64_t tiles = narrow ? dh::ceil_div(std::max(N, K), 128) : dh::ceil_div(N, edge) * dh::ceil_div(K, edge), resident = edge == 256 ? CUS : 2 * CUS;
    const int64_t chunks = resident / tiles > 1 ? resident / tiles : 1;
    const int64_t rows = std::max<int64_t>(dh::ceil_div(positions, chunks), 64);
    p = {edge, rows};
    if (narrow || rows >= 4096) break;  // (1563 rows a chunk: 50000 x 1000 -> 304 76 us with the 256 tile, 62 with 128)
  }
  return p;
}

template <class TileT>
int wgrad_grid(const char* me, WgradArgs& a) {
  const int64_t tiles_k = dh::ceil_div(a.K, TileT::BN), tiles = dh::ceil_div(a.N, TileT::BM) * tiles_k;
  if (tiles > MAX_GRID || a.chunks * tiles > MAX_GRID - a.zeroers)
    return dh::fail(DH_ERR_INVALID, "%s: %lld tiles in one launch", me, (long long)(a.chunks * tiles));
  a.tiles_k = (int)tiles_k;
  a.tiles = (int)tiles;
  return DH_OK;
}

template <class T, class TileT>
int wgrad_launch(const char* me, WgradArgs a, hipStream_t st) {
  static std::atomic<uint64_t> done{0};
  const int allowed = allow_lds(me, reinterpret_cast<const void*>(grouped_wgrad_kernel<T, TileT>), TileT::LDS_BYTES, done);
  const int rc = allowed == DH_OK ? wgrad_grid<TileT>(me, a) : allowed;
  if (rc != DH_OK) return rc;
  hipLaunchKernelGGL((grouped_wgrad_kernel<T, TileT>), dim3((unsigned)(a.chunks * a.tiles + a.zeroers)), dim3(TileT::THREADS), TileT::LDS_BYTES, st, a);
  return dh::check_launch(me);
}

template <class TileT>
int wgrad_dma_launch(const char* me, WgradArgs a, hipStream_t st) {
  static std::atomic<uint64_t> done{0};
  const int allowed = allow_lds(me, reinterpret_cast<const void*>(grouped_wgrad_dma_kernel<TileT>), TileT::LDS_BYTES, done);
  const int rc = allowed == DH_OK ? wgrad_grid<TileT>(me, a) : allowed;
  if (rc != DH_OK) return rc;
  hipLaunchKernelGGL((grouped_wgrad_dma_kernel<TileT>), dim3((unsigned)(a.chunks * a.tiles + a.zeroers)), dim3(TileT::THREADS), TileT::LDS_BYTES, st, a);
  return dh::check_launch(me);
}

int check_grouped(const char* me, int64_t M, int64_t N, int64_t K, int64_t G, int dtype) {
  if (M < 0 || N < 0 || K < 0 || G < 0) return dh::fail(DH_ERR_INVALID, "%s: negative size", me);
  if (M > 0x7fffffff || G > 0x7fffff00) return dh::fail(DH_ERR_INVALID, "%s: more rows than an int32 bound can number", me);
  if (dtype != DH_DTYPE_F32 && dtype != DH_DTYPE_BF16) return dh::fail(DH_ERR_INVALID, "%s: dtype %d", me, dtype);
  return DH_OK;
}

}  // namespace

extern "C" int dh_gemm_grouped(int64_t M, int64_t N, int64_t K, int64_t G, int trans_b, int dtype, const void* X, int64_t ldx, const void* W,
                               int64_t ldw, int64_t stride_w, const int32_t* group_ptr, const float* bias, int64_t ld_bias, int act, void* Y,
                               int64_t ldy, int y_dtype, int zero_outside, dh_stream_t stream) {
  const char* me = "dh_gemm_grouped";
  const int rc = check_grouped(me, M, N, K, G, dtype);
  if (rc != DH_OK) return rc;
  if (y_dtype != DH_DTYPE_F32 && y_dtype != DH_DTYPE_BF16) return dh::fail(DH_ERR_INVALID, "%s: output dtype %d", me, y_dtype);
  if (act != DH_ACT_NONE && act != DH_ACT_RELU) return dh::fail(DH_ERR_INVALID, "%s: activation %d", me, act);
  if (M == 0 || N == 0) return DH_OK;
  if (!Y || !group_ptr || (K > 0 && (!X || (G > 0 && !W)))) return dh::fail(DH_ERR_INVALID, "%s: null tensor", me);
  const int64_t wc = trans_b ? K : N;
  if (ldx < K || ldw < wc || ldy < N || (bias && ld_bias < N) || (G > 1 && stride_w < 0)) return dh::fail(DH_ERR_INVALID, "%s: leading dimension below the row length", me);
  FwdArgs a{};
  a.gr = {group_ptr, M, (int)G};
  a.N = N; a.K = K; a.X = X; a.W = W; a.ldx = ldx; a.ldw = ldw; a.stride_w = stride_w; a.bias = bias; a.ld_bias = ld_bias; a.Y = Y; a.ldy = ldy;
  a.act = act; a.y_bf16 = y_dtype == DH_DTYPE_BF16; a.zero_outside = zero_outside != 0;
  hipStream_t st = dh::as_stream(stream);
  if (dtype == DH_DTYPE_BF16) return trans_b ? forward_pick<uint16_t, false>(me, a, st) : forward_pick<uint16_t, true>(me, a, st);
  return trans_b ? forward_pick<float, false>(me, a, st) : forward_pick<float, true>(me, a, st);
}

extern "C" size_t dh_gemm_grouped_wgrad_workspace_bytes(int64_t M, int64_t N, int64_t K, int64_t G, int dtype) {
  if (M <= 0 || N <= 0 || K <= 0 || G <= 0) return 16;
  const int64_t chunks = dh::ceil_div(wgrad_positions(M, G), wgrad_plan(M, N, K, G, dtype).chunk);
  return chunks < 2 ? 16 : 16 + (size_t)(2 * chunks) * (size_t)N * (size_t)(K + 1) * 4;
}

extern "C" int dh_gemm_grouped_wgrad(int64_t M, int64_t N, int64_t K, int64_t G, int dtype, const void* dY, int64_t ldy, const void* X, int64_t ldx,
                                     const int32_t* group_ptr, void* dW, int64_t ldw, int64_t stride_w, int dw_dtype, float* db, int64_t ld_db,
                                     void* workspace, size_t workspace_bytes, dh_stream_t stream) {
  const char* me = "dh_gemm_grouped_wgrad";
  const int rc = check_grouped(me, M, N, K, G, dtype);
  if (rc != DH_OK) return rc;
  if (dw_dtype != DH_DTYPE_F32 && dw_dtype != DH_DTYPE_BF16) return dh::fail(DH_ERR_INVALID, "%s: output dtype %d", me, dw_dtype);
  if (db && G > 0 && N > 0 && K == 0) return dh::fail(DH_ERR_INVALID, "%s: db without a column of X", me);
  if (G == 0 || N == 0 || K == 0) return DH_OK;
  if (!dW || !group_ptr || (M > 0 && (!dY || !X))) return dh::fail(DH_ERR_INVALID, "%s: null tensor", me);
  if (ldy < N || ldx < K || ldw < K || (G > 1 && stride_w < (N - 1) * ldw + K) || (db && ld_db < N))
    return dh::fail(DH_ERR_INVALID, "%s: leading dimension below the row length", me);
  const size_t need = dh_gemm_grouped_wgrad_workspace_bytes(M, N, K, G, dtype);
  if (!workspace || workspace_bytes < need) return dh::fail(DH_ERR_WORKSPACE, "%s: workspace of %zu bytes, need %zu", me, workspace_bytes, need);
  if (!dh::aligned16(workspace)) return dh::fail(DH_ERR_INVALID, "%s: workspace must be 16-byte aligned", me);
  WgradArgs a{};
  a.gr = {group_ptr, M, (int)G};
  a.N = N; a.K = K; a.dY = dY; a.X = X; a.ldy = ldy; a.ldx = ldx; a.dW = dW; a.ldw = ldw; a.stride_w = stride_w; a.dw_bf16 = dw_dtype == DH_DTYPE_BF16;
  a.db = db; a.ld_db = ld_db;
  const WgradPlan plan = wgrad_plan(M, N, K, G, dtype);
  a.chunk = plan.chunk;
  // a workgroup writes about 20 GB/s: runs of at most 64 KB (2 rows of 10 types, 328 -> 140 bf16: 38 us with whole groups, 12 so)
  a.slices = (int)std::min((double)std::min<int64_t>(N, 1 << 20), 1 + (double)N * K * (a.dw_bf16 ? 2 : 4) / 65536);
  a.zeroers = 8 * (int)std::min<int64_t>(32, dh::ceil_div(G * a.slices, 8));
  a.chunks = M > 0 ? dh::ceil_div(wgrad_positions(M, G), a.chunk) : 1;
  a.part_w = static_cast<float*>(workspace);
  a.part_b = a.part_w + 2 * a.chunks * N * K;
  hipStream_t st = dh::as_stream(stream);
  const int vec = dtype == DH_DTYPE_BF16 ? 8 : 4;
  const bool dma = dma_rows(dY, ldy, vec) && dma_rows(X, ldx, vec) && N % vec == 0 && K % vec == 0;
  int launched;
  if (plan.edge == NARROW) {
    if (dtype == DH_DTYPE_BF16)
      launched = N <= NARROW ? wgrad_launch<uint16_t, Tile<uint16_t, true, true, 1, 1, 1, 4>>(me, a, st) : wgrad_launch<uint16_t, Tile<uint16_t, true, true, 1, 1, 4, 1>>(me, a, st);
    else
      launched = N <= NARROW ? wgrad_launch<float, Tile<float, true, true, 1, 1, 1, 4>>(me, a, st) : wgrad_launch<float, Tile<float, true, true, 1, 1, 4, 1>>(me, a, st);
  } else if (dtype != DH_DTYPE_BF16) {
    if (!dma) launched = plan.edge == 128 ? wgrad_launch<float, Tile<float, true, true, 2, 2, 2, 2>>(me, a, st) : wgrad_launch<float, Tile<float, true, true, 1, 1, 2, 2>>(me, a, st);
    else launched = plan.edge == 128 ? wgrad_dma_launch<DmaTile<float, true, true, 2, 2, 2, 2>>(me, a, st) : wgrad_dma_launch<DmaTile<float, true, true, 1, 1, 2, 2>>(me, a, st);
  } else {
    if (!dma) launched = wgrad_launch<uint16_t, Tile<uint16_t, true, true, 2, 2, 2, 2>>(me, a, st);
    else launched = plan.edge == 256 ? wgrad_dma_launch<DmaTile<uint16_t, true, true, 4, 2, 2, 4>>(me, a, st) : wgrad_dma_launch<DmaTile<uint16_t, true, true, 2, 2, 2, 2>>(me, a, st);
  }
  if (launched != DH_OK) return launched;
  if (a.chunks > 1)
    hipLaunchKernelGGL(wgrad_join_kernel, dim3((unsigned)dh::ceil_div(N * K, 1024), (unsigned)(a.chunks - 1)), dim3(256), 0, st, a);
  return dh::check_launch(me);
}
