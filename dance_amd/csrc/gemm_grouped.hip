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
#include <type_traits>

#include "common.h"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4u __attribute__((ext_vector_type(4), aligned(2)));  // 16 bytes at an element's own alignment

__device__ __forceinline__ float bf16_f32(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ uint16_t f32_bf16(float x) {  // nearest even; NaN stays a quiet NaN
  const uint32_t u = __float_as_uint(x);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);
  return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
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
  int64_t begin, end, start;  // the slot's rows; start: the group's first row
  int index;       // number of the slot within its group
  bool live;
};

// slot s of R rows (R a power of two: shift)
__device__ __forceinline__ Slot find_slot(const Groups& gr, int64_t s, int shift) {
  const int n = gr.G + 2;
  const int i = search(n, s, [&](int j) { return (gr.edge(j) >> shift) + j; });
  const int64_t a = gr.edge(i), b = gr.edge(i + 1);
  const int64_t first = (a >> shift) + i;
  Slot r;
  r.group = i == 0 || i == n - 1 ? -1 : i - 1;
  r.start = a;
  r.index = (int)(s - first);
  r.begin = a + ((int64_t)r.index << shift);
  r.end = min(b, r.begin + ((int64_t)1 << shift));
  r.live = r.index >= 0 && r.begin < b;
  return r;
}

// the logical number of a workgroup: the dispatcher deals workgroups round robin to the 8 XCDs; handing each XCD a contiguous run keeps
// the tiles that share an operand panel on one L2
__device__ __forceinline__ int64_t xcd_run(int64_t bid, int64_t n) {
  const int64_t q = n / 8, r = n % 8, xcd = bid % 8;
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

// R rows (m or n) x BK of an operand.  KM = false: memory is [row][k]; true: [k][row].  Both stay as they lie in memory in LDS too:
// a [k][row] image is read back transposed (bf16: ds_read_b64_tr_b16) or by single elements (fp32).
template <class T, bool KM, int R, int THREADS>
struct Operand {
  static constexpr int VEC = Geo<T>::VEC, BK = Geo<T>::BK;
  // [k][row] images: bf16 rows of R + 32 elements (64 bytes past a multiple of 256: the four k rows that one transposing read takes from
  // lie on distinct banks); fp32 rows of R + 8 (the two half waves read rows 4 apart: 32 banks apart)
  static constexpr int LD = KM ? (sizeof(T) == 2 ? R + 32 : R + 8) : Geo<T>::LD_MK;
  static constexpr int ELEMS = KM ? BK * LD : R * LD;
  static constexpr int CPR = KM ? R / VEC : 8;                        // 16-byte pieces per image row
  static constexpr int PIECES = (KM ? BK : R) * CPR / THREADS;        // per thread
  static constexpr int ROWS_PER_PASS = THREADS / CPR;
  static_assert(PIECES >= 1 && PIECES * THREADS == (KM ? BK : R) * CPR, "tile does not divide among the threads");

  u32x4 reg[PIECES];

  static __device__ __forceinline__ u32x4 guarded(const T* p, int64_t n_valid) {
    if (n_valid >= VEC) return *reinterpret_cast<const u32x4u*>(p);
    T e[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) e[i] = i < n_valid ? p[i] : T(0);
    u32x4 v;
    __builtin_memcpy(&v, e, 16);
    return v;
  }
  // rows [r0, rlim) of the operand, k in [k0, klim).  Rows beyond rlim read some row below it (their products are never stored);
  // k beyond klim reads as zero.  FULL: the whole BK lies below klim (and for KM all R rows below rlim).
  template <bool FULL>
  __device__ __forceinline__ void load(const T* base, int64_t ld, int64_t r0, int64_t rlim, int64_t k0, int64_t klim) {
    const int tid = threadIdx.x;
#pragma unroll
    for (int q = 0; q < PIECES; ++q) {
      const int ir = tid / CPR + q * ROWS_PER_PASS, ic = (tid % CPR) * VEC;
      if (!KM) {
        const int64_t row = min(r0 + ir, rlim - 1), k = k0 + ic;
        const T* p = base + row * ld + k;
        if (FULL) reg[q] = *reinterpret_cast<const u32x4u*>(p);
        else reg[q] = guarded(p, klim - k);
      } else {
        const int64_t k = k0 + ir, row = r0 + ic;
        const T* p = base + k * ld + row;
        if (FULL) reg[q] = *reinterpret_cast<const u32x4u*>(p);
        else reg[q] = guarded(p, k < klim ? rlim - row : 0);
      }
    }
  }
  __device__ __forceinline__ void store(T* img) const {
    const int tid = threadIdx.x;
#pragma unroll
    for (int q = 0; q < PIECES; ++q) {
      const int ir = tid / CPR + q * ROWS_PER_PASS, ic = (tid % CPR) * VEC;
      *reinterpret_cast<u32x4*>(img + ir * LD + ic) = reg[q];
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
// (with A first a lane holds 16 rows of one column: four times as many, two-byte, stores: 818 against 726 us at 200003 x 2000 -> 512 bf16)
template <int MI, int NI, int WC, class F>
__device__ __forceinline__ void each4(const f32x16 (&acc)[MI][NI], int64_t m0, int64_t mlim, int64_t n0, int64_t nlim, F&& f) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
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
// BM x BN of C = A B^T over k in [0, K): WR x WC waves of MI x NI 32 x 32 accumulators.  Two LDS stages: while the products of one step
// run, the next one's pieces (requested a step earlier) are written and the ones after that requested.
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
  // seen(opB or opA): called with the A operand's registers of every step (the bias gradient's column sums)
  template <class Seen>
  __device__ __forceinline__ void run(const T* A, int64_t lda, int64_t m0, int64_t mlim, const T* B, int64_t ldb, int64_t n0, int64_t nlim,
                                      int64_t k_begin, int64_t k_end, T* lds, Seen&& seen) {
    zero();
    if (k_end <= k_begin) return;
    const bool whole = (!A_KM || m0 + BM <= mlim) && (!B_KM || n0 + BN <= nlim);
    OpA a;
    OpB b;
    auto fetch = [&](int64_t k0) __attribute__((always_inline)) {
      if (whole && k0 + BK <= k_end) {
        a.template load<true>(A, lda, m0, mlim, k0, k_end);
        b.template load<true>(B, ldb, n0, nlim, k0, k_end);
      } else {
        a.template load<false>(A, lda, m0, mlim, k0, k_end);
        b.template load<false>(B, ldb, n0, nlim, k0, k_end);
      }
    };
    auto put = [&](int stage) __attribute__((always_inline)) {
      a.store(lds + stage * STAGE);
      b.store(lds + stage * STAGE + OpA::ELEMS);
      seen(a);
    };
    const int64_t steps = (k_end - k_begin + BK - 1) / BK;
    fetch(k_begin);
    put(0);
    if (steps > 1) fetch(k_begin + BK);
    __syncthreads();
    for (int64_t t = 0; t < steps; ++t) {
      if (t + 1 < steps) {
        put((t + 1) & 1);
        if (t + 2 < steps) fetch(k_begin + (t + 2) * BK);
      }
      products(lds + (t & 1) * STAGE);
      __syncthreads();
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
  typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
  typedef unsigned int u32x2u __attribute__((ext_vector_type(2), aligned(2)));
  if (BF16) {
    uint16_t* p = static_cast<uint16_t*>(row) + n;
    const uint16_t h[4] = {f32_bf16(v[0]), f32_bf16(v[1]), f32_bf16(v[2]), f32_bf16(v[3])};
    if (n + 4 <= nlim) {
      *reinterpret_cast<u32x2u*>(p) = u32x2u{(unsigned)h[0] | (unsigned)h[1] << 16, (unsigned)h[2] | (unsigned)h[3] << 16};
    } else {
      for (int e = 0; e < 3; ++e)
        if (n + e < nlim) p[e] = h[e];
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

// ---- the bf16 tile filled by LDS DMA ---------------------------------------------------------------------------------------------------
// The same product with the operands going from memory to LDS without passing registers (global_load_lds, 16 bytes a lane): what the big
// products run on.  The DMA writes a wave's 64 pieces to 1 KB of LDS in lane order, so images cannot be padded; bank conflicts are avoided by
// choosing WHICH piece a lane fetches: piece c of an image row lies at position c ^ x,
//   [row][k] images (128-byte rows):  x = (row >> 1) & 7: the 16 rows that a 16-byte fragment read takes at a time cover all 16 slots of
//                                     two rows;
//   [k][row] images (2 R-byte rows):  x = (k & 3) << 2: the four k rows that a transposing read takes from lie 64 bytes apart.
// Needs 16-byte aligned rows (address and stride) and, for a [k][row] operand, a row count that is a multiple of 8 (a piece is whole or
// absent).  In the last, partial step of k the lanes whose pieces lie behind the end fetch a piece of zeros instead.
typedef const __attribute__((address_space(1))) void* global_ptr;
typedef __attribute__((address_space(3))) void* lds_ptr;

__device__ __attribute__((aligned(16))) const uint32_t zero_piece[4] = {0, 0, 0, 0};

template <bool KM, int R, int THREADS>
struct DmaOperand {
  static constexpr int BK = 64, CPR = KM ? R / 8 : 8, PIECES = R * 8 / THREADS, ELEMS = R * BK;
  static_assert(PIECES * THREADS == R * 8 && (!KM || R >= 128), "tile does not divide among the threads");

  const uint16_t* p[PIECES];

  static __device__ __forceinline__ int image_row(int q) { return (q * THREADS + (int)threadIdx.x) / CPR; }
  static __device__ __forceinline__ int piece(int q) {
    const int row = image_row(q), c = (q * THREADS + (int)threadIdx.x) % CPR;
    return KM ? c ^ ((row & 3) << 2) : c ^ ((row >> 1) & 7);
  }
  __device__ __forceinline__ void start(const uint16_t* base, int64_t ld, int64_t r0, int64_t rlim, int64_t k0) {
#pragma unroll
    for (int q = 0; q < PIECES; ++q) {
      if (KM) p[q] = base + (k0 + image_row(q)) * ld + min(r0 + piece(q) * 8, rlim - 8);
      else p[q] = base + min(r0 + image_row(q), rlim - 1) * ld + k0 + piece(q) * 8;
    }
  }
  // the next BK of k into an image
  __device__ __forceinline__ void issue(uint16_t* img, int64_t ld) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int q = 0; q < PIECES; ++q) {
      __builtin_amdgcn_global_load_lds((global_ptr)p[q], (lds_ptr)(img + (q * THREADS + wave * 64) * 8), 16, 0, 0);
      p[q] += KM ? BK * ld : BK;
    }
  }
  // the last `left` < BK of k, zeros behind them
  __device__ __forceinline__ void issue_last(uint16_t* img, int left) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int q = 0; q < PIECES; ++q) {
      const int k = KM ? image_row(q) : piece(q) * 8;
      const void* from = k < left ? static_cast<const void*>(p[q]) : static_cast<const void*>(zero_piece);
      __builtin_amdgcn_global_load_lds((global_ptr)from, (lds_ptr)(img + (q * THREADS + wave * 64) * 8), 16, 0, 0);
    }
  }
  // the fragment of rows [32 tile, 32 tile + 32), k [kk, kk + 16): lane l holds row l & 31, k (l >> 5) * 8 .. + 8
  static __device__ __forceinline__ bf16x8 frag(const uint16_t* img, int tile, int kk) {
    const int lane = threadIdx.x & 63;
    if (!KM) {
      const int c = (kk >> 3) + (lane >> 5);
      return *reinterpret_cast<const bf16x8*>(img + (tile * 32 + (lane & 31)) * BK + ((c ^ ((lane >> 1) & 7)) << 3));
    }
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef s16x4 __attribute__((address_space(3))) * lds_s16x4;
    const int b = lane >> 4, i = lane & 15, x = i >> 2;  // x = k & 3 of the lane's row
    const uint16_t* at = img + (kk + (b >> 1) * 8 + x) * R + (tile ^ x) * 32 + (b & 1) * 16 + (i & 3) * 4;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)at);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at + 4 * R));
    bf16x8 f;
    __builtin_memcpy(&f, &lo, 8);
    __builtin_memcpy(reinterpret_cast<char*>(&f) + 8, &hi, 8);
    return f;
  }
};

// every wave's DMA has landed and its image reads are done: what the barrier by itself does not wait for is the DMA (vmcnt)
__device__ __forceinline__ void images_ready() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Schedule of a step: its first fragments are in registers when it begins; the fragments of k group kk + 1 are read while the products of
// group kk run, the barrier that hands over the next image stands in front of the LAST group, and behind it the next step's first fragments
// are read and the step after that is requested: a wave never waits for LDS with nothing to multiply, and the DMA has a whole step to land.
template <bool A_KM, bool B_KM, int MI, int NI, int WR, int WC>
struct DmaTile {
  static constexpr int BM = MI * WR * 32, BN = NI * WC * 32, THREADS = WR * WC * 64, BK = 64;
  typedef DmaOperand<A_KM, BM, THREADS> OpA;
  typedef DmaOperand<B_KM, BN, THREADS> OpB;
  static constexpr int STAGE = OpA::ELEMS + OpB::ELEMS, OUT = 4096, LDS_BYTES = 2 * STAGE * 2 + WR * WC * OUT;

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
    bf16x8 a[MI], b[NI];
    __device__ __forceinline__ void read(const uint16_t* st, int kk) {
      const int wave = threadIdx.x >> 6, tm = (wave / WC) * MI, tn = (wave % WC) * NI;
#pragma unroll
      for (int i = 0; i < MI; ++i) a[i] = OpA::frag(st, tm + i, kk);
#pragma unroll
      for (int j = 0; j < NI; ++j) b[j] = OpB::frag(st + OpA::ELEMS, tn + j, kk);
    }
  };
  template <bool SUMS>
  __device__ __forceinline__ void multiply(const Frags& f) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.b[j], f.a[i], acc[i][j], 0, 0, 0);
    if (SUMS) {
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        u32x4 v;
        __builtin_memcpy(&v, &f.a[i], 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) row_sum[i] += __uint_as_float(v[e] << 16) + __uint_as_float(v[e] & 0xffff0000u);
      }
    }
  }
  // LDS reads of one fragment set per group of MI x NI products: spread one behind each product
  static constexpr int READS = (A_KM ? 2 : 1) * MI + (B_KM ? 2 : 1) * NI, PER = (READS + MI * NI - 1) / (MI * NI);
  static __device__ __forceinline__ void interleave() {
#pragma unroll
    for (int i = 0; i < MI * NI; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
    }
  }
  template <bool SUMS>
  __device__ __forceinline__ void run(const uint16_t* A, int64_t lda, int64_t m0, int64_t mlim, const uint16_t* B, int64_t ldb, int64_t n0,
                                      int64_t nlim, int64_t k_begin, int64_t k_end, uint16_t* lds) {
    zero();
    if (k_end <= k_begin) return;
    OpA a;
    OpB b;
    a.start(A, lda, m0, mlim, k_begin);
    b.start(B, ldb, n0, nlim, k_begin);
    const int64_t full = (k_end - k_begin) / BK;
    const int left = (int)((k_end - k_begin) % BK);
    const int64_t steps = full + (left > 0);
    auto image = [&](int64_t t) __attribute__((always_inline)) { return lds + (t & 1) * STAGE; };
    auto issue = [&](int64_t t) __attribute__((always_inline)) {
      if (t < full) {
        a.issue(image(t), lda);
        b.issue(image(t) + OpA::ELEMS, ldb);
      } else {
        a.issue_last(image(t), left);
        b.issue_last(image(t) + OpA::ELEMS, left);
      }
    };
    Frags f[2];
    issue(0);
    if (steps > 1) issue(1);
    images_ready();
    f[0].read(image(0), 0);
    int64_t t = 0;
    for (; t + 1 < steps; ++t) {
      const uint16_t* st = image(t);
#pragma unroll
      for (int g = 0; g < 3; ++g) {
        f[(g + 1) & 1].read(st, (g + 1) * 16);
        multiply<SUMS>(f[g & 1]);
        interleave();
      }
      images_ready();
      if (t + 2 < steps) issue(t + 2);
      f[0].read(image(t + 1), 0);
      multiply<SUMS>(f[1]);
      interleave();
    }
    const int groups = left > 0 ? (left + 15) / 16 : 4;
    for (int g = 0; g < groups; ++g) {
      if (g + 1 < groups) f[1].read(image(t), (g + 1) * 16);
      multiply<SUMS>(f[0]);
      f[0] = f[1];
    }
  }
  // The tile to memory: base[m * ld + n] = value(n, four accumulators) for m < mlim, n < nlim.  A lane holds four-runs of one row each 8
  // columns apart; written like that, every store instruction scatters 16-byte bits over 32 rows.  Each wave turns 32 rows x 128 bytes at
  // a time in its own 4 KB of LDS (16-byte piece c of row r at c ^ (r >> 1) & 7, as in the images) and stores whole 128-byte row pieces.
  template <bool BF16, class V>
  __device__ __forceinline__ void store(void* base, int64_t ld, int64_t m0, int64_t mlim, int64_t n0, int64_t nlim, uint16_t* lds, V&& value) const {
    constexpr int SIZE = BF16 ? 2 : 4, COLS = 128 / SIZE, PER = COLS / 32;  // columns and accumulator tiles of a 128-byte row piece
    static_assert(NI % PER == 0, "a wave's columns do not divide into row pieces");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    unsigned char* out = reinterpret_cast<unsigned char*>(lds + 2 * STAGE) + wave * OUT;
    const int r = lane & 31, x = (r >> 1) & 7;
    const int64_t wm = m0 + (wave / WC) * MI * 32, wn = n0 + (wave % WC) * NI * 32;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int jj = 0; jj < NI; jj += PER) {
        if (wm + i * 32 >= mlim || wn + jj * 32 >= nlim) continue;  // (uniform)
#pragma unroll
        for (int j = jj; j < jj + PER; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4 v = value(wn + j * 32 + 8 * q + 4 * (lane >> 5),
                                  f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]});
            const int col = (j - jj) * 32 + 8 * q + 4 * (lane >> 5);
            if (BF16) {
              *reinterpret_cast<u32x2*>(out + r * 128 + (((col >> 3) ^ x) << 4) + (col & 4) * 2) =
                  u32x2{(unsigned)f32_bf16(v[0]) | (unsigned)f32_bf16(v[1]) << 16, (unsigned)f32_bf16(v[2]) | (unsigned)f32_bf16(v[3]) << 16};
            } else {
              *reinterpret_cast<f32x4*>(out + r * 128 + (((col >> 2) ^ x) << 4)) = v;
            }
          }
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          const int row = it * 8 + (lane >> 3), c = lane & 7;
          const u32x4 v = *reinterpret_cast<const u32x4*>(out + row * 128 + ((c ^ ((row >> 1) & 7)) << 4));
          const int64_t m = wm + i * 32 + row, n = wn + jj * 32 + c * (16 / SIZE);
          if (m < mlim && n < nlim) {
            unsigned char* to = static_cast<unsigned char*>(base) + (m * ld + n) * SIZE;
            if (n + 16 / SIZE <= nlim) {
              *reinterpret_cast<u32x4u*>(to) = v;
            } else {
              for (int e = 0; e < 16 / SIZE - 1; ++e) {
                if (n + e >= nlim) break;
                if (BF16) reinterpret_cast<uint16_t*>(to)[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
                else reinterpret_cast<uint32_t*>(to)[e] = v[e];
              }
            }
          }
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

template <class T, class TileT, bool DMA>
__global__ __launch_bounds__(TileT::THREADS) void grouped_forward_kernel(const FwdArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char raw_lds[];
  const int64_t tiles_n = (a.N + TileT::BN - 1) / TileT::BN;
  const int64_t id = xcd_run(blockIdx.x, gridDim.x);
  const Slot s = find_slot(a.gr, id / tiles_n, __builtin_ctz(TileT::BM));
  if (!s.live || (s.group < 0 && !a.zero_outside)) return;
  const int64_t n0 = (id % tiles_n) * TileT::BN;
  T* lds = reinterpret_cast<T*>(raw_lds);
  TileT t;
  const float* bias = nullptr;
  if (s.group < 0) {
    t.zero();
  } else {
    const T *X = static_cast<const T*>(a.X), *W = static_cast<const T*>(a.W) + s.group * a.stride_w;
    if constexpr (DMA) t.template run<false>(X, a.ldx, s.begin, s.end, W, a.ldw, n0, a.N, 0, a.K, lds);
    else t.run(X, a.ldx, s.begin, s.end, W, a.ldw, n0, a.N, 0, a.K, lds, [](const auto&) {});
    if (a.bias) bias = a.bias + s.group * a.ld_bias;
  }
  auto value = [&](int64_t n, f32x4 v) __attribute__((always_inline)) {
    if (bias) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += bias[min(n + e, a.N - 1)];
    }
    if (a.act == DH_ACT_RELU) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = v[e] < 0.f ? 0.f : v[e];  // (a NaN passes)
    }
    return v;
  };
  if constexpr (DMA) {
    if (a.y_bf16) t.template store<true>(a.Y, a.ldy, s.begin, s.end, n0, a.N, lds, value);
    else t.template store<false>(a.Y, a.ldy, s.begin, s.end, n0, a.N, lds, value);
  } else {
    t.each(s.begin, s.end, n0, a.N, [&](int64_t m, int64_t n, f32x4 v) __attribute__((always_inline)) {
      v = value(n, v);
      if (a.y_bf16) put4<true>(static_cast<uint16_t*>(a.Y) + m * a.ldy, n, a.N, v);
      else put4<false>(static_cast<float*>(a.Y) + m * a.ldy, n, a.N, v);
    });
  }
}

// ---- dW, db --------------------------------------------------------------------------------------------------------------------------
// dW_g [N][K] = sum over the group's rows of dY[i, n] X[i, k]: both operands [k][row] images with the rows as the contraction.  Long groups
// are cut into chunks of 2^shift rows; a group of one chunk is finished in place, the chunks of a longer one go to partial slots that
// wgrad_join_kernel adds in chunk order (no atomics).  The slot of chunk j that starts at row s: 2 (s >> shift) + (j > 0): two chunks of
// longer groups that start inside the same 2^shift rows are the last of one group (j > 0) and the first of the next (j = 0).
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
  float* part_w;  // [slots][N][K]
  float* part_b;  // [slots][N]
  int shift;
  int64_t tiles_k, tiles;
};

template <class T, class TileT, bool DMA>
__global__ __launch_bounds__(TileT::THREADS) void grouped_wgrad_kernel(const WgradArgs a) {
  typedef typename TileT::OpA OpA;
  extern __shared__ __attribute__((aligned(16))) unsigned char raw_lds[];
  const int64_t id = xcd_run(blockIdx.x, gridDim.x);
  const Slot s = find_slot(a.gr, id / a.tiles, a.shift);
  if (s.group < 0) return;
  const int64_t glen = a.gr.edge(s.group + 2) - s.start;
  if (!s.live && !(glen <= 0 && s.index == 0)) return;  // an empty group's one slot writes its zeros
  const int64_t tile = id % a.tiles, n0 = (tile / a.tiles_k) * TileT::BM, k0 = (tile % a.tiles_k) * TileT::BN;
  const bool alone = glen <= ((int64_t)1 << a.shift);
  const bool sums = a.db && k0 == 0;
  const int64_t end = s.live ? s.end : s.begin;
  const T *dY = static_cast<const T*>(a.dY), *X = static_cast<const T*>(a.X);
  T* stages = reinterpret_cast<T*>(raw_lds);
  TileT t;
  constexpr int VEC = Geo<T>::VEC;
  float cs[VEC];
  if constexpr (DMA) {
    if (sums) t.template run<true>(dY, a.ldy, n0, a.N, X, a.ldx, k0, a.K, s.begin, end, stages);
    else t.template run<false>(dY, a.ldy, n0, a.N, X, a.ldx, k0, a.K, s.begin, end, stages);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) cs[e] = 0.f;
    t.run(dY, a.ldy, n0, a.N, X, a.ldx, k0, a.K, s.begin, end, stages, [&](const OpA& op) __attribute__((always_inline)) {
      if (!sums) return;
#pragma unroll
      for (int q = 0; q < OpA::PIECES; ++q) {
        T e[VEC];
        __builtin_memcpy(e, &op.reg[q], 16);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          if constexpr (sizeof(T) == 2) cs[i] += bf16_f32(e[i]);
          else cs[i] += e[i];
        }
      }
    });
  }
  const int64_t slot = alone ? 0 : 2 * (s.begin >> a.shift) + (s.index > 0 ? 1 : 0);
  void* out = a.part_w + slot * a.N * a.K;
  int64_t ld = a.K;
  bool bf16 = false;
  if (alone) {
    bf16 = a.dw_bf16;
    ld = a.ldw;
    out = static_cast<char*>(a.dW) + s.group * a.stride_w * (bf16 ? 2 : 4);
  }
  if constexpr (DMA) {
    auto value = [](int64_t, f32x4 v) __attribute__((always_inline)) { return v; };
    if (bf16) t.template store<true>(out, ld, n0, a.N, k0, a.K, stages, value);
    else t.template store<false>(out, ld, n0, a.N, k0, a.K, stages, value);
  } else {
    t.each(n0, a.N, k0, a.K, [&](int64_t n, int64_t k, f32x4 v) __attribute__((always_inline)) {
      if (bf16) put4<true>(static_cast<uint16_t*>(out) + n * ld, k, a.K, v);
      else put4<false>(static_cast<float*>(out) + n * ld, k, a.K, v);
    });
  }
  if (sums) {
    auto put = [&](int i, float v) __attribute__((always_inline)) {
      if (n0 + i >= a.N) return;
      if (alone) a.db[s.group * a.ld_db + n0 + i] = v;
      else a.part_b[slot * a.N + n0 + i] = v;
    };
    if constexpr (DMA) t.row_sums(put);
    else {  // thread t summed columns (t % CPR) * VEC of the rows it staged
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
        put(i, v);
      }
    }
  }
}

// The chunks of every group longer than one chunk.  blockIdx.y = b: the group that starts inside rows [b << shift, (b + 1) << shift) and
// reaches beyond them, if there is one, contains the last of these rows.
__global__ __launch_bounds__(256) void wgrad_join_kernel(const WgradArgs a) {
  const int64_t b = blockIdx.y, last = ((b + 1) << a.shift) - 1;
  if (last >= a.gr.M) return;
  const int i = search(a.gr.G + 2, last, [&](int j) { return a.gr.edge(j); });
  const int64_t start = a.gr.edge(i), end = a.gr.edge(i + 1);
  if (i == 0 || i == a.gr.G + 1 || start < (b << a.shift) || start > last || end - start <= ((int64_t)1 << a.shift)) return;
  const int group = i - 1, chunks = (int)((end - start + ((int64_t)1 << a.shift) - 1) >> a.shift);
  const int64_t nk = a.N * a.K, total = nk + (a.db ? a.N : 0);
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= total) return;
  const bool is_b = at >= nk;
  const float* p = is_b ? a.part_b + 2 * b * a.N + (at - nk) : a.part_w + 2 * b * nk + at;
  const int64_t step = is_b ? a.N : nk;
  float v = p[0];
  int c = 1;
  for (; c + 8 <= chunks; c += 8) {  // chunk c > 0 of the group: slot 2 (b + c) + 1
    float t[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) t[u] = p[(2 * (int64_t)(c + u) + 1) * step];
#pragma unroll
    for (int u = 0; u < 8; ++u) v += t[u];
  }
  for (; c < chunks; ++c) v += p[(2 * (int64_t)c + 1) * step];
  if (is_b) {
    a.db[group * a.ld_db + (at - nk)] = v;
  } else {
    const int64_t o = group * a.stride_w + (at / a.K) * a.ldw + at % a.K;
    if (a.dw_bf16) static_cast<uint16_t*>(a.dW)[o] = f32_bf16(v);
    else static_cast<float*>(a.dW)[o] = v;
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------------
constexpr int64_t MAX_GRID = 0x7fffffff;

template <class T, class TileT, bool DMA>
int forward_launch(const char* me, const FwdArgs& a, hipStream_t st) {
  const int64_t slots = a.gr.M / TileT::BM + a.gr.G + 2, grid = slots * dh::ceil_div(a.N, TileT::BN);
  if (grid > MAX_GRID) return dh::fail(DH_ERR_INVALID, "%s: %lld tiles in one launch", me, (long long)grid);
  auto* kernel = grouped_forward_kernel<T, TileT, DMA>;
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, TileT::LDS_BYTES);
  if (attr != hipSuccess) return dh::fail(DH_ERR_LAUNCH, "%s: %d bytes of LDS: %s", me, TileT::LDS_BYTES, hipGetErrorString(attr));
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(TileT::THREADS), TileT::LDS_BYTES, st, a);
  return dh::check_launch(me);
}

bool dma_rows(const void* p, int64_t ld) { return dh::aligned16(p) && ld % 8 == 0; }

template <class T, bool W_KM>
int forward_pick(const char* me, const FwdArgs& a, hipStream_t st) {
  // few rows per group: a 32-row tile wastes less of the matrix cores and of the slots
  if (a.gr.M <= (int64_t)48 * a.gr.G) return forward_launch<T, Tile<T, false, W_KM, 1, 1, 1, 4>, false>(me, a, st);
  if constexpr (sizeof(T) == 2) {
    const bool dma = dma_rows(a.X, a.ldx) && dma_rows(a.W, a.ldw) && a.stride_w % 8 == 0 && a.K % 8 == 0 && (!W_KM || a.N % 8 == 0);
    if (dma && a.gr.M >= (int64_t)1024 * a.gr.G) return forward_launch<T, DmaTile<false, W_KM, 4, 2, 2, 4>, true>(me, a, st);
    if (dma) return forward_launch<T, DmaTile<false, W_KM, 2, 2, 2, 2>, true>(me, a, st);
  }
  return forward_launch<T, Tile<T, false, W_KM, 2, 2, 2, 2>, false>(me, a, st);
}

constexpr int WG_TILE = 128;

// rows per chunk: enough chunks x tiles to fill the chip a few times, no chunk below 256 rows
int wgrad_shift(int64_t M, int64_t N, int64_t K) {
  const int64_t tiles = dh::ceil_div(N, WG_TILE) * dh::ceil_div(K, WG_TILE);
  const int64_t want = dh::ceil_div(1024, tiles);  // chunks
  int shift = 8;
  while (shift < 30 && (M >> shift) > want) ++shift;
  return shift;
}

int64_t wgrad_slots(int64_t M, int shift) { return 2 * ((M >> shift) + 1); }

template <class T, class TileT, bool DMA>
int wgrad_launch(const char* me, WgradArgs a, hipStream_t st) {
  a.tiles_k = dh::ceil_div(a.K, TileT::BN);
  a.tiles = dh::ceil_div(a.N, TileT::BM) * a.tiles_k;
  const int64_t grid = ((a.gr.M >> a.shift) + a.gr.G + 2) * a.tiles;
  if (grid > MAX_GRID) return dh::fail(DH_ERR_INVALID, "%s: %lld tiles in one launch", me, (long long)grid);
  auto* kernel = grouped_wgrad_kernel<T, TileT, DMA>;
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, TileT::LDS_BYTES);
  if (attr != hipSuccess) return dh::fail(DH_ERR_LAUNCH, "%s: %d bytes of LDS: %s", me, TileT::LDS_BYTES, hipGetErrorString(attr));
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(TileT::THREADS), TileT::LDS_BYTES, st, a);
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
  if (!Y || (G > 0 && !group_ptr) || (K > 0 && (!X || (G > 0 && !W)))) return dh::fail(DH_ERR_INVALID, "%s: null tensor", me);
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

extern "C" size_t dh_gemm_grouped_wgrad_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K < 0) return 16;
  return 16 + (size_t)wgrad_slots(M, wgrad_shift(M, N, K)) * (size_t)N * (size_t)(K + 1) * 4;
}

extern "C" int dh_gemm_grouped_wgrad(int64_t M, int64_t N, int64_t K, int64_t G, int dtype, const void* dY, int64_t ldy, const void* X, int64_t ldx,
                                     const int32_t* group_ptr, void* dW, int64_t ldw, int64_t stride_w, int dw_dtype, float* db, int64_t ld_db,
                                     void* workspace, size_t workspace_bytes, dh_stream_t stream) {
  const char* me = "dh_gemm_grouped_wgrad";
  const int rc = check_grouped(me, M, N, K, G, dtype);
  if (rc != DH_OK) return rc;
  if (dw_dtype != DH_DTYPE_F32 && dw_dtype != DH_DTYPE_BF16) return dh::fail(DH_ERR_INVALID, "%s: output dtype %d", me, dw_dtype);
  if (G == 0 || N == 0 || K == 0) return DH_OK;
  if (!dW || !group_ptr || (M > 0 && (!dY || !X))) return dh::fail(DH_ERR_INVALID, "%s: null tensor", me);
  if (ldy < N || ldx < K || ldw < K || (G > 1 && stride_w < (N - 1) * ldw + K) || (db && ld_db < N))
    return dh::fail(DH_ERR_INVALID, "%s: leading dimension below the row length", me);
  const size_t need = dh_gemm_grouped_wgrad_workspace_bytes(M, N, K);
  if (!workspace || workspace_bytes < need) return dh::fail(DH_ERR_WORKSPACE, "%s: workspace of %zu bytes, need %zu", me, workspace_bytes, need);
  if (!dh::aligned16(workspace)) return dh::fail(DH_ERR_INVALID, "%s: workspace must be 16-byte aligned", me);
  WgradArgs a{};
  a.gr = {group_ptr, M, (int)G};
  a.N = N; a.K = K; a.dY = dY; a.X = X; a.ldy = ldy; a.ldx = ldx; a.dW = dW; a.ldw = ldw; a.stride_w = stride_w; a.dw_bf16 = dw_dtype == DH_DTYPE_BF16;
  a.db = db; a.ld_db = ld_db; a.shift = wgrad_shift(M, N, K);
  const int64_t slots = wgrad_slots(M, a.shift);
  a.part_w = static_cast<float*>(workspace);
  a.part_b = a.part_w + slots * N * K;
  hipStream_t st = dh::as_stream(stream);
  int launched;
  if (dtype != DH_DTYPE_BF16) launched = wgrad_launch<float, Tile<float, true, true, 2, 2, 2, 2>, false>(me, a, st);
  else if (dma_rows(dY, ldy) && dma_rows(X, ldx) && N % 8 == 0 && K % 8 == 0) launched = wgrad_launch<uint16_t, DmaTile<true, true, 2, 2, 2, 2>, true>(me, a, st);
  else launched = wgrad_launch<uint16_t, Tile<uint16_t, true, true, 2, 2, 2, 2>, false>(me, a, st);
  if (launched != DH_OK) return launched;
  if ((M >> a.shift) > 0)
    hipLaunchKernelGGL(wgrad_join_kernel, dim3((unsigned)dh::ceil_div(N * K + N, 256), (unsigned)(M >> a.shift)), dim3(256), 0, st, a);
  return dh::check_launch(me);
}
