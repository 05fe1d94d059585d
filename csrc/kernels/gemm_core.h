// Block-tile matrix product on gfx950 MFMA, shared by the classifier loss (linear_xent.hip) and the
// orthogonalisation (newton_schulz.hip): acc[m][n] = sum_k sum_(p,q) A_p(m, k) B_q(n, k).
//
// Operands are 16-bit matrices in memory, in one of two forms:
//   rows  (T = false): element (r, k) at r * ld + k, the reduction runs along the row
//   cols  (T = true):  element (r, k) at k * ld + r, the reduction runs down the column
// (a `rows` operand whose extent is no multiple of 8 holds zeros up to the next one), so all of
// A B^T, A B and A^T B run without a transposed copy: a `rows` fragment is one ds_read_b128,
// a `cols` fragment two ds_read_b64_tr_b16 (the hardware's transposed read).
//
// PL planes: a value may be held as a sum of PL 16-bit numbers (PL = 2: two fp16, 22 bits; PL = 3:
// three bf16, 24 bits), each plane a matrix of its own.  A step then multiplies the pairs (p, q) with
// p + q < PL: what is left out is below 2^-22 (2^-24) of the product of the two largest.
//
// One step covers BK reduction elements.  All planes of both operands are copied to LDS by buffer
// loads that bypass the registers (raw_ptr_buffer_load_lds, 16 bytes a lane): the lane's offset is
// fixed for the whole loop, only a scalar moves, and the buffer's bound turns rows past the end into
// zeros.  The copy fills LDS in lane order, so the XOR swizzle that keeps fragment reads free of bank
// conflicts is applied to the source chunk.  NST buffers in a ring, one barrier a step: it publishes
// the step's tiles and retires the reads of the buffer that the next copy overwrites.
//
// The MFMA takes B as its row operand: a lane then holds, for one m (lane & 15), four neighbouring n
// (4 (lane >> 4) + e), which makes row-wise softmax statistics cheap and stores 8- or 16-byte wide.
#pragma once
#include "common.h"

namespace pmd {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(8))) short s16x8;

template <bool F16>
__device__ __forceinline__ f32x4 mm16(const s16x8& a, const s16x8& b, const f32x4& c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
}

// One operand of the whole product.  ld and the plane pointers are multiples of 8 elements / 16 bytes.
template <int PL>
struct GemmOperand {
  const unsigned short* plane[PL];
  long long ld;
  int rows;  // extent of m (or n)
};

constexpr unsigned kGemmOob = 0x80000000u;  // a buffer offset past every bound: reads zero
constexpr long long kGemmMaxLd = 1ll << 21; // 256 rows of this many 16-bit elements stay below 2^31 bytes

template <int BM_, int BN_, int WM_, int WN_, int BK_, int NST_, int PL_, bool TA_, bool TB_, bool F16_>
struct Gemm {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, BK = BK_, NST = NST_, PL = PL_;
  static constexpr bool TA = TA_, TB = TB_, F16 = F16_;
  static constexpr int NW = WM * WN, NT = 64 * NW;
  static constexpr int TM = BM / WM, TN = BN / WN, MI = TM / 16, NI = TN / 16;
  static constexpr int A_PLANE = BM * BK * 2, B_PLANE = BN * BK * 2;
  static constexpr int STAGE = PL * (A_PLANE + B_PLANE), LDS = NST * STAGE;
  static constexpr int LA = A_PLANE / (NT * 16), LB = B_PLANE / (NT * 16);  // loads per thread and plane
  static_assert(LA >= 1 && LB >= 1 && BK % 32 == 0 && LDS <= 160 * 1024, "tile shape");
  typedef f32x4 Acc[MI][NI];

  // swizzle of the 16-byte chunks of a `rows` tile (BK * 2 bytes a row)
  static __device__ __forceinline__ int swz_rows(int row) { return BK == 64 ? row & 7 : (row >> 2) & 2; }
  // swizzle of the 32-byte windows of a `cols` tile (COLS * 2 bytes a row)
  template <int COLS>
  static __device__ __forceinline__ int swz_cols(int row) {
    if constexpr (COLS >= 128) return (row & 3) | (((row >> 3) & 1) << 2);
    return ((row >> 1) & 1) | ((row >> 2) & 2);
  }

  // byte offset, within the operand's tile in memory, of the chunk that lane `tid` copies in load i
  template <int ROWS, bool T>
  static __device__ __forceinline__ unsigned src_off(int i, int tid, long long ld, int row_end, int* kchunk) {
    constexpr int CH = T ? ROWS / 8 : BK / 8;  // chunks of an LDS row
    const int L = i * NT + tid, row = L / CH, slot = L - row * CH;
    if constexpr (T) {
      const int chunk = (((slot >> 1) ^ swz_cols<ROWS>(row)) << 1) | (slot & 1);
      *kchunk = 0;
      return chunk * 8 < row_end ? (unsigned)(row * ld * 2 + chunk * 16) : kGemmOob;
    } else {
      const int chunk = slot ^ swz_rows(row);
      *kchunk = chunk * 8;
      return row < row_end ? (unsigned)(row * ld * 2 + chunk * 16) : kGemmOob;
    }
  }

  struct Loader {
    unsigned off[LA + LB];
    int kc[LA + LB];
    const char *a[PL], *b[PL];
    long long lda, ldb;
    int ra, rb;  // rows left from the tile's start
    int K;

    __device__ __forceinline__ Loader(const GemmOperand<PL>& A, const GemmOperand<PL>& B, int m0, int n0, int K_,
                                      int tid)
        : lda(A.ld), ldb(B.ld), ra(A.rows - m0), rb(B.rows - n0), K(K_) {
#pragma unroll
      for (int i = 0; i < LA; ++i) off[i] = src_off<BM, TA>(i, tid, lda, ra, &kc[i]);
#pragma unroll
      for (int i = 0; i < LB; ++i) off[LA + i] = src_off<BN, TB>(i, tid, ldb, rb, &kc[LA + i]);
#pragma unroll
      for (int p = 0; p < PL; ++p) {
        a[p] = reinterpret_cast<const char*>(A.plane[p]) + (TA ? (long long)m0 * 2 : (long long)m0 * lda * 2);
        b[p] = reinterpret_cast<const char*>(B.plane[p]) + (TB ? (long long)n0 * 2 : (long long)n0 * ldb * 2);
      }
    }

    // bytes that may be read from the base of a tile whose reduction starts at k
    template <bool T, int ROWS>
    __device__ __forceinline__ int bound(long long ld, int rows, int k) const {
      const int r = min(rows, ROWS);
      if (r <= 0) return 0;
      if (T) return (int)((long long)(min(BK, K - k) - 1) * ld * 2 + (long long)r * 2);
      return (int)((long long)(r - 1) * ld * 2 + (long long)((K + 7) & ~7) * 2);
    }

    template <bool T, int N, int O>
    __device__ __forceinline__ void copy(const char* base, long long ld, int bytes, int k, char* dst, int wid) const {
      // `rows`: the reduction offset is the scalar offset; `cols`: it moves the 64-bit base
      const char* p = T ? base + (long long)k * ld * 2 : base;
      const __amdgpu_buffer_rsrc_t rs =
          __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p), 0, bytes, 0x00020000);
      const int so = T ? 0 : k * 2;
      const bool tail = !T && k + BK > K;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        unsigned vo = off[O + i];
        if (tail && k + kc[O + i] >= K) vo = kGemmOob;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rs, (__attribute__((address_space(3))) void*)(dst + (i * NW + wid) * 1024), 16, (int)vo, so, 0, 0);
      }
    }

    __device__ __forceinline__ void load(int k, char* stage, int wid) const {
      const int ba = bound<TA, BM>(lda, ra, k), bb = bound<TB, BN>(ldb, rb, k);
#pragma unroll
      for (int p = 0; p < PL; ++p) copy<TA, LA, 0>(a[p], lda, ba, k, stage + p * A_PLANE, wid);
#pragma unroll
      for (int p = 0; p < PL; ++p) copy<TB, LB, LA>(b[p], ldb, bb, k, stage + PL * A_PLANE + p * B_PLANE, wid);
    }
  };

  // N fragments of 16 rows x 32 reduction elements: rows r0 + 16 i + (lane & 15), k = ks * 32 + 8 (lane >> 4) ..
  template <int ROWS, bool T, int N>
  static __device__ __forceinline__ void frags(const char* tile, int r0, int ks, int lane, s16x8 (&f)[N]) {
    if constexpr (!T) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int row = r0 + i * 16 + (lane & 15), chunk = ks * 4 + (lane >> 4);
        f[i] = *reinterpret_cast<const s16x8*>(tile + row * (BK * 2) + ((chunk ^ swz_rows(row)) << 4));
      }
    } else {
      const int k = ks * 32 + 8 * (lane >> 4) + ((lane >> 2) & 3);
      unsigned addr[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int byte = (r0 + i * 16 + 4 * (lane & 3)) * 2;
        const char* p = tile + k * (ROWS * 2) + (((byte >> 5) ^ swz_cols<ROWS>(k)) << 5) + (byte & 31);
        addr[i] = (unsigned)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
      }
      read_tr<4 * ROWS * 2>(addr, f);  // rows k and k + 4 have the same swizzle
    }
  }

  // Transposed reads, lo halves at the addresses and hi halves OFF bytes further, with their wait: ahead of
  // the builtin (__builtin_amdgcn_ds_read_tr16_b64_v4i16) the compiler waits for every copy to LDS in
  // flight, the next step's too, so loads and products took turns.  All of an operand's reads share one wait.
  template <int OFF>
  static __device__ __forceinline__ void read_tr(const unsigned (&p)[1], s16x8 (&f)[1]) {
    s16x4 l0, h0;
    asm volatile("ds_read_b64_tr_b16 %0, %2\n\tds_read_b64_tr_b16 %1, %2 offset:%3\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(l0), "=&v"(h0) : "v"(p[0]), "n"(OFF));
    f[0] = join(l0, h0);
  }
  template <int OFF>
  static __device__ __forceinline__ void read_tr(const unsigned (&p)[2], s16x8 (&f)[2]) {
    s16x4 l0, h0, l1, h1;
    asm volatile("ds_read_b64_tr_b16 %0, %4\n\tds_read_b64_tr_b16 %1, %4 offset:%6\n\t"
                 "ds_read_b64_tr_b16 %2, %5\n\tds_read_b64_tr_b16 %3, %5 offset:%6\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(l0), "=&v"(h0), "=&v"(l1), "=&v"(h1) : "v"(p[0]), "v"(p[1]), "n"(OFF));
    f[0] = join(l0, h0);
    f[1] = join(l1, h1);
  }
  template <int OFF>
  static __device__ __forceinline__ void read_tr(const unsigned (&p)[4], s16x8 (&f)[4]) {
    s16x4 l0, h0, l1, h1, l2, h2, l3, h3;
    asm volatile("ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %10 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %6, %11\n\tds_read_b64_tr_b16 %7, %11 offset:%12\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(l0), "=&v"(h0), "=&v"(l1), "=&v"(h1), "=&v"(l2), "=&v"(h2), "=&v"(l3), "=&v"(h3)
                 : "v"(p[0]), "v"(p[1]), "v"(p[2]), "v"(p[3]), "n"(OFF));
    f[0] = join(l0, h0);
    f[1] = join(l1, h1);
    f[2] = join(l2, h2);
    f[3] = join(l3, h3);
  }
  template <int OFF>
  static __device__ __forceinline__ void read_tr(const unsigned (&p)[8], s16x8 (&f)[8]) {
    s16x4 l0, h0, l1, h1, l2, h2, l3, h3, l4, h4, l5, h5, l6, h6, l7, h7;
    asm volatile("ds_read_b64_tr_b16 %0, %16\n\tds_read_b64_tr_b16 %1, %16 offset:%24\n\t"
                 "ds_read_b64_tr_b16 %2, %17\n\tds_read_b64_tr_b16 %3, %17 offset:%24\n\t"
                 "ds_read_b64_tr_b16 %4, %18\n\tds_read_b64_tr_b16 %5, %18 offset:%24\n\t"
                 "ds_read_b64_tr_b16 %6, %19\n\tds_read_b64_tr_b16 %7, %19 offset:%24\n\t"
                 "ds_read_b64_tr_b16 %8, %20\n\tds_read_b64_tr_b16 %9, %20 offset:%24\n\t"
                 "ds_read_b64_tr_b16 %10, %21\n\tds_read_b64_tr_b16 %11, %21 offset:%24\n\t"
                 "ds_read_b64_tr_b16 %12, %22\n\tds_read_b64_tr_b16 %13, %22 offset:%24\n\t"
                 "ds_read_b64_tr_b16 %14, %23\n\tds_read_b64_tr_b16 %15, %23 offset:%24\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(l0), "=&v"(h0), "=&v"(l1), "=&v"(h1), "=&v"(l2), "=&v"(h2), "=&v"(l3), "=&v"(h3), "=&v"(l4),
                   "=&v"(h4), "=&v"(l5), "=&v"(h5), "=&v"(l6), "=&v"(h6), "=&v"(l7), "=&v"(h7)
                 : "v"(p[0]), "v"(p[1]), "v"(p[2]), "v"(p[3]), "v"(p[4]), "v"(p[5]), "v"(p[6]), "v"(p[7]), "n"(OFF));
    f[0] = join(l0, h0);
    f[1] = join(l1, h1);
    f[2] = join(l2, h2);
    f[3] = join(l3, h3);
    f[4] = join(l4, h4);
    f[5] = join(l5, h5);
    f[6] = join(l6, h6);
    f[7] = join(l7, h7);
  }
  static __device__ __forceinline__ s16x8 join(const s16x4& l, const s16x4& h) {
    return s16x8{l[0], l[1], l[2], l[3], h[0], h[1], h[2], h[3]};
  }

  // `rows` operands: the fragments of one 32-deep slice are read ahead of the MFMAs of the slice before; in
  // the 256-wide one-plane tile (64 MFMAs a step) the schedule is pinned to a read every second MFMA, which
  // measured 3-4% over the compiler's own order (reads just ahead of their use): 3.91 against 4.05 ms for
  // 8,192 x 131,072 x 2,048.
  static __device__ __forceinline__ void step(const char* stage, Acc& acc, int wm, int wn, int lane) {
    const char* At = stage;
    const char* Bt = stage + PL * A_PLANE;
    if constexpr (PL == 1 && MI * NI == 32 && !TA && !TB) {
      s16x8 af[2][MI], bf[2][NI];
#pragma unroll
      for (int ks = 0; ks <= BK / 32; ++ks) {
        if (ks < BK / 32) {
          frags<BN, TB>(Bt, wn * TN, ks, lane, bf[ks & 1]);
          frags<BM, TA>(At, wm * TM, ks, lane, af[ks & 1]);
        }
        if (ks > 0) {
#pragma unroll
          for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j)
              acc[i][j] = mm16<F16>(bf[(ks - 1) & 1][j], af[(ks - 1) & 1][i], acc[i][j]);
        }
      }
      __builtin_amdgcn_sched_group_barrier(0x100, MI + NI, 0);  // LDS reads of the first slice
#pragma unroll
      for (int q = 0; q < MI + NI; ++q) {
        __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);  // MFMAs
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      return;
    }
#pragma unroll
    for (int ks = 0; ks < BK / 32; ++ks) {
      s16x8 af[PL][MI], bf[PL][NI];
#pragma unroll
      for (int p = 0; p < PL; ++p) {  // `rows` operands first: their reads share the others' wait
        if constexpr (TA) {
          frags<BN, TB>(Bt + p * B_PLANE, wn * TN, ks, lane, bf[p]);
          frags<BM, TA>(At + p * A_PLANE, wm * TM, ks, lane, af[p]);
        } else {
          frags<BM, TA>(At + p * A_PLANE, wm * TM, ks, lane, af[p]);
          frags<BN, TB>(Bt + p * B_PLANE, wn * TN, ks, lane, bf[p]);
        }
      }
      // the smallest products first: they would vanish against a sum that holds the largest
#pragma unroll
      for (int s = PL - 1; s >= 0; --s)
#pragma unroll
        for (int p = 0; p <= s; ++p)
#pragma unroll
          for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = mm16<F16>(bf[s - p][j], af[p][i], acc[i][j]);
    }
  }

  template <int N>
  static __device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
  }

  // acc = product over k in [k0, k1) (k0 a multiple of BK; k1 = the operands' extent, or a multiple of
  // BK below it).  Ends with every wave past its LDS reads: the caller may reuse smem.
  static __device__ __forceinline__ void run(const GemmOperand<PL>& A, const GemmOperand<PL>& B, int m0, int n0,
                                             int k0, int k1, char* smem, Acc& acc) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wid / WN, wn = wid % WN;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const Loader ld(A, B, m0, n0, k1, tid);
    constexpr int LPS = PL * (LA + LB);  // loads of a step
    static_assert(NST >= 2 && NST <= 5 && (NST - 2) * LPS <= 63, "counted waits");
    const int steps = (k1 - k0 + BK - 1) / BK;
#pragma unroll
    for (int s = 0; s < NST - 1; ++s)
      if (s < steps) ld.load(k0 + s * BK, smem + s * STAGE, wid);
    int buf = 0;
    for (int t = 0; t < steps; ++t) {
      // step t's copies have landed once at most those of the steps behind it are in flight
      const int later = min(NST - 2, steps - 1 - t);
      if (NST >= 5 && later >= 3) wait_loads<3 * LPS>();
      else if (NST >= 4 && later == 2) wait_loads<2 * LPS>();
      else if (NST >= 3 && later == 1) wait_loads<LPS>();
      else wait_loads<0>();
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (t + NST - 1 < steps) {
        int nb = buf + NST - 1;
        if (nb >= NST) nb -= NST;
        ld.load(k0 + (t + NST - 1) * BK, smem + nb * STAGE, wid);
      }
      step(smem + buf * STAGE, acc, wm, wn, lane);
      if (++buf == NST) buf = 0;
    }
    __syncthreads();
  }
};

// Order of a grid of tm x tn tiles: each XCD takes a contiguous run of the order (xcd_remap), and the
// order walks bands of 8 row tiles column by column, so that the blocks of an XCD that run together
// share both operands' tiles in its L2.
__device__ __forceinline__ void tile_of(int bid, int nblocks, int tm, int tn, int& im, int& in) {
  const int L = xcd_remap(bid, nblocks);
  const int band = 8 * tn, b = L / band, r = L - b * band;
  const int h = min(8, tm - b * 8);
  in = r / h;
  im = b * 8 + (r - in * h);
}

}  // namespace pmd
