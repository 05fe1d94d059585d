// Newton-Schulz orthogonalisation of weight updates, many matrices in a launch (gfx950).
//
//   X_0 = U / (|U|_F + eps), taken with its shorter side s first (l the longer)
//   S = X X^T,  P = b S + c S S,  X <- a X + P X          `steps` times
//   out = beta out + alpha X                              (alpha times a device scalar, if given)
//
// The odd polynomial a + b t^3 + c t^5 acts on the singular values and leaves the singular vectors;
// a = 3.4445 multiplies the smallest ones by 484 in five steps, and every rounding error with them, so
// one bf16 product is off by percents here.  Matrices are held as two fp16 planes (22 bits) and every
// product takes three MFMAs (gemm_core.h): errors stay near those of fp32 arithmetic, at several
// times the rate of the fp32 MFMA.  fp16 needs scaling: |X|_2 <= 1 at the start, and the largest value
// the polynomial takes bounds every entry of X, S and P at every step, so the host picks powers of
// two that put the bound just below fp16's range (ns_scales).
//
// S and P are symmetric (polynomials of X X^T): only tiles on and below the diagonal are computed, and
// stored twice.  X is read as the `cols` operand of P X, so no transposed copy of it exists.
//
// One launch covers every matrix of the group: the grid is the list of all their tiles.  The Gram
// product runs down the long side; its reduction is split, for enough blocks, into fp32 slabs that a
// second kernel joins in order.  No atomics.
#include "gemm_core.h"

#include <math.h>

#include <algorithm>
#include <vector>

namespace pmd {

namespace {

typedef _Float16 f16_t;

// The matrices of a group, by value in the kernel arguments of the first kernel (which writes the table
// below) and of the one-block kernel.
struct NsDim {
  int s, l;          // shorter, longer side
  long long xo, so;  // element offsets in the workspace: X (2 buffers x 2 planes), S and P (2 planes each)
};
struct NsIo {
  const void* src;
  void* dst;
  float alpha;
  int tall;          // src is l x s: taken transposed
};
struct NsGroup {
  int count;
  NsDim d[kNsGroup];
  NsIo io[kNsGroup];
};

__host__ __device__ inline int up8(int v) { return (v + 7) & ~7; }
__host__ __device__ inline long long cdiv(long long a, long long b) { return (a + b - 1) / b; }
__host__ __device__ inline int tri(int t) { return t * (t + 1) / 2; }

// How the phases of a group are cut into blocks.
enum NsPhase { kNorm, kStart, kGram, kJoin, kPoly, kUpdate, kPhases };
constexpr int kNormBlocks = 256;  // partial sums of a matrix's norm, at most
struct NsCut {
  int kc;                                   // reduction of a Gram block
  int gram_small, poly_small, upd_small;    // 64-wide tiles for all
  int gram_wide, poly_wide;                 // 192-wide tiles for all
  int upd_big;                              // 256-wide tiles for all
};
struct NsBlocks {
  int tile, splits, blocks;  // splits: blocks that share a sum (of a Gram tile, of the norm)
};
__host__ __device__ inline NsBlocks ns_blocks(int phase, int s, int l, const NsCut& c) {
  const int t = s <= 64 ? 64 : 128, lp = up8(l);
  NsBlocks b{t, 1, 0};
  if (phase == kNorm) {
    const long long n = cdiv((long long)s * l, 16384);
    b.splits = b.blocks = n < kNormBlocks ? (int)n : kNormBlocks;
  } else if (phase == kStart) {
    b.blocks = (int)(cdiv(s, 64) * cdiv(lp, 64));
  } else if (phase == kGram || phase == kJoin) {
    b.tile = c.gram_wide ? 192 : c.gram_small ? 64 : t;
    b.splits = (int)cdiv(l, c.kc);
    const int tiles = tri((int)cdiv(s, b.tile));
    b.blocks = phase == kGram ? tiles * b.splits : b.splits > 1 ? tiles * (b.tile * b.tile / 1024) : 0;
  } else if (phase == kPoly) {
    b.tile = c.poly_wide ? 192 : c.poly_small ? 64 : t;
    b.blocks = tri((int)cdiv(s, b.tile));
  } else {
    b.tile = c.upd_big ? 256 : c.upd_small ? 64 : t;
    b.blocks = (int)(cdiv(s, b.tile) * cdiv(lp, b.tile));
  }
  return b;
}

// The same in device memory, written by the first kernel of a call: one load finds a block's matrix, and
// the later launches carry no descriptions.
struct NsTable {
  int t0[kPhases][64];  // first block of each matrix (past the last matrix: never reached)
  NsBlocks b[kPhases][kNsGroup];
  NsDim d[kNsGroup];
  NsIo io[kNsGroup];
};

// the matrix of a block: one load and a ballot
__device__ __forceinline__ int find_matrix(const NsTable* t, int phase, int block) {
  const unsigned long long m = __ballot(t->t0[phase][threadIdx.x & 63] <= block);
  return 63 - __clzll(m);
}

__device__ __forceinline__ float ns_ld(const void* p, long long i, bool f32) {
  return f32 ? static_cast<const float*>(p)[i] : bf2f(static_cast<const bf16_t*>(p)[i]);
}

// v is pinned to its fp32 rounding: where it is a product, the compiler else rounds the product straight to fp16
// for one of hi and its use in lo, and twice for the other, and the two differ now and then by a whole fp16 step
__device__ __forceinline__ void split2(float v, unsigned short& hi, unsigned short& lo) {
  asm("" : "+v"(v));
  const f16_t h = (f16_t)v, l = (f16_t)(v - (float)h);
  hi = __builtin_bit_cast(unsigned short, h);
  lo = __builtin_bit_cast(unsigned short, l);
}
__device__ __forceinline__ float join2(unsigned short hi, unsigned short lo) {
  return (float)__builtin_bit_cast(f16_t, hi) + (float)__builtin_bit_cast(f16_t, lo);
}

// four neighbours of a matrix in two planes, o a multiple of 4
__device__ __forceinline__ void put_planes(unsigned short* p, long long plane, long long o, const float (&v)[4]) {
  unsigned short h[4], l[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) split2(v[e], h[e], l[e]);
  *reinterpret_cast<uint2*>(p + o) = make_uint2(h[0] | ((uint32_t)h[1] << 16), h[2] | ((uint32_t)h[3] << 16));
  *reinterpret_cast<uint2*>(p + plane + o) = make_uint2(l[0] | ((uint32_t)l[1] << 16), l[2] | ((uint32_t)l[3] << 16));
}

// ------------------------------------------------------------- norm, start
// part [matrix][kNormBlocks] = sums of squares, in fp64 (entries of 1e-30 or 1e30 neither vanish nor
// overflow); a block takes at least 16,384 elements.  Block 0 also writes the table.
__global__ __launch_bounds__(256) void ns_norm_kernel(NsGroup g, NsCut cut, int f32, double* __restrict__ part,
                                                      NsTable* __restrict__ table) {
  __shared__ double red[4];
  // a lane per matrix (every wave of the block alike): prefix sums of the phases' blocks
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const bool have = lane < g.count;
  const int ms = have ? g.d[lane].s : 0, ml = have ? g.d[lane].l : 0;
  auto first_block = [&](int n) {
    int t = n;
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(t, o, 64);
      if (lane >= o) t += v;
    }
    return have ? t - n : 0x7fffffff;
  };
  const int nb0 = have ? ns_blocks(kNorm, ms, ml, cut).blocks : 0, f0 = first_block(nb0);
  const int k = 63 - __clzll(__ballot(f0 <= (int)blockIdx.x));
  const int b = blockIdx.x - __shfl(f0, k, 64), nb = __shfl(nb0, k, 64);
  if (blockIdx.x == 0) {
    for (int ph = wid; ph < kPhases; ph += 4) {
      const NsBlocks n = have ? ns_blocks(ph, ms, ml, cut) : NsBlocks{0, 0, 0};
      table->t0[ph][lane] = first_block(n.blocks);
      if (have) table->b[ph][lane] = n;
    }
    if (have && wid == 3) {
      table->d[lane] = g.d[lane];
      table->io[lane] = g.io[lane];
    }
  }
  const long long n = (long long)g.d[k].s * g.d[k].l;
  const void* src = g.io[k].src;
  double s = 0.0;
  const long long n4 = reinterpret_cast<uintptr_t>(src) % 16 == 0 ? n >> 2 : 0;  // whole vectors
  for (long long i = b * 256ll + threadIdx.x; i < n4; i += nb * 256ll) {
    float v[4];
    if (f32) {
      const float4 t = static_cast<const float4*>(src)[i];
      v[0] = t.x;
      v[1] = t.y;
      v[2] = t.z;
      v[3] = t.w;
    } else {
      const uint2 t = static_cast<const uint2*>(src)[i];
      v[0] = bf2f(t.x & 0xffff);
      v[1] = bf2f(t.x >> 16);
      v[2] = bf2f(t.y & 0xffff);
      v[3] = bf2f(t.y >> 16);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) s += (double)v[e] * v[e];
  }
  for (long long i = n4 * 4 + b * 256ll + threadIdx.x; i < n; i += nb * 256ll) {
    const double v = ns_ld(src, i, f32);
    s += v * v;
  }
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[k * kNormBlocks + b] = ((red[0] + red[1]) + red[2]) + red[3];
}

// X_0 planes [s][up8(l)] of one 64 x 64 tile, through LDS when the matrix is taken transposed
__global__ __launch_bounds__(256) void ns_start_kernel(const NsTable* __restrict__ tab, int f32,
                                                       const double* __restrict__ part, unsigned short* __restrict__ ws,
                                                       float eps, float scale) {
  __shared__ float tile[64][65];
  __shared__ float inv_s;
  const int k = find_matrix(tab, kStart, blockIdx.x), t = blockIdx.x - tab->t0[kStart][k];
  const NsDim d = tab->d[k];
  const NsIo io = tab->io[k];
  const int s = d.s, l = d.l, lp = up8(l), sums = tab->b[kNorm][k].splits;
  const int tl = (lp + 63) / 64, r0 = (t / tl) * 64, c0 = (t % tl) * 64;
  if (threadIdx.x < 64) {
    double v = 0.0;
    for (int i = threadIdx.x; i < sums; i += 64) v += part[k * kNormBlocks + i];
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if (threadIdx.x == 0) inv_s = (float)(1.0 / (sqrt(v) + (double)eps)) * scale;
  }
  const bool tall = io.tall;
  const int a = threadIdx.x & 63, b = threadIdx.x >> 6;
#pragma unroll 8
  for (int i = b; i < 64; i += 4) {  // a: along the source's rows
    const int r = tall ? r0 + a : r0 + i, c = tall ? c0 + i : c0 + a;
    const float v = r < s && c < l ? ns_ld(io.src, tall ? (long long)c * s + r : (long long)r * l + c, f32) : 0.f;
    if (tall) tile[a][i] = v;
    else tile[i][a] = v;
  }
  __syncthreads();
  const float inv = inv_s;
  unsigned short* x = ws + d.xo;
  const long long plane = (long long)s * lp;
  const int q = (threadIdx.x & 15) * 4;
#pragma unroll
  for (int i = threadIdx.x >> 4; i < 64; i += 16) {
    const int r = r0 + i, c = c0 + q;
    if (r >= s || c >= lp) continue;
    const float v[4] = {tile[i][q] * inv, tile[i][q + 1] * inv, tile[i][q + 2] * inv, tile[i][q + 3] * inv};
    put_planes(x, plane, (long long)r * lp + c, v);
  }
}

// ------------------------------------------------------------------ products
__device__ __forceinline__ GemmOperand<2> ns_operand(const unsigned short* p, long long plane, int ld, int rows) {
  GemmOperand<2> o;
  o.plane[0] = p;
  o.plane[1] = p + plane;
  o.ld = ld;
  o.rows = rows;
  return o;
}

// tile t of the lower triangle, row by row
__device__ __forceinline__ void tri_of(int t, int& im, int& in) {
  int r = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
  while ((r + 1) * (r + 2) / 2 <= t) ++r;
  while (r * (r + 1) / 2 > t) --r;
  im = r;
  in = t - r * (r + 1) / 2;
}

// four neighbours n.. of row m of a symmetric matrix [s][up8(s)] (2 planes), and their mirror images.
// Four neighbouring lanes hold four neighbouring rows m; they transpose their 4 x 4 values among
// themselves, so that the mirror image is stored 8 bytes wide too (all 64 lanes call this, with m and n
// multiples of 4 apart from the lane's own m & 3).
__device__ __forceinline__ void put_sym(unsigned short* p, int s, int m, int n, const float (&v)[4], bool mirror) {
  const int ld = up8(s);
  const long long plane = (long long)s * ld;
  if (m < s && n < ld) put_planes(p, plane, (long long)m * ld + n, v);
  if (!mirror) return;
  float t[4] = {v[0], v[1], v[2], v[3]};
  const int q = threadIdx.x & 3;
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    const bool up = q & o;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (!(e & o)) {
        const float r = __shfl_xor(up ? t[e] : t[e | o], o, 64);
        if (up) t[e] = r;
        else t[e | o] = r;
      }
  }
  const int row = n + q, col = m & ~3;  // now t[e] belongs to (m & ~3) + e, n + q
  if (row < s && col < ld) put_planes(p, plane, (long long)row * ld + col, t);
}

__device__ __forceinline__ void join4(const uint2& h, const uint2& l, float (&v)[4]) {
  v[0] = join2(h.x & 0xffff, l.x & 0xffff);
  v[1] = join2(h.x >> 16, l.x >> 16);
  v[2] = join2(h.y & 0xffff, l.y & 0xffff);
  v[3] = join2(h.y >> 16, l.y >> 16);
}

// An epilogue's rows of 16, in runs short enough that the run's operands (4 registers a tile) fit beside
// the accumulators: all of a run's loads are issued before the first is used.
template <class G, typename F>
__device__ __forceinline__ void for_rows(F&& f) {
  constexpr int R = G::MI * G::NI > 16 ? 16 / G::NI : G::MI;
  static_assert(G::MI % R == 0, "whole runs");
  f(std::integral_constant<int, 0>{}, std::integral_constant<int, R>{});
  if constexpr (G::MI > R) f(std::integral_constant<int, R>{}, std::integral_constant<int, R>{});
  if constexpr (G::MI > 2 * R) f(std::integral_constant<int, 2 * R>{}, std::integral_constant<int, R>{});
  static_assert(G::MI <= 3 * R, "three runs");
}

// the tiles (m + 16 i, n + 16 j) of a matrix in two planes (zero outside [rows][cols])
template <class G, int R>
__device__ __forceinline__ void load_planes(const unsigned short* p, long long plane, int ld, int rows, int cols, int m,
                                            int n, uint2 (&h)[R][G::NI], uint2 (&l)[R][G::NI]) {
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < G::NI; ++j) {
      const bool ok = m + i * 16 < rows && n + j * 16 < cols;
      const long long o = ok ? (long long)(m + i * 16) * ld + n + j * 16 : 0;
      const uint2 a = *reinterpret_cast<const uint2*>(p + o), b = *reinterpret_cast<const uint2*>(p + plane + o);
      h[i][j] = ok ? a : make_uint2(0, 0);
      l[i][j] = ok ? b : make_uint2(0, 0);
    }
}

// The kernels below take their tile per matrix: the grid of a group mixes 128- and 64-wide tiles (G1,
// G2: 256 threads each), a group of large matrices runs on 192- or 256-wide ones alone (G1 = G2).
template <class G1, class G2>
constexpr int ns_lds() {
  return G1::LDS > G2::LDS ? G1::LDS : G2::LDS;
}

// S = X X^T: planes scaled by out_scale / (X's scale)^2 in one go, or (split sums) slabs
// [block][BM][BN] of raw sums
template <class G>
__device__ __forceinline__ void ns_gram_tile(const NsDim& d, int splits, int L, int r, unsigned short* ws, int xbuf,
                                             int kc, float mul, float* slab, int slab_stride, char* smem) {
  const int t = r / splits, z = r - t * splits;
  int im, in;
  tri_of(t, im, in);
  const int lp = up8(d.l);
  const long long plane = (long long)d.s * lp;
  const GemmOperand<2> x = ns_operand(ws + d.xo + xbuf * 2 * plane, plane, lp, d.s);
  typename G::Acc acc;
  G::run(x, x, im * G::BM, in * G::BN, z * kc, min(d.l, (z + 1) * kc), smem, acc);
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, wm = wid / G::WN, wn = wid % G::WN;
#pragma unroll
  for (int i = 0; i < G::MI; ++i)
#pragma unroll
    for (int j = 0; j < G::NI; ++j) {
      const int ml = wm * G::TM + i * 16 + (lane & 15), nl = wn * G::TN + j * 16 + (lane >> 4) * 4;
      if (splits > 1) {
        *reinterpret_cast<float4*>(slab + (long long)L * slab_stride + ml * G::BN + nl) =
            make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
      } else {
        const float v[4] = {acc[i][j][0] * mul, acc[i][j][1] * mul, acc[i][j][2] * mul, acc[i][j][3] * mul};
        put_sym(ws + d.so, d.s, im * G::BM + ml, in * G::BN + nl, v, im != in);
      }
    }
}
template <class G1, class G2>
__global__ __launch_bounds__(G1::NT) void ns_gram_kernel(const NsTable* __restrict__ tab,
                                                         unsigned short* __restrict__ ws, int xbuf, int kc, float mul,
                                                         float* __restrict__ slab, int slab_stride) {
  __shared__ __attribute__((aligned(16))) char smem[ns_lds<G1, G2>()];
  const int L = xcd_remap(blockIdx.x, gridDim.x);
  const int k = find_matrix(tab, kGram, L), r = L - tab->t0[kGram][k];
  const NsDim d = tab->d[k];
  const NsBlocks b = tab->b[kGram][k];
  if (b.tile == G1::BM) ns_gram_tile<G1>(d, b.splits, L, r, ws, xbuf, kc, mul, slab, slab_stride, smem);
  else ns_gram_tile<G2>(d, b.splits, L, r, ws, xbuf, kc, mul, slab, slab_stride, smem);
}

// joins the slabs of the Gram tiles in order, 1,024 values a block
__global__ __launch_bounds__(256) void ns_join_kernel(const NsTable* __restrict__ tab, unsigned short* __restrict__ ws,
                                                      const float* __restrict__ slab, int slab_stride, float mul) {
  const int k = find_matrix(tab, kJoin, blockIdx.x), b = blockIdx.x - tab->t0[kJoin][k];
  const NsDim d = tab->d[k];
  const int BT = tab->b[kJoin][k].tile, splits = tab->b[kJoin][k].splits;
  const int per = BT * BT / 1024, t = b / per, part = b - t * per;
  int im, in;
  tri_of(t, im, in);
  const float* s0 = slab + (tab->t0[kGram][k] + (long long)t * splits) * slab_stride;
  const int u = part * 256 + threadIdx.x, q = u >> 2;  // four neighbouring lanes: four rows (put_sym)
  const int m = q / (BT / 4) * 4 + (u & 3), n = q % (BT / 4) * 4;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int z = 0; z < splits; ++z) {
    const float4 w = *reinterpret_cast<const float4*>(s0 + (long long)z * slab_stride + m * BT + n);
    v[0] += w.x;
    v[1] += w.y;
    v[2] += w.z;
    v[3] += w.w;
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) v[c] *= mul;
  put_sym(ws + d.so, d.s, im * BT + m, in * BT + n, v, im != in);
}

// P = b S + c S S (S's scale ss, P's scale sp)
template <class G>
__device__ __forceinline__ void ns_poly_tile(const NsDim& d, int t, unsigned short* ws, float b, float c, float inv_ss,
                                             float sp, char* smem) {
  int im, in;
  tri_of(t, im, in);
  const int ld = up8(d.s);
  const long long plane = (long long)d.s * ld;
  const unsigned short* S = ws + d.so;
  const GemmOperand<2> x = ns_operand(S, plane, ld, d.s);
  typename G::Acc acc;
  G::run(x, x, im * G::BM, in * G::BN, 0, d.s, smem, acc);
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, wm = wid / G::WN, wn = wid % G::WN;
  const float kc = c * inv_ss * inv_ss * sp, kb = b * inv_ss * sp;
  const int mb = im * G::BM + wm * G::TM + (lane & 15), nb = in * G::BN + wn * G::TN + (lane >> 4) * 4;
  for_rows<G>([&](auto i0, auto rows) {
    uint2 h[rows][G::NI], l[rows][G::NI];
    load_planes<G, rows>(S, plane, ld, d.s, ld, mb + i0 * 16, nb, h, l);
#pragma unroll
    for (int i = 0; i < rows; ++i)
#pragma unroll
      for (int j = 0; j < G::NI; ++j) {
        float sv[4], v[4];
        join4(h[i][j], l[i][j], sv);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fmaf(kc, acc[i0 + i][j][e], kb * sv[e]);
        put_sym(ws + d.so + 2 * plane, d.s, mb + (i0 + i) * 16, nb + j * 16, v, im != in);
      }
  });
}
template <class G1, class G2>
__global__ __launch_bounds__(G1::NT) void ns_poly_kernel(const NsTable* __restrict__ tab,
                                                         unsigned short* __restrict__ ws, float b, float c, float inv_ss,
                                                         float sp) {
  __shared__ __attribute__((aligned(16))) char smem[ns_lds<G1, G2>()];
  const int L = xcd_remap(blockIdx.x, gridDim.x);
  const int k = find_matrix(tab, kPoly, L), t = L - tab->t0[kPoly][k];
  const NsDim d = tab->d[k];
  if (tab->b[kPoly][k].tile == G1::BM) ns_poly_tile<G1>(d, t, ws, b, c, inv_ss, sp, smem);
  else ns_poly_tile<G2>(d, t, ws, b, c, inv_ss, sp, smem);
}

// four values (m, n..) of out = beta out + alpha X
__device__ __forceinline__ void ns_out(const NsIo& io, int f32, int s, int l, int m, int n, const float (&v)[4],
                                       float alpha, float beta) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (n + e >= l) continue;
    const long long q = io.tall ? (long long)(n + e) * s + m : (long long)m * l + n + e;
    if (f32) {
      float* dst = static_cast<float*>(io.dst) + q;
      *dst = beta != 0.f ? fmaf(alpha, v[e], beta * *dst) : alpha * v[e];
    } else {
      bf16_t* dst = static_cast<bf16_t*>(io.dst) + q;
      *dst = f2bf(beta != 0.f ? fmaf(alpha, v[e], beta * bf2f(*dst)) : alpha * v[e]);
    }
  }
}

struct NsStep {  // of the update: a, 1 / scales of X and P, scale of the next X; the last step's output
  float a, inv_sx, inv_sp, so, beta;
  int f32;
  const float* alpha_dev;
};

// X' = a X + P X into the other buffer, or (LAST) out = beta out + alpha X'
template <class G, bool LAST>
__device__ __forceinline__ void ns_update_tile(const NsDim& d, int t, const NsIo& io, unsigned short* ws, int xbuf,
                                               const NsStep& st, char* smem) {
  const int lp = up8(d.l), ld = up8(d.s);
  const int tm = (d.s + G::BM - 1) / G::BM, tn = (lp + G::BN - 1) / G::BN;
  const int band = 8 * tn, bb = t / band, rr = t - bb * band, h = min(8, tm - bb * 8);
  const int in = rr / h, im = bb * 8 + (rr - in * h);
  const long long xplane = (long long)d.s * lp, splane = (long long)d.s * ld;
  const unsigned short* X = ws + d.xo + xbuf * 2 * xplane;
  const GemmOperand<2> p = ns_operand(ws + d.so + 2 * splane, splane, ld, d.s);
  const GemmOperand<2> x = ns_operand(X, xplane, lp, lp);
  typename G::Acc acc;
  G::run(p, x, im * G::BM, in * G::BN, 0, d.s, smem, acc);
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, wm = wid / G::WN, wn = wid % G::WN;
  unsigned short* Y = ws + d.xo + (xbuf ^ 1) * 2 * xplane;
  const float kp = st.inv_sp * st.inv_sx, ka = st.a * st.inv_sx;
  float alpha = 0.f;
  if constexpr (LAST) alpha = io.alpha * (st.alpha_dev ? st.alpha_dev[0] : 1.f);
  const int mb = im * G::BM + wm * G::TM + (lane & 15), nb = in * G::BN + wn * G::TN + (lane >> 4) * 4;
  for_rows<G>([&](auto i0, auto rows) {
    uint2 hh[rows][G::NI], ll[rows][G::NI];
    load_planes<G, rows>(X, xplane, lp, d.s, lp, mb + i0 * 16, nb, hh, ll);
#pragma unroll
    for (int i = 0; i < rows; ++i)
#pragma unroll
      for (int j = 0; j < G::NI; ++j) {
        const int m = mb + (i0 + i) * 16, n = nb + j * 16;
        if (m >= d.s || n >= lp) continue;
        float xv[4], v[4];
        join4(hh[i][j], ll[i][j], xv);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fmaf(kp, acc[i0 + i][j][e], ka * xv[e]);
        if constexpr (LAST) {
          ns_out(io, st.f32, d.s, d.l, m, n, v, alpha, st.beta);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] *= st.so;
          put_planes(Y, xplane, (long long)m * lp + n, v);
        }
      }
  });
}
template <class G1, class G2, bool LAST>
__global__ __launch_bounds__(G1::NT) void ns_update_kernel(const NsTable* __restrict__ tab,
                                                           unsigned short* __restrict__ ws, int xbuf, NsStep st) {
  __shared__ __attribute__((aligned(16))) char smem[ns_lds<G1, G2>()];
  const int L = xcd_remap(blockIdx.x, gridDim.x);
  const int k = find_matrix(tab, kUpdate, L), t = L - tab->t0[kUpdate][k];
  const NsDim d = tab->d[k];
  const NsIo io = LAST ? tab->io[k] : NsIo{};
  if (tab->b[kUpdate][k].tile == G1::BM) ns_update_tile<G1, LAST>(d, t, io, ws, xbuf, st, smem);
  else ns_update_tile<G2, LAST>(d, t, io, ws, xbuf, st, smem);
}

// ------------------------------------------------------------ small matrices
// A matrix that fits LDS runs all its steps in one block of 16 waves on v_mfma_f32_16x16x4_f32: no
// launches between the products, and fp32's own precision.  With a shorter side of at most 16 the
// products run in fp64 (v_mfma_f64_16x16x4_f64): the few singular values share few errors, which then
// do not average out.  X stays fp32 in LDS.
// Measured as captured graphs against the many-block kernels: 64 x 27 26 / 62 us, 64 x 64 44 / 76, 16 x 1,000
// 51 / 85, 64 x 256 81 / 89, 96 x 96 95 / 87, 8 x 4,096 136 / 92 -- the bound on the work keeps the gain, and
// shorter sides of at most 16 stay here for their accuracy.
constexpr int kSmallThreads = 1024, kSmallWaves = kSmallThreads / 64;
constexpr int kSmallElems = 32768;          // s * l: the matrix in at most 136 KiB of LDS
constexpr int kSmallSide = 96;              // s: S and P beside it
constexpr long long kSmallWork = 1 << 18;   // s * s * l

typedef __attribute__((ext_vector_type(4))) double f64x4;

template <bool F64>
struct SmallT {
  typedef float R;
  typedef f32x4 Acc;
  static constexpr int kSplit = kSmallWaves;  // waves that may share a Gram tile
  static __device__ __forceinline__ Acc mm(R a, R b, Acc c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ int row(int lane, int e) { return (lane >> 4) * 4 + e; }
};
template <>
struct SmallT<true> {
  typedef double R;
  typedef f64x4 Acc;
  static constexpr int kSplit = kSmallWaves / 2;
  static __device__ __forceinline__ Acc mm(R a, R b, Acc c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ int row(int lane, int e) { return e * 4 + (lane >> 4); }
};

__host__ __device__ inline bool small_f64(int s) { return s <= 16; }
// row strides: X's a multiple of 64 floats + 4 (the 16 rows x 4 columns of a fragment hit all banks)
__host__ __device__ inline int small_ldx(int l) { return (l + 63) / 64 * 64 + 4; }
__host__ __device__ inline int small_lds(int s) { return (s + 15) / 16 * 16 + 4; }
inline long long small_bytes(int s, int l) {
  const long long T = (s + 15) / 16, rows = (long long)s * small_ldx(l) * 4;
  return small_f64(s) ? rows + (2 * 16 * small_lds(s) + SmallT<true>::kSplit * 256) * 8
                      : rows + (2 * T * 16 * small_lds(s) + SmallT<false>::kSplit * 256) * 4;
}
inline bool small_ok(int s, int l) {
  return s <= kSmallSide && (long long)s * l <= kSmallElems && (small_f64(s) || (long long)s * s * l <= kSmallWork) &&
         small_bytes(s, l) <= 160 * 1024 - 512;
}

// one 16 x 16 tile of A B^T over k0 <= k < k1 (multiples of 16): rows m0.. of A, n0.. of B (zero past
// `rows`), k along the rows
template <bool F64, typename E>
__device__ __forceinline__ typename SmallT<F64>::Acc small_dot(const E* M, int ld, int m0, int n0, int rows, int k0,
                                                               int k1, int lane) {
  typedef typename SmallT<F64>::R R;
  const int r = lane & 15, kk = lane >> 4;
  const bool oka = m0 + r < rows, okb = n0 + r < rows;
  const E* pa = M + (oka ? m0 + r : 0) * ld + kk;
  const E* pb = M + (okb ? n0 + r : 0) * ld + kk;
  typename SmallT<F64>::Acc acc = {0, 0, 0, 0};
  for (int k = k0; k < k1; k += 16) {
    E a[4], b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      a[j] = pa[k + 4 * j];
      b[j] = pb[k + 4 * j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) acc = SmallT<F64>::mm((R)(oka ? a[j] : 0), (R)(okb ? b[j] : 0), acc);
  }
  return acc;
}

template <bool F64>
__device__ __forceinline__ void small_body(const NsDim& dim, const NsIo& o, int f32, int steps, float a, float b,
                                           float c, float eps, float beta, const float* alpha_dev, char* lds,
                                           double* red) {
  typedef SmallT<F64> ST;
  typedef typename ST::R R;
  const int s = dim.s, l = dim.l, T = F64 ? 1 : (s + 15) / 16;
  const int ldx = small_ldx(l), ld = small_lds(s), l16 = (l + 15) & ~15;
  R* S = reinterpret_cast<R*>(lds);    // [16 T][ld]
  R* P = S + 16 * T * ld;              // [16 T][ld]
  R* part = P + 16 * T * ld;           // [kSplit][256]
  float* X = reinterpret_cast<float*>(part + ST::kSplit * 256);  // [s][ldx], zero past column l
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int n = s * l;
  for (int i = tid; i < s * (ldx - l); i += kSmallThreads) X[i / (ldx - l) * ldx + l + i % (ldx - l)] = 0.f;
  double ss = 0.0;
  for (int i = tid; i < n; i += kSmallThreads) {
    const float v = ns_ld(o.src, i, f32);
    const int r = o.tall ? i % s : i / l, q = o.tall ? i / s : i % l;
    X[r * ldx + q] = v;
    ss += (double)v * v;
  }
  for (int d = 32; d > 0; d >>= 1) ss += __shfl_xor(ss, d, 64);
  if (lane == 0) red[wid] = ss;
  __syncthreads();
  ss = 0.0;
  for (int w = 0; w < kSmallWaves; ++w) ss += red[w];
  const double inv = 1.0 / (sqrt(ss) + (double)eps);
  for (int i = tid; i < s * ldx; i += kSmallThreads) X[i] = (float)(X[i] * inv);
  const int tiles = T * (T + 1) / 2;
  const int split = tiles < ST::kSplit ? ST::kSplit / tiles : 1;  // waves that share a Gram tile's sum
  const int kc = (((l16 + split - 1) / split) + 15) & ~15;
  for (int step = 0; step < steps; ++step) {
    __syncthreads();
    // S = X X^T: lower triangle, then mirrored.  split > 1: partial tiles joined in order
    for (int u = wid; u < tiles * split; u += kSmallWaves) {
      const int t = u / split, z = u - t * split;
      int im, in;
      tri_of(t, im, in);
      const typename ST::Acc v = small_dot<F64>(X, ldx, im * 16, in * 16, s, z * kc, min(l16, (z + 1) * kc), lane);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = ST::row(lane, e), q = lane & 15;
        if (split > 1) {
          part[u * 256 + r * 16 + q] = v[e];
        } else {
          S[(im * 16 + r) * ld + in * 16 + q] = v[e];
          if (im != in) S[(in * 16 + q) * ld + im * 16 + r] = v[e];
        }
      }
    }
    __syncthreads();
    if (split > 1) {
      for (int i = tid; i < tiles * 256; i += kSmallThreads) {
        const int t = i >> 8, r = (i >> 4) & 15, q = i & 15;
        int im, in;
        tri_of(t, im, in);
        R v = 0;
        for (int z = 0; z < split; ++z) v += part[(t * split + z) * 256 + (i & 255)];
        S[(im * 16 + r) * ld + in * 16 + q] = v;
        if (im != in) S[(in * 16 + q) * ld + im * 16 + r] = v;
      }
      __syncthreads();
    }
    // P = b S + c S S
    for (int t = wid; t < T * T; t += kSmallWaves) {
      const int im = t / T, in = t - im * T;
      const typename ST::Acc v = small_dot<F64>(S, ld, im * 16, in * 16, 16 * T, 0, 16 * T, lane);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = (im * 16 + ST::row(lane, e)) * ld + in * 16 + (lane & 15);
        P[i] = (R)c * v[e] + (R)b * S[i];
      }
    }
    __syncthreads();
    // X <- a X + P X: a wave owns 16 columns and reads them all before it writes any (P is zero past
    // row and column s: the rows of X past s are taken as its last one)
    constexpr int MT = F64 ? 1 : kSmallSide / 16;
    for (int q0 = wid * 16; q0 < l16; q0 += kSmallWaves * 16) {
      const int q = q0 + (lane & 15), kk = lane >> 4;
      typename ST::Acc acc[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i] = typename ST::Acc{0, 0, 0, 0};
      for (int r = 0; r < 16 * T; r += 16) {
        float xb[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) xb[j] = X[min(r + 4 * j + kk, s - 1) * ldx + q];
#pragma unroll
        for (int i = 0; i < MT; ++i)
          if (i < T) {
            R pa[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) pa[j] = P[(i * 16 + (lane & 15)) * ld + r + 4 * j + kk];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i] = ST::mm(pa[j], (R)xb[j], acc[i]);
          }
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
        if (i < T)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = i * 16 + ST::row(lane, e);
            if (r < s) X[r * ldx + q] = (float)((R)a * (R)X[r * ldx + q] + acc[i][e]);
          }
    }
  }
  __syncthreads();
  const float alpha = o.alpha * (alpha_dev ? alpha_dev[0] : 1.f);
  for (int i = tid; i < n; i += kSmallThreads) {
    const int r = o.tall ? i % s : i / l, q = o.tall ? i / s : i % l;
    const float v = X[r * ldx + q];
    if (f32) {
      float* dst = static_cast<float*>(o.dst) + i;
      *dst = beta != 0.f ? fmaf(alpha, v, beta * *dst) : alpha * v;
    } else {
      bf16_t* dst = static_cast<bf16_t*>(o.dst) + i;
      *dst = f2bf(beta != 0.f ? fmaf(alpha, v, beta * bf2f(*dst)) : alpha * v);
    }
  }
}

__global__ __launch_bounds__(kSmallThreads) void ns_small_kernel(NsGroup g, int f32, int steps, float a, float b,
                                                                 float c, float eps, float beta,
                                                                 const float* __restrict__ alpha_dev) {
  extern __shared__ __attribute__((aligned(16))) char small_lds_mem[];
  __shared__ double red[kSmallWaves];
  const NsDim d = g.d[blockIdx.x];
  const NsIo io = g.io[blockIdx.x];
  if (small_f64(d.s)) small_body<true>(d, io, f32, steps, a, b, c, eps, beta, alpha_dev, small_lds_mem, red);
  else small_body<false>(d, io, f32, steps, a, b, c, eps, beta, alpha_dev, small_lds_mem, red);
}

// ------------------------------------------------ the optimizer's first pass
// One pass over the flat arenas before the orthogonalisation.  kinds [n / 4]: 1 marks matrices
// (buf = first ? g : mom buf + g, upd = nesterov ? g + mom buf : buf, p *= 1 - lr wd), 0 the rest, which
// get torch.optim.SGD's whole step here.  Parameters start at multiples of 4 elements.  lr_dev: device
// learning rates [2] of the two kinds, for captured steps.
__global__ __launch_bounds__(256) void muon_prep_kernel(float* __restrict__ p, const float* __restrict__ g,
                                                        float* __restrict__ buf, float* __restrict__ upd,
                                                        const uint8_t* __restrict__ kinds, long long n4, MuonRule m,
                                                        MuonRule r, const float* __restrict__ lr_dev, int first) {
  const float lm = lr_dev ? lr_dev[0] : m.lr, lr = lr_dev ? lr_dev[1] : r.lr;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n4; i += (long long)gridDim.x * 256) {
    const bool mat = kinds[i] != 0;
    const MuonRule k = mat ? m : r;
    const float4 p4 = reinterpret_cast<const float4*>(p)[i], g4 = reinterpret_cast<const float4*>(g)[i];
    float pv[4] = {p4.x, p4.y, p4.z, p4.w}, gv[4] = {g4.x, g4.y, g4.z, g4.w}, bv[4] = {0.f, 0.f, 0.f, 0.f};
    if (!first && k.momentum != 0.f) {
      const float4 b4 = reinterpret_cast<const float4*>(buf)[i];
      bv[0] = b4.x;
      bv[1] = b4.y;
      bv[2] = b4.z;
      bv[3] = b4.w;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float d = mat ? gv[e] : gv[e] + k.weight_decay * pv[e];
      if (k.momentum != 0.f) {
        bv[e] = first ? d : k.momentum * bv[e] + d;
        d = k.nesterov ? d + k.momentum * bv[e] : bv[e];
      }
      gv[e] = d;
      pv[e] = mat ? pv[e] * (1.f - lm * k.weight_decay) : pv[e] - lr * d;
    }
    if (k.momentum != 0.f) reinterpret_cast<float4*>(buf)[i] = make_float4(bv[0], bv[1], bv[2], bv[3]);
    if (mat) reinterpret_cast<float4*>(upd)[i] = make_float4(gv[0], gv[1], gv[2], gv[3]);
    if (!mat || k.weight_decay != 0.f) reinterpret_cast<float4*>(p)[i] = make_float4(pv[0], pv[1], pv[2], pv[3]);
  }
}

// ------------------------------------------------------------------- host
template <bool TB>
using NsBig = Gemm<256, 256, 2, 4, 32, 2, 2, false, TB, true>;
template <bool TB>
using NsMid = Gemm<128, 128, 2, 2, 32, 2, 2, false, TB, true>;
template <bool TB>
using NsSmall = Gemm<64, 64, 2, 2, 64, 2, 2, false, TB, true>;
// up to kNsFew blocks, about one a compute unit: eight waves and longer steps, for a block is then bound
// by the latency of its loads and barriers
constexpr int kNsFew = 320;
template <bool TB>
using NsMidL = Gemm<128, 128, 2, 4, 64, 2, 2, false, TB, true>;
template <bool TB>
using NsSmallL = Gemm<64, 64, 2, 4, 64, 4, 2, false, TB, true>;
// twelve waves, three to a SIMD: 222 us for a Gram product of 4,096 x 4,096 (four waves: 242)
using NsWide = Gemm<192, 192, 4, 3, 32, 3, 2, false, false, true>;
// f(G1, G2) with the tiles of a phase of so many blocks
template <bool TB, typename F>
void ns_with(bool latency, F&& f, bool wide = false) {
  if constexpr (!TB)
    if (wide) return f(NsWide{}, NsWide{});
  if (latency) f(NsMidL<TB>{}, NsSmallL<TB>{});
  else f(NsMid<TB>{}, NsSmall<TB>{});
}

struct NsPlan {
  NsCut cut;
  NsGroup group;
  int blocks[kPhases], slab_stride;
  long long elems, slab_floats;
};

// Tiles: a 64-wide tile for matrices whose shorter side it covers, else 128 -- unless a phase then has
// fewer than 128 blocks, which leaves half of the compute units idle: then 64 for all.  The update takes
// 256 where that still fills the device and no matrix is much narrower (4,096 x 4,096: 335 us on 256, 430 on
// 128; ResNet-50's mixture: 162 on 256, 144 on 128).
NsPlan ns_plan(const NsMatrix* mats, int n) {
  NsPlan p{};
  long long upd256 = 0, off = 0;
  int longest = 1, shortest = kNsMaxSide;
  p.group.count = n;
  for (int i = 0; i < n; ++i) {
    NsDim& d = p.group.d[i];
    d.s = std::min(mats[i].rows, mats[i].cols);
    d.l = std::max(mats[i].rows, mats[i].cols);
    d.xo = off;
    off += 4ll * d.s * up8(d.l);
    d.so = off;
    off += 4ll * d.s * up8(d.s);
    off = (off + 63) / 64 * 64;
    p.group.io[i] = NsIo{mats[i].src, mats[i].dst, mats[i].alpha, mats[i].rows > mats[i].cols ? 1 : 0};
    upd256 += cdiv(d.s, 256) * cdiv(up8(d.l), 256);
    longest = std::max(longest, d.l);
    shortest = std::min(shortest, d.s);
  }
  p.elems = off;
  auto blocks = [&](int phase) {
    long long b = 0;
    for (int i = 0; i < n; ++i) b += ns_blocks(phase, p.group.d[i].s, p.group.d[i].l, p.cut).blocks;
    return b;
  };
  p.cut.kc = 256;
  p.cut.gram_small = blocks(kGram) < 128;
  p.cut.poly_small = blocks(kPoly) < 128;
  const long long upd128 = blocks(kUpdate);
  p.cut.upd_small = upd128 < 128;
  p.cut.upd_big = upd256 >= 192 && shortest > 192;
  // the Gram reduction is cut into pieces of kc (at least 256), for at most about 1,000 blocks in all
  // (ResNet-50's mixture: 58 us, and 20 for the join; 68 and 17 with 600 blocks)
  while (p.cut.kc < longest && blocks(kGram) > 1000) p.cut.kc += 64;
  // The symmetric products on 192-wide tiles, one a compute unit, where their rounds take less than those of
  // 128-wide ones, two a unit (a last round of at most 256 has the units to itself): 4,096 x 4,096 in 253 tiles
  // takes 222 + 227 us (Gram and polynomial), in 528 285 + 292.
  auto wide = [&](int phase, int& on) {
    const long long b = blocks(phase), rest = b % 512;
    const long long mid = (b / 512 * 2 + (rest > 256 ? 2 : rest > 0 ? 1 : 0)) * 128 * 128;
    on = 1;
    on = shortest > 192 && cdiv(blocks(phase), 256) * 192 * 192 < mid;
  };
  if (p.cut.kc >= longest) wide(kGram, p.cut.gram_wide);
  wide(kPoly, p.cut.poly_wide);
  for (int ph = 0; ph < kPhases; ++ph) p.blocks[ph] = (int)blocks(ph);
  p.slab_stride = p.cut.gram_small ? 64 * 64 : 128 * 128;
  p.slab_floats = p.blocks[kJoin] ? (long long)p.blocks[kGram] * p.slab_stride : 0;
  return p;
}

struct NsScales {
  float x, s, p;  // of X, S and P of one step
};

// Powers of two for every step.  [0, hi] holds the singular values, so hi bounds the entries of X,
// hi^2 those of S and max |b t + c t^2| over t <= hi^2 those of P; each is scaled to at most 2^15
// (fp16 ends at 65,504: a factor of two covers the roundings).  The largest values lie at the ends or
// where the derivative vanishes: b + 2 c t = 0 for P, a + 3 b w + 5 c w^2 = 0 (w = v^2) for the next X.
bool ns_scales(int steps, float a, float b, float c, NsScales* out) {
  if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
  double hi = 1.0;
  auto pow2 = [](double bound) { return (float)std::ldexp(1.0, std::min(40, (int)std::floor(15.0 - std::log2(bound)))); };
  for (int k = 0; k < steps; ++k) {
    double mp = 1e-6, mx = 1e-6;
    const double end = hi * hi;
    auto at_p = [&](double t) {
      if (t > 0 && t <= end) mp = std::max(mp, std::fabs(t * ((double)b + (double)c * t)));
    };
    auto at_x = [&](double w) {
      if (w > 0 && w <= end) mx = std::max(mx, std::fabs(std::sqrt(w) * ((double)a + w * ((double)b + (double)c * w))));
    };
    at_p(end);
    at_x(end);
    if (c != 0.f) {
      at_p(-(double)b / (2.0 * c));
      const double d = 9.0 * b * b - 20.0 * (double)a * c;
      if (d >= 0) {
        at_x((-3.0 * b + std::sqrt(d)) / (10.0 * c));
        at_x((-3.0 * b - std::sqrt(d)) / (10.0 * c));
      }
    } else if (b != 0.f) {
      at_x(-(double)a / (3.0 * b));
    }
    mp *= 1.01;
    mx *= 1.01;
    if (!(hi <= 1024.0 && mp <= 1e6 && mx <= 1024.0)) return false;
    out[k] = NsScales{pow2(hi), pow2(hi * hi), pow2(mp)};
    hi = mx;
  }
  return true;
}

bool ns_matrix_ok(const NsMatrix& m) {
  return m.rows >= 1 && m.cols >= 1 && m.rows <= kNsMaxSide && m.cols <= kNsMaxSide;
}

struct NsSpace {  // of a group, in bytes
  long long slab, part, table, total;
};
NsSpace ns_space(const NsPlan& p) {
  auto up = [](long long b) { return (b + 255) / 256 * 256; };
  NsSpace o;
  o.slab = up(p.elems * 2);
  o.part = o.slab + up(p.slab_floats * 4);
  o.table = o.part + up((long long)p.group.count * kNormBlocks * 8);
  o.total = o.table + up(sizeof(NsTable));
  return o;
}

}  // namespace

int muon_prep_launch(float* p, const float* g, float* buf, float* upd, const uint8_t* kinds, long long n,
                     const MuonRule& matrices, const MuonRule& rest, const float* lr_dev, bool first, hipStream_t st) {
  if (n < 0 || n % 4) return 1;
  if (n == 0) return 0;
  const long long nb = cdiv(n / 4, 256);
  hipLaunchKernelGGL(muon_prep_kernel, dim3((int)std::min<long long>(nb, 8192)), dim3(256), 0, st, p, g, buf, upd,
                     kinds, n / 4, matrices, rest, lr_dev, first ? 1 : 0);
  return 0;
}

int ns_check(int steps, float a, float b, float c) {
  NsScales sc[kNsMaxSteps];
  if (steps < 1 || steps > kNsMaxSteps) return 1;
  return ns_scales(steps, a, b, c, sc) ? 0 : 2;
}

namespace {

// Matrices for the one-block kernel go first; the others in order of their shorter side, the largest
// first, so that the longest blocks of a grid start first.
std::vector<NsMatrix> ns_order(const NsMatrix* mats, int n, int* small) {
  std::vector<NsMatrix> v, rest;
  for (int i = 0; i < n; ++i) {
    const int s = std::min(mats[i].rows, mats[i].cols), l = std::max(mats[i].rows, mats[i].cols);
    (small_ok(s, l) ? v : rest).push_back(mats[i]);
  }
  *small = (int)v.size();
  std::stable_sort(rest.begin(), rest.end(), [](const NsMatrix& x, const NsMatrix& y) {
    return std::min(x.rows, x.cols) > std::min(y.rows, y.cols);
  });
  v.insert(v.end(), rest.begin(), rest.end());
  return v;
}

}  // namespace

long long ns_workspace_bytes(const NsMatrix* mats, int n) {
  int small;
  const std::vector<NsMatrix> v = ns_order(mats, n, &small);
  long long most = 0;
  for (int i = small; i < n; i += kNsGroup)
    most = std::max(most, ns_space(ns_plan(v.data() + i, std::min(n - i, kNsGroup))).total);
  return most;
}

int ns_launch(const NsMatrix* mats, int n, bool f32, int steps, float a, float b, float c, float eps, float beta,
              const float* alpha_dev, void* ws, hipStream_t st) {
  NsScales sc[kNsMaxSteps];
  if (steps < 1 || steps > kNsMaxSteps || !ns_scales(steps, a, b, c, sc)) return 1;
  for (int i = 0; i < n; ++i)
    if (!ns_matrix_ok(mats[i])) return 2;
  const int f = f32 ? 1 : 0;
  int small;
  const std::vector<NsMatrix> v = ns_order(mats, n, &small);
  for (int g0 = 0; g0 < small; g0 += kNsGroup) {
    const NsPlan p = ns_plan(v.data() + g0, std::min(small - g0, kNsGroup));
    long long bytes = 0;
    for (int i = 0; i < p.group.count; ++i) bytes = std::max(bytes, small_bytes(p.group.d[i].s, p.group.d[i].l));
    if (bytes > 64 * 1024 &&
        hipFuncSetAttribute(reinterpret_cast<const void*>(ns_small_kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                            (int)bytes) != hipSuccess)
      return 3;
    hipLaunchKernelGGL(ns_small_kernel, dim3(p.group.count), dim3(kSmallThreads), (size_t)bytes, st, p.group, f, steps, a,
                       b, c, eps, beta, alpha_dev);
  }
  for (int g0 = small; g0 < n; g0 += kNsGroup) {
    const NsPlan p = ns_plan(v.data() + g0, std::min(n - g0, kNsGroup));
    const NsSpace o = ns_space(p);
    char* base = static_cast<char*>(ws);
    unsigned short* W = static_cast<unsigned short*>(ws);
    float* slab = reinterpret_cast<float*>(base + o.slab);
    double* part = reinterpret_cast<double*>(base + o.part);
    NsTable* tab = reinterpret_cast<NsTable*>(base + o.table);
    hipLaunchKernelGGL(ns_norm_kernel, dim3(p.blocks[kNorm]), dim3(256), 0, st, p.group, p.cut, f, part, tab);
    hipLaunchKernelGGL(ns_start_kernel, dim3(p.blocks[kStart]), dim3(256), 0, st, tab, f, part, W, eps, sc[0].x);
    for (int k = 0; k < steps; ++k) {
      const int xb = k & 1;
      const float gmul = sc[k].s / (sc[k].x * sc[k].x);
      ns_with<false>(p.blocks[kGram] <= kNsFew, [&](auto g1, auto g2) {
        hipLaunchKernelGGL((ns_gram_kernel<decltype(g1), decltype(g2)>), dim3(p.blocks[kGram]), dim3(g1.NT), 0, st, tab,
                           W, xb, p.cut.kc, gmul, slab, p.slab_stride);
      }, p.cut.gram_wide);
      if (p.blocks[kJoin])
        hipLaunchKernelGGL(ns_join_kernel, dim3(p.blocks[kJoin]), dim3(256), 0, st, tab, W, slab, p.slab_stride, gmul);
      ns_with<false>(p.blocks[kPoly] <= kNsFew, [&](auto g1, auto g2) {
        hipLaunchKernelGGL((ns_poly_kernel<decltype(g1), decltype(g2)>), dim3(p.blocks[kPoly]), dim3(g1.NT), 0, st, tab,
                           W, b, c, 1.f / sc[k].s, sc[k].p);
      }, p.cut.poly_wide);
      const bool last = k + 1 == steps;
      const NsStep u{a, 1.f / sc[k].x, 1.f / sc[k].p, last ? 1.f : sc[k + 1].x, beta, f, alpha_dev};
      auto update = [&](auto g1, auto g2) {
        using G1 = decltype(g1);
        using G2 = decltype(g2);
        if (last)
          hipLaunchKernelGGL((ns_update_kernel<G1, G2, true>), dim3(p.blocks[kUpdate]), dim3(G1::NT), 0, st, tab, W, xb,
                             u);
        else
          hipLaunchKernelGGL((ns_update_kernel<G1, G2, false>), dim3(p.blocks[kUpdate]), dim3(G1::NT), 0, st, tab, W, xb,
                             u);
      };
      if (p.cut.upd_big) update(NsBig<true>{}, NsBig<true>{});
      else ns_with<true>(p.blocks[kUpdate] <= kNsFew, update);
    }
  }
  return 0;
}

}  // namespace pmd
