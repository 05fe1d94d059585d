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

namespace pmd {

namespace {

typedef _Float16 f16_t;

struct NsDim {
  int s, l;          // shorter, longer side
  long long xo, so;  // element offsets in the workspace: X (2 buffers x 2 planes), S and P (2 planes each)
  int t0;            // first block of this matrix in the phase's grid
  int splits;        // of the Gram product
};
struct NsIo {
  const void* src;
  void* dst;
  float alpha;
  int tall;          // src is l x s: taken transposed
};
struct NsGroup {
  int count, blocks;
  NsDim d[kNsGroup];
};
struct NsIoGroup {
  NsIo io[kNsGroup];
};

__device__ __forceinline__ int up8(int v) { return (v + 7) & ~7; }

__device__ __forceinline__ int find_matrix(const NsGroup& g, int block) {
  int lo = 0, hi = g.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (g.d[mid].t0 <= block) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ float ns_ld(const void* p, long long i, bool f32) {
  return f32 ? static_cast<const float*>(p)[i] : bf2f(static_cast<const bf16_t*>(p)[i]);
}

__device__ __forceinline__ void split2(float v, unsigned short& hi, unsigned short& lo) {
  const f16_t h = (f16_t)v, l = (f16_t)(v - (float)h);
  hi = __builtin_bit_cast(unsigned short, h);
  lo = __builtin_bit_cast(unsigned short, l);
}
__device__ __forceinline__ float join2(unsigned short hi, unsigned short lo) {
  return (float)__builtin_bit_cast(f16_t, hi) + (float)__builtin_bit_cast(f16_t, lo);
}

// ------------------------------------------------------------- norm, start
constexpr int kNormBlocks = 64;  // partial sums per matrix

// part [matrix][kNormBlocks] = sums of squares, in fp64 (entries of 1e-30 or 1e30 neither vanish nor
// overflow)
__global__ __launch_bounds__(256) void ns_norm_kernel(NsGroup g, NsIoGroup io, int f32, double* __restrict__ part) {
  __shared__ double red[4];
  const int k = blockIdx.x / kNormBlocks, b = blockIdx.x % kNormBlocks;
  const long long n = (long long)g.d[k].s * g.d[k].l;
  double s = 0.0;
  for (long long i = b * 256ll + threadIdx.x; i < n; i += kNormBlocks * 256ll) {
    const double v = ns_ld(io.io[k].src, i, f32);
    s += v * v;
  }
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = ((red[0] + red[1]) + red[2]) + red[3];
}

// X_0 planes [s][up8(l)] of one 64 x 64 tile, through LDS when the matrix is taken transposed
__global__ __launch_bounds__(256) void ns_start_kernel(NsGroup g, NsIoGroup io, int f32, const double* __restrict__ part,
                                                       unsigned short* __restrict__ ws, float eps, float scale) {
  __shared__ float tile[64][65];
  __shared__ float inv_s;
  const int k = find_matrix(g, blockIdx.x), t = blockIdx.x - g.d[k].t0;
  const int s = g.d[k].s, l = g.d[k].l, lp = up8(l);
  const int tl = (lp + 63) / 64, r0 = (t / tl) * 64, c0 = (t % tl) * 64;
  if (threadIdx.x < 64) {
    double v = part[k * kNormBlocks + threadIdx.x];
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if (threadIdx.x == 0) inv_s = (float)(1.0 / (sqrt(v) + (double)eps)) * scale;
  }
  const bool tall = io.io[k].tall;
  const int a = threadIdx.x & 63, b = threadIdx.x >> 6;
  for (int i = b; i < 64; i += 4) {  // a: along the source's rows
    const int r = tall ? r0 + a : r0 + i, c = tall ? c0 + i : c0 + a;
    const float v = r < s && c < l ? ns_ld(io.io[k].src, tall ? (long long)c * s + r : (long long)r * l + c, f32) : 0.f;
    if (tall) tile[a][i] = v;
    else tile[i][a] = v;
  }
  __syncthreads();
  const float inv = inv_s;
  unsigned short* x = ws + g.d[k].xo;
  const long long plane = (long long)s * lp;
  for (int i = b; i < 64; i += 4) {
    const int r = r0 + i, c = c0 + a;
    if (r >= s || c >= lp) continue;
    unsigned short hi, lo;
    split2(tile[i][a] * inv, hi, lo);
    x[(long long)r * lp + c] = hi;
    x[plane + (long long)r * lp + c] = lo;
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
  while ((long long)(r + 1) * (r + 2) / 2 <= t) ++r;
  while ((long long)r * (r + 1) / 2 > t) --r;
  im = r;
  in = t - r * (r + 1) / 2;
}

// four neighbours n.. of row m of a symmetric matrix [s][up8(s)] (2 planes), and their mirror images
__device__ __forceinline__ void put_sym(unsigned short* p, int s, int m, int n, const float (&v)[4], bool mirror) {
  const int ld = up8(s);
  const long long plane = (long long)s * ld;
  unsigned short h[4], l[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) split2(v[e], h[e], l[e]);
  if (m < s && n < ld) {
    const long long o = (long long)m * ld + n;
    *reinterpret_cast<uint2*>(p + o) = make_uint2(h[0] | ((uint32_t)h[1] << 16), h[2] | ((uint32_t)h[3] << 16));
    *reinterpret_cast<uint2*>(p + plane + o) = make_uint2(l[0] | ((uint32_t)l[1] << 16), l[2] | ((uint32_t)l[3] << 16));
  }
  if (mirror && m < ld)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < s) {
        p[(long long)(n + e) * ld + m] = h[e];
        p[plane + (long long)(n + e) * ld + m] = l[e];
      }
}

// S = X X^T: planes scaled by out_scale / (X's scale)^2 in one go, or slabs [block][BM][BN] (raw sums)
template <class G>
__global__ __launch_bounds__(G::NT) void ns_gram_kernel(NsGroup g, unsigned short* __restrict__ ws, int xbuf, int kc,
                                                        float mul, float* __restrict__ slab) {
  __shared__ __attribute__((aligned(16))) char smem[G::LDS];
  const int L = xcd_remap(blockIdx.x, gridDim.x);
  const int k = find_matrix(g, L);
  const NsDim d = g.d[k];
  const int r = L - d.t0, t = r / d.splits, z = r - t * d.splits;
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
      if (slab) {
        *reinterpret_cast<float4*>(slab + ((long long)L * G::BM + ml) * G::BN + nl) =
            make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
      } else {
        const float v[4] = {acc[i][j][0] * mul, acc[i][j][1] * mul, acc[i][j][2] * mul, acc[i][j][3] * mul};
        put_sym(ws + d.so, d.s, im * G::BM + ml, in * G::BN + nl, v, im != in);
      }
    }
}

// joins the slabs of the Gram product's tiles in order; 4 blocks a tile
template <int BT>
__global__ __launch_bounds__(256) void ns_join_kernel(NsGroup g, unsigned short* __restrict__ ws,
                                                      const float* __restrict__ slab, float mul) {
  // g.t0 counts the Gram product's blocks (tile x split); this grid has 4 blocks for every one of
  // them, and those of a split z > 0 have nothing to do
  const int b = blockIdx.x >> 2, part = blockIdx.x & 3;
  const int k = find_matrix(g, b);
  const NsDim d = g.d[k];
  const int r = b - d.t0, t = r / d.splits;
  if (r - t * d.splits != 0) return;
  int im, in;
  tri_of(t, im, in);
  const float* s0 = slab + (long long)b * BT * BT;
  for (int e = threadIdx.x; e < BT * BT / 16; e += 256) {
    const int i = (part * (BT * BT / 16) + e) * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int z = 0; z < d.splits; ++z) {
      const float4 q = *reinterpret_cast<const float4*>(s0 + (long long)z * BT * BT + i);
      v[0] += q.x;
      v[1] += q.y;
      v[2] += q.z;
      v[3] += q.w;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] *= mul;
    put_sym(ws + d.so, d.s, im * BT + i / BT, in * BT + i % BT, v, im != in);
  }
}

// P = b S + c S S (S's scale ss, P's scale sp)
template <class G>
__global__ __launch_bounds__(G::NT) void ns_poly_kernel(NsGroup g, unsigned short* __restrict__ ws, float b, float c,
                                                        float inv_ss, float sp) {
  __shared__ __attribute__((aligned(16))) char smem[G::LDS];
  const int L = xcd_remap(blockIdx.x, gridDim.x);
  const NsDim d = g.d[find_matrix(g, L)];
  int im, in;
  tri_of(L - d.t0, im, in);
  const int ld = up8(d.s);
  const long long plane = (long long)d.s * ld;
  const unsigned short* S = ws + d.so;
  const GemmOperand<2> x = ns_operand(S, plane, ld, d.s);
  typename G::Acc acc;
  G::run(x, x, im * G::BM, in * G::BN, 0, d.s, smem, acc);
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, wm = wid / G::WN, wn = wid % G::WN;
  const float kc = c * inv_ss * inv_ss * sp, kb = b * inv_ss * sp;
#pragma unroll
  for (int i = 0; i < G::MI; ++i)
#pragma unroll
    for (int j = 0; j < G::NI; ++j) {
      const int m = im * G::BM + wm * G::TM + i * 16 + (lane & 15);
      const int n = in * G::BN + wn * G::TN + j * 16 + (lane >> 4) * 4;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      if (m < d.s && n < ld) {
        const long long o = (long long)m * ld + n;
        const uint2 h = *reinterpret_cast<const uint2*>(S + o), l = *reinterpret_cast<const uint2*>(S + plane + o);
        const float sv[4] = {join2(h.x & 0xffff, l.x & 0xffff), join2(h.x >> 16, l.x >> 16),
                             join2(h.y & 0xffff, l.y & 0xffff), join2(h.y >> 16, l.y >> 16)};
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fmaf(kc, acc[i][j][e], kb * sv[e]);
      }
      put_sym(ws + d.so + 2 * plane, d.s, m, n, v, im != in);
    }
}

// X' = a X + P X into the other buffer, or (LAST) out = beta out + alpha X'
template <class G, bool LAST>
__global__ __launch_bounds__(G::NT) void ns_update_kernel(NsGroup g, NsIoGroup io, unsigned short* __restrict__ ws,
                                                          int xbuf, float a, float inv_sx, float inv_sp, float so,
                                                          int f32, float beta, const float* __restrict__ alpha_dev) {
  __shared__ __attribute__((aligned(16))) char smem[G::LDS];
  const int L = xcd_remap(blockIdx.x, gridDim.x);
  const int k = find_matrix(g, L);
  const NsDim d = g.d[k];
  const int t = L - d.t0, lp = up8(d.l), ld = up8(d.s);
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
  const float kp = inv_sp * inv_sx, ka = a * inv_sx;
  float alpha = 0.f;
  if constexpr (LAST) alpha = io.io[k].alpha * (alpha_dev ? alpha_dev[0] : 1.f);
#pragma unroll
  for (int i = 0; i < G::MI; ++i)
#pragma unroll
    for (int j = 0; j < G::NI; ++j) {
      const int m = im * G::BM + wm * G::TM + i * 16 + (lane & 15);
      const int n = in * G::BN + wn * G::TN + j * 16 + (lane >> 4) * 4;
      if (m >= d.s || n >= lp) continue;
      const long long o = (long long)m * lp + n;
      const uint2 hh = *reinterpret_cast<const uint2*>(X + o), ll = *reinterpret_cast<const uint2*>(X + xplane + o);
      const float xv[4] = {join2(hh.x & 0xffff, ll.x & 0xffff), join2(hh.x >> 16, ll.x >> 16),
                           join2(hh.y & 0xffff, ll.y & 0xffff), join2(hh.y >> 16, ll.y >> 16)};
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = fmaf(kp, acc[i][j][e], ka * xv[e]);
      if constexpr (LAST) {
        const bool tall = io.io[k].tall;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (n + e >= d.l) continue;
          const long long q = tall ? (long long)(n + e) * d.s + m : (long long)m * d.l + n + e;
          if (f32) {
            float* dst = static_cast<float*>(io.io[k].dst) + q;
            *dst = beta != 0.f ? fmaf(alpha, v[e], beta * *dst) : alpha * v[e];
          } else {
            bf16_t* dst = static_cast<bf16_t*>(io.io[k].dst) + q;
            *dst = f2bf(beta != 0.f ? fmaf(alpha, v[e], beta * bf2f(*dst)) : alpha * v[e]);
          }
        }
      } else {
        unsigned short hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) split2(v[e] * so, hi[e], lo[e]);
        *reinterpret_cast<uint2*>(Y + o) = make_uint2(hi[0] | ((uint32_t)hi[1] << 16), hi[2] | ((uint32_t)hi[3] << 16));
        *reinterpret_cast<uint2*>(Y + xplane + o) =
            make_uint2(lo[0] | ((uint32_t)lo[1] << 16), lo[2] | ((uint32_t)lo[3] << 16));
      }
    }
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
using NsSmall = Gemm<64, 64, 2, 2, 32, 3, 2, false, TB, true>;

template <bool TB, typename F>
void ns_with_tile(int tile, F&& f) {
  if (tile == 256) f(NsBig<TB>{});
  else if (tile == 128) f(NsMid<TB>{});
  else f(NsSmall<TB>{});
}

inline long long cdiv(long long a, long long b) { return (a + b - 1) / b; }
inline long long tri(long long t) { return t * (t + 1) / 2; }

struct NsPlan {
  int gram_tile, poly_tile, upd_tile, kc;
  NsGroup start, gram, poly, upd;
  bool slabs;
  long long elems, slab_floats;
};

// tile of a phase: the largest that gives at least 192 blocks, else the smallest
template <typename F>
int ns_pick(const NsMatrix* m, int n, F&& blocks) {
  for (int t : {256, 128}) {
    long long b = 0;
    for (int i = 0; i < n; ++i) b += blocks(m[i], t);
    if (b >= 192) return t;
  }
  return 64;
}

NsPlan ns_plan(const NsMatrix* mats, int n) {
  NsPlan p{};
  auto S = [](const NsMatrix& m) { return std::min(m.rows, m.cols); };
  auto Lg = [](const NsMatrix& m) { return std::max(m.rows, m.cols); };
  auto tri_tiles = [&](const NsMatrix& m, int t) { return tri(cdiv(S(m), t)); };
  auto upd_tiles = [&](const NsMatrix& m, int t) { return cdiv(S(m), t) * cdiv((Lg(m) + 7) / 8 * 8, t); };
  p.poly_tile = ns_pick(mats, n, tri_tiles);
  p.upd_tile = ns_pick(mats, n, upd_tiles);
  // the Gram reduction is cut into pieces of kc, about 512 blocks in all, each at least 256 long
  p.gram_tile = ns_pick(mats, n, [&](const NsMatrix& m, int t) { return tri_tiles(m, t) * cdiv(Lg(m), 1024); });
  long long work = 0, longest = 0;
  for (int i = 0; i < n; ++i) {
    work += tri_tiles(mats[i], p.gram_tile) * Lg(mats[i]);
    longest = std::max<long long>(longest, Lg(mats[i]));
  }
  long long kc = std::max<long long>(256, cdiv(work, 512));
  p.kc = (int)(std::min(kc, std::max<long long>(longest, 256) + 63) / 64 * 64);
  long long off = 0, bs = 0, bg = 0, bp = 0, bu = 0;
  for (int i = 0; i < n; ++i) {
    NsDim d{};
    d.s = S(mats[i]);
    d.l = Lg(mats[i]);
    const long long lp = (d.l + 7) / 8 * 8, ld = (d.s + 7) / 8 * 8;
    d.xo = off;
    off += 4 * d.s * lp;
    d.so = off;
    off += 4 * d.s * ld;
    off = (off + 63) / 64 * 64;
    d.splits = (int)cdiv(d.l, p.kc);
    p.slabs = p.slabs || d.splits > 1;
    d.t0 = (int)bs;
    p.start.d[i] = d;
    d.t0 = (int)bg;
    p.gram.d[i] = d;
    d.t0 = (int)bp;
    p.poly.d[i] = d;
    d.t0 = (int)bu;
    p.upd.d[i] = d;
    bs += cdiv(d.s, 64) * cdiv(lp, 64);
    bg += tri_tiles(mats[i], p.gram_tile) * d.splits;
    bp += tri_tiles(mats[i], p.poly_tile);
    bu += upd_tiles(mats[i], p.upd_tile);
  }
  p.start.count = p.gram.count = p.poly.count = p.upd.count = n;
  p.start.blocks = (int)bs;
  p.gram.blocks = (int)bg;
  p.poly.blocks = (int)bp;
  p.upd.blocks = (int)bu;
  p.elems = off;
  p.slab_floats = p.slabs ? bg * p.gram_tile * p.gram_tile : 0;
  return p;
}

struct NsScales {
  float x, s, p;  // of X, S and P of one step
};

// Powers of two for every step.  [0, hi] holds the singular values, so hi bounds the entries of X,
// hi^2 those of S and max |b t + c t^2| over t <= hi^2 those of P; each is scaled to at most 2^15
// (fp16 ends at 65,504: a factor of two covers the bound's sampling and the roundings).
bool ns_scales(int steps, float a, float b, float c, NsScales* out) {
  if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
  double hi = 1.0;
  auto pow2 = [](double bound) { return (float)std::ldexp(1.0, std::min(40, (int)std::floor(15.0 - std::log2(bound)))); };
  for (int k = 0; k < steps; ++k) {
    double mp = 1e-6, mx = 1e-6;
    for (int i = 1; i <= 4096; ++i) {
      const double v = hi * i / 4096, t = v * v;
      mp = std::max(mp, std::fabs(b * t + c * t * t));
      mx = std::max(mx, std::fabs(v * (a + b * t + c * t * t)));
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

long long ns_group_bytes(const NsPlan& p, int n, long long* slab_off, long long* part_off) {
  long long b = (p.elems * 2 + 255) / 256 * 256;
  *slab_off = b;
  b += (p.slab_floats * 4 + 255) / 256 * 256;
  *part_off = b;
  return b + (long long)n * kNormBlocks * 8;
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

long long ns_workspace_bytes(const NsMatrix* mats, int n) {
  long long most = 0, so, po;
  for (int i = 0; i < n; i += kNsGroup) {
    const int c = std::min(n - i, kNsGroup);
    most = std::max(most, ns_group_bytes(ns_plan(mats + i, c), c, &so, &po));
  }
  return most;
}

int ns_launch(const NsMatrix* mats, int n, bool f32, int steps, float a, float b, float c, float eps, float beta,
              const float* alpha_dev, void* ws, hipStream_t st) {
  NsScales sc[kNsMaxSteps];
  if (steps < 1 || steps > kNsMaxSteps || !ns_scales(steps, a, b, c, sc)) return 1;
  for (int i = 0; i < n; ++i)
    if (!ns_matrix_ok(mats[i])) return 2;
  for (int g0 = 0; g0 < n; g0 += kNsGroup) {
    const int cnt = std::min(n - g0, kNsGroup);
    const NsPlan p = ns_plan(mats + g0, cnt);
    long long slab_off, part_off;
    ns_group_bytes(p, cnt, &slab_off, &part_off);
    unsigned short* W = static_cast<unsigned short*>(ws);
    float* slab = p.slabs ? reinterpret_cast<float*>(static_cast<char*>(ws) + slab_off) : nullptr;
    double* part = reinterpret_cast<double*>(static_cast<char*>(ws) + part_off);
    NsIoGroup io{};
    for (int i = 0; i < cnt; ++i) {
      const NsMatrix& m = mats[g0 + i];
      io.io[i] = NsIo{m.src, m.dst, m.alpha, m.rows > m.cols ? 1 : 0};
    }
    const int f = f32 ? 1 : 0;
    hipLaunchKernelGGL(ns_norm_kernel, dim3(cnt * kNormBlocks), dim3(256), 0, st, p.start, io, f, part);
    hipLaunchKernelGGL(ns_start_kernel, dim3(p.start.blocks), dim3(256), 0, st, p.start, io, f, part, W, eps, sc[0].x);
    for (int k = 0; k < steps; ++k) {
      const int xb = k & 1;
      const float gmul = sc[k].s / (sc[k].x * sc[k].x);
      ns_with_tile<false>(p.gram_tile, [&](auto gm) {
        using G = decltype(gm);
        hipLaunchKernelGGL(ns_gram_kernel<G>, dim3(p.gram.blocks), dim3(G::NT), 0, st, p.gram, W, xb, p.kc, gmul,
                           slab);
        if (slab)
          hipLaunchKernelGGL(ns_join_kernel<G::BM>, dim3(p.gram.blocks * 4), dim3(256), 0, st, p.gram, W, slab, gmul);
      });
      ns_with_tile<false>(p.poly_tile, [&](auto gm) {
        using G = decltype(gm);
        hipLaunchKernelGGL(ns_poly_kernel<G>, dim3(p.poly.blocks), dim3(G::NT), 0, st, p.poly, W, b, c, 1.f / sc[k].s,
                           sc[k].p);
      });
      const bool last = k + 1 == steps;
      ns_with_tile<true>(p.upd_tile, [&](auto gm) {
        using G = decltype(gm);
        if (last)
          hipLaunchKernelGGL((ns_update_kernel<G, true>), dim3(p.upd.blocks), dim3(G::NT), 0, st, p.upd, io, W, xb, a,
                             1.f / sc[k].x, 1.f / sc[k].p, 1.f, f, beta, alpha_dev);
        else
          hipLaunchKernelGGL((ns_update_kernel<G, false>), dim3(p.upd.blocks), dim3(G::NT), 0, st, p.upd, io, W, xb, a,
                             1.f / sc[k].x, 1.f / sc[k].p, sc[k + 1].x, f, 0.f, nullptr);
      });
    }
  }
  return 0;
}

}  // namespace pmd
