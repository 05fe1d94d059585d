// Softmax cross-entropy of a linear classifier, straight from the features (gfx950).
//
//   l = x W^T + b   x [N][D], W [V][D]      loss = sum_{rows kept} (lse(l_i) - l_i[t_i]) / max(kept, 1)
//   dl = (softmax(l) - onehot(t)) gloss / kept   (rows kept; zero elsewhere)
//   dx = dl W,  dW = dl^T x,  db = column sums of dl
//
// The logits are never stored.  Forward: the product's epilogue reduces its tile to (max, sum of
// exponentials, argmax) per row, one combine pass joins the column tiles, one block sums the rows.
// When a backward will follow, the epilogue also keeps the exponentials it has at hand, about the
// maximum of their row in the wave's columns, if they take at most kKeepBytes (with the weight's copy, where
// it is not read in place).
// Backward, per piece of the vocabulary: softmax - onehot is written in 16 bits (a piece holds at most
// kPieceBytes, which the last-level cache keeps) and the two gradient products read it from there.  It
// comes from the kept exponentials, times exp(their maximum - lse), in a pass bound by memory; or, past
// kKeepBytes, from the piece's logits computed again, 8 N V D operations instead of 6.
//
// Rounding: operands are bf16 (products are then exact in fp32), or fp32 held as three bf16 planes
// (gemm_core.h).  softmax - onehot is rounded to the same: one bf16 when the operands are bf16 --
// half a bf16 step of each probability, the size of the gradients' own rounding -- or three planes.
// Exponentials are kept in fp32 for fp32 operands, else in fp16 times 2^15: half an fp16 step (an
// eighth of a bf16 one) down to 2^-29 of the maximum, and below that 2^-40 of it.
// Sums, statistics, the loss and db stay in fp32 (db sums the probabilities before that rounding).
// No atomics: partial results are joined in a fixed order.
//
// Rows whose target is ignore_index count for nothing whatever they hold (their features are
// replaced by zeros before the product).  A target outside [0, V) makes the row's loss NaN.
#include "gemm_core.h"

namespace pmd {

namespace {

constexpr long long kPieceBytes = 192ll << 20;
constexpr long long kKeepBytes = 4ll << 30;
constexpr float kKeepScale = 32768.f;  // exponentials of at most 1 as fp16: up to 2^15 (its largest is 65504)

__device__ __forceinline__ float ld_any(const void* p, long long i, bool f32) {
  return f32 ? static_cast<const float*>(p)[i] : bf2f(static_cast<const bf16_t*>(p)[i]);
}

// v as a sum of PL bf16 (each the rounding of what the ones before it leave)
template <int PL>
__device__ __forceinline__ void to_planes(float v, bf16_t (&o)[PL]) {
#pragma unroll
  for (int p = 0; p < PL; ++p) {
    o[p] = f2bf(v);
    v -= bf2f(o[p]);
  }
}

// src [rows][cols] (bf16 or fp32, row stride lds) -> PL planes [rows][ld], zero-padded columns; with
// target: rows to ignore become zero
template <int PL>
__global__ __launch_bounds__(256) void lx_prep_kernel(const void* __restrict__ src, int f32, long long lds, int rows,
                                                      int cols, bf16_t* __restrict__ dst, long long plane, int ld,
                                                      const long long* __restrict__ target, long long ignore) {
  const int c8 = ld >> 3;
  const long long total = (long long)rows * c8;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const int r = (int)(i / c8), c = (int)(i - (long long)r * c8) * 8;
    const bool skip = target && target[r] == ignore;
    bf16_t o[8][PL];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      to_planes<PL>(!skip && c + k < cols ? ld_any(src, r * lds + c + k, f32) : 0.f, o[k]);
#pragma unroll
    for (int p = 0; p < PL; ++p) {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = (uint32_t)o[2 * k][p] | ((uint32_t)o[2 * k + 1][p] << 16);
      *reinterpret_cast<uint4*>(dst + p * plane + (long long)r * ld + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

template <int PL>
struct LxArgs {
  GemmOperand<PL> x, w;  // rows N x D, V x D (w from the piece's first row in the backward)
  int N, V, D;           // V: classes (of the piece)
  const void* bias;      // nullable, from the piece's first class
  int bias_f32;
  const long long* target;
  long long ignore;
  int v0;                // first class of the piece
  // forward
  float *pmax, *psum;    // [column tiles][N]
  int* pidx;
  float* tlogit;         // [N]
  void* keep;            // nullable: exponentials [N][ldk], fp32 or (one plane) fp16 times kKeepScale
  float* kref;           // [V / the waves' columns][N]: what they are about
  long long ldk;
  // backward
  const float* lse;      // [N]
  bf16_t* prob;          // PL planes [N][ldp]
  long long pplane;
  int ldp;
  float* dbpart;         // [row tiles][ldp], nullable
};

__device__ __forceinline__ float bias_of(const void* bias, int f32, int n, int V) {
  return bias && n < V ? ld_any(bias, n, f32) : 0.f;
}

typedef float f32x4_keep __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8_keep __attribute__((ext_vector_type(8)));

// Exponentials are kept in the order in which lanes hold them: of 32 columns, column 16 j + 4 q + e at
// 8 q + 4 j + e, so that a lane (row, q) stores 16 bytes and four of them 64 bytes of a row.  (In column order,
// 8 bytes a lane, the forward of 8,192 x 2,048 x 131,072 takes 4.9 ms; so it takes 4.2, keeping nothing 3.7;
// nontemporal stores change nothing.)
template <int PL, int NI>
__device__ __forceinline__ void keep_store(void* p, long long o, const float (&v)[NI][4]) {
  static_assert(NI % 2 == 0, "a wave's columns are multiples of 32");
#pragma unroll
  for (int j = 0; j < NI; j += 2) {
    if constexpr (PL == 1) {
      f16x8_keep h;
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = (_Float16)(v[j + e / 4][e % 4] * kKeepScale);
      *reinterpret_cast<f16x8_keep*>(static_cast<_Float16*>(p) + o + j * 16) = h;
    } else {
      f32x4_keep* d = reinterpret_cast<f32x4_keep*>(static_cast<float*>(p) + o + j * 16);
      const f32x4_keep h0 = {v[j][0], v[j][1], v[j][2], v[j][3]};
      const f32x4_keep h1 = {v[j + 1][0], v[j + 1][1], v[j + 1][2], v[j + 1][3]};
      d[0] = h0;
      d[1] = h1;
    }
  }
}
// the 8 values kept at o (a multiple of 8), of 4 + 4 columns; pairs of lanes then exchange four, so that each
// has 8 columns in a row
template <int PL>
__device__ __forceinline__ void keep_load(const void* p, long long o, float (&v)[8]) {
  if constexpr (PL == 1) {
    const f16x8_keep h =
        __builtin_nontemporal_load(reinterpret_cast<const f16x8_keep*>(static_cast<const _Float16*>(p) + o));
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)h[e];
  } else {
    const f32x4_keep* q = reinterpret_cast<const f32x4_keep*>(static_cast<const float*>(p) + o);
    const f32x4_keep h0 = __builtin_nontemporal_load(q), h1 = __builtin_nontemporal_load(q + 1);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = h0[e];
      v[4 + e] = h1[e];
    }
  }
}
__device__ __forceinline__ int keep_column(int o) { return (o & ~31) + (o & 8) * 2 + ((o & 16) >> 1); }
__device__ __forceinline__ void keep_exchange(float (&v)[8], bool odd) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float t = __shfl_xor(odd ? v[e] : v[4 + e], 1, 64);
    if (odd) v[e] = t;
    else v[4 + e] = t;
  }
}

// ---------------------------------------------------------------- forward
template <class G>
__global__ __launch_bounds__(G::NT) void lx_fwd_kernel(LxArgs<G::PL> a) {
  __shared__ __attribute__((aligned(16))) char smem[G::LDS];
  const int tm = (a.N + G::BM - 1) / G::BM, tn = (a.V + G::BN - 1) / G::BN;
  int im, in;
  tile_of(blockIdx.x, tm * tn, tm, tn, im, in);
  const int m0 = im * G::BM, n0 = in * G::BN;
  typename G::Acc acc;
  G::run(a.x, a.w, m0, n0, 0, a.D, smem, acc);
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, wm = wid / G::WN, wn = wid % G::WN;
  const int nb = n0 + wn * G::TN + (lane >> 4) * 4;
  float bias[G::NI][4];
#pragma unroll
  for (int j = 0; j < G::NI; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[j][e] = bias_of(a.bias, a.bias_f32, nb + j * 16 + e, a.V);
  float* sm = reinterpret_cast<float*>(smem);  // [WN][BM] max, sum, index
  float* ss = sm + G::WN * G::BM;
  int* si = reinterpret_cast<int*>(ss + G::WN * G::BM);
  long long target[G::MI];
#pragma unroll
  for (int i = 0; i < G::MI; ++i) {
    const int m = m0 + wm * G::TM + i * 16 + (lane & 15);
    target[i] = m < a.N ? a.target[m] : -1;
  }
#pragma unroll
  for (int i = 0; i < G::MI; ++i) {
    const int ml = wm * G::TM + i * 16 + (lane & 15), m = m0 + ml;
    const long long t = target[i];
    float mx = -INFINITY;
    int mi = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < G::NI; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = nb + j * 16 + e;
        float v = acc[i][j][e] + bias[j][e];
        if (n >= a.V) v = -INFINITY;
        acc[i][j][e] = v;
        if (v > mx) {
          mx = v;
          mi = n;
        }
        if (n == t && n < a.V) a.tlogit[m] = v;
      }
#pragma unroll
    for (int o = 16; o <= 32; o <<= 1) {
      const float om = __shfl_xor(mx, o, 64);
      const int oi = __shfl_xor(mi, o, 64);
      if (om > mx || (om == mx && oi < mi)) {
        mx = om;
        mi = oi;
      }
    }
    const float ref = mx == -INFINITY ? 0.f : mx;  // nothing above -inf: the sum is 0, not NaN
    float s = 0.f, v[G::NI][4];
#pragma unroll
    for (int j = 0; j < G::NI; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[j][e] = __expf(acc[i][j][e] - ref);
        s += v[j][e];
      }
    const int nw = n0 + wn * G::TN;
    if (a.keep && m < a.N && nw < a.ldk)
      keep_store<G::PL, G::NI>(a.keep, m * a.ldk + nw + (lane >> 4) * 8, v);
    if (a.keep && lane < 16 && m < a.N) a.kref[(long long)(in * G::WN + wn) * a.N + m] = mx;
    s += __shfl_xor(s, 16, 64);
    s += __shfl_xor(s, 32, 64);
    if (lane < 16) {
      sm[wn * G::BM + ml] = mx;
      ss[wn * G::BM + ml] = s;
      si[wn * G::BM + ml] = mi;
    }
  }
  __syncthreads();
  for (int r = tid; r < G::BM; r += G::NT) {
    if (m0 + r >= a.N) continue;
    float mx = sm[r];
    int mi = si[r];
#pragma unroll
    for (int q = 1; q < G::WN; ++q)
      if (sm[q * G::BM + r] > mx) {  // a tie stays with the lower columns
        mx = sm[q * G::BM + r];
        mi = si[q * G::BM + r];
      }
    const float ref = mx == -INFINITY ? 0.f : mx;
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < G::WN; ++q) s += ss[q * G::BM + r] * __expf((sm[q * G::BM + r] == -INFINITY ? ref : sm[q * G::BM + r]) - ref);
    const long long o = (long long)in * a.N + m0 + r;
    a.pmax[o] = mx;
    a.psum[o] = s;
    a.pidx[o] = mi;
  }
}

struct LxRows {  // the forward's per-tile results and what joining them gives
  const float *pmax, *psum, *tlogit;
  const int* pidx;
  const long long* target;
  long long ignore;
  int N, V, tiles;
  float *lse, *rloss;  // [N]; the loss of rows to ignore is 0
  int* hit;            // [N] 0: to ignore, 1: kept, 2: kept and top-1 right
};

// Joins the column tiles of RB rows m0..; thread (r, q) takes every Q-th tile of row r.  All RB Q threads of
// the block call this.
template <int RB, int Q>
__device__ __forceinline__ void lx_join_rows(const LxRows& a, int m0, float (*sm)[RB + 1], float (*ss)[RB + 1],
                                             int (*si)[RB + 1]) {
  const int r = threadIdx.x % RB, q = threadIdx.x / RB, m = m0 + r;
  float mx = -INFINITY, s = 0.f;
  int mi = 0x7fffffff;
  if (m < a.N)
    for (int c = q; c < a.tiles; c += Q) {
      const long long o = (long long)c * a.N + m;
      const float om = a.pmax[o], os = a.psum[o];
      const int oi = a.pidx[o];
      if (om > mx || (om == mx && oi < mi)) {
        s = (mx == om ? s : s * __expf(mx - om)) + os;  // equal: both may be -inf
        mx = om;
        mi = oi;
      } else {
        s += mx == om ? os : os * __expf(om - mx);
      }
    }
  sm[q][r] = mx;
  ss[q][r] = s;
  si[q][r] = mi;
  __syncthreads();
  if (q == 0 && m < a.N) {
    for (int k = 1; k < Q; ++k)
      if (sm[k][r] > mx || (sm[k][r] == mx && si[k][r] < mi)) {
        mx = sm[k][r];
        mi = si[k][r];
      }
    const float ref = mx == -INFINITY ? 0.f : mx;
    s = 0.f;
    for (int k = 0; k < Q; ++k) s += sm[k][r] == -INFINITY ? ss[k][r] : ss[k][r] * __expf(sm[k][r] - ref);
    const long long t0 = a.target[m];
    const bool keep = t0 != a.ignore, in = t0 >= 0 && t0 < a.V;
    const float l = mx + __logf(s);
    a.lse[m] = keep && !in ? NAN : l;
    a.rloss[m] = !keep ? 0.f : in ? l - a.tlogit[m] : NAN;
    a.hit[m] = !keep ? 0 : (t0 == mi ? 2 : 1);
  }
}

__global__ __launch_bounds__(256) void lx_combine_kernel(LxRows a) {
  __shared__ float sm[16][17], ss[16][17];
  __shared__ int si[16][17];
  lx_join_rows<16, 16>(a, blockIdx.x * 16, sm, ss, si);
}

// loss = sum of the row losses / kept, correct, 1 / kept
__device__ __forceinline__ void lx_total(const float* rloss, const int* hit, int N, float* loss, long long* correct,
                                         float* inv_count) {
  __shared__ float sl[16];
  __shared__ int sk[16], sc[16];
  float l = 0.f;
  int k = 0, c = 0;
  for (int i = threadIdx.x; i < N; i += 1024) {
    l += rloss[i];
    k += hit[i] > 0;
    c += hit[i] == 2;
  }
  for (int o = 32; o > 0; o >>= 1) {
    l += __shfl_xor(l, o, 64);
    k += __shfl_xor(k, o, 64);
    c += __shfl_xor(c, o, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    sl[threadIdx.x >> 6] = l;
    sk[threadIdx.x >> 6] = k;
    sc[threadIdx.x >> 6] = c;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) {
      l += sl[w];
      k += sk[w];
      c += sc[w];
    }
    const float n = k > 0 ? (float)k : 1.f;
    loss[0] = l / n;
    correct[0] = c;
    inv_count[0] = 1.f / n;
  }
}
__global__ __launch_bounds__(1024) void lx_loss_kernel(const float* __restrict__ rloss, const int* __restrict__ hit,
                                                       int N, float* __restrict__ loss, long long* __restrict__ correct,
                                                       float* __restrict__ inv_count) {
  lx_total(rloss, hit, N, loss, correct, inv_count);
}
// both in one block, 256 rows at a time, for up to 512 rows and 64 tiles: 256 rows of 16 tiles take 5.7 us (1,030
// rows of 65 tiles take lx_combine_kernel 10.4 and lx_loss_kernel 3.9)
constexpr int kOneBlockRows = 512, kOneBlockTiles = 64;
__global__ __launch_bounds__(1024) void lx_finish_kernel(LxRows a, float* loss, long long* correct, float* inv_count) {
  __shared__ float sm[4][257], ss[4][257];
  __shared__ int si[4][257];
  for (int m0 = 0; m0 < a.N; m0 += 256) {
    lx_join_rows<256, 4>(a, m0, sm, ss, si);
    __syncthreads();
  }
  __threadfence_block();
  lx_total(a.rloss, a.hit, a.N, loss, correct, inv_count);
}

// --------------------------------------------------------------- backward
// prob = softmax - onehot of the piece (rows to ignore: 0; columns past V: 0), dbpart = its column
// sums over the row tile
template <class G>
__global__ __launch_bounds__(G::NT) void lx_prob_kernel(LxArgs<G::PL> a) {
  __shared__ __attribute__((aligned(16))) char smem[G::LDS];
  const int tm = (a.N + G::BM - 1) / G::BM, tn = (a.ldp + G::BN - 1) / G::BN;
  int im, in;
  tile_of(blockIdx.x, tm * tn, tm, tn, im, in);
  const int m0 = im * G::BM, n0 = in * G::BN;
  typename G::Acc acc;
  G::run(a.x, a.w, m0, n0, 0, a.D, smem, acc);
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, wm = wid / G::WN, wn = wid % G::WN;
  const int nb = n0 + wn * G::TN + (lane >> 4) * 4;
  float bias[G::NI][4], col[G::NI][4];
#pragma unroll
  for (int j = 0; j < G::NI; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      bias[j][e] = bias_of(a.bias, a.bias_f32, nb + j * 16 + e, a.V);
      col[j][e] = 0.f;
    }
  long long target[G::MI];
  float lses[G::MI];
#pragma unroll
  for (int i = 0; i < G::MI; ++i) {
    const int m = m0 + wm * G::TM + i * 16 + (lane & 15);
    target[i] = m < a.N ? a.target[m] : a.ignore;
    lses[i] = m < a.N ? a.lse[m] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < G::MI; ++i) {
    const int m = m0 + wm * G::TM + i * 16 + (lane & 15);
    if (m >= a.N) continue;
    const long long t = target[i];
    const bool keep = t != a.ignore;
    const float lse = lses[i];
#pragma unroll
    for (int j = 0; j < G::NI; ++j) {
      const int n = nb + j * 16;
      if (n >= a.ldp) continue;
      bf16_t o[4][G::PL];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float p = 0.f;
        if (keep && n + e < a.V) {
          p = __expf(acc[i][j][e] + bias[j][e] - lse);
          if (t == a.v0 + n + e) p -= 1.f;
        }
        col[j][e] += p;
        to_planes<G::PL>(p, o[e]);
      }
#pragma unroll
      for (int q = 0; q < G::PL; ++q) {
        const uint2 w = make_uint2((uint32_t)o[0][q] | ((uint32_t)o[1][q] << 16),
                                   (uint32_t)o[2][q] | ((uint32_t)o[3][q] << 16));
        *reinterpret_cast<uint2*>(a.prob + q * a.pplane + (long long)m * a.ldp + n) = w;
      }
    }
  }
  if (a.dbpart) {
    float* sc = reinterpret_cast<float*>(smem);  // [WM][BN]
#pragma unroll
    for (int j = 0; j < G::NI; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v = col[j][e];
        for (int o = 1; o < 16; o <<= 1) v += __shfl_xor(v, o, 64);
        if ((lane & 15) == 0) sc[wm * G::BN + wn * G::TN + j * 16 + (lane >> 4) * 4 + e] = v;
      }
    __syncthreads();
    for (int c = tid; c < G::BN; c += G::NT)
      if (n0 + c < a.ldp) {
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < G::WM; ++q) v += sc[q * G::BN + c];
        a.dbpart[(long long)im * a.ldp + n0 + c] = v;
      }
  }
}

// The same from the exponentials that the forward kept, in blocks of `rows` rows x CW vectors of 8 columns;
// the 256 / CW groups of threads take consecutive rows each.  8,192 rows x 8,192 columns in 53 us (5.0 TB/s
// read and written); computing the logits again takes 265 us.
template <int PL>
struct LxScale {
  const void* keep;       // from the piece's first class
  const float *kref, *lse, *tlogit;
  long long ldk;
  int kshift;             // log2 of the columns that share a kref
  const long long* target;
  long long ignore;
  int N, V, v0;           // V: classes of the piece
  bf16_t* prob;
  long long pplane;
  int ldp, CW, rows, cblocks;
  float* dbpart;
};
template <int PL>
__global__ __launch_bounds__(256) void lx_scale_kernel(LxScale<PL> a) {
  __shared__ float sc[256 * 9];
  const int tid = threadIdx.x, tc = tid & (a.CW - 1), grp = tid / a.CW, per = a.rows * a.CW / 256;
  const int im = blockIdx.x / a.cblocks, cb = blockIdx.x - im * a.cblocks;
  const int o8 = (cb * a.CW + tc) * 8, n = keep_column(o8), ms = im * a.rows + grp * per, me = min(a.N, ms + per);
  float col[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) col[e] = 0.f;
  if (n < a.ldp) {
    const float* ref = a.kref + (long long)((a.v0 + n) >> a.kshift) * a.N;
#pragma unroll 4
    for (int m = ms; m < me; ++m) {
      float v[8];
      keep_load<PL>(a.keep, m * a.ldk + o8, v);
      keep_exchange(v, tc & 1);
      const long long t = a.target[m];
      const bool keep = t != a.ignore;
      const float lse = a.lse[m];
      const float s = __expf(ref[m] - lse) * (PL == 1 ? 1.f / kKeepScale : 1.f);
      const long long d = t - a.v0 - n;  // the target among the 8
      bf16_t o[8][PL];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float p = 0.f;
        if (keep && n + e < a.V) p = d == e ? __expf(a.tlogit[m] - lse) - 1.f : v[e] * s;
        col[e] += p;
        to_planes<PL>(p, o[e]);
      }
#pragma unroll
      for (int q = 0; q < PL; ++q) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = (uint32_t)o[2 * k][q] | ((uint32_t)o[2 * k + 1][q] << 16);
        *reinterpret_cast<uint4*>(a.prob + q * a.pplane + (long long)m * a.ldp + n) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
  if (!a.dbpart) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) sc[tid * 9 + e] = col[e];
  __syncthreads();
  if (grp == 0 && n < a.ldp) {
    for (int g = 1; g < 256 / a.CW; ++g)
#pragma unroll
      for (int e = 0; e < 8; ++e) col[e] += sc[(g * a.CW + tc) * 9 + e];
    float* d = a.dbpart + (long long)im * a.ldp + n;
    *reinterpret_cast<float4*>(d) = make_float4(col[0], col[1], col[2], col[3]);
    *reinterpret_cast<float4*>(d + 4) = make_float4(col[4], col[5], col[6], col[7]);
  }
}

__device__ __forceinline__ void st4(void* p, bool f32, long long o, const float (&v)[4], int n, bool acc) {
  if (f32) {
    float* d = static_cast<float*>(p) + o;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) d[e] = acc ? d[e] + v[e] : v[e];
  } else {
    bf16_t* d = static_cast<bf16_t*>(p) + o;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) d[e] = f2bf(v[e]);
  }
}

__device__ __forceinline__ void st4v(void* p, bool f32, long long o, const float (&v)[4], bool acc) {
  if (f32) {
    float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + o);
    float4 t = make_float4(v[0], v[1], v[2], v[3]);
    if (acc) {
      const float4 u = *d;
      t = make_float4(u.x + t.x, u.y + t.y, u.z + t.z, u.w + t.w);
    }
    *d = t;
  } else {
    *reinterpret_cast<uint2*>(static_cast<bf16_t*>(p) + o) =
        make_uint2(f2bf(v[0]) | ((uint32_t)f2bf(v[1]) << 16), f2bf(v[2]) | ((uint32_t)f2bf(v[3]) << 16));
  }
}

// a gradient product: dst [M][N] = or += scale * A B^T.  ws: split z of the reduction adds to slab z
// ([splits][M][N] fp32, unscaled) instead.
template <int PL>
struct LxGradArgs {
  GemmOperand<PL> A, B;
  int M, N, K, ksplit;        // ksplit: reduction elements of a split
  float* slab;                // nullable
  int slab_add;               // slabs hold earlier pieces
  void* dst;
  long long ldd;
  int dst_f32, accumulate;
  const float *gloss, *inv_count;
};

template <class G>
__device__ __forceinline__ void lx_grad_tile(const LxGradArgs<G::PL>& a, int block, int blocks, int split, char* smem) {
  const int tm = (a.M + G::BM - 1) / G::BM, tn = (a.N + G::BN - 1) / G::BN;
  int im, in;
  tile_of(block, blocks, tm, tn, im, in);
  const int m0 = im * G::BM, n0 = in * G::BN;
  const int k0 = split * a.ksplit, k1 = min(a.K, k0 + a.ksplit);
  typename G::Acc acc;
  G::run(a.A, a.B, m0, n0, k0, k1, smem, acc);
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, wm = wid / G::WN, wn = wid % G::WN;
  const float sc = a.slab ? 1.f : a.gloss[0] * a.inv_count[0];
  const bool vec = a.ldd % 4 == 0 && reinterpret_cast<uintptr_t>(a.dst) % 16 == 0;
#pragma unroll
  for (int i = 0; i < G::MI; ++i) {
    const int m = m0 + wm * G::TM + i * 16 + (lane & 15);
    if (m >= a.M) continue;
#pragma unroll
    for (int j = 0; j < G::NI; ++j) {
      const int n = n0 + wn * G::TN + j * 16 + (lane >> 4) * 4;
      if (n >= a.N) continue;
      if (a.slab) {
        float* d = a.slab + ((long long)split * a.M + m) * a.N + n;  // N % 8 == 0: whole float4
        float4 v = make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
        if (a.slab_add) {
          const float4 o = *reinterpret_cast<const float4*>(d);
          v = make_float4(v.x + o.x, v.y + o.y, v.z + o.z, v.w + o.w);
        }
        *reinterpret_cast<float4*>(d) = v;
      } else {
        const float v[4] = {acc[i][j][0] * sc, acc[i][j][1] * sc, acc[i][j][2] * sc, acc[i][j][3] * sc};
        const long long o = (long long)m * a.ldd + n;
        if (vec && n + 4 <= a.ldd) st4v(a.dst, a.dst_f32, o, v, a.accumulate);
        else st4(a.dst, a.dst_f32, o, v, (int)min(4ll, a.ldd - n), a.accumulate);
      }
    }
  }
}

// dx (blocks of GX, splits of its reduction one after the other) and dW (GW) in one grid
template <class GX, class GW>
__global__ __launch_bounds__(GX::NT) void lx_grads_kernel(LxGradArgs<GX::PL> x, LxGradArgs<GW::PL> w, int xtiles,
                                                          int xblocks, int wblocks) {
  __shared__ __attribute__((aligned(16))) char smem[GX::LDS > GW::LDS ? GX::LDS : GW::LDS];
  const int b = blockIdx.x;
  if (b < xblocks) lx_grad_tile<GX>(x, b % xtiles, xtiles, b / xtiles, smem);
  else lx_grad_tile<GW>(w, b - xblocks, wblocks, 0, smem);
}

// The last kernel of a piece: db [V] = or += scale * column sums of part [tiles][ldp], in blocks of 64
// classes; and after the last piece dx [M][cols] = scale * sum over the slabs [splits][M][ld] (rows to
// ignore are zero), in the blocks behind them.
struct LxTail {
  const float *part, *slab;
  void *db, *dx;
  int tiles, ldp, V, db_f32, accumulate, db_blocks;
  int splits, M, ld, dx_f32, cols;
  const float *gloss, *inv_count;
  const long long* target;
  long long ignore;
};
__global__ __launch_bounds__(256) void lx_tail_kernel(LxTail a) {
  const float sc = a.gloss[0] * a.inv_count[0];
  if ((int)blockIdx.x < a.db_blocks) {
    __shared__ float part[4][64];
    const int g = threadIdx.x >> 6, n = blockIdx.x * 64 + (threadIdx.x & 63);
    float s = 0.f;
    if (n < a.V) {
#pragma unroll 8
      for (int t = g; t < a.tiles; t += 4) s += a.part[(long long)t * a.ldp + n];
    }
    part[g][threadIdx.x & 63] = s;
    __syncthreads();
    if (g || n >= a.V) return;
    for (int k = 1; k < 4; ++k) s += part[k][threadIdx.x];
    s *= sc;
    if (a.db_f32) {
      float* d = static_cast<float*>(a.db) + n;
      *d = a.accumulate ? *d + s : s;
    } else {
      static_cast<bf16_t*>(a.db)[n] = f2bf(s);
    }
    return;
  }
  const int c4 = a.ld >> 2, blocks = gridDim.x - a.db_blocks;
  const long long total = (long long)a.M * c4, step = (long long)a.M * a.ld;
  for (long long i = (blockIdx.x - a.db_blocks) * 256ll + threadIdx.x; i < total; i += blocks * 256ll) {
    const int r = (int)(i / c4), c = (int)(i - (long long)r * c4) * 4;
    if (c >= a.cols) continue;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (a.target[r] != a.ignore) {
      const float* s = a.slab + (long long)r * a.ld + c;
#pragma unroll 4
      for (int z = 0; z < a.splits; ++z) {
        const float4 t = *reinterpret_cast<const float4*>(s + z * step);
        v[0] += t.x;
        v[1] += t.y;
        v[2] += t.z;
        v[3] += t.w;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] *= sc;
    }
    st4(a.dx, a.dx_f32, (long long)r * a.cols + c, v, min(4, a.cols - c), false);
  }
}

// ------------------------------------------------------------------- host
template <int PL, bool TA, bool TB>
struct LxTiles {  // 256 only for one plane: three planes of it would not fit LDS twice
  typedef Gemm<128, 128, 2, 2, PL == 1 ? 64 : 32, 2, PL, TA, TB, false> Mid;
  // few blocks, bound by the latency of their loads: more steps in flight
  typedef Gemm<64, 64, 2, 2, PL == 1 ? 64 : 32, PL == 1 ? 4 : 3, PL, TA, TB, false> Small;
};
template <bool TA, bool TB>
using LxBig = Gemm<256, 256, 2, 4, 64, 2, 1, TA, TB, false>;

inline long long tiles_of(long long m, long long n, int t) { return ((m + t - 1) / t) * ((n + t - 1) / t); }

// Tile of an m x n product (times the splits of its reduction): the largest that still gives the 256
// compute units a block each, else the smallest.
inline int pick_tile(long long m, long long n, int splits, int pl) {
  if (pl == 1 && tiles_of(m, n, 256) * splits >= 192) return 256;
  if (tiles_of(m, n, 128) * splits >= 192) return 128;
  return 64;
}

template <int PL, bool TA, bool TB, typename F>
int with_tile(int tile, F&& f) {
  if constexpr (PL == 1)
    if (tile == 256) return f(LxBig<TA, TB>{});
  if (tile == 128) return f(typename LxTiles<PL, TA, TB>::Mid{});
  return f(typename LxTiles<PL, TA, TB>::Small{});
}

// f(tile of dx, tile of dW); the two share a kernel, so a 256-wide one needs the other to be
template <int PL, typename F>
void with_tiles(int x, int w, F&& f) {
  typedef LxTiles<PL, false, true> X;
  typedef LxTiles<PL, true, true> W;
  if constexpr (PL == 1)
    if (x == 256 && w == 256) return f(LxBig<false, true>{}, LxBig<true, true>{});
  if (x >= 128 && w >= 128) return f(typename X::Mid{}, typename W::Mid{});
  if (x >= 128) return f(typename X::Mid{}, typename W::Small{});
  if (w >= 128) return f(typename X::Small{}, typename W::Mid{});
  return f(typename X::Small{}, typename W::Small{});
}

inline int grid_cap(long long n, int cap) {
  if (n > cap) n = cap;
  return n < 1 ? 1 : (int)n;
}

struct LxPlan {
  int Dp;                   // features, padded to 8
  bool w_direct;            // the weight is read in place
  int fwd_tile, fwd_ct;     // forward tile and column tiles
  int piece, pieces;        // classes of a piece (multiple of 64 unless it is all of V), pieces
  int kshift;               // log2 of the forward's columns of a wave
  long long ldk;            // row of the kept exponentials
  bool keep;                // they are within kKeepBytes
  int bwd_tile, bwd_rt;     // tile of the recomputation; its row tiles, or those of lx_scale_kernel
  int sc_cw, sc_rows;       // lx_scale_kernel's column vectors and rows of a block
  int dx_tile, dx_splits, dx_ksplit, dw_tile;
};

inline int up(long long v, int m) { return (int)((v + m - 1) / m * m); }

// The piece-dependent part of the plan.
void lx_plan_piece(const LxShape& s, long long piece, LxPlan& p) {
  p.piece = (int)piece;
  p.pieces = (s.V + p.piece - 1) / p.piece;
  p.bwd_tile = pick_tile(s.N, p.piece, 1, s.planes);
  p.bwd_rt = (s.N + p.bwd_tile - 1) / p.bwd_tile;
  if (p.keep) {  // at least 4 rows a thread, and four blocks a compute unit where that leaves them
    const int vecs = up(p.piece, 64) / 8;
    for (p.sc_cw = 8; p.sc_cw < 64 && p.sc_cw * 2 <= vecs;) p.sc_cw *= 2;
    const long long cb = (vecs + p.sc_cw - 1) / p.sc_cw;
    for (p.sc_rows = 128; p.sc_rows > 4 * 256 / p.sc_cw && cb * ((s.N + p.sc_rows - 1) / p.sc_rows) < 1024;)
      p.sc_rows /= 2;
    p.bwd_rt = (s.N + p.sc_rows - 1) / p.sc_rows;
  }
  p.dw_tile = pick_tile(p.piece, p.Dp, 1, s.planes);
  // dx reduces over the classes: split them until the compute units are full, at least 512 a split
  p.dx_tile = pick_tile(s.N, p.Dp, (int)(p.piece / 512 > 0 ? p.piece / 512 : 1), s.planes);
  const long long t = tiles_of(s.N, p.Dp, p.dx_tile);
  long long sp = (256 + t - 1) / t;
  if (sp > p.piece / 512) sp = p.piece / 512;
  if (sp < 1) sp = 1;
  p.dx_ksplit = up((p.piece + sp - 1) / sp, 64);
  p.dx_splits = (p.piece + p.dx_ksplit - 1) / p.dx_ksplit;
}

// Time of the backward in tile steps: every product runs in rounds of 256 blocks (one 256-wide tile a
// compute unit), and a last round that is not full costs a whole one.
long long lx_piece_cost(const LxShape& s, const LxPlan& p) {
  auto rounds = [](long long blocks) { return (blocks + 255) / 256; };
  const long long prob = rounds(tiles_of(s.N, p.piece, 256)) * p.Dp;
  const long long dw = rounds(tiles_of(p.piece, p.Dp, 256)) * s.N;
  const long long dx = rounds(tiles_of(s.N, p.Dp, 256) * p.dx_splits) * p.dx_ksplit;
  return p.pieces * (prob + dw + dx);
}

// kept: the exponentials are kept if they are few enough
LxPlan lx_plan(const LxShape& s, bool kept) {
  LxPlan p;
  p.Dp = up(s.D, 8);
  p.w_direct = s.planes == 1 && !s.w_f32 && s.D % 8 == 0 && s.w_aligned;
  p.fwd_tile = pick_tile(s.N, s.V, 1, s.planes);
  p.fwd_ct = (s.V + p.fwd_tile - 1) / p.fwd_tile;
  p.kshift = p.fwd_tile == 64 ? 5 : 6;
  p.ldk = up(s.V, 64);
  p.keep = kept && s.N * (p.ldk + (p.ldk >> p.kshift) * 2) * (s.planes == 1 ? 2 : 4) +
                           (p.w_direct ? 0 : 2ll * s.planes * s.V * p.Dp) <= kKeepBytes;
  const int vp = up(s.V, 64);
  long long piece = kPieceBytes / (2ll * s.planes * s.N) / 256 * 256;
  if (piece < 1024) piece = 1024;
  if (piece > (1 << 20)) piece = 1 << 20;  // a tile's offsets within the piece stay below 2^31 bytes
  lx_plan_piece(s, piece < vp ? piece : vp, p);
  if (p.pieces > 1 && p.bwd_tile == 256 && p.dw_tile == 256 && p.dx_tile == 256) {
    // a smaller piece may fill the last rounds better: 8,192 rows x 2,048 features x 131,072 classes take
    // 16 pieces of 8,192 rather than 11 of 12,288, whose dW products have 384 blocks (18.9 ms, when the pieces of
    // 8,192 took 16.6)
    long long best = lx_piece_cost(s, p), at = p.piece;
    for (long long c = piece - 256; c >= piece / 4; c -= 256) {
      lx_plan_piece(s, c, p);
      const long long cost = lx_piece_cost(s, p);
      if (cost < best) {
        best = cost;
        at = c;
      }
    }
    lx_plan_piece(s, at, p);
  }
  return p;
}

// workspace layout (bytes, 256-aligned)
struct Carver {
  char* base;
  long long off = 0;
  template <typename T>
  T* take(long long n) {
    T* p = reinterpret_cast<T*>(base + off);
    off += (n * (long long)sizeof(T) + 255) / 256 * 256;
    return base ? p : nullptr;
  }
};

struct LxBuf {
  bf16_t *x, *w;  // x: the caller's xp
  float *pmax, *psum, *tlogit, *rloss;
  int *pidx, *hit;
  bf16_t* prob;
  float *dbpart, *slab;
};

LxBuf lx_carve(const LxShape& s, const LxPlan& p, bool bwd, char* base, long long* bytes) {
  Carver c{base};
  LxBuf b{};
  if (!p.w_direct && !p.keep) b.w = c.take<bf16_t>((long long)s.planes * s.V * p.Dp);
  if (!bwd) {
    const long long n = (long long)p.fwd_ct * s.N;
    b.pmax = c.take<float>(n);
    b.psum = c.take<float>(n);
    b.pidx = c.take<int>(n);
    b.tlogit = c.take<float>(s.N);
    b.rloss = c.take<float>(s.N);
    b.hit = c.take<int>(s.N);
  } else {
    b.prob = c.take<bf16_t>((long long)s.planes * s.N * p.piece);
    b.dbpart = c.take<float>((long long)p.bwd_rt * p.piece);
    b.slab = c.take<float>((long long)p.dx_splits * s.N * p.Dp);
  }
  *bytes = c.off;
  return b;
}

struct LxKept {  // what a forward keeps for its backward
  void* e;
  float *ref, *tlogit;
  bf16_t* w;             // the weight laid out, unless it is read in place
};
LxKept lx_kept(const LxShape& s, const LxPlan& p, void* base, long long* bytes) {
  Carver c{static_cast<char*>(base)};
  LxKept k{};
  k.e = c.take<char>(s.N * p.ldk * (s.planes == 1 ? 2 : 4));
  k.ref = c.take<float>((long long)s.N * (up(s.V, p.fwd_tile) >> p.kshift));
  k.tlogit = c.take<float>(s.N);
  if (!p.w_direct) k.w = c.take<bf16_t>((long long)s.planes * s.V * p.Dp);
  *bytes = c.off;
  return k;
}

template <int PL>
GemmOperand<PL> planes_of(const bf16_t* p, long long plane, long long ld, int rows) {
  GemmOperand<PL> o;
  for (int q = 0; q < PL; ++q) o.plane[q] = p + q * plane;
  o.ld = ld;
  o.rows = rows;
  return o;
}

template <int PL>
void lx_prep(const void* src, bool f32, int rows, int cols, bf16_t* dst, int ld, const long long* target,
             long long ignore, hipStream_t st) {
  const long long n = (long long)rows * (ld / 8);
  hipLaunchKernelGGL(lx_prep_kernel<PL>, dim3(grid_cap((n + 255) / 256, 8192)), dim3(256), 0, st, src, f32 ? 1 : 0,
                     (long long)cols, rows, cols, dst, (long long)rows * ld, ld, target, ignore);
}

bool lx_ok(const LxShape& s) {
  return s.N >= 1 && s.V >= 1 && s.D >= 1 && (s.planes == 1 || s.planes == 3) && s.D <= kGemmMaxLd - 8 &&
         s.V <= (1 << 30) && s.N <= (1 << 24) && (long long)s.N * s.V <= (1ll << 38);
}

template <int PL>
int lx_fwd_t(const LxShape& s, const LxIo& io, hipStream_t st) {
  const LxPlan p = lx_plan(s, io.kept != nullptr);
  long long bytes;
  LxBuf b = lx_carve(s, p, false, static_cast<char*>(io.ws), &bytes);
  const LxKept kept = lx_kept(s, p, io.kept, &bytes);
  if (io.kept) {
    b.tlogit = kept.tlogit;
    b.w = kept.w;
  }
  b.x = static_cast<bf16_t*>(io.xp);
  lx_prep<PL>(io.x, s.x_f32, s.N, s.D, b.x, p.Dp, io.target, io.ignore, st);
  if (!p.w_direct) lx_prep<PL>(io.w, s.w_f32, s.V, s.D, b.w, p.Dp, nullptr, 0, st);
  LxArgs<PL> a{};
  a.x = planes_of<PL>(b.x, (long long)s.N * p.Dp, p.Dp, s.N);
  a.w = p.w_direct ? planes_of<PL>(static_cast<const bf16_t*>(io.w), 0, s.D, s.V)
                   : planes_of<PL>(b.w, (long long)s.V * p.Dp, p.Dp, s.V);
  a.N = s.N; a.V = s.V; a.D = p.Dp;
  a.bias = io.bias; a.bias_f32 = s.b_f32;
  a.target = io.target; a.ignore = io.ignore;
  a.pmax = b.pmax; a.psum = b.psum; a.pidx = b.pidx; a.tlogit = b.tlogit;
  a.keep = kept.e; a.kref = kept.ref; a.ldk = p.ldk;
  const int rc = with_tile<PL, false, false>(p.fwd_tile, [&](auto g) {
    using G = decltype(g);
    hipLaunchKernelGGL(lx_fwd_kernel<G>, dim3((unsigned)tiles_of(s.N, s.V, G::BM)), dim3(G::NT), 0, st, a);
    return 0;
  });
  if (rc) return rc;
  const LxRows r{b.pmax, b.psum, b.tlogit, b.pidx, io.target, io.ignore, s.N, s.V, p.fwd_ct, io.lse, b.rloss, b.hit};
  if (s.N <= kOneBlockRows && p.fwd_ct <= kOneBlockTiles) {
    hipLaunchKernelGGL(lx_finish_kernel, dim3(1), dim3(1024), 0, st, r, io.loss, io.correct, io.inv_count);
  } else {
    hipLaunchKernelGGL(lx_combine_kernel, dim3((s.N + 15) / 16), dim3(256), 0, st, r);
    hipLaunchKernelGGL(lx_loss_kernel, dim3(1), dim3(1024), 0, st, b.rloss, b.hit, s.N, io.loss, io.correct,
                       io.inv_count);
  }
  return 0;
}

template <int PL>
int lx_bwd_t(const LxShape& s, const LxIo& io, hipStream_t st) {
  const LxPlan p = lx_plan(s, io.kept != nullptr);
  long long bytes;
  LxBuf b = lx_carve(s, p, true, static_cast<char*>(io.ws), &bytes);
  b.x = static_cast<bf16_t*>(io.xp);  // the forward's
  const LxKept kept = lx_kept(s, p, io.kept, &bytes);
  if (!p.w_direct && !io.kept) lx_prep<PL>(io.w, s.w_f32, s.V, s.D, b.w, p.Dp, nullptr, 0, st);
  const bf16_t* wbase = p.w_direct ? static_cast<const bf16_t*>(io.w) : io.kept ? kept.w : b.w;
  const long long wplane = p.w_direct ? 0 : (long long)s.V * p.Dp;
  for (int k = 0; k < p.pieces; ++k) {
    const int v0 = k * p.piece, V = s.V - v0 < p.piece ? s.V - v0 : p.piece;
    LxArgs<PL> a{};
    a.x = planes_of<PL>(b.x, (long long)s.N * p.Dp, p.Dp, s.N);
    a.w = planes_of<PL>(wbase + (long long)v0 * p.Dp, wplane, p.Dp, V);
    a.N = s.N; a.V = V; a.D = p.Dp; a.v0 = v0;
    const int bsz = s.b_f32 ? 4 : 2;
    a.bias = io.bias ? static_cast<const char*>(io.bias) + (long long)v0 * bsz : nullptr;
    a.bias_f32 = s.b_f32;
    a.target = io.target; a.ignore = io.ignore; a.lse = io.lse;
    a.ldp = up(V, 64);
    a.prob = b.prob; a.pplane = (long long)s.N * a.ldp;
    a.dbpart = io.db ? b.dbpart : nullptr;
    if (io.kept) {
      LxScale<PL> c{};
      c.keep = static_cast<const char*>(kept.e) + (long long)v0 * (PL == 1 ? 2 : 4);
      c.kref = kept.ref; c.lse = io.lse; c.tlogit = kept.tlogit;
      c.ldk = p.ldk; c.kshift = p.kshift; c.target = io.target; c.ignore = io.ignore;
      c.N = s.N; c.V = V; c.v0 = v0;
      c.prob = b.prob; c.pplane = a.pplane; c.ldp = a.ldp; c.dbpart = a.dbpart;
      c.CW = p.sc_cw; c.rows = p.sc_rows; c.cblocks = (a.ldp / 8 + c.CW - 1) / c.CW;
      hipLaunchKernelGGL(lx_scale_kernel<PL>, dim3((unsigned)(c.cblocks * p.bwd_rt)), dim3(256), 0, st, c);
    } else with_tile<PL, false, false>(p.bwd_tile, [&](auto g) {
      using G = decltype(g);
      hipLaunchKernelGGL(lx_prob_kernel<G>, dim3((unsigned)tiles_of(s.N, a.ldp, G::BM)), dim3(G::NT), 0, st, a);
      return 0;
    });
    LxGradArgs<PL> x{}, w{};
    if (io.dx) {  // slabs [splits][N][Dp] += prob W
      x.A = planes_of<PL>(b.prob, a.pplane, a.ldp, s.N);
      x.B = planes_of<PL>(wbase + (long long)v0 * p.Dp, wplane, p.Dp, p.Dp);
      x.M = s.N; x.N = p.Dp; x.K = V; x.ksplit = p.dx_ksplit;
      x.slab = b.slab; x.slab_add = k > 0;
    }
    if (io.dw) {  // dW[v0 ..] = or += scale prob^T x
      w.A = planes_of<PL>(b.prob, a.pplane, a.ldp, a.ldp);
      w.B = planes_of<PL>(b.x, (long long)s.N * p.Dp, p.Dp, p.Dp);
      w.M = V; w.N = p.Dp; w.K = s.N; w.ksplit = up(s.N, 64);
      w.dst = static_cast<char*>(io.dw) + (long long)v0 * s.D * (io.dw_f32 ? 4 : 2);
      w.ldd = s.D; w.dst_f32 = io.dw_f32; w.accumulate = io.accumulate;
      w.gloss = io.gloss; w.inv_count = io.inv_count;
    }
    if (io.dx || io.dw) with_tiles<PL>(p.dx_tile, p.dw_tile, [&](auto gx, auto gw) {
      using GX = decltype(gx);
      using GW = decltype(gw);
      const int xt = io.dx ? (int)tiles_of(s.N, p.Dp, GX::BM) : 1, xb = io.dx ? xt * p.dx_splits : 0;
      const int wb = io.dw ? (int)tiles_of(V, p.Dp, GW::BM) : 0;
      auto launch = [&](int xblocks, int wblocks) {
        hipLaunchKernelGGL((lx_grads_kernel<GX, GW>), dim3((unsigned)(xblocks + wblocks)), dim3(GX::NT), 0, st, x, w, xt,
                           xblocks, wblocks);
      };
      // one grid where a product alone leaves compute units idle; two where each has rounds of its own
      if (xb < 256 || wb < 256) {
        launch(xb, wb);
      } else {
        launch(xb, 0);
        launch(0, wb);
      }
    });
    const bool last = k + 1 == p.pieces;
    if (io.db || (last && io.dx)) {
      LxTail t{};
      t.gloss = io.gloss; t.inv_count = io.inv_count; t.target = io.target; t.ignore = io.ignore;
      if (io.db) {
        t.part = b.dbpart; t.tiles = p.bwd_rt; t.ldp = a.ldp; t.V = V;
        t.db = static_cast<char*>(io.db) + (long long)v0 * bsz; t.db_f32 = s.b_f32; t.accumulate = io.accumulate;
        t.db_blocks = (V + 63) / 64;
      }
      long long nb = 0;
      if (last && io.dx) {
        t.slab = b.slab; t.splits = p.dx_splits; t.M = s.N; t.ld = p.Dp; t.dx = io.dx; t.dx_f32 = s.x_f32; t.cols = s.D;
        nb = grid_cap(((long long)s.N * (p.Dp / 4) + 255) / 256, 4096);
      }
      hipLaunchKernelGGL(lx_tail_kernel, dim3((unsigned)(t.db_blocks + nb)), dim3(256), 0, st, t);
    }
  }
  return 0;
}

}  // namespace

long long lx_xplanes(const LxShape& s) { return (long long)s.planes * s.N * up(s.D, 8); }

long long lx_workspace_bytes(const LxShape& s, bool bwd, bool kept) {
  if (!lx_ok(s)) return 0;
  long long bytes;
  lx_carve(s, lx_plan(s, kept), bwd, nullptr, &bytes);
  return bytes;
}

long long lx_kept_bytes(const LxShape& s) {
  if (!lx_ok(s)) return 0;
  const LxPlan p = lx_plan(s, true);
  long long bytes = 0;
  if (p.keep) lx_kept(s, p, nullptr, &bytes);
  return bytes;
}

int lx_fwd_launch(const LxShape& s, const LxIo& io, hipStream_t st) {
  if (!lx_ok(s)) return 1;
  return s.planes == 1 ? lx_fwd_t<1>(s, io, st) : lx_fwd_t<3>(s, io, st);
}

int lx_bwd_launch(const LxShape& s, const LxIo& io, hipStream_t st) {
  if (!lx_ok(s)) return 1;
  return s.planes == 1 ? lx_bwd_t<1>(s, io, st) : lx_bwd_t<3>(s, io, st);
}

}  // namespace pmd
