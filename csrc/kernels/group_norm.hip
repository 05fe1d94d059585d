// Group normalisation with the residual add and the activation, channels last (gfx950).
//
//   x [N][HW][C], G groups of cg = C/G consecutive channels, per (n, g) over HW x cg elements:
//     mu, var (biased),  rstd = 1/sqrt(var + eps),  xhat = (x - mu) rstd
//     z = gamma xhat + beta (+ residual),  out = act(z)           act: none, relu, silu
//   backward, dz = act'(z) dout (the residual's gradient), per (n, g):
//     dx = rstd (gamma dz - mean(gamma dz) - xhat mean(gamma dz xhat))
//     dgamma = sum_{n,hw} dz xhat,  dbeta = sum_{n,hw} dz
//
// These kernels read the data twice; samples whose groups fit a block's registers are taken by
// kernels/group_norm_one.hip, which reads them once.
//
// Every pass is bound by memory; a thread owns VEC consecutive channels (16 bytes where the
// channel count and the pointers allow) and walks down the pixels, so any group width works
// the same way: statistics are taken per channel and joined into groups through LDS.
//
// A sample's pixels are split over `chunks` blocks.  Forward: stats kernel (one partial per
// (n, chunk, g)), then the apply kernel, whose blocks join the partials themselves.  Backward: the
// same pair over (dz, dz xhat), then the sums of the per-channel partials to dgamma / dbeta.
//
// With a residual and ReLU the forward keeps the slope as one bit per element (a byte per vector, as
// bn_apply does), and the backward reads that instead of the residual.
//
// Variances are (count, mean, M2) triples in fp32: a thread sums up to kSeg pixels about the mean of its
// first four, and such triples are joined pairwise (Chan, Golub, LeVeque 1983).  Plain sums of x and x^2
// would lose (mu/sigma)^2 of their precision; this loses at most kSeg 2^-24, when one of the four is far
// off.  All joins run in a fixed order: results do not depend on the scheduling.
#include "group_norm.h"

#include <algorithm>
#include <initializer_list>
#include <type_traits>

namespace pmd {

namespace {

constexpr int GT = 256;   // threads of a block
constexpr int GU = 4;    // pixels a thread loads at once
constexpr int kSeg = 64;  // pixels a thread sums about one shift

// Block geometry: cols = C / VEC channel vectors; CW of them side by side, R pixel rows at once.
struct GnGeo {
  int cols, CW, R;
  __device__ __forceinline__ GnGeo(int C, int VEC) {
    cols = C / VEC;
    CW = cols < GT ? cols : GT;
    R = GT / CW;
  }
};

// lanes for one value a chunk (at most kMaxChunks of them)
constexpr int kMaxChunks = 64;
__device__ __forceinline__ int chunk_lanes(int chunks) {
  int L = 1;
  while (L < chunks) L <<= 1;
  return L;
}
// f(g, part[lane][g] or 0) for every group, by L lanes each; the loads of eight rounds are under way at once
template <typename F>
__device__ __forceinline__ void join_chunks(const float2* part, int chunks, int G, int L, F&& f) {
  const int lane = threadIdx.x & (L - 1), step = GT / L;
  for (int g0 = threadIdx.x / L; g0 < G; g0 += 8 * step) {
    float2 t[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int g = g0 + k * step;
      t[k] = lane < chunks && g < G ? part[(size_t)lane * G + g] : make_float2(0.f, 0.f);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (g0 + k * step < G) f(g0 + k * step, t[k]);
  }
}

// ---------------------------------------------------------------- forward
// part [N][chunks][G] = (mean, M2) over the chunk's pixels x cg channels
template <typename T, int VEC>
__global__ __launch_bounds__(GT) void gn_stats_kernel(const T* __restrict__ x, float2* __restrict__ part, int HW,
                                                      int C, int G, int chunks, int P) {
  extern __shared__ float lds[];  // [R][C] means, [R][C] M2
  __shared__ float lc[GT];        // pixels of a slot
  const GnGeo geo(C, VEC);
  const int n = blockIdx.x / chunks, ch = blockIdx.x - n * chunks;
  const int p0 = ch * P, np = min(P, HW - p0);
  const T* xb = x + ((size_t)n * HW + p0) * C;
  const int tid = threadIdx.x, row = tid / geo.CW, tc = tid - row * geo.CW;
  float* lm = lds;
  float* l2 = lds + geo.R * C;
  if (row < geo.R) {
    for (int col = tc; col < geo.cols; col += geo.CW) {
      float* lmc = lm + row * C + col * VEC;  // this thread's mean and M2 so far: LDS, to leave registers
      float* l2c = l2 + row * C + col * VEC;
#pragma unroll
      for (int k = 0; k < VEC; ++k) lmc[k] = l2c[k] = 0.f;
      int cnt = 0;
      const T* xc = xb + col * VEC;
      for (int p = row; p < np;) {
        float sh[VEC], s1[VEC], s2[VEC];
        GnVec<T, VEC> v[GU];
        const int have = min(kSeg, (np - p + geo.R - 1) / geo.R);  // pixels of this segment
        auto batch = [&](int i) {  // pixels i .. of the segment, its last one again past the end
#pragma unroll
          for (int u = 0; u < GU; ++u)
            v[u] = *reinterpret_cast<const GnVec<T, VEC>*>(xc + (size_t)(p + min(i + u, have - 1) * geo.R) * C);
        };
        auto add = [&](int i) {
#pragma unroll
          for (int u = 0; u < GU; ++u) {
            const float w = i + u < have ? 1.f : 0.f;
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
              const float d = (GnIo<T>::up(v[u].v[k]) - sh[k]) * w;
              s1[k] += d;
              s2[k] = fmaf(d, d, s2[k]);
            }
          }
        };
        batch(0);
        const float w0 = 1.f / min(GU, have);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          float t = GnIo<T>::up(v[0].v[k]);
#pragma unroll
          for (int u = 1; u < GU; ++u) t += u < have ? GnIo<T>::up(v[u].v[k]) : 0.f;
          sh[k] = t * w0;
          s1[k] = s2[k] = 0.f;
        }
        add(0);
        for (int i = GU; i < have; i += GU) {
          batch(i);
          add(i);
        }
        const float in = 1.f / have, w = (float)have / (cnt + have), nn = (float)cnt * w;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float dm = s1[k] * in, q = fmaxf(s2[k] - s1[k] * dm, 0.f), d = sh[k] + dm - lmc[k];
          lmc[k] += d * w;
          l2c[k] += (s2[k] != s2[k] ? s2[k] : q) + d * d * nn;  // fmaxf drops a NaN
        }
        cnt += have;
        p += have * geo.R;
      }
    }
  }
  __syncthreads();
  // The triples of a channel first: its rows s, s + S, ..  (64 x 112 x 112 x 64 takes 28 us; 43 with all R x cg
  // triples of a group joined at once, which leaves many groups to few waves, one after the other.)
  const int S = C < GT ? GT / C : 1, each = np / geo.R, more = np - each * geo.R;
  for (int e = tid; e < S * C; e += GT) {
    const int s = e / C, c = e - s * C;
    float cnt = 0.f, t = 0.f, q = 0.f;
    for (int r = s; r < geo.R; r += S) {
      const float nr = (float)(each + (r < more ? 1 : 0));  // pixels of row r
      cnt += nr;
      t += nr * lm[r * C + c];
    }
    const float mu = t / fmaxf(cnt, 1.f);
    for (int r = s; r < geo.R; r += S) {
      const float nr = (float)(each + (r < more ? 1 : 0)), d = lm[r * C + c] - mu;
      q += nr > 0.f ? l2[r * C + c] + nr * d * d : 0.f;
    }
    lm[s * C + c] = mu;  // row s is this thread's alone
    l2[s * C + c] = q;
    if (c == 0) lc[s] = cnt;
  }
  __syncthreads();
  const int cg = C / G, ent = S * cg;
  const int L = seg_lanes(ent), lane = tid & (L - 1);
  const float inv = 1.f / ((float)np * cg);
  for (int g = tid / L; g < G; g += GT / L) {
    float t = 0.f;
    for (int e = lane; e < ent; e += L) {
      const int s = e / cg, c = e - s * cg;
      t += lc[s] * lm[s * C + g * cg + c];
    }
    const float mu = seg_sum(t, L) * inv;
    float q = 0.f;
    for (int e = lane; e < ent; e += L) {
      const int s = e / cg, c = e - s * cg;
      const float n = lc[s], d = lm[s * C + g * cg + c] - mu;
      q += n > 0.f ? l2[s * C + g * cg + c] + n * d * d : 0.f;
    }
    q = seg_sum(q, L);
    if (lane == 0) part[((size_t)n * chunks + ch) * G + g] = make_float2(mu, q);
  }
}

// out = act(gamma (x - mu) rstd + beta + res); the blocks of chunk 0 store mu, rstd [N][G] for the
// backward
template <typename T, int VEC, int ACT, bool RES, bool MASK>
__global__ __launch_bounds__(GT) void gn_apply_kernel(const T* __restrict__ x, const T* __restrict__ res,
                                                      const float* __restrict__ gamma, const float* __restrict__ beta,
                                                      const float2* __restrict__ part, float2* __restrict__ stats,
                                                      T* __restrict__ out, uint8_t* __restrict__ mask, int HW,
                                                      int C, int G, int chunks, int P, float eps) {
  extern __shared__ float lds[];  // mu [G], rstd [G]
  const GnGeo geo(C, VEC);
  const int n = blockIdx.x / chunks, ch = blockIdx.x - n * chunks;
  const int tid = threadIdx.x, cg = C / G;
  {
    const int L = chunk_lanes(chunks), lane = tid & (L - 1);
    const float np = lane < chunks ? (float)min(P, HW - lane * P) : 0.f, total = (float)HW * cg;
    join_chunks(part + (size_t)n * chunks * G, chunks, G, L, [&](int g, const float2& t) {
      const float mu = seg_sum(np * t.x, L) / HW, d = t.x - mu;
      const float rstd = rsqrtf(seg_sum(np > 0.f ? t.y + np * cg * d * d : 0.f, L) / total + eps);
      if (lane == 0) {
        lds[g] = mu;
        lds[G + g] = rstd;
        if (ch == 0) stats[(size_t)n * G + g] = make_float2(mu, rstd);
      }
    });
  }
  __syncthreads();
  const int row = tid / geo.CW, tc = tid - row * geo.CW;
  if (row >= geo.R) return;
  const int p0 = ch * P, np = min(P, HW - p0);
  const size_t base = ((size_t)n * HW + p0) * C;
  for (int col = tc; col < geo.cols; col += geo.CW) {
    float mu[VEC], a[VEC], b[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const int c = col * VEC + k, g = c / cg;
      mu[k] = lds[g];
      a[k] = gamma[c] * lds[G + g];
      b[k] = beta[c];
    }
    for (int p = row; p < np; p += geo.R) {
      const size_t o = base + (size_t)p * C + col * VEC;
      float v[VEC];
      gn_load<T, VEC>(x + o, v);
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[k] = fmaf(v[k] - mu[k], a[k], b[k]);
      if constexpr (RES) {
        float r[VEC];
        gn_load<T, VEC>(res + o, r);
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] += r[k];
      }
      if constexpr (MASK) {
        unsigned bits = 0;
#pragma unroll
        for (int k = 0; k < VEC; ++k) bits |= v[k] <= 0.f ? 0u : 1u << k;
        mask[o / VEC] = (uint8_t)bits;
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[k] = gn_act<ACT>(v[k]);
      gn_store<T, VEC>(out + o, v);
    }
  }
}

// --------------------------------------------------------------- backward
// cpart [rows of (n, chunk)][2][C] = sums over the chunk's pixels of dz and dz xhat (per channel);
// gpart [N][chunks][G] = their gamma-weighted sums over the group
template <typename T, int VEC, int ACT, int SLOPE>
__global__ __launch_bounds__(GT) void gn_bwd_stats_kernel(
    const T* __restrict__ dout, const T* __restrict__ x, const T* __restrict__ res, const uint8_t* __restrict__ mask,
    const float* __restrict__ gamma, const float* __restrict__ beta, const float2* __restrict__ stats,
    float* __restrict__ cpart, float2* __restrict__ gpart, int HW, int C, int G, int chunks, int P) {
  extern __shared__ float lds[];  // [R][C] sums of dz, [R][C] sums of dz xhat
  const GnGeo geo(C, VEC);
  const int n = blockIdx.x / chunks, ch = blockIdx.x - n * chunks;
  const int p0 = ch * P, np = min(P, HW - p0);
  const size_t base = ((size_t)n * HW + p0) * C;
  const int tid = threadIdx.x, row = tid / geo.CW, tc = tid - row * geo.CW, cg = C / G;
  float* l1 = lds;
  float* l2 = lds + geo.R * C;
  if (row < geo.R) {
    for (int col = tc; col < geo.cols; col += geo.CW) {
      float mu[VEC], rs[VEC], a[VEC], be[VEC], s1[VEC], s2[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const int c = col * VEC + k;
        const float2 st = stats[(size_t)n * G + c / cg];
        mu[k] = st.x;
        rs[k] = st.y;
        a[k] = gamma[c] * st.y;
        be[k] = beta[c];
        s1[k] = s2[k] = 0.f;
      }
      for (int p = row; p < np; p += geo.R) {
        const size_t o = base + (size_t)p * C + col * VEC;
        float v[VEC], g[VEC], r[VEC], dz[VEC];
        gn_load<T, VEC>(x + o, v);
        gn_load<T, VEC>(dout + o, g);
        if constexpr (SLOPE == kOfXRes && ACT != 0) gn_load<T, VEC>(res + o, r);
        unsigned bits = 0;
        if constexpr (SLOPE == kOfMask) bits = mask[o / VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] -= mu[k];
        gn_dz<VEC, ACT, SLOPE>(v, g, r, bits, a, be, dz);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          s1[k] += dz[k];
          s2[k] = fmaf(dz[k], v[k], s2[k]);
        }
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        l1[row * C + col * VEC + k] = s1[k];
        l2[row * C + col * VEC + k] = s2[k] * rs[k];
      }
    }
  }
  __syncthreads();
  float* cp = cpart + ((size_t)n * chunks + ch) * 2 * C;
  for (int c = tid; c < C; c += GT) {  // rows -> row 0 (a thread's own column: no race)
    float a = 0.f, b = 0.f;
    for (int r = 0; r < geo.R; ++r) {
      a += l1[r * C + c];
      b += l2[r * C + c];
    }
    cp[c] = a;
    cp[C + c] = b;
    l1[c] = a;
    l2[c] = b;
  }
  __syncthreads();
  const int L = seg_lanes(cg), lane = tid & (L - 1);
  for (int g = tid / L; g < G; g += GT / L) {
    float a = 0.f, b = 0.f;
    for (int c = lane; c < cg; c += L) {
      const float w = gamma[g * cg + c];
      a += w * l1[g * cg + c];
      b += w * l2[g * cg + c];
    }
    a = seg_sum(a, L);
    b = seg_sum(b, L);
    if (lane == 0) gpart[((size_t)n * chunks + ch) * G + g] = make_float2(a, b);
  }
}

// dx, and the residual's gradient dz when it is wanted
template <typename T, int VEC, int ACT, int SLOPE>
__global__ __launch_bounds__(GT) void gn_bwd_apply_kernel(
    const T* __restrict__ dout, const T* __restrict__ x, const T* __restrict__ res, const uint8_t* __restrict__ mask,
    const float* __restrict__ gamma, const float* __restrict__ beta, const float2* __restrict__ stats,
    const float2* __restrict__ gpart, T* __restrict__ dx, T* __restrict__ dres, int HW, int C, int G, int chunks, int P) {
  extern __shared__ float lds[];  // mean(gamma dz) [G], mean(gamma dz xhat) [G]
  const GnGeo geo(C, VEC);
  const int n = blockIdx.x / chunks, ch = blockIdx.x - n * chunks;
  const int tid = threadIdx.x, cg = C / G;
  {
    const int L = chunk_lanes(chunks), lane = tid & (L - 1);
    const float inv = 1.f / ((float)HW * cg);
    join_chunks(gpart + (size_t)n * chunks * G, chunks, G, L, [&](int g, const float2& t) {
      const float a = seg_sum(t.x, L), b = seg_sum(t.y, L);
      if (lane == 0) {
        lds[g] = a * inv;
        lds[G + g] = b * inv;
      }
    });
  }
  __syncthreads();
  const int row = tid / geo.CW, tc = tid - row * geo.CW;
  if (row >= geo.R) return;
  const int p0 = ch * P, np = min(P, HW - p0);
  const size_t base = ((size_t)n * HW + p0) * C;
  for (int col = tc; col < geo.cols; col += geo.CW) {
    // dx = a dz - (m1 rstd + (x - mu) m2 rstd^2)
    float mu[VEC], a[VEC], be[VEC], c1[VEC], c2[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const int c = col * VEC + k, g = c / cg;
      const float2 st = stats[(size_t)n * G + g];
      mu[k] = st.x;
      a[k] = gamma[c] * st.y;
      be[k] = beta[c];
      c1[k] = lds[g] * st.y;
      c2[k] = lds[G + g] * st.y * st.y;
    }
    for (int p = row; p < np; p += geo.R) {
      const size_t o = base + (size_t)p * C + col * VEC;
      float v[VEC], g[VEC], r[VEC], dz[VEC], d[VEC];
      gn_load<T, VEC>(x + o, v);
      gn_load<T, VEC>(dout + o, g);
      if constexpr (SLOPE == kOfXRes && ACT != 0) gn_load<T, VEC>(res + o, r);
      unsigned bits = 0;
      if constexpr (SLOPE == kOfMask) bits = mask[o / VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[k] -= mu[k];
      gn_dz<VEC, ACT, SLOPE>(v, g, r, bits, a, be, dz);
#pragma unroll
      for (int k = 0; k < VEC; ++k) d[k] = fmaf(a[k], dz[k], -fmaf(v[k], c2[k], c1[k]));
      gn_store<T, VEC>(dx + o, d);
      if (dres) gn_store<T, VEC>(dres + o, dz);
    }
  }
}

// Column sums of src [rows][2][C] in fp64: block (x, y) sums 64 columns over its share of the rows, 16 row
// lanes joined in a fixed order.  One share: d_beta (half 0) and d_gamma (half 1) are written or added to;
// more: mid [shares][2 C], which a second pass of this kernel sums.
template <typename S>
__global__ __launch_bounds__(1024) void gn_dparam_kernel(const S* __restrict__ src, double* __restrict__ mid,
                                                         float* __restrict__ dgamma, float* __restrict__ dbeta,
                                                         long long rows, int C, int accumulate) {
  __shared__ double part[16][64];
  const int c = threadIdx.x & 63, r = threadIdx.x >> 6;
  const int j = blockIdx.x * 64 + c;
  const long long per = (rows + gridDim.y - 1) / gridDim.y, lo = blockIdx.y * per, hi = min(rows, lo + per);
  double s = 0.0;
  if (j < 2 * C) {
#pragma unroll 8
    for (long long i = lo + r; i < hi; i += 16) s += src[(size_t)i * 2 * C + j];
  }
  part[r][c] = s;
  __syncthreads();
  if (r == 0 && j < 2 * C) {
    for (int k = 1; k < 16; ++k) s += part[k][c];
    if (mid) {
      mid[(size_t)blockIdx.y * 2 * C + j] = s;
    } else {
      float* d = j < C ? dbeta + j : dgamma + (j - C);
      *d = accumulate ? *d + (float)s : (float)s;
    }
  }
}

// ------------------------------------------------------------------- host
struct GnPlan {
  int vec, chunks, P, R;
};

int gn_vec(int C, int esize, uintptr_t align) {
  int v = 16 / esize;
  while (v > 1 && (C % v != 0 || align % (uintptr_t)(v * esize) != 0)) v >>= 1;
  return v;
}

// Chunks of about N HW / blocks pixels: 2,048 blocks forward, 4,096 backward (256 x 56 x 56 x 256 bf16:
// 117 us + 242 us against 124 + 243 for stats and apply forward, 186 + 320 against 225 + 347 backward), but
// at least 48 KiB each and 4 pixels a thread, for a block joins all of its sample's partials first (64 x 112 x
// 112 x 64 forward: 83 us in chunks of 49 KiB, 109 in 25), and at most 64 a sample.
GnPlan gn_plan(int N, int HW, int C, int esize, uintptr_t align, int blocks) {
  GnPlan p;
  p.vec = gn_vec(C, esize, align);
  const int cols = C / p.vec;
  const int CW = cols < GT ? cols : GT;
  p.R = GT / CW;
  long long per = ((long long)N * HW + blocks - 1) / blocks;
  // the floor on the bytes holds where the device is full all the same (512 blocks of it)
  const long long floor_px = (48 << 10) / ((long long)C * esize);
  if ((long long)N * HW / 512 >= floor_px) per = std::max(per, floor_px);
  per = std::max<long long>({per, (HW + kMaxChunks - 1) / kMaxChunks, (long long)p.R * GU});
  if (per > HW) per = HW;
  p.P = (int)per;
  p.chunks = (HW + p.P - 1) / p.P;
  return p;
}
constexpr int kFwdBlocks = 2048, kBwdBlocks = 4096;

size_t gn_lds_stats(const GnPlan& p, int C) { return (size_t)2 * p.R * C * sizeof(float); }

template <typename F>
int gn_dispatch_vec(int esize, int vec, F&& f) {
  if (esize == 2) {
    if (vec == 8) return f(bf16_t{}, std::integral_constant<int, 8>{});
    if (vec == 4) return f(bf16_t{}, std::integral_constant<int, 4>{});
    if (vec == 2) return f(bf16_t{}, std::integral_constant<int, 2>{});
    return f(bf16_t{}, std::integral_constant<int, 1>{});
  }
  if (vec == 4) return f(float{}, std::integral_constant<int, 4>{});
  if (vec == 2) return f(float{}, std::integral_constant<int, 2>{});
  return f(float{}, std::integral_constant<int, 1>{});
}

// f(activation, slope): without a residual the slope is of x; ReLU's may be in the mask
template <typename F>
int gn_dispatch_act(int act, bool res, bool mask, F&& f) {
  typedef std::integral_constant<int, 0> N;
  typedef std::integral_constant<int, 1> R;
  typedef std::integral_constant<int, 2> S;
  if (act == 0) return f(N{}, std::integral_constant<int, kOfX>{});  // its slope is 1 with a residual too
  if (act == 1 && mask) return f(R{}, std::integral_constant<int, kOfMask>{});
  if (act == 1) return res ? f(R{}, std::integral_constant<int, kOfXRes>{}) : f(R{}, std::integral_constant<int, kOfX>{});
  return res ? f(S{}, std::integral_constant<int, kOfXRes>{}) : f(S{}, std::integral_constant<int, kOfX>{});
}

// the statistics kernels keep two fp32 [R][C] arrays in LDS
template <typename K>
int gn_allow_lds(K kernel, size_t bytes) {
  if (bytes <= 64 * 1024) return 0;
  return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                             (int)bytes) == hipSuccess ? 0 : 3;
}

bool gn_args_ok(const GnArgs& a) {
  return a.N >= 1 && a.HW >= 1 && a.C >= 1 && a.C <= kGnMaxChannels && a.G >= 1 && a.C % a.G == 0 &&
         (a.esize == 2 || a.esize == 4) && a.act >= 0 && a.act <= 2 && a.N <= (1 << 23);
}

uintptr_t gn_align(std::initializer_list<const void*> ps) {
  uintptr_t o = 16;
  for (const void* p : ps) o |= reinterpret_cast<uintptr_t>(p);
  return o & (~o + 1);  // lowest set bit: every pointer is a multiple of it
}

}  // namespace

namespace {

int gn_shares(long long rows) {  // of dparam's first pass: about 64 rows each, where two passes pay
  const long long n = rows <= 512 ? 1 : (rows + 63) / 64;
  return n > 64 ? 64 : (int)n;
}

// the narrowest vectors make the most chunks; the caller's pointers decide the width later
long long gn_max_chunks(int N, int HW, int C, int esize, int blocks) {
  long long m = 0;
  for (int v = 16 / esize; v >= 1; v >>= 1) {
    if (C % v) continue;
    const GnPlan p = gn_plan(N, HW, C, esize, (uintptr_t)(v * esize), blocks);
    if (p.chunks > m) m = p.chunks;
  }
  return m;
}

}  // namespace

bool gn_wants_mask(int C, int esize, int act, bool res) {
  return act == 1 && res && C % (16 / esize) == 0;
}

long long gn_fwd_workspace_floats(int N, int HW, int C, int G, int esize) {
  return 2 * (long long)N * gn_max_chunks(N, HW, C, esize, kFwdBlocks) * G;
}

long long gn_bwd_workspace_floats(int N, int HW, int C, int G, int esize) {
  const long long rows = N * gn_max_chunks(N, HW, C, esize, kBwdBlocks);
  return rows * (2ll * C + 2ll * G) + 64 * 2ll * C * 2 + 2;
}

int gn_fwd_launch(const GnArgs& a, hipStream_t st) {
  if (!gn_args_ok(a)) return 1;
  GnOne one;
  if (gn_one_plan(a.N, a.HW, a.C, a.G, a.esize, gn_align({a.x, a.res, a.out}), false, one))
    return gn_one_fwd(a, one, st);
  const GnPlan p = gn_plan(a.N, a.HW, a.C, a.esize, gn_align({a.x, a.res, a.out}), kFwdBlocks);
  if (a.mask && p.vec * a.esize != 16) return 2;  // one byte per 16-byte vector
  float2* part = reinterpret_cast<float2*>(a.ws);
  const size_t lds = gn_lds_stats(p, a.C), l2 = 2 * (size_t)a.G * sizeof(float);
  return gn_dispatch_vec(a.esize, p.vec, [&](auto t, auto vec) {
    using T = decltype(t);
    constexpr int V = decltype(vec)::value;
    const T* x = static_cast<const T*>(a.x);
    auto ks = gn_stats_kernel<T, V>;
    if (gn_allow_lds(ks, lds)) return 3;
    auto run = [&](auto ka) {
      if (gn_allow_lds(ka, l2)) return 3;
      hipLaunchKernelGGL(ks, dim3(a.N * p.chunks), dim3(GT), lds, st, x, part, a.HW, a.C, a.G, p.chunks, p.P);
      hipLaunchKernelGGL(ka, dim3(a.N * p.chunks), dim3(GT), l2, st, x, static_cast<const T*>(a.res), a.gamma, a.beta,
                         part, reinterpret_cast<float2*>(a.stats), static_cast<T*>(a.out), a.mask, a.HW, a.C, a.G,
                         p.chunks, p.P, a.eps);
      return 0;
    };
    if (a.mask) {
      if constexpr (V * sizeof(T) == 16) return run(gn_apply_kernel<T, V, 1, true, true>);
      return 2;
    }
    return gn_dispatch_act(a.act, a.res != nullptr, false, [&](auto act, auto) {
      constexpr int A = decltype(act)::value;
      return a.res ? run(gn_apply_kernel<T, V, A, true, false>) : run(gn_apply_kernel<T, V, A, false, false>);
    });
  });
}

int gn_bwd_launch(const GnArgs& a, hipStream_t st) {
  if (!gn_args_ok(a)) return 1;
  const uintptr_t align = gn_align({a.x, a.res, a.dout, a.dx, a.dres});
  const GnPlan p = gn_plan(a.N, a.HW, a.C, a.esize, align, kBwdBlocks);
  if (a.mask && p.vec * a.esize != 16) return 2;
  GnOne one;
  const bool in_one = (!a.res || a.act == 0) && gn_one_plan(a.N, a.HW, a.C, a.G, a.esize, align, a.act == 2, one);
  const long long rows = in_one ? a.N : (long long)a.N * p.chunks;
  float* cpart = a.ws;
  float2* gpart = reinterpret_cast<float2*>(a.ws + rows * 2 * a.C);
  const size_t lds = gn_lds_stats(p, a.C), l2 = 2 * (size_t)a.G * sizeof(float);
  const int rc = in_one ? gn_one_bwd(a, one, cpart, st) : gn_dispatch_vec(a.esize, p.vec, [&](auto t, auto vec) {
    using T = decltype(t);
    constexpr int V = decltype(vec)::value;
    return gn_dispatch_act(a.act, a.res != nullptr, a.mask != nullptr, [&](auto act, auto slope) {
      constexpr int A = decltype(act)::value, S = decltype(slope)::value;
      const T* x = static_cast<const T*>(a.x);
      const T* dy = static_cast<const T*>(a.dout);
      const T* rs = static_cast<const T*>(a.res);
      const float2* stt = reinterpret_cast<const float2*>(a.stats);
      auto ks = gn_bwd_stats_kernel<T, V, A, S>;
      auto ka = gn_bwd_apply_kernel<T, V, A, S>;
      if (gn_allow_lds(ks, lds) || gn_allow_lds(ka, l2)) return 3;
      hipLaunchKernelGGL(ks, dim3((unsigned)rows), dim3(GT), lds, st, dy, x, rs, a.mask, a.gamma, a.beta, stt, cpart,
                         gpart, a.HW, a.C, a.G, p.chunks, p.P);
      hipLaunchKernelGGL(ka, dim3((unsigned)rows), dim3(GT), l2, st, dy, x, rs, a.mask, a.gamma, a.beta, stt, gpart,
                         static_cast<T*>(a.dx), static_cast<T*>(a.dres), a.HW, a.C, a.G, p.chunks, p.P);
      return 0;
    });
  });
  if (rc) return rc;
  const int shares = gn_shares(rows), acc = a.accumulate ? 1 : 0;
  const dim3 cols((2 * a.C + 63) / 64);
  if (shares == 1) {
    hipLaunchKernelGGL(gn_dparam_kernel<float>, cols, dim3(1024), 0, st, cpart, nullptr, a.dgamma, a.dbeta, rows, a.C,
                       acc);
    return 0;
  }
  const uintptr_t end = reinterpret_cast<uintptr_t>(a.ws + rows * (2 * (size_t)a.C + 2 * (size_t)a.G));
  double* mid = reinterpret_cast<double*>((end + 7) & ~(uintptr_t)7);
  hipLaunchKernelGGL(gn_dparam_kernel<float>, dim3(cols.x, shares), dim3(1024), 0, st, cpart, mid, nullptr, nullptr, rows,
                     a.C, 0);
  hipLaunchKernelGGL(gn_dparam_kernel<double>, cols, dim3(1024), 0, st, mid, nullptr, a.dgamma, a.dbeta,
                     (long long)shares, a.C, acc);
  return 0;
}

}  // namespace pmd
