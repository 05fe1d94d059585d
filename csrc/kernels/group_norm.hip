// Group normalisation with the residual add and the activation, channels last (gfx950).
//
//   x [N][HW][C], G groups of cg = C/G consecutive channels, per (n, g) over HW x cg elements:
//     mu, var (biased),  rstd = 1/sqrt(var + eps),  xhat = (x - mu) rstd
//     z = gamma xhat + beta (+ residual),  out = act(z)           act: none, relu, silu
//   backward, dz = act'(z) dout (the residual's gradient), per (n, g):
//     dx = rstd (gamma dz - mean(gamma dz) - xhat mean(gamma dz xhat))
//     dgamma = sum_{n,hw} dz xhat,  dbeta = sum_{n,hw} dz
//
// Every pass is bound by memory; a thread owns VEC consecutive channels (16 bytes where the
// channel count and the pointers allow) and walks down the pixels, so any group width works
// the same way: statistics are taken per channel and joined into groups through LDS.
//
// A sample's pixels are split over `chunks` blocks.  Forward: stats kernel (one partial per
// (n, chunk, g)), then the apply kernel, whose blocks join the partials themselves.  Backward: the
// same pair over (dz, dz xhat), and one kernel that sums the per-channel partials to dgamma / dbeta.
//
// Variances are (count, mean, M2) triples in fp32: M2 about the mean of the few pixels a thread
// holds in registers, then joined pairwise (Chan, Golub, LeVeque 1983).  Sum and sum of squares
// would lose (mu/sigma)^2 of their precision.  All joins run in a fixed order: results do not depend
// on the scheduling.
#include "common.h"

namespace pmd {

namespace {

constexpr int GT = 256;   // threads of a block
constexpr int GU = 4;     // pixels a thread holds at once

template <typename T>
struct GnIo;
template <>
struct GnIo<bf16_t> {
  static __device__ __forceinline__ float up(bf16_t v) { return bf2f(v); }
  static __device__ __forceinline__ bf16_t down(float v) { return f2bf(v); }
};
template <>
struct GnIo<float> {
  static __device__ __forceinline__ float up(float v) { return v; }
  static __device__ __forceinline__ float down(float v) { return v; }
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) GnVec {
  T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ void gn_load(const T* p, float (&f)[VEC]) {
  const GnVec<T, VEC> r = *reinterpret_cast<const GnVec<T, VEC>*>(p);
#pragma unroll
  for (int k = 0; k < VEC; ++k) f[k] = GnIo<T>::up(r.v[k]);
}
template <typename T, int VEC>
__device__ __forceinline__ void gn_store(T* p, const float (&f)[VEC]) {
  GnVec<T, VEC> r;
#pragma unroll
  for (int k = 0; k < VEC; ++k) r.v[k] = GnIo<T>::down(f[k]);
  *reinterpret_cast<GnVec<T, VEC>*>(p) = r;
}

// NaN stays NaN (as torch's relu)
template <int ACT>
__device__ __forceinline__ float gn_act(float z) {
  if constexpr (ACT == 1) return z <= 0.f ? 0.f : z;
  if constexpr (ACT == 2) return z / (1.f + __expf(-z));
  return z;
}
template <int ACT>
__device__ __forceinline__ float gn_dact(float z, float g) {
  if constexpr (ACT == 1) return z <= 0.f ? 0.f : g;
  if constexpr (ACT == 2) {
    const float s = 1.f / (1.f + __expf(-z));
    return g * (s * (1.f + z * (1.f - s)));
  }
  return g;
}

// Block geometry: cols = C / VEC channel vectors; CW of them side by side, R pixel rows at once.
struct GnGeo {
  int cols, CW, R;
  __device__ __forceinline__ GnGeo(int C, int VEC) {
    cols = C / VEC;
    CW = cols < GT ? cols : GT;
    R = GT / CW;
  }
};

// sum over the L (power of two) lanes of a segment, every lane gets it
__device__ __forceinline__ float seg_sum(float v, int L) {
  for (int o = L >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// lanes that share one group's entries: the largest power of two <= min(64, entries)
__device__ __forceinline__ int seg_lanes(int entries) {
  int L = 1;
  while (L < 64 && L * 2 <= entries) L <<= 1;
  return L;
}

// ---------------------------------------------------------------- forward
// part [N][chunks][G] = (mean, M2) over the chunk's pixels x cg channels
template <typename T, int VEC>
__global__ __launch_bounds__(GT) void gn_stats_kernel(const T* __restrict__ x, float2* __restrict__ part, int HW,
                                                      int C, int G, int chunks, int P) {
  extern __shared__ float lds[];  // [R][C] means, [R][C] M2
  const GnGeo geo(C, VEC);
  const int n = blockIdx.x / chunks, ch = blockIdx.x - n * chunks;
  const int p0 = ch * P, np = min(P, HW - p0);
  const T* xb = x + ((size_t)n * HW + p0) * C;
  const int tid = threadIdx.x, row = tid / geo.CW, tc = tid - row * geo.CW;
  float* lm = lds;
  float* l2 = lds + geo.R * C;
  if (row < geo.R) {
    for (int col = tc; col < geo.cols; col += geo.CW) {
      float mean[VEC], m2[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) mean[k] = m2[k] = 0.f;
      int cnt = 0;
      for (int p = row; p < np; p += geo.R * GU) {
        float v[GU][VEC];
        int nu = 0;
#pragma unroll
        for (int u = 0; u < GU; ++u) {
          const int q = p + u * geo.R;
          if (q < np) {
            gn_load<T, VEC>(xb + (size_t)q * C + col * VEC, v[u]);
            nu = u + 1;
          }
        }
        const float inu = 1.f / nu, w = (float)nu / (cnt + nu), nn = (float)cnt * w;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          float s = 0.f, q = 0.f;
#pragma unroll
          for (int u = 0; u < GU; ++u)
            if (u < nu) s += v[u][k];
          s *= inu;
#pragma unroll
          for (int u = 0; u < GU; ++u)
            if (u < nu) q += (v[u][k] - s) * (v[u][k] - s);
          const float d = s - mean[k];
          mean[k] += d * w;
          m2[k] += q + d * d * nn;
        }
        cnt += nu;
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        lm[row * C + col * VEC + k] = mean[k];
        l2[row * C + col * VEC + k] = m2[k];
      }
    }
  }
  __syncthreads();
  // join the R x cg triples of a group
  const int cg = C / G, ent = geo.R * cg;
  const int L = seg_lanes(ent), lane = tid & (L - 1);
  const float inv = 1.f / ((float)np * cg);
  for (int g = tid / L; g < G; g += GT / L) {
    float s = 0.f;
    for (int e = lane; e < ent; e += L) {
      const int r = e / cg, c = e - r * cg;
      const int nr = (np - r + geo.R - 1) / geo.R;  // pixels of row r (0 when np <= r)
      s += nr * lm[r * C + g * cg + c];
    }
    const float mu = seg_sum(s, L) * inv;
    float q = 0.f;
    for (int e = lane; e < ent; e += L) {
      const int r = e / cg, c = e - r * cg;
      const int nr = (np - r + geo.R - 1) / geo.R;
      const float d = lm[r * C + g * cg + c] - mu;
      q += l2[r * C + g * cg + c] + nr * d * d;
    }
    q = seg_sum(q, L);
    if (lane == 0) part[((size_t)n * chunks + ch) * G + g] = make_float2(mu, q);
  }
}

// out = act(gamma (x - mu) rstd + beta + res); the blocks of chunk 0 store mu, rstd [N][G] for the
// backward
template <typename T, int VEC, int ACT, bool RES>
__global__ __launch_bounds__(GT) void gn_apply_kernel(const T* __restrict__ x, const T* __restrict__ res,
                                                      const float* __restrict__ gamma, const float* __restrict__ beta,
                                                      const float2* __restrict__ part, float2* __restrict__ stats,
                                                      T* __restrict__ out, int HW, int C, int G, int chunks, int P,
                                                      float eps) {
  extern __shared__ float lds[];  // mu [G], rstd [G]
  const GnGeo geo(C, VEC);
  const int n = blockIdx.x / chunks, ch = blockIdx.x - n * chunks;
  const int tid = threadIdx.x, cg = C / G;
  {
    const float2* pn = part + (size_t)n * chunks * G;
    const int L = seg_lanes(chunks), lane = tid & (L - 1);
    const float total = (float)HW * cg;
    for (int g = tid / L; g < G; g += GT / L) {
      float s = 0.f;
      for (int c = lane; c < chunks; c += L) s += (float)min(P, HW - c * P) * pn[(size_t)c * G + g].x;
      const float mu = seg_sum(s, L) / HW;
      float q = 0.f;
      for (int c = lane; c < chunks; c += L) {
        const float2 t = pn[(size_t)c * G + g];
        const float d = t.x - mu;
        q += t.y + (float)min(P, HW - c * P) * cg * d * d;
      }
      const float rstd = rsqrtf(seg_sum(q, L) / total + eps);
      if (lane == 0) {
        lds[g] = mu;
        lds[G + g] = rstd;
        if (ch == 0) stats[(size_t)n * G + g] = make_float2(mu, rstd);
      }
    }
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
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[k] = gn_act<ACT>(v[k]);
      gn_store<T, VEC>(out + o, v);
    }
  }
}

// --------------------------------------------------------------- backward
// cpart [N][chunks][2][C] = sums over the chunk's pixels of dz and dz xhat (per channel);
// gpart [N][chunks][G] = their gamma-weighted sums over the group
template <typename T, int VEC, int ACT, bool RES>
__global__ __launch_bounds__(GT) void gn_bwd_stats_kernel(
    const T* __restrict__ dout, const T* __restrict__ x, const T* __restrict__ res, const float* __restrict__ gamma,
    const float* __restrict__ beta, const float2* __restrict__ stats, float* __restrict__ cpart,
    float2* __restrict__ gpart, int HW, int C, int G, int chunks, int P) {
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
      float mu[VEC], rs[VEC], ga[VEC], be[VEC], s1[VEC], s2[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const int c = col * VEC + k;
        const float2 st = stats[(size_t)n * G + c / cg];
        mu[k] = st.x;
        rs[k] = st.y;
        ga[k] = gamma[c];
        be[k] = beta[c];
        s1[k] = s2[k] = 0.f;
      }
      for (int p = row; p < np; p += geo.R) {
        const size_t o = base + (size_t)p * C + col * VEC;
        float v[VEC], g[VEC], r[VEC];
        gn_load<T, VEC>(x + o, v);
        gn_load<T, VEC>(dout + o, g);
        if constexpr (RES) gn_load<T, VEC>(res + o, r);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          // z in the forward's own steps (a = gamma rstd, one fma): its sign is the forward's
          float z = fmaf(v[k] - mu[k], ga[k] * rs[k], be[k]);
          if constexpr (RES) z += r[k];
          const float dz = gn_dact<ACT>(z, g[k]);
          s1[k] += dz;
          s2[k] += dz * ((v[k] - mu[k]) * rs[k]);
        }
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        l1[row * C + col * VEC + k] = s1[k];
        l2[row * C + col * VEC + k] = s2[k];
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

// dx, and with RES the residual's gradient dz
template <typename T, int VEC, int ACT, bool RES>
__global__ __launch_bounds__(GT) void gn_bwd_apply_kernel(
    const T* __restrict__ dout, const T* __restrict__ x, const T* __restrict__ res, const float* __restrict__ gamma,
    const float* __restrict__ beta, const float2* __restrict__ stats, const float2* __restrict__ gpart,
    T* __restrict__ dx, T* __restrict__ dres, int HW, int C, int G, int chunks, int P) {
  extern __shared__ float lds[];  // mean(gamma dz) [G], mean(gamma dz xhat) [G]
  const GnGeo geo(C, VEC);
  const int n = blockIdx.x / chunks, ch = blockIdx.x - n * chunks;
  const int tid = threadIdx.x, cg = C / G;
  {
    const float2* pn = gpart + (size_t)n * chunks * G;
    const int L = seg_lanes(chunks), lane = tid & (L - 1);
    const float inv = 1.f / ((float)HW * cg);
    for (int g = tid / L; g < G; g += GT / L) {
      float a = 0.f, b = 0.f;
      for (int c = lane; c < chunks; c += L) {
        const float2 t = pn[(size_t)c * G + g];
        a += t.x;
        b += t.y;
      }
      a = seg_sum(a, L);
      b = seg_sum(b, L);
      if (lane == 0) {
        lds[g] = a * inv;
        lds[G + g] = b * inv;
      }
    }
  }
  __syncthreads();
  const int row = tid / geo.CW, tc = tid - row * geo.CW;
  if (row >= geo.R) return;
  const int p0 = ch * P, np = min(P, HW - p0);
  const size_t base = ((size_t)n * HW + p0) * C;
  for (int col = tc; col < geo.cols; col += geo.CW) {
    float mu[VEC], rs[VEC], ga[VEC], be[VEC], m1[VEC], m2[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const int c = col * VEC + k, g = c / cg;
      const float2 st = stats[(size_t)n * G + g];
      mu[k] = st.x;
      rs[k] = st.y;
      ga[k] = gamma[c];
      be[k] = beta[c];
      m1[k] = lds[g];
      m2[k] = lds[G + g];
    }
    for (int p = row; p < np; p += geo.R) {
      const size_t o = base + (size_t)p * C + col * VEC;
      float v[VEC], g[VEC], r[VEC], d[VEC];
      gn_load<T, VEC>(x + o, v);
      gn_load<T, VEC>(dout + o, g);
      if constexpr (RES) gn_load<T, VEC>(res + o, r);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        float z = fmaf(v[k] - mu[k], ga[k] * rs[k], be[k]);
        if constexpr (RES) z += r[k];
        const float dz = gn_dact<ACT>(z, g[k]);
        const float xh = (v[k] - mu[k]) * rs[k];
        d[k] = (ga[k] * dz - m1[k] - xh * m2[k]) * rs[k];
        if constexpr (RES) r[k] = dz;
      }
      gn_store<T, VEC>(dx + o, d);
      if constexpr (RES) gn_store<T, VEC>(dres + o, r);
    }
  }
}

// dst [C] (+)= sum over rows of src [rows][2][C], half 0 -> dbeta, half 1 -> dgamma; the rows are
// split over the 16 row lanes of a block of 64 columns and joined in a fixed order
__global__ __launch_bounds__(1024) void gn_dparam_kernel(const float* __restrict__ src, float* __restrict__ dgamma,
                                                         float* __restrict__ dbeta, long long rows, int C,
                                                         int accumulate) {
  __shared__ double part[16][64];
  const int c = threadIdx.x & 63, r = threadIdx.x >> 6;
  const int j = blockIdx.x * 64 + c;
  double s = 0.0;
  if (j < 2 * C)
    for (long long i = r; i < rows; i += 16) s += src[(size_t)i * 2 * C + j];
  part[r][c] = s;
  __syncthreads();
  if (r == 0 && j < 2 * C) {
    for (int k = 1; k < 16; ++k) s += part[k][c];
    float* d = j < C ? dbeta + j : dgamma + (j - C);
    *d = accumulate ? *d + (float)s : (float)s;
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

GnPlan gn_plan(int N, int HW, int C, int esize, uintptr_t align) {
  GnPlan p;
  p.vec = gn_vec(C, esize, align);
  const int cols = C / p.vec;
  const int CW = cols < GT ? cols : GT;
  p.R = GT / CW;
  // about 2048 blocks over the batch, each at least 4 pixels a thread and at most 64 chunks a sample
  long long per = ((long long)N * HW + 2047) / 2048;
  const long long lo = (HW + 63) / 64;
  if (per < lo) per = lo;
  if (per < (long long)p.R * GU) per = (long long)p.R * GU;
  if (per > HW) per = HW;
  p.P = (int)per;
  p.chunks = (HW + p.P - 1) / p.P;
  return p;
}

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

template <typename F>
int gn_dispatch_act(int act, bool res, F&& f) {
  if (res) {
    if (act == 0) return f(std::integral_constant<int, 0>{}, std::true_type{});
    if (act == 1) return f(std::integral_constant<int, 1>{}, std::true_type{});
    return f(std::integral_constant<int, 2>{}, std::true_type{});
  }
  if (act == 0) return f(std::integral_constant<int, 0>{}, std::false_type{});
  if (act == 1) return f(std::integral_constant<int, 1>{}, std::false_type{});
  return f(std::integral_constant<int, 2>{}, std::false_type{});
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
         (a.esize == 2 || a.esize == 4) && a.act >= 0 && a.act <= 2 && (long long)a.N * 64 < (1ll << 31);
}

uintptr_t gn_align(std::initializer_list<const void*> ps) {
  uintptr_t o = 16;
  for (const void* p : ps) o |= reinterpret_cast<uintptr_t>(p);
  return o & (~o + 1);  // lowest set bit: every pointer is a multiple of it
}

}  // namespace

long long gn_fwd_workspace_floats(int N, int HW, int C, int G, int esize) {
  // the narrowest vectors make the most chunks; the caller's pointers decide the width later
  long long m = 0;
  for (int v = 16 / esize; v >= 1; v >>= 1) {
    if (C % v) continue;
    const GnPlan p = gn_plan(N, HW, C, esize, (uintptr_t)(v * esize));
    if (p.chunks > m) m = p.chunks;
  }
  return 2 * (long long)N * m * G;
}

long long gn_bwd_workspace_floats(int N, int HW, int C, int G, int esize) {
  const long long rows = gn_fwd_workspace_floats(N, HW, C, G, esize) / (2 * G);
  return rows * (2ll * C + 2ll * G);
}

int gn_fwd_launch(const GnArgs& a, hipStream_t st) {
  if (!gn_args_ok(a)) return 1;
  const GnPlan p = gn_plan(a.N, a.HW, a.C, a.esize, gn_align({a.x, a.res, a.out}));
  float2* part = reinterpret_cast<float2*>(a.ws);
  const size_t lds = gn_lds_stats(p, a.C);
  return gn_dispatch_vec(a.esize, p.vec, [&](auto t, auto vec) {
    using T = decltype(t);
    constexpr int V = decltype(vec)::value;
    const T* x = static_cast<const T*>(a.x);
    auto ks = gn_stats_kernel<T, V>;
    if (gn_allow_lds(ks, lds)) return 3;
    hipLaunchKernelGGL(ks, dim3(a.N * p.chunks), dim3(GT), lds, st, x, part, a.HW, a.C, a.G, p.chunks, p.P);
    return gn_dispatch_act(a.act, a.res != nullptr, [&](auto act, auto res) {
      auto ka = gn_apply_kernel<T, V, decltype(act)::value, decltype(res)::value>;
      const size_t l2 = 2 * (size_t)a.G * sizeof(float);
      if (gn_allow_lds(ka, l2)) return 3;
      hipLaunchKernelGGL(ka, dim3(a.N * p.chunks), dim3(GT), l2, st, x, static_cast<const T*>(a.res), a.gamma, a.beta,
                         part, reinterpret_cast<float2*>(a.stats), static_cast<T*>(a.out), a.HW, a.C, a.G, p.chunks,
                         p.P, a.eps);
      return 0;
    });
  });
}

int gn_bwd_launch(const GnArgs& a, hipStream_t st) {
  if (!gn_args_ok(a)) return 1;
  const GnPlan p = gn_plan(a.N, a.HW, a.C, a.esize, gn_align({a.x, a.res, a.dout, a.dx, a.dres}));
  const long long rows = (long long)a.N * p.chunks;
  float* cpart = a.ws;
  float2* gpart = reinterpret_cast<float2*>(a.ws + rows * 2 * a.C);
  const size_t lds = gn_lds_stats(p, a.C);
  const int rc = gn_dispatch_vec(a.esize, p.vec, [&](auto t, auto vec) {
    using T = decltype(t);
    constexpr int V = decltype(vec)::value;
    return gn_dispatch_act(a.act, a.res != nullptr, [&](auto act, auto res) {
      constexpr int A = decltype(act)::value;
      constexpr bool RS = decltype(res)::value;
      const T* x = static_cast<const T*>(a.x);
      const T* dy = static_cast<const T*>(a.dout);
      const T* rs = static_cast<const T*>(a.res);
      const float2* stt = reinterpret_cast<const float2*>(a.stats);
      auto ks = gn_bwd_stats_kernel<T, V, A, RS>;
      if (gn_allow_lds(ks, lds)) return 3;
      hipLaunchKernelGGL(ks, dim3((unsigned)rows), dim3(GT), lds, st, dy, x, rs, a.gamma, a.beta, stt, cpart, gpart,
                         a.HW, a.C, a.G, p.chunks, p.P);
      auto ka = gn_bwd_apply_kernel<T, V, A, RS>;
      const size_t l2 = 2 * (size_t)a.G * sizeof(float);
      if (gn_allow_lds(ka, l2)) return 3;
      hipLaunchKernelGGL(ka, dim3((unsigned)rows), dim3(GT), l2, st, dy, x, rs, a.gamma, a.beta, stt, gpart,
                         static_cast<T*>(a.dx), static_cast<T*>(a.dres), a.HW, a.C, a.G, p.chunks, p.P);
      return 0;
    });
  });
  if (rc) return rc;
  hipLaunchKernelGGL(gn_dparam_kernel, dim3((2 * a.C + 63) / 64), dim3(1024), 0, st, cpart, a.dgamma, a.dbeta, rows,
                     a.C, a.accumulate ? 1 : 0);
  return 0;
}

}  // namespace pmd
