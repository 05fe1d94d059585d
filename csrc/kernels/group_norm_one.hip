// Group normalisation in one pass over the data, for samples whose groups fit a block's registers (gfx950).
//
// A block takes the pixels of one sample x CB channels (whole groups; 48 to 512 bytes of a pixel, so that
// lines are read whole or by neighbours at once), every thread up to K vectors of 16 bytes of the same channels.  It reads each input
// once, takes the statistics from its registers, and writes: the formulas are those of
// kernels/group_norm.hip, whose kernels read the data twice.
//
// Statistics: a thread takes mean and M2 of each of its channels (two sweeps of its registers), triples
// (count, mean, M2) are joined through LDS, rows of threads first, then the channels of a group, always in
// the same order.
#include "group_norm.h"

#include <type_traits>

namespace pmd {

namespace {

constexpr int kOneThreads = 512;

typedef u32x4_nt Raw;  // 16 bytes as they lie in memory: 8 bf16 or 4 fp32

// One sample of a tensor as a buffer of the hardware's: loads past its end give 0 and stores there are dropped,
// so that the K pixels of a thread need neither branches nor an address register each.
struct GnBuf {
  __amdgpu_buffer_rsrc_t r;
  __device__ __forceinline__ GnBuf(const void* p, size_t offset, unsigned bytes)
      : r(__builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(static_cast<const char*>(p)) + offset, 0, bytes,
                                            0x00020000)) {}
  __device__ __forceinline__ Raw load(unsigned o) const { return __builtin_amdgcn_raw_buffer_load_b128(r, o, 0, 0); }
  __device__ __forceinline__ unsigned load_byte(unsigned o) const {
    return __builtin_amdgcn_raw_buffer_load_b8(r, o, 0, 0);
  }
  __device__ __forceinline__ void store(const Raw& v, unsigned o) const {
    __builtin_amdgcn_raw_buffer_store_b128(v, r, o, 0, 0);
  }
  __device__ __forceinline__ void store_byte(unsigned v, unsigned o) const {
    __builtin_amdgcn_raw_buffer_store_b8((unsigned char)v, r, o, 0, 0);
  }
};

// The compiler is to unpack r anew in every sweep, one vector after the other: kept unpacked, or taken several
// at a time, the vectors take twice the registers.
__device__ __forceinline__ void again(Raw& r) {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" : "+v"(r));
}

__device__ __forceinline__ Raw gn_down(const float (&f)[8]) {
  const uint4 w = pack8(f);
  return Raw{w.x, w.y, w.z, w.w};
}
__device__ __forceinline__ Raw gn_down(const float (&f)[4]) {
  return Raw{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
}
__device__ __forceinline__ void gn_up(const Raw& r, float (&f)[8]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f[2 * k] = __uint_as_float(r[k] << 16);
    f[2 * k + 1] = __uint_as_float(r[k] & 0xffff0000u);
  }
}
__device__ __forceinline__ void gn_up(const Raw& r, float (&f)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) f[k] = __uint_as_float(r[k]);
}
// element k becomes 0 unless keep
template <int VEC>
__device__ __forceinline__ void gn_clear(Raw& r, int k, bool keep) {
  if constexpr (VEC == 4) r[k] = keep ? r[k] : 0u;
  else r[k / 2] &= keep ? 0xffffffffu : k % 2 ? 0x0000ffffu : 0xffff0000u;
}

// A block's place: sample n, channels c0 .. c0 + CB, this thread's vector tc of them and its first pixel row
struct GnSpot {
  int n, c0, tc, row, R, CB, each, more, have;
  __device__ __forceinline__ GnSpot(int HW, int C, int CB_, int VEC) : CB(CB_) {
    const int nb = C / CB, b = xcd_remap(blockIdx.x, gridDim.x);  // neighbours share lines of 128 bytes
    n = b / nb;
    c0 = (b - n * nb) * CB;
    const int cols = CB / VEC;
    R = blockDim.x / cols;
    row = threadIdx.x / cols;
    tc = threadIdx.x - row * cols;
    each = HW / R;
    more = HW - each * R;
    have = pixels(row);
  }
  __device__ __forceinline__ int pixels(int r) const { return each + (r < more ? 1 : 0); }  // of a row of threads
};

template <typename T, int VEC, int ACT, bool RES, bool MASK, int K>
__global__ __launch_bounds__(kOneThreads) void gn_one_fwd_kernel(const T* __restrict__ x, const T* __restrict__ res,
                                                                 const float* __restrict__ gamma,
                                                                 const float* __restrict__ beta,
                                                                 float2* __restrict__ stats, T* __restrict__ out,
                                                                 uint8_t* __restrict__ mask, int HW, int C, int G,
                                                                 int CB, float eps) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const GnSpot at(HW, C, CB, VEC);
  const int tid = threadIdx.x, NT = blockDim.x, cg = C / G, S = NT / CB, groups = CB / cg;
  const unsigned bytes = (unsigned)HW * C * sizeof(T);
  const size_t sample = (size_t)at.n * bytes;
  const unsigned o0 = ((unsigned)at.row * C + at.c0 + at.tc * VEC) * sizeof(T), step = (unsigned)at.R * C * sizeof(T);
  const GnBuf xb(x, sample, bytes), rb(RES ? res : x, sample, bytes), ob(out, sample, bytes);
  const GnBuf mb(MASK ? mask : nullptr, sample / 16, MASK ? bytes / 16 : 0);
  Raw v[K];
#pragma unroll
  for (int i = 0; i < K; ++i) v[i] = xb.load(o0 + i * step);
  float* lm = lds;                 // [R][CB]
  float* l2 = lm + NT * VEC;
  float* sm = l2 + NT * VEC;       // [S][CB]
  float* s2 = sm + NT;
  float* sc = s2 + NT;             // [S]
  float* gm = sc + S;              // [groups] mean, rstd
  {
    float mean[VEC], m2[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) mean[k] = m2[k] = 0.f;
#pragma unroll
    for (int i = 0; i < K; ++i) {
      float f[VEC];
      again(v[i]);
    gn_up(v[i], f);
#pragma unroll
      for (int k = 0; k < VEC; ++k) mean[k] += f[k];
    }
    const float in = 1.f / max(1, at.have);
#pragma unroll
    for (int k = 0; k < VEC; ++k) mean[k] *= in;
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const float w = i < at.have ? 1.f : 0.f;
      float f[VEC];
      again(v[i]);
      gn_up(v[i], f);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float d = (f[k] - mean[k]) * w;
        m2[k] = fmaf(d, d, m2[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < VEC; k += 4) {
      *reinterpret_cast<float4*>(lm + tid * VEC + k) = make_float4(mean[k], mean[k + 1], mean[k + 2], mean[k + 3]);
      *reinterpret_cast<float4*>(l2 + tid * VEC + k) = make_float4(m2[k], m2[k + 1], m2[k + 2], m2[k + 3]);
    }
  }
  // K = 25: one block a compute unit; its loads of the residual are under way while the sums are joined (256 x 56
  // x 56 x 256: 322 us without, 281 with).  Otherwise other blocks' loads are, and it changes nothing.
  constexpr int P = RES && K == 25 ? K : 0;
  Raw pre[P ? P : 1];
  if constexpr (P > 0) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < P; ++i) pre[i] = rb.load(o0 + i * step);
  }
  __syncthreads();
  {  // a channel's rows s, s + S, ..
    const int c = tid % CB, s = tid / CB;
    float cnt = 0.f, t = 0.f, q = 0.f;
    for (int r = s; r < at.R; r += S) {
      const float nr = (float)at.pixels(r);
      cnt += nr;
      t += nr * lm[r * CB + c];
    }
    const float mu = t / fmaxf(cnt, 1.f);
    for (int r = s; r < at.R; r += S) {
      const float nr = (float)at.pixels(r), d = lm[r * CB + c] - mu;
      q += nr > 0.f ? l2[r * CB + c] + nr * d * d : 0.f;
    }
    sm[tid] = mu;
    s2[tid] = q;
    if (c == 0) sc[s] = cnt;
  }
  __syncthreads();
  {  // a group's S x cg triples
    const int ent = S * cg, L = seg_lanes(ent), lane = tid & (L - 1);
    for (int g = tid / L; g < groups; g += NT / L) {
      float t = 0.f, q = 0.f;
      for (int e = lane; e < ent; e += L) {
        const int s = e / cg, c = g * cg + e - s * cg;
        t += sc[s] * sm[s * CB + c];
      }
      const float mu = seg_sum(t, L) / ((float)HW * cg);
      for (int e = lane; e < ent; e += L) {
        const int s = e / cg, c = g * cg + e - s * cg;
        const float d = sm[s * CB + c] - mu;
        q += sc[s] > 0.f ? s2[s * CB + c] + sc[s] * d * d : 0.f;
      }
      const float rstd = rsqrtf(seg_sum(q, L) / ((float)HW * cg) + eps);
      if (lane == 0) {
        gm[g] = mu;
        gm[groups + g] = rstd;
        stats[(size_t)at.n * G + at.c0 / cg + g] = make_float2(mu, rstd);
      }
    }
  }
  __syncthreads();
  float mu[VEC], a[VEC], b[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    const int c = at.tc * VEC + k, g = c / cg;
    mu[k] = gm[g];
    a[k] = gamma[at.c0 + c] * gm[groups + g];
    b[k] = beta[at.c0 + c];
  }
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const unsigned o = o0 + i * step;
    float f[VEC];
    again(v[i]);
    gn_up(v[i], f);
#pragma unroll
    for (int k = 0; k < VEC; ++k) f[k] = fmaf(f[k] - mu[k], a[k], b[k]);
    if constexpr (RES) {
      float r[VEC];
      if constexpr (P > 0) {
        again(pre[i]);
        gn_up(pre[i], r);
      } else {
        gn_up(rb.load(o), r);
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) f[k] += r[k];
    }
    if constexpr (MASK) {
      unsigned bits = 0;
#pragma unroll
      for (int k = 0; k < VEC; ++k) bits |= f[k] <= 0.f ? 0u : 1u << k;
      mb.store_byte(bits, o / 16);
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k) f[k] = gn_act<ACT>(f[k]);
    ob.store(gn_down(f), o);
  }
}

// ReLU's slope is 0 or 1: dz replaces dout in its registers.  SiLU's dz is computed again for dx.
template <typename T, int VEC, int ACT, int SLOPE, int K>
__global__ __launch_bounds__(kOneThreads) void gn_one_bwd_kernel(const T* __restrict__ dout, const T* __restrict__ x,
                                                                 const uint8_t* __restrict__ mask,
                                                                 const float* __restrict__ gamma,
                                                                 const float* __restrict__ beta,
                                                                 const float2* __restrict__ stats,
                                                                 float* __restrict__ cpart, T* __restrict__ dx,
                                                                 T* __restrict__ dres, int HW, int C, int G, int CB) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const GnSpot at(HW, C, CB, VEC);
  const int tid = threadIdx.x, NT = blockDim.x, cg = C / G, S = NT / CB, groups = CB / cg;
  const unsigned bytes = (unsigned)HW * C * sizeof(T);
  const size_t sample = (size_t)at.n * bytes;
  const unsigned o0 = ((unsigned)at.row * C + at.c0 + at.tc * VEC) * sizeof(T), step = (unsigned)at.R * C * sizeof(T);
  const GnBuf xb(x, sample, bytes), gb(dout, sample, bytes), db(dx, sample, bytes);
  const GnBuf rb(dres ? dres : dx, sample, dres ? bytes : 0);
  const GnBuf mb(SLOPE == kOfMask ? mask : nullptr, sample / 16, SLOPE == kOfMask ? bytes / 16 : 0);
  Raw v[K], g[K];  // past the end: 0, which adds nothing
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const unsigned o = o0 + i * step;
    v[i] = xb.load(o);
    g[i] = gb.load(o);
    if constexpr (SLOPE == kOfMask) {
      const unsigned bits = mb.load_byte(o / 16);
#pragma unroll
      for (int k = 0; k < VEC; ++k) gn_clear<VEC>(g[i], k, (bits >> k) & 1);
    }
  }
  float* l1 = lds;                 // [R][CB]
  float* l2 = l1 + NT * VEC;
  float* s1 = l2 + NT * VEC;       // [S][CB]
  float* s2 = s1 + NT;
  float* gm = s2 + NT;             // [groups] mean(gamma dz), mean(gamma dz xhat)
  constexpr bool kOfZ = ACT != 0 && SLOPE == kOfX;  // the slope takes z
  float mu[VEC], a[VEC], be[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    const int c = at.c0 + at.tc * VEC + k;
    const float2 st = stats[(size_t)at.n * G + c / cg];
    mu[k] = st.x;
    if constexpr (kOfZ) {
      a[k] = gamma[c] * st.y;
      be[k] = beta[c];
    }
  }
  {
    float t1[VEC], t2[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) t1[k] = t2[k] = 0.f;
#pragma unroll
    for (int i = 0; i < K; ++i) {
      float f[VEC], dz[VEC], r[VEC];
      again(v[i]);
      gn_up(v[i], f);
#pragma unroll
      for (int k = 0; k < VEC; ++k) f[k] -= mu[k];
      again(g[i]);
      if constexpr (ACT == 1 && SLOPE == kOfX) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) gn_clear<VEC>(g[i], k, !(fmaf(f[k], a[k], be[k]) <= 0.f));
        again(g[i]);
      }
      gn_up(g[i], dz);
      if constexpr (ACT == 2) gn_dz<VEC, ACT, SLOPE>(f, dz, r, 0u, a, be, dz);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        t1[k] += dz[k];
        t2[k] = fmaf(dz[k], f[k], t2[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < VEC; k += 4) {
      *reinterpret_cast<float4*>(l1 + tid * VEC + k) = make_float4(t1[k], t1[k + 1], t1[k + 2], t1[k + 3]);
      *reinterpret_cast<float4*>(l2 + tid * VEC + k) = make_float4(t2[k], t2[k + 1], t2[k + 2], t2[k + 3]);
    }
  }
  if constexpr (ACT != 2)
    if (dres) {  // under way while the sums are joined (256 x 56 x 56 x 256: 426 us without, 408 with)
#pragma unroll
      for (int i = 0; i < K; ++i) rb.store(g[i], o0 + i * step);
    }
  __syncthreads();
  {
    const int c = tid % CB, s = tid / CB;
    float t = 0.f, q = 0.f;
    for (int r = s; r < at.R; r += S) {
      t += l1[r * CB + c];
      q += l2[r * CB + c];
    }
    s1[tid] = t;
    s2[tid] = q;
  }
  __syncthreads();
  for (int c = tid; c < CB; c += NT) {
    float t = 0.f, q = 0.f;
    for (int s = 0; s < S; ++s) {
      t += s1[s * CB + c];
      q += s2[s * CB + c];
    }
    q *= stats[(size_t)at.n * G + (at.c0 + c) / cg].y;
    float* cp = cpart + (size_t)at.n * 2 * C + at.c0 + c;
    cp[0] = t;
    cp[C] = q;
    const float w = gamma[at.c0 + c];
    l1[c] = w * t;  // the rows were summed before the last barrier
    l2[c] = w * q;
  }
  __syncthreads();
  {
    const int L = seg_lanes(cg), lane = tid & (L - 1);
    const float in = 1.f / ((float)HW * cg);
    for (int q = tid / L; q < groups; q += NT / L) {
      float t = 0.f, u = 0.f;
      for (int c = lane; c < cg; c += L) {
        t += l1[q * cg + c];
        u += l2[q * cg + c];
      }
      t = seg_sum(t, L);
      u = seg_sum(u, L);
      if (lane == 0) {
        gm[q] = t * in;
        gm[groups + q] = u * in;
      }
    }
  }
  __syncthreads();
  float c1[VEC], c2[VEC];  // dx = a dz - (m1 rstd + (x - mu) m2 rstd^2)
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    const int c = at.tc * VEC + k, q = c / cg;
    const float rstd = stats[(size_t)at.n * G + (at.c0 + c) / cg].y;
    c1[k] = gm[q] * rstd;
    c2[k] = gm[groups + q] * rstd * rstd;
    if constexpr (!kOfZ) a[k] = gamma[at.c0 + c] * rstd;
  }
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const unsigned o = o0 + i * step;
    float f[VEC], dz[VEC], d[VEC];
    again(v[i]);
    gn_up(v[i], f);
    again(g[i]);
    gn_up(g[i], dz);
#pragma unroll
    for (int k = 0; k < VEC; ++k) f[k] -= mu[k];
    if constexpr (ACT == 2) {
      float r[VEC];
      gn_dz<VEC, ACT, SLOPE>(f, dz, r, 0u, a, be, dz);
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k) d[k] = fmaf(a[k], dz[k], -fmaf(f[k], c2[k], c1[k]));
    db.store(gn_down(d), o);
    if constexpr (ACT == 2) rb.store(gn_down(dz), o);
  }
}

size_t gn_one_lds(const GnOne& o, int vec, int groups) {
  return ((size_t)2 * o.NT * vec + 2 * o.NT + o.NT / o.CB + 2 * groups) * sizeof(float);
}

template <typename F>
int with_k(int k, F&& f) {
  if (k <= 7) return f(std::integral_constant<int, 7>{});
  if (k <= 13) return f(std::integral_constant<int, 13>{});
  return f(std::integral_constant<int, 25>{});
}

}  // namespace

// The smallest K that takes all pixels with at most 512 threads, lines of 128 bytes first: 64 bytes take 256 x 14 x 14
// x 1,024 from 67 + 98 us (forward + backward) to 79 + 116, and 32 bytes 256 x 56 x 56 x 256 from 322 + 427 to 365 +
// 457, although K is then 13.  The kernels that read twice take 355 + 533 us there, 90 + 157 for 256 x 14 x 14 x 1,024,
// 17 + 15 for 16 x 7 x 7 x 512 (these 8.6 + 10).  K = 25 is for 256 blocks at least, one a compute unit: with two, 1 x
// 56 x 56 x 64 takes 19 + 22 us, and 19 + 15 split over more.  SiLU's backward would spill at K = 25.
bool gn_one_plan(int N, int HW, int C, int G, int esize, uintptr_t align, bool silu_bwd, GnOne& o) {
  const int vec = 16 / esize, cg = C / G;
  if (align % 16 || C % vec) return false;
  // the widths behind the first four are for groups whose channels are no power of two (256 x 28 x 28 x 96 in 8
  // groups: 29 + 48 us, 39 + 58 read twice)
  const int limits[] = {7, 13, 25}, widths[] = {8, 4, 16, 32, 12, 6, 24, 10, 20, 14, 28, 5, 7, 3};
  for (int k : limits)
    for (int cols : widths) {
      const int CB = cols * vec;
      if (CB % cg || C % CB) continue;
      if (k == 25 && (silu_bwd || (long long)N * (C / CB) < 256)) continue;
      // whole rows, and whole slots of CB threads; powers of two where the columns are one (256 x 28 x 28 x 512: 147 +
      // 203 us with 512 threads, 149 + 214 with the 448 that would do)
      const bool two = (cols & (cols - 1)) == 0;
      for (int nt = 128; nt <= kOneThreads; nt += two ? nt : 64)
        if (nt % CB == 0 && HW <= (long long)k * (nt / cols) && (long long)N * (C / CB) * nt < (1ll << 32)) {
          o = GnOne{CB, nt, k};
          return true;
        }
    }
  return false;
}

int gn_one_fwd(const GnArgs& a, const GnOne& o, hipStream_t st) {
  const dim3 grid((unsigned)((long long)a.N * (a.C / o.CB))), block(o.NT);
  const size_t lds = gn_one_lds(o, 16 / a.esize, o.CB / (a.C / a.G));
  return with_k(o.K, [&](auto k) {
    constexpr int K = decltype(k)::value;
    auto run = [&](auto t, auto act, auto res, auto mask) {
      using T = decltype(t);
      constexpr int V = 16 / sizeof(T);
      hipLaunchKernelGGL((gn_one_fwd_kernel<T, V, decltype(act)::value, decltype(res)::value, decltype(mask)::value, K>),
                         grid, block, lds, st, static_cast<const T*>(a.x), static_cast<const T*>(a.res), a.gamma, a.beta,
                         reinterpret_cast<float2*>(a.stats), static_cast<T*>(a.out), a.mask, a.HW, a.C, a.G, o.CB, a.eps);
      return 0;
    };
    auto typed = [&](auto t) {
      auto acts = [&](auto res) {
        if (a.act == 0) return run(t, std::integral_constant<int, 0>{}, res, std::false_type{});
        if (a.act == 2) return run(t, std::integral_constant<int, 2>{}, res, std::false_type{});
        if constexpr (decltype(res)::value)
          if (a.mask) return run(t, std::integral_constant<int, 1>{}, res, std::true_type{});
        return run(t, std::integral_constant<int, 1>{}, res, std::false_type{});
      };
      return a.res ? acts(std::true_type{}) : acts(std::false_type{});
    };
    return a.esize == 2 ? typed(bf16_t{}) : typed(float{});
  });
}

int gn_one_bwd(const GnArgs& a, const GnOne& o, float* cpart, hipStream_t st) {
  const dim3 grid((unsigned)((long long)a.N * (a.C / o.CB))), block(o.NT);
  const size_t lds = gn_one_lds(o, 16 / a.esize, o.CB / (a.C / a.G));
  return with_k(o.K, [&](auto k) {
    constexpr int K = decltype(k)::value;
    auto run = [&](auto t, auto act, auto slope) {
      using T = decltype(t);
      constexpr int V = 16 / sizeof(T);
      hipLaunchKernelGGL((gn_one_bwd_kernel<T, V, decltype(act)::value, decltype(slope)::value, K>), grid, block, lds, st,
                         static_cast<const T*>(a.dout), static_cast<const T*>(a.x), a.mask, a.gamma, a.beta,
                         reinterpret_cast<const float2*>(a.stats), cpart, static_cast<T*>(a.dx), static_cast<T*>(a.dres),
                         a.HW, a.C, a.G, o.CB);
      return 0;
    };
    auto typed = [&](auto t) {
      typedef std::integral_constant<int, kOfX> X;
      if (a.act == 0) return run(t, std::integral_constant<int, 0>{}, X{});
      if constexpr (K <= 13)  // gn_one_plan
        if (a.act == 2) return run(t, std::integral_constant<int, 2>{}, X{});
      if (a.act == 2) return 2;
      if (a.mask) return run(t, std::integral_constant<int, 1>{}, std::integral_constant<int, kOfMask>{});
      return run(t, std::integral_constant<int, 1>{}, X{});
    };
    return a.esize == 2 ? typed(bf16_t{}) : typed(float{});
  });
}

}  // namespace pmd
