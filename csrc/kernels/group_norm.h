// What the group norm's kernels share: vectors of 16 bytes or less, activations, lane sums.
#pragma once
#include "common.h"

namespace pmd {

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

// Where the activation's slope comes from: z of x alone, z of x and the residual, or the forward's bits.
enum GnSlope { kOfX, kOfXRes, kOfMask };

// dz of one vector; xc = x - mu
template <int VEC, int ACT, int SLOPE>
__device__ __forceinline__ void gn_dz(const float (&xc)[VEC], const float (&g)[VEC], const float (&r)[VEC],
                                      unsigned bits, const float (&a)[VEC], const float (&be)[VEC], float (&dz)[VEC]) {
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    if constexpr (ACT == 0) {
      dz[k] = g[k];
    } else if constexpr (SLOPE == kOfMask) {
      dz[k] = (bits >> k) & 1 ? g[k] : 0.f;
    } else {
      // z in the forward's own steps (a = gamma rstd, one fma): its sign is the forward's
      float z = fmaf(xc[k], a[k], be[k]);
      if constexpr (SLOPE == kOfXRes) z += r[k];
      dz[k] = gn_dact<ACT>(z, g[k]);
    }
  }
}

// Kernels that keep a sample's channels of whole groups in registers (kernels/group_norm_one.hip).
struct GnOne {
  int CB, NT, K;  // channels and threads of a block, pixels of a thread
};
bool gn_one_plan(int N, int HW, int C, int G, int esize, uintptr_t align, bool silu_bwd, GnOne& o);
int gn_one_fwd(const GnArgs& a, const GnOne& o, hipStream_t st);
// cpart [N][2][C]: per sample and channel the sums of dz and dz xhat
int gn_one_bwd(const GnArgs& a, const GnOne& o, float* cpart, hipStream_t st);

}  // namespace pmd
