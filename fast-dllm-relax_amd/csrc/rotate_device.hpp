// Norms and rotation of heads: what a thread does with its part of one.
#pragma once
#include "paged_device.hpp"
#include "rotate.hpp"

namespace fdllm {

// Eight threads take a head.  Thread u has two runs of 8 dims, from `lo` and `hi`, in which pairs 8 u .. 8 u + 7 lie
// whatever the layout: the halves' runs side by side, or 16 neighbouring dims.  Behind the turned dims (u >= rot / 16): 16
// neighbouring dims too.
struct HeadPart { int lo, hi; bool turned; };
__device__ __forceinline__ HeadPart head_part(const TurnP& t, int u) {
  const bool turned = 16 * u < t.rot;
  return turned && !t.inter ? HeadPart{8 * u, 8 * u + t.rot / 2, true} : HeadPart{16 * u, 16 * u + 8, turned};
}

template <int DT, class R>
__device__ __forceinline__ void load_part(const uint16_t* head, HeadPart p, R (&x)[16]) {
  float a[8], b[8];
  unpack8<DT>(*reinterpret_cast<const u32x4*>(head + p.lo), a);
  unpack8<DT>(*reinterpret_cast<const u32x4*>(head + p.hi), b);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = a[e];
    x[8 + e] = b[e];
  }
}
// Normed by w, the norm's weights of this part.  The sum of squares is taken in 64 bits, which hold that of any value of the
// dtype; its root by the hardware's estimate and two steps of Newton's method, r (3 - v r^2) / 2.
template <class R>
__device__ __forceinline__ void norm_part(R (&x)[16], const float (&w)[16], float eps) {
  double v = 0;
#pragma unroll
  for (int e = 0; e < 16; ++e) v = __builtin_fma((double)x[e], (double)x[e], v);
#pragma unroll
  for (int k = 1; k < 8; k *= 2) v += __shfl_xor(v, k, WAVE);
  v = __builtin_fma(v, 1.0 / HD, (double)eps);
  double r = __builtin_amdgcn_rsq(v);
#pragma unroll
  for (int k = 0; k < 2; ++k) r *= __builtin_fma(-0.5 * v * r, r, 1.5);
  r = v < INFINITY ? r : 1.0 / v;  // (infinite: 0)
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] *= (R)r * (R)w[e];
}
// pair e of this part (e < 8) turned
template <bool INTER, class R>
__device__ __forceinline__ void turn_pair(R (&x)[16], int e, R sn, R cs) {
  const int i = INTER ? 2 * e : e, j = INTER ? 2 * e + 1 : 8 + e;
  const R a = x[i], b = x[j];
  x[i] = a * cs - b * sn;
  x[j] = b * cs + a * sn;
}

}  // namespace fdllm
