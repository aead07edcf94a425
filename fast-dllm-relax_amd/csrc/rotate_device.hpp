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

// the values of the other lanes of eight: lane ^ 1, ^ 2 and (equal among each four lanes then) 7 - lane
template <int CTRL> __device__ __forceinline__ float other_lane(float v) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xf, 0xf, false));
}
template <int CTRL> __device__ __forceinline__ double other_lane(double v) {
  const long long b = __double_as_longlong(v);
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)b, CTRL, 0xf, 0xf, false);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, 0xf, 0xf, false);
  return __longlong_as_double((long long)((unsigned long long)hi << 32 | lo));
}
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_MIRROR8 = 0x141;

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
// dtype; its root by the hardware's estimate (within 2^-24) and a step of Newton's method, r (3 - v r^2) / 2.
// Its inverse r may be beyond fp32 (a row of bf16's largest or least values), and times w sooner: x, which r leaves at most
// sqrt(128) of, takes r's power of two by itself, r's fraction next and w last.
template <class R>
__device__ __forceinline__ void norm_part(R (&x)[16], const float (&w)[16], float eps) {
  double part[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 16; ++e) part[e & 3] = __builtin_fma((double)x[e], (double)x[e], part[e & 3]);
  double v = (part[0] + part[1]) + (part[2] + part[3]);
  v += other_lane<DPP_XOR1>(v);
  v += other_lane<DPP_XOR2>(v);
  v += other_lane<DPP_MIRROR8>(v);
  v = __builtin_fma(v, 1.0 / HD, (double)eps);
  double r = __builtin_amdgcn_rsq(v);
  r *= __builtin_fma(-0.5 * v * r, r, 1.5);
  r = v < INFINITY ? r : 1.0 / v;  // (infinite: 0)
  if constexpr (sizeof(R) == 8) {
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] *= r * w[e];
  } else {
    const int k = __builtin_amdgcn_frexp_exp(r);
    const float m = (float)__builtin_amdgcn_frexp_mant(r);
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = __builtin_amdgcn_ldexpf(x[e], k) * m * w[e];
  }
}
// pair e of this part (e < 8) turned
template <bool INTER, class R>
__device__ __forceinline__ void turn_pair(R (&x)[16], int e, R sn, R cs) {
  const int i = INTER ? 2 * e : e, j = INTER ? 2 * e + 1 : 8 + e;
  const R a = x[i], b = x[j];
  x[i] = a * cs - b * sn;
  x[j] = b * cs + a * sn;
}
// sine and cosine of t turns, times gain: the angle is reduced in 64 bits; the hardware's sine and cosine take turns and are
// within 2^-22.9 here (the results are rounded to 16 bits)
__device__ __forceinline__ void turn_sincos16(double t, float gain, float& sn, float& cs) {
  const float f = (float)(t - __builtin_rint(t));
  sn = __builtin_amdgcn_sinf(f) * gain;
  cs = __builtin_amdgcn_cosf(f) * gain;
}

// Up to H of a row's heads, from head h0, from `in` to `out` (which may be one): normed where `norm`, turned by position pos,
// rounded once to the model dtype.  All is read before anything of the same head is written.
template <int DT, bool INTER, int H>
__device__ __forceinline__ void turn_heads(const TurnP& t, int u, double pos, const uint16_t* in, const uint16_t* norm,
                                           uint16_t* out, int h0, int heads) {
  const HeadPart p = head_part(t, u);
  float x[H][16], w[16];
#pragma unroll
  for (int h = 0; h < H; ++h)
    if (h0 + h < heads) load_part<DT>(in + (h0 + h) * HD, p, x[h]);
  if (norm) {
    load_part<DT>(norm, p, w);
#pragma unroll
    for (int h = 0; h < H; ++h)
      if (h0 + h < heads) norm_part(x[h], w, t.eps);
  }
  if (p.turned) {
    const float gain = (float)t.gain;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float sn, cs;
      turn_sincos16(pos * t.turn[8 * u + e], gain, sn, cs);
#pragma unroll
      for (int h = 0; h < H; ++h) turn_pair<INTER>(x[h], e, sn, cs);
    }
  }
#pragma unroll
  for (int h = 0; h < H; ++h) {
    if (h0 + h >= heads) break;
    uint16_t* dst = out + (h0 + h) * HD;
    u32x4 lo, hi;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      lo[e] = pack_f32x2<DT>(x[h][2 * e], x[h][2 * e + 1]);
      hi[e] = pack_f32x2<DT>(x[h][8 + 2 * e], x[h][9 + 2 * e]);
    }
    *reinterpret_cast<u32x4*>(dst + p.lo) = lo;
    *reinterpret_cast<u32x4*>(dst + p.hi) = hi;
  }
}

}  // namespace fdllm
