// Device helpers of the paged caches' kernels: rows and pages of a sequence, rotation by position.
#pragma once
#include "common.hpp"
#include "paged.hpp"
#include "paged_index.hpp"

namespace fdllm {

constexpr int HD = 128;

// a load from memory that the launch only reads, at a uniform address: through the scalar cache, a fraction of a vector
// load's latency
__device__ __forceinline__ int ld_const(const int32_t* p) {
  return *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)p;
}
__device__ __forceinline__ RowSpan seq_rows(const SeqRowsP& s, int b) {
  if (s.row_start == nullptr) return seq_span(nullptr, s.rows, s.max_rows, b);
  const int32_t two[2] = {ld_const(s.row_start + b), ld_const(s.row_start + b + 1)};
  return seq_span(two, s.rows, s.max_rows, 0);
}
template <class C>
__device__ __forceinline__ int page_of(const C& c, int b, long long j) {
  return page_at(c.table + b * c.table_ld, c.table_w, c.num_pages, j);
}

// sine and cosine of t turns
__device__ __forceinline__ void turn_sincos(double t, float& sn, float& cs) {
  sincospif(2.0f * (float)(t - __builtin_rint(t)), &sn, &cs);
}
// as their series to the 11th and 10th power of at most pi / 4: within 2^-33.  The coefficients: (2 pi)^k / k!, signed
constexpr double SIN1 = 6.283185307179586, SIN3 = -41.34170224039976, SIN5 = 81.60524927607506, SIN7 = -76.70585975306139,
                 SIN9 = 42.058693944897655, SIN11 = -15.09464257682299;
constexpr double COS2 = -19.739208802178716, COS4 = 64.9393940226683, COS6 = -85.45681720669373, COS8 = 60.24464137187666,
                 COS10 = -26.4262567833744;
__device__ __forceinline__ void turn_sincos(double t, double& sn, double& cs) {
  constexpr double BIG = 6755399441055744.0;  // 1.5 x 2^52: adding it rounds to whole numbers, its low word holds them
  const double m = __builtin_fma(t, 4.0, BIG);
  const int k = (int)__double_as_longlong(m);
  const double z = __builtin_fma(m - BIG, -0.25, t), w = z * z;  // |z| <= 1 / 8 of a turn
  double s = SIN11, c = COS10;
  s = __builtin_fma(s, w, SIN9);
  c = __builtin_fma(c, w, COS8);
  s = __builtin_fma(s, w, SIN7);
  c = __builtin_fma(c, w, COS6);
  s = __builtin_fma(s, w, SIN5);
  c = __builtin_fma(c, w, COS4);
  s = __builtin_fma(s, w, SIN3);
  c = __builtin_fma(c, w, COS2);
  s = __builtin_fma(s, w, SIN1) * z;
  c = __builtin_fma(c, w, 1.0);
  sn = k & 1 ? c : s;
  cs = k & 1 ? s : c;
  sn = k & 2 ? -sn : sn;
  cs = (k + 1) & 2 ? -cs : cs;
}
template <int DT>
__device__ __forceinline__ void unpack8(u32x4 w, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = lo_f32<DT>(w[e]);
    x[2 * e + 1] = hi_f32<DT>(w[e]);
  }
}
// the pair x, y turned
template <class R>
__device__ __forceinline__ void rotate(float& x, float& y, R sn, R cs) {
  const R a = x, b = y;
  x = (float)(a * cs - b * sn);
  y = (float)(b * cs + a * sn);
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

}  // namespace fdllm
