// The paged 8-bit cache: appending rotated keys and values, and attention over it.
#include <algorithm>

#include "common.hpp"
#include "paged.hpp"
#include "paged_index.hpp"

namespace fdllm {

namespace {

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
__device__ __forceinline__ int page_of(const PagedP& c, int b, long long j) {
  return page_at(c.table + b * c.table_ld, c.table_w, c.num_pages, j);
}

// ---- append ------------------------------------------------------------------------------------
// Rotation by position: pair (i, i + 64) turns by pos theta^(-i/64) radians.  The angle is reduced in 64 bits (in
// turns: its whole part is dropped), so far positions keep their angle.  Queries, rounded to the model dtype after, are
// turned in fp32.  Keys are turned in 64 bits with one rounding to fp32, so that their bytes are those of the definition but
// where it lies within 2^-24 of a tie (in fp32 a few in a million lie on the other side of e4m3's rounding; us, fp32 / 64 bits,
// at an earlier step: 8192 rows 14.5 / 14.6, a ragged batch of 6200 rows 14.4 / 16.5).  A thread takes the 8 pairs of unit
// u (pairs 8 u .. 8 u + 7).  All sines and cosines together, against a build with constants in their place: 8192 rows
// 14.7 / 13.9, the ragged batch, whose workgroups compute those of a page anew for each kv head and four query heads, 14.9 / 12.0.
__device__ __forceinline__ double first_turn(const PagedAppendP& a, int u) {
  double t = 0.15915494309189533577;  // 1 / (2 pi)
  t *= (u & 1) ? a.turn8 : 1.0;
  t *= (u & 2) ? a.turn16 : 1.0;
  t *= (u & 4) ? a.turn32 : 1.0;
  return t;
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

// the least power of two s with amax <= 448 s, at least 2^-100 (448, e4m3's largest, is 0.875 x 2^9)
__device__ __forceinline__ float pow2_scale(float amax) {
  if (!(amax > 0.f)) return 0x1p-100f;
  int e;
  const float m = frexpf(amax, &e);
  e = e - 9 + (m > 0.875f ? 1 : 0);
  return ldexpf(1.0f, max(e, -100));
}
// four values as e4m3 bytes; what is not finite becomes NaN
__device__ __forceinline__ uint32_t to_e4m3(float a, float b, float c, float d) {
  const float nan = __uint_as_float(0x7fc00000u);
  a = finite(a) ? a : nan;
  b = finite(b) ? b : nan;
  c = finite(c) ? c : nan;
  d = finite(d) ? d : nan;
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
  return (uint32_t)r;
}
// four e4m3 bytes times r, as e4m3 bytes
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float r) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return to_e4m3(lo[0] * r, lo[1] * r, hi[0] * r, hi[1] * r);
}

// One workgroup takes one page of one sequence: of one kv head (blockIdx.y < nkv), or the queries of QH heads of
// the rows that fall into that page.  The page's new rows [w0, w1) (slots) are encoded with one scale per tensor:
// the least power of two that holds them, or the page's own where rows that stay are live in it and need more.
// Where the new rows need more than the page has, the rows that stay are encoded again with the larger scale:
// powers of two, so that only loses what falls under e4m3's least step.  Values go through LDS, since a row's
// values are a column of V's page, and leave it as 16-byte pieces; a piece with other rows in it is read first
// and keeps them (a page belongs to one sequence).
// (us with 2 / 4 / 6 / 12 heads, at an earlier step: 8192 rows 16.4 / 14.6 / 15.2 / 16.1, 24 prompts of up to 509 rows 18.0 /
// 16.4 / 16.9 / 16.3.)
// 8192 rows: 63 MB in 14.0 us, 4.5 TB/s, near a plain copy's 4.9.  The ragged batch: 47 MB in 13.7 us, its waves waiting for half
// of their cycles (lengths, table, page and rows one after the other in each workgroup).  One token is a launch of 5.5 us: those
// reads, which depend on each other.
constexpr int QH = 4;
// W: the slots that a workgroup has threads for: the whole page or, where a call has no more than 32 rows of a sequence,
// 32 from w0 on.  us, whole / 32: a token of each of 256 sequences in pages of 64 9.9 / 7.2, of 128 17.1 / 7.3; 32 rows
// of 64 sequences in pages of 128 14.4 / 9.5.  (16 from w0 on: 256 sequences 7.3 / 6.8, 16 of 8 rows 5.6 / 6.0.)
template <int DT, int PAGE, int W>
__global__ __launch_bounds__(W * 8) void paged_append_kernel(PagedAppendP a) {
  constexpr int NT = W * 8;                     // a thread takes one (slot, pair unit) item of K
  constexpr int VU = 2;                         // and two (slot, 8 dims) items of V
  constexpr int PP = W < PAGE ? W / 16 + 1 : PAGE / 16;  // 16-byte pieces of V's page that the rows may touch, for each dim
  constexpr int VP = (HD * PP + NT - 1) / NT;   // and for each thread
  constexpr int LDV = 16 * PP + 4;              // bytes from dim to dim in LDS
  __shared__ float red[2][NT / 64];
  __shared__ __align__(16) uint8_t vt[HD * LDV];
  const int tid = threadIdx.x;
  const int npp = (int)(gridDim.x / (unsigned)a.s.nseq);  // pages a sequence's rows can touch
  const int b = (int)blockIdx.x / npp, jj = (int)blockIdx.x % npp;
  const RowSpan rs = seq_rows(a.s, b);
  const int start = a.start[b];
  const PageSpan ps = page_span(start, rs.n, a.live ? a.live[b] : start, jj, a.c.shift);
  const int w0 = ps.w0, w1 = ps.w1;
  if (w0 >= w1) return;
  const long long row0 = rs.first - ps.rel;  // slot s is the call's row row0 + s
  const long long pos0 = (a.pos ? a.pos[b] : start) - ps.rel;
  const int base = W < PAGE ? w0 : 0, vbase = base & ~15;  // the first slots of this workgroup's items, and in LDS
  const int u = tid & 7;
  double f = first_turn(a, u);  // turns per position of this thread's next pair

  if ((int)blockIdx.y >= a.c.nkv) {
    // queries: rotated, rounded once to the model dtype
    const int h0 = ((int)blockIdx.y - a.c.nkv) * QH;
    const int s = base + (tid >> 3);
    if (s >= w0 && s < w1) {
      float sn[8], cs[8];
#pragma unroll
      for (int e = 0; e < 8; ++e, f *= a.turn1) turn_sincos((double)(pos0 + s) * f, sn[e], cs[e]);
      const uint16_t* src = a.q + (row0 + s) * a.ldq;
      uint16_t* dst = a.q_out + (row0 + s) * a.nq * HD;
#pragma unroll
      for (int h = 0; h < QH; ++h) {
        if (h0 + h >= a.nq) break;
        const int o = (h0 + h) * HD + 8 * u;
        float lo[8], hi[8];
        unpack8<DT>(*reinterpret_cast<const u32x4*>(src + o), lo);
        unpack8<DT>(*reinterpret_cast<const u32x4*>(src + o + 64), hi);
#pragma unroll
        for (int e = 0; e < 8; ++e) rotate(lo[e], hi[e], sn[e], cs[e]);
        u32x4 x, y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = pack2(from_f32<DT>(lo[2 * e]), from_f32<DT>(lo[2 * e + 1]));
          y[e] = pack2(from_f32<DT>(hi[2 * e]), from_f32<DT>(hi[2 * e + 1]));
        }
        *reinterpret_cast<u32x4*>(dst + o) = x;
        *reinterpret_cast<u32x4*>(dst + o + 64) = y;
      }
    }
    return;
  }

  const int pg = page_of(a.c, b, ps.j);
  if (pg < 0) return;
  const int h = blockIdx.y;
  const size_t ph = (size_t)pg * a.c.nkv + h;
  uint8_t* kp = a.c.k + ph * PAGE * HD;
  uint8_t* vp = a.c.v + ph * PAGE * HD;
  const int lv = ps.live;
  const bool keeps = ps.keeps;
  const float ks_old = a.c.ks[ph], vs_old = a.c.vs[ph];

  const int s = base + (tid >> 3);  // this thread's slot of K, and its unit u
  const bool mine = s >= w0 && s < w1;
  float klo[8], khi[8], vv[VU][8];
#pragma unroll
  for (int e = 0; e < 8; ++e) klo[e] = khi[e] = 0.f;
  if (mine) {
    const uint16_t* src = a.k + (row0 + s) * a.ldk + h * HD + 8 * u;
    unpack8<DT>(*reinterpret_cast<const u32x4*>(src), klo);
    unpack8<DT>(*reinterpret_cast<const u32x4*>(src + 64), khi);
  }
#pragma unroll
  for (int i = 0; i < VU; ++i) {
    const int sv = base + (tid >> 4) + W / 2 * i;
#pragma unroll
    for (int e = 0; e < 8; ++e) vv[i][e] = 0.f;
    if (sv >= w0 && sv < w1) unpack8<DT>(*reinterpret_cast<const u32x4*>(a.v + (row0 + sv) * a.ldv + h * HD + 8 * (tid & 15)), vv[i]);
  }
  // this thread's pieces of V's page: dim d, slots s0 .. s0 + 15, none from w1 on; read where they hold other rows too
  u32x4 held[VP];
  auto piece = [&](int k, int& d, int& s0) {
    const int p = tid + NT * k;
    d = W < PAGE ? p % HD : p / PP;
    s0 = vbase + 16 * (W < PAGE ? p / HD : p % PP);
    return p < HD * PP && s0 < w1 && s0 + 16 > w0;
  };
#pragma unroll
  for (int k = 0; k < VP; ++k) {
    int d, s0;
    held[k] = u32x4{0, 0, 0, 0};
    if (piece(k, d, s0) && (s0 < w0 || s0 + 16 > w1)) held[k] = *reinterpret_cast<const u32x4*>(vp + d * PAGE + s0);
  }
  float ka = 0.f, va = 0.f;
  if (mine) {
#pragma unroll
    for (int e = 0; e < 8; ++e, f *= a.turn1) {
      double sn, cs;
      turn_sincos((double)(pos0 + s) * f, sn, cs);
      rotate(klo[e], khi[e], sn, cs);
      ka = fmaxf(ka, finite(klo[e]) ? fabsf(klo[e]) : 0.f);
      ka = fmaxf(ka, finite(khi[e]) ? fabsf(khi[e]) : 0.f);
    }
  }
#pragma unroll
  for (int i = 0; i < VU; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) va = fmaxf(va, finite(vv[i][e]) ? fabsf(vv[i][e]) : 0.f);
  ka = wave_max(ka);
  va = wave_max(va);
  if ((tid & 63) == 0) {
    red[0][tid >> 6] = ka;
    red[1][tid >> 6] = va;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    ka = fmaxf(ka, red[0][w]);
    va = fmaxf(va, red[1][w]);
  }
  float ks = pow2_scale(ka), vs = pow2_scale(va);
  if (keeps) {
    ks = fmaxf(ks, ks_old);
    vs = fmaxf(vs, vs_old);
  }
  const float ki = 1.0f / ks, vi = 1.0f / vs;
  if (mine) {
    const auto& x = klo;
    const auto& y = khi;
    uint8_t* dst = kp + s * HD + 8 * u;
    *reinterpret_cast<u32x2*>(dst) = u32x2{to_e4m3(x[0] * ki, x[1] * ki, x[2] * ki, x[3] * ki),
                                           to_e4m3(x[4] * ki, x[5] * ki, x[6] * ki, x[7] * ki)};
    *reinterpret_cast<u32x2*>(dst + 64) = u32x2{to_e4m3(y[0] * ki, y[1] * ki, y[2] * ki, y[3] * ki),
                                                to_e4m3(y[4] * ki, y[5] * ki, y[6] * ki, y[7] * ki)};
  }
  if (keeps && ks > ks_old) {
    const float r = ks_old / ks;
#pragma unroll 1
    for (int p = tid; p < PAGE * 8; p += NT) {
      const int sl = p >> 3;  // (16 bytes of slot sl)
      if ((sl >= w0 && sl < w1) || sl >= lv) continue;
      u32x4 w = *reinterpret_cast<const u32x4*>(kp + 16 * p);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = rescale4(w[e], r);
      *reinterpret_cast<u32x4*>(kp + 16 * p) = w;
    }
  }
  // V: bytes of (slot, 8 dims) items into their dims' rows
#pragma unroll
  for (int i = 0; i < VU; ++i) {
    const int sv = base + (tid >> 4) + W / 2 * i;
    if (sv < w0 || sv >= w1) continue;
    const auto& x = vv[i];
    const uint32_t lo = to_e4m3(x[0] * vi, x[1] * vi, x[2] * vi, x[3] * vi);
    const uint32_t hi = to_e4m3(x[4] * vi, x[5] * vi, x[6] * vi, x[7] * vi);
    uint8_t* t = vt + 8 * (tid & 15) * LDV + sv - vbase;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      t[e * LDV] = (uint8_t)(lo >> (8 * e));
      t[(4 + e) * LDV] = (uint8_t)(hi >> (8 * e));
    }
  }
  __syncthreads();
  const bool grow = keeps && vs > vs_old;
  const float r = vs_old / vs;
#pragma unroll
  for (int k = 0; k < VP; ++k) {
    int d, s0;
    if (!piece(k, d, s0)) continue;
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t fresh = *reinterpret_cast<const uint32_t*>(vt + d * LDV + s0 - vbase + 4 * e);
      const uint32_t old = held[k][e], moved = grow ? rescale4(old, r) : old;
      uint32_t out = 0;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int sl = s0 + 4 * e + t;
        const uint32_t m = 0xffu << (8 * t);
        out |= m & (sl >= w0 && sl < w1 ? fresh : sl < lv ? moved : old);
      }
      w[e] = out;
    }
    *reinterpret_cast<u32x4*>(vp + d * PAGE + s0) = w;
  }
  if (grow) {  // the other pieces
#pragma unroll 1
    for (int p = tid; p < PAGE * 8; p += NT) {
      const int s0 = 16 * (p % (PAGE / 16));
      if ((s0 < w1 && s0 + 16 > w0) || s0 >= lv) continue;
      u32x4 w = *reinterpret_cast<const u32x4*>(vp + 16 * p);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int live = min(max(lv - s0 - 4 * e, 0), 4);  // bytes of this word that are live
        const uint32_t m = live == 4 ? 0xffffffffu : (1u << (8 * live)) - 1u;
        w[e] = (rescale4(w[e], r) & m) | (w[e] & ~m);
      }
      *reinterpret_cast<u32x4*>(vp + 16 * p) = w;
    }
  }
  if (tid == 0) {
    a.c.ks[ph] = ks;
    a.c.vs[ph] = vs;
  }
}

// ---- attention ---------------------------------------------------------------------------------
// Rows: a sequence's n query rows x the G query heads of a kv head, flattened as row i, head g -> i G + g, in
// tiles of 16.  Keys: tiles of 64.  A wave computes S^T = K Q^T (rows: keys, columns: queries) and
// O^T = V^T P^T (rows: dims, columns: queries), both by 16x16x32 MFMAs, without LDS: every operand is a load
// from the pages, four bytes of e4m3 becoming four 16-bit values by two conversions.
//   Lane l = 16 g + c.  Key 16 g + 8 h + 4 a + i of a tile (g, i < 4; h, a < 2) is row 4 g + i of S^T's product
//   (h, a): so lane l holds after those four products the scores of query c with the 16 keys 16 g .. 16 g + 15, which
//   lie in one page (a page is a multiple of 16) and share its scales, and p of (h, a, i) is just what the second
//   product's operand wants as element 4 a + i of its k step h (keys 16 g + 8 h + 0..7 in lane group g): the
//   probabilities never change lanes.
//   K's scale and the softmax's factor multiply the scores; V's scale, 2^e f with f in [1, 2), is split: 2^e goes
//   into V's conversion, which takes one, as far as it leaves every byte in the model dtype's range (`Range`), and what is
//   left, f for any usual scale, into the exponent of p.
// p x f is rounded to the model dtype, half a step of its own size as the result's rounding.  Where a workgroup has one tile of
// rows (a token of each sequence, which waits for memory) what the rounding leaves goes through the second product too, so
// that the result's rounding is the only one that counts; two tiles would pay for that.  Error against 64 bits, once / in two
// parts: a token over 2080 keys 0.0022 / 0.0017, 64 of up to 8192 0.0018 / 0.0016, 2048 rows over 8192 0.0018 / 0.0017, and
// us 10.6 / 10.6, 29.6 / 30.2 (one pass over the same input after the other), 123 / 152; 16 sequences of 32 rows 13.3 / 15.4.
//   fp16 has no step of its own size below 2^-14 and nothing below 2^-25, and many keys of small p may carry a row: there p (and
// with it the sum) is 2^14 times as large.
// The running maximum is that of p x f over the query's whole row, which so is at most 1, held in each of its four lanes; the
// sum, of p, is each lane's own part until the end.

// The exponents that V's conversion takes (as a float's bits).  fp16: 448 x 2^7 is in range (256 x 2^8, as which 65504 is
// stored, is not), e4m3's least, 2^-9, is a whole number of fp16's least steps at 2^-15.  bf16: sums of many 448 x 2^60 stay
// in fp32's range (256 x 2^120, as which bf16's largest value is stored, is not).  A value past the range would be infinite, and
// 0 x inf NaN in the rows that do not attend it.
template <int DT> struct Range {
  static constexpr uint32_t LO = (DT == DT_F16 ? 127 - 15 : 127 - 100) << 23, HI = (DT == DT_F16 ? 127 + 7 : 127 + 60) << 23;
};
template <int DT>
__device__ __forceinline__ u32x4 e4m3x8(uint32_t w0, uint32_t w1, float s) {
  if constexpr (DT == DT_BF16) {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, true))};
  } else {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, s, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, s, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, s, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, s, true))};
  }
}

// bytes [n, 4) of word w (of keys) cleared; n may be anything
__device__ __forceinline__ uint32_t first_bytes(uint32_t w, int n) {
  return n >= 4 ? w : n <= 0 ? 0u : w & ((1u << (8 * n)) - 1u);
}
__device__ __forceinline__ u32x4 first_bytes16(u32x4 w, int n) {
  return u32x4{first_bytes(w[0], n), first_bytes(w[1], n - 4), first_bytes(w[2], n - 8), first_bytes(w[3], n - 12)};
}
// bit 7 of each byte of w that is e4m3's NaN (0x7f or 0xff: without its sign, the one that carries into bit 7 by + 1)
__device__ __forceinline__ uint32_t nan_bits(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// two probabilities rounded to the model dtype (2^x is no product, so fp16 needs none of pack_f32x2's care)
template <int DT>
__device__ __forceinline__ uint32_t pack_p(float a, float b) {
  if constexpr (DT == DT_BF16) return pack_f32x2<DT>(a, b);
  else return pack2(f32_to_f16(a), f32_to_f16(b));
}
// hides where w came from: what was computed of it before is computed again instead of kept in registers
__device__ __forceinline__ void anew(u32x4& w) { asm volatile("" : "+v"(w)); }

constexpr int KW = 4;  // waves of a workgroup
// One workgroup: T tiles of 16 flattened rows of one (sequence, kv head), a split of their keys, its key tiles taken in turn
// by KW waves, whose results are joined through LDS.  A wave converts each K and V operand once for its T tiles.
// The next tile's K is requested as soon as this one's scores are done, the next V after the second product, so each
// is on its way during the other half of the work without registers of its own; page numbers are requested a tile
// earlier.  The queries' operands stay in LDS (T tiles of them would be 16 T registers in every wave).
// 2048 rows over 8192 keys (90 GFLOP): 122 us, 0.74 PFLOP/s, bound by the pages' way from L2, 1.44 GB at 11.8 TB/s (89 us
// with the first tiles alone; no part of the arithmetic is worth more than 5 us).  A token of each of 64 sequences over
// 1024 to 8192 keys: 36 us, 3.7 TB/s of the pages.  32 rows over 32768 keys: 20 us and 4.5 to join the splits.
template <int DT, int T>
__global__ __launch_bounds__(64 * KW, 2) void paged_attn_kernel(PagedAttnP a) {
  __shared__ __align__(16) u32x4 qs[T][4][WAVE];
  __shared__ __align__(16) f32x4 so[KW][8][WAVE];
  __shared__ float sm[KW][16], sl[KW][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  // Workgroup id lies on XCD id % 8 (round robin).  A group's workgroups take the query tiles of one key range in
  // turn, all on one XCD, whose L2 then reads that range once; where there are fewer than eight ranges their
  // queries are cut into `cuts` groups.
  const int id = (int)blockIdx.x, xcd = id & 7, slot = id >> 3;
  const int group = slot / a.group_wgs * 8 + xcd, range = group / a.cuts;
  const int tile = slot % a.group_wgs * a.cuts + group % a.cuts;
  const int split = range % a.S, hk = range / a.S % a.c.nkv, b = range / a.S / a.c.nkv;
  if (b >= a.s.nseq) return;
  const int G = a.nq / a.c.nkv;
  const int page = a.c.page, shift = a.c.shift;
  const int32_t* table = a.c.table + b * a.c.table_ld;
  // the page numbers of a tile's four runs of 16 keys, as the table has them; pages() makes them -1 where they are
  // past the end or none
  struct Four { int p[4]; };
  auto entries = [&](int t) {
    Four f;
#pragma unroll
    for (int k = 0; k < 4; ++k) f.p[k] = ld_const(table + min((64 * t + 16 * k) >> shift, a.c.table_w - 1));
    return f;
  };
  // each of these is a memory's latency, so they go out together: the length, the queries, and without key splits
  // (whose place follows from the length) the wave's first pages
  const int len = ld_const(a.kv_len + b);
  const Four early = entries(a.S == 1 ? wave : 0);
  const RowSpan rs = seq_rows(a.s, b);
  const int first = rs.first, n = rs.n, M = n * G;
  const int m0 = 16 * T * tile;  // first flattened row of this workgroup
  if (m0 >= M) return;
  const int lk = min(max(len, 0), a.c.table_w * a.c.page);
  // flattened row m0 + r is query row i0 + row_of(r) of the sequence
  const int i0 = __builtin_amdgcn_readfirstlane(m0 / G), g0 = m0 - i0 * G;
  auto row_of = [&](int r) { return (int)(((unsigned)(g0 + r) * a.div24) >> 24); };
  // queries: dims 64 jj + 16 g + 8 h + 0..7 of column c are its part of k step (jj, h), which wave 2 jj + h reads for all tiles
  u32x4 qr[T];
#pragma unroll
  for (int k = 0; k < T; ++k) {
    const int r = 16 * k + c, jj = wave >> 1, h = wave & 1, i = row_of(r);
    qr[k] = u32x4{0, 0, 0, 0};
    if (m0 + r < M)
      qr[k] = *reinterpret_cast<const u32x4*>(a.q + (long long)(first + i0 + i) * a.ldq + (hk * G + g0 + r - i * G) * HD + 64 * jj +
                                              16 * g + 8 * h);
  }
  // keeps memory accesses on their side
  auto stay = [] { asm volatile("" ::: "memory"); };
  stay();
  // limits grow from row to row: all attend keys below kmin, none those from kmax on
  const int kmin = key_limit(len, lk, n, i0, a.mask_block);
  const int kmax = key_limit(len, lk, n, min(i0 + row_of(16 * T - 1), n - 1), a.mask_block);

  const int tiles = (kmax + 63) / 64, per = (tiles + a.S - 1) / a.S;
  const int t1 = min(tiles, (split + 1) * per);
  float m[T], l[T];
  uint32_t spoilt[T];  // bit 4 d + i: o[q][d][i] is NaN
  f32x4 o[T][8];
#pragma unroll
  for (int q = 0; q < T; ++q) {
    m[q] = -INFINITY;
    l[q] = 0.f;
    spoilt[q] = 0;
#pragma unroll
    for (int d = 0; d < 8; ++d) o[q][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const unsigned stride = (unsigned)(a.c.nkv * page) * HD;  // bytes from page to page
  const uint8_t *kbase = a.c.k + hk * page * HD, *vbase = a.c.v + hk * page * HD;
  const float *ksbase = a.c.ks + hk, *vsbase = a.c.vs + hk;
  auto pages = [&](int t, Four f) {
#pragma unroll
    for (int k = 0; k < 4; ++k) f.p[k] = 64 * t + 16 * k < lk && f.p[k] >= 0 && f.p[k] < a.c.num_pages ? f.p[k] : -1;
    return f;
  };
  auto pick = [](Four f, int k) { return k & 2 ? (k & 1 ? f.p[3] : f.p[2]) : (k & 1 ? f.p[1] : f.p[0]); };
  auto all_pages = [](Four f) { return (f.p[0] | f.p[1] | f.p[2] | f.p[3]) >= 0; };
  u32x4 kw[2][2][2], vw[8];  // K [h][a][jj]
  float ksn = 0.f, vsn = 0.f;
  auto load_k = [&](int t, Four f) {
    const int pk = pick(f, c >> 2);
    const uint8_t* kp = kbase + (unsigned long long)(unsigned)max(pk, 0) * stride +
                        ((((64 * t + 16 * (c >> 2)) & (page - 1)) + (c & 3)) * HD + 16 * g);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int aa = 0; aa < 2; ++aa)
#pragma unroll
        for (int jj = 0; jj < 2; ++jj)
          kw[h][aa][jj] = *reinterpret_cast<const u32x4*>(kp + (8 * h + 4 * aa) * HD + 64 * jj);
  };
  auto load_v = [&](int t, Four f) {
    const int pv = pick(f, g);
    const unsigned p = (unsigned)max(pv, 0);
    const uint8_t* vp = vbase + (unsigned long long)p * stride + (c * page + ((64 * t + 16 * g) & (page - 1)));
    const unsigned long long at = (unsigned long long)p * (unsigned)a.c.nkv;
    ksn = ksbase[at];
    vsn = vsbase[at];
#pragma unroll
    for (int d = 0; d < 8; ++d) vw[d] = *reinterpret_cast<const u32x4*>(vp + 16 * d * page);
  };

  // of a lane's 16 keys from key0, those that its query of tile q attends: the first so many (a column without a
  // query asks for no mask of its own)
  auto first_keys = [&](int q, bool none, int key0) {
    const int r = 16 * q + c;
    return none ? 0 : (m0 + r < M ? key_limit(len, lk, n, i0 + row_of(r), a.mask_block) : kmax) - key0;
  };
  // Tile t in the pages now, whose K, V and scales are loaded; the next tile's are requested on the way.
  int t = split * per + wave;
  Four now{}, next{};
  auto step = [&] {
    stay();  // (the queries' operands are read from LDS each time)
    // edge: some key is past a query's limit or the end, or in no page
    const bool edge = 64 * t + 64 > kmin || !all_pages(now);
    const int key0 = 64 * t + 16 * g;
    const bool none = edge && pick(now, g) < 0;
    const float ks = (none ? 1.0f : fmaxf(ksn, 0x1p-100f)) * a.scale_log2e;
    const float vs = none ? 1.0f : fmaxf(vsn, 0x1p-100f);
    if (edge) {  // (here, where few registers are in use)
      // what lies behind the sequence's end or in no page is nothing, NaN among it
      uint32_t nan = 0;
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        vw[d] = first_bytes16(vw[d], none ? 0 : lk - key0);
        nan |= nan_bits(vw[d][0]) | nan_bits(vw[d][1]) | nan_bits(vw[d][2]) | nan_bits(vw[d][3]);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (__any(nan != 0)) {
        // A masked probability is 0, and 0 x NaN is not.  So NaN is taken out of V, and put into the dims of those
        // queries that attend such a key: where the product of "is NaN" and "is attended" counts any.
#pragma unroll
        for (int q = 0; q < T; ++q) {
          const int lim = first_keys(q, none, key0);
          u32x4 at[2];
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              at[h][e] = pack2(from_f32<DT>(8 * h + 2 * e < lim ? 1.0f : 0.0f), from_f32<DT>(8 * h + 2 * e + 1 < lim ? 1.0f : 0.0f));
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            anew(vw[d]);
            u32x4 is;
#pragma unroll
            for (int e = 0; e < 4; ++e) is[e] = (nan_bits(vw[d][e]) >> 7) * 0x38;  // e4m3's 1
            f32x4 hit = mfma16<DT>(e4m3x8<DT>(is[0], is[1], 1.0f), at[0], f32x4{0.f, 0.f, 0.f, 0.f});
            hit = mfma16<DT>(e4m3x8<DT>(is[2], is[3], 1.0f), at[1], hit);
#pragma unroll
            for (int i = 0; i < 4; ++i) spoilt[q] |= hit[i] > 0.f ? 1u << (4 * d + i) : 0u;
            __builtin_amdgcn_sched_barrier(0);
          }
        }
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          anew(vw[d]);
#pragma unroll
          for (int e = 0; e < 4; ++e) vw[d][e] &= ~((nan_bits(vw[d][e]) >> 7) * 0xff);
        }
      }
    }
    f32x4 s[T][2][2];
    u32x4 qf[T][4];
#pragma unroll
    for (int q = 0; q < T; ++q)
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) qf[q][kk] = qs[q][kk][lane];
    // k step by k step, so that the products that follow each other add to different sums
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int aa = 0; aa < 2; ++aa) {
          const u32x4 w = kw[h][aa][kk >> 1];
          const u32x4 kf = kk & 1 ? e4m3x8<DT>(w[2], w[3], 1.0f) : e4m3x8<DT>(w[0], w[1], 1.0f);
#pragma unroll
          for (int q = 0; q < T; ++q)
            s[q][h][aa] = mfma16<DT>(kf, qf[q][kk], kk == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[q][h][aa]);
        }
      __builtin_amdgcn_sched_barrier(0);
    }
    stay();
    const bool more = t + KW < t1;
    if (more) {
      now = pages(t + KW, next);
      next = entries(t + 2 * KW);  // (looked at a tile later; past the table its last)
      load_k(t + KW, now);
    }
    stay();
    __builtin_amdgcn_sched_barrier(0);
    const uint32_t eb = min(max(__float_as_uint(vs) & 0x7f800000u, Range<DT>::LO), Range<DT>::HI);
    const float ve = __uint_as_float(eb);
    const float vf = vs * __uint_as_float((254u << 23) - eb);  // (vs / ve, exact)
    const float lvf = __builtin_amdgcn_logf(vf), rvf = __builtin_amdgcn_rcpf(vf);  // (log2; 0 and 1 for a power of two in range)
    u32x4 pf[T][2], rest[T][2];
#pragma unroll
    for (int q = 0; q < T; ++q) {
      if (edge) {
        const int lim = first_keys(q, none, key0);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int aa = 0; aa < 2; ++aa)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[q][h][aa][i] = 8 * h + 4 * aa + i < lim ? s[q][h][aa][i] : -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int aa = 0; aa < 2; ++aa)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[q][h][aa][i]);
      mx = __builtin_fmaf(mx, ks, lvf);
      if (__any(mx > m[q])) {
        const float mn = fmaxf(m[q], rows_max(mx));
        const float al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[q] - mn);
        m[q] = mn;
        l[q] *= al;
#pragma unroll
        for (int d = 0; d < 8; ++d) o[q][d] *= al;
      }
      const float sub = (m[q] == -INFINITY ? 0.f : m[q]) - (DT == DT_F16 ? lvf + 14.0f : lvf);
      float ls = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float p[8];
#pragma unroll
        for (int aa = 0; aa < 2; ++aa)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            p[4 * aa + i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[q][h][aa][i], ks, -sub));
            ls += p[4 * aa + i];
          }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          pf[q][h][e] = pack_p<DT>(p[2 * e], p[2 * e + 1]);
          if constexpr (T == 1) rest[q][h][e] = pack_p<DT>(p[2 * e] - lo_f32<DT>(pf[q][h][e]), p[2 * e + 1] - hi_f32<DT>(pf[q][h][e]));
        }
      }
      l[q] += ls * rvf;
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      const u32x4 v0 = e4m3x8<DT>(vw[d][0], vw[d][1], ve), v1 = e4m3x8<DT>(vw[d][2], vw[d][3], ve);
#pragma unroll
      for (int q = 0; q < T; ++q) {
        o[q][d] = mfma16<DT>(v0, pf[q][0], o[q][d]);
        o[q][d] = mfma16<DT>(v1, pf[q][1], o[q][d]);
        if constexpr (T == 1) {
          o[q][d] = mfma16<DT>(v0, rest[q][0], o[q][d]);
          o[q][d] = mfma16<DT>(v1, rest[q][1], o[q][d]);
        }
      }
      if (d & 1) __builtin_amdgcn_sched_barrier(0);
    }
    stay();
    t += KW;
    if (more) load_v(t, now);
  };

  if (t < t1) now = pages(t, a.S == 1 ? early : entries(t));
#pragma unroll
  for (int k = 0; k < T; ++k) qs[k][wave][lane] = qr[k];
  stay();
  if (t < t1) {
    load_k(t, now);
    load_v(t, now);
    next = entries(t + KW);
  }
  // the queries are in LDS for all waves; K and V stay under way
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  stay();
  while (t < t1) step();

  // the waves' parts of the keys, joined in wave order: each wave takes 32 dims of all queries
  const long long rq = (long long)a.s.rows * a.nq;
#pragma unroll
  for (int q = 0; q < T; ++q) {
    if (m0 + 16 * q >= M) break;
    l[q] = rows_sum(l[q]);
    if (__any(spoilt[q] != 0)) {
#pragma unroll
      for (int d = 0; d < 8; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (spoilt[q] >> (4 * d + i) & 1) o[q][d][i] = __uint_as_float(0x7fc00000u);
    }
#pragma unroll
    for (int d = 0; d < 8; ++d) so[wave][d][lane] = o[q][d];
    if (g == 0) {
      sm[wave][c] = m[q];
      sl[wave][c] = l[q];
    }
    __syncthreads();
    const int r = 16 * q + c;
    if (m0 + r < M) {
      float mm = -INFINITY, ll = 0.f, wgt[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sm[w][c]);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        wgt[w] = sm[w][c] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(sm[w][c] - mm);  // (without keys: zeros)
        ll += wgt[w] * sl[w][c];
      }
      const int i = row_of(r);
      const long long idx = (long long)(first + i0 + i) * a.nq + hk * G + g0 + r - i * G;
      const float inv = a.S > 1 ? 1.0f : ll == 0.f ? 0.f : 1.0f / ll;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int d = 2 * wave + k;
        f32x4 v = wgt[0] * so[0][d][lane];
#pragma unroll
        for (int w = 1; w < 4; ++w) v += wgt[w] * so[w][d][lane];
        v *= inv;
        if (a.S > 1)
          *reinterpret_cast<f32x4*>(a.part + (split * rq + idx) * HD + 16 * d + 4 * g) = v;
        else
          *reinterpret_cast<u32x2*>(a.out + idx * HD + 16 * d + 4 * g) =
              u32x2{pack_f32x2<DT>(v[0], v[1]), pack_f32x2<DT>(v[2], v[3])};
      }
      if (a.S > 1 && wave == 0 && g == 0) {
        float* pm = a.part + a.S * rq * HD + (split * rq + idx) * 2;
        pm[0] = mm;
        pm[1] = ll;
      }
    }
    if (q + 1 < T) __syncthreads();
  }
}

// The key splits of each (row, head) joined in a fixed order: one wave each, its four groups of 16 lanes taking every
// fourth split (8 dims a lane), so that the splits' loads go out together.
template <int DT>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttnP a) {
  const int lane = threadIdx.x & 63, b = blockIdx.y, g = lane >> 4, c = lane & 15;
  const RowSpan rs = seq_rows(a.s, b);
  const int item = (int)blockIdx.x * 4 + (threadIdx.x >> 6);  // row i, head
  if (item >= rs.n * a.nq) return;
  const long long rq = (long long)a.s.rows * a.nq, idx = (long long)rs.first * a.nq + item;
  const float* ml = a.part + a.S * rq * HD;
  // lane s holds split s's statistics (at most 64 splits)
  float ms = -INFINITY, ls = 0.f;
  if (lane < a.S) {
    const f32x2_t v = *reinterpret_cast<const f32x2_t*>(ml + (lane * rq + idx) * 2);
    ms = v[0];
    ls = v[1];
  }
  const float mm = wave_max(ms);
  const bool keys = ms != -INFINITY || ls != 0.f;  // (else nothing was attended, or lane >= S)
  const float wgt = ms == -INFINITY ? (keys ? 1.0f : 0.f) : __builtin_amdgcn_exp2f(ms - mm);
  const unsigned long long some = __ballot(keys);  // the splits to join, those of weight 0 too: 0 x NaN is NaN, as within a workgroup
  const float ll = wave_sum(wgt * ls);
  f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f}, y = x;
#pragma unroll 4
  for (int s0 = 0; s0 < a.S; s0 += 4) {
    const int s = s0 + g;
    const float w = __shfl(wgt, s & 63, WAVE);
    if (some >> (s & 63) & 1) {
      const f32x4* p = reinterpret_cast<const f32x4*>(a.part + (s * rq + idx) * HD + 8 * c);
      x += w * p[0];
      y += w * p[1];
    }
  }
  const float inv = ll == 0.f ? 0.f : 1.0f / ll;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = rows_sum(x[i]) * inv;
    y[i] = rows_sum(y[i]) * inv;
  }
  if (g == 0)
    *reinterpret_cast<u32x4*>(a.out + idx * HD + 8 * c) =
        u32x4{pack_f32x2<DT>(x[0], x[1]), pack_f32x2<DT>(x[2], x[3]), pack_f32x2<DT>(y[0], y[1]), pack_f32x2<DT>(y[2], y[3])};
}

template <int DT, int PAGE>
hipError_t launch_append_page(const PagedAppendP& a, hipStream_t st) {
  const dim3 grid((unsigned)append_wgs(a.s.nseq, a.s.max_rows, PAGE), a.c.nkv + (a.q ? (a.nq + QH - 1) / QH : 0));
  auto launch = [&](auto kernel, int threads) { hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, st, a); };
  if (PAGE > 32 && a.s.max_rows <= 32) launch(paged_append_kernel<DT, PAGE, PAGE < 32 ? PAGE : 32>, 256);
  else launch(paged_append_kernel<DT, PAGE, PAGE>, 8 * PAGE);
  return hipGetLastError();
}
template <int DT>
hipError_t launch_append_dt(const PagedAppendP& a, hipStream_t st) {
  switch (a.c.page) {
    case 16: return launch_append_page<DT, 16>(a, st);
    case 32: return launch_append_page<DT, 32>(a, st);
    case 64: return launch_append_page<DT, 64>(a, st);
    case 128: return launch_append_page<DT, 128>(a, st);
  }
  return hipErrorInvalidValue;
}

long long attn_wgs(const PagedAttnP& a) {
  return ((long long)a.S * a.c.nkv * a.s.nseq * a.cuts + 7) / 8 * 8 * a.group_wgs;
}
template <int DT>
hipError_t launch_attn_dt(const PagedAttnP& a, hipStream_t st) {
  const dim3 grid((unsigned)attn_wgs(a));
  if (a.tiles16 == 1) hipLaunchKernelGGL((paged_attn_kernel<DT, 1>), grid, dim3(64 * KW), 0, st, a);
  else hipLaunchKernelGGL((paged_attn_kernel<DT, 2>), grid, dim3(64 * KW), 0, st, a);
  if (const hipError_t e = hipGetLastError(); e != hipSuccess || a.S == 1) return e;
  hipLaunchKernelGGL(paged_merge_kernel<DT>, dim3((a.s.max_rows * a.nq + 3) / 4, a.s.nseq), dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_append(int dt, const PagedAppendP& a, hipStream_t st) {
  return dt == DT_BF16 ? launch_append_dt<DT_BF16>(a, st) : launch_append_dt<DT_F16>(a, st);
}

// Tiles of 16 flattened rows that a workgroup takes: one where a kv head has no more, else two, which share the conversion
// of K and V (us, one / two tiles: 16 sequences of 32 rows 13.9 / 13.5, one of 32 rows over 32768 keys 28.0 / 25.3, 2048
// rows over 8192 keys 196 / 124).  Three or four would leave one wave a SIMD (184 and 220 at the last, at an earlier step).
// Key splits: as many as leave the workgroups within one to a compute unit, of two tiles, or two to one, of one tile (a token
// of many sequences waits on memory more than it computes) and where a wave would have more than 20 tiles of keys
// otherwise; none below a tile of keys for each wave.  us, one / two to a compute unit, of two tiles: 16 sequences of 32
// rows over up to 1055 keys 13.5 / 19.3 (no second launch to join them), over 4096 32.3 / 33.1, over 8192 57.6 / 52.5, over
// 32768 206 / 177; one of 32 rows over 32768 keys 25.3 / 27.6, four 52.8 / 47.1; of one tile: one row of 64 sequences over
// 1024 to 8192 keys 39.3 / 37.4.  Up to three tiles (five, where workgroups have one) for each wave are not split: joining
// costs a launch.  us, split / whole: a row over 256 keys 10.2 / 6.9, over 1024 11.5 / 9.6, over 2080 11.3 / 15.0, of 64
// sequences over 1024 13.4 / 10.6; four sequences of 32 rows over 512 keys 11.8 / 10.7, eight rows over 1024 11.0 / 12.0.
bool paged_attn_plan(PagedAttnP& a, int cus) {
  const long long M = (long long)a.s.max_rows * (a.nq / a.c.nkv), pairs = (long long)a.c.nkv * a.s.nseq;
  a.tiles16 = M <= 16 ? 1 : 2;
  const long long rows = 16 * a.tiles16, wide = (M + rows - 1) / rows, tiles = ((long long)a.max_len + 63) / 64;
  const long long wgs = wide * pairs;
  long long S = 1;
  if (tiles > (a.tiles16 == 1 ? 5 : 3) * KW) {
    S = std::max(1ll, cus / wgs);
    if (a.tiles16 == 1 || tiles > 20 * KW * S) S = 2ll * cus / wgs;
    S = std::max(1ll, std::min({S, (tiles + KW - 1) / KW, 64ll}));
  }
  // ranges in whole rounds of the eight XCDs, where their workgroups follow each other there (without: 32 rows over
  // 32768 keys 30.6 instead of 25.4)
  while (wide > 1 && S > 8 && S * pairs % 8 != 0) --S;
  a.S = (int)S;
  const long long ranges = S * pairs;
  a.cuts = (int)std::min(ranges >= 8 ? 1ll : (8 + ranges - 1) / ranges, wide);
  a.group_wgs = (int)((wide + a.cuts - 1) / a.cuts);
  return grid_fits(attn_wgs(a), 64 * KW) && grid_fits(((long long)a.s.max_rows * a.nq + 3) / 4, 256);
}
size_t paged_attn_floats(const PagedAttnP& a) {
  return a.S > 1 ? (size_t)a.S * a.s.rows * a.nq * (HD + 2) : 0;
}
hipError_t launch_paged_attn(int dt, const PagedAttnP& a, hipStream_t st) {
  return dt == DT_BF16 ? launch_attn_dt<DT_BF16>(a, st) : launch_attn_dt<DT_F16>(a, st);
}

}  // namespace fdllm
