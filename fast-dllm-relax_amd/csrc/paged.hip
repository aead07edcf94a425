// The paged 8-bit cache: appending rotated keys and values, and attention over it.
#include <algorithm>

#include "common.hpp"
#include "paged.hpp"
#include "paged_index.hpp"

namespace fdllm {

namespace {

constexpr int HD = 128;

__device__ __forceinline__ RowSpan seq_rows(const SeqRowsP& s, int b) {
  return seq_span(s.row_start, s.rows, s.max_rows, b);
}
__device__ __forceinline__ int page_of(const PagedP& c, int b, long long j) {
  return page_at(c.table + b * c.table_ld, c.table_w, c.num_pages, j);
}

// ---- append ------------------------------------------------------------------------------------
// Rotation by position: pair (i, i + 64) turns by pos theta^(-i/64) radians.  The angle is reduced in 64 bits (in
// turns: its whole part is dropped), so far positions keep their angle; sine and cosine are fp32 and not rounded
// to the model dtype.  A thread takes the 8 pairs of unit u (pairs 8 u .. 8 u + 7).
__device__ __forceinline__ void unit_turns(const PagedAppendP& a, int u, double (&f)[8]) {
  double t = 0.15915494309189533577;  // 1 / (2 pi)
  t *= (u & 1) ? a.turn8 : 1.0;
  t *= (u & 2) ? a.turn16 : 1.0;
  t *= (u & 4) ? a.turn32 : 1.0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    f[e] = t;
    t *= a.turn1;
  }
}
__device__ __forceinline__ void unit_sincos(const double (&f)[8], long long pos, float (&sn)[8], float (&cs)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const double t = (double)pos * f[e];
    sincospif(2.0f * (float)(t - __builtin_rint(t)), &sn[e], &cs[e]);
  }
}
template <int DT>
__device__ __forceinline__ void unpack8(u32x4 w, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = lo_f32<DT>(w[e]);
    x[2 * e + 1] = hi_f32<DT>(w[e]);
  }
}
__device__ __forceinline__ void rotate8(float (&lo)[8], float (&hi)[8], const float (&sn)[8], const float (&cs)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float x = lo[e], y = hi[e];
    lo[e] = x * cs[e] - y * sn[e];
    hi[e] = y * cs[e] + x * sn[e];
  }
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
constexpr int QH = 4;
template <int DT, int PAGE>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendP a) {
  constexpr int KU = (PAGE * 8 + 255) / 256;    // (slot, pair unit) items per thread
  constexpr int VU = (PAGE * 16 + 255) / 256;   // (slot, 8 dims) items per thread
  constexpr int VP = (HD * PAGE / 16 + 255) / 256;  // 16-byte pieces of V's page per thread
  constexpr int LDV = PAGE + 4;                 // bytes from dim to dim in LDS
  __shared__ float red[2][4];
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
  const int u = tid & 7;
  double f[8];

  if ((int)blockIdx.y >= a.c.nkv) {
    // queries: rotated, rounded once to the model dtype
    const int h0 = ((int)blockIdx.y - a.c.nkv) * QH;
    unit_turns(a, u, f);
    for (int s = w0 + (tid >> 3); s < w1; s += 32) {
      float sn[8], cs[8];
      unit_sincos(f, pos0 + s, sn, cs);
      const uint16_t* src = a.q + (row0 + s) * a.ldq;
      uint16_t* dst = a.q_out + (row0 + s) * a.nq * HD;
#pragma unroll
      for (int h = 0; h < QH; ++h) {
        if (h0 + h >= a.nq) break;
        const int o = (h0 + h) * HD + 8 * u;
        float lo[8], hi[8];
        unpack8<DT>(*reinterpret_cast<const u32x4*>(src + o), lo);
        unpack8<DT>(*reinterpret_cast<const u32x4*>(src + o + 64), hi);
        rotate8(lo, hi, sn, cs);
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

  float klo[KU][8], khi[KU][8], vv[VU][8];
#pragma unroll
  for (int i = 0; i < KU; ++i) {
    const int s = (tid >> 3) + 32 * i;
    if (s >= w0 && s < w1) {
      const uint16_t* src = a.k + (row0 + s) * a.ldk + h * HD + 8 * u;
      unpack8<DT>(*reinterpret_cast<const u32x4*>(src), klo[i]);
      unpack8<DT>(*reinterpret_cast<const u32x4*>(src + 64), khi[i]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) klo[i][e] = khi[i][e] = 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < VU; ++i) {
    const int s = (tid >> 4) + 16 * i;
    if (s >= w0 && s < w1) {
      unpack8<DT>(*reinterpret_cast<const u32x4*>(a.v + (row0 + s) * a.ldv + h * HD + 8 * (tid & 15)), vv[i]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) vv[i][e] = 0.f;
    }
  }
  // V's pieces that hold other rows too
  u32x4 held[VP];
#pragma unroll
  for (int i = 0; i < VP; ++i) {
    const int p = tid + 256 * i;  // piece: dim p / (PAGE / 16), slots 16 (p % (PAGE / 16)) .. + 15
    const int s0 = 16 * (p % (PAGE / 16));
    held[i] = u32x4{0, 0, 0, 0};
    if (p < HD * PAGE / 16 && (keeps || (s0 < w1 && s0 + 16 > w0 && (s0 < w0 || s0 + 16 > w1))))
      held[i] = *reinterpret_cast<const u32x4*>(vp + 16 * (size_t)p);
  }
  unit_turns(a, u, f);
  float ka = 0.f, va = 0.f;
#pragma unroll
  for (int i = 0; i < KU; ++i) {
    const int s = (tid >> 3) + 32 * i;
    float sn[8], cs[8];
    unit_sincos(f, pos0 + s, sn, cs);
    rotate8(klo[i], khi[i], sn, cs);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (s < w0 || s >= w1) klo[i][e] = khi[i][e] = 0.f;
      ka = fmaxf(ka, finite(klo[i][e]) ? fabsf(klo[i][e]) : 0.f);
      ka = fmaxf(ka, finite(khi[i][e]) ? fabsf(khi[i][e]) : 0.f);
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
  ka = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  va = fmaxf(fmaxf(red[1][0], red[1][1]), fmaxf(red[1][2], red[1][3]));
  float ks = pow2_scale(ka), vs = pow2_scale(va);
  if (keeps) {
    ks = fmaxf(ks, ks_old);
    vs = fmaxf(vs, vs_old);
  }
  const float ki = 1.0f / ks, vi = 1.0f / vs;
#pragma unroll
  for (int i = 0; i < KU; ++i) {
    const int s = (tid >> 3) + 32 * i;
    if (s < w0 || s >= w1) continue;
    const auto& x = klo[i];
    const auto& y = khi[i];
    uint8_t* dst = kp + s * HD + 8 * u;
    *reinterpret_cast<u32x2*>(dst) = u32x2{to_e4m3(x[0] * ki, x[1] * ki, x[2] * ki, x[3] * ki),
                                           to_e4m3(x[4] * ki, x[5] * ki, x[6] * ki, x[7] * ki)};
    *reinterpret_cast<u32x2*>(dst + 64) = u32x2{to_e4m3(y[0] * ki, y[1] * ki, y[2] * ki, y[3] * ki),
                                                to_e4m3(y[4] * ki, y[5] * ki, y[6] * ki, y[7] * ki)};
  }
  if (keeps && ks > ks_old) {
    const float r = ks_old / ks;
    for (int p = tid; p < PAGE * HD / 16; p += 256) {
      const int s = p >> 3;
      if (s >= lv || (s >= w0 && s < w1)) continue;
      u32x4 w = *reinterpret_cast<const u32x4*>(kp + 16 * p);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = rescale4(w[e], r);
      *reinterpret_cast<u32x4*>(kp + 16 * p) = w;
    }
  }
  // V: bytes of (slot, 8 dims) items into their dims' rows
#pragma unroll
  for (int i = 0; i < VU; ++i) {
    const int s = (tid >> 4) + 16 * i;
    if (s < w0 || s >= w1) continue;
    const auto& x = vv[i];
    const uint32_t lo = to_e4m3(x[0] * vi, x[1] * vi, x[2] * vi, x[3] * vi);
    const uint32_t hi = to_e4m3(x[4] * vi, x[5] * vi, x[6] * vi, x[7] * vi);
    uint8_t* t = vt + 8 * (tid & 15) * LDV + s;
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
  for (int i = 0; i < VP; ++i) {
    const int p = tid + 256 * i;
    if (p >= HD * PAGE / 16) break;
    const int d = p / (PAGE / 16), s0 = 16 * (p % (PAGE / 16));
    const bool touched = s0 < w1 && s0 + 16 > w0;
    if (!touched && !(grow && s0 < lv)) continue;
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t fresh = *reinterpret_cast<const uint32_t*>(vt + d * LDV + s0 + 4 * e);
      uint32_t old = held[i][e], moved = old;
      if (grow) moved = rescale4(old, r);
      uint32_t out = 0;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int s = s0 + 4 * e + t;
        const uint32_t m = 0xffu << (8 * t);
        out |= m & (s >= w0 && s < w1 ? fresh : s < lv ? moved : old);
      }
      w[e] = out;
    }
    *reinterpret_cast<u32x4*>(vp + 16 * (size_t)p) = w;
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
//   into V's conversion, which takes one, f into the exponent of p.
// The running maximum is that of the query's whole row, held in each of its four lanes; the sum is each lane's own part
// until the end.
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
// whether any byte of w is e4m3's NaN (0x7f or 0xff)
__device__ __forceinline__ bool has_nan(u32x4 w) {
  uint32_t any = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    // bytes 0x7f after the sign is dropped carry into bit 7 by + 1, others do not
    any |= ((w[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
  }
  return any != 0;
}


template <int DT, int KW>
__global__ __launch_bounds__(64 * KW) void paged_attn_kernel(PagedAttnP a) {
  __shared__ float sm[KW][16], sl[KW][16];
  __shared__ __align__(16) float so[KW][16][HD + 4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = lane & 15, g = lane >> 4;
  const int b = blockIdx.z, hk = (int)blockIdx.y / a.S, split = (int)blockIdx.y % a.S;
  const int G = a.nq / a.c.nkv;
  const RowSpan rs = seq_rows(a.s, b);
  const int first = rs.first, n = rs.n;
  const int m0 = 16 * (int)blockIdx.x;  // first flattened row of this tile
  if (m0 >= n * G) return;
  const int lk = min(max(a.kv_len[b], 0), a.c.table_w * a.c.page);
  // this lane's query
  const int mr = m0 + c, qi = mr / G, qh = hk * G + mr % G;
  const bool row_ok = mr < n * G;
  int klim = key_limit(a.kv_len[b], lk, n, qi, a.mask_block);  // keys [0, klim) are attended
  int kmax = row_ok ? klim : 0;
#pragma unroll
  for (int k = 8; k >= 1; k >>= 1) kmax = max(kmax, __shfl_xor(kmax, k, WAVE));
  kmax = __builtin_amdgcn_readfirstlane(kmax);
  if (!row_ok) klim = kmax;  // (a column without a query asks for no mask of its own)

  // queries: dims 64 jj + 16 g + 8 h + 0..7 of this lane's query are k step (jj, h)
  u32x4 qf[2][2];
#pragma unroll
  for (int jj = 0; jj < 2; ++jj)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      qf[jj][h] = row_ok ? *reinterpret_cast<const u32x4*>(a.q + (long long)(first + qi) * a.ldq + qh * HD + 64 * jj + 16 * g + 8 * h)
                         : u32x4{0, 0, 0, 0};

  const int tiles = (kmax + 63) / 64, per = (tiles + a.S - 1) / a.S;
  const int t1 = min(tiles, (split + 1) * per);
  float m = -INFINITY, l = 0.f;
  f32x4 o[8];
#pragma unroll
  for (int d = 0; d < 8; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int page = a.c.page, shift = a.c.shift;
  const size_t pstride = (size_t)page * HD;

  for (int t = split * per + wave; t < t1; t += KW) {
    // this lane's 16 keys (scores, V) and the 16 keys its K rows come from
    const int key0 = 64 * t + 16 * g, kc0 = 64 * t + 16 * (c >> 2);
    const int pv = key0 < lk ? page_of(a.c, b, key0 >> shift) : -1;
    const int pk = kc0 < lk ? page_of(a.c, b, kc0 >> shift) : -1;
    const size_t ov = (size_t)max(pv, 0) * a.c.nkv + hk, ok = (size_t)max(pk, 0) * a.c.nkv + hk;
    const uint8_t* kp = a.c.k + ok * pstride + (size_t)((kc0 & (page - 1)) + (c & 3)) * HD + 16 * g;
    const uint8_t* vp = a.c.v + ov * pstride + (size_t)c * page + (key0 & (page - 1));
    u32x4 kw[2][2][2], vw[8];  // K [h][a][jj]
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int aa = 0; aa < 2; ++aa)
#pragma unroll
        for (int jj = 0; jj < 2; ++jj)
          kw[h][aa][jj] = *reinterpret_cast<const u32x4*>(kp + (8 * h + 4 * aa) * HD + 64 * jj);
#pragma unroll
    for (int d = 0; d < 8; ++d) vw[d] = *reinterpret_cast<const u32x4*>(vp + (size_t)16 * d * page);
    const float ks = (pv < 0 ? 1.0f : fmaxf(a.c.ks[ov], 0x1p-100f)) * a.scale_log2e;
    const float vs = pv < 0 ? 1.0f : fmaxf(a.c.vs[ov], 0x1p-100f);
    f32x4 s[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int aa = 0; aa < 2; ++aa) {
        f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int jj = 0; jj < 2; ++jj) {
          const u32x4 w = kw[h][aa][jj];
          acc = mfma16<DT>(e4m3x8<DT>(w[0], w[1], 1.0f), qf[jj][0], acc);
          acc = mfma16<DT>(e4m3x8<DT>(w[2], w[3], 1.0f), qf[jj][1], acc);
        }
        s[h][aa] = acc;
      }
    // keys past this query's limit, and pages that are none
    const bool edge = __any(64 * t + 64 > klim || pv < 0);
    const int lim = pv < 0 ? 0 : klim - key0;  // of this lane's 16 keys, the first lim are attended
    if (edge) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int aa = 0; aa < 2; ++aa)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[h][aa][i] = 8 * h + 4 * aa + i < lim ? s[h][aa][i] : -INFINITY;
      // what lies behind the sequence's end or in no page is nothing, NaN among it
#pragma unroll
      for (int d = 0; d < 8; ++d) vw[d] = first_bytes16(vw[d], pv < 0 ? 0 : lk - key0);
    }
    float mx = -INFINITY;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int aa = 0; aa < 2; ++aa)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[h][aa][i]);
    mx *= ks;
    if (__any(mx > m)) {
      const float mn = fmaxf(m, rows_max(mx));
      const float al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= al;
#pragma unroll
      for (int d = 0; d < 8; ++d) o[d] *= al;
    }
    const float mref = m == -INFINITY ? 0.f : m;
    const float ve = __uint_as_float(__float_as_uint(vs) & 0x7f800000u);
    const float vf = __uint_as_float((__float_as_uint(vs) & 0x007fffffu) | 0x3f800000u);
    const float sub = mref - __builtin_amdgcn_logf(vf);  // (log2; 0 for a power of two)
    float ls = 0.f;
    u32x4 pf[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float p[8];
#pragma unroll
      for (int aa = 0; aa < 2; ++aa)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[4 * aa + i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][aa][i], ks, -sub));
          ls += p[4 * aa + i];
        }
#pragma unroll
      for (int e = 0; e < 4; ++e) pf[h][e] = pack_f32x2<DT>(p[2 * e], p[2 * e + 1]);
    }
    l += ls * __builtin_amdgcn_rcpf(vf);
    // a masked probability is 0, and 0 x NaN is not: where a key that some query of the tile does not attend holds
    // NaN, each group of queries with the same limit takes its product with the keys behind that limit cleared
    bool nan = false;
    if (edge) {
#pragma unroll
      for (int d = 0; d < 8; ++d) nan |= has_nan(vw[d]);
    }
    if (edge && __any(nan)) {
      f32x4 keep[8];
#pragma unroll
      for (int d = 0; d < 8; ++d) keep[d] = o[d];
      for (int q = 0; q < 16; ++q) {
        const int kl = __builtin_amdgcn_readlane(klim, q);
        if (q > 0 && kl == __builtin_amdgcn_readlane(klim, q - 1)) continue;
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          const u32x4 w = first_bytes16(vw[d], kl - key0);
          f32x4 acc = keep[d];
          acc = mfma16<DT>(e4m3x8<DT>(w[0], w[1], ve), pf[0], acc);
          acc = mfma16<DT>(e4m3x8<DT>(w[2], w[3], ve), pf[1], acc);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[d][i] = klim == kl ? acc[i] : o[d][i];
        }
      }
    } else {
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        o[d] = mfma16<DT>(e4m3x8<DT>(vw[d][0], vw[d][1], ve), pf[0], o[d]);
        o[d] = mfma16<DT>(e4m3x8<DT>(vw[d][2], vw[d][3], ve), pf[1], o[d]);
      }
    }
  }
  l = rows_sum(l);
  // the waves' parts of the keys, joined in wave order
  if (g == 0) {
    sm[wave][c] = m;
    sl[wave][c] = l;
  }
#pragma unroll
  for (int d = 0; d < 8; ++d) *reinterpret_cast<f32x4*>(&so[wave][c][16 * d + 4 * g]) = o[d];
  __syncthreads();
  constexpr int TPQ = 4 * KW;  // threads per query
  const int qc = threadIdx.x / TPQ, dim0 = (threadIdx.x % TPQ) * (HD / TPQ);
  const int omr = m0 + qc;
  if (omr >= n * G) return;
  float mm = -INFINITY, ll = 0.f;
#pragma unroll
  for (int w = 0; w < KW; ++w) mm = fmaxf(mm, sm[w][qc]);
  float wgt[KW];
#pragma unroll
  for (int w = 0; w < KW; ++w) {
    wgt[w] = sm[w][qc] == -INFINITY && !(sl[w][qc] != sl[w][qc]) ? 0.f : __builtin_amdgcn_exp2f(sm[w][qc] - mm);
    ll += wgt[w] * sl[w][qc];
  }
  const long long idx = (long long)(first + omr / G) * a.nq + hk * G + omr % G;
  const float inv = a.S > 1 ? 1.0f : ll == 0.f ? 0.f : 1.0f / ll;
  float v[HD / TPQ];
#pragma unroll
  for (int i = 0; i < HD / TPQ; ++i) {
    v[i] = 0.f;
#pragma unroll
    for (int w = 0; w < KW; ++w)
      if (wgt[w] != 0.f) v[i] += wgt[w] * so[w][qc][dim0 + i];
    v[i] *= inv;
  }
  if (a.S > 1) {
    const long long rq = (long long)a.s.rows * a.nq;
    float* po = a.part + (split * rq + idx) * HD + dim0;
#pragma unroll
    for (int i = 0; i < HD / TPQ; i += 4) *reinterpret_cast<f32x4*>(po + i) = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
    if (dim0 == 0) {
      float* pm = a.part + a.S * rq * HD + (split * rq + idx) * 2;
      pm[0] = mm;
      pm[1] = ll;
    }
  } else {
    uint16_t* po = a.out + idx * HD + dim0;
#pragma unroll
    for (int i = 0; i < HD / TPQ; i += 8)
      *reinterpret_cast<u32x4*>(po + i) =
          u32x4{pack_f32x2<DT>(v[i], v[i + 1]), pack_f32x2<DT>(v[i + 2], v[i + 3]), pack_f32x2<DT>(v[i + 4], v[i + 5]),
                pack_f32x2<DT>(v[i + 6], v[i + 7])};
  }
}

// the key splits of each (row, head), one wave each, joined in split order
template <int DT>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttnP a) {
  const int lane = threadIdx.x & 63, b = blockIdx.y;
  const RowSpan rs = seq_rows(a.s, b);
  const int first = rs.first, n = rs.n;
  const int item = (int)blockIdx.x * 4 + (threadIdx.x >> 6);  // row i, head
  if (item >= n * a.nq) return;
  const long long rq = (long long)a.s.rows * a.nq, idx = (long long)first * a.nq + item;
  const float* ml = a.part + a.S * rq * HD;
  float mm = -INFINITY;
  for (int s = 0; s < a.S; ++s) mm = fmaxf(mm, ml[(s * rq + idx) * 2]);
  float ll = 0.f, x = 0.f, y = 0.f;
  for (int s = 0; s < a.S; ++s) {
    const float ms = ml[(s * rq + idx) * 2], ls = ml[(s * rq + idx) * 2 + 1];
    if (ls == 0.f) continue;  // (a split without keys; NaN is not 0)
    const float w = ms == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ms - mm);
    const f32x2_t v = *reinterpret_cast<const f32x2_t*>(a.part + (s * rq + idx) * HD + 2 * lane);
    ll += w * ls;
    x += w * v[0];
    y += w * v[1];
  }
  const float inv = ll == 0.f ? 0.f : 1.0f / ll;
  reinterpret_cast<uint32_t*>(a.out + idx * HD)[lane] = pack_f32x2<DT>(x * inv, y * inv);
}

constexpr int ATTN_KW = 4;

template <int DT>
hipError_t launch_append_dt(const PagedAppendP& a, hipStream_t st) {
  const int page = a.c.page, npp = (int)pages_touched(a.s.max_rows, page);
  const dim3 grid((unsigned)(a.s.nseq * npp), a.c.nkv + (a.q ? (a.nq + QH - 1) / QH : 0));
  switch (page) {
    case 16: hipLaunchKernelGGL((paged_append_kernel<DT, 16>), grid, dim3(256), 0, st, a); break;
    case 32: hipLaunchKernelGGL((paged_append_kernel<DT, 32>), grid, dim3(256), 0, st, a); break;
    case 64: hipLaunchKernelGGL((paged_append_kernel<DT, 64>), grid, dim3(256), 0, st, a); break;
    case 128: hipLaunchKernelGGL((paged_append_kernel<DT, 128>), grid, dim3(256), 0, st, a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

template <int DT>
hipError_t launch_attn_dt(const PagedAttnP& a, hipStream_t st) {
  const int G = a.nq / a.c.nkv;
  const dim3 grid((a.s.max_rows * G + 15) / 16, a.c.nkv * a.S, a.s.nseq);
  hipLaunchKernelGGL((paged_attn_kernel<DT, ATTN_KW>), grid, dim3(64 * ATTN_KW), 0, st, a);
  if (const hipError_t e = hipGetLastError(); e != hipSuccess || a.S == 1) return e;
  hipLaunchKernelGGL(paged_merge_kernel<DT>, dim3((a.s.max_rows * a.nq + 3) / 4, a.s.nseq), dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_append(int dt, const PagedAppendP& a, hipStream_t st) {
  return dt == DT_BF16 ? launch_append_dt<DT_BF16>(a, st) : launch_append_dt<DT_F16>(a, st);
}

int paged_attn_splits(const PagedAttnP& a, int cus) {
  const int G = a.nq / a.c.nkv;
  const long long wgs = (long long)((a.s.max_rows * G + 15) / 16) * a.c.nkv * a.s.nseq;
  const int tiles = (a.max_len + 63) / 64;
  return (int)std::max(1ll, std::min({(2ll * cus + wgs - 1) / wgs, (long long)(tiles + ATTN_KW - 1) / ATTN_KW, 64ll}));
}
size_t paged_attn_floats(const PagedAttnP& a) {
  return a.S > 1 ? (size_t)a.S * a.s.rows * a.nq * (HD + 2) : 0;
}
hipError_t launch_paged_attn(int dt, const PagedAttnP& a, hipStream_t st) {
  return dt == DT_BF16 ? launch_attn_dt<DT_BF16>(a, st) : launch_attn_dt<DT_F16>(a, st);
}

}  // namespace fdllm
