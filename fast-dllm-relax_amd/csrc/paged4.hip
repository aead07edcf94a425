// The paged 4-bit cache: appending normed and rotated keys and values, reading rows back, and attention over it.
#include <algorithm>

#include "common.hpp"
#include "paged4.hpp"
#include "rotate_device.hpp"

namespace fdllm {

namespace {

constexpr int ROW = HD / 2;  // bytes of a row's codes

// bytes of a slot's scale of block 0 in its page's; blocks are 4 apart
__device__ __forceinline__ int key_scale_at(int slot) { return (slot >> 4) * 64 + (slot & 3) * 16 + (slot >> 2 & 3); }

// the row's place in a page of its sequence: -1 where there is none
struct Place { int page, slot; };
__device__ __forceinline__ Place place_of(const Paged4P& c, int b, long long pos) {
  return Place{pos < 0 ? -1 : page_of(c, b, pos >> c.shift), (int)pos & (c.page - 1)};
}

// Row r of the call as row i of sequence b; b < 0: of none.  A wave takes 8 rows in turn, a lane's the (lane / 8)-th from
// row0; all its lanes come here.  A launch so has workgroups for the call's rows and none for the rows that a ragged batch's
// sequences do not have (24 sequences of up to 509 rows, us, by sequence / by row: 15.0 / 11.6).
struct CallRow { int b, i; };
__device__ __forceinline__ CallRow call_row(const SeqRowsP& s, int row0) {
  const int lane = threadIdx.x & 63, row = row0 + (lane >> 3);
  if (s.row_start == nullptr) {
    const int b = (int)((unsigned)row / (unsigned)s.max_rows);
    return CallRow{row < s.rows && b < s.nseq ? b : -1, row - b * s.max_rows};
  }
  int b = -1;
  // row starts by 64, each of the eight rows counting those that do not lie behind it; of many sequences by halving, seven or more
  // loads that wait for each other (us, appends of one row a sequence, counted / halved: 24 sequences 4.45 / 4.61, 64 4.73 / 4.81,
  // 128 5.03 / 4.98, 256 5.54 / 5.12, 1000 8.13 / 5.57)
  if (s.nseq < 128) {
    for (int k0 = 0; k0 <= s.nseq; k0 += 64) {
      const int v = k0 + lane <= s.nseq ? s.row_start[k0 + lane] : 0x7fffffff;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int n = __builtin_popcountll(__ballot(v <= row0 + k));
        b += (lane >> 3) == k ? n : 0;
      }
    }
  } else {
    b = seq_of_row(s.row_start, s.nseq, row);
  }
  if (row >= s.rows || b < 0 || b >= s.nseq) return CallRow{-1, 0};
  const RowSpan rs = seq_span(s.row_start + b, s.rows, s.max_rows, 0);
  return row >= rs.first && row < rs.first + rs.n ? CallRow{b, row - rs.first} : CallRow{-1, 0};
}

// ---- append ------------------------------------------------------------------------------------
// e2m1 holds 0, .5, 1, 1.5, 2, 3, 4 and 6 with a sign.  Keys: the least power of two s, 2^-60 <= s <= 2^125, with
// |x| <= 7 s for the block's 32 values (up to 7, half way to what would follow, 6 is the nearest).  Values: a sixth of the
// row's largest, rounded to bf16, at least 2^-60.
__device__ __forceinline__ int key_exponent(float amax) {  // + 127
  if (!(amax > 0.f)) return 127 - 60;
  int e;
  const float m = frexpf(amax, &e);  // 7 = 0.875 x 2^3
  return 127 + min(max(e - 3 + (m > 0.875f ? 1 : 0), -60), 125);
}
// x as fp32 that compares as x does with any value of 19 bits (borders between codes and scales among them): cut off after 20
// bits, the last one set where something was cut
__device__ __forceinline__ float to_f32_odd(double x) {
  const auto b = (unsigned long long)__double_as_longlong(x);
  return (float)__longlong_as_double((long long)((b >> 32 | ((uint32_t)b != 0 ? 1u : 0u)) << 32));
}
// 8 values as codes, nearest, ties to even, at most 6 (the conversion saturates)
__device__ __forceinline__ uint32_t to_e2m1x8(const float* x) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], 1.0f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], 1.0f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], 1.0f, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], 1.0f, 3);
  return w;
}
template <int N>
__device__ __forceinline__ float largest(const float* x) {  // NaN where one is not finite
  float m = 0.f;
  bool ok = true;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    m = fmaxf(m, fabsf(x[e]));
    ok = ok && finite(x[e]);
  }
  return ok ? m : __uint_as_float(0x7fc00000u);
}
// the larger, NaN where one is
__device__ __forceinline__ float larger(float a, float b) { return a != a || b != b ? __uint_as_float(0x7fc00000u) : fmaxf(a, b); }

// A workgroup, a wave, takes eight rows of the call, eight threads a row: the queries of QH heads, the keys of KH
// or the values of KH (blockIdx.y in that order).  Two neighbouring threads hold a block of 32 dims and eight a row, so its
// largest value is three lane exchanges away; rows share nothing, so a wave is a workgroup.  Bound by memory and the chain of
// dependent loads before it (row starts, lengths, table): 8192 rows of 12 + 2 heads 15.6 us, 3.9 TB/s; a ragged batch of 6131
// 12.0 us; a token 4.1 us.  Rows requested before their sequence is known delay the chain: 11.9 / 13.3 us ragged.
constexpr int KLD = HD + 4;  // floats from row to row in LDS
template <int DT, bool INTER, int QH, int KH>
__global__ __launch_bounds__(64) void paged4_append_kernel(Paged4AppendP a) {
  __shared__ __align__(16) float rows_lds[8 * KLD];
  const int u = threadIdx.x & 7, r = threadIdx.x >> 3, row0 = 8 * (int)blockIdx.x;
  const CallRow cr = call_row(a.s, row0);
  if (cr.b < 0) return;  // (the eight threads of a row together)
  const int b = cr.b, i = cr.i, start = a.start[b];
  if (start < 0) return;
  const long long row = row0 + r;
  const int qg = a.q ? (a.nq + QH - 1) / QH : 0, kg = (a.c.nkv + KH - 1) / KH, y = (int)blockIdx.y;

  const double pos = (double)((a.pos ? a.pos[b] : start) + (long long)i);
  if (y < qg) {
    turn_heads<DT, INTER, QH>(a.t, u, pos, a.q + row * a.ldq, a.q_norm, a.q_out + row * a.nq * HD, QH * y, a.nq);
    return;
  }
  if (y < qg + kg) {
    const HeadPart p = head_part(a.t, u);
    // keys: turned and encoded from 64 bits, so that their codes are those of the definition but where it lies within 2^-30 of
    // the pair's size of a tie (sines are within 2^-33)
    const int h0 = (y - qg) * KH;
    const Place at = place_of(a.c, b, (long long)start + i);
    double x[KH][16];
    float w[16];
#pragma unroll
    for (int h = 0; h < KH; ++h)
      if (h0 + h < a.c.nkv) load_part<DT>(a.k + row * a.ldk + (h0 + h) * HD, p, x[h]);
    if (a.k_norm) {
      load_part<DT>(a.k_norm, p, w);
#pragma unroll
      for (int h = 0; h < KH; ++h)
        if (h0 + h < a.c.nkv) norm_part(x[h], w, a.t.eps);
    }
    if (p.turned) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        double sn, cs;
        turn_sincos(pos * a.t.turn[8 * u + e], sn, cs);
        sn *= a.t.gain;
        cs *= a.t.gain;
#pragma unroll
        for (int h = 0; h < KH; ++h) turn_pair<INTER>(x[h], e, sn, cs);
      }
    }
    if (at.page < 0) return;
    float* mine = rows_lds + r * KLD;  // the row's dims in order: 16 neighbouring ones for each thread, two to a block
#pragma unroll
    for (int h = 0; h < KH; ++h) {
      if (h0 + h >= a.c.nkv) break;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        *reinterpret_cast<f32x4*>(mine + (e < 2 ? p.lo + 4 * e : p.hi + 4 * (e - 2))) =
            f32x4{to_f32_odd(x[h][4 * e]), to_f32_odd(x[h][4 * e + 1]), to_f32_odd(x[h][4 * e + 2]), to_f32_odd(x[h][4 * e + 3])};
      }
      __builtin_amdgcn_wave_barrier();  // (a row is one wave's, whose LDS accesses stay in order)
      asm volatile("" ::: "memory");
      float v[16];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f32x4 f = *reinterpret_cast<const f32x4*>(mine + 16 * u + 4 * e);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[4 * e + k] = f[k];
      }
      asm volatile("" ::: "memory");
      __builtin_amdgcn_wave_barrier();
      float m = largest<16>(v);
      m = larger(m, other_lane<DPP_XOR1>(m));
      const int e = m != m ? 255 : key_exponent(m);
      const float inv = __uint_as_float((uint32_t)(e == 255 ? 127 : 254 - e) << 23);
#pragma unroll
      for (int k = 0; k < 16; ++k) v[k] *= inv;
      const size_t ph = (size_t)at.page * a.c.nkv + h0 + h;
      *reinterpret_cast<u32x2*>(a.c.k + (ph * a.c.page + at.slot) * ROW + 8 * u) = u32x2{to_e2m1x8(v), to_e2m1x8(v + 8)};
      if ((u & 1) == 0) a.c.ks[ph * a.c.page * 4 + key_scale_at(at.slot) + 4 * (u >> 1)] = (uint8_t)e;
    }
    return;
  }

  const int h0 = (y - qg - kg) * KH;
  const Place at = place_of(a.c, b, (long long)start + i);
  if (at.page < 0) return;
#pragma unroll
  for (int h = 0; h < KH; ++h) {
    if (h0 + h >= a.c.nkv) break;
    float x[16];
    load_part<DT>(a.v + row * a.ldv + (h0 + h) * HD, HeadPart{16 * u, 16 * u + 8, false}, x);
    float m = largest<16>(x);
    m = larger(m, other_lane<DPP_XOR1>(m));
    m = larger(m, other_lane<DPP_XOR2>(m));
    m = larger(m, other_lane<DPP_MIRROR8>(m));
    const uint16_t sb = m != m ? 0x7fc0 : f32_to_bf16(fmaxf(m / 6.0f, 0x1p-60f));
    const float inv = m != m ? 1.0f : 1.0f / bf16_to_f32(sb);
    // x / s is a border between two codes (3 bits), or off by 2^-11 of its size or more, since x has 11 bits and s 8: what the
    // reciprocal's rounding does to a border is taken back by keeping 16 bits
#pragma unroll
    for (int k = 0; k < 16; ++k) x[k] = __uint_as_float((__float_as_uint(x[k] * inv) + 0x80u) & 0xffffff00u);
    const size_t ph = (size_t)at.page * a.c.nkv + h0 + h;
    *reinterpret_cast<u32x2*>(a.c.v + (ph * a.c.page + at.slot) * ROW + 8 * u) = u32x2{to_e2m1x8(x), to_e2m1x8(x + 8)};
    if (u == 0) a.c.vs[ph * a.c.page + at.slot] = sb;
  }
}

// ---- read --------------------------------------------------------------------------------------
// eight codes as values times s, rounded once to the model dtype
template <int DT>
__device__ __forceinline__ u32x4 from_e2m1x8(uint32_t w, float s) {
  u32x4 o;
  auto two = [&](auto v) { return pack_f32x2<DT>(v[0] * s, v[1] * s); };
  o[0] = two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0));
  o[1] = two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1));
  o[2] = two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2));
  o[3] = two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3));
  return o;
}
__device__ __forceinline__ float key_scale(uint32_t e) {  // (255: NaN)
  return __uint_as_float(e == 255 ? 0x7fc00000u : e == 0 ? 0x00400000u : e << 23);
}
// Eight threads take a row of one head (blockIdx.y), keys and values; rows whose page is none get zeros.  Bound by the results'
// bytes: 32768 rows of two heads 10.2 us, 4.1 TB/s.
template <int DT>
__global__ __launch_bounds__(64) void paged4_read_kernel(Paged4ReadP a) {
  const int u = threadIdx.x & 7, r = threadIdx.x >> 3, h = blockIdx.y, row0 = 8 * (int)blockIdx.x;
  const CallRow cr = call_row(a.s, row0);
  if (cr.b < 0) return;
  const long long row = row0 + r;
  const Place at = place_of(a.c, cr.b, (long long)a.start[cr.b] + cr.i);
  u32x2 k{0, 0}, v{0, 0};
  float ks = 0.f, vs = 0.f;
  if (at.page >= 0) {
    const size_t ph = (size_t)at.page * a.c.nkv + h, slot = ph * a.c.page + at.slot;
    k = *reinterpret_cast<const u32x2*>(a.c.k + slot * ROW + 8 * u);
    v = *reinterpret_cast<const u32x2*>(a.c.v + slot * ROW + 8 * u);
    ks = key_scale(a.c.ks[ph * a.c.page * 4 + key_scale_at(at.slot) + 4 * (u >> 1)]);
    vs = bf16_to_f32(a.c.vs[slot]);
  }
  u32x4* ko = reinterpret_cast<u32x4*>(a.k + row * a.ldk + h * HD + 16 * u);
  u32x4* vo = reinterpret_cast<u32x4*>(a.v + row * a.ldv + h * HD + 16 * u);
  ko[0] = from_e2m1x8<DT>(k[0], ks);
  ko[1] = from_e2m1x8<DT>(k[1], ks);
  vo[0] = from_e2m1x8<DT>(v[0], vs);
  vo[1] = from_e2m1x8<DT>(v[1], vs);
}

// ---- attention ---------------------------------------------------------------------------------
// Rows: a sequence's n query rows x the G query heads of a kv head, flattened as row i, head g -> i G + g, in
// tiles of 16.  Keys: tiles of 64.  A wave computes S^T = K Q^T (rows: keys, columns: queries) and
// O^T = V^T P^T (rows: dims, columns: queries).
//   Bounds: many rows, the matrix and vector instructions, which share the SIMDs' issue (2048 rows over 8192 keys 97 us, 0.93
// PFLOP/s); one row of many sequences, memory (64 of them over 1024 to 8192 keys 22 us with the join, 3.2 TB/s).
//   First product: 16x16x128 with scales, K's codes and powers of two as they are stored, the queries in e4m3 in two parts
// (bf16, whose 8 bits they hold) or three (fp16's 11): hi, the rest of it times 16, the rest of that; one power of two for
// each block of 32 dims, so that what falls under a part's least step is 2^-21 of the block's largest or less.  Lane
// l = 16 g + c holds the 32 dims of block g of key c, and of query c the dims 16 g .. 16 g + 15 and 64 + 16 g .. 64 + 16 g + 15.
//   Product p takes the tile's keys 16 p .. 16 p + 15, which lie in one page (a page is a multiple of 16), as its rows: so lane l
// holds after the four products the scores of query c with the keys 16 p + 4 g + 0..3, and what its softmax leaves is the
// second product's operand as it stands (those of p = 2 h and 2 h + 1 for k step h).
//   Second product: V's codes as bf16, which holds them; their rows are turned into columns on the way through LDS (a
// transposing read of 16 keys x 16 dims for each 16 lanes, whose keys are those above).  A key's scale goes on its probability,
// in fp32.
// The running maximum is that of the query's whole row, held in each of its four lanes; the sum is each lane's own part
// until the end.
//   bf16: p x scale is rounded to bf16, half a step of its own size as the result's rounding.  Where a workgroup has one tile of
// rows (a token of each sequence, which waits for memory) what the rounding leaves goes through the second product too.
// The probabilities, and so their sum, are 2^-24 times as large: p x scale x code stays in range for any scale and 2^24 keys.
// The maximum is exact: the largest probability is 1 then, which is not rounded (2048 rows over 8192 keys, exact / lagging by
// up to 2^8: 99 / 93 us, but an error against 64 bits of 0.0018 / 0.0021, where the result's own rounding gives 0.0017).
//   fp16: p x scale is rounded to fp16, half a step of its own size as the result's rounding.  So that it is in range the
// maximum is that of score + log2 scale, and the largest p x scale 2^11 to 2^15 (the maximum may lag by up to 2^4); what lies
// under 2^-25 of the largest is off by at most 2^-36 of it.  The sum takes p x scale / scale.  Scales are taken as 2^-60 to 2^31: a
// p x scale that leaves fp32's range (2^-137 of the largest) then belongs to a probability of 2^-46 or less beside another.
// (us, bf16 in two parts / this: 2048 rows over 8192 keys 138 / 115, then with three tiles 101; 16 sequences of 32 rows
// 12.9 / 11.9.  Scales of any size and sign cost 0.5 and 0.2 us of these.)

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// K (fp4, its scales the lowest byte of ks) x query part R (e4m3, byte R of qs)
template <int R>
__device__ __forceinline__ f32x4 mfma_kq(u32x4 k, const u32x4 (&q)[2], f32x4 c, uint32_t ks, uint32_t qs) {
  const i32x4 kk = __builtin_bit_cast(i32x4, k);
  const i32x8 a = __builtin_shufflevector(kk, kk, 0, 1, 2, 3, -1, -1, -1, -1);
  const i32x8 b = __builtin_shufflevector(__builtin_bit_cast(i32x4, q[0]), __builtin_bit_cast(i32x4, q[1]), 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 0, 0, (int)ks, R, (int)qs);
}
template <int DT>
__device__ __forceinline__ u32x4 e2m1x8(uint32_t w) {
  if constexpr (DT == DT_BF16)
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 0)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 1)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 2)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 3))};
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 0)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 1)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 2)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 3))};
}
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t larger_halves(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
// four values as e4m3; then x is what they leave, times 16
__device__ __forceinline__ uint32_t e4m3_part(float (&x)[4]) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], r, true);
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(r, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(r, true);
  x[0] = (x[0] - lo[0]) * 16.0f;
  x[1] = (x[1] - lo[1]) * 16.0f;
  x[2] = (x[2] - hi[0]) * 16.0f;
  x[3] = (x[3] - hi[1]) * 16.0f;
  return (uint32_t)r;
}

// what the products in fp16 take of a scale of V: its size, at least 2^-60 (less would have its key leave the range that the sum is
// kept in, and adds no value of fp16's), NaN above 2^31 (fp16 holds no value of such a row)
__device__ __forceinline__ float fp16_scale(float s) {
  s = fabsf(s);
  return s <= 0x1p31f ? fmaxf(s, 0x1p-60f) : __uint_as_float(0x7fc00000u);
}

constexpr int VLD = 72;   // bytes from key to key of V in LDS: the rows that lanes read together lie in different banks
template <int DT> constexpr int PARTS = DT == DT_BF16 ? 2 : 3;

// One workgroup: T tiles of 16 flattened rows of one (sequence, kv head), a split of their keys, its key tiles taken in turn
// by KW waves, whose results are joined through LDS.  The next tile's V is requested as soon as this one's is in LDS, the next
// K when this one's scores are done; page numbers a tile earlier.
template <int DT, int T, int KW>
__global__ __launch_bounds__(64 * KW, KW > 4 ? 1 : T == 1 ? 3 : 2) void paged4_attn_kernel(Paged4AttnP a) {
  constexpr int NP = PARTS<DT>;
  constexpr bool HALFP = DT == DT_F16, TWO = T == 1 && !HALFP;
  constexpr float LAG = HALFP ? 4.f : 0.f, SHIFT = HALFP ? 11.f : -24.f;
  constexpr int PDT = HALFP ? DT_F16 : DT_BF16;
  constexpr int QBYTES = T * NP * 2 * WAVE * 16, VT = 64 * VLD + (HALFP ? 512 : 256), VBYTES = KW * VT;
  constexpr int JOIN = T == 2 ? 2 : 1, SOBYTES = JOIN * KW * 8 * WAVE * 16;
  __shared__ __align__(16) uint8_t lds[QBYTES + VBYTES > SOBYTES ? QBYTES + VBYTES : SOBYTES];
  __shared__ float sm[JOIN][KW][16], sl[JOIN][KW][16];
  __shared__ uint32_t qscale[T][4][16];
  auto qs = reinterpret_cast<u32x4(*)[NP][2][WAVE]>(lds);
  auto so = reinterpret_cast<f32x4(*)[KW][8][WAVE]>(lds);  // (when the queries and V are done with)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  uint8_t* vt = lds + QBYTES + wave * VT;  // a wave's V, and its scales
  float* vscale = reinterpret_cast<float*>(vt + 64 * VLD);
  // Workgroup id lies on XCD id % 8 (round robin).  A group's workgroups take the query tiles of one key range in
  // turn, all on one XCD, whose L2 then reads that range once; where there are fewer than eight ranges their
  // queries are cut into `cuts` groups.
  const int id = (int)blockIdx.x, xcd = id & 7, slot = id >> 3;
  const int group = slot / a.group_wgs * 8 + xcd, range = group / a.cuts;
  // the tiles of most keys (under a mask the last) come first; where all workgroups are resident at once, two to a compute
  // unit (or one, of eight waves), the second ones in the other order (us, by position / this: 2048 rows over 8192 keys
  // 109 / 102, 8192 over themselves 257 / 227)
  const int at = slot % a.group_wgs, half = a.one_round ? a.group_wgs / 2 : a.group_wgs;
  const int tile = (at < half ? a.group_wgs - 1 - at : at - half) * a.cuts + group % a.cuts;
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
  // queries: two waves take a tile, half of the dims each; of three tiles one wave takes one (us, all of a row's dims read by four
  // waves of a tile, two of two tiles / this: a token over 2080 keys 9.1 / 8.7, 16 sequences of 32 rows 11.9 / 11.7)
  constexpr int HALVES = T <= 2 ? 1 : 2;
  const int qt = wave % T, half0 = HALVES == 1 ? wave / T : 0;
  u32x4 qr[2 * HALVES];
  if (wave < 2 * T / HALVES) {
    const int r = 16 * qt + c, i = row_of(r);
    const uint16_t* src = a.q + (long long)(first + i0 + i) * a.ldq + (hk * G + g0 + r - i * G) * HD + 16 * g + 64 * half0;
#pragma unroll
    for (int k = 0; k < 2 * HALVES; ++k)
      qr[k] = m0 + r < M ? *reinterpret_cast<const u32x4*>(src + 64 * (k >> 1) + 8 * (k & 1)) : u32x4{0, 0, 0, 0};
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
  f32x4 o[T][8];
#pragma unroll
  for (int q = 0; q < T; ++q) {
    m[q] = -INFINITY;
    l[q] = 0.f;
#pragma unroll
    for (int d = 0; d < 8; ++d) o[q][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const unsigned heads = (unsigned)(a.c.nkv * page), head = (unsigned)(hk * page);  // slots from page to page, to this head
  auto pages = [&](int t, Four f) {
#pragma unroll
    for (int k = 0; k < 4; ++k) f.p[k] = 64 * t + 16 * k < lk && f.p[k] >= 0 && f.p[k] < a.c.num_pages ? f.p[k] : -1;
    return f;
  };
  auto all_pages = [](Four f) { return (f.p[0] | f.p[1] | f.p[2] | f.p[3]) >= 0; };
  // first of the 16 slots that run k of tile t has in page p (any page's where it has none)
  auto slots = [&](int t, int k, int p) {
    return (unsigned long long)(unsigned)max(p, 0) * heads + head + ((64 * t + 16 * k) & (page - 1));
  };
  u32x4 kw[4], vw[4];
  uint32_t ksw[4], vsw = 0;
  auto load_k = [&](int t, Four f) {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const unsigned long long s0 = slots(t, p, f.p[p]);
      kw[p] = *reinterpret_cast<const u32x4*>(a.c.k + s0 * ROW + (unsigned)(c * ROW + 16 * g));
      ksw[p] = *reinterpret_cast<const uint32_t*>(a.c.ks + s0 * 4 + (unsigned)((c & 3) * 16 + 4 * g));
    }
  };
  auto load_v = [&](int t, Four f) {
#pragma unroll
    for (int k = 0; k < 4; ++k) vw[k] = *reinterpret_cast<const u32x4*>(a.c.v + slots(t, k, f.p[k]) * ROW + (unsigned)(16 * lane));
    const int pg = g & 2 ? (g & 1 ? f.p[3] : f.p[2]) : (g & 1 ? f.p[1] : f.p[0]);
    vsw = a.c.vs[slots(t, g, pg) + c];
  };

  // how many keys from 64 t + 4 g on the lane's query of tile q attends (a column without a query asks for no mask of its own)
  auto first_keys = [&](int q, int t) {
    int r = 16 * q + c;
    if constexpr (T > 2 && HALFP) asm volatile("" : "+v"(r));  // (not kept from step to step)
    return (m0 + r < M ? key_limit(len, lk, n, i0 + row_of(r), a.mask_block) : kmax) - 64 * t - 4 * g;
  };
  // Tile t in the pages now, whose K, V and scales are loaded; the next tile's are requested on the way.
  int t = split * per + wave;
  Four now{};
  // the entries of the tile after: lane k has that of run k & 3.  (Through the vector cache: a wait for LDS would wait for
  // scalar loads too.)
  int next = 0;
  auto entry = [&](int t) { return table[min((64 * t + 16 * (lane & 3)) >> shift, a.c.table_w - 1)]; };
  auto spread = [](int v) {
    return Four{{__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 1), __builtin_amdgcn_readlane(v, 2),
                 __builtin_amdgcn_readlane(v, 3)}};
  };
  // edge: some key is past a query's limit or the end, or in no page
  auto step = [&](auto is_edge) {
    constexpr bool EDGE = decltype(is_edge)::value;
    const Four here = now;
    // the next tile, or this one again: then nothing that is loaded is used
    const bool more = t + KW < t1;
    const int tn = more ? t + KW : t;
    if (more) {
      now = pages(tn, spread(next));
      next = entry(t + 2 * KW);  // (looked at a tile later; past the table its last)
    }
    stay();
    uint32_t ks[4];  // of the word's four slots c & 3, + 4, + 8, + 12 the lane's
#pragma unroll
    for (int p = 0; p < 4; ++p) ks[p] = ksw[p] >> (8 * (c >> 2));
    auto scores = [&](int q, f32x4 (&s)[4]) {
      const uint32_t qsc = qscale[q][g][c];
      const f32x4 zero{0.f, 0.f, 0.f, 0.f};
      const u32x4 q0[2] = {qs[q][0][0][lane], qs[q][0][1][lane]}, q1[2] = {qs[q][1][0][lane], qs[q][1][1][lane]};
      s[0] = mfma_kq<0>(kw[0], q0, zero, ks[0], qsc);
      s[1] = mfma_kq<0>(kw[1], q0, zero, ks[1], qsc);
      s[2] = mfma_kq<0>(kw[2], q0, zero, ks[2], qsc);
      s[3] = mfma_kq<0>(kw[3], q0, zero, ks[3], qsc);
      s[0] = mfma_kq<1>(kw[0], q1, s[0], ks[0], qsc);
      s[1] = mfma_kq<1>(kw[1], q1, s[1], ks[1], qsc);
      s[2] = mfma_kq<1>(kw[2], q1, s[2], ks[2], qsc);
      s[3] = mfma_kq<1>(kw[3], q1, s[3], ks[3], qsc);
      if constexpr (NP == 3) {
        const u32x4 q2[2] = {qs[q][2][0][lane], qs[q][2][1][lane]};
        s[0] = mfma_kq<2>(kw[0], q2, s[0], ks[0], qsc);
        s[1] = mfma_kq<2>(kw[1], q2, s[1], ks[1], qsc);
        s[2] = mfma_kq<2>(kw[2], q2, s[2], ks[2], qsc);
        s[3] = mfma_kq<2>(kw[3], q2, s[3], ks[3], qsc);
      }
    };
    unsigned long long minus = 0;  // (fp16) keys whose scale is negative
    u32x4 pf[T][2], rest[T][2];
    constexpr bool AHEAD = T <= 2, LATE = EDGE && T > 2 && HALFP;  // (three tiles in fp16 have no registers to spare)
    f32x4 sc[2][4];
    if constexpr (AHEAD) scores(0, sc[0]);
#pragma unroll
    for (int q = 0; q < T; ++q) {
      f32x4(&s)[4] = sc[q & 1];
      if constexpr (!AHEAD) scores(q, s);
      else if (q + 1 < T) scores(q + 1, sc[(q + 1) & 1]);
      if (!LATE && q == (AHEAD && T > 1 ? T - 2 : T - 1)) {
        stay();
        load_k(tn, now);
        stay();
      }
      if (q == 0) {  // V into LDS
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint8_t* dst = vt + (16 * k + (lane >> 2)) * VLD + 16 * (lane & 3);
          *reinterpret_cast<u32x2*>(dst) = u32x2{vw[k][0], vw[k][1]};
          *reinterpret_cast<u32x2*>(dst + 8) = u32x2{vw[k][2], vw[k][3]};
        }
        if constexpr (HALFP) {
          minus = __ballot(vsw >> 15);
          const float vs = fp16_scale(__uint_as_float(vsw << 16));
          vscale[lane] = __builtin_amdgcn_logf(vs);
          vscale[64 + lane] = __builtin_amdgcn_rcpf(vs);
        } else {
          vscale[lane] = __uint_as_float(vsw << 16);
        }
        stay();
      }
      const int lim = EDGE ? first_keys(q, t) : 64;
      if constexpr (HALFP) {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const f32x4 lv = *reinterpret_cast<const f32x4*>(vscale + 16 * p + 4 * g);
#pragma unroll
          for (int i = 0; i < 4; ++i) s[p][i] = __builtin_fmaf(s[p][i], a.scale_log2e, lv[i]);
        }
      }
      if constexpr (EDGE) {
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[p][i] = 16 * p + i < (here.p[p] < 0 ? 0 : lim) ? s[p][i] : -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[p][i]);
      if constexpr (!HALFP) mx *= a.scale_log2e;
      if (__any(mx > m[q] + LAG)) {
        const float mn = fmaxf(m[q], rows_max(mx));
        const float al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[q] - mn);
        m[q] = mn;
        l[q] *= al;
#pragma unroll
        for (int d = 0; d < 8; ++d) o[q][d] *= al;
      }
      const float sub = (m[q] == -INFINITY ? 0.f : m[q]) - SHIFT;
      float ls = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        f32x4 p[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const f32x4 vs = *reinterpret_cast<const f32x4*>(vscale + (HALFP ? 64 : 0) + 32 * h + 16 * k + 4 * g);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            // (what lies behind may be NaN)
            if constexpr (HALFP) {
              p[k][i] = __builtin_amdgcn_exp2f(s[2 * h + k][i] - sub);
              ls = __builtin_fmaf(p[k][i], !EDGE || p[k][i] != 0.f ? vs[i] : 0.f, ls);
            } else {
              p[k][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * h + k][i], a.scale_log2e, -sub));
              ls += p[k][i];
              p[k][i] = !EDGE || 32 * h + 16 * k + i < (here.p[2 * h + k] < 0 ? 0 : lim) ? p[k][i] * vs[i] : 0.f;
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = p[e >> 1][2 * (e & 1)], y = p[e >> 1][2 * (e & 1) + 1];
          if constexpr (HALFP) pf[q][h][e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x, y}), f16x2));
          else pf[q][h][e] = pack_f32x2<PDT>(x, y);
          if constexpr (TWO)
            rest[q][h][e] = pack_f32x2<DT_BF16>(x - lo_f32<DT_BF16>(pf[q][h][e]), y - hi_f32<DT_BF16>(pf[q][h][e]));
        }
      }
      l[q] += ls;
    }
    stay();
    if (HALFP && minus != 0) {  // the sign goes to the key's codes
      // (the lane's number made here again: three tiles have no register to keep it in)
      unsigned l = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0));
      asm volatile("" : "+v"(l));
      const uint32_t flip = minus >> l & 1 ? 0x88888888u : 0;
#pragma unroll 1
      for (int k = 0; k < 8; ++k) *reinterpret_cast<u32x2*>(vt + l * VLD + 8 * k) ^= flip;
    }
    if constexpr (LATE) load_k(tn, now);
    load_v(tn, now);
    stay();
    typedef int i32x2 __attribute__((ext_vector_type(2)));
    auto column = [&](int d) {  // of dim 16 d + c the codes of keys 4 g + 0..3, 16 + 4 g + 0..3, 32 .., 48 ..
      return __builtin_amdgcn_ds_read_tr4_b64_v2i32(
          (__attribute__((address_space(3))) i32x2*)(vt + (16 * (c >> 2) + 4 * g + (c & 3)) * VLD + 8 * d));
    };
    // (the products' wave goes first: the other one of the SIMD has its softmax to do meanwhile; us, without / with: 2048 rows over
    // 8192 keys 99.4 / 94.8, 8192 over themselves 220 / 215)
    __builtin_amdgcn_s_setprio(1);
    i32x2 col[2] = {column(0), column(1)};
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      const i32x2 w = col[d & 1];
      if (d + 2 < 8) col[d & 1] = column(d + 2);
      const u32x4 v0 = e2m1x8<PDT>((uint32_t)w[0]), v1 = e2m1x8<PDT>((uint32_t)w[1]);
#pragma unroll
      for (int q = 0; q < T; ++q) {
        o[q][d] = mfma16<PDT>(v0, pf[q][0], o[q][d]);
        o[q][d] = mfma16<PDT>(v1, pf[q][1], o[q][d]);
        if constexpr (TWO) {
          o[q][d] = mfma16<DT_BF16>(v0, rest[q][0], o[q][d]);
          o[q][d] = mfma16<DT_BF16>(v1, rest[q][1], o[q][d]);
        }
      }
    }
    __builtin_amdgcn_s_setprio(0);
    stay();
    t += KW;
  };

  if (t < t1) now = pages(t, a.S == 1 ? early : entries(t));
  stay();
  if (t < t1) {
    load_k(t, now);
    load_v(t, now);
    next = entry(t + KW);
  }
  stay();
  if (wave < 2 * T / HALVES) {
    // the exponents of the largest values of the blocks that the runs lie in: block g / 2 and 2 + g / 2
    uint32_t E[HALVES];
    float f[HALVES];
#pragma unroll
    for (int k = 0; k < HALVES; ++k) {
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = larger_halves(top, qr[2 * k + (e >> 2)][e & 3] & 0x7fff7fffu);
      const uint32_t mine = __float_as_uint(fmaxf(lo_f32<DT>(top), hi_f32<DT>(top)));
      // (not finite: the dtype's own largest exponent, which larger_halves keeps and the maximum of floats might not)
      const uint32_t bits = larger_halves(top, top << 16) >> 16;
      const bool finite_ = DT == DT_BF16 ? bits < 0x7f80u : bits < 0x7c00u;
      const auto two = __builtin_amdgcn_permlane16_swap(finite_ ? mine : 0x7f800000u, finite_ ? mine : 0x7f800000u, false, false);
      const uint32_t e = max(two[0], two[1]) >> 23;
      E[k] = e < 255 ? max(e, 24u) : 255u;
      f[k] = __uint_as_float((e < 255 ? 261 - E[k] : 127) << 23);  // (values below 2^8 then)
    }
    if ((g & 1) == 0) {
#pragma unroll
      for (int k = 0; k < HALVES; ++k)
        qscale[qt][2 * (half0 + k) + (g >> 1)][c] = E[k] < 255 ? E[k] - 7 | (E[k] - 11) << 8 | (E[k] - 15) << 16 : 0xffffffffu;
    }
    // part by part, four dims at a time
#pragma unroll
    for (int j = 0; j < 4 * HALVES; ++j) {
      const u32x4 w = qr[j >> 1];
      float x[4] = {lo_f32<DT>(w[2 * (j & 1)]) * f[j >> 2], hi_f32<DT>(w[2 * (j & 1)]) * f[j >> 2],
                    lo_f32<DT>(w[2 * (j & 1) + 1]) * f[j >> 2], hi_f32<DT>(w[2 * (j & 1) + 1]) * f[j >> 2]};
#pragma unroll
      for (int r = 0; r < NP; ++r) reinterpret_cast<uint32_t*>(&qs[qt][r][half0 + (j >> 2)][lane])[j & 3] = e4m3_part(x);
    }
  }
  // the queries are in LDS for all waves; K and V stay under way
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  stay();
  // (two loops: with both forms in one the compiler keeps the sums in two places and spills)
  while (t < t1 && 64 * t + 64 <= kmin && all_pages(now)) step(std::false_type{});
  while (t < t1) step(std::true_type{});

  // the waves' parts of the keys, joined in wave order: each wave takes 128 / KW dims of all queries; of two tiles at once where
  // LDS has room (16 sequences of 32 rows over up to 1056 keys, one by one / this: 11.9 / 11.6 us)
  __syncthreads();
  const long long rq = (long long)a.s.rows * a.nq;
#pragma unroll
  for (int q0 = 0; q0 < T; q0 += JOIN) {
    if (m0 + 16 * q0 >= M) break;
#pragma unroll
    for (int z = 0; z < JOIN; ++z) {
      const int q = q0 + z;
      l[q] = rows_sum(l[q]);
#pragma unroll
      for (int d = 0; d < 8; ++d) so[z][wave][d][lane] = o[q][d];
      if (g == 0) {
        sm[z][wave][c] = m[q];
        sl[z][wave][c] = l[q];
      }
    }
    __syncthreads();
#pragma unroll
    for (int z = 0; z < JOIN; ++z) {
      const int r = 16 * (q0 + z) + c;
      if (m0 + r < M) {
        float mm = -INFINITY, ll = 0.f, wgt[KW];
#pragma unroll
        for (int w = 0; w < KW; ++w) mm = fmaxf(mm, sm[z][w][c]);
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          wgt[w] = sm[z][w][c] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(sm[z][w][c] - mm);  // (without keys: zeros)
          ll += wgt[w] * sl[z][w][c];
        }
        const int i = row_of(r);
        const long long idx = (long long)(first + i0 + i) * a.nq + hk * G + g0 + r - i * G;
        const float inv = a.S > 1 ? 1.0f : ll == 0.f ? 0.f : 1.0f / ll;
#pragma unroll
        for (int k = 0; k < 8 / KW; ++k) {
          const int d = 8 / KW * wave + k;
          f32x4 v = wgt[0] * so[z][0][d][lane];
#pragma unroll
          for (int w = 1; w < KW; ++w) v += wgt[w] * so[z][w][d][lane];
          if (a.S > 1) {
            *reinterpret_cast<f32x4*>(a.part + (split * rq + idx) * HD + 16 * d + 4 * g) = v;
          } else {
            v *= inv;
            *reinterpret_cast<u32x2*>(a.out + idx * HD + 16 * d + 4 * g) =
                u32x2{pack_f32x2<DT>(v[0], v[1]), pack_f32x2<DT>(v[2], v[3])};
          }
        }
        if (a.S > 1 && wave == 0 && g == 0) {
          float* pm = a.part + a.S * rq * HD + (split * rq + idx) * 2;
          pm[0] = mm;
          pm[1] = ll;
        }
      }
    }
    if (q0 + JOIN < T) __syncthreads();
  }
}

long long row_wgs(int rows) { return (rows + 7ll) / 8; }
long long attn_wgs(const Paged4AttnP& a) {
  return ((long long)a.S * a.c.nkv * a.s.nseq * a.cuts + 7) / 8 * 8 * a.group_wgs;
}
template <int DT>
hipError_t launch_attn_dt(const Paged4AttnP& a, hipStream_t st) {
  const dim3 grid((unsigned)attn_wgs(a));
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(64 * a.waves), 0, st, a); };
  if (a.waves == 8) launch(paged4_attn_kernel<DT, 2, 8>);
  else if (a.tiles16 == 1) launch(paged4_attn_kernel<DT, 1, 4>);
  else if (a.tiles16 == 2) launch(paged4_attn_kernel<DT, 2, 4>);
  else launch(paged4_attn_kernel<DT, 3, 4>);
  if (const hipError_t e = hipGetLastError(); e != hipSuccess || a.S == 1) return e;
  return launch_paged_merge(DT, PagedMergeP{a.s, a.nq, a.S, a.part, a.out}, st);
}

}  // namespace

namespace {
// Heads that a workgroup takes: four query heads or two kv heads share the sines and cosines, which are in 64 bits for the keys,
// but few workgroups are a chain of instructions, which two and one make shorter.  The more heads, the fewer rows make enough
// workgroups (us, two and one / four and two, of 12 + 2 heads: 1024 rows 4.7 / 5.7, 3008 rows 9.0 / 9.5, 4096 rows 10.7 / 10.4,
// 8192 rows 16.3 / 15.6; 4 + 2 heads: 6000 rows 8.7 / 9.1, 16384 rows 16.5 / 15.8; 8 + 8: 2048 rows 8.7 / 9.2, 3008 rows 12.0 /
// 11.6; 32 + 8: 1024 rows 8.8 / 9.5, 2048 rows 13.0 / 12.8; 64 + 8: 1024 rows 11.5 / 12.1, 2048 rows 19.4 / 18.9; 16 + 1, whose
// keys share nothing: 512 rows 4.4 / 4.6, 3008 rows 10.1 / 9.5).
template <int DT, bool INTER>
hipError_t launch_append(const Paged4AppendP& a, hipStream_t st) {
  auto heads = [&](int qh, int kh) { return (a.q ? (a.nq + qh - 1) / qh : 0) + 2 * ((a.c.nkv + kh - 1) / kh); };
  const bool few = row_wgs(a.s.rows) * heads(4, 2) <= 3100;
  const dim3 grid((unsigned)row_wgs(a.s.rows), few ? heads(2, 1) : heads(4, 2));
  if (few) hipLaunchKernelGGL((paged4_append_kernel<DT, INTER, 2, 1>), grid, dim3(64), 0, st, a);
  else hipLaunchKernelGGL((paged4_append_kernel<DT, INTER, 4, 2>), grid, dim3(64), 0, st, a);
  return hipGetLastError();
}
}  // namespace
hipError_t launch_paged4_append(int dt, const Paged4AppendP& a, hipStream_t st) {
  if (dt == DT_BF16) return a.t.inter ? launch_append<DT_BF16, true>(a, st) : launch_append<DT_BF16, false>(a, st);
  return a.t.inter ? launch_append<DT_F16, true>(a, st) : launch_append<DT_F16, false>(a, st);
}

bool paged4_rows_fit(int rows) { return grid_fits(row_wgs(rows), 64); }

hipError_t launch_paged4_read(int dt, const Paged4ReadP& a, hipStream_t st) {
  const dim3 grid((unsigned)row_wgs(a.s.rows), a.c.nkv);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(64), 0, st, a); };
  dt == DT_BF16 ? launch(paged4_read_kernel<DT_BF16>) : launch(paged4_read_kernel<DT_F16>);
  return hipGetLastError();
}

// Tiles of 16 flattened rows that a workgroup takes: one where a kv head has no more; else two, or three where that still
// leaves two workgroups for each compute unit (us, two / three: 2048 rows over 8192 keys 114 / 109, in fp16 116 / 102,
// 16 sequences of 128 rows 37.2 / 35.8, 16 of 32 rows 12.7 / 17.7).
// Waves: eight where two tiles leave one workgroup or less to a compute unit, so that each SIMD still has two (us, four /
// eight: 512 rows over 4608 keys 33.3 / 27.6, 64 sequences of 8 rows over 1000 to 2056 keys 20.6 / 17.3, 32 rows over 32768
// keys 22.7 / 20.7, 16 sequences of 32 rows over up to 1056 keys 12.5 / 11.6, in fp16 14.6 / 13.1).  One tile: four, and
// more splits (a token over 2080 keys 9.0, with eight waves and no split 12.5; of 64 sequences 23.4 / 24.6).
// Key splits: as many as leave the workgroups within one (one tile: two) to a compute unit, none below a tile of keys for each
// wave; up to three tiles (five, where workgroups have one) for each wave are not split, since joining costs a launch.
bool paged4_attn_plan(Paged4AttnP& a, int cus) {
  const long long M = (long long)a.s.max_rows * (a.nq / a.c.nkv), pairs = (long long)a.c.nkv * a.s.nseq;
  a.tiles16 = M <= 16 ? 1 : (M + 47) / 48 * pairs >= 2 * cus ? 3 : 2;
  const long long rows = 16 * a.tiles16, wide = (M + rows - 1) / rows, tiles = ((long long)a.max_len + 63) / 64;
  const long long wgs = wide * pairs;
  a.waves = a.tiles16 == 2 && wgs <= cus ? 8 : 4;
  long long S = 1;
  if (tiles > (a.tiles16 == 1 ? 5 : 3) * a.waves)
    S = std::max(1ll, std::min({(a.tiles16 == 1 ? 2ll : 1ll) * cus / wgs, (tiles + a.waves - 1) / a.waves, 64ll}));
  // ranges in whole rounds of the eight XCDs, where their workgroups follow each other there
  while (wide > 1 && S > 8 && S * pairs % 8 != 0) --S;
  a.S = (int)S;
  const long long ranges = S * pairs;
  a.cuts = (int)std::min(ranges >= 8 ? 1ll : (8 + ranges - 1) / ranges, wide);
  a.group_wgs = (int)((wide + a.cuts - 1) / a.cuts);
  a.one_round = attn_wgs(a) <= 8ll / a.waves * cus;
  return grid_fits(attn_wgs(a), 64 * a.waves) && grid_fits(((long long)a.s.max_rows * a.nq + 3) / 4, 256);
}
size_t paged4_attn_floats(const Paged4AttnP& a) {
  return a.S > 1 ? (size_t)a.S * a.s.rows * a.nq * (HD + 2) : 0;
}
hipError_t launch_paged4_attn(int dt, const Paged4AttnP& a, hipStream_t st) {
  return dt == DT_BF16 ? launch_attn_dt<DT_BF16>(a, st) : launch_attn_dt<DT_F16>(a, st);
}

}  // namespace fdllm
