// Log probabilities of given tokens, with each row's entropy and most probable alternatives, in one pass over the
// logits.
#include <algorithm>

#include "common.hpp"
#include "logprobs.hpp"

namespace fdllm {

namespace {

typedef unsigned long long u64;
constexpr float LOG2E = 1.44269504088896340736f;
constexpr int EPL = 16;                        // elements a lane takes per iteration
constexpr int CHUNK = EPL * WAVE;              // elements a wave takes per iteration
constexpr int LIST = LP_MAX_TOP * (EPL + 1);   // a wave's candidates: the best so far and 64 lanes' at most
// Iterations whose maxima a wave keeps, a multiple of 8 (they are read 16 bytes at a time): the most with which a workgroup's LDS,
// 39.5 KB, leaves room for four on a compute unit, as its registers do.  Longer rows are taken in such parts, each with a bound
// of its own.  us of 600 rows with 32 / 40 / 48: of 151936 bf16 55.1 / 52.0 / 52.2, of 163840 (one part of 40) 57.0 / 53.7 / 53.8,
// of 167936 (two) 58.1 / 56.8 / 54.9, of 262144 86.4 / 86.0 / 85.8; of fp32 76.8 / 76.5 / 77.2, 78.4 / 77.9 / 78.2, 79.4 / 81.6 /
// 80.2 and 124.6 / 123.5 / 124.5.
constexpr int REC = 40;
constexpr int WAVES = 4;
constexpr int AHEAD = 8;                       // keys that a ranking loop requests at once
constexpr int MAX_SPLITS = 64;

// A logit and its index as one number whose order is that of the alternatives: by value (-0 is 0, NaN lies with -inf),
// equal ones by index, the lower first.
__device__ __forceinline__ u64 key_of(float x, int idx) {
  x = x == x ? x + 0.0f : -INFINITY;
  const uint32_t b = __float_as_uint(x);
  const uint32_t o = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  return ((u64)o << 32) | (uint32_t)~idx;
}
__device__ __forceinline__ float key_value(u64 k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ int key_index(u64 k) { return (int)~(uint32_t)k; }

// One row's softmax as far as a lane, a wave or a split has seen it: the largest logit m (at least -FLT_MAX), s = sum
// exp(x - m), u = sum exp(x - m) (x - m).  log-sum-exp = m + log s, entropy = log s - u / s.
struct Stat { float m, s, u; };
__device__ __forceinline__ Stat stat_join(Stat a, Stat b) {
  const float m = fmaxf(a.m, b.m);
  const float da = a.m - m, db = b.m - m;
  const float ea = __builtin_amdgcn_exp2f(da * LOG2E), eb = __builtin_amdgcn_exp2f(db * LOG2E);
  Stat r;
  r.m = m;
  r.s = ea * a.s + eb * b.s;
  // (a part with nothing in it has s = u = 0 and adds nothing, whatever its distance)
  r.u = ea * (a.u + fmaxf(da, -1e30f) * a.s) + eb * (b.u + fmaxf(db, -1e30f) * b.s);
  return r;
}

template <int LT> struct Elem { typedef u16 type; static constexpr int E = 8; };
template <> struct Elem<LT_F32> { typedef float type; static constexpr int E = 4; };

template <int LT> __device__ __forceinline__ float one(const typename Elem<LT>::type* p) {
  if constexpr (LT == LT_F32) return *p;
  else return to_f32<LT == LT_BF16 ? DT_BF16 : DT_F16>(*p);
}
// the E elements of a 16-byte unit
template <int LT> __device__ __forceinline__ void unpack(u32x4 w, float* x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (LT == LT_F32) x[i] = __uint_as_float(w[i]);
    else {
      x[2 * i] = lo_f32<LT == LT_BF16 ? DT_BF16 : DT_F16>(w[i]);
      x[2 * i + 1] = hi_f32<LT == LT_BF16 ? DT_BF16 : DT_F16>(w[i]);
    }
  }
}

// lane p's key, p uniform
__device__ __forceinline__ u64 lane_key(u64 k, int p) {
  return ((u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(k >> 32), p) << 32) |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)k, p);
}
// At most the n-th largest (from 1) of the lanes' values, and within 2^-7 of it: its order's upper 16 bits, found from the
// top by counting the lanes that reach them (a vector compare and a few scalar operations each; ranking the lanes
// against each other takes 200 vector instructions).
__device__ __forceinline__ float nth_lane(float v, int n) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  const uint32_t o = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  uint32_t t = 0;
#pragma unroll
  for (int k = 31; k >= 16; --k) {
    const uint32_t up = t | (1u << k);
    t = __popcll(__ballot(o >= up)) >= n ? up : t;
  }
  // (below the order of -inf lie NaN's bits)
  return t <= 0x007fffffu ? -INFINITY : __uint_as_float(t & 0x80000000u ? t ^ 0x80000000u : ~t);
}
// the n-th largest of the lanes' keys
__device__ __forceinline__ u64 nth_lane_key(u64 v, int n, int lane) {
  int rank = 0;
  for (int p = 0; p < WAVE; ++p) {
    const u64 o = lane_key(v, p);
    rank += (o > v || (o == v && p < lane)) ? 1 : 0;
  }
  const unsigned long long who = __ballot(rank == n - 1);
  return lane_key(v, __ffsll(who) - 1);
}

// how many of the n keys in LDS (zeros up to the next multiple of AHEAD) are larger than k
__device__ __forceinline__ int rank_of(u64 k, const u64* list, int n) {
  int rank = 0;
  for (int q = 0; q < n; q += AHEAD) {
    u64 v[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) v[i] = list[q + i];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) rank += v[i] > k ? 1 : 0;
  }
  return rank;
}

// The wave's candidates in LDS: the `top` best logits taken are always among its `n` keys; logits above `t` enter it.
// Elements are taken in ascending order of their indices from one call to the next, so a later one equal to t has the
// higher index and stays out.
struct Cand { u64* list; int n; float t; };

// the list cut down to its `top` best, in order (any list: one that ran full, or has many equal logits)
__device__ __forceinline__ void cand_cut(Cand& c, int top, int lane) {
  u64 mine[(LIST + 63) / 64];
  int rank[(LIST + 63) / 64];
#pragma unroll
  for (int i = 0; i < (LIST + 63) / 64; ++i) {
    const int p = lane + 64 * i;
    mine[i] = p < c.n ? c.list[p] : 0;
    rank[i] = 0;
  }
  for (int p = 0; p < c.n; ++p) {
    const u64 k = c.list[p];
#pragma unroll
    for (int i = 0; i < (LIST + 63) / 64; ++i)
      if (64 * i < c.n) rank[i] += k > mine[i] ? 1 : 0;
  }
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < (LIST + 63) / 64; ++i)
    if (lane + 64 * i < c.n && rank[i] < top) c.list[rank[i]] = mine[i];
  __builtin_amdgcn_wave_barrier();
  c.n = min(c.n, top);
  if (c.n == top) c.t = fmaxf(c.t, key_value(c.list[top - 1]));
}

// The lanes' elements above c.t, and not below `from`, into the list: x[i] has index idx(i), -inf where there is none; mx is the
// lane's largest.
template <class IDX>
__device__ __forceinline__ void cand_take(Cand& c, const float (&x)[EPL], float mx, float from, IDX idx, int top, int lane) {
  int total = EPL * __popcll(__ballot(mx > c.t && mx >= from));  // at most
  if (c.n + total > LIST) {
    total = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) total += __popcll(__ballot(x[i] > c.t && x[i] >= from));
  }
  u64 floor_key = 0;
  if (c.n + total > LIST) {
    cand_cut(c, top, lane);
    // the `top` best of the lanes' own best are at least as many elements, so nothing below the last of them is
    // wanted; no more than `top` lanes have elements that reach it
    u64 best = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const u64 k = x[i] > c.t ? key_of(x[i], idx(i)) : 0;
      best = k > best ? k : best;
    }
    floor_key = nth_lane_key(best, top, lane);
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    bool in = x[i] > c.t && x[i] >= from;
    if (__any(in)) {
      const u64 k = key_of(x[i], idx(i));
      in = in && k >= floor_key;
      const unsigned long long b = __ballot(in);
      if (in) c.list[c.n + __popcll(b & ((1ull << lane) - 1))] = k;
      c.n += __popcll(b);
    }
  }
  __builtin_amdgcn_wave_barrier();
}

// the largest of a lane's elements as 16 bits, rounded up
__device__ __forceinline__ u16 up16(float x) {
  const uint32_t b = __float_as_uint(x);
  return (u16)((b & 0x80000000u ? b : b + 0xffffu) >> 16);
}

// an iteration's elements, mx the lane's largest of them, into its statistics
__device__ __forceinline__ void stat_take(Stat& st, const float (&x)[EPL], float mx) {
  if (mx > st.m) {
    const float d = st.m - mx, e = __builtin_amdgcn_exp2f(d * LOG2E);
    st.u = e * (st.u + fmaxf(d, -1e30f) * st.s);
    st.s *= e;
    st.m = mx;
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const float d = x[i] - st.m;
    const float e = __builtin_amdgcn_exp2f(d * LOG2E);
    st.s += e;
    st.u += e * fmaxf(d, -1e30f);  // (an excluded token's logit is -inf and its e 0)
  }
}

// the logit of the row's given token (0 without one), asked for long before row_results needs it
template <int LT>
__device__ __forceinline__ float given_logit(const LogprobsP& a, int r) {
  if (a.ids == nullptr) return 0.f;
  const int id = a.ids[r];
  return id >= 0 && id < a.vocab ? one<LT>((const typename Elem<LT>::type*)a.logits + r * a.ld + id) : 0.f;
}

// the results of a row whose statistics and `n` best keys (in order, LDS) are complete
template <int LT>
__device__ __forceinline__ void row_results(const LogprobsP& a, int r, Stat st, const u64* best, int n, float given) {
  const float ls = logf(st.s), lse_m = st.m;
  // only -inf: no distribution (0 / 0); +inf: inf - inf
  const bool none = !(st.s > 0.f) || !(fabsf(lse_m) < INFINITY);
  const float nan = __uint_as_float(0x7fc00000u);
  const int t = threadIdx.x;
  if (t == 0) {
    a.entropy[r] = none ? nan : ls - st.u / st.s;
    if (a.ids != nullptr) {
      const int id = a.ids[r];
      float v = 0.f;
      if (id >= a.vocab) v = nan;
      else if (id >= 0) v = none ? nan : (given - lse_m) - ls;
      a.logprob[r] = v;
    }
  }
  if (t < a.top) {
    int id;
    float v;
    if (t < n) {
      id = key_index(best[t]);
      v = key_value(best[t]);
    } else {
      // fewer tokens than alternatives have a probability: the others by index
      int skip = t - n;
      id = 0;
      for (;; ++id) {
        bool listed = false;
        for (int i = 0; i < n; ++i) listed |= key_index(best[i]) == id;
        if (!listed && skip-- == 0) break;
      }
      v = one<LT>((const typename Elem<LT>::type*)a.logits + r * a.ld + id);
    }
    a.top_ids[(long long)r * a.top + t] = id;
    a.top_logprob[(long long)r * a.top + t] = none ? nan : (v - lse_m) - ls;
  }
}

// One workgroup takes split blockIdx.y of row blockIdx.x: a range of the row's whole 16-byte units, a quarter per
// wave, in order.  The elements before the first unit belong to the first wave of the first split, those behind the
// last to the last wave of the last.
// The stream itself only gathers statistics and each lane's largest logit of each iteration.  The alternatives are found
// afterwards: the top-th largest of the lanes' largest logits is a bound that `top` logits reach, and few others do (24
// of a wave's reach that of 20); the lanes and iterations that hold any are known, and their 16 elements are read
// again.  (Looking for them in the stream cost 2800 clocks an iteration, four times the statistics.)
// 1024 rows of 151936 float32 with 20 alternatives: 622 MB in 118 us, 5.3 TB/s.  One row of 151643 bfloat16: 8.8 us and 4.8
// to join its splits, the stages' latencies (load, bound, reading again, ranking).
template <int LT>
__global__ __launch_bounds__(64 * WAVES) void logprobs_kernel(LogprobsP a) {
  typedef typename Elem<LT>::type T;
  constexpr int E = Elem<LT>::E, UPL = EPL / E;  // units per lane and iteration
  __shared__ __align__(16) u64 lists[WAVES][LIST + AHEAD];
  __shared__ u64 best[LP_MAX_TOP];
  __shared__ Stat stats[WAVES];
  __shared__ float bounds[WAVES];
  __shared__ int counts[WAVES];
  __shared__ __align__(16) u16 recs[WAVES][WAVE][REC];
  __shared__ int who[WAVES][WAVE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = blockIdx.x, split = blockIdx.y;
  const T* row = (const T*)a.logits + r * a.ld;
  const int head = min(a.vocab, (int)(((16 - ((uintptr_t)row & 15)) & 15) / sizeof(T)));
  const int units = (a.vocab - head) / E, tail0 = head + units * E;
  const u32x4* body = reinterpret_cast<const u32x4*>(row + head);
  const int parts = a.S * WAVES, part = split * WAVES + wave;
  const int per = (units + parts - 1) / parts;
  const int u0 = min(units, part * per), u1 = min(units, u0 + per);
  const int top = a.top;
  const float given = a.S == 1 && threadIdx.x == 0 ? given_logit<LT>(a, r) : 0.f;
  Cand c{lists[wave], 0, -INFINITY};
  Stat st{-3.402823466e38f, 0.f, 0.f};
  float lane_max = -INFINITY;  // (st.m starts above -inf)
#define FD_INLINE __attribute__((always_inline))
  auto load = [&](u32x4 (&w)[UPL], int u) FD_INLINE {  // this lane's units of an iteration, u its first
#pragma unroll
    for (int i = 0; i < UPL; ++i)
      if (u + 64 * i < u1) w[i] = body[u + 64 * i];
  };
  auto values = [&](const u32x4 (&w)[UPL], int u, float (&x)[EPL]) FD_INLINE {
#pragma unroll
    for (int i = 0; i < UPL; ++i) {
      unpack<LT>(w[i], x + i * E);
#pragma unroll
      for (int e = 0; e < E; ++e) x[i * E + e] = u + 64 * i < u1 ? x[i * E + e] : -INFINITY;
    }
  };
  auto largest = [](const float (&x)[EPL]) FD_INLINE {
    float mx = x[0];
#pragma unroll
    for (int i = 1; i < EPL; ++i) mx = fmaxf(mx, x[i]);
    return mx;
  };
  // the row's ends: its first `head` elements are the first wave's, those from tail0 the last one's
  auto ends = [&](int from, int n) FD_INLINE {
    const float x = lane < n ? one<LT>(row + from + lane) : -INFINITY;
    lane_max = fmaxf(lane_max, x);
    float xs[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) xs[i] = i == 0 ? x : -INFINITY;
    stat_take(st, xs, x);
  };
  constexpr int HEAD = -1, TAIL = -2;
  bool head_item = part == 0 && head > 0, tail_item = part == parts - 1 && tail0 < a.vocab;
  if (head_item) ends(0, head);
  if (tail_item) ends(tail0, a.vocab - tail0);

  constexpr int STEP = UPL * WAVE;  // units of an iteration
  // 64 bytes a lane requested ahead: one iteration of fp32, two of 16 bits (us, one / two: 1200 rows of 151936 fp32 147 / 166,
  // with fewer waves for the registers, of bf16 111 / 90)
  constexpr int DEPTH = E / 4;
  u32x4 next[DEPTH][UPL];
#pragma unroll
  for (int h = 0; h < DEPTH; ++h) load(next[h], u0 + h * STEP + lane);
  int u = u0;
  bool last;
  do {
    // at most REC iterations
    const int base = u;
    int n = 0;
    while (u < u1 && n < REC) {
      static_assert(REC % DEPTH == 0 && REC % 8 == 0 && REC < 64);
#pragma unroll
      for (int h = 0; h < DEPTH; ++h) {
        if (u >= u1) break;
        float x[EPL];
        values(next[h], u + lane, x);
        load(next[h], u + DEPTH * STEP + lane);
        const float mx = largest(x);
        lane_max = fmaxf(lane_max, mx);
        if (top > 0) recs[wave][lane][n] = up16(mx);
        stat_take(st, x, mx);
        u += STEP;
        ++n;
      }
    }
    last = u >= u1;
    if (top == 0) continue;
    // the last ones against the best bound of the four waves (each wave comes here once)
    float bound = nth_lane(lane_max, top);
    if (last) {
      if (lane == 0) bounds[wave] = bound;
      __syncthreads();
      bound = fmaxf(fmaxf(bounds[0], bounds[1]), fmaxf(bounds[2], bounds[3]));
    }
    // the iterations in which some lane reaches it, and this lane's
    unsigned long long any = 0, mine = 0;
    for (int i0 = 0; i0 < n; i0 += 8) {
      const u32x4 v = *reinterpret_cast<const u32x4*>(&recs[wave][lane][i0]);
      unsigned a8 = 0, m8 = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool in = (i & 1 ? hi_f32<DT_BF16>(v[i / 2]) : lo_f32<DT_BF16>(v[i / 2])) >= bound;
        a8 |= __ballot(in) != 0 ? 1u << i : 0u;
        m8 |= in ? 1u << i : 0u;
      }
      any |= (unsigned long long)a8 << i0;
      mine |= (unsigned long long)m8 << i0;
    }
    any &= (1ull << n) - 1;  // (n <= REC < 64)
    // Up to 64 (iteration, lane) pairs at a time: whole iterations, and the ends before and after all of them, so that
    // indices ascend from one cand_take to the next.  Lane l takes the elements of the l-th pair.
    int cnt = 0;
    if (head_item) {
      if (lane == 0) who[wave][0] = HEAD;
      cnt = 1;
      head_item = false;
    }
    bool more;
    do {
      while (any != 0) {
        const int i = __builtin_ctzll(any);
        const bool in = mine >> i & 1;
        const unsigned long long b = __ballot(in);
        const int k = __popcll(b);
        if (cnt + k > WAVE) break;
        if (in) who[wave][cnt + __popcll(b & ((1ull << lane) - 1))] = i << 6 | lane;
        cnt += k;
        any &= any - 1;
      }
      more = any != 0;
      if (!more && last && tail_item) {
        if (cnt < WAVE) {
          if (lane == 0) who[wave][cnt] = TAIL;
          ++cnt;
          tail_item = false;
        } else {
          more = true;
        }
      }
      if (cnt > 0) {
        __builtin_amdgcn_wave_barrier();
        const int p = lane < cnt ? who[wave][lane] : 0;
        __builtin_amdgcn_wave_barrier();
        const int at = lane < cnt && p >= 0 ? base + (p >> 6) * STEP + (p & 63) : u1;  // (u1: nothing)
        u32x4 w[UPL];
        load(w, at);
        float x[EPL];
        values(w, at, x);
        int from = head + at * E, step = WAVE * E;  // element i's index: from + i / E step + i % E
        if (p < 0) {
          from = p == HEAD ? 0 : tail0;
          step = E;
          const int m = p == HEAD ? head : a.vocab - tail0;
#pragma unroll
          for (int i = 0; i < E - 1; ++i)
            if (i < m) x[i] = one<LT>(row + from + i);
        }
        cand_take(c, x, largest(x), bound, [&](int i) { return from + i / E * step + i % E; }, top, lane);
        cnt = 0;
      }
    } while (more);
  } while (!last);
#undef FD_INLINE
  // the wave's lanes, in a fixed order
  for (int k = 32; k >= 1; k >>= 1) {
    const Stat o{__shfl_xor(st.m, k, WAVE), __shfl_xor(st.s, k, WAVE), __shfl_xor(st.u, k, WAVE)};
    st = lane & k ? stat_join(o, st) : stat_join(st, o);
  }
  if (c.n > WAVE) cand_cut(c, top, lane);  // (many equal logits, or segments with rising bounds)
  if (lane < AHEAD) c.list[c.n + lane] = 0;  // (no key: the ranking reads AHEAD at a time)
  if (lane == 0) {
    stats[wave] = st;
    counts[wave] = c.n;
  }
  __syncthreads();
  st = stat_join(stat_join(stats[0], stats[1]), stat_join(stats[2], stats[3]));
  int n = 0;
  for (int w = 0; w < WAVES; ++w) n += counts[w];
  n = min(n, top);
  if (top > 0 && lane < counts[wave]) {  // (at most a wave's 64 each)
    const u64 k = lists[wave][lane];
    int rank = 0;
    for (int o = 0; o < WAVES; ++o) rank += rank_of(k, lists[o], counts[o]);
    if (rank < top) best[rank] = k;
  }
  __syncthreads();
  if (a.S == 1) {
    row_results<LT>(a, r, st, best, n, given);
    return;
  }
  const size_t slot = (size_t)r * a.S + split;
  u64* keys = (u64*)a.ws + (size_t)r * a.S * top + split;
  float* sp = (float*)((u64*)a.ws + (size_t)a.rows * a.S * top) + slot * 4;
  if ((int)threadIdx.x < top) keys[(size_t)threadIdx.x * a.S] = (int)threadIdx.x < n ? best[threadIdx.x] : 0;
  if (threadIdx.x == 0) {
    sp[0] = st.m;
    sp[1] = st.s;
    sp[2] = st.u;
  }
}

// the splits of row blockIdx.x, one wave: the statistics joined in split order, the sorted lists merged
template <int LT>
__global__ __launch_bounds__(64) void logprobs_join_kernel(LogprobsP a) {
  __shared__ u64 best[LP_MAX_TOP], all[MAX_SPLITS * LP_MAX_TOP + AHEAD];
  const int r = blockIdx.x, lane = threadIdx.x;
  const float given = lane == 0 ? given_logit<LT>(a, r) : 0.f;
  const size_t slot = (size_t)r * a.S + lane;
  const float* sp = (const float*)((const u64*)a.ws + (size_t)a.rows * a.S * a.top) + slot * 4;
  Stat st{-3.402823466e38f, 0.f, 0.f};
  if (lane < a.S) st = Stat{sp[0], sp[1], sp[2]};
  for (int k = 32; k >= 1; k >>= 1) {
    const Stat o{__shfl_xor(st.m, k, WAVE), __shfl_xor(st.s, k, WAVE), __shfl_xor(st.u, k, WAVE)};
    st = lane & k ? stat_join(o, st) : stat_join(st, o);
  }
  int n = 0;
  if (a.top > 0) {
    // The splits' lists are sorted.  With `each` keys of a split counted, ceil(top / each) splits have that many keys
    // not below the ceil(top / each)-th largest of the splits' logits in that place: a bound that `top` keys reach,
    // and those of few splits pass.
    const int top = a.top, each = (top + a.S - 1) / a.S, lists = (top + each - 1) / each;
    // [key place][split]: a place's keys of all splits lie together
    const u64* keys = (const u64*)a.ws + (size_t)r * a.S * top + lane;
    const u64 at_each = lane < a.S ? keys[(each - 1) * a.S] : 0;
    const float bound = nth_lane(at_each != 0 ? key_value(at_each) : -INFINITY, lists);
    int m = 0;
    for (int t0 = 0; t0 < top; t0 += 4) {  // (four places requested at once; the first is seldom not enough)
      u64 k[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) k[i] = lane < a.S && t0 + i < top ? keys[(t0 + i) * a.S] : 0;
      bool any = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool in = k[i] != 0 && key_value(k[i]) >= bound;
        const unsigned long long b = __ballot(in);
        if (in) all[m + __popcll(b & ((1ull << lane) - 1))] = k[i];
        m += __popcll(b);
        any = b != 0;
      }
      if (!any) break;  // (lists are sorted: nothing behind the last place is wanted)
    }
    if (lane < AHEAD) all[m + lane] = 0;
    __syncthreads();
    for (int p = lane; p < m; p += WAVE) {
      const u64 k = all[p];
      const int rank = rank_of(k, all, m);
      if (rank < top) best[rank] = k;
    }
    n = min(m, top);
  }
  __syncthreads();
  row_results<LT>(a, r, st, best, n, given);
}

template <int LT>
hipError_t launch_lt(const LogprobsP& a, hipStream_t st) {
  hipLaunchKernelGGL(logprobs_kernel<LT>, dim3(a.rows, a.S), dim3(64 * WAVES), 0, st, a);
  if (const hipError_t e = hipGetLastError(); e != hipSuccess || a.S == 1) return e;
  hipLaunchKernelGGL(logprobs_join_kernel<LT>, dim3(a.rows), dim3(64), 0, st, a);
  return hipGetLastError();
}

}  // namespace

// Splits of a row: as many as make at most two workgroups to a compute unit, none below an iteration of each wave (us with
// one / two / four / eight to a unit, 64 rows of 151936 float32: 24.7 / 18.5 / 20.1 / 25.8; rounded up, 300 and 400 rows
// take 48.9 and 62.6 instead of 44.3 and 50.7).  None where they spare a wave no more than eleven iterations: joining them
// costs a launch, and each has to find its alternatives.  us, split / whole: one row of 5000 logits 13.6 / 9.7, of 33001
// 13.8 / 12.4, of 65001 12.9 / 15.9; 100 rows of 50001 17.8 / 15.9, of 90001 20.4 / 21.1; 200 rows of 65001 22.6 / 18.0, of
// 151936 35.9 / 39.8.
int logprobs_splits(const LogprobsP& a, int cus) {
  const int its = (a.vocab + WAVES * CHUNK - 1) / (WAVES * CHUNK);
  const int S = std::max(1, std::min({2 * cus / a.rows, its, MAX_SPLITS}));
  return (long long)its * (S - 1) <= 11ll * S ? 1 : S;
}
size_t logprobs_bytes(const LogprobsP& a) { return a.S > 1 ? (size_t)a.rows * a.S * (8 * a.top + 16) : 0; }

hipError_t launch_logprobs(const LogprobsP& a, hipStream_t st) {
  if (a.type == LT_BF16) return launch_lt<LT_BF16>(a, st);
  if (a.type == LT_F16) return launch_lt<LT_F16>(a, st);
  return launch_lt<LT_F32>(a, st);
}

}  // namespace fdllm
