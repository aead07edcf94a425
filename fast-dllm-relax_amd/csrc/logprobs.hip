// Log probabilities of given tokens, with each row's entropy and most probable alternatives, in one pass over the
// logits.
#include <algorithm>

#include "common.hpp"
#include "logprobs.hpp"

namespace fdllm {

namespace {

typedef unsigned long long u64;
constexpr int EPL = 16;                        // elements a lane takes per iteration
constexpr int CHUNK = EPL * WAVE;              // elements a wave takes per iteration
constexpr int LIST = LP_MAX_TOP * (EPL + 1);   // a wave's candidates: the best so far and one iteration's at most
constexpr int WAVES = 4;
constexpr int MAX_SPLITS = 64;
constexpr float LOG2E = 1.44269504088896340736f;

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
  const float ea = expf(da), eb = expf(db);
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

// The wave's candidates in LDS: the `top` best logits seen are always among its `n` keys; logits above `t` enter it.
// t is about the top-th largest of the lanes' largest logits so far: that many logits are at least as large, all of
// them in the list.  It is renewed when the logits seen have doubled, so each doubling brings about top more candidates (24 of
// 20: as many logits as 20 of 64 lanes hold the largest of), without any ordering until the end.  A wave takes its
// elements in ascending order of their indices between iterations, so a later one equal to t has the higher index and
// stays out.
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

// One iteration's elements above c.t, and not below `from`, into the list: x[i] has index idx(i), -inf where there is none;
// mx is the lane's largest.
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

// the results of a row whose statistics and `n` best keys (in order, LDS) are complete
template <int LT>
__device__ __forceinline__ void row_results(const LogprobsP& a, int r, Stat st, const u64* best, int n) {
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
      else if (id >= 0) v = none ? nan : (one<LT>((const typename Elem<LT>::type*)a.logits + r * a.ld + id) - lse_m) - ls;
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
template <int LT>
__global__ __launch_bounds__(64 * WAVES) void logprobs_kernel(LogprobsP a) {
  typedef typename Elem<LT>::type T;
  constexpr int E = Elem<LT>::E, UPL = EPL / E;  // units per lane and iteration
  __shared__ u64 lists[WAVES][LIST];
  __shared__ u64 best[LP_MAX_TOP];
  __shared__ Stat stats[WAVES];
  __shared__ int counts[WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = blockIdx.x, split = blockIdx.y;
  const T* row = (const T*)a.logits + r * a.ld;
  const int head = min(a.vocab, (int)(((16 - ((uintptr_t)row & 15)) & 15) / sizeof(T)));
  const int units = (a.vocab - head) / E, tail0 = head + units * E;
  const u32x4* body = reinterpret_cast<const u32x4*>(row + head);
  const int parts = a.S * WAVES, part = split * WAVES + wave;
  const int per = (units + parts - 1) / parts;
  const int u0 = min(units, part * per), u1 = min(units, u0 + per);
  Cand c{lists[wave], 0, -INFINITY};
  Stat st{-3.402823466e38f, 0.f, 0.f};
  const int top = a.top;
  float lane_max = -INFINITY;  // (st.m starts above -inf)
  int seen = 0, renew = 1;
  auto take = [&](const float (&x)[EPL], auto idx) {
    float mx = x[0];
#pragma unroll
    for (int i = 1; i < EPL; ++i) mx = fmaxf(mx, x[i]);
    if (top > 0) {
      lane_max = fmaxf(lane_max, mx);
      float from = -INFINITY;
      if (++seen == renew) {
        renew *= 2;
        from = nth_lane(lane_max, top);
      }
      if (__any(mx > c.t && mx >= from)) cand_take(c, x, mx, from, idx, top, lane);
      c.t = fmaxf(c.t, from);
    }
    stat_take(st, x, mx);
  };
  auto edge = [&](int from, int n) {  // n < 64 elements from index `from`, one per lane
    float x[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) x[i] = -INFINITY;
    if (lane < n) x[0] = one<LT>(row + from + lane);
    take(x, [&](int) { return from + lane; });
  };
  if (part == 0 && head > 0) edge(0, head);
  // the next iteration's units are on their way while one is worked on
  u32x4 next[UPL];
  auto fetch = [&](int u) {
#pragma unroll
    for (int i = 0; i < UPL; ++i) {
      const int at = u + 64 * i + lane;
      if (at < u1) next[i] = body[at];
    }
  };
  fetch(u0);
  for (int u = u0; u < u1; u += UPL * WAVE) {
    float x[EPL];
#pragma unroll
    for (int i = 0; i < UPL; ++i) {
      unpack<LT>(next[i], x + i * E);
      if (u + 64 * i + lane >= u1) {
#pragma unroll
        for (int e = 0; e < E; ++e) x[i * E + e] = -INFINITY;
      }
    }
    fetch(u + UPL * WAVE);
    take(x, [&](int i) { return head + (u + 64 * (i / E) + lane) * E + i % E; });
  }
  if (part == parts - 1 && tail0 < a.vocab) edge(tail0, a.vocab - tail0);
  // the wave's lanes, in a fixed order
  for (int k = 32; k >= 1; k >>= 1) {
    const Stat o{__shfl_xor(st.m, k, WAVE), __shfl_xor(st.s, k, WAVE), __shfl_xor(st.u, k, WAVE)};
    st = lane & k ? stat_join(o, st) : stat_join(st, o);
  }
  if (top > 0 && c.n > WAVE) {
    // what the final bound leaves; more than a lane's one each only where many logits are equal
    const float t = nth_lane(lane_max, top);
    int n = 0;
    for (int p0 = 0; p0 < c.n; p0 += WAVE) {
      const u64 k = p0 + lane < c.n ? c.list[p0 + lane] : 0;
      const bool in = k != 0 && key_value(k) >= t;
      const unsigned long long b = __ballot(in);
      __builtin_amdgcn_wave_barrier();
      if (in) c.list[n + __popcll(b & ((1ull << lane) - 1))] = k;
      __builtin_amdgcn_wave_barrier();
      n += __popcll(b);
    }
    c.n = n;
    if (c.n > WAVE) cand_cut(c, top, lane);
  }
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
    for (int o = 0; o < WAVES; ++o)
      for (int q = 0; q < counts[o]; ++q) rank += lists[o][q] > k ? 1 : 0;
    if (rank < top) best[rank] = k;
  }
  __syncthreads();
  if (a.S == 1) {
    row_results<LT>(a, r, st, best, n);
    return;
  }
  const size_t slot = (size_t)r * a.S + split;
  u64* keys = (u64*)a.ws + slot * top;
  float* sp = (float*)((u64*)a.ws + (size_t)a.rows * a.S * top) + slot * 4;
  if ((int)threadIdx.x < top) keys[threadIdx.x] = (int)threadIdx.x < n ? best[threadIdx.x] : 0;
  if (threadIdx.x == 0) {
    sp[0] = st.m;
    sp[1] = st.s;
    sp[2] = st.u;
  }
}

// the splits of row blockIdx.x, one wave: the statistics joined in split order, the sorted lists merged
template <int LT>
__global__ __launch_bounds__(64) void logprobs_join_kernel(LogprobsP a) {
  __shared__ u64 best[LP_MAX_TOP], all[MAX_SPLITS * LP_MAX_TOP];
  const int r = blockIdx.x, lane = threadIdx.x;
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
    // not below the ceil(top / each)-th largest of the splits' keys in that place: a bound that `top` keys reach, and
    // those of few splits pass.
    const int top = a.top, each = (top + a.S - 1) / a.S, lists = (top + each - 1) / each;
    const u64* keys = (const u64*)a.ws + slot * top;
    const u64 bound = nth_lane_key(lane < a.S ? keys[each - 1] : 0, lists, lane);
    int m = 0;
    for (int t = 0; t < top; ++t) {
      const u64 k = lane < a.S ? keys[t] : 0;
      const bool in = k != 0 && k >= bound;
      const unsigned long long b = __ballot(in);
      if (b == 0) break;
      if (in) all[m + __popcll(b & ((1ull << lane) - 1))] = k;
      m += __popcll(b);
    }
    __syncthreads();
    for (int p = lane; p < m; p += WAVE) {
      const u64 k = all[p];
      int rank = 0;
      for (int q = 0; q < m; ++q) rank += all[q] > k ? 1 : 0;
      if (rank < top) best[rank] = k;
    }
    n = min(m, top);
  }
  __syncthreads();
  row_results<LT>(a, r, st, best, n);
}

template <int LT>
hipError_t launch_lt(const LogprobsP& a, hipStream_t st) {
  hipLaunchKernelGGL(logprobs_kernel<LT>, dim3(a.rows, a.S), dim3(64 * WAVES), 0, st, a);
  if (const hipError_t e = hipGetLastError(); e != hipSuccess || a.S == 1) return e;
  hipLaunchKernelGGL(logprobs_join_kernel<LT>, dim3(a.rows), dim3(64), 0, st, a);
  return hipGetLastError();
}

}  // namespace

int logprobs_splits(const LogprobsP& a, int cus) {
  const int want = (2 * cus + a.rows - 1) / a.rows, most = (a.vocab + WAVES * CHUNK - 1) / (WAVES * CHUNK);
  return std::max(1, std::min({want, most, MAX_SPLITS}));
}
size_t logprobs_bytes(const LogprobsP& a) { return a.S > 1 ? (size_t)a.rows * a.S * (8 * a.top + 16) : 0; }

hipError_t launch_logprobs(const LogprobsP& a, hipStream_t st) {
  if (a.type == LT_BF16) return launch_lt<LT_BF16>(a, st);
  if (a.type == LT_F16) return launch_lt<LT_F16>(a, st);
  return launch_lt<LT_F32>(a, st);
}

}  // namespace fdllm
