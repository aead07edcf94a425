// Norms of queries and keys for each head, with their rotation by position, in one pass.
#include "rotate_device.hpp"

namespace fdllm {

namespace {

constexpr int HG = 4;  // heads that a workgroup takes of its rows: they share the sines and cosines

// A workgroup takes blockDim.x / 8 rows of up to HG heads (blockIdx.y: groups of the queries' heads, then of the keys').
// All is read before anything of the same head is written, so a result may lie over its input.
template <int DT, bool INTER>
__global__ __launch_bounds__(256) void rotate_heads_kernel(RotateP a) {
  const int u = threadIdx.x & 7;
  const long long row = (long long)blockIdx.x * (blockDim.x >> 3) + (threadIdx.x >> 3);
  const int qg = a.q ? (a.nq + HG - 1) / HG : 0, y = (int)blockIdx.y;
  const bool keys = y >= qg;
  const int heads = keys ? a.nkv : a.nq, h0 = HG * (keys ? y - qg : y);
  const uint16_t *in = keys ? a.k : a.q, *norm = keys ? a.k_norm : a.q_norm;
  uint16_t* out = keys ? a.k_out : a.q_out;
  const long long ld = keys ? a.ldk : a.ldq, ldo = keys ? a.ldko : a.ldqo;
  if (row >= a.rows) return;  // (the eight threads of a row together)
  const HeadPart p = head_part(a.t, u);
  const long long pos = a.pos ? a.pos[row] : a.pos0 + row;
  float x[HG][16], w[16];
#pragma unroll
  for (int h = 0; h < HG; ++h)
    if (h0 + h < heads) load_part<DT>(in + row * ld + (h0 + h) * HD, p, x[h]);
  if (norm) {
    load_part<DT>(norm, p, w);
#pragma unroll
    for (int h = 0; h < HG; ++h)
      if (h0 + h < heads) norm_part(x[h], w, a.t.eps);
  }
  if (p.turned) {
    const float gain = (float)a.t.gain;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float sn, cs;
      turn_sincos((double)pos * a.t.turn[8 * u + e], sn, cs);
      sn *= gain;
      cs *= gain;
#pragma unroll
      for (int h = 0; h < HG; ++h) turn_pair<INTER>(x[h], e, sn, cs);
    }
  }
#pragma unroll
  for (int h = 0; h < HG; ++h) {
    if (h0 + h >= heads) break;
    uint16_t* dst = out + row * ldo + (h0 + h) * HD;
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

// rows of few: workgroups of one wave, spread over the compute units
int rotate_threads(int rows) { return rows <= 8 ? 64 : 256; }

}  // namespace

bool rotate_fits(const RotateP& a) { return grid_fits(((long long)a.rows + 7) / 8, 64); }

hipError_t launch_rotate_heads(int dt, const RotateP& a, hipStream_t st) {
  const int threads = rotate_threads(a.rows), rows = threads / 8;
  const dim3 grid((a.rows + rows - 1) / rows, (a.q ? (a.nq + HG - 1) / HG : 0) + (a.k ? (a.nkv + HG - 1) / HG : 0));
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, st, a); };
  if (dt == DT_BF16) a.t.inter ? launch(rotate_heads_kernel<DT_BF16, true>) : launch(rotate_heads_kernel<DT_BF16, false>);
  else a.t.inter ? launch(rotate_heads_kernel<DT_F16, true>) : launch(rotate_heads_kernel<DT_F16, false>);
  return hipGetLastError();
}

}  // namespace fdllm
