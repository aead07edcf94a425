// Norms of queries and keys for each head, with their rotation by position, in one pass.
#include "rotate_device.hpp"

namespace fdllm {

namespace {

constexpr int HG = 4;  // heads that a workgroup takes of its rows: they share the sines and cosines

// A workgroup takes blockDim.x / 8 rows of up to HG heads (blockIdx.y: groups of the queries' heads, then of the keys').
template <int DT, bool INTER>
__global__ __launch_bounds__(256) void rotate_heads_kernel(RotateP a) {
  const long long row = (long long)blockIdx.x * (blockDim.x >> 3) + (threadIdx.x >> 3);
  if (row >= a.rows) return;  // (the eight threads of a row together)
  const int qg = a.q ? (a.nq + HG - 1) / HG : 0, y = (int)blockIdx.y;
  const double pos = (double)(a.pos ? a.pos[row] : a.pos0 + row);
  if (y < qg) turn_heads<DT, INTER, HG>(a.t, threadIdx.x & 7, pos, a.q + row * a.ldq, a.q_norm, a.q_out + row * a.ldqo, HG * y, a.nq);
  else turn_heads<DT, INTER, HG>(a.t, threadIdx.x & 7, pos, a.k + row * a.ldk, a.k_norm, a.k_out + row * a.ldko, HG * (y - qg), a.nkv);
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
