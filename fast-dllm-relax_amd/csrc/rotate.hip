// Norms of queries and keys for each head, with their rotation by position, in one pass.
#include "rotate_device.hpp"

namespace fdllm {

namespace {

// A workgroup takes eight rows of one head (blockIdx.y: the queries' heads, then the keys').  Sharing the sines and cosines
// among heads gains nothing (us, four heads and 256 threads / one: a row 4.3 / 2.7, 1024 rows 4.8 / 3.7, 8192 rows 13.1 / 12.9,
// near a copy's time): a launch is the workgroups' chain of instructions, or memory's.
template <int DT, bool INTER>
__global__ __launch_bounds__(64) void rotate_heads_kernel(RotateP a) {
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 3);
  if (row >= a.rows) return;  // (the eight threads of a row together)
  const int nq = a.q ? a.nq : 0, y = (int)blockIdx.y, u = threadIdx.x & 7;
  const double pos = (double)(a.pos ? a.pos[row] : a.pos0 + row);
  if (y < nq) turn_heads<DT, INTER, 1>(a.t, u, pos, a.q + row * a.ldq, a.q_norm, a.q_out + row * a.ldqo, y, nq);
  else turn_heads<DT, INTER, 1>(a.t, u, pos, a.k + row * a.ldk, a.k_norm, a.k_out + row * a.ldko, y - nq, a.nkv);
}

}  // namespace

bool rotate_fits(const RotateP& a) { return grid_fits(((long long)a.rows + 7) / 8, 64); }

hipError_t launch_rotate_heads(int dt, const RotateP& a, hipStream_t st) {
  const dim3 grid((unsigned)(((long long)a.rows + 7) / 8), (a.q ? a.nq : 0) + (a.k ? a.nkv : 0));
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(64), 0, st, a); };
  if (dt == DT_BF16) a.t.inter ? launch(rotate_heads_kernel<DT_BF16, true>) : launch(rotate_heads_kernel<DT_BF16, false>);
  else a.t.inter ? launch(rotate_heads_kernel<DT_F16, true>) : launch(rotate_heads_kernel<DT_F16, false>);
  return hipGetLastError();
}

}  // namespace fdllm
