// Launch interfaces of the heads' norms and rotation (rotate.hip), and the rotation's plan, which the paged 4-bit cache
// (paged4.hip) shares.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fdllm {

// What a head of 128 goes through: with `w`, x (mean x^2 + eps)^-1/2 w; then its first `rot` dims (a multiple of 16) are
// turned in pairs, pair j by position x turn[j] turns, times gain.  Pair j: dims (j, j + rot / 2), or (2 j, 2 j + 1) where
// `inter`.
struct TurnP {
  double turn[64];
  double gain;
  int rot, inter;
  float eps;
};

struct RotateP {
  TurnP t;
  const uint16_t *q, *k; long long ldq, ldk;  // elements from row to row; null: none
  uint16_t *q_out, *k_out; long long ldqo, ldko;
  const uint16_t *q_norm, *k_norm;            // [128]; null: no norm
  int nq, nkv, rows;
  const int32_t* pos; long long pos0;         // position of row r: pos[r], or pos0 + r
};
hipError_t launch_rotate_heads(int dt, const RotateP& a, hipStream_t st);
// whether its launch holds so many rows
bool rotate_fits(const RotateP& a);

}  // namespace fdllm
