// Launch interfaces of the paged 8-bit cache (paged.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fdllm {

// ---- the paged cache ---------------------------------------------------------------------------
// One layer's pages: K [num_pages][nkv][page][128] and V [num_pages][nkv][128][page] in e4m3, one fp32 scale per
// page and kv head for each ([num_pages][nkv]); the value a byte stands for is e4m3(byte) x scale.  Position p of
// sequence b is slot p % page of page table[b table_ld + p / page].  V is stored with its slots innermost: the
// attention's second product sums over keys, and its MFMA operand (8 consecutive keys of one dim per lane) is
// then a plain load, as K's (8 consecutive dims of one key) is.
// Every index that comes from device memory is checked before it is used: a page outside [0, num_pages) is neither
// read nor written.
struct PagedP {
  uint8_t *k, *v;
  float *ks, *vs;
  int num_pages, page, shift, nkv;  // page = 1 << shift
  const int32_t* table; long long table_ld; int table_w;  // table_w pages per sequence
};

// The rows of a ragged batch: sequence b has rows [row_start[b], row_start[b + 1]) of the call's `rows`, at most
// max_rows of them; row_start null: sequence b has rows [b max_rows, (b + 1) max_rows).
struct SeqRowsP {
  const int32_t* row_start;
  int rows, nseq, max_rows;
};

struct PagedAppendP {
  PagedP c;
  SeqRowsP s;
  const uint16_t *q, *k, *v; long long ldq, ldk, ldv;  // elements from row to row; q null: no queries
  uint16_t* q_out;                                     // [rows][nq][128]
  int nq;
  const int32_t *start, *live, *pos;                   // per sequence: first written position, live rows before, rotation
  double turn1, turn8, turn16, turn32;                 // theta^(-1/64), ^(-8/64), ...: pair i turns theta^(-i/64) per position
};
hipError_t launch_paged_append(int dt, const PagedAppendP& a, hipStream_t st);

struct PagedAttnP {
  PagedP c;
  SeqRowsP s;
  const uint16_t* q; long long ldq;
  uint16_t* out;             // [rows][nq][128]
  int nq;
  unsigned div24;            // 2^24 / G + 1, G = nq / nkv: x / G = x div24 >> 24 for x < G + 64
  const int32_t* kv_len;     // per sequence: attended keys [0, kv_len)
  int mask_block;            // 0: none; else row at position p attends keys below (p / mask_block + 1) mask_block
  float scale_log2e;         // log2(e) / sqrt(128)
  int max_len;               // no sequence is longer (the key split is planned for it)
  int tiles16;               // tiles of 16 flattened rows that a workgroup takes
  int S;                     // key splits
  int group_wgs, cuts;       // the grid: see paged_attn_kernel
  float* part;               // S > 1: partial outputs [S][rows nq][128], then (m, l) [S][rows nq][2]
};
// plans a call (its shapes are set) on a device of `cus` compute units: the key splits and the grid; false: too large for a
// launch.  Then the floats of workspace it needs.
bool paged_attn_plan(PagedAttnP& a, int cus);
size_t paged_attn_floats(const PagedAttnP& a);
hipError_t launch_paged_attn(int dt, const PagedAttnP& a, hipStream_t st);

}  // namespace fdllm
