// Launch interfaces of the paged 4-bit cache (paged4.hip).
#pragma once
#include "paged.hpp"
#include "rotate.hpp"

namespace fdllm {

// One layer's pages: K and V [num_pages][nkv][page][64], two e2m1 codes a byte, the lower dim in the lower half.
// K: one power of two, its exponent + 127 (255: NaN), for each block of 32 dims, [num_pages][nkv][page / 16][4][4][4] by
// (slot / 16, slot % 4, block, slot / 4 % 4).  A lane of the attention's first product, whose rows are slots and whose steps
// are blocks, so finds the scales of its four products in one word, which is how the matrix instruction takes them.
// V: one bf16 scale for each slot and head, [num_pages][nkv][page]; it goes on the probabilities.
// Every row stands by itself: a row is written without reading another.
struct Paged4P {
  uint8_t *k, *v, *ks;
  uint16_t* vs;
  int num_pages, page, shift, nkv;  // page = 1 << shift
  const int32_t* table; long long table_ld; int table_w;  // table_w pages per sequence
};

// whether the append's and the read's launches hold so many rows
bool paged4_rows_fit(int rows);

struct Paged4AppendP {
  Paged4P c;
  SeqRowsP s;
  TurnP t;
  const uint16_t *q, *k, *v; long long ldq, ldk, ldv;  // elements from row to row; q null: no queries
  uint16_t* q_out;                                     // [rows][nq][128]
  const uint16_t *q_norm, *k_norm;                     // [128]; null: no norm
  int nq;
  const int32_t *start, *pos;                          // per sequence: first written position, rotation (null: start)
};
hipError_t launch_paged4_append(int dt, const Paged4AppendP& a, hipStream_t st);

struct Paged4ReadP {
  Paged4P c;
  SeqRowsP s;
  const int32_t* start;                      // per sequence: position of its first row
  uint16_t *k, *v; long long ldk, ldv;       // results, elements from row to row
};
hipError_t launch_paged4_read(int dt, const Paged4ReadP& a, hipStream_t st);

// As PagedAttnP (whose plan for the joining launch it carries), over 4-bit pages.
struct Paged4AttnP {
  Paged4P c;
  SeqRowsP s;
  const uint16_t* q; long long ldq;
  uint16_t* out;
  int nq;
  unsigned div24;
  const int32_t* kv_len;
  int mask_block;
  float scale_log2e;
  int max_len, tiles16, waves, S, group_wgs, cuts;  // waves of a workgroup
  int one_round;  // whether all workgroups are resident at once
  float* part;
};
bool paged4_attn_plan(Paged4AttnP& a, int cus);
size_t paged4_attn_floats(const Paged4AttnP& a);
hipError_t launch_paged4_attn(int dt, const Paged4AttnP& a, hipStream_t st);

}  // namespace fdllm
