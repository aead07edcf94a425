// Where a paged call's rows, pages and keys are: every index that comes from device memory (row starts, lengths, page
// numbers) passes through here before it becomes an address.  No GPU header, so that the CPU can check it
// (tests/paged_index_check.cpp).
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define FD_BOTH __host__ __device__ __forceinline__
#else
#define FD_BOTH inline
#endif

namespace fdllm {

// first row and number of rows of sequence b: inside [0, rows) and at most max_rows, whatever row_start holds
struct RowSpan { int first, n; };
FD_BOTH RowSpan seq_span(const int32_t* row_start, int rows, int max_rows, int b) {
  long long first = (long long)b * max_rows, n = max_rows;
  if (row_start != nullptr) {
    first = row_start[b];
    n = (long long)row_start[b + 1] - first;
    n = n < max_rows ? n : max_rows;
  }
  if (first < 0 || first >= rows) return RowSpan{0, 0};
  n = n < rows - first ? n : rows - first;
  return RowSpan{(int)first, (int)(n > 0 ? n : 0)};
}

// The sequence that row r of a call belongs to, the last whose rows do not start behind it, by halving (ascending row_start;
// others give some number of [-1, nseq]).
FD_BOTH int seq_of_row(const int32_t* row_start, int nseq, int r) {
  int lo = 0, hi = nseq + 1;  // row_start[< lo] <= r < row_start[>= hi]
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (row_start[mid] <= r) lo = mid + 1;
    else hi = mid;
  }
  return lo - 1;
}

// entry j of a sequence's row of the page table: -1 where it has none or a number that is no page
FD_BOTH int page_at(const int32_t* row, int width, int num_pages, long long j) {
  if (j < 0 || j >= width) return -1;
  const int p = row[j];
  return p >= 0 && p < num_pages ? p : -1;
}

// Page jj (from 0) of those that n rows from position `start` touch, of 1 << shift positions: j its place in the
// sequence, its slots [w0, w1) are written (none: w0 >= w1), slot s by the sequence's row s - rel; its first `live` slots
// held something before (live positions of the sequence), and some of those stay where `keeps`.
struct PageSpan { long long j, rel; int w0, w1, live; bool keeps; };
FD_BOTH PageSpan page_span(int start, int n, long long live, int jj, int shift) {
  PageSpan s{0, 0, 0, 0, 0, false};
  if (start < 0 || n <= 0) return s;
  const long long page = 1ll << shift, end = (long long)start + n;
  s.j = (start >> shift) + (long long)jj;
  const long long p0 = s.j << shift;
  s.rel = start - p0;
  if (p0 >= end) return s;
  s.w0 = (int)(s.rel > 0 ? s.rel : 0);
  s.w1 = (int)(end - p0 < page ? end - p0 : page);
  s.live = (int)(live <= p0 ? 0 : live - p0 < page ? live - p0 : page);
  s.keeps = s.live > 0 && (s.w0 > 0 || s.live > s.w1);
  return s;
}
// the most pages that `rows` consecutive positions touch
FD_BOTH long long pages_touched(int rows, int page) { return ((long long)rows + 2 * page - 2) / page; }

// Row i of a sequence's n attends keys [0, key_limit) of the first lk (its length, no more than its table holds).
FD_BOTH int key_limit(int kv_len, int lk, int n, int i, int mask_block) {
  if (mask_block <= 0) return lk;
  if (kv_len < n - i) return 0;  // before the first position
  const unsigned pos = (unsigned)kv_len - (unsigned)(n - i), end = pos / (unsigned)mask_block * (unsigned)mask_block + (unsigned)mask_block;
  return end < (unsigned)lk ? (int)end : lk;
}

// the workgroups that take a call's pages, one for each of a sequence's
FD_BOTH long long append_wgs(int nseq, int max_rows, int page) { return nseq * pages_touched(max_rows, page); }
// Queries [rows][heads][128], ldq elements from row to row, written over by a contiguous result: only where they are contiguous
// too (a single row is) does a workgroup write what it alone has read.
FD_BOTH bool place_fits(const void* q, long long ldq, int rows, int heads, const void* out) {
  return q == nullptr || q != out || rows <= 1 || ldq == heads * 128ll;
}
// a launch's x axis holds fewer than 2^32 threads
FD_BOTH bool grid_fits(long long wgs, int threads) { return wgs >= 0 && wgs <= 0xffffffffll / threads; }
// positions of a table: a tile that lies ahead of the last one still has a position of 31 bits
FD_BOTH bool table_fits(int pages_per_seq, int page) { return (long long)pages_per_seq * page <= 0x7fffffffll - 4096; }

}  // namespace fdllm
