// Checks the index arithmetic of the paged cache (csrc/paged_index.hpp) against loops over positions, with hostile device
// values among them; compiled and run by tests/test_paged.py.
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "paged_index.hpp"

using namespace fdllm;

#define CHECK(x)                                               \
  do {                                                         \
    if (!(x)) {                                                \
      std::printf("line %d: %s\n", __LINE__, #x);              \
      std::exit(1);                                            \
    }                                                          \
  } while (0)

static const int hostile[] = {INT_MIN, INT_MIN + 1, -1000, -1, 0, 1, 5, 31, 32, 33, 100, 1 << 20, INT_MAX - 64, INT_MAX - 1, INT_MAX};

int main() {
  // rows: always inside [0, rows), at most max_rows, and the given ones where they are sane
  for (int rows : {1, 2, 33, 1000})
    for (int max_rows : {1, 2, 32, 1000}) {
      for (int a : hostile)
        for (int b : hostile) {
          const int32_t rs[2] = {a, b};
          const RowSpan s = seq_span(rs, rows, max_rows, 0);
          CHECK(s.n >= 0 && s.n <= max_rows && s.first >= 0 && s.first + s.n <= rows);
          if (a >= 0 && a <= b && b <= rows && b - a <= max_rows && a < rows) CHECK(s.first == a && s.n == b - a);
          if (b <= a) CHECK(s.n == 0);
        }
      for (int b = 0; (b + 1) * max_rows <= rows; ++b) {
        const RowSpan s = seq_span(nullptr, rows, max_rows, b);
        CHECK(s.first == b * max_rows && s.n == max_rows);
      }
    }
  // pages
  for (int width : {1, 3})
    for (int pages : {1, 7})
      for (int p : hostile)
        for (long long j : {-1ll, 0ll, 1ll, 2ll, 3ll, 1ll << 27, LLONG_MAX / 2}) {
          const std::vector<int32_t> row(width, p);
          const int got = page_at(row.data(), width, pages, j);
          CHECK(got == (j >= 0 && j < width && p >= 0 && p < pages ? p : -1));
        }
  // slots of every page that rows touch, against the positions one by one
  for (int shift : {4, 5, 6, 7}) {
    const int page = 1 << shift;
    for (int start : {0, 1, 15, 16, 31, 32, 63, 127, 128, 1000})
      for (int n : {1, 2, 16, 17, 32, 33, 128, 129, 300})
        for (long long live : {0ll, 1ll, (long long)start, start + 1ll, (long long)start + n, start + n + 5ll, 5000ll, -3ll, (long long)INT_MIN}) {
          int seen = 0;
          const long long np = pages_touched(n, page);
          for (int jj = 0; jj < np + 2; ++jj) {
            const PageSpan s = page_span(start, n, live, jj, shift);
            if (s.w0 >= s.w1) continue;
            CHECK(jj < np);
            CHECK(s.w0 >= 0 && s.w1 <= page && s.live >= 0 && s.live <= page);
            bool keeps = false;
            for (int k = 0; k < page; ++k) {
              const long long p = (s.j << shift) + k;
              const bool is_new = p >= start && p < start + n, is_live = p < live;
              CHECK(is_new == (k >= s.w0 && k < s.w1));
              CHECK(is_live == (k < s.live));
              if (is_new) {
                CHECK(k - s.rel == p - start && k - s.rel >= 0 && k - s.rel < n);
                ++seen;
              }
              keeps |= is_live && !is_new;
            }
            CHECK(keeps == s.keeps);
          }
          CHECK(seen == n);
        }
    for (int start : hostile)
      for (int n : {0, 1, 40})
        for (int jj : {0, 1, 2}) {
          const PageSpan s = page_span(start, n, start, jj, shift);
          CHECK(s.w0 >= 0 && s.w1 <= page);
          if (start < 0 || n == 0) CHECK(s.w0 >= s.w1);
          if (s.w0 < s.w1) CHECK(s.w0 - s.rel >= 0 && s.w1 - 1 - s.rel < n && s.j >= 0);
        }
  }
  // keys
  for (int kv : hostile)
    for (int cap : {16, 4096})
      for (int n : {1, 7, 300})
        for (int i : {0, 3, 299})
          for (int block : {0, 1, 32, INT_MAX}) {
            const int lk = kv < 0 ? 0 : kv < cap ? kv : cap;
            const int lim = key_limit(kv, lk, n, i, block);
            CHECK(lim >= 0 && lim <= lk);
            const long long pos = (long long)kv - n + i;
            for (int key = 0; key < (lk < 400 ? lk : 400); ++key) {
              const bool sees = block == 0 || (pos >= 0 && key / block <= pos / block);
              CHECK((key < lim) == sees);
            }
          }
  // launches and tables
  for (int nseq : {1, 64, 65535})
    for (int rows : {1, 100, 1 << 20, INT_MAX})
      for (int page : {16, 128}) {
        const long long wgs = append_wgs(nseq, rows, page);
        CHECK(wgs >= (long long)nseq * (((long long)rows + page - 1) / page) && wgs <= (long long)nseq * ((long long)rows / page + 2));
        CHECK(grid_fits(wgs, 8 * page) == (wgs * 8 * page < 1ll << 32));
      }
  CHECK(!grid_fits(-1, 256));
  CHECK(table_fits(1, 16) && !table_fits(INT_MAX, 128) && !table_fits(INT_MAX / 16, 16));
  for (int page : {16, 32, 64, 128}) {
    const int most = (INT_MAX - 4096) / page;
    CHECK(table_fits(most, page) && !table_fits(most + 1, page));
    // the last tile, and those asked for ahead of it
    CHECK((long long)(most * page + 63) / 64 * 64 + 64 * 8 + 63 < INT_MAX);
  }
  std::puts("ok");
  return 0;
}
