// Checks how a row of a call finds its sequence (csrc/paged_index.hpp) against a loop over the sequences, with hostile row
// starts among them; compiled and run by tests/test_paged4.py.
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "paged_index.hpp"

using namespace fdllm;

int main() {
  unsigned state = 7;
  auto rnd = [&](int n) { return (int)((state = state * 1664525u + 1013904223u) >> 8) % n; };
  for (int nseq : {1, 2, 3, 63, 64, 65, 511, 512, 1000})
    for (int most : {0, 1, 5}) {
      std::vector<int32_t> rs{rnd(3)};
      for (int b = 0; b < nseq; ++b) rs.push_back(rs.back() + rnd(most + 1));
      for (int r = -2; r < rs.back() + 4; ++r) {
        int want = -1;
        for (int b = 0; b <= nseq; ++b)
          if (rs[b] <= r) want = b;
        const int got = seq_of_row(rs.data(), nseq, r);
        if (got != want) {
          std::printf("row %d of %d sequences: %d, not %d\n", r, nseq, got, want);
          return 1;
        }
        // its rows are the ones of seq_span
        if (got >= 0 && got < nseq) {
          const RowSpan s = seq_span(rs.data(), rs.back() + 4, 1000, got);
          if ((r >= s.first && r < s.first + s.n) != (r < rs[got + 1])) return 1;
        }
      }
    }
  const int hostile[] = {INT_MIN, -1, 0, 1, 7, INT_MAX - 1, INT_MAX};
  for (int a : hostile)
    for (int b : hostile)
      for (int c : hostile)
        for (int r : hostile) {
          const int32_t rs[] = {a, b, c};
          const int got = seq_of_row(rs, 2, r);
          if (got < -1 || got > 2) return 1;
        }
  std::printf("ok\n");
}
