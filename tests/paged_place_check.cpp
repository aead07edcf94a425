// Checks where a paged call's result may lie over its queries (csrc/paged_index.hpp): wherever the rule says yes, no row of the
// result covers an element of another row's queries; compiled and run by tests/test_paged.py.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "paged_index.hpp"

using namespace fdllm;

int main() {
  std::vector<unsigned short> mem(64 * 40 * 128);
  bool refused = false;
  for (int heads : {1, 4, 12})
    for (int rows : {0, 1, 2, 3, 40})
      for (long long ld : {heads * 128ll, heads * 128ll + 8, heads * 128ll + 512, 2ll * heads * 128}) {
        bool clear = true;
        for (int r = 0; r < rows; ++r)      // the result's row r ...
          for (int o = 0; o < rows; ++o) {  // ... and the queries' row o, from the same place
            const long long a = (long long)r * heads * 128, b = o * ld;
            if (r != o && a < b + heads * 128 && b < a + heads * 128) clear = false;
            if (r == o && a != b) clear = false;
          }
        if (place_fits(mem.data(), ld, rows, heads, mem.data()) != clear) {
          std::printf("%d heads, %d rows, stride %lld: %d\n", heads, rows, ld, (int)clear);
          return 1;
        }
        refused |= !clear;
        if (!place_fits(mem.data(), ld, rows, heads, mem.data() + 64 * 20 * 128) || !place_fits(nullptr, ld, rows, heads, nullptr)) return 1;
      }
  if (!refused) return 1;
  std::puts("ok");
  return 0;
}
