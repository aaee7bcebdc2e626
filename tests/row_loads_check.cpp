// Every pack that is loaded for a row of n elements lies inside the row, and puts its elements where they belong.
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <vector>

#include "../bayesiannetwork_amd/csrc/row_loads.h"

template <typename U>
int check() {
  constexpr int V = 16 / (int)sizeof(U);
  for (int n = V; n <= 140; ++n) {
    std::vector<U> row(n);
    for (int i = 0; i < n; ++i) row[i] = (U)(1000 + i);
    for (int from = 0; from < n + 64; ++from) {
      const int start = bn_rows::pack_start(from, n, V);
      if (start < 0 || start + V > n || start > from) return std::printf("n %d from %d: loads %d..%d\n", n, from, start, start + V), 1;
      bn_rows::Raw raw;
      std::memcpy(raw.w, row.data() + start, 16);
      raw = bn_rows::moved_down<sizeof(U)>(raw, from - start);
      U got[V];
      std::memcpy(got, raw.w, 16);
      for (int j = 0; j < V; ++j)
        if (from + j < n && got[j] != row[from + j]) return std::printf("n %d from %d: element %d\n", n, from, j), 1;
    }
  }
  return 0;
}

int main() { return check<uint16_t>() || check<uint32_t>() || check<uint64_t>(); }
