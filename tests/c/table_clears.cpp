// How the rows of a table's gradient that have no token are shared out over workgroups (octex_amd/csrc/table.hpp), for tables
// of any size: prints "ok", or the first one whose launch would not fit.
#include "../../octex_amd/csrc/table.hpp"

#include <cstdio>

using namespace cuvs::neighbors::octex::detail;

int main()
{
  constexpr int64_t kMostRows = (int64_t{1} << 31) - 1, kMemory = int64_t{288} << 30;
  constexpr int64_t kMostGroups = ((int64_t{1} << 32) - 1) / 256 - (int64_t{1} << 21);  // beside those that sum
  for (int64_t bytes = 2; bytes <= int64_t{4} << 24; bytes += bytes < 70000 ? 2 : bytes / 3) {
    const int64_t most = std::min(kMostRows, kMemory / bytes);
    for (int64_t left = 1;; left = std::min(left * 2, most)) {
      const int64_t rows = rows_to_clear(left, bytes), groups = (left + rows - 1) / rows;
      if (rows < 1 || rows > kClearRows || groups > kMostGroups) {
        std::printf("%lld rows of %lld bytes: %lld a workgroup, %lld workgroups\n", static_cast<long long>(left),
                    static_cast<long long>(bytes), static_cast<long long>(rows), static_cast<long long>(groups));
        return 1;
      }
      if (left == most) break;
    }
  }
  std::puts("ok");
  return 0;
}
