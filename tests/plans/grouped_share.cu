// Host-side check of grouped_share: every tile of a group gets rows, none more than a tile holds, in multiples of what an MMA takes, also for groups
// whose rows and tiles together are more than an int holds.  Exit status 0 if all of that holds.
#include <cstdio>
#include "../../fgms_b200/csrc/grouped_umma.cuh"

int main() {
  long long checked = 0, bad = 0;
  for (int unit : {16, 32})
    for (int tile = 2 * unit; tile <= 256; tile *= 2) {
      const auto check = [&](long long n) {
        const int rows = (int)n, count = (int)((n + tile - 1) / tile), share = fgms::grouped_share(rows, count, unit);
        const long long behind = (long long)(count - 1) * share;  // the last tile's first row
        if (share < 1 || share > tile || share % unit || behind >= n || behind + share < n) {
          if (++bad < 10) std::printf("%d rows, %d tiles of at most %d: shares of %d\n", rows, count, tile, share);
        }
        ++checked;
      };
      for (long long n = 1; n <= 5000; ++n) check(n);
      for (long long most = 0x7fffffffll - 1024, n = most; n > most - 3000; --n) check(n);
      for (long long n = 5000; n < 0x7fffffffll - 1024; n += n / 1000) check(n);
    }
  std::printf("%lld checked, %lld bad\n", checked, bad);
  return bad == 0 ? 0 : 1;
}
