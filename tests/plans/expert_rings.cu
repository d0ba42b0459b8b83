// The rings of a layer of experts for every number of tokens that an expert may have: all that is copied and all that is read lies inside them.
#include <cstdio>
#include "../../fgms_b200/csrc/expert_layer.cuh"

int main() {
  using namespace fgms;
  const int bytes = 232448 - 1024 - EL_FIXED_BYTES;  // the most there is, less what is aligned away and what stands in front
  for (int most = 1; most <= EL_MAX_TOKENS; ++most) {
    const ElRings r = el_rings(bytes, most);
    bool ok = r.stages >= 6 && r.stages <= EL_MAX_STAGES && r.x_stages >= 2 && r.x_stages <= EL_MAX_STAGES;
    const int x0 = r.stages * EL_TILE_BYTES;
    for (int n = 1; n <= most; ++n)              // of the expert at hand
      for (int rest = 0; rest < 2; ++rest) {     // h, and its remainders
        const int first = x0 + (r.x_stages - 1) * r.x_bytes + rest * r.x_bytes / 2;
        const int copied = first + (n - 1) * EL_X_PITCH + EL_K * 2;
        int read = 0;
        for (int j = 0; j * 8 < n; j += 2) read = first + (j * 8 + 15) * EL_X_PITCH + 7 * 32 + 32;  // the last warp's 16 values of the last row
        ok = ok && copied <= bytes && read <= bytes && copied <= x0 + r.x_stages * r.x_bytes;
      }
    if (!ok) {
      printf("most %d: %d stages, %d of rows of %d bytes do not fit %d\n", most, r.stages, r.x_stages, r.x_bytes, bytes);
      return 1;
    }
  }
  printf("ok\n");
  return 0;
}
