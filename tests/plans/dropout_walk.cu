// The ways of dropout's threads over rows and chunks, against the same in 64 bits: every chunk once, and nothing behind the last row, however many rows there are.
#include <climits>
#include <cstdio>
#include "../../fgms_b200/csrc/dropout.cuh"

int main() {
  using namespace fgms;
  for (const long long rows : {1ll, 2ll, 1000ll, (long long)INT_MAX - 2, (long long)INT_MAX - 1, (long long)INT_MAX})
    for (unsigned per_row = 1; per_row <= 9; ++per_row)
      for (const int sms : {1, 84, 148}) {
        const unsigned long long step = (unsigned long long)DROP_THREADS * DROP_BLOCKS * sms, chunks = (unsigned long long)rows * per_row;
        const int step_row = (int)(step / per_row);
        const unsigned step_chunk = (unsigned)(step - (unsigned long long)step_row * per_row);
        for (unsigned long long thread = 0; thread < step; thread += 1 + step / 1000) {
          // from the last few steps before the end on, and eight steps behind it
          unsigned long long at = thread;
          if (chunks > 4 * step + thread) at += (chunks - thread) / step * step - 3 * step;
          int row = at / per_row < (unsigned long long)rows ? (int)(at / per_row) : (int)rows;
          unsigned chunk = (unsigned)(at % per_row);
          for (int behind = 0; behind < 8; at += step) {
            const bool there = at < chunks;
            if (there ? row != (int)(at / per_row) || chunk != at % per_row : row != (int)rows) {
              printf("%lld rows of %u chunks, %d SMs, thread %llu: row %d, chunk %u at %llu\n", rows, per_row, sms, thread, row, chunk, at);
              return 1;
            }
            behind += !there;
            row = drop_row_after(row, step_row, (int)rows);
            chunk += step_chunk;
            if (chunk >= per_row) {
              chunk -= per_row;
              row = drop_next_row(row, (int)rows);
            }
          }
        }
      }
  printf("ok\n");
  return 0;
}
