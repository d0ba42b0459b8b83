// Dropout and the residual's addition: out = residual + keep ? x factor : 0, and the gradient of x, keep ? g factor : 0, with the same lots (row_values.cuh).
// A dropped value is gone whatever it was: NaN too.
#pragma once
#include "row_values.cuh"

namespace fgms {

constexpr int DROP_THREADS = 256, DROP_BLOCKS = 4;  // of an SM
constexpr int DROP_AT_ONCE = 2;  // chunks whose loads are on their way together, while their lots are drawn

struct DropoutParams {
  const void *x, *residual;  // residual: or null
  void* out;
  long long rows, x_pitch, residual_pitch, out_pitch;
  int width;
  bool x_vec, residual_vec, out_vec;
  DropParams drop;
  int alone;  // see GmsParams
};

// The row `step` rows further, and the next one: n_rows where there is none, and from n_rows on.  (Rows and steps together may leave an int; 2^31 - 1 rows and one more do, but
// for a number without a sign.)
__host__ __device__ __forceinline__ int drop_row_after(int row, int step, int n_rows) { return row < n_rows - step ? row + step : n_rows; }
__host__ __device__ __forceinline__ int drop_next_row(int row, int n_rows) { return (int)min((unsigned)row + 1u, (unsigned)n_rows); }

// A chunk is a thread's; threads go on by the whole grid, whose width in rows and columns is divided once, and so are the ways through the tensors.  What
// bounds it are instructions as much as memory: 228 a chunk of eight at first (masks of bits, products for addresses, conversions one by one), 168 now, of
// which the lots are some 70: 32768 x 2048 in bf16 with a residual 72 us, its gradient 64, 85 and 64 % of the measured copy rate.  SOME: something is dropped.
template <typename T, bool BACKWARD, bool SOME>
__global__ void __launch_bounds__(DROP_THREADS, DROP_BLOCKS) dropout_kernel(const __grid_constant__ DropoutParams p) {
  umma::griddep_wait();
  if (!p.alone) umma::griddep_launch_dependents();
  const DropKey key = drop_key(BACKWARD ? p.drop.used : p.drop.state);
  const uint32_t below = drop_below(p.drop.threshold);
  const unsigned per_row = ((unsigned)p.width + ROW_CHUNK - 1) / ROW_CHUNK;
  const unsigned long long at = (unsigned long long)blockIdx.x * DROP_THREADS + threadIdx.x, step = (unsigned long long)gridDim.x * DROP_THREADS;
  const int step_row = (int)(step / per_row);
  const unsigned step_chunk = (unsigned)(step - (unsigned long long)step_row * per_row);
  const int n_rows = (int)p.rows;
  const unsigned first_row = (unsigned)(at / per_row);
  unsigned chunk = (unsigned)(at - (unsigned long long)first_row * per_row);
  int row = first_row < (unsigned)n_rows ? (int)first_row : n_rows;
  // from one chunk to the next, and what is more where the next one is a row further
  struct Way {
    long long at, step, wrap;
    __device__ __forceinline__ Way(long long pitch, int row, unsigned chunk, int step_row, unsigned step_chunk, unsigned per_row)
        : at(row * pitch + (long long)chunk * ROW_CHUNK), step(step_row * pitch + (long long)step_chunk * ROW_CHUNK), wrap(pitch - (long long)per_row * ROW_CHUNK) {}
  };
  Way x_way(p.x_pitch, row, chunk, step_row, step_chunk, per_row), add_way(p.residual_pitch, row, chunk, step_row, step_chunk, per_row),
      out_way(p.out_pitch, row, chunk, step_row, step_chunk, per_row);
  while (__any_sync(0xffffffffu, row < n_rows)) {
    int rows[DROP_AT_ONCE], cols[DROP_AT_ONCE], there[DROP_AT_ONCE];
    T* out[DROP_AT_ONCE];
    RowRaw<T> x[DROP_AT_ONCE], add[DROP_AT_ONCE];
#pragma unroll
    for (int i = 0; i < DROP_AT_ONCE; ++i) {
      cols[i] = (int)(chunk * ROW_CHUNK);
      there[i] = row < n_rows ? p.width - cols[i] : 0;
      rows[i] = row;
      out[i] = static_cast<T*>(p.out) + out_way.at;
      x[i] = row_load(static_cast<const T*>(p.x) + x_way.at, there[i], p.x_vec);
      if (!BACKWARD && p.residual) add[i] = row_load(static_cast<const T*>(p.residual) + add_way.at, there[i], p.residual_vec);
      row = drop_row_after(row, step_row, n_rows);
      chunk += step_chunk;
      x_way.at += x_way.step;
      out_way.at += out_way.step;
      if (!BACKWARD) add_way.at += add_way.step;
      if (chunk >= per_row) {
        chunk -= per_row;
        row = drop_next_row(row, n_rows);
        x_way.at += x_way.wrap;
        out_way.at += out_way.wrap;
        if (!BACKWARD) add_way.at += add_way.wrap;
      }
    }
    DropLots lots[DROP_AT_ONCE];
    if (SOME) {
#pragma unroll
      for (int i = 0; i < DROP_AT_ONCE; ++i) lots[i] = drop_lots(key, (uint32_t)cols[i] / ROW_CHUNK, (uint32_t)rows[i]);
    }
#pragma unroll
    for (int i = 0; i < DROP_AT_ONCE; ++i) {
      float y[ROW_CHUNK];
      row_values(x[i], y);
      if (SOME) {
#pragma unroll
        for (int e = 0; e < ROW_CHUNK; ++e) y[e] = lots[i].kept(e, below) ? y[e] * p.drop.factor : 0.f;
      }
      if (!BACKWARD && p.residual) {
        float r[ROW_CHUNK];
        row_values(add[i], r);
#pragma unroll
        for (int e = 0; e < ROW_CHUNK; ++e) y[e] += r[e];
      }
      row_store(out[i], y, there[i], p.out_vec, cols[i] == 0);
    }
  }
  if (!BACKWARD) drop_count(p.drop);
}

}  // namespace fgms
