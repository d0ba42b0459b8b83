// Dropout and the residual's addition: out = residual + keep ? x factor : 0, and the gradient of x, keep ? g factor : 0, with the same lots (row_values.cuh).
// A dropped value is gone whatever it was: NaN too.
#pragma once
#include "row_values.cuh"

namespace fgms {

constexpr int DROP_THREADS = 256;
constexpr int DROP_AT_ONCE = 4;  // chunks whose loads are on their way together

struct DropoutParams {
  const void *x, *residual;  // residual: or null
  void* out;
  long long rows, x_pitch, residual_pitch, out_pitch;
  int width;
  bool x_vec, residual_vec, out_vec;
  DropParams drop;
  int alone;  // see GmsParams
};

// A chunk is a thread's; threads go on by the whole grid, whose width in rows and columns is divided once.
template <typename T, bool BACKWARD>
__global__ void __launch_bounds__(DROP_THREADS) dropout_kernel(const __grid_constant__ DropoutParams p) {
  umma::griddep_wait();
  if (!p.alone) umma::griddep_launch_dependents();
  const DropKey key = drop_key(BACKWARD ? p.drop.used : p.drop.state);
  const unsigned per_row = ((unsigned)p.width + ROW_CHUNK - 1) / ROW_CHUNK;
  const unsigned long long at = (unsigned long long)blockIdx.x * DROP_THREADS + threadIdx.x, step = (unsigned long long)gridDim.x * DROP_THREADS;
  const long long step_row = (long long)(step / per_row);
  const unsigned step_chunk = (unsigned)(step - (unsigned long long)step_row * per_row);
  long long row = (long long)(at / per_row);
  unsigned chunk = (unsigned)(at - (unsigned long long)row * per_row);
  const auto next = [&] {
    row += step_row;
    chunk += step_chunk;
    if (chunk >= per_row) {
      chunk -= per_row;
      ++row;
    }
  };
  while (row < p.rows) {
    long long rows[DROP_AT_ONCE];
    unsigned chunks[DROP_AT_ONCE];
    RowRaw<T> x[DROP_AT_ONCE], add[DROP_AT_ONCE];
    int n = 0;
#pragma unroll
    for (int i = 0; i < DROP_AT_ONCE; ++i) {
      rows[i] = row;
      chunks[i] = chunk;
      if (row < p.rows) {
        const int col = (int)(chunk * ROW_CHUNK), there = p.width - col;
        x[i] = row_load(static_cast<const T*>(p.x) + row * p.x_pitch + col, there, p.x_vec);
        if (!BACKWARD && p.residual) add[i] = row_load(static_cast<const T*>(p.residual) + row * p.residual_pitch + col, there, p.residual_vec);
        n = i + 1;
        next();
      }
    }
#pragma unroll
    for (int i = 0; i < DROP_AT_ONCE; ++i) {
      if (i >= n) continue;
      const int col = (int)(chunks[i] * ROW_CHUNK);
      const uint32_t keep = drop_keep(key, chunks[i], (uint32_t)rows[i], p.drop.threshold);
      float y[ROW_CHUNK];
#pragma unroll
      for (int e = 0; e < ROW_CHUNK; ++e) {
        y[e] = keep >> e & 1u ? row_value(x[i], e) * p.drop.factor : 0.f;
        if (!BACKWARD && p.residual) y[e] += row_value(add[i], e);
      }
      row_store(static_cast<T*>(p.out) + rows[i] * p.out_pitch + col, y, p.width - col, p.out_vec);
    }
  }
  if (!BACKWARD) drop_count(p.drop);
}

}  // namespace fgms
