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

// A chunk is a thread's; threads go on by the whole grid, whose width in rows and columns is divided once.
template <typename T, bool BACKWARD>
__global__ void __launch_bounds__(DROP_THREADS, DROP_BLOCKS) dropout_kernel(const __grid_constant__ DropoutParams p) {
  umma::griddep_wait();
  if (!p.alone) umma::griddep_launch_dependents();
  const DropKey key = drop_key(BACKWARD ? p.drop.used : p.drop.state);
  const unsigned per_row = ((unsigned)p.width + ROW_CHUNK - 1) / ROW_CHUNK;
  const unsigned long long at = (unsigned long long)blockIdx.x * DROP_THREADS + threadIdx.x, step = (unsigned long long)gridDim.x * DROP_THREADS;
  const long long step_row = (long long)(step / per_row);
  const unsigned step_chunk = (unsigned)(step - (unsigned long long)step_row * per_row);
  long long row = (long long)(at / per_row);
  unsigned chunk = (unsigned)(at - (unsigned long long)row * per_row);
  while (__any_sync(0xffffffffu, row < p.rows)) {
    long long rows[DROP_AT_ONCE];
    int cols[DROP_AT_ONCE], there[DROP_AT_ONCE];
    RowRaw<T> x[DROP_AT_ONCE], add[DROP_AT_ONCE];
#pragma unroll
    for (int i = 0; i < DROP_AT_ONCE; ++i) {
      cols[i] = (int)(chunk * ROW_CHUNK);
      there[i] = row < p.rows ? p.width - cols[i] : 0;
      rows[i] = row < p.rows ? row : 0;
      x[i] = row_load(static_cast<const T*>(p.x) + rows[i] * p.x_pitch + cols[i], there[i], p.x_vec);
      if (!BACKWARD && p.residual) add[i] = row_load(static_cast<const T*>(p.residual) + rows[i] * p.residual_pitch + cols[i], there[i], p.residual_vec);
      row += step_row;
      chunk += step_chunk;
      if (chunk >= per_row) {
        chunk -= per_row;
        ++row;
      }
    }
    uint32_t keep[DROP_AT_ONCE];
#pragma unroll
    for (int i = 0; i < DROP_AT_ONCE; ++i) keep[i] = drop_keep(key, (uint32_t)cols[i] / ROW_CHUNK, (uint32_t)rows[i], p.drop.threshold);
#pragma unroll
    for (int i = 0; i < DROP_AT_ONCE; ++i) {
      float y[ROW_CHUNK];
#pragma unroll
      for (int e = 0; e < ROW_CHUNK; ++e) {
        y[e] = keep[i] >> e & 1u ? row_value(x[i], e) * p.drop.factor : 0.f;
        if (!BACKWARD && p.residual) y[e] += row_value(add[i], e);
      }
      row_store(static_cast<T*>(p.out) + rows[i] * p.out_pitch + cols[i], y, there[i], p.out_vec, cols[i] == 0);
    }
  }
  if (!BACKWARD) drop_count(p.drop);
}

}  // namespace fgms
