// Root-mean-square norm of rows with the residual's addition, and its gradient.
//
//   h = residual + drop(x)        r = 1 / sqrt(mean(h^2) + eps)        y = h r w
//   gradient, with n = h r and g = dy w:
//   dh = r (g - n mean(g n)) + dsum        dx = drop'(dh)        dresidual = dh        dw = sum over the rows of dy n
//
// Sums, statistics and everything in between are fp32; h is rounded once where it is stored, and y comes from the h before that.  An output in 8 bits is
// round(y 127 / a) with the scale a / 127, a = max |y| of the row: symmetric, so that a product needs no offsets.  A row whose largest value is
// below 2^-100 is zeros with a scale of zero; a row that holds a value which is not finite has a scale of NaN and codes of zero, so that a product with
// it is NaN.
//
// One pass: a row's values stay in registers from their load to their store, CH chunks of eight a thread.  Rows of up to 256 values are a warp's each, wider
// ones a block's (of the gradient, up to 512, two warps' of eight such pairs in a block, so that the blocks' shares of the weight's gradient
// stay few), with one exchange through shared memory for each reduction.  16384 x 4096 in bf16 with the residual 87 us, 94 % of the measured copy rate: memory.  With
// dropout the lots (70 of 300 instructions for eight values) and the loads, one row after the other, bound it: 8192 x 2048 34 us forward, 43 the gradient, 5 to
// 7 the sum of the blocks' shares of the weight's.  (A pass of all three through autograd takes 77 to 119 us: at this size the host may set the pace.)
#pragma once
#include "row_values.cuh"

namespace fgms {

constexpr int NORM_MAX_THREADS = 1024;
constexpr int NORM_WARP_ROWS = 4;   // rows (warps) of a block where a row is a warp's
constexpr int NORM_GRAD_ROWS = 8;   // rows that a block of the gradient has at a time where a row is a warp's or two

struct NormParams {
  const void *x, *residual, *weight;  // residual: or null; weight: null without a norm (norm = 0)
  void *out, *sum;                    // sum: or null
  float *scale, *rstd;                // scale: of an output in 8 bits; rstd: or null
  long long rows, x_pitch, residual_pitch, out_pitch, sum_pitch;
  int width, norm;
  bool x_vec, residual_vec, out_vec, sum_vec, weight_vec;
  float eps, inverse_width;
  DropParams drop;
  int alone;  // see GmsParams
};

// |x| as an unsigned number: larger values are larger numbers, and NaN is above them all
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sum over the threads of a row; `part`: 32 words of shared memory that no reduction shortly before has used.
template <bool WARP>
__device__ __forceinline__ float row_sum(float v, float* part) {
  v = warp_sum(v);
  if (WARP) return v;
  const int lane = threadIdx.x & 31, warps = (int)blockDim.x >> 5;
  if (lane == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum(lane < warps ? part[lane] : 0.f);
}
template <bool WARP>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* part) {
  v = __reduce_max_sync(0xffffffffu, v);
  if (WARP) return v;
  const int lane = threadIdx.x & 31, warps = (int)blockDim.x >> 5;
  if (lane == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  return __reduce_max_sync(0xffffffffu, lane < warps ? part[lane] : 0u);
}

// Of the gradient: `GROUP` warps a row, 0 the whole block.
template <int GROUP>
__device__ __forceinline__ float group_sum(float v, float* part) {
  if (GROUP <= 1) return row_sum<GROUP == 1>(v, part);
  v = warp_sum(v);
  const int warp = (int)threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) part[warp] = v;
  asm volatile("barrier.cta.sync %0, %1;" ::"r"(1 + warp / GROUP), "n"(32 * (GROUP ? GROUP : 1)) : "memory");
  return part[warp / 2 * 2] + part[warp / 2 * 2 + 1];  // (of two)
}

// T: rows; W: the weight; CH: chunks a thread; WARP: a row is a warp's; EIGHT: the output is codes of 8 bits
template <typename T, typename W, int CH, bool WARP, bool EIGHT, bool DROP, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 512 ? (CH == 1 ? 3 : 2) : 1) rms_norm_kernel(const __grid_constant__ NormParams p) {
  __shared__ float parts[4][32];
  umma::griddep_wait();
  if (!p.alone) umma::griddep_launch_dependents();
  DropKey key;
  if (DROP) key = drop_key(p.drop.state);
  const uint32_t below = drop_below(p.drop.threshold);
  const int per_row = WARP ? 32 : (int)blockDim.x, thread = WARP ? (int)threadIdx.x & 31 : (int)threadIdx.x;
  const long long rows_at_once = WARP ? (long long)gridDim.x * NORM_WARP_ROWS : (long long)gridDim.x;
  int turn = 0;  // a row's reductions use other words than the last one's, which a slower warp may still read
  for (long long row = WARP ? (long long)blockIdx.x * NORM_WARP_ROWS + (threadIdx.x >> 5) : (long long)blockIdx.x; row < p.rows; row += rows_at_once) {
    RowRaw<T> raw[CH], add[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * per_row + thread) * ROW_CHUNK, there = p.width - col;
      raw[c] = row_load(static_cast<const T*>(p.x) + row * p.x_pitch + col, there, p.x_vec);
      if (p.residual) add[c] = row_load(static_cast<const T*>(p.residual) + row * p.residual_pitch + col, there, p.residual_vec);
    }
    float h[CH][ROW_CHUNK], sum = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int chunk = c * per_row + thread, col = chunk * ROW_CHUNK;
      DropLots lots;
      if (DROP) lots = drop_lots(key, (uint32_t)chunk, (uint32_t)row);
      row_values(raw[c], h[c]);
      if (DROP) {
#pragma unroll
        for (int e = 0; e < ROW_CHUNK; ++e) h[c][e] = lots.kept(e, below) ? h[c][e] * p.drop.factor : 0.f;
      }
      if (p.residual) {
        float r[ROW_CHUNK];
        row_values(add[c], r);
#pragma unroll
        for (int e = 0; e < ROW_CHUNK; ++e) h[c][e] += r[e];
      }
#pragma unroll
      for (int e = 0; e < ROW_CHUNK; ++e) sum += h[c][e] * h[c][e];
      if (p.sum) row_store(static_cast<T*>(p.sum) + row * p.sum_pitch + col, h[c], p.width - col, p.sum_vec, chunk == 0);
    }
    float r = 1.f;
    if (p.norm) {
      r = 1.f / sqrtf(row_sum<WARP>(sum, parts[turn]) * p.inverse_width + p.eps);
      if (p.rstd && thread == 0) p.rstd[row] = r;
    }
    uint32_t largest = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * per_row + thread) * ROW_CHUNK, there = p.width - col;
      if (p.norm && there > 0) {
        float w[ROW_CHUNK];
        const W* from = static_cast<const W*>(p.weight) + col;
        if (p.weight_vec && there >= ROW_CHUNK) {  // every row reads it again: from L1
          RowRaw<W> v;
#pragma unroll
          for (int q = 0; q < (int)sizeof(W) / 2; ++q) *reinterpret_cast<uint4*>(v.w + 4 * q) = __ldg(reinterpret_cast<const uint4*>(from) + q);
          row_values(v, w);
        } else {
#pragma unroll
          for (int e = 0; e < ROW_CHUNK; ++e) w[e] = e < there ? to_f32(from[e]) : 0.f;
        }
#pragma unroll
        for (int e = 0; e < ROW_CHUNK; ++e) h[c][e] = h[c][e] * r * w[e];
      }
      if (EIGHT) {
#pragma unroll
        for (int e = 0; e < ROW_CHUNK; ++e) largest = max(largest, e < there ? magnitude(h[c][e]) : 0u);
      } else {
        row_store(static_cast<T*>(p.out) + row * p.out_pitch + col, h[c], there, p.out_vec, col == 0);
      }
    }
    if (EIGHT) {
      const float a = __uint_as_float(row_max<WARP>(largest, reinterpret_cast<uint32_t*>(parts[turn + 1])));
      const bool finite = a < __uint_as_float(0x7f800000u), some = finite && a >= 7.88860905e-31f;  // 2^-100
      const float to_code = some ? 127.f / a : 0.f;
      if (thread == 0) p.scale[row] = finite ? (some ? a / 127.f : 0.f) : __uint_as_float(0x7fc00000u);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int col = (c * per_row + thread) * ROW_CHUNK, there = p.width - col;
        int8_t* to = static_cast<int8_t*>(p.out) + row * p.out_pitch + col;
        uint32_t code[ROW_CHUNK];
#pragma unroll
        for (int e = 0; e < ROW_CHUNK; ++e) code[e] = some ? (uint32_t)__float2int_rn(h[c][e] * to_code) & 0xffu : 0u;
        if (p.out_vec && there >= ROW_CHUNK) {
          *reinterpret_cast<uint2*>(to) = make_uint2(code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24, code[4] | code[5] << 8 | code[6] << 16 | code[7] << 24);
        } else {
#pragma unroll
          for (int e = 0; e < ROW_CHUNK; ++e)
            if (e < there) to[e] = (int8_t)code[e];
        }
      }
    }
    if (!WARP) turn ^= 2;
  }
  if (DROP) drop_count(p.drop);
}

struct NormGradParams {
  const void *dy, *sum, *x, *residual, *dsum, *weight;  // h: read from sum, or with x computed again; residual, dsum: or null
  const float* rstd;
  void *dx, *dresidual;  // either may be null
  float* parts;          // [blocks][width]: what each block's rows add to the weight's gradient, or null
  long long rows, dy_pitch, sum_pitch, residual_pitch, dsum_pitch, dx_pitch, dresidual_pitch;  // sum_pitch: x's
  int width;
  bool dy_vec, sum_vec, residual_vec, dsum_vec, dx_vec, dresidual_vec, weight_vec;
  float inverse_width;
  DropParams drop;
  int alone;
};

// The block's rows one after the other, their share of the weight's gradient in registers until the last one: 1024 threads an SM with 64 registers each, where the
// next row's values on their way meanwhile and half as many threads took 58 us instead of 43 (8192 x 2048, bf16, with dropout).
// FROM_X: h = residual + drop(x) once more, unrounded, for rows in 16 bits: from the h that was stored the weight's gradient is off by 0.0024 of its norm in bf16, and 0.0003 in
// fp16, whatever the weight's type; so an fp32 weight has it to 2^-22, and one of the rows' type to its own rounding, 0.0016 and 0.0002.  A tensor more to read: 8192 x 2048
// without dropout 32.7 us instead of 27.0, 16384 x 4096 120 instead of 105.
template <typename T, typename W, int CH, int GROUP, bool DROP, bool FROM_X, int THREADS>
__global__ void __launch_bounds__(THREADS, CH == 1 ? 1024 / THREADS : 1) rms_norm_grad_kernel(const __grid_constant__ NormGradParams p) {
  __shared__ float parts[2][32];
  __shared__ float share[GROUP ? NORM_GRAD_ROWS : 1][GROUP ? 32 * GROUP * CH * ROW_CHUNK : 1];
  umma::griddep_wait();
  if (!p.alone) umma::griddep_launch_dependents();
  DropKey key;
  if (DROP) key = drop_key(p.drop.used);
  const uint32_t below = drop_below(p.drop.threshold);
  constexpr int EACH = GROUP ? 32 * GROUP : 1;  // threads of a row
  const int per_row = GROUP ? EACH : (int)blockDim.x, thread = GROUP ? (int)threadIdx.x % EACH : (int)threadIdx.x, group = GROUP ? (int)threadIdx.x / EACH : 0;
  const long long rows_at_once = GROUP ? (long long)gridDim.x * NORM_GRAD_ROWS : (long long)gridDim.x;
  float dw[CH][ROW_CHUNK];
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int e = 0; e < ROW_CHUNK; ++e) dw[c][e] = 0.f;
  RowRaw<T> dy[CH], h[CH], add[CH], extra[CH];
  int turn = 0;
  for (long long row = GROUP ? (long long)blockIdx.x * NORM_GRAD_ROWS + group : (long long)blockIdx.x; row < p.rows; row += rows_at_once) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * per_row + thread) * ROW_CHUNK, there = p.width - col;
      dy[c] = row_load(static_cast<const T*>(p.dy) + row * p.dy_pitch + col, there, p.dy_vec);
      h[c] = row_load(static_cast<const T*>(FROM_X ? p.x : p.sum) + row * p.sum_pitch + col, there, p.sum_vec);
      if (FROM_X && p.residual) add[c] = row_load(static_cast<const T*>(p.residual) + row * p.residual_pitch + col, there, p.residual_vec);
      if (p.dsum) extra[c] = row_load(static_cast<const T*>(p.dsum) + row * p.dsum_pitch + col, there, p.dsum_vec);
    }
    const float r = __ldg(p.rstd + row);
    DropLots lots[CH];
    float n[CH][ROW_CHUNK], g[CH][ROW_CHUNK], dot = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int chunk = c * per_row + thread, col = chunk * ROW_CHUNK, there = p.width - col;
      if (DROP) lots[c] = drop_lots(key, (uint32_t)chunk, (uint32_t)row);
      row_values(h[c], n[c]);
      if (FROM_X) {
        if (DROP) {
#pragma unroll
          for (int e = 0; e < ROW_CHUNK; ++e) n[c][e] = lots[c].kept(e, below) ? n[c][e] * p.drop.factor : 0.f;
        }
        if (p.residual) {
          float v[ROW_CHUNK];
          row_values(add[c], v);
#pragma unroll
          for (int e = 0; e < ROW_CHUNK; ++e) n[c][e] += v[e];
        }
      }
      RowRaw<W> raw;
      const W* from = static_cast<const W*>(p.weight) + col;
      if (p.weight_vec && there >= ROW_CHUNK) {  // every row reads it again: from L1
#pragma unroll
        for (int q = 0; q < (int)sizeof(W) / 2; ++q) {
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(from) + q);
          raw.w[4 * q] = v.x; raw.w[4 * q + 1] = v.y; raw.w[4 * q + 2] = v.z; raw.w[4 * q + 3] = v.w;
        }
      } else {
        raw = row_load(from, there, false);
      }
      float w[ROW_CHUNK];
      row_values(raw, w);
      row_values(dy[c], g[c]);
#pragma unroll
      for (int e = 0; e < ROW_CHUNK; ++e) {
        n[c][e] *= r;
        dw[c][e] += g[c][e] * n[c][e];
        g[c][e] *= w[e];
        dot += g[c][e] * n[c][e];
      }
    }
    const float mean = group_sum<GROUP>(dot, parts[turn]) * p.inverse_width;
    if (GROUP != 1) turn ^= 1;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int chunk = c * per_row + thread, col = chunk * ROW_CHUNK, there = p.width - col;
      float dh[ROW_CHUNK];
#pragma unroll
      for (int e = 0; e < ROW_CHUNK; ++e) dh[e] = r * (g[c][e] - n[c][e] * mean);
      if (p.dsum) {
        float v[ROW_CHUNK];
        row_values(extra[c], v);
#pragma unroll
        for (int e = 0; e < ROW_CHUNK; ++e) dh[e] += v[e];
      }
      if (p.dresidual) row_store(static_cast<T*>(p.dresidual) + row * p.dresidual_pitch + col, dh, there, p.dresidual_vec, chunk == 0);
      if (p.dx) {
        if (DROP) {
#pragma unroll
          for (int e = 0; e < ROW_CHUNK; ++e) dh[e] = lots[c].kept(e, below) ? dh[e] * p.drop.factor : 0.f;
        }
        row_store(static_cast<T*>(p.dx) + row * p.dx_pitch + col, dh, there, p.dx_vec, chunk == 0);
      }
    }
  }
  if (!p.parts) return;
  float* to = p.parts + (size_t)blockIdx.x * p.width;
  if (GROUP) {  // the block's groups in their order
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int e = 0; e < ROW_CHUNK; ++e) share[group][(c * per_row + thread) * ROW_CHUNK + e] = dw[c][e];
    __syncthreads();
    for (int col = (int)threadIdx.x; col < p.width; col += EACH * NORM_GRAD_ROWS) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < NORM_GRAD_ROWS; ++i) sum += share[i][col];
      to[col] = sum;
    }
  } else {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * per_row + thread) * ROW_CHUNK;
      if ((p.width & 3) == 0) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
          if (col + 4 * q < p.width) *reinterpret_cast<float4*>(to + col + 4 * q) = make_float4(dw[c][4 * q], dw[c][4 * q + 1], dw[c][4 * q + 2], dw[c][4 * q + 3]);
      } else {
#pragma unroll
        for (int e = 0; e < ROW_CHUNK; ++e)
          if (col + e < p.width) to[col + e] = dw[c][e];
      }
    }
  }
}

// The blocks' shares in their order, 32 columns a block: 32 rows of threads take every 32nd share each and are added up in their order.
constexpr int NORM_SHARES_Y = 32;
template <typename W>
__global__ void __launch_bounds__(32 * NORM_SHARES_Y) rms_norm_weight_grad_kernel(const float* __restrict__ parts, int n, int width, W* dw, int alone) {
  __shared__ float sums[NORM_SHARES_Y][32];
  umma::griddep_wait();
  if (!alone) umma::griddep_launch_dependents();
  const int col = (int)blockIdx.x * 32 + (threadIdx.x & 31), y = (int)threadIdx.x >> 5;
  float sum = 0.f;
  if (col < width) {
#pragma unroll 8
    for (int i = y; i < n; i += NORM_SHARES_Y) sum += __ldcg(parts + (size_t)i * width + col);
  }
  sums[y][threadIdx.x & 31] = sum;
  __syncthreads();
  if (y == 0 && col < width) {
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < NORM_SHARES_Y; ++i) sum += sums[i][threadIdx.x & 31];
    dw[col] = from_f32<W>(sum);
  }
}

// Threads that a row of a block gets with CH chunks each.
inline int norm_threads(int width, int ch) {
  const int chunks = (width + ROW_CHUNK - 1) / ROW_CHUNK;
  return ((chunks + ch - 1) / ch + 31) / 32 * 32;
}

template <typename T, typename W, int CH, bool WARP, bool EIGHT, int THREADS>
cudaError_t launch_rms_norm_as(const NormParams& p, cudaStream_t st, int sms) {
  const int threads = WARP ? 32 * NORM_WARP_ROWS : norm_threads(p.width, CH);
  const long long blocks = WARP ? (p.rows + NORM_WARP_ROWS - 1) / NORM_WARP_ROWS : p.rows;
  const long long at_once = (long long)sms * ((THREADS == 512 ? (CH == 1 ? 1536 : 1024) : 2048) / threads);
  const dim3 grid((unsigned)(blocks < at_once ? blocks : at_once));
  if (!EIGHT && p.drop.threshold > 0) return launch_pdl(rms_norm_kernel<T, W, CH, WARP, false, true, THREADS>, grid, threads, 0, st, p);
  return launch_pdl(rms_norm_kernel<T, W, CH, WARP, EIGHT, false, THREADS>, grid, threads, 0, st, p);
}
template <typename T, typename W, bool EIGHT>
cudaError_t launch_rms_norm(const NormParams& p, cudaStream_t st, int sms) {
  constexpr int WARPS = 32 * NORM_WARP_ROWS;
  if (p.width <= 256) return launch_rms_norm_as<T, W, 1, true, EIGHT, WARPS>(p, st, sms);
  // A warp with two chunks a lane, if nothing is dropped (23491 x 288 in fp16 12.4 us, two warps with one 18.9; with the lots of two chunks it has 103 registers).
  if (p.width <= 512 && p.drop.threshold == 0) return launch_rms_norm_as<T, W, 2, true, EIGHT, WARPS>(p, st, sms);
  // Few rows, or lots to draw: as many threads as there are chunks.
  const bool drop = p.drop.threshold > 0;
  if (p.width <= (p.rows < sms || drop ? 4096 : 2048)) return launch_rms_norm_as<T, W, 1, false, EIGHT, 512>(p, st, sms);
  if (p.width <= 8192 && p.rows < sms) return launch_rms_norm_as<T, W, 1, false, EIGHT, NORM_MAX_THREADS>(p, st, sms);
  if (p.width <= 8192) return launch_rms_norm_as<T, W, 2, false, EIGHT, 512>(p, st, sms);
  return launch_rms_norm_as<T, W, 4, false, EIGHT, NORM_MAX_THREADS>(p, st, sms);
}
constexpr int NORM_MAX_WIDTH = NORM_MAX_THREADS * 4 * ROW_CHUNK;

// What a gradient is cut into: the blocks each leave a share of the weight's gradient.
struct NormGradCut {
  int ch, group, threads, blocks;  // group: warps a row, 0 a block
};
inline NormGradCut norm_grad_cut(long long rows, int width, int sms) {
  NormGradCut c;
  c.group = width <= 256 ? 1 : width <= 512 ? 2 : 0;
  // as many threads as there are chunks, 64 registers each: 920 x 4448 in fp16 with its forward 37.6 us with two chunks a thread, 35.7 so
  c.ch = width <= 8192 ? 1 : width <= 16384 ? 2 : 4;
  c.threads = c.group ? 32 * c.group * NORM_GRAD_ROWS : norm_threads(width, c.ch);
  const long long blocks = c.group ? (rows + NORM_GRAD_ROWS - 1) / NORM_GRAD_ROWS : rows, at_once = (long long)sms * (c.threads <= 1024 ? 1024 / c.threads : 1);
  c.blocks = (int)(blocks < at_once ? blocks : at_once);
  return c;
}
template <typename T, typename W, int CH, int GROUP, int THREADS>
cudaError_t launch_rms_norm_grad_as(const NormGradParams& p, const NormGradCut& cut, cudaStream_t st) {
  const dim3 grid((unsigned)cut.blocks);
  const bool drop = p.drop.threshold > 0;
  if constexpr (sizeof(T) == 2) {
    if (p.x)
      return drop ? launch_pdl(rms_norm_grad_kernel<T, W, CH, GROUP, true, true, THREADS>, grid, cut.threads, 0, st, p)
                  : launch_pdl(rms_norm_grad_kernel<T, W, CH, GROUP, false, true, THREADS>, grid, cut.threads, 0, st, p);
  }
  return drop ? launch_pdl(rms_norm_grad_kernel<T, W, CH, GROUP, true, false, THREADS>, grid, cut.threads, 0, st, p)
              : launch_pdl(rms_norm_grad_kernel<T, W, CH, GROUP, false, false, THREADS>, grid, cut.threads, 0, st, p);
}
template <typename T, typename W>
cudaError_t launch_rms_norm_grad(const NormGradParams& p, const NormGradCut& cut, cudaStream_t st) {
  if (cut.group == 1) return launch_rms_norm_grad_as<T, W, 1, 1, 32 * NORM_GRAD_ROWS>(p, cut, st);
  if (cut.group == 2) return launch_rms_norm_grad_as<T, W, 1, 2, 64 * NORM_GRAD_ROWS>(p, cut, st);
  if (cut.ch == 1) return cut.threads <= 512 ? launch_rms_norm_grad_as<T, W, 1, 0, 512>(p, cut, st) : launch_rms_norm_grad_as<T, W, 1, 0, 1024>(p, cut, st);
  return cut.ch == 2 ? launch_rms_norm_grad_as<T, W, 2, 0, 1024>(p, cut, st) : launch_rms_norm_grad_as<T, W, 4, 0, 1024>(p, cut, st);
}
template <typename W>
cudaError_t launch_rms_norm_weight_grad(const float* parts, int n, int width, void* dw, int alone, cudaStream_t st) {
  return launch_pdl(rms_norm_weight_grad_kernel<W>, dim3((unsigned)((width + 31) / 32)), 32 * NORM_SHARES_Y, 0, st, parts, n, width, static_cast<W*>(dw), alone);
}

}  // namespace fgms
