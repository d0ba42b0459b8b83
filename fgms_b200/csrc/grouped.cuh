// Products of ragged groups of rows with a weight matrix each: what the kernels of grouped_ffma.cuh and grouped_umma.cuh share.
//
//   rows of group g: kpos[g] <= r < kpos[g + 1]
//   forward          out[r]     = in[r] . W[g]                      one accumulator per output value, written once
//   input gradient   in_grad[r] = out_grad[r] . W[g]^T
//   weight gradient  dW[g]      = sum over the rows of g of in[r]^T (x) out_grad[r]     (zeros for a group without rows)
//
// Rows of no group (before kpos[0], from kpos[groups] on) are neither read nor, unless `zero_rest` is set, written.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "umma.cuh"

namespace fgms {

enum GroupedPass { GROUPED_FWD = 0, GROUPED_DGRAD = 1, GROUPED_WGRAD = 2 };

struct GroupedParams {
  const void* a;        // forward, weight gradient: in [n_rows, c_in]; input gradient: out_grad [n_rows, c_out]
  const void* b;        // forward, input gradient: W [groups, c_in, c_out]; weight gradient: out_grad
  void* d;              // out / in_grad / dW
  const int32_t* kpos;  // [groups + 1]
  int n_rows, c_in, c_out, groups;
  int zero_rest;  // forward, input gradient: rows of no group become zeros
  int a_pitch, b_pitch, d_pitch;  // values from a row to the next: the widths, except on the tensor cores with copied rows
  int alone;      // see GmsParams
};

// kpos comes from device memory and is not trusted: entries are clamped to [0, n_rows], and one that is smaller than an entry before it
// takes that one's value, so that no row belongs to two groups and no two tiles write the same row.  Each entry that had to be changed
// is counted once per launch.  first[g] is the first row of group g (first[groups]: one past the last), tiles[g] the number of
// tiles of `tile` rows of the groups before g.
__device__ __forceinline__ void build_group_table(int tile, const int32_t* __restrict__ kpos, int n_rows, int groups, int* first /* [groups + 1] */,
                                                  int* tiles /* [groups + 1] */) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int highest = 0, carry = 0;
    for (int s0 = 0; s0 <= groups; s0 += 32) {
      const int s = s0 + lane;
      const int raw = s <= groups ? __ldg(kpos + s) : 0;
      int c = min(max(raw, 0), n_rows);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, c, o);
        if (lane >= o) c = max(c, n);
      }
      c = max(c, highest);
      if (s <= groups) {
        if (raw != c && blockIdx.x == 0) report_problem();
        first[s] = c;
      }
      // the first row of the group behind this lane's: the next lane's, or the first one of the next 32
      int next = __shfl_down_sync(0xffffffffu, c, 1);
      if (lane == 31) next = s < groups ? max(c, min(max(__ldg(kpos + s + 1), 0), n_rows)) : c;
      int v = s < groups ? (next - c + tile - 1) / tile : 0;
      const int own = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += n;
      }
      if (s <= groups) tiles[s] = carry + v - own;
      carry += __shfl_sync(0xffffffffu, v, 31);
      highest = __shfl_sync(0xffffffffu, c, 31);
    }
  }
  __syncthreads();
}

// zeros to the rows of no group, `row_bytes` bytes each, by `threads` threads of every CTA
__device__ __forceinline__ void zero_other_rows(void* d, size_t row_bytes, const int* first, int groups, int n_rows, int thread, int threads) {
  const size_t head = (size_t)first[0] * row_bytes, from = (size_t)first[groups] * row_bytes, to = (size_t)n_rows * row_bytes;
  uint8_t* base = static_cast<uint8_t*>(d);
  const size_t at = (size_t)blockIdx.x * threads + thread, step = (size_t)gridDim.x * threads;
  const auto zero = [&](size_t lo, size_t hi) {
    if (((reinterpret_cast<uintptr_t>(base) | lo | hi) & 15) == 0) {
      for (size_t i = lo + at * 16; i < hi; i += step * 16) *reinterpret_cast<uint4*>(base + i) = make_uint4(0, 0, 0, 0);
    } else {  // elements are at least two bytes, and so are all the offsets
      for (size_t i = lo + at * 2; i < hi; i += step * 2) *reinterpret_cast<uint16_t*>(base + i) = 0;
    }
  };
  zero(0, head);
  zero(from, to);
}

template <typename T> __device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

}  // namespace fgms
