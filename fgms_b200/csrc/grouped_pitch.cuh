// 16-bit rows whose channel counts are no multiples of 8, or that start off a 16-byte boundary, for the tensor cores: a tensor map wants rows
// that are multiples of 16 bytes apart.  Operands are copied to such rows first and outputs copied back: two passes over memory and three
// launches, against the products on the CUDA cores (grouped_worth_copying has both sides).  The maps still say where
// a row ends, so what lies between the rows is read as zeros and need not be cleared.
#pragma once
#include "grouped.cuh"

namespace fgms {

// `len` values of each of `rows` rows
struct GroupedRows {
  const uint16_t* src;
  uint16_t* dst;
  long long rows, src_pitch, dst_pitch;
  int len;
};
constexpr int GP_THREADS = 256;
constexpr int GP_SEGMENT = 256;  // columns of a warp at a time: 64 bytes an access

__device__ __forceinline__ void grouped_copy_rows(const GroupedRows& r, long long lo, long long hi, bool zero_rest) {
  const int segments = (r.len + GP_SEGMENT - 1) / GP_SEGMENT, lane = threadIdx.x & 31;
  const long long warps = (long long)gridDim.x * (GP_THREADS / 32);
  for (long long i = (long long)blockIdx.x * (GP_THREADS / 32) + (threadIdx.x >> 5); i < r.rows * segments; i += warps) {
    const long long row = i / segments;
    const int c0 = (int)(i - row * segments) * GP_SEGMENT + lane;
    const bool inside = row >= lo && row < hi;
    if (!inside && !zero_rest) continue;
    const uint16_t* from = r.src + row * r.src_pitch;
    uint16_t* to = r.dst + row * r.dst_pitch;
    uint16_t v[GP_SEGMENT / 32];
#pragma unroll
    for (int k = 0; k < GP_SEGMENT / 32; ++k) v[k] = inside && c0 + 32 * k < r.len ? from[c0 + 32 * k] : (uint16_t)0;
#pragma unroll
    for (int k = 0; k < GP_SEGMENT / 32; ++k)
      if (c0 + 32 * k < r.len) to[c0 + 32 * k] = v[k];
  }
}

// two matrices (either may have no rows); alone: see GmsParams
__global__ void __launch_bounds__(GP_THREADS) grouped_copy_kernel(GroupedRows x, GroupedRows y, int alone) {
  umma::griddep_wait();
  if (!alone) umma::griddep_launch_dependents();
  grouped_copy_rows(x, 0, x.rows, false);
  grouped_copy_rows(y, 0, y.rows, false);
}

// the rows of the groups; the others are left as they were, or become zeros
__global__ void __launch_bounds__(GP_THREADS) grouped_copy_back_kernel(GroupedRows r, const int32_t* __restrict__ kpos, int groups, int zero_rest,
                                                                      int alone) {
  __shared__ int ends[2];
  umma::griddep_wait();
  if (!alone) umma::griddep_launch_dependents();
  if (threadIdx.x < 32) {  // as build_group_table has them (which has counted the entries that were changed)
    int last = 0;
    for (int s = threadIdx.x; s <= groups; s += 32) last = max(last, (int)min((long long)max(__ldg(kpos + s), 0), r.rows));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
    if (threadIdx.x == 0) {
      ends[0] = (int)min((long long)max(__ldg(kpos), 0), r.rows);
      ends[1] = last;
    }
  }
  __syncthreads();
  grouped_copy_rows(r, ends[0], ends[1], zero_rest != 0);
}

// What of a call has to be copied, and where to.
struct GroupedCopies {
  struct One { bool needed; long long rows; int len, pitch; size_t at; } a, b, d;
  size_t total;  // bytes of workspace; 0: nothing is copied
};

// Copying pays where the CUDA cores (16-bit rows of odd widths: 16 TFLOP/s and 5 us) would take longer than reading and writing everything once more at
// 2 TB/s, nine microseconds of launches and latency, and the product itself: 1000 rows 1001 -> 1003 109 us there, 15 with copies; 6007 rows in 9 groups
// 260 -> 516 79 / 17, the gradient of a 65 x 67 matrix over 20000 rows 164 / 27; 3000 rows in 4 groups 99 -> 333 21 / 10.5.
// `steps`: of 16 of the contraction that one CTA there goes through after the other, 0.7 us each.
inline bool grouped_worth_copying(double bytes, double flops, double steps) {
  const double there = flops / 16e6 > 0.7 * steps ? flops / 16e6 : 0.7 * steps;  // microseconds
  return 5.0 + there > 9.0 + bytes / 2e6 + flops / 1e9;
}

template <int PASS>
GroupedCopies grouped_copies(const void* a, const void* b, const void* d, int n_rows, int c_in, int c_out, int groups) {
  GroupedCopies c;
  const auto one = [](const void* p, long long rows, int width) {
    GroupedCopies::One o;
    o.rows = rows;
    o.len = width;
    o.pitch = (width + 7) / 8 * 8;
    o.needed = o.pitch != width || (reinterpret_cast<uintptr_t>(p) & 15) != 0;
    o.at = 0;
    return o;
  };
  const long long mats = (long long)groups * c_in;
  c.a = one(a, n_rows, PASS == GROUPED_DGRAD ? c_out : c_in);
  c.b = one(b, PASS == GROUPED_WGRAD ? n_rows : mats, c_out);
  c.d = one(d, PASS == GROUPED_WGRAD ? mats : n_rows, PASS == GROUPED_DGRAD ? c_in : c_out);
  c.total = 0;
  double bytes = 0;
  for (GroupedCopies::One* o : {&c.a, &c.b, &c.d}) {
    if (!o->needed) continue;
    o->at = c.total;
    c.total += ((size_t)o->rows * o->pitch * 2 + 255) / 256 * 256;
    bytes += 4.0 * (double)o->rows * o->len;
  }
  // a tile's contraction is shared by eight CTAs where tiles are few: see launch_grouped_ffma
  double steps = (PASS == GROUPED_WGRAD ? (double)n_rows / groups : PASS == GROUPED_DGRAD ? (double)c_out : (double)c_in) / 16;
  const double tiles = PASS == GROUPED_WGRAD ? (double)groups * ((c_in + 63) / 64) * ((c_out + 63) / 64) : (double)((n_rows + 63) / 64) * ((c.d.len + 63) / 64);
  if (tiles < 148) steps /= tiles * 8 < 148 ? 8.0 : 148 / tiles;
  if (n_rows < 1 || !grouped_worth_copying(bytes, 2.0 * n_rows * (double)c_in * c_out, steps)) c.total = 0;
  return c;
}

}  // namespace fgms
