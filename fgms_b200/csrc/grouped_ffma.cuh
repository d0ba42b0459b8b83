// Grouped products on the CUDA cores: fp32 storage in exact fp32, and fp16 / bf16 whose rows do not start on 16-byte boundaries (widths
// that are no multiples of 8, views), which a tensor map cannot describe.  Any size, any alignment.
//
// A CTA computes tiles of TILE x TILE values of D, the contraction in steps of 16: both operands are widened to fp32 on their way
// into shared memory, laid out with the contraction index outermost, and every thread keeps (TILE / 16)^2 sums in registers as
// packed pairs (fma.rn.f32x2).  The next step's operands are fetched to registers while the current one is multiplied.
#pragma once
#include "ffma_rows.cuh"  // ff_fma2, ff_two, ff_half
#include "grouped.cuh"

namespace fgms {

constexpr int GF_THREADS = 256;
constexpr int GF_K = 16;

// four values from p on, zeros from the `there`-th on
template <typename T>
__device__ __forceinline__ float4 gf_load4(const T* p, int there, bool vec) {
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (there <= 0) return v;
  if (vec && there >= 4) {
    if constexpr (sizeof(T) == 4) {
      v = __ldg(reinterpret_cast<const float4*>(p));
    } else {
      const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
      T h[4];
      memcpy(h, &u, 8);
      v = make_float4(to_f32(h[0]), to_f32(h[1]), to_f32(h[2]), to_f32(h[3]));
    }
    return v;
  }
  v.x = to_f32(p[0]);
  if (there > 1) v.y = to_f32(p[1]);
  if (there > 2) v.z = to_f32(p[2]);
  if (there > 3) v.w = to_f32(p[3]);
  return v;
}

// One operand of a tile: `outer` rows or columns of D from `base` on, `inner` contraction steps.  ALONG: the contraction index is
// contiguous, and outer ones are `pitch` values apart; otherwise the other way around.
template <typename T, bool ALONG, int TILE>
struct GfOperand {
  static constexpr int QUADS = TILE * GF_K / 4 / GF_THREADS, LD = TILE + 4;
  const T* base;
  size_t pitch;
  int outer, inner;
  bool vec;
  float4 held[QUADS];
  __device__ __forceinline__ void fetch(int k0) {
#pragma unroll
    for (int q = 0; q < QUADS; ++q) {
      const int i = (int)threadIdx.x + q * GF_THREADS;
      if (ALONG) {
        const int o = i / (GF_K / 4), k = k0 + i % (GF_K / 4) * 4;
        held[q] = gf_load4(base + (size_t)o * pitch + k, o < outer ? inner - k : 0, vec);
      } else {
        const int o = i % (TILE / 4) * 4, k = k0 + i / (TILE / 4);
        held[q] = gf_load4(base + (size_t)k * pitch + o, k < inner ? outer - o : 0, vec);
      }
    }
  }
  __device__ __forceinline__ void put(float* to) const {
#pragma unroll
    for (int q = 0; q < QUADS; ++q) {
      const int i = (int)threadIdx.x + q * GF_THREADS;
      if (ALONG) {
        const int o = i / (GF_K / 4), k = i % (GF_K / 4) * 4;
        to[(k + 0) * LD + o] = held[q].x;
        to[(k + 1) * LD + o] = held[q].y;
        to[(k + 2) * LD + o] = held[q].z;
        to[(k + 3) * LD + o] = held[q].w;
      } else {
        *reinterpret_cast<float4*>(to + i / (TILE / 4) * LD + i % (TILE / 4) * 4) = held[q];
      }
    }
  }
};

template <typename T, int PASS, int TILE>
__global__ void __launch_bounds__(GF_THREADS) grouped_ffma_kernel(GroupedParams p) {
  constexpr int SUB = TILE / 16;  // rows and columns of D per thread: 4 or 8, in quads 64 apart
  constexpr int LD = TILE + 4;
  constexpr bool A_ALONG = PASS != GROUPED_WGRAD, B_ALONG = PASS == GROUPED_DGRAD;
  __shared__ __align__(16) float as[2][GF_K * LD], bs[2][GF_K * LD];
  extern __shared__ int gf_table[];
  int *first = gf_table, *tiles = gf_table + p.groups + 1;
  umma::griddep_wait();
  if (!p.alone) umma::griddep_launch_dependents();
  build_group_table(TILE, p.kpos, p.n_rows, p.groups, first, tiles);

  const T *a = static_cast<const T*>(p.a), *b = static_cast<const T*>(p.b);
  T* d = static_cast<T*>(p.d);
  const int d_cols = PASS == GROUPED_DGRAD ? p.c_in : p.c_out, col_tiles = (d_cols + TILE - 1) / TILE;
  const int row_tiles = (p.c_in + TILE - 1) / TILE;  // of a group's dW
  const long long total = PASS == GROUPED_WGRAD ? (long long)p.groups * row_tiles * col_tiles : (long long)tiles[p.groups] * col_tiles;
  if (PASS != GROUPED_WGRAD && p.zero_rest) zero_other_rows(d, (size_t)d_cols * sizeof(T), first, p.groups, p.n_rows, threadIdx.x, GF_THREADS);
  const auto aligned = [](const void* q, int width) { return (reinterpret_cast<uintptr_t>(q) % (4 * sizeof(T))) == 0 && width % 4 == 0; };
  GfOperand<T, A_ALONG, TILE> oa;
  GfOperand<T, B_ALONG, TILE> ob;
  oa.pitch = PASS == GROUPED_DGRAD ? p.c_out : p.c_in;
  ob.pitch = p.c_out;
  oa.vec = aligned(a, PASS == GROUPED_DGRAD ? p.c_out : p.c_in);
  ob.vec = aligned(b, p.c_out);
  const bool d_vec = aligned(d, d_cols);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;

  for (long long t = blockIdx.x; t < total; t += gridDim.x) {
    const int c0 = (int)(t % col_tiles) * TILE;
    const int mt = (int)(t / col_tiles);
    T* out;
    int n_k, d_rows;
    if (PASS == GROUPED_WGRAD) {
      const int g = mt / row_tiles, r0 = mt % row_tiles * TILE;
      oa.base = a + (size_t)first[g] * p.c_in + r0;
      ob.base = b + (size_t)first[g] * p.c_out + c0;
      n_k = first[g + 1] - first[g];
      oa.outer = d_rows = p.c_in - r0;
      ob.outer = p.c_out - c0;
      out = d + ((size_t)g * p.c_in + r0) * p.c_out + c0;
    } else {
      const int g = find_segment(tiles, p.groups, mt);
      const int r0 = first[g] + (mt - tiles[g]) * TILE;
      const T* w = b + (size_t)g * p.c_in * p.c_out;
      oa.base = a + (size_t)r0 * oa.pitch;
      ob.base = PASS == GROUPED_FWD ? w + c0 : w + (size_t)c0 * p.c_out;
      n_k = PASS == GROUPED_FWD ? p.c_in : p.c_out;
      oa.outer = d_rows = first[g + 1] - r0;
      ob.outer = d_cols - c0;
      out = d + (size_t)r0 * d_cols + c0;
    }
    oa.inner = ob.inner = n_k;
    uint64_t sum[SUB][SUB / 2];
#pragma unroll
    for (int i = 0; i < SUB; ++i)
#pragma unroll
      for (int j = 0; j < SUB / 2; ++j) sum[i][j] = 0;
    oa.fetch(0);
    ob.fetch(0);
    int buf = 0;
    for (int k0 = 0; k0 < n_k; k0 += GF_K) {
      oa.put(as[buf]);
      ob.put(bs[buf]);
      __syncthreads();  // (the other buffer's readers have passed the one before)
      if (k0 + GF_K < n_k) {
        oa.fetch(k0 + GF_K);
        ob.fetch(k0 + GF_K);
      }
      const float *pa = as[buf] + ty * 4, *pb = bs[buf] + tx * 4;
#pragma unroll
      for (int k = 0; k < GF_K; ++k) {
        uint64_t fb[SUB / 2];
        float fa[SUB];
#pragma unroll
        for (int h = 0; h < SUB / 4; ++h) {
          ff_lds2(ff_smem(pb + k * LD + h * 64), fb[2 * h], fb[2 * h + 1]);
          *reinterpret_cast<float4*>(fa + 4 * h) = *reinterpret_cast<const float4*>(pa + k * LD + h * 64);
        }
#pragma unroll
        for (int i = 0; i < SUB; ++i) {
          const uint64_t two = ff_two(fa[i], fa[i]);
#pragma unroll
          for (int j = 0; j < SUB / 2; ++j) ff_fma2(sum[i][j], two, fb[j]);
        }
      }
      buf ^= 1;
    }
    __syncthreads();  // before the next tile's first step overwrites what may still be read
#pragma unroll
    for (int i = 0; i < SUB; ++i) {
      const int r = ty * 4 + i % 4 + i / 4 * 64;
      if (r >= d_rows) continue;
#pragma unroll
      for (int h = 0; h < SUB / 4; ++h) {
        const int c = tx * 4 + h * 64;
        T v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = from_f32<T>(ff_half(sum[i][2 * h + e / 2], e & 1));
        T* to = out + (size_t)r * d_cols + c;
        if (d_vec && c + 4 <= d_cols - c0) {
          if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(v);
          else *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(v);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c + e < d_cols - c0) to[e] = v[e];
        }
      }
    }
  }
}

template <typename T, int PASS>
int launch_grouped_ffma(const GroupedParams& p, cudaStream_t st, int sms) {
  const int d_cols = PASS == GROUPED_DGRAD ? p.c_in : p.c_out;
  const auto tiles = [&](int tile) {  // at most
    const long long rows = PASS == GROUPED_WGRAD ? (long long)p.groups * ((p.c_in + tile - 1) / tile) : (long long)p.n_rows / tile + p.groups;
    return rows * ((d_cols + tile - 1) / tile);
  };
  const size_t table = (size_t)(2 * p.groups + 2) * sizeof(int);
  // 128 x 128 reads each operand half as often; below two such tiles per SM smaller ones keep more of the chip busy
  const bool wide = tiles(128) >= 2ll * sms;
  const long long n = wide ? tiles(128) : tiles(64), most = (long long)sms * (wide ? 2 : 4);
  const dim3 grid((unsigned)(n < 1 ? 1 : n < most ? n : most));
  const cudaError_t e = wide ? launch_pdl(grouped_ffma_kernel<T, PASS, 128>, grid, GF_THREADS, table, st, p)
                             : launch_pdl(grouped_ffma_kernel<T, PASS, 64>, grid, GF_THREADS, table, st, p);
  return e == cudaSuccess ? 0 : -1;
}

}  // namespace fgms
