// Grouped products on the CUDA cores: fp32 storage in exact fp32, and fp16 / bf16 whose rows do not start on 16-byte boundaries (widths
// that are no multiples of 8, views), which a tensor map cannot describe, where copying them does not pay (grouped_pitch.cuh).  Any size, any alignment.
//
// A CTA computes tiles of TILE x TILE values of D, the contraction in steps of 16: both operands are widened to fp32 on their way
// into shared memory, laid out with the contraction index outermost, and every thread keeps 8 rows by TILE / 16 columns of sums in registers as packed
// pairs (fma.rn.f32x2).  The next step's operands are on their way to registers while one is multiplied; more steps ahead gained nothing.
//
// Bound by the FMA pipe (a packed FMA is 2.4 cycles a scheduler: 62 TFLOP/s) and by the registers that want pairs: 16384 rows of 16 groups 1024 -> 1024
// 742 / 708 / 677 us (forward, input gradient, weight gradient; 46 to 51 TFLOP/s; with single FMAs 895 / 894 / 837), 6007 rows of 9 groups 260 -> 516 64 / 65 / 76
// (with 256 threads of 4 x 4 sums for a tile of 64 69 / 81 / 94).
#pragma once
#include "ffma_rows.cuh"  // ff_fma2, ff_two, ff_half
#include "grouped.cuh"

namespace fgms {

__host__ __device__ constexpr int gf_threads(int tile) { return tile == 128 ? 256 : 128; }  // 16 by 16, or 16 by 8
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
  static constexpr int THREADS = gf_threads(TILE), QUADS = TILE * GF_K / 4 / THREADS, LD = TILE + 4;
  const T* base;
  size_t pitch;
  int outer, inner;
  bool vec;
  float4 held[QUADS];
  __device__ __forceinline__ void fetch(int k0) {
#pragma unroll
    for (int q = 0; q < QUADS; ++q) {
      const int i = (int)threadIdx.x + q * THREADS;
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
      const int i = (int)threadIdx.x + q * THREADS;
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

// PARTS: the CTAs of a cluster share a tile's contraction; each adds up some of its rows at the end, in the order of the parts.
template <typename T, int PASS, int TILE, bool PARTS>
__global__ void __launch_bounds__(gf_threads(TILE), TILE == 128 ? 2 : 4) grouped_ffma_kernel(GroupedParams p, int parts) {
  constexpr int THREADS = gf_threads(TILE);
  constexpr int SUB = TILE / 16;  // columns of D per thread: 4 or 8, in quads 64 apart; rows: 8, in quads TILE / 2 apart
  constexpr int LD = TILE + 4;
  constexpr bool A_ALONG = PASS != GROUPED_WGRAD, B_ALONG = PASS == GROUPED_DGRAD;
  __shared__ __align__(16) float as[2][GF_K * LD], bs[2][GF_K * LD];
  __shared__ __align__(16) float sums[PARTS ? TILE * TILE : 4];
  extern __shared__ int gf_table[];
  int *first = gf_table, *tiles = gf_table + p.groups + 1;
  umma::griddep_wait();
  if (!p.alone) umma::griddep_launch_dependents();
  build_group_table(TILE, p.kpos, p.n_rows, p.groups, first, tiles);
  if (PARTS) umma::cluster_sync();  // all parts have started: their shared memory may be written

  const T *a = static_cast<const T*>(p.a), *b = static_cast<const T*>(p.b);
  T* d = static_cast<T*>(p.d);
  const int d_cols = PASS == GROUPED_DGRAD ? p.c_in : p.c_out, col_tiles = (d_cols + TILE - 1) / TILE;
  const int row_tiles = (p.c_in + TILE - 1) / TILE;  // of a group's dW
  const long long total = PASS == GROUPED_WGRAD ? (long long)p.groups * row_tiles * col_tiles : (long long)tiles[p.groups] * col_tiles;
  if (PASS != GROUPED_WGRAD && p.zero_rest) zero_other_rows(d, (size_t)d_cols * sizeof(T), first, p.groups, p.n_rows, threadIdx.x, THREADS);
  const auto aligned = [](const void* q, int width) { return (reinterpret_cast<uintptr_t>(q) % (4 * sizeof(T))) == 0 && width % 4 == 0; };
  GfOperand<T, A_ALONG, TILE> oa;
  GfOperand<T, B_ALONG, TILE> ob;
  oa.pitch = PASS == GROUPED_DGRAD ? p.c_out : p.c_in;
  ob.pitch = p.c_out;
  oa.vec = aligned(a, PASS == GROUPED_DGRAD ? p.c_out : p.c_in);
  ob.vec = aligned(b, p.c_out);
  const bool d_vec = aligned(d, d_cols);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int ctas = PARTS ? parts : 1, part = PARTS ? (int)blockIdx.x % parts : 0;

  const auto store4 = [&](T* to, const float (&x)[4], int left) {  // the first `left` of four columns
    T v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = from_f32<T>(x[e]);
    if (d_vec && left >= 4) {
      if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(v);
      else *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(v);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) to[e] = v[e];
    }
  };

  for (long long t = blockIdx.x / ctas; t < total; t += gridDim.x / ctas) {  // PARTS: at most one
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
    // this CTA's share of the contraction, in whole steps
    const int steps = (n_k + GF_K - 1) / GF_K;
    const int k_from = PARTS ? (int)((long long)steps * part / parts) * GF_K : 0;
    const int k_to = PARTS ? min(n_k, (int)((long long)steps * (part + 1) / parts) * GF_K) : n_k;
    oa.inner = ob.inner = k_to;
    uint64_t sum[8][SUB / 2];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < SUB / 2; ++j) sum[i][j] = 0;
    oa.fetch(k_from);
    ob.fetch(k_from);
    int buf = 0;
    for (int k0 = k_from; k0 < k_to; k0 += GF_K) {
      oa.put(as[buf]);
      ob.put(bs[buf]);
      __syncthreads();  // (the other buffer's readers have passed the one before)
      oa.fetch(k0 + GF_K);  // (zeros behind the last step)
      ob.fetch(k0 + GF_K);
      const float *pa = as[buf] + ty * 4, *pb = bs[buf] + tx * 4;
#pragma unroll 8  // of 16: with all of them written out 128 x 128 needs more registers than there are (forward 900 us instead of 742)
      for (int k = 0; k < GF_K; ++k) {
        float fa[8];
        uint64_t fb[SUB / 2];
#pragma unroll
        for (int h = 0; h < 2; ++h) *reinterpret_cast<float4*>(fa + 4 * h) = *reinterpret_cast<const float4*>(pa + k * LD + h * (TILE / 2));
#pragma unroll
        for (int h = 0; h < SUB / 4; ++h) {
          const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(pb + k * LD + h * 64);
          fb[2 * h] = v.x;
          fb[2 * h + 1] = v.y;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint64_t two = ff_two(fa[i], fa[i]);
#pragma unroll
          for (int j = 0; j < SUB / 2; ++j) ff_fma2(sum[i][j], two, fb[j]);
        }
      }
      buf ^= 1;
    }
    if constexpr (PARTS) {
      // rows [share q, share (q + 1)) to part q: [part][row][column]
      const int share = TILE / parts;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = ty * 4 + i % 4 + i / 4 * (TILE / 2);
        const uint32_t at = ff_smem(sums) + (uint32_t)(((part * share + r % share) * TILE + tx * 4) * 4);
        asm volatile("{\n\t.reg .b32 there;\n\tmapa.shared::cluster.u32 there, %0, %1;\n\tst.shared::cluster.v4.f32 [there], {%2, %3, %4, %5};\n\t}" ::"r"(at),
                     "r"(r / share), "f"(ff_half(sum[i][0], 0)), "f"(ff_half(sum[i][0], 1)), "f"(ff_half(sum[i][1], 0)), "f"(ff_half(sum[i][1], 1))
                     : "memory");
      }
    } else {
      __syncthreads();  // before the next tile's first step overwrites what may still be read
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = ty * 4 + i % 4 + i / 4 * (TILE / 2);
        if (r >= d_rows) continue;
#pragma unroll
        for (int h = 0; h < SUB / 4; ++h) {
          const float x[4] = {ff_half(sum[i][2 * h], 0), ff_half(sum[i][2 * h], 1), ff_half(sum[i][2 * h + 1], 0), ff_half(sum[i][2 * h + 1], 1)};
          const int c = tx * 4 + h * 64;
          store4(out + (size_t)r * d_cols + c, x, d_cols - c0 - c);
        }
      }
    }
    if constexpr (PARTS) {
      umma::cluster_sync();
      const int share = TILE / parts;
      for (int i = threadIdx.x; i < share * (TILE / 4); i += THREADS) {
        const int r = i / (TILE / 4), c = i % (TILE / 4) * 4;
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        for (int q = 0; q < parts; ++q) {
          const float4 v = *reinterpret_cast<const float4*>(sums + (q * share + r) * TILE + c);
          x[0] += v.x; x[1] += v.y; x[2] += v.z; x[3] += v.w;
        }
        if (part * share + r < d_rows) store4(out + (size_t)(part * share + r) * d_cols + c, x, d_cols - c0 - c);
      }
      return;  // a cluster has one tile; nothing is sent to a CTA after the barrier
    }
  }
}

template <typename T, int PASS>
int launch_grouped_ffma(const GroupedParams& p, cudaStream_t st, int sms) {
  const int d_cols = PASS == GROUPED_DGRAD ? p.c_in : p.c_out;
  const auto tiles = [&](int tile) {  // at most
    const long long rows = PASS == GROUPED_WGRAD ? (long long)p.groups * ((p.c_in + tile - 1) / tile)
                                                 : (long long)p.n_rows / tile + (p.n_rows < p.groups ? p.n_rows : p.groups);
    return rows * ((d_cols + tile - 1) / tile);
  };
  const size_t table = (size_t)(2 * p.groups + 2) * sizeof(int);
  // Few tiles with many steps: clusters of up to eight CTAs share them, as far as the host knows how many there are.  (The gradient of a 65 x 67 matrix
  // over 20000 rows 944 us, so 125; 2 rows 512 -> 512 24, so 8.6.)
  const long long steps = (PASS == GROUPED_WGRAD ? (long long)p.n_rows / p.groups : PASS == GROUPED_DGRAD ? p.c_out : p.c_in) / GF_K;
  int parts = 1;
  while (parts < 8 && tiles(64) * parts * 2 <= 2ll * sms && steps >= 8ll * parts) parts *= 2;
  if (parts > 1) {
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)(tiles(64) * parts));
    lc.blockDim = dim3(gf_threads(64));
    lc.dynamicSmemBytes = table;
    lc.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)parts;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    lc.attrs = at;
    lc.numAttrs = 2;
    return cudaLaunchKernelEx(&lc, grouped_ffma_kernel<T, PASS, 64, true>, p, parts) == cudaSuccess ? 0 : -1;
  }
  // 128 x 128 reads each operand half as often; below two such tiles per SM smaller ones keep more of the chip busy
  // (6007 rows in 9 groups, 260 -> 516, tiles of 64 / 128: 64 / 62 us, input gradient 65 / 109, weight gradient 76 / 79)
  const bool wide = tiles(128) >= 2ll * sms;
  const long long n = wide ? tiles(128) : tiles(64), most = (wide ? 2ll : 4ll) * sms;
  const dim3 grid((unsigned)(n < 1 ? 1 : n < most ? n : most));
  const cudaError_t e = wide ? launch_pdl(grouped_ffma_kernel<T, PASS, 128, false>, grid, gf_threads(128), table, st, p, 1)
                             : launch_pdl(grouped_ffma_kernel<T, PASS, 64, false>, grid, gf_threads(64), table, st, p, 1);
  return e == cudaSuccess ? 0 : -1;
}

}  // namespace fgms
