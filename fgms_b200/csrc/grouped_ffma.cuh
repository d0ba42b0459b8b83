// Grouped products on the CUDA cores: fp32 storage in exact fp32, and fp16 / bf16 whose rows do not start on 16-byte boundaries (widths
// that are no multiples of 8, views), which a tensor map cannot describe.  Any size, any alignment.
//
// A CTA computes tiles of TILE x TILE values of D, the contraction in steps of 16: both operands are widened to fp32 on their way
// into shared memory, laid out with the contraction index outermost, and every thread keeps (TILE / 16)^2 sums in registers as
// packed pairs (fma.rn.f32x2).  The operands of the steps ahead are on their way to registers while one is multiplied: one step for tiles of 128, which
// have no registers for more, four for tiles of 64, whose time is the latency of their loads (2 rows 512 -> 512 24 us with one, 8.6 with four).  16384 rows of
// 16 groups 1024 -> 1024 744 us, 46 TFLOP/s; what bounds the large tiles are the registers that a packed FMA wants aligned and doubled.
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
template <typename T, bool ALONG, int TILE, int DEPTH>
struct GfOperand {
  static constexpr int QUADS = TILE * GF_K / 4 / GF_THREADS, LD = TILE + 4;
  const T* base;
  size_t pitch;
  int outer, inner;
  bool vec;
  float4 held[DEPTH][QUADS];
  __device__ __forceinline__ void fetch(float4 (&held)[QUADS], int k0) {
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
  __device__ __forceinline__ void put(const float4 (&held)[QUADS], float* to) const {
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

// PARTS: the CTAs of a cluster share a tile's contraction; each adds up some of its rows at the end, in the order of the parts.
template <typename T, int PASS, int TILE, bool PARTS>
__global__ void __launch_bounds__(GF_THREADS, 2) grouped_ffma_kernel(GroupedParams p, int parts) {
  constexpr int SUB = TILE / 16;  // rows and columns of D per thread: 4 or 8, in quads 64 apart
  constexpr int LD = TILE + 4;
  constexpr int DEPTH = TILE == 64 ? 4 : 1;  // steps on their way, in registers
  constexpr bool A_ALONG = PASS != GROUPED_WGRAD, B_ALONG = PASS == GROUPED_DGRAD;
  __shared__ __align__(16) float as[2][GF_K * LD], bs[2][GF_K * LD];
  __shared__ __align__(16) float sums[PARTS ? TILE * TILE : 4];
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
  GfOperand<T, A_ALONG, TILE, DEPTH> oa;
  GfOperand<T, B_ALONG, TILE, DEPTH> ob;
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
    uint64_t sum[SUB][SUB / 2];
#pragma unroll
    for (int i = 0; i < SUB; ++i)
#pragma unroll
      for (int j = 0; j < SUB / 2; ++j) sum[i][j] = 0;
#pragma unroll
    for (int s = 0; s < DEPTH; ++s) {
      oa.fetch(oa.held[s], k_from + s * GF_K);
      ob.fetch(ob.held[s], k_from + s * GF_K);
    }
    int buf = 0;
    for (int k0 = k_from; k0 < k_to; k0 += DEPTH * GF_K) {
#pragma unroll
      for (int s = 0; s < DEPTH; ++s) {
        if (k0 + s * GF_K >= k_to) break;
        oa.put(oa.held[s], as[buf]);
        ob.put(ob.held[s], bs[buf]);
        __syncthreads();  // (the other buffer's readers have passed the one before)
        oa.fetch(oa.held[s], k0 + (s + DEPTH) * GF_K);
        ob.fetch(ob.held[s], k0 + (s + DEPTH) * GF_K);
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
    }
    if constexpr (PARTS) {
      // rows [share q, share (q + 1)) to part q: [part][row][column]
      const int share = TILE / parts;
#pragma unroll
      for (int i = 0; i < SUB; ++i) {
        const int r = ty * 4 + i;
        const uint32_t at = ff_smem(sums) + (uint32_t)(((part * share + r % share) * TILE + tx * 4) * 4);
        asm volatile("{\n\t.reg .b32 there;\n\tmapa.shared::cluster.u32 there, %0, %1;\n\tst.shared::cluster.v2.b64 [there], {%2, %3};\n\t}" ::"r"(at),
                     "r"(r / share), "l"(sum[i][0]), "l"(sum[i][1])
                     : "memory");
      }
    } else {
      __syncthreads();  // before the next tile's first step overwrites what may still be read
#pragma unroll
      for (int i = 0; i < SUB; ++i) {
        const int r = ty * 4 + i % 4 + i / 4 * 64;
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
      for (int i = threadIdx.x; i < share * (TILE / 4); i += GF_THREADS) {
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
  // over 20000 rows 944 us, so 117; 200 rows 1000 -> 300 48, so 14.)
  const long long steps = (PASS == GROUPED_WGRAD ? (long long)p.n_rows / p.groups : PASS == GROUPED_DGRAD ? p.c_out : p.c_in) / GF_K;
  int parts = 1;
  while (parts < 8 && tiles(64) * parts * 2 <= 2ll * sms && steps >= 8ll * parts) parts *= 2;
  if (parts > 1) {
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)(tiles(64) * parts));
    lc.blockDim = dim3(GF_THREADS);
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
  // 128 x 128 reads each operand half as often; below two such tiles per SM smaller ones, with more steps on their way, keep more of the chip busy
  // (6007 rows in 9 groups: 260 -> 516 69 us with 64, 62 with 128; its input gradient 81 / 109, its weight gradient 94 / 79)
  const bool wide = tiles(128) >= 2ll * sms;
  const long long n = wide ? tiles(128) : tiles(64), most = 2ll * sms;
  const dim3 grid((unsigned)(n < 1 ? 1 : n < most ? n : most));
  const cudaError_t e = wide ? launch_pdl(grouped_ffma_kernel<T, PASS, 128, false>, grid, GF_THREADS, table, st, p, 1)
                             : launch_pdl(grouped_ffma_kernel<T, PASS, 64, false>, grid, GF_THREADS, table, st, p, 1);
  return e == cudaSuccess ? 0 : -1;
}

}  // namespace fgms
