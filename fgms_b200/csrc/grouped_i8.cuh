// Products of 8-bit integers with a scale for each row and each output channel, over ragged groups of rows, on tcgen05 (kind::i8):
//
//   out[r, c] = float(sum over k of a[r, k] b[g, c, k]) * row_scale[r] * channel_scale[g, c]         for the rows r of group g
//
// Sums are 32-bit integers and exact (at most 2^17 - 1 products of at most 2^14), so neither the cut nor the order changes a bit; what is
// rounded is the sum to fp32 (beyond 2^24), the two multiplications and the output's type.
//
// Both operands have the contraction side by side in memory (weights are [groups, c_out, c_in]: a channel's row is what has a scale), 128 values a
// stage: the bytes of a stage, the walk over the tiles and the cut of a call are those of the input gradient in 16 bits (grouped_umma.cuh), which
// is told half as many channels.  An MMA takes 32 values where that one takes 16, in the same time: 16384 rows 2048 -> 4096 to bf16 90 us, 3.06 POP/s, kept
// busy 110 (the power limit), the tensor pipe active 78 % of it; one row 8.6 us, latency.
//
//   warp 0      producer          warp 1      MMA issuer (of the pair's even CTA)
//   warps 4-11  epilogue: scales, a transposition through shared memory and 16-byte stores; outputs off 16-byte boundaries go straight to
//               memory, 32 channels a store (9444 rows 1232 -> 952 in fp32 32 us so, 26 through the patch)
#pragma once
#include "grouped_umma.cuh"
#include "row_values.cuh"

namespace fgms {

constexpr int GI_MAX_CONTRACTION = (1 << 17) - 1;

struct GroupedI8Params {
  GroupedParams g;  // as the walk takes it: c_in the output's channels, c_out the contraction in units of two values; a: rows, b: weights; kpos: or null
  const float *row_scale, *channel_scale;
  int dtype;   // of the output: 0 fp32, 1 fp16, 2 bf16
  int store;   // 0: 16-bit rows through the patch, 1: fp32 rows through it, 2: straight to memory
};

namespace umma {
template <int CG>
__device__ __forceinline__ void pair_mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  const uint32_t acc = accumulate ? 1u : 0u;
  if (CG == 1)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
                 "r"(idesc), "r"(acc)
                 : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
                 "r"(idesc), "r"(acc)
                 : "memory");
}
}  // namespace umma

__device__ __forceinline__ float i8_scaled(uint32_t sum, float a, float b) { return (float)(int)sum * a * b; }

__device__ __forceinline__ void i8_store(const GroupedI8Params& p, size_t at, float v) {
  if (p.dtype == 0) static_cast<float*>(p.g.d)[at] = v;
  else if (p.dtype == 1) static_cast<__half*>(p.g.d)[at] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p.g.d)[at] = __float2bfloat16_rn(v);
}

template <int CG, bool SPLIT>
__global__ void __launch_bounds__(GU_THREADS, 1)
    grouped_i8_kernel(GroupedI8Params q, GuConfig cfg, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                      const __grid_constant__ CUtensorMap map_b16) {
  using namespace umma;
  const GroupedParams& p = q.g;
  extern __shared__ uint8_t gi_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(gi_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  GuShared* sh = reinterpret_cast<GuShared*>(smem + (size_t)cfg.stages * cfg.stage_bytes + GU_EPI_WARPS / 4 * GU_PATCH_BYTES);
  int* first = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(sh) + GU_SHARED_BYTES);  // [groups + 1]
  int* tiles = first + p.groups + 1;                                                     // [groups + 1]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? blockIdx.x & 1u : 0u;
  volatile int* abort_flag = &sh->abort_flag;

  if (threadIdx.x == 0) {
    for (int s = 0; s < cfg.stages; ++s) {
      mbar_init(smem_u32(&sh->full[s]), CG);
      mbar_init(smem_u32(&sh->empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&sh->tmem_full[b]), 1);
      mbar_init(smem_u32(&sh->tmem_empty[b]), GU_EPI_WARPS * CG);
    }
    mbar_init(smem_u32(&sh->drained), 1);
    sh->abort_flag = 0;
    mbar_fence_init();
  }
  uint32_t tmem_cols = 32;
  while (tmem_cols < 2u * (uint32_t)cfg.tile_n) tmem_cols <<= 1;
  if (warp == 1) pair_alloc<CG>(smem_u32(&sh->tmem_base), tmem_cols);
  griddep_wait();
  if (!p.alone) griddep_launch_dependents();
  if (p.kpos != nullptr) {
    build_group_table(cfg.tile_n, p.kpos, p.n_rows, p.groups, first, tiles);
  } else {
    if (threadIdx.x == 0) {
      first[0] = tiles[0] = 0;
      first[1] = p.n_rows;
      tiles[1] = (p.n_rows + cfg.tile_n - 1) / cfg.tile_n;
    }
    __syncthreads();
  }
  tc_fence_before();
  pair_sync<CG>();  // barriers and tensor memory of both CTAs are there
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;
  GuTiles<GROUPED_DGRAD, CG, SPLIT> tile(p, cfg, first, tiles, nullptr);
  const uint32_t stage0 = smem_u32(smem);
  const int channels = p.c_in;
  bool ok = true;

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    if (elect_one()) {
      int s = 0;
      uint32_t ph = 1;
      for (; tile.left > 0 && ok; tile.next()) {
        const int m0 = tile.m0 + (int)rank * 128, half = tile.n_mma / CG, n0 = tile.n0 + (int)rank * half;
        for (int kb = tile.b0; kb < tile.b1; ++kb) {
          ok = pair_wait<false>(smem_u32(&sh->empty[s]), ph, abort_flag);
          if (!ok) break;
          const uint32_t a = stage0 + (uint32_t)(s * cfg.stage_bytes), b = a + GU_A_BYTES;
          const int k = kb * 128;
          const uint32_t bar = at_leader<CG>(smem_u32(&sh->full[s]));
          pair_expect(bar, GU_A_BYTES + (uint32_t)half * 128u);
          pair_load_3d<CG>(a, &map_a, bar, k, m0, tile.g);
          if (half == cfg.tile_n / CG) {
            pair_load_2d<CG>(b, &map_b, bar, k, n0);
          } else {
            for (int r = 0; r < half; r += 16) pair_load_2d<CG>(b + (uint32_t)r * 128u, &map_b16, bar, k, n0 + r);
          }
          if (++s == cfg.stages) { s = 0; ph ^= 1u; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (rank == 0 && elect_one()) {
      // [4,6) sums: 2, int32   [7,10) and [10,13) operands: 1, int8   both K-major   [17,23) N >> 3   [24,29) M >> 4
      const uint32_t idesc0 = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(128 * CG >> 4) << 24);
      const uint64_t a_desc0 = make_sdesc(stage0, 16u, 1024u), b_desc0 = make_sdesc(stage0 + GU_A_BYTES, 16u, 1024u);
      int s = 0, buf = 0;
      uint32_t ph = 0, buf_ph = 1;
      for (; tile.left > 0 && ok; tile.next()) {
        const int steps = min((tile.k_len + 15) / 16, tile.b1 * 4) - tile.b0 * 4;  // of the contraction: 32 values each, four a stage
        if (steps <= 0) continue;
        ok = pair_wait<true>(smem_u32(&sh->tmem_empty[buf]), buf_ph, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(buf * cfg.tile_n), idesc = idesc0 | (uint32_t)(tile.n_mma >> 3) << 17;
        for (int k = 0; k < steps; k += 4) {
          ok = pair_wait<true>(smem_u32(&sh->full[s]), ph, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint64_t off = (uint64_t)((uint32_t)(s * cfg.stage_bytes) >> 4);
          const uint64_t a = a_desc0 + off, b = b_desc0 + off;
          if (k + 4 <= steps) {
#pragma unroll
            for (int i = 0; i < 4; ++i) pair_mma_i8<CG>(d, a + (uint64_t)(i * 2), b + (uint64_t)(i * 2), idesc, k > 0 || i > 0);
          } else {
            for (int i = 0; k + i < steps; ++i) pair_mma_i8<CG>(d, a + (uint64_t)(i * 2), b + (uint64_t)(i * 2), idesc, k > 0 || i > 0);
          }
          pair_commit<CG>(smem_u32(&sh->empty[s]));
          if (++s == cfg.stages) { s = 0; ph ^= 1u; }
        }
        if (!ok) break;
        pair_commit<CG>(smem_u32(&sh->tmem_full[buf]));
        buf ^= 1;
        if (buf == 0) buf_ph ^= 1u;
      }
      // what was issued has finished before the pair's memory is given up
      pair_commit<CG>(smem_u32(&sh->drained));
      mbar_wait(smem_u32(&sh->drained), 0u, nullptr);
    }
    __syncwarp();
  } else if (warp >= GU_EPI_WARP0) {
    // ------------------------------------------------------------------ epilogue
    const int quarter = warp & 3;  // lanes of tensor memory that this warp may read
    const int half = (warp - GU_EPI_WARP0) >> 2;  // of the tile's columns, in turns of 32
    if (p.zero_rest)
      zero_other_rows(p.d, (size_t)p.d_pitch * (q.dtype == 0 ? 4 : 2), first, p.groups, p.n_rows, threadIdx.x - GU_EPI_WARP0 * 32, GU_EPI_WARPS * 32);
    const uint32_t patch = stage0 + (uint32_t)(cfg.stages * cfg.stage_bytes) + (uint32_t)half * GU_PATCH_BYTES;
    const auto chunk_at = [&](int row, int chunk) { return patch + (uint32_t)(row * 256 + (chunk ^ (row & 7)) * 16); };
    const uint32_t put = chunk_at(lane & 7, quarter * 4 + (lane >> 3));  // rows eight apart: 2048 bytes on
    int buf = 0;
    uint32_t ph = 0;
    for (; !SPLIT && tile.left > 0 && ok; tile.next()) {
      const int m0 = tile.m0 + (int)rank * 128;
      const float* scales = q.channel_scale + (size_t)tile.g * channels;
      // the scales of the channels that this thread holds sums of, on their way while the sums are awaited
      float channel[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = m0 + quarter * 32 + (q.store > 0 ? lane : i * 8 + (lane >> 2));
        channel[i] = c < channels ? __ldg(scales + c) : 0.f;
      }
      ok = four_agree(half, pair_wait<false>(smem_u32(&sh->tmem_full[buf]), ph, abort_flag, tile_wait_limit(tile.blocks)));
      if (!ok) break;
      tc_fence_after();
      const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * cfg.tile_n);
      if (q.store == 1) {
        const int c = m0 + lane * 4;
        float* to = static_cast<float*>(p.d) + (size_t)tile.n0 * p.d_pitch + c;
        for (int j0 = half * 16; j0 < tile.n_mma; j0 += 32) {  // 16 rows of the warp's 32 channels, then four rows of all 128
          uint32_t v[16];
          tmem_ld16(from + (uint32_t)j0, v);
          const float scale = lane < 16 && j0 + lane < tile.n ? __ldg(q.row_scale + tile.n0 + j0 + lane) : 0.f;
          tmem_ld_wait();
          four_sync(half);  // the patch has been read
#pragma unroll
          for (int j = 0; j < 16; ++j)
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(patch + (uint32_t)(j * 512 + (quarter * 32 + lane) * 4)),
                         "f"(i8_scaled(v[j], __shfl_sync(0xffffffffu, scale, j), channel[0]))
                         : "memory");
          four_sync(half);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = quarter * 4 + i;
            float4 o;
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(o.x), "=f"(o.y), "=f"(o.z), "=f"(o.w) : "r"(patch + (uint32_t)(row * 512 + lane * 16)) : "memory");
            if (j0 + row < tile.n && c < channels) *reinterpret_cast<float4*>(to + (size_t)(j0 + row) * p.d_pitch) = o;
          }
        }
      } else if (q.store == 2) {
        const int c = m0 + quarter * 32 + lane;
        for (int j0 = half * 32; j0 < tile.n_mma; j0 += 64) {
#pragma unroll
          for (int part = 0; part < 32; part += 16) {
            if (j0 + part >= tile.n_mma) break;
            uint32_t v[16];
            tmem_ld16(from + (uint32_t)(j0 + part), v);
            const int r0 = j0 + part;
            const float scale = lane < 16 && r0 + lane < tile.n ? __ldg(q.row_scale + tile.n0 + r0 + lane) : 0.f;
            tmem_ld_wait();
            size_t at = (size_t)(tile.n0 + r0) * p.d_pitch + c;
#pragma unroll
            for (int j = 0; j < 16; ++j, at += p.d_pitch) {
              const float row = __shfl_sync(0xffffffffu, scale, j);
              if (r0 + j < tile.n && c < channels) i8_store(q, at, i8_scaled(v[j], row, channel[0]));
            }
          }
        }
      } else {
        const int ch = m0 + (lane & 15) * 8;
        uint16_t* to = static_cast<uint16_t*>(p.d) + (size_t)tile.n0 * p.d_pitch + ch;
        const bool mine = ch < channels;
        for (int j0 = half * 32; j0 < tile.n_mma; j0 += 64) {
          // 32 rows (columns of the accumulator, of which the last 16 may not be used) of the warp's 32 channels
          uint32_t v[32];
          tmem_ld_16x8x4(from + (uint32_t)j0, reinterpret_cast<uint32_t(&)[16]>(v[0]));
          tmem_ld_16x8x4(from + (uint32_t)j0 + (16u << 16), reinterpret_cast<uint32_t(&)[16]>(v[16]));
          float row[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = j0 + (i >> 1) * 8 + (lane & 3) * 2 + (i & 1);
            row[i] = r < tile.n ? __ldg(q.row_scale + tile.n0 + r) : 0.f;
          }
          tmem_ld_wait();
          four_sync(half);  // the patch has been read
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // eight rows
            uint32_t h[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {  // of eight channels each
              const uint32_t* s = v + (c >> 1) * 16 + i * 4 + (c & 1) * 2;
              const float lo = i8_scaled(s[0], row[2 * i], channel[c]), hi = i8_scaled(s[1], row[2 * i + 1], channel[c]);
              if (cfg.bf16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(h[c]) : "f"(hi), "f"(lo));
              else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(h[c]) : "f"(hi), "f"(lo));
            }
            asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(put + (uint32_t)i * 2048u), "r"(h[0]), "r"(h[1]), "r"(h[2]),
                         "r"(h[3])
                         : "memory");
          }
          four_sync(half);
          const int r0 = quarter * 8 + (lane >> 4);  // two rows a store, eight a warp
          uint4 o[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(o[i].x), "=r"(o[i].y), "=r"(o[i].z), "=r"(o[i].w) : "r"(chunk_at(r0 + 2 * i, lane & 15)) : "memory");
          uint16_t* row_to = to + (size_t)(j0 + r0) * p.d_pitch;
          const int rows = mine ? tile.n - j0 - r0 : 0;
#pragma unroll
          for (int i = 0; i < 4; ++i, row_to += 2 * (size_t)p.d_pitch)
            if (2 * i < rows) *reinterpret_cast<uint4*>(row_to) = o[i];
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) pair_arrive(at_leader<CG>(smem_u32(&sh->tmem_empty[buf])));
      buf ^= 1;
      if (buf == 0) ph ^= 1u;
    }
  }
  if (!ok) report_problem();
  // The odd CTA: the commits' arrivals at its barriers are behind it before it may end.  (Its epilogue has seen all of them but the last.)
  if (CG == 2 && rank != 0 && warp == GU_EPI_WARP0) mbar_parked_wait(smem_u32(&sh->drained), 0u, nullptr);
  __syncwarp();
  tc_fence_before();
  if constexpr (SPLIT) {
    // ------------------------------------------------------------------ sums of the parts
    // Every CTA has the sums over its share of the contraction in tensor memory and hands the columns (rows of the output) to the CTA that
    // finishes them, in shared memory over its ring, [part][column][128 channels].
    cluster_sync();  // all copies and MMAs of all parts are done
    tc_fence_after();
    const int part = (int)blockIdx.x % cfg.parts, width = (tile.n_mma + cfg.parts - 1) / cfg.parts;
    if (warp >= GU_EPI_WARP0 && tile.left > 0) {
      const int quarter = warp & 3, half = (warp - GU_EPI_WARP0) >> 2;
      for (int j0 = half * 16; j0 < tile.n_mma; j0 += 32) {
        uint32_t v[16];
        if (tile.b1 > tile.b0) {
          tmem_ld16(tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)j0, v);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = 0u;
        }
        int to = j0 / width, c = j0 - to * width;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if (j0 + j < tile.n) put_at(to, stage0 + (uint32_t)(((part * width + c) * 128 + quarter * 32 + lane) * 4), v[j]);
          if (++c == width) { c = 0; ++to; }
        }
      }
    }
    cluster_sync();
    if (warp >= GU_EPI_WARP0 && tile.left > 0) {
      const int thread = (int)threadIdx.x - GU_EPI_WARP0 * 32, lane_ch = thread & 127, c_at = tile.m0 + lane_ch;
      const int n = min(width, tile.n - part * width);
      if (c_at < channels) {
        const float channel = __ldg(q.channel_scale + (size_t)tile.g * channels + c_at);
        for (int c = thread >> 7; c < n; c += GU_EPI_WARPS / 4) {
          int sum = 0;
          for (int i = 0; i < cfg.parts; ++i) sum += ld_shared_i32(stage0 + (uint32_t)(((i * width + c) * 128 + lane_ch) * 4));
          const int r = tile.n0 + part * width + c;
          i8_store(q, (size_t)r * p.d_pitch + c_at, i8_scaled((uint32_t)sum, __ldg(q.row_scale + r), channel));
        }
      }
    }
    tc_fence_before();
  }
  if (*abort_flag) {  // copies may still be on their way into this CTA's memory
    const long long start = clock64();
    while (clock64() - start < 2000000) __nanosleep(1000);
  }
  __syncwarp();
  pair_sync<CG>();  // nothing arrives at the other CTA's barriers, and nothing reads its memory, after this
  if (warp == 1) {
    tc_fence_after();
    pair_free<CG>(tmem, tmem_cols);
  }
}

// A tensor map of 8-bit values, boxes of 128 values (swizzled) by `box` rows, rows `pitch` bytes apart (a multiple of 16).
inline int grouped_i8_tensor_map(CUtensorMap* map, const void* data, int cols, long long pitch, int rows, int mats, int box) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  const Encode encode = reinterpret_cast<Encode>(tensor_map_encoder());
  if (encode == nullptr) return -1000 - (int)CUDA_ERROR_NOT_FOUND;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)(mats > 0 ? mats : 1)};
  const cuuint64_t pitches[2] = {(cuuint64_t)pitch, (cuuint64_t)pitch * (cuuint64_t)rows};
  const cuuint32_t boxes[3] = {128, (cuuint32_t)box, 1}, steps[3] = {1, 1, 1};
  const auto made = [&] {
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, mats > 0 ? 3 : 2, const_cast<void*>(data), dims, pitches, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult rc = made();
  if (rc == CUDA_ERROR_INVALID_CONTEXT) {  // a host thread that has launched nothing yet: see weight_tensor_map
    int dev = 0;
    if (cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) rc = made();
  }
  return rc == CUDA_SUCCESS ? 0 : -1000 - (int)rc;
}

template <int CG, bool SPLIT>
int grant_grouped_i8(int max_smem) {
  static std::atomic<int> granted[64];
  return ensure_smem(grouped_i8_kernel<CG, SPLIT>, max_smem, granted);
}

// rows and weights: `contraction` values a row, `row_pitch` and `weight_pitch` bytes apart (multiples of 16, from 16-byte boundaries)
template <int CG, bool SPLIT>
int launch_grouped_i8_as(const GroupedI8Params& q, int contraction, long long row_pitch, long long weight_pitch, const GuCut& cut, cudaStream_t st, int sms,
                         int max_smem) {
  const GroupedParams& p = q.g;
  GuConfig cfg;
  cfg.parts = SPLIT ? cut.parts : 1;
  cfg.tile_n = cut.tile_n;
  cfg.bf16 = q.dtype == 2;
  cfg.by_size = 0;
  cfg.stage_bytes = GU_A_BYTES + cfg.tile_n / CG * 128;
  const int rest = 1024 + GU_EPI_WARPS / 4 * GU_PATCH_BYTES + GU_SHARED_BYTES + (2 * p.groups + 2) * (int)sizeof(int);
  cfg.stages = (max_smem - rest) / cfg.stage_bytes;
  if (cfg.stages > GU_MAX_STAGES) cfg.stages = GU_MAX_STAGES;
  if (cfg.stages < 2 || (SPLIT && cfg.stages * cfg.stage_bytes < (cfg.tile_n + cut.parts) * 512)) return -1;
  cfg.smem = rest + cfg.stages * cfg.stage_bytes;
  long long clusters = grouped_tiles<GROUPED_DGRAD>(p, cut);
  if (!SPLIT && clusters > sms / CG) clusters = sms / CG;
  if (clusters < 1) clusters = 1;
  const int ctas = SPLIT ? cut.parts : CG;
  CUtensorMap a, b, b16;
  int rc = grouped_i8_tensor_map(&a, p.b, contraction, weight_pitch, p.c_in, p.groups, 128);
  if (rc == 0) rc = grouped_i8_tensor_map(&b, p.a, contraction, row_pitch, p.n_rows, 0, cfg.tile_n / CG);
  if (rc == 0) rc = grouped_i8_tensor_map(&b16, p.a, contraction, row_pitch, p.n_rows, 0, 16);
  if (rc != 0) return rc;
  if (grant_grouped_i8<CG, SPLIT>(max_smem) != 0) return -1;
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3((unsigned)(clusters * ctas));
  lc.blockDim = dim3(GU_THREADS);
  lc.dynamicSmemBytes = (size_t)cfg.smem;
  lc.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)ctas;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  lc.attrs = at;
  lc.numAttrs = ctas > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&lc, grouped_i8_kernel<CG, SPLIT>, q, cfg, a, b, b16) == cudaSuccess ? 0 : -1;
}

// see grouped_clusters_at_once
inline int grouped_i8_clusters_at_once(int parts, int sms, int max_smem) {
  static std::atomic<int> known[64][4];
  int dev = 0, all = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64 || parts < 2) return 0;
  std::atomic<int>& at = known[dev][parts == 2 ? 0 : parts == 4 ? 1 : 2];
  if (cudaDeviceGetAttribute(&all, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  int n = at.load(std::memory_order_acquire) - 1;
  if (n < 0) {
    if (grant_grouped_i8<1, true>(max_smem) != 0) return 0;
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)(parts * all));
    lc.blockDim = dim3(GU_THREADS);
    lc.dynamicSmemBytes = (size_t)max_smem;
    cudaLaunchAttribute cluster[1];
    cluster[0].id = cudaLaunchAttributeClusterDimension;
    cluster[0].val.clusterDim.x = (unsigned)parts;
    cluster[0].val.clusterDim.y = cluster[0].val.clusterDim.z = 1;
    lc.attrs = cluster;
    lc.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, grouped_i8_kernel<1, true>, &lc) != cudaSuccess || n < 0) {
      cudaGetLastError();
      return 0;
    }
    at.store(n + 1, std::memory_order_release);
  }
  return n * sms / all;
}

inline int launch_grouped_i8(const GroupedI8Params& q, int contraction, long long row_pitch, long long weight_pitch, cudaStream_t st, int sms, int max_smem) {
  const GuCut cut = grouped_cut<GROUPED_DGRAD>(q.g, sms, [&](int parts) { return grouped_i8_clusters_at_once(parts, sms, max_smem); });
  if (cut.parts > 1) return launch_grouped_i8_as<1, true>(q, contraction, row_pitch, weight_pitch, cut, st, sms, max_smem);
  return cut.cg == 2 ? launch_grouped_i8_as<2, false>(q, contraction, row_pitch, weight_pitch, cut, st, sms, max_smem)
                     : launch_grouped_i8_as<1, false>(q, contraction, row_pitch, weight_pitch, cut, st, sms, max_smem);
}

// ---------------------------------------------------------------------------------------------
// Codes whose rows no tensor map describes (not a multiple of 16 bytes apart, or off a 16-byte boundary) are copied to rows that it does, four bytes at
// a time; the maps still say where a row ends.  One launch and one more pass over them: codes from quantize_rows need none.
// ---------------------------------------------------------------------------------------------
struct ByteRows {
  const uint8_t* src;
  uint8_t* dst;
  long long rows, src_pitch, dst_pitch;
  int len;
};
constexpr int BR_THREADS = 256;
__device__ __forceinline__ void copy_byte_rows(const ByteRows& r) {
  const int words = (r.len + 3) / 4, lane = threadIdx.x & 31;
  const long long warps = (long long)gridDim.x * (BR_THREADS / 32);
  for (long long row = (long long)blockIdx.x * (BR_THREADS / 32) + (threadIdx.x >> 5); row < r.rows; row += warps) {
    const uint8_t* from = r.src + row * r.src_pitch;
    const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(from) & 3u);
    const uint32_t* aligned = reinterpret_cast<const uint32_t*>(from - off);
    uint32_t* to = reinterpret_cast<uint32_t*>(r.dst + row * r.dst_pitch);
    for (int w = lane; w < words; w += 32) {
      uint32_t v = 0;
      if ((w > 0 || off == 0) && 4 * w + 8 - (int)off <= r.len) {  // both words that it lies in are the row's own
        v = off == 0 ? aligned[w] : __funnelshift_r(aligned[w], aligned[w + 1], off * 8);
      } else {
        for (int i = 0; i < 4; ++i)
          if (4 * w + i < r.len) v |= (uint32_t)from[4 * w + i] << (8 * i);
      }
      to[w] = v;
    }
  }
}
static __global__ void __launch_bounds__(BR_THREADS) copy_byte_rows_kernel(ByteRows x, ByteRows y, int alone) {
  umma::griddep_wait();
  if (!alone) umma::griddep_launch_dependents();
  copy_byte_rows(x);
  copy_byte_rows(y);
}

}  // namespace fgms
