// Grouped products on tcgen05: fp16 / bf16 rows that tensor maps can describe (channel counts that are multiples of 8, 16-byte aligned tensors).
//
// The channels of the output are the M side of the MMA and what the ragged groups are cut along is its N side: an MMA takes any N
// that is a multiple of 16, so the last rows of a group cost what they are, not a whole tile of 128.
//
//                       M, 128 a CTA             N, at most `tile_n`        contraction, 64 a stage
//   forward             channels of out (W)      rows of a group (in)       c_in
//   input gradient      channels of in_grad (W)  rows of a group (out_grad) c_out
//   weight gradient     c_out (out_grad)         c_in (in)                  rows of a group
//
// Operands come by TMA into 128-byte-swizzled tiles: the side whose contraction index is contiguous in memory K-major, the other one MN-major.  With
// CG = 2 a pair of CTAs on two SMs works on one tile (M = 256): each loads its own half of both operands, the even one issues the MMAs of
// both, each has its 128 channels of the sums in its tensor memory.
//
//   warp 0      producer: one lane issues the stage's copies, a ring of stages ahead
//   warp 1      MMA issuer (of the pair's even CTA)
//   warp 2      weight gradient: the rows behind a group's last one in its last stage are the next group's; they are cleared in
//               shared memory between the copy and the MMA
//   warps 4-7   epilogue: tcgen05.ld, neighbouring lanes exchange halves of two rows so that each stores two channels
//
// Two accumulators in tensor memory: the epilogue of a tile runs beside the next one's MMAs.  All waits are bounded; a wait that runs out sets the
// CTA's abort flag and is counted.
#pragma once
#include "grouped.cuh"

namespace fgms {

constexpr int GU_K = 64;  // contraction length of a stage: 128 bytes
constexpr int GU_THREADS = 256;
constexpr int GU_MAX_STAGES = 12;
constexpr int GU_A_BYTES = 128 * GU_K * 2;

struct GuShared {
  uint64_t full[GU_MAX_STAGES];    // of the even CTA: both CTAs' halves of the stage are there
  uint64_t empty[GU_MAX_STAGES];   // of each CTA
  uint64_t landed[GU_MAX_STAGES];  // a stage whose rows are to be cleared is there
  uint64_t tmem_full[2];
  uint64_t tmem_empty[2];  // of the even CTA
  uint64_t drained;
  uint32_t tmem_base;
  int abort_flag;
};
constexpr int GU_SHARED_BYTES = (sizeof(GuShared) + 15) & ~15;

struct GuConfig {
  int tile_n;       // rows (weight gradient: input channels) of a tile at most: a multiple of 16 CG, at most 256
  int stages;
  int stage_bytes;  // of a CTA: a multiple of 1024
  int bf16;
  int smem;
};

namespace umma {
template <int CG>
__device__ __forceinline__ void pair_alloc(uint32_t smem_dst, uint32_t cols) {
  if (CG == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_dst), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_dst), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CG>
__device__ __forceinline__ void pair_free(uint32_t taddr, uint32_t cols) {
  if (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
  else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
template <int CG>
__device__ __forceinline__ void pair_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  const uint32_t acc = accumulate ? 1u : 0u;
  if (CG == 1)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
                 "r"(idesc), "r"(acc)
                 : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
                 "r"(idesc), "r"(acc)
                 : "memory");
}
// an arrival at `bar` of every CTA of the pair once the MMAs issued so far have finished
template <int CG>
__device__ __forceinline__ void pair_commit(uint32_t bar) {
  if (CG == 1) asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((unsigned short)3)
                 : "memory");
}
// the address of this CTA's `addr` in the pair's even CTA
template <int CG>
__device__ __forceinline__ uint32_t at_leader(uint32_t addr) {
  if (CG == 1) return addr;
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
// arrivals at a barrier of either CTA of the pair
__device__ __forceinline__ void pair_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void pair_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.release.cluster.shared::cluster.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool pair_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool pair_park(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
// the bounded waits of mbar_wait (SPIN) and mbar_parked_wait, for barriers that the other CTA of a pair arrives at
template <bool SPIN>
__device__ __forceinline__ bool pair_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  if (pair_test(bar, parity)) return true;
  const long long start = clock64();
  for (uint32_t it = 1;; ++it) {
    if (SPIN ? pair_test(bar, parity) : pair_park(bar, parity)) return true;
    if (!SPIN || (it & 255u) == 0) {
      if (*abort_flag) return false;
      if (clock64() - start > WAIT_LIMIT_CYCLES) break;
    }
  }
  *abort_flag = 1;
  return false;
}
// box of a tensor map, into this CTA's shared memory; its bytes are reported to `bar`, with CG = 2 of either CTA
template <int CG>
__device__ __forceinline__ void pair_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  if (CG == 1)
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(map), "r"(bar),
                 "r"(x), "r"(y)
                 : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
                 "l"(map), "r"(bar), "r"(x), "r"(y)
                 : "memory");
}
template <int CG>
__device__ __forceinline__ void pair_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  if (CG == 1)
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(map), "r"(bar),
                 "r"(x), "r"(y), "r"(z)
                 : "memory");
  else
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
                 "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
                 : "memory");
}
template <int CG>
__device__ __forceinline__ void pair_sync() {
  if (CG == 1) __syncthreads();
  else asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
}  // namespace umma

// What a tile is: the same for every role.
struct GuTile {
  int g, m0, n0, n, n_mma;  // group; first channel (of the pair); first row or column; how many; the same as the MMA takes it
  int k0, k_len;            // weight gradient: the group's first row and how many; otherwise 0 and the channels of the contraction
};
template <int PASS, int CG>
struct GuTiles {
  const int *first, *tiles;
  int groups, tile_n, m_tiles, n_tiles, c_k, c_in;
  long long total;
  __device__ __forceinline__ GuTiles(const GroupedParams& p, int tile_n_, const int* first_, const int* tiles_)
      : first(first_), tiles(tiles_), groups(p.groups), tile_n(tile_n_), c_in(p.c_in) {
    const int channels = PASS == GROUPED_DGRAD ? p.c_in : p.c_out;
    c_k = PASS == GROUPED_DGRAD ? p.c_out : p.c_in;
    m_tiles = (channels + 128 * CG - 1) / (128 * CG);
    n_tiles = (p.c_in + tile_n - 1) / tile_n;
    total = PASS == GROUPED_WGRAD ? (long long)groups * n_tiles * m_tiles : (long long)tiles[groups] * m_tiles;
  }
  __device__ __forceinline__ GuTile at(long long t) const {
    GuTile r;
    const int q = (int)(t / m_tiles);
    r.m0 = (int)(t - (long long)q * m_tiles) * (128 * CG);
    if (PASS == GROUPED_WGRAD) {
      r.g = q / n_tiles;
      r.n0 = (q - r.g * n_tiles) * tile_n;
      r.n = min(tile_n, c_in - r.n0);
      r.k0 = first[r.g];
      r.k_len = first[r.g + 1] - r.k0;
    } else {
      r.g = find_segment(tiles, groups, q);
      // a group's rows are shared out evenly over its tiles: (tiles - 1) * share is less than its rows, as share <= tile_n
      const int rows = first[r.g + 1] - first[r.g], count = tiles[r.g + 1] - tiles[r.g], i = q - tiles[r.g];
      const int share = ((rows + count - 1) / count + 16 * CG - 1) / (16 * CG) * (16 * CG);
      r.n0 = first[r.g] + i * share;
      r.n = min(share, rows - i * share);
      r.k0 = 0;
      r.k_len = c_k;
    }
    r.n_mma = (r.n + 16 * CG - 1) / (16 * CG) * (16 * CG);
    return r;
  }
};

template <int PASS, int CG>
__global__ void __launch_bounds__(GU_THREADS, 1)
    grouped_umma_kernel(GroupedParams p, GuConfig cfg, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                        const __grid_constant__ CUtensorMap map_b16) {
  using namespace umma;
  constexpr bool A_MN = PASS != GROUPED_DGRAD, B_MN = PASS == GROUPED_WGRAD;
  extern __shared__ uint8_t gu_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(gu_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  GuShared* sh = reinterpret_cast<GuShared*>(smem + (size_t)cfg.stages * cfg.stage_bytes);
  int* first = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(sh) + GU_SHARED_BYTES);  // [groups + 1]
  int* tiles = first + p.groups + 1;                                                     // [groups + 1]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? blockIdx.x & 1u : 0u;
  volatile int* abort_flag = &sh->abort_flag;

  if (threadIdx.x == 0) {
    for (int s = 0; s < cfg.stages; ++s) {
      mbar_init(smem_u32(&sh->full[s]), CG);
      mbar_init(smem_u32(&sh->empty[s]), 1);
      mbar_init(smem_u32(&sh->landed[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&sh->tmem_full[b]), 1);
      mbar_init(smem_u32(&sh->tmem_empty[b]), 4 * CG);
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
  build_group_table(cfg.tile_n, p.kpos, p.n_rows, p.groups, first, tiles);
  tc_fence_before();
  pair_sync<CG>();  // barriers and tensor memory of both CTAs are there
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;
  const GuTiles<PASS, CG> all(p, cfg.tile_n, first, tiles);
  const long long t0 = blockIdx.x / CG, step = gridDim.x / CG;
  const uint32_t stage0 = smem_u32(smem);
  bool ok = true;

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    if (elect_one()) {
      int s = 0;
      uint32_t ph = 1;
      for (long long t = t0; t < all.total && ok; t += step) {
        const GuTile tile = all.at(t);
        const int m0 = tile.m0 + (int)rank * 128, half = tile.n_mma / CG, n0 = tile.n0 + (int)rank * half;
        const int blocks = (tile.k_len + GU_K - 1) / GU_K;
        const uint32_t b_bytes = B_MN ? (uint32_t)((half + 63) / 64) * 8192u : (uint32_t)half * 128u;
        for (int kb = 0; kb < blocks; ++kb) {
          ok = pair_wait<false>(smem_u32(&sh->empty[s]), ph, abort_flag);
          if (!ok) break;
          const uint32_t a = stage0 + (uint32_t)(s * cfg.stage_bytes), b = a + GU_A_BYTES;
          const int k = tile.k0 + kb * GU_K;
          const bool clear = PASS == GROUPED_WGRAD && (tile.k_len - kb * GU_K) % 16 != 0 && kb + 1 == blocks;
          // a stage to be cleared is reported to this CTA's warp 2, which reports it on
          const uint32_t bar = clear ? smem_u32(&sh->landed[s]) : at_leader<CG>(smem_u32(&sh->full[s]));
          pair_expect(bar, GU_A_BYTES + b_bytes);
          if (PASS == GROUPED_FWD) {
            pair_load_3d<CG>(a, &map_a, bar, m0, k, tile.g);
            pair_load_3d<CG>(a + 8192, &map_a, bar, m0 + 64, k, tile.g);
          } else if (PASS == GROUPED_DGRAD) {
            pair_load_3d<CG>(a, &map_a, bar, k, m0, tile.g);
          } else {
            pair_load_2d<CG>(a, &map_a, bar, m0, k);
            pair_load_2d<CG>(a + 8192, &map_a, bar, m0 + 64, k);
          }
          if (B_MN) {
            for (int c = 0; c < half; c += 64) pair_load_2d<CG>(b + (uint32_t)c * 128u, &map_b, bar, n0 + c, k);
          } else if (half == cfg.tile_n / CG) {
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
      // bits 7 and 10: the operands' type (0 fp16, 1 bf16)
      const uint32_t idesc0 = make_idesc(false, A_MN, B_MN, 128 * CG, 0) | (cfg.bf16 ? (1u << 7) | (1u << 10) : 0u);
      const uint64_t a_desc0 = make_sdesc(stage0, A_MN ? 8192u : 16u, 1024u), b_desc0 = make_sdesc(stage0 + GU_A_BYTES, B_MN ? 8192u : 16u, 1024u);
      constexpr uint32_t a_step = (A_MN ? 2048u : 32u) >> 4, b_step = (B_MN ? 2048u : 32u) >> 4;
      int s = 0, buf = 0;
      uint32_t ph = 0, buf_ph = 1;
      for (long long t = t0; t < all.total && ok; t += step) {
        const GuTile tile = all.at(t);
        const int steps = (tile.k_len + 15) / 16;  // of the contraction: 16 each, four a stage
        if (steps == 0) continue;
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
            for (int i = 0; i < 4; ++i) pair_mma<CG>(d, a + (uint64_t)(i * a_step), b + (uint64_t)(i * b_step), idesc, k > 0 || i > 0);
          } else {
            for (int i = 0; k + i < steps; ++i) pair_mma<CG>(d, a + (uint64_t)(i * a_step), b + (uint64_t)(i * b_step), idesc, k > 0 || i > 0);
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
  } else if (warp == 2 && PASS == GROUPED_WGRAD) {
    // ------------------------------------------------------------------ rows behind a group's last one
    int s = 0;
    uint32_t odd = 0;  // phases of the barriers, a bit a stage
    for (long long t = t0; t < all.total && ok; t += step) {
      const GuTile tile = all.at(t);
      const int blocks = (tile.k_len + GU_K - 1) / GU_K, there = tile.k_len % GU_K;
      if (blocks == 0) continue;
      s = (s + blocks - 1) % cfg.stages;
      if (there % 16 != 0) {
        ok = pair_wait<false>(smem_u32(&sh->landed[s]), (odd >> s) & 1u, abort_flag);
        if (!ok) break;
        odd ^= 1u << s;
        // to the next multiple of 16: the MMA goes no further.  A row is 128 bytes of each block of 64 channels.
        const uint32_t base = stage0 + (uint32_t)(s * cfg.stage_bytes);
        const int rows = 16 - there % 16, chans = GU_A_BYTES / 8192 + (tile.n_mma / CG + 63) / 64;
        for (int i = lane; i < rows * chans * 8; i += 32) {
          const int chunk = i & 7, r = (i >> 3) % rows, c = (i >> 3) / rows;
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(base + (uint32_t)(c * 8192 + (there + r) * 128 + chunk * 16)), "r"(0) : "memory");
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) pair_arrive(at_leader<CG>(smem_u32(&sh->full[s])));
      }
      s = s + 1 == cfg.stages ? 0 : s + 1;
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ epilogue
    const int quarter = warp - 4;  // lanes of tensor memory that this warp may read
    const int channels = PASS == GROUPED_DGRAD ? p.c_in : p.c_out;
    uint16_t* out = static_cast<uint16_t*>(p.d);
    if (PASS != GROUPED_WGRAD && p.zero_rest) zero_other_rows(p.d, (size_t)channels * 2, first, p.groups, p.n_rows, threadIdx.x - 128, 128);
    int buf = 0;
    uint32_t ph = 0;
    for (long long t = t0; t < all.total && ok; t += step) {
      const GuTile tile = all.at(t);
      const bool some = tile.k_len > 0;  // a group without rows has a gradient of zeros
      // Even lanes store row j, odd ones row j + 1, two channels each.
      const int ch = tile.m0 + (int)rank * 128 + quarter * 32 + (lane & ~1);
      const bool mine = ch < channels;
      uint16_t* to = out + (PASS == GROUPED_WGRAD ? ((size_t)tile.g * p.c_in + tile.n0) * channels : (size_t)tile.n0 * channels) + ch + (size_t)(lane & 1) * channels;
      if (some) {
        ok = pair_wait<false>(smem_u32(&sh->tmem_full[buf]), ph, abort_flag);
        ok = __all_sync(0xffffffffu, ok) != 0;
        if (!ok) break;
        tc_fence_after();
      }
      const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * cfg.tile_n);
      for (int j0 = 0; j0 < tile.n_mma; j0 += 16) {
        uint32_t v[16];
        if (some) {
          tmem_ld16(from + (uint32_t)j0, v);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = 0u;
        }
        if (some && j0 + 16 >= tile.n_mma) {  // the last of them: the accumulator is free
          tc_fence_before();
          __syncwarp();
          if (lane == 0) pair_arrive(at_leader<CG>(smem_u32(&sh->tmem_empty[buf])));
        }
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          const uint32_t give = (lane & 1) ? v[j] : v[j + 1], got = __shfl_xor_sync(0xffffffffu, give, 1);
          const float lo = __uint_as_float((lane & 1) ? got : v[j]), hi = __uint_as_float((lane & 1) ? v[j + 1] : got);
          uint32_t two;
          if (cfg.bf16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(two) : "f"(hi), "f"(lo));
          else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(two) : "f"(hi), "f"(lo));
          if (mine && j0 + j + (lane & 1) < tile.n) *reinterpret_cast<uint32_t*>(to + (size_t)(j0 + j) * channels) = two;
        }
      }
      if (some) {
        buf ^= 1;
        if (buf == 0) ph ^= 1u;
      }
    }
  }
  if (!ok) report_problem();
  __syncwarp();
  tc_fence_before();
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

// A tensor map of 16-bit values, boxes of 64 values (128 bytes, swizzled) by `box` rows: of a matrix [rows][cols], or with `mats` > 0 of that
// many of them.
inline int grouped_tensor_map(CUtensorMap* map, const void* data, int cols, int rows, int mats, int box, bool bf16) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  const Encode encode = reinterpret_cast<Encode>(tensor_map_encoder());
  if (encode == nullptr) return -1000 - (int)CUDA_ERROR_NOT_FOUND;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)(mats > 0 ? mats : 1)};
  const cuuint64_t pitch[2] = {(cuuint64_t)cols * 2, (cuuint64_t)cols * 2 * (cuuint64_t)rows};
  const cuuint32_t boxes[3] = {64, (cuuint32_t)box, 1}, steps[3] = {1, 1, 1};
  const auto made = [&] {
    return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, mats > 0 ? 3 : 2, const_cast<void*>(data), dims, pitch, boxes,
                  steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult rc = made();
  if (rc == CUDA_ERROR_INVALID_CONTEXT) {  // a host thread that has launched nothing yet: see weight_tensor_map
    int dev = 0;
    if (cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) rc = made();
  }
  return rc == CUDA_SUCCESS ? 0 : -1000 - (int)rc;
}

// Whether the kernel takes a call: what the tensor maps and the stores ask for.
inline bool grouped_umma_takes(const GroupedParams& p, bool* shape) {
  *shape = p.c_in % 8 == 0 && p.c_out % 8 == 0 && p.n_rows > 0;
  return *shape && ((reinterpret_cast<uintptr_t>(p.a) | reinterpret_cast<uintptr_t>(p.b) | reinterpret_cast<uintptr_t>(p.d)) & 15) == 0;
}

template <int PASS, int CG>
int launch_grouped_umma_as(const GroupedParams& p, bool bf16, int tile_n, cudaStream_t st, int sms, int max_smem) {
  GuConfig cfg;
  cfg.tile_n = tile_n;
  cfg.bf16 = bf16;
  const int b_bytes = PASS == GROUPED_WGRAD ? (tile_n / CG + 63) / 64 * 8192 : tile_n / CG * 128;
  cfg.stage_bytes = GU_A_BYTES + b_bytes;
  const int rest = 1024 + GU_SHARED_BYTES + (2 * p.groups + 2) * (int)sizeof(int);
  cfg.stages = (max_smem - rest) / cfg.stage_bytes;
  if (cfg.stages > GU_MAX_STAGES) cfg.stages = GU_MAX_STAGES;
  if (cfg.stages < 2) return -1;
  cfg.smem = rest + cfg.stages * cfg.stage_bytes;
  const int channels = PASS == GROUPED_DGRAD ? p.c_in : p.c_out, m_tiles = (channels + 128 * CG - 1) / (128 * CG);
  const long long n_tiles = PASS == GROUPED_WGRAD ? (long long)p.groups * ((p.c_in + tile_n - 1) / tile_n) : (long long)p.n_rows / tile_n + p.groups;
  long long pairs = n_tiles * m_tiles;
  if (pairs > sms / CG) pairs = sms / CG;
  if (pairs < 1) pairs = 1;
  CUtensorMap a, b, b16;
  int rc;
  if (PASS == GROUPED_WGRAD) {  // p.a: in, p.b: out_grad
    rc = grouped_tensor_map(&a, p.b, p.c_out, p.n_rows, 0, 64, bf16);
    if (rc == 0) rc = grouped_tensor_map(&b, p.a, p.c_in, p.n_rows, 0, 64, bf16);
    b16 = b;
  } else {
    rc = grouped_tensor_map(&a, p.b, p.c_out, p.c_in, p.groups, PASS == GROUPED_FWD ? 64 : 128, bf16);
    const int width = PASS == GROUPED_FWD ? p.c_in : p.c_out;
    if (rc == 0) rc = grouped_tensor_map(&b, p.a, width, p.n_rows, 0, tile_n / CG, bf16);
    if (rc == 0) rc = grouped_tensor_map(&b16, p.a, width, p.n_rows, 0, 16, bf16);
  }
  if (rc != 0) return rc;
  static std::atomic<int> granted[64];
  if (ensure_smem(grouped_umma_kernel<PASS, CG>, cfg.smem, granted) != 0) return -1;
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3((unsigned)(pairs * CG));
  lc.blockDim = dim3(GU_THREADS);
  lc.dynamicSmemBytes = (size_t)cfg.smem;
  lc.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = CG;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  lc.attrs = at;
  lc.numAttrs = CG == 2 ? 2 : 1;
  return cudaLaunchKernelEx(&lc, grouped_umma_kernel<PASS, CG>, p, cfg, a, b, b16) == cudaSuccess ? 0 : -1;
}

template <int PASS>
int launch_grouped_umma(const GroupedParams& p, bool bf16, cudaStream_t st, int sms, int max_smem) {
  if (sms >= 2 && (PASS == GROUPED_DGRAD ? p.c_in : p.c_out) > 128) return launch_grouped_umma_as<PASS, 2>(p, bf16, 256, st, sms, max_smem);
  return launch_grouped_umma_as<PASS, 1>(p, bf16, 128, st, sms, max_smem);
}

}  // namespace fgms
