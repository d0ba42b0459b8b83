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
//   warps 4-11  epilogue: tcgen05.ld in the shape of MMA fragments, a transposition through shared memory (stmatrix), 16-byte stores along the rows
//
// Two accumulators in tensor memory: the epilogue of a tile runs beside the next one's MMAs.  All waits are bounded; a wait that runs out sets the
// CTA's abort flag and is counted.
//
// 32768 rows of 32 even groups 2048 -> 4096, bf16, kept busy for half a second: forward 445-452 us (1225 TFLOP/s), input gradient 451-457, weight gradient 464,
// where the library's batched product takes 441-444 and one product of that many operations 403-416; all run into the power limit.  A short burst 385
// (1430 TFLOP/s), 97 us a quarter of it.  What bounds that is the tensor pipe, busy for 87 % of it: 78 us without loads
// behind the first ring, 91 without the epilogue or its stores, which share the way to L2 with the 64 KB a stage that a pair reads.  96 rows in 64 groups 2048 -> 1024 46 us, 5.8 TB/s of weights.
#pragma once
#include "grouped.cuh"

namespace fgms {

constexpr int GU_K = 64;  // contraction length of a stage: 128 bytes
constexpr int GU_EPI_WARP0 = 4, GU_EPI_WARPS = 8;
constexpr int GU_THREADS = (GU_EPI_WARP0 + GU_EPI_WARPS) * 32;
constexpr int GU_MAX_STAGES = 12;
constexpr int GU_A_BYTES = 128 * GU_K * 2;
constexpr int GU_PATCH_BYTES = 32 * 128 * 2;  // of four epilogue warps

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
  int parts;        // CTAs that share a tile's contraction (SPLIT), 1 otherwise
  int tile_n;       // rows (weight gradient: input channels) of a tile at most: a multiple of 16 CG, at most 256
  int stages;
  int stage_bytes;  // of a CTA: a multiple of 1024
  int bf16;
  int by_size;      // weight gradient: the groups with the most rows first
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
// Arrivals at a barrier of either CTA of the pair.  No write to memory goes with them: the accumulator has been read, a copy will report its
// bytes.  So they do not release at cluster scope, which waits until all earlier copies and stores of the thread have been performed: 1300 cycles
// a stage in the producer, as much as the whole product takes without (2048 -> 4096 on 8192 rows 194 us, so 112).
__device__ __forceinline__ void pair_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void pair_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cluster.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// An arrival that writes go with: rows that the odd CTA has cleared, which MMAs issued by the even one's thread read.  It releases at cluster
// scope, and that thread looks at the completed phase with pair_acquire before it issues them.  Once a ragged tile, 0.3 us of it that nothing
// hides: 16 ragged groups of 16411 rows 2048 x 1024 74.4 us, with arrivals of the other kind 72.3 (the look itself costs nothing).
__device__ __forceinline__ void pair_arrive_release(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void pair_acquire(uint32_t bar, uint32_t parity) {
  uint32_t ok;  // true: the phase has been waited for
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
}
__device__ __forceinline__ bool pair_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool pair_park(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
// the bounded waits of mbar_wait (SPIN) and mbar_parked_wait, for barriers that the other CTA of a pair arrives at
template <bool SPIN>
__device__ __forceinline__ bool pair_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, long long limit = WAIT_LIMIT_CYCLES) {
  if (pair_test(bar, parity)) return true;
  const long long start = clock64();
  for (uint32_t it = 1;; ++it) {
    if (SPIN ? pair_test(bar, parity) : pair_park(bar, parity)) return true;
    if (!SPIN || (it & 255u) == 0) {
      if (*abort_flag) return false;
      if (clock64() - start > limit) break;
    }
  }
  *abort_flag = 1;
  return false;
}
// a wait for whole tiles: what a wait has, and a microsecond for each of their stages (a group may have millions)
__device__ __forceinline__ long long tile_wait_limit(long long stages) { return WAIT_LIMIT_CYCLES + 2000ll * stages; }
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
// 16 lanes by 32 consecutive columns, as four fragments of 16 x 8: thread t has lanes t / 4 and t / 4 + 8, columns 2 (t % 4) and the next
__device__ __forceinline__ void tmem_ld_16x8x4(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}
// Four warps of the epilogue meet.  Every one of them comes: the waits before are bounded, and whether they go on is decided together.
__device__ __forceinline__ void four_sync(int half) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(1 + half) : "memory"); }
__device__ __forceinline__ bool four_agree(int half, bool ok) {
  uint32_t all;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(all) : "r"((uint32_t)ok), "r"(1 + half) : "memory");
  return all != 0;
}
// a word to this CTA's address `addr` in CTA `to` of the cluster
__device__ __forceinline__ void put_at(int to, uint32_t addr, uint32_t value) {
  asm volatile("{\n\t.reg .b32 there;\n\tmapa.shared::cluster.u32 there, %0, %1;\n\tst.shared::cluster.b32 [there], %2;\n\t}" ::"r"(addr), "r"(to), "r"(value) : "memory");
}
template <int CG>
__device__ __forceinline__ void pair_sync() {
  if (CG == 1) __syncthreads();
  else cluster_sync();
}
}  // namespace umma

// How many of a group's rows its tiles take, `count` of at most `tile` rows, as evenly as multiples of `unit` (which divides `tile`) allow: (count - 1)
// shares are less than its rows, as none is more than `tile`.  Rows and tiles together may be more than an int holds.
__host__ __device__ __forceinline__ int grouped_share(int rows, int count, int unit) {
  return (int)(((unsigned)rows + (unsigned)count - 1u) / (unsigned)count + (unsigned)unit - 1u) / unit * unit;
}

// The tiles of a pair, one after the other: the same walk in every role.  Steps are added up, without a division a tile: those of 64-bit numbers
// and the search for the group took the epilogue of a short tile as long as its stores.
template <int PASS, int CG, bool SPLIT>
struct GuTiles {
  int g, m0, n0, n, n_mma;  // group; first channel (of the pair); first row or column; how many; the same as the MMA takes it
  int k0, k_len;            // weight gradient: the group's first row and how many; otherwise 0 and the channels of the contraction
  int blocks, b0, b1;       // stages of the contraction; those of this CTA
  const int *first, *tiles, *order;
  int left, index, total, m, q, m_tiles;  // q: row tile, or of the weight gradient tile of input channels
  int tile_n, c_in, n_tiles, share, parts, place;  // place: of the group in `order`
  int step, step_m, step_q, step_g, back, back_m, back_q, back_g;
  bool snake, odd;
  __device__ __forceinline__ GuTiles(const GroupedParams& p, const GuConfig& cfg, const int* first_, const int* tiles_, const int* order_)
      : first(first_), tiles(tiles_), order(order_), tile_n(cfg.tile_n), c_in(p.c_in), parts(cfg.parts) {
    const int channels = PASS == GROUPED_DGRAD ? p.c_in : p.c_out;
    const int ctas = SPLIT ? parts : CG, at = (int)blockIdx.x / ctas, all = (int)gridDim.x / ctas;
    m_tiles = (channels + 128 * CG - 1) / (128 * CG);
    n_tiles = (p.c_in + tile_n - 1) / tile_n;
    total = (PASS == GROUPED_WGRAD ? p.groups * n_tiles : tiles[p.groups]) * m_tiles;  // the launch sees to it that this is an int
    // Round after round of tiles in the order of the pairs; by size every other round the other way around, so that who had the larger tile of a
    // round has the smaller one of the next.
    snake = PASS == GROUPED_WGRAD && !SPLIT && cfg.by_size;
    odd = false;
    index = at;
    left = index < total;
    q = at / m_tiles;
    m = at - q * m_tiles;
    step = snake ? 2 * (all - at) - 1 : all;
    step_q = step / m_tiles;
    step_m = step - step_q * m_tiles;
    back = snake ? 2 * at + 1 : all;
    back_q = back / m_tiles;
    back_m = back - back_q * m_tiles;
    g = share = place = 0;
    step_g = back_g = 0;
    if (PASS == GROUPED_WGRAD) {
      place = q / n_tiles;
      q -= place * n_tiles;
      step_g = step_q / n_tiles;
      step_q -= step_g * n_tiles;
      back_g = back_q / n_tiles;
      back_q -= back_g * n_tiles;
      k_len = -1;
    } else {
      k0 = 0;
      k_len = PASS == GROUPED_DGRAD ? p.c_out : p.c_in;
    }
    n_mma = n = blocks = b0 = b1 = 0;
    if (left > 0) fill();
  }
  __device__ __forceinline__ void fill() {
    m0 = m * (128 * CG);
    if (PASS == GROUPED_WGRAD) {
      g = snake ? order[place] : place;
      n0 = q * tile_n;
      n = min(tile_n, c_in - n0);
      k0 = first[g];
      k_len = first[g + 1] - k0;
    } else {
      while (tiles[g + 1] <= q) { ++g; share = 0; }
      const int rows = first[g + 1] - first[g], count = tiles[g + 1] - tiles[g], i = q - tiles[g];
      if (share == 0) share = grouped_share(rows, count, 16 * CG);
      n0 = first[g] + i * share;
      n = min(share, rows - i * share);
    }
    n_mma = (n + 16 * CG - 1) / (16 * CG) * (16 * CG);
    blocks = b1 = (k_len + GU_K - 1) / GU_K;
    if (SPLIT) {
      const int part = (int)blockIdx.x % parts;
      b0 = (int)((long long)blocks * part / parts);
      b1 = (int)((long long)blocks * (part + 1) / parts);
    }
  }
  __device__ __forceinline__ void next() {
    index += odd ? back : step;
    left = index < total;
    if (left == 0) return;
    m += odd ? back_m : step_m;
    q += odd ? back_q : step_q;
    if (m >= m_tiles) { m -= m_tiles; ++q; }
    if (PASS == GROUPED_WGRAD) {
      place += odd ? back_g : step_g;
      if (q >= n_tiles) { q -= n_tiles; ++place; }
    }
    odd = snake && !odd;
    fill();
  }
};

template <int PASS, int CG, bool SPLIT>
__global__ void __launch_bounds__(GU_THREADS, 1)
    grouped_umma_kernel(GroupedParams p, GuConfig cfg, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                        const __grid_constant__ CUtensorMap map_b16) {
  using namespace umma;
  constexpr bool A_MN = PASS != GROUPED_DGRAD, B_MN = PASS == GROUPED_WGRAD;
  extern __shared__ uint8_t gu_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(gu_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  GuShared* sh = reinterpret_cast<GuShared*>(smem + (size_t)cfg.stages * cfg.stage_bytes + GU_EPI_WARPS / 4 * GU_PATCH_BYTES);
  int* first = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(sh) + GU_SHARED_BYTES);  // [groups + 1]
  int* tiles = first + p.groups + 1;                                                     // [groups + 1]
  int* order = tiles + p.groups + 1;                                                     // [groups], weight gradient by size
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
  build_group_table(cfg.tile_n, p.kpos, p.n_rows, p.groups, first, tiles);
  if (PASS == GROUPED_WGRAD && cfg.by_size) {
    // A tile's time is its group's rows; dealt out in the order of the groups some pairs have half as much again as others.
    for (int g = threadIdx.x; g < p.groups; g += GU_THREADS) {
      const int rows = first[g + 1] - first[g];
      int before = 0;
      for (int h = 0; h < p.groups; ++h) {
        const int other = first[h + 1] - first[h];
        before += other > rows || (other == rows && h < g);
      }
      order[before] = g;
    }
    __syncthreads();
  }
  tc_fence_before();
  pair_sync<CG>();  // barriers and tensor memory of both CTAs are there
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;
  GuTiles<PASS, CG, SPLIT> tile(p, cfg, first, tiles, order);
  const uint32_t stage0 = smem_u32(smem);
  bool ok = true;

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    if (elect_one()) {
      int s = 0;
      uint32_t ph = 1;
      for (; tile.left > 0 && ok; tile.next()) {
        const int m0 = tile.m0 + (int)rank * 128, half = tile.n_mma / CG, n0 = tile.n0 + (int)rank * half;
        const uint32_t b_bytes = B_MN ? (uint32_t)((half + 63) / 64) * 8192u : (uint32_t)half * 128u;
        for (int kb = tile.b0; kb < tile.b1; ++kb) {
          ok = pair_wait<false>(smem_u32(&sh->empty[s]), ph, abort_flag);
          if (!ok) break;
          const uint32_t a = stage0 + (uint32_t)(s * cfg.stage_bytes), b = a + GU_A_BYTES;
          const int k = tile.k0 + kb * GU_K;
          const bool clear = PASS == GROUPED_WGRAD && (tile.k_len - kb * GU_K) % 16 != 0 && kb + 1 == tile.blocks;
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
      for (; tile.left > 0 && ok; tile.next()) {
        const int steps = min((tile.k_len + 15) / 16, tile.b1 * 4) - tile.b0 * 4;  // of the contraction: 16 each, four a stage
        if (steps <= 0) continue;
        ok = pair_wait<true>(smem_u32(&sh->tmem_empty[buf]), buf_ph, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const int cleared = tile.k_len % 16 != 0 ? steps - 4 : steps;  // weight gradient: from there on the stage in which both CTAs have cleared rows
        const uint32_t d = tmem + (uint32_t)(buf * cfg.tile_n), idesc = idesc0 | (uint32_t)(tile.n_mma >> 3) << 17;
        for (int k = 0; k < steps; k += 4) {
          ok = pair_wait<true>(smem_u32(&sh->full[s]), ph, abort_flag);
          if (!ok) break;
          if (PASS == GROUPED_WGRAD && CG == 2 && k >= cleared) pair_acquire(smem_u32(&sh->full[s]), ph);
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
    long long passed = 0;  // stages since the last wait: tiles without such rows are not waited for
    for (; tile.left > 0 && ok; tile.next()) {
      const int there = tile.k_len % GU_K;
      if (tile.b0 == tile.b1) continue;
      passed += tile.b1 - tile.b0;
      s = (s + tile.b1 - tile.b0 - 1) % cfg.stages;
      if (there % 16 != 0 && tile.b1 == tile.blocks) {
        ok = pair_wait<false>(smem_u32(&sh->landed[s]), (odd >> s) & 1u, abort_flag, tile_wait_limit(passed));
        if (!ok) break;
        passed = 0;
        odd ^= 1u << s;
        // to the next multiple of 16: the MMA goes no further.  A row is 128 bytes of each block of 64 channels.
        const uint32_t base = stage0 + (uint32_t)(s * cfg.stage_bytes);
        const int blocks_there = GU_A_BYTES / 8192 + (tile.n_mma / CG + 63) / 64;
        for (int c = lane >> 3; c < blocks_there; c += 4)
          for (int r = there; r % 16 != 0; ++r)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(base + (uint32_t)(c * 8192 + r * 128 + (lane & 7) * 16)), "r"(0) : "memory");
        fence_proxy_async();  // what the tensor cores read of this CTA's memory from here on
        __syncwarp();
        if (lane == 0) {
          if (CG == 2 && rank != 0) pair_arrive_release(at_leader<CG>(smem_u32(&sh->full[s])));
          else pair_arrive(smem_u32(&sh->full[s]));
        }
      }
      s = s + 1 == cfg.stages ? 0 : s + 1;
    }
  } else if (warp >= GU_EPI_WARP0) {
    // ------------------------------------------------------------------ epilogue
    const int quarter = warp & 3;  // lanes of tensor memory that this warp may read
    const int half = (warp - GU_EPI_WARP0) >> 2;  // of the tile's columns, in turns of 32
    const int channels = PASS == GROUPED_DGRAD ? p.c_in : p.c_out;
    uint16_t* out = static_cast<uint16_t*>(p.d);
    if (PASS != GROUPED_WGRAD && p.zero_rest)
      zero_other_rows(p.d, (size_t)p.d_pitch * 2, first, p.groups, p.n_rows, threadIdx.x - GU_EPI_WARP0 * 32, GU_EPI_WARPS * 32);
    const size_t pitch = 2 * (size_t)p.d_pitch;
    // The patch of four warps: 32 rows of 128 channels, 256 bytes each, whose 16-byte chunks are permuted so that neither the eight rows of a
    // matrix nor eight consecutive chunks of a row meet in a bank.
    const uint32_t patch = stage0 + (uint32_t)(cfg.stages * cfg.stage_bytes) + (uint32_t)half * GU_PATCH_BYTES;
    const auto chunk_at = [&](int row, int chunk) { return patch + (uint32_t)(row * 256 + (chunk ^ (row & 7)) * 16); };
    const uint32_t put = chunk_at(lane & 7, quarter * 4 + (lane >> 3));  // rows eight apart: 2048 bytes on
    int buf = 0;
    uint32_t ph = 0;
    for (; !SPLIT && tile.left > 0 && ok; tile.next()) {
      const bool some = tile.k_len > 0;  // a group without rows has a gradient of zeros
      const int ch = tile.m0 + (int)rank * 128 + (lane & 15) * 8;
      uint16_t* to = out + (PASS == GROUPED_WGRAD ? (size_t)tile.g * p.c_in + tile.n0 : (size_t)tile.n0) * p.d_pitch + ch;
      const bool mine = ch < channels;
      if (some) {
        ok = four_agree(half, pair_wait<false>(smem_u32(&sh->tmem_full[buf]), ph, abort_flag, tile_wait_limit(tile.blocks)));
        if (!ok) break;
        tc_fence_after();
      }
      const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * cfg.tile_n);
      for (int j0 = half * 32; j0 < tile.n_mma; j0 += 64) {
        // 32 rows (columns of the accumulator, of which the last 16 may not be used) of the warp's 32 channels
        uint32_t v[32];
        if (some) {
          tmem_ld_16x8x4(from + (uint32_t)j0, reinterpret_cast<uint32_t(&)[16]>(v[0]));
          tmem_ld_16x8x4(from + (uint32_t)j0 + (16u << 16), reinterpret_cast<uint32_t(&)[16]>(v[16]));
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = 0u;
        }
        four_sync(half);  // the patch has been read
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // eight rows
          uint32_t h[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {  // of eight channels each
            const float lo = __uint_as_float(v[(c >> 1) * 16 + i * 4 + (c & 1) * 2]), hi = __uint_as_float(v[(c >> 1) * 16 + i * 4 + (c & 1) * 2 + 1]);
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
        uint16_t* row = to + (size_t)(j0 + r0) * p.d_pitch;
        const int rows = mine ? tile.n - j0 - r0 : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i, row += pitch)
          if (2 * i < rows) {
            // a weight gradient is read once, when the step is over: 64 groups of a few rows, 2048 -> 1024, 57 us without the hint, 52 with
            if (PASS == GROUPED_WGRAD) __stcs(reinterpret_cast<uint4*>(row), o[i]);
            else *reinterpret_cast<uint4*>(row) = o[i];
          }
      }
      if (some) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) pair_arrive(at_leader<CG>(smem_u32(&sh->tmem_empty[buf])));
        buf ^= 1;
        if (buf == 0) ph ^= 1u;
      }
    }
  }
  if (!ok) report_problem();
  // The odd CTA: the commits' arrivals at its barriers are behind it before it may end.  (Its epilogue has seen all of them but the last.)
  if (CG == 2 && rank != 0 && warp == GU_EPI_WARP0) mbar_parked_wait(smem_u32(&sh->drained), 0u, nullptr);
  __syncwarp();
  tc_fence_before();
  if constexpr (SPLIT) {
    // ------------------------------------------------------------------ sums of the parts
    // Every CTA has the sums over its share of the contraction in tensor memory.  It hands the columns (rows of the output) to the CTA that finishes
    // them, in shared memory over its ring, [part][column][128 channels]; that one adds them in the order of the parts: the same bits on every run.
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
          put_at(to, stage0 + (uint32_t)(((part * width + c) * 128 + quarter * 32 + lane) * 4), v[j]);
          if (++c == width) { c = 0; ++to; }
        }
      }
    }
    cluster_sync();
    if (warp >= GU_EPI_WARP0 && tile.left > 0) {
      const int channels = PASS == GROUPED_DGRAD ? p.c_in : p.c_out, thread = (int)threadIdx.x - GU_EPI_WARP0 * 32;
      const int ch = 2 * (thread & 63);
      const int n = min(width, tile.n - part * width);
      uint16_t* out = static_cast<uint16_t*>(p.d) +
                      ((PASS == GROUPED_WGRAD ? (size_t)tile.g * p.c_in + tile.n0 : (size_t)tile.n0) + part * width) * p.d_pitch + tile.m0 + ch;
      if (tile.m0 + ch < channels)
        for (int c = thread >> 6; c < n; c += GU_EPI_WARPS / 2) {
          float lo = 0.f, hi = 0.f;
          for (int q = 0; q < cfg.parts; ++q) {
            float a, b;
            asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(a), "=f"(b) : "r"(stage0 + (uint32_t)(((q * width + c) * 128 + ch) * 4)) : "memory");
            lo += a;
            hi += b;
          }
          uint32_t two;
          if (cfg.bf16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(two) : "f"(hi), "f"(lo));
          else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(two) : "f"(hi), "f"(lo));
          *reinterpret_cast<uint32_t*>(out + (size_t)c * p.d_pitch) = two;
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

// A tensor map of 16-bit values, boxes of 64 values (128 bytes, swizzled) by `box` rows: of a matrix [rows][cols] of rows `row` values apart, or with
// `mats` > 0 of that many of them.
inline int grouped_tensor_map(CUtensorMap* map, const void* data, int cols, int row, int rows, int mats, int box, bool bf16) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  const Encode encode = reinterpret_cast<Encode>(tensor_map_encoder());
  if (encode == nullptr) return -1000 - (int)CUDA_ERROR_NOT_FOUND;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)(mats > 0 ? mats : 1)};
  const cuuint64_t pitch[2] = {(cuuint64_t)row * 2, (cuuint64_t)row * 2 * (cuuint64_t)rows};
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

// Whether the kernel takes a call: what the tensor maps and the stores ask for; tiles (of 64 x 128 values at least) are counted in an int.
inline bool grouped_umma_takes(const GroupedParams& p, bool* shape) {
  const long long wide = p.c_in > p.c_out ? p.c_in : p.c_out, rows = (long long)p.n_rows > (long long)p.groups * p.c_in ? p.n_rows : (long long)p.groups * p.c_in;
  *shape = p.a_pitch % 8 == 0 && p.b_pitch % 8 == 0 && p.d_pitch % 8 == 0 && p.n_rows > 0 && (rows / 64 + p.groups) * (wide / 128 + 1) < 0x7fff0000ll;
  return *shape && ((reinterpret_cast<uintptr_t>(p.a) | reinterpret_cast<uintptr_t>(p.b) | reinterpret_cast<uintptr_t>(p.d)) & 15) == 0;
}

// A way to cut a product up.
struct GuCut {
  int cg, tile_n, parts;
};

// at most: no more groups have rows than there are rows
template <int PASS>
long long grouped_tiles(const GroupedParams& p, const GuCut& cut) {
  const int channels = PASS == GROUPED_DGRAD ? p.c_in : p.c_out;
  const long long m = (channels + 128 * cut.cg - 1) / (128 * cut.cg);
  if (PASS == GROUPED_WGRAD) return m * p.groups * ((p.c_in + cut.tile_n - 1) / cut.tile_n);
  return m * (p.n_rows / cut.tile_n + (p.n_rows < p.groups ? p.n_rows : p.groups));
}

// The cut that is expected to take the least time, from the sizes that the host knows: rows are taken to be spread evenly.
//
// Measured, microseconds (bf16, launches in a row; c, a stage of a tile: on an idle chip / on a full one):
//   n columns             64            128           256
//   one CTA          0.21 / 0.24   0.22 / 0.30   0.29 / 0.50
//   a pair           0.21 / 0.23   0.21 / 0.28   0.29 / 0.42
// and 4 for everything around it (a pair 0.8 more), 0.5 and 0.0055 a column for the epilogue, beside the next tile's stages.  So pairs of 256 columns
// where there is work for all: 16 groups of 1024 rows 2048 -> 2048 98 us, single CTAs 112, 128 columns 125 and 134; narrower tiles and single CTAs
// (of tiles that do as well the narrowest: they leave room for more stages, and 96 rows in 64 groups 2048 -> 1024 take 46.4 us instead of 50.4) where
// there is not: 1000 rows 1024 -> 1024 11.1 us, so 8.1; 4096 rows in 8 groups 512 -> 512 9.1, so 7.3.
// Parts: a cluster for every tile, whose CTAs share the contraction; 2 and 0.024 a column more for adding up.  One row 4096 -> 4096 17.4 us, with four
// parts 9.2; the gradient of a 256 x 256 matrix over 30000 rows 94, with eight parts 19; but only while all clusters run at once, as every further round of
// them starts from nothing (1000 rows 1024 -> 1024 with four parts 28).
inline float grouped_stage_us(int cg, float n, float load) {
  const float idle = n <= 128.f ? 0.2f + 0.02f * n / 128.f : 0.22f + 0.07f * (n - 128.f) / 128.f;
  const float full = cg == 2 ? (n <= 128.f ? 0.2f + 0.08f * n / 128.f : 0.28f + 0.14f * (n - 128.f) / 128.f)
                             : (n <= 128.f ? 0.2f + 0.1f * n / 128.f : 0.3f + 0.2f * (n - 128.f) / 128.f);
  return idle + (full - idle) * (load < 1.f ? load : 1.f);
}

template <int PASS, typename Clusters>
GuCut grouped_cut(const GroupedParams& p, int sms, Clusters clusters_at_once) {
  static constexpr GuCut CUTS[] = {{1, 64, 1},  {1, 128, 1}, {1, 256, 1}, {2, 128, 1}, {2, 256, 1}, {1, 32, 2},  {1, 64, 2},
                                   {1, 128, 2}, {1, 32, 4},  {1, 64, 4},  {1, 128, 4}, {1, 32, 8},  {1, 64, 8},  {1, 128, 8}};
  const int channels = PASS == GROUPED_DGRAD ? p.c_in : p.c_out;
  const float groups = (float)(PASS == GROUPED_WGRAD || p.groups < p.n_rows ? p.groups : p.n_rows), rows = (float)p.n_rows / groups;
  const float blocks = PASS == GROUPED_WGRAD ? rows / 64.f + 0.5f : (float)(((PASS == GROUPED_DGRAD ? p.c_out : p.c_in) + 63) / 64);
  GuCut best = CUTS[0];
  float least = 0.f;
  for (const GuCut& cut : CUTS) {
    if (cut.cg > sms) continue;
    const float m = (float)((channels + 128 * cut.cg - 1) / (128 * cut.cg)), width = (float)cut.tile_n;
    float tiles, n;
    if (PASS == GROUPED_WGRAD) {
      tiles = groups * (float)((p.c_in + cut.tile_n - 1) / cut.tile_n);
      n = p.c_in < cut.tile_n ? (float)p.c_in : width;
    } else {
      tiles = groups * (rows <= width ? 1.f : rows / width + 0.5f);
      n = rows < width ? rows : width;
    }
    tiles *= m;
    const float epilogue = 0.5f + 0.0055f * n, slots = (float)(sms / cut.cg);
    float us;
    if (cut.parts > 1) {
      if (blocks < 2.f * (float)cut.parts || grouped_tiles<PASS>(p, cut) > clusters_at_once(cut.parts)) continue;
      us = 4.f + blocks / (float)cut.parts * grouped_stage_us(1, n, tiles * (float)cut.parts / slots) + 2.f + 0.024f * n;
    } else {
      const float rounds = tiles <= slots ? 1.f : tiles / slots + 0.5f, tile = blocks * grouped_stage_us(cut.cg, n, tiles / slots);
      us = (cut.cg == 2 ? 4.8f : 4.f) + tile + (rounds - 1.f) * (tile > epilogue ? tile : epilogue) + epilogue;
    }
    if (least == 0.f || us < least) {
      least = us;
      best = cut;
    }
  }
  return best;
}

// The shared memory that the kernel may be launched with, always the most there is: a launch of a smaller size would set the limit down for a question
// about the largest (grouped_clusters_at_once), whose answer would then depend on which call came first.
template <int PASS, int CG, bool SPLIT>
int grant_grouped_umma(int max_smem) {
  static std::atomic<int> granted[64];
  return ensure_smem(grouped_umma_kernel<PASS, CG, SPLIT>, max_smem, granted);
}

template <int PASS, int CG, bool SPLIT>
int launch_grouped_umma_as(const GroupedParams& p, bool bf16, const GuCut& cut, cudaStream_t st, int sms, int max_smem) {
  GuConfig cfg;
  cfg.parts = SPLIT ? cut.parts : 1;
  cfg.tile_n = cut.tile_n;
  cfg.bf16 = bf16;
  const int b_bytes = PASS == GROUPED_WGRAD ? (cfg.tile_n / CG + 63) / 64 * 8192 : cfg.tile_n / CG * 128;
  cfg.stage_bytes = GU_A_BYTES + b_bytes;
  const int rest = 1024 + GU_EPI_WARPS / 4 * GU_PATCH_BYTES + GU_SHARED_BYTES + (3 * p.groups + 2) * (int)sizeof(int);
  cfg.stages = (max_smem - rest) / cfg.stage_bytes;
  if (cfg.stages > GU_MAX_STAGES) cfg.stages = GU_MAX_STAGES;
  if (cfg.stages < 2 || (SPLIT && cfg.stages * cfg.stage_bytes < (cfg.tile_n + cut.parts) * 512)) return -1;
  cfg.smem = rest + cfg.stages * cfg.stage_bytes;
  // SPLIT: a cluster for every tile there may be; otherwise pairs (or CTAs) go from tile to tile
  long long clusters = grouped_tiles<PASS>(p, cut);
  // By size: 20 ragged groups of 20000 rows 512 x 512 21.5 us, so 16.1; 16 of 16384 2048 x 1024 56.2 / 55.4.  More than 64 groups even out by themselves, and every
  // CTA ranks them: 300 of 3000 rows 512 x 512 42.6 / 45.1, 1000 128 x 256 43 / 90.
  cfg.by_size = PASS == GROUPED_WGRAD && !SPLIT && p.groups > 1 && p.groups <= 64 && clusters > sms / CG;
  if (!SPLIT && clusters > sms / CG) clusters = sms / CG;
  if (clusters < 1) clusters = 1;
  const int ctas = SPLIT ? cut.parts : CG;
  CUtensorMap a, b, b16;
  int rc;
  if (PASS == GROUPED_WGRAD) {  // p.a: in, p.b: out_grad
    rc = grouped_tensor_map(&a, p.b, p.c_out, p.b_pitch, p.n_rows, 0, 64, bf16);
    if (rc == 0) rc = grouped_tensor_map(&b, p.a, p.c_in, p.a_pitch, p.n_rows, 0, 64, bf16);
    b16 = b;
  } else {
    rc = grouped_tensor_map(&a, p.b, p.c_out, p.b_pitch, p.c_in, p.groups, PASS == GROUPED_FWD ? 64 : 128, bf16);
    const int width = PASS == GROUPED_FWD ? p.c_in : p.c_out;
    if (rc == 0) rc = grouped_tensor_map(&b, p.a, width, p.a_pitch, p.n_rows, 0, cfg.tile_n / CG, bf16);
    if (rc == 0) rc = grouped_tensor_map(&b16, p.a, width, p.a_pitch, p.n_rows, 0, 16, bf16);
  }
  if (rc != 0) return rc;
  if (grant_grouped_umma<PASS, CG, SPLIT>(max_smem) != 0) return -1;
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
  return cudaLaunchKernelEx(&lc, grouped_umma_kernel<PASS, CG, SPLIT>, p, cfg, a, b, b16) == cudaSuccess ? 0 : -1;
}

// Clusters of `parts` CTAs that the device runs at the same time, each with all of an SM's shared memory: clusters do not straddle its groups
// of SMs, so 128 CTAs in clusters of eight do not fit on 148.  Answered once a device (a question that failed is asked again); fewer SMs than
// all of them: in proportion.
template <int PASS>
int grouped_clusters_at_once(int parts, int sms, int max_smem) {
  static std::atomic<int> known[64][4];  // and one, 0: not known
  int dev = 0, all = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64 || parts < 2) return 0;
  std::atomic<int>& at = known[dev][parts == 2 ? 0 : parts == 4 ? 1 : 2];
  if (cudaDeviceGetAttribute(&all, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  int n = at.load(std::memory_order_acquire) - 1;
  if (n < 0) {
    if (grant_grouped_umma<PASS, 1, true>(max_smem) != 0) return 0;
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
    if (cudaOccupancyMaxActiveClusters(&n, grouped_umma_kernel<PASS, 1, true>, &lc) != cudaSuccess || n < 0) {
      cudaGetLastError();
      return 0;
    }
    at.store(n + 1, std::memory_order_release);
  }
  return n * sms / all;
}

template <int PASS>
int launch_grouped_umma_cut(const GroupedParams& p, bool bf16, const GuCut& cut, cudaStream_t st, int sms, int max_smem) {
  if (cut.parts > 1) return launch_grouped_umma_as<PASS, 1, true>(p, bf16, cut, st, sms, max_smem);
  return cut.cg == 2 ? launch_grouped_umma_as<PASS, 2, false>(p, bf16, cut, st, sms, max_smem)
                     : launch_grouped_umma_as<PASS, 1, false>(p, bf16, cut, st, sms, max_smem);
}

template <int PASS>
int launch_grouped_umma(const GroupedParams& p, bool bf16, cudaStream_t st, int sms, int max_smem) {
  const auto at_once = [&](int parts) { return grouped_clusters_at_once<PASS>(parts, sms, max_smem); };
  return launch_grouped_umma_cut<PASS>(p, bf16, grouped_cut<PASS>(p, sms, at_once), st, sms, max_smem);
}

}  // namespace fgms
