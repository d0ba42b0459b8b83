// A whole layer of experts for a few tokens, in two kernels:
//
//   logit[t, e] = x[t] . router[e]                        the top_k largest of a token, the lower index first where two are equal
//   gate[t, j]  = softmax of the chosen logits
//   u = x[t] . W_in[e]      h = act(u), or act(first half of u) * second half where W_in is twice as wide as W_out is high
//   out[t] = sum over j of gate[t, j] (h . W_out[e(t, j)])
//
// expert_logits_kernel has a block for an expert and eight tokens.  A choice hangs on the difference of two logits, so they are summed in 64 bits; every
// expert's in the same order, so that equal rows of the router are equal.
//
// expert_layer_kernel is cooperative, a CTA an SM.  What bounds it is the weights of the experts that some token goes to, each read once: a tile of a weight
// is 64 of the contraction by 128 columns (a TMA copy for each 64 of them, a ring of tiles ahead), and the tiles of all experts, column blocks and
// contractions are one list, cut into as many equal shares as there are CTAs.  A share may start and end inside a column block: whoever has the
// block's first tile adds what the others hand over, in their order, so that the sums are the same bits on every run.  The products are
// mma.sync.m16n8k16 with the columns of the weight as M and an expert's tokens as N, eight a step (rows that are no token are computed and thrown
// away): beside 16 KB from memory, 0.35 us of an SM's share, eight steps for each of up to eight such groups are nothing.
//
//   warps 0-7   tokens' rows (cp.async, three tiles ahead), products, activation          warp 8   TMA producer
//
// The producer goes on to W_out while the others wait for the last h: what a grid barrier costs, the ring has bridged.  All waits are bounded.
#pragma once
#include "grouped_umma.cuh"
#include "row_values.cuh"

namespace fgms {

constexpr int EL_MAX_TOKENS = 64, EL_MAX_TOP_K = 16, EL_MAX_EXPERTS = 512;
constexpr int EL_MAX_PAIRS = EL_MAX_TOKENS * EL_MAX_TOP_K;
constexpr int EL_K = 64;                           // contraction of a tile
constexpr int EL_TILE_BYTES = EL_K * 128 * 2;      // two blocks of 64 columns
constexpr int EL_MAX_STAGES = 12;
constexpr int EL_X_STAGES = 4;                     // tokens' rows: 64 values each
constexpr int EL_X_BYTES = EL_MAX_TOKENS * EL_K * 2;
constexpr int EL_CONSUMERS = 256, EL_THREADS = EL_CONSUMERS + 32;
constexpr int EL_SLOT = EL_CONSUMERS * 32;         // fp32 sums that a CTA may hand over
constexpr int EL_ROUTER_THREADS = 128, EL_ROUTER_TOKENS = 8;

struct ExpertParams {
  const void *x, *router;
  void* out;
  int32_t* experts;  // [tokens][top_k]
  float* gates;      // [tokens][top_k]
  int tokens, n_experts, top_k, width, hidden, out_width, gated, activation;  // activation: 0 relu, 1 silu
  long long x_pitch, out_pitch;
  // workspace
  double* logits;    // [tokens][n_experts]
  uint32_t* flags;   // [2][ctas], a share's sums are there; then [3], CTAs that have arrived at a barrier
  float* slots;      // [ctas][EL_SLOT]
  uint16_t* h;       // [tokens top_k][hidden], in the order of the experts
  float* part;       // [tokens top_k][out_width]
  int ctas, stages, bf16;
  bool x_vec;
  int alone;
};

template <typename T, typename R>
__global__ void __launch_bounds__(EL_ROUTER_THREADS) expert_logits_kernel(const __grid_constant__ ExpertParams p) {
  __shared__ double sums[EL_ROUTER_TOKENS][EL_ROUTER_THREADS / 32];
  umma::griddep_wait();
  if (!p.alone) umma::griddep_launch_dependents();
  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (int i = threadIdx.x; i < 2 * p.ctas + 3; i += EL_ROUTER_THREADS) p.flags[i] = 0u;
  const int e = (int)blockIdx.x, t0 = (int)blockIdx.y * EL_ROUTER_TOKENS, n = min(EL_ROUTER_TOKENS, p.tokens - t0);
  double sum[EL_ROUTER_TOKENS];
#pragma unroll
  for (int t = 0; t < EL_ROUTER_TOKENS; ++t) sum[t] = 0.0;
  const R* row = static_cast<const R*>(p.router) + (size_t)e * p.width;
  for (int col = (int)threadIdx.x * ROW_CHUNK; col < p.width; col += EL_ROUTER_THREADS * ROW_CHUNK) {  // the width is a multiple of a chunk
    const RowRaw<R> w = row_load(row + col, ROW_CHUNK, true);
    double wd[ROW_CHUNK];
#pragma unroll
    for (int i = 0; i < ROW_CHUNK; ++i) wd[i] = (double)row_value(w, i);
#pragma unroll
    for (int t = 0; t < EL_ROUTER_TOKENS; ++t) {
      if (t >= n) break;
      const RowRaw<T> x = row_load(static_cast<const T*>(p.x) + (t0 + t) * p.x_pitch + col, ROW_CHUNK, p.x_vec);
#pragma unroll
      for (int i = 0; i < ROW_CHUNK; ++i) sum[t] += (double)row_value(x, i) * wd[i];
    }
  }
#pragma unroll
  for (int t = 0; t < EL_ROUTER_TOKENS; ++t) {
    if (t >= n) break;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum[t] += __shfl_xor_sync(0xffffffffu, sum[t], o);
    if ((threadIdx.x & 31) == 0) sums[t][threadIdx.x >> 5] = sum[t];
  }
  __syncthreads();
  if ((int)threadIdx.x < n) {
    double v = 0.0;
#pragma unroll
    for (int i = 0; i < EL_ROUTER_THREADS / 32; ++i) v += sums[threadIdx.x][i];
    p.logits[(size_t)(t0 + threadIdx.x) * p.n_experts + e] = v;
  }
}

struct ElShared {
  uint64_t full[EL_MAX_STAGES], empty[EL_MAX_STAGES];
  int abort_flag, used;
  float gates[EL_MAX_PAIRS];
  uint16_t chosen[EL_MAX_PAIRS], list[EL_MAX_PAIRS];        // pairs: token * top_k + j; list: in the order of their experts
  uint16_t count[EL_MAX_EXPERTS], place[EL_MAX_EXPERTS];    // of an expert: pairs, and the next one's place in the list
  uint16_t expert[EL_MAX_EXPERTS], first[EL_MAX_EXPERTS + 1];  // of those that are used: which, and the first pair's place
};

// A share of the list of tiles: tile `at` is contraction step kb of column block m of the used expert u.
struct ElWalk {
  int at, end, u, m, kb, steps, blocks;
  __device__ __forceinline__ ElWalk(int from, int to, int blocks_, int steps_) : at(from), end(to), steps(steps_), blocks(blocks_) {
    const int block = from / steps;
    kb = from - block * steps;
    u = block / blocks;
    m = block - u * blocks;
  }
  __device__ __forceinline__ bool left() const { return at < end; }
  __device__ __forceinline__ void next() {
    ++at;
    if (++kb == steps) {
      kb = 0;
      if (++m == blocks) {
        m = 0;
        ++u;
      }
    }
  }
};
__device__ __forceinline__ int el_share(int total, int cta, int ctas) { return (int)((long long)total * cta / ctas); }

__device__ __forceinline__ void el_sync() { asm volatile("barrier.cta.sync 1, %0;" ::"n"(EL_CONSUMERS) : "memory"); }
__device__ __forceinline__ uint32_t el_acquire(const uint32_t* at) {
  uint32_t v;
  asm volatile("ld.acquire.gpu.global.b32 %0, [%1];" : "=r"(v) : "l"(at) : "memory");
  return v;
}
// until *at is `want` at least
__device__ __forceinline__ bool el_await(const uint32_t* at, uint32_t want, volatile int* abort_flag) {
  const long long start = clock64();
  while (el_acquire(at) < want) {
    if (*abort_flag) return false;
    if (clock64() - start > umma::WAIT_LIMIT_CYCLES) {
      *abort_flag = 1;
      return false;
    }
  }
  return true;
}
// All consumers of all CTAs: what was written before is there behind it.
__device__ __forceinline__ void el_grid_sync(uint32_t* counter, int ctas, volatile int* abort_flag) {
  el_sync();
  if (threadIdx.x == 0) {
    __threadfence();
    atomicAdd(counter, 1u);
    el_await(counter, (uint32_t)ctas, abort_flag);
    __threadfence();
  }
  el_sync();
}

__device__ __forceinline__ void el_ldmatrix(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void el_ldmatrix_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <bool BF16>
__device__ __forceinline__ void el_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float el_activated(int activation, float v) { return activation == 0 ? (v != v ? v : fmaxf(v, 0.f)) : v / (1.f + __expf(-v)); }
template <bool BF16>
__device__ __forceinline__ uint16_t el_round(float v) {
  return BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}

// The top_k largest logits of a token, by a warp: (*expert, *gate) of lane j are the j-th one's.  A logit that is not a number counts as minus infinity (and
// makes the gates such).
__device__ __forceinline__ void el_choose(const ExpertParams& p, int t, int* expert, float* gate) {
  const int lane = threadIdx.x & 31;
  constexpr int EACH = EL_MAX_EXPERTS / 32;
  const double lowest = __longlong_as_double((long long)0xfff0000000000000ull);
  double v[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    v[i] = lowest;
    if (lane + 32 * i < p.n_experts) {
      v[i] = __ldcg(p.logits + (size_t)t * p.n_experts + lane + 32 * i);
      if (!(v[i] >= lowest)) v[i] = lowest;
    }
  }
  uint32_t taken = 0;
  double top = 0.0;
  float mine = 0.f, total = 0.f;
  for (int j = 0; j < p.top_k; ++j) {
    double best = lowest;
    int at = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      if (32 * i >= p.n_experts) break;
      const int e = lane + 32 * i;
      if (e < p.n_experts && !(taken >> i & 1u) && (v[i] > best || (v[i] == best && e < at))) {
        best = v[i];
        at = e;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double other = __shfl_xor_sync(0xffffffffu, best, o);
      const int where = __shfl_xor_sync(0xffffffffu, at, o);
      if (other > best || (other == best && where < at)) {
        best = other;
        at = where;
      }
    }
    if ((at & 31) == lane) taken |= 1u << (at >> 5);
    if (j == 0) top = best;
    const float share = expf((float)(best - top));
    total += share;
    if (lane == j) {
      mine = share;
      *expert = at;
    }
  }
  *gate = mine / total;
}
// Of all tokens, in every CTA.  Up to EL_CHOOSE_ALONE tokens each CTA does it for itself, two rounds of its warps at most; more are dealt out, a token
// a CTA, and met at a grid barrier, which costs as much as two or three rounds.
constexpr int EL_CHOOSE_ALONE = 2 * EL_THREADS / 32;
__device__ __forceinline__ void el_choose_all(const ExpertParams& p, ElShared* sh) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cta = (int)blockIdx.x;
  const bool alone = p.tokens <= EL_CHOOSE_ALONE;
  for (int t = alone ? warp : cta; t < p.tokens && (alone || warp == 0); t += alone ? EL_THREADS / 32 : p.ctas) {
    int expert = 0;
    float gate = 0.f;
    el_choose(p, t, &expert, &gate);
    if (lane >= p.top_k) continue;
    const int pair = t * p.top_k + lane;
    sh->chosen[pair] = (uint16_t)expert;
    sh->gates[pair] = gate;
    if (!alone || cta == 0) {
      __stcg(p.experts + pair, expert);
      __stcg(p.gates + pair, gate);
    }
  }
  if (!alone) {
    if (warp < EL_CONSUMERS / 32) {
      el_grid_sync(p.flags + 2 * p.ctas + 2, p.ctas, &sh->abort_flag);
      for (int i = threadIdx.x; i < p.tokens * p.top_k; i += EL_CONSUMERS) {
        // (a value that no CTA has written, after a wait that ran out, is no expert)
        sh->chosen[i] = (uint16_t)min(max(__ldcg(p.experts + i), 0), p.n_experts - 1);
        sh->gates[i] = __ldcg(p.gates + i);
      }
    }
  }
  __syncthreads();
}

// The pairs in the order of their experts (of an expert: of the tokens), by one warp.
__device__ __forceinline__ void el_sort(const ExpertParams& p, ElShared* sh) {
  const int lane = threadIdx.x & 31, pairs = p.tokens * p.top_k;
  for (int e = lane; e < p.n_experts; e += 32) sh->count[e] = 0;
  __syncwarp();
  for (int i0 = 0; i0 < pairs; i0 += 32) {
    const int e = i0 + lane < pairs ? (int)sh->chosen[i0 + lane] : 0x10000 + lane;  // no pair: equal to none
    const uint32_t peers = __match_any_sync(0xffffffffu, e);
    if (i0 + lane < pairs && (peers >> lane) == 1u) sh->count[e] += (uint16_t)__popc(peers);  // the last of its expert
    __syncwarp();
  }
  int used = 0, first = 0;
  for (int e0 = 0; e0 < p.n_experts; e0 += 32) {
    const int n = e0 + lane < p.n_experts ? (int)sh->count[e0 + lane] : 0;
    const uint32_t some = __ballot_sync(0xffffffffu, n > 0);
    int before = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += v;
    }
    const int place = first + before - n;
    if (n > 0) {
      const int u = used + __popc(some & ((1u << lane) - 1u));
      sh->expert[u] = (uint16_t)(e0 + lane);
      sh->first[u] = (uint16_t)place;
      sh->place[e0 + lane] = (uint16_t)place;
    }
    used += __popc(some);
    first += __shfl_sync(0xffffffffu, before, 31);
  }
  if (lane == 0) {
    sh->used = used;
    sh->first[used] = (uint16_t)pairs;
  }
  __syncwarp();
  for (int i0 = 0; i0 < pairs; i0 += 32) {
    const int e = i0 + lane < pairs ? (int)sh->chosen[i0 + lane] : 0x10000 + lane;
    const uint32_t peers = __match_any_sync(0xffffffffu, e);
    int place = 0;
    if (i0 + lane < pairs) {
      place = (int)sh->place[e] + __popc(peers & ((1u << lane) - 1u));
      sh->list[place] = (uint16_t)(i0 + lane);
    }
    __syncwarp();
    if (i0 + lane < pairs && (peers >> lane) == 1u) sh->place[e] = (uint16_t)(place + 1);
    __syncwarp();
  }
}

template <bool BF16>
__global__ void __launch_bounds__(EL_THREADS, 1)
    expert_layer_kernel(const __grid_constant__ ExpertParams p, const __grid_constant__ CUtensorMap map_in, const __grid_constant__ CUtensorMap map_out) {
  using namespace umma;
  extern __shared__ uint8_t el_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(el_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  ElShared* sh = reinterpret_cast<ElShared*>(smem + (size_t)p.stages * EL_TILE_BYTES + EL_X_STAGES * EL_X_BYTES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cta = (int)blockIdx.x;
  volatile int* abort_flag = &sh->abort_flag;
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(smem_u32(&sh->full[s]), 1);
      mbar_init(smem_u32(&sh->empty[s]), EL_CONSUMERS / 32);
    }
    sh->abort_flag = 0;
    mbar_fence_init();
  }
  __syncthreads();
  el_choose_all(p, sh);
  if (warp == 0) el_sort(p, sh);
  __syncthreads();
  const int used = sh->used;
  const uint32_t tiles0 = smem_u32(smem), x0 = tiles0 + (uint32_t)(p.stages * EL_TILE_BYTES);
  // of the two products: steps of the contraction, blocks of columns, tiles
  const int columns = p.gated ? 64 : 128;  // of h that a block stands for
  int steps[2] = {(p.width + EL_K - 1) / EL_K, (p.hidden + EL_K - 1) / EL_K};
  int blocks[2] = {(p.hidden + columns - 1) / columns, (p.out_width + 127) / 128};
  bool ok = true;

  if (warp == EL_CONSUMERS / 32) {
    // ------------------------------------------------------------------ producer
    if (elect_one()) {
      int s = 0;
      uint32_t ph = 1;
      for (int product = 0; product < 2 && ok; ++product) {
        const int total = used * blocks[product] * steps[product];
        const CUtensorMap* map = product == 0 ? &map_in : &map_out;
        const int second = product == 0 && p.gated ? p.hidden : 64, width = product == 0 ? columns : 128;
        for (ElWalk w(el_share(total, cta, p.ctas), el_share(total, cta + 1, p.ctas), blocks[product], steps[product]); w.left(); w.next()) {
          ok = mbar_parked_wait(smem_u32(&sh->empty[s]), ph, abort_flag);
          if (!ok) break;
          const uint32_t to = tiles0 + (uint32_t)(s * EL_TILE_BYTES), bar = smem_u32(&sh->full[s]);
          const int e = sh->expert[w.u];
          mbar_expect_tx(bar, EL_TILE_BYTES);
          pair_load_3d<1>(to, map, bar, w.m * width, w.kb * EL_K, e);
          pair_load_3d<1>(to + EL_TILE_BYTES / 2, map, bar, w.m * width + second, w.kb * EL_K, e);
          if (++s == p.stages) { s = 0; ph ^= 1u; }
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ consumers
    const int g = lane >> 2, c = lane & 3;  // of a fragment: column of the weight; pair of tokens
    int s = 0;
    uint32_t ph = 0;
    for (int product = 0; product < 2; ++product) {
      if (product == 1) el_grid_sync(p.flags + 2 * p.ctas, p.ctas, abort_flag);
      const int total = used * blocks[product] * steps[product], from = el_share(total, cta, p.ctas), to = el_share(total, cta + 1, p.ctas);
      const bool gated = product == 0 && p.gated;
      uint32_t* flags = p.flags + product * p.ctas;
      // a warp's 16 columns: two groups of eight, side by side, or one of each half
      const int block_a = gated ? 0 : warp >> 2, chunk_a = gated ? warp : (warp & 3) * 2, block_b = gated ? 1 : block_a, chunk_b = gated ? warp : chunk_a + 1;
      ElWalk ahead(from, to, blocks[product], steps[product]);
      int x_slot = 0;
      const auto fetch = [&] {  // the rows of the expert's tokens that the next tile is multiplied with
        if (ahead.left()) {
          const int first = sh->first[ahead.u], n = sh->first[ahead.u + 1] - first, k0 = ahead.kb * EL_K;
          const int width = product == 0 ? p.width : p.hidden;
          for (int i = threadIdx.x; i < n * 8; i += EL_CONSUMERS) {
            const int row = i >> 3, chunk = i & 7, k = k0 + chunk * 8;
            const uint16_t* src;
            if (product == 0) src = static_cast<const uint16_t*>(p.x) + (size_t)(sh->list[first + row] / (uint32_t)p.top_k) * p.x_pitch;
            else src = p.h + (size_t)(first + row) * p.hidden;
            cp_async16(x0 + (uint32_t)(x_slot * EL_X_BYTES + row * 128 + (chunk ^ (row & 7)) * 16), k < width ? src + k : src, k < width);
          }
          ahead.next();
        }
        cp_async_commit();
        x_slot = (x_slot + 1) % EL_X_STAGES;
      };
#pragma unroll
      for (int i = 0; i < EL_X_STAGES - 1; ++i) fetch();
      float acc[8][4];
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
      int head = from;  // where the segment in `acc` began
      int x_at = 0;
      for (ElWalk w(from, to, blocks[product], steps[product]); w.left(); w.next()) {
        cp_async_wait<EL_X_STAGES - 2>();
        el_sync();  // all have the tile's rows, and are done with the last one's
        fetch();
        const int first = sh->first[w.u], n = sh->first[w.u + 1] - first;
        if (ok) ok = mbar_parked_wait(smem_u32(&sh->full[s]), ph, abort_flag);
        const uint32_t tile = tiles0 + (uint32_t)(s * EL_TILE_BYTES), x = x0 + (uint32_t)(x_at * EL_X_BYTES);
        {
          const int matrix = lane >> 3, row = lane & 7;
          const uint32_t block = (matrix & 1 ? block_b : block_a) * (EL_TILE_BYTES / 2), chunk = (matrix & 1 ? chunk_b : chunk_a) ^ row;
          const uint32_t weights = tile + block + (uint32_t)((matrix >> 1) * 8 + row) * 128u + chunk * 16u;
          uint32_t a[4][4];
#pragma unroll
          for (int k = 0; k < 4; ++k) el_ldmatrix_trans(a[k], weights + (uint32_t)k * 2048u);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (j * 8 >= n) break;
            uint32_t b[4];
            const uint32_t tokens = x + (uint32_t)((j * 8 + row) * 128);
            el_ldmatrix(b, tokens + (uint32_t)((matrix ^ row) * 16));
            el_mma<BF16>(acc[j], a[0], b[0], b[1]);
            el_mma<BF16>(acc[j], a[1], b[2], b[3]);
            el_ldmatrix(b, tokens + (uint32_t)(((matrix + 4) ^ row) * 16));
            el_mma<BF16>(acc[j], a[2], b[0], b[1]);
            el_mma<BF16>(acc[j], a[3], b[2], b[3]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh->empty[s]));
        if (++s == p.stages) { s = 0; ph ^= 1u; }
        x_at = (x_at + 1) % EL_X_STAGES;
        const bool last = w.kb + 1 == steps[product];
        if (!last && w.at + 1 < to) continue;
        // ---------------------------------------------------------------- the end of a segment
        const int block_first = w.at - w.kb, block_end = block_first + steps[product];
        if (head != block_first) {  // the first segment of this share: its sums go to whoever has the block's first tile
          float* slot = p.slots + (size_t)cta * EL_SLOT + threadIdx.x;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (j * 8 >= n) break;
#pragma unroll
            for (int i = 0; i < 4; ++i) __stcg(slot + (j * 4 + i) * EL_CONSUMERS, acc[j][i]);
          }
          el_sync();
          if (threadIdx.x == 0) {
            __threadfence();
            asm volatile("st.release.gpu.global.b32 [%0], %1;" ::"l"(flags + cta), "r"(1u) : "memory");
          }
        } else {
          if (!last) {
            int others = 0;  // shares behind this one that begin inside the block
            while (cta + 1 + others < p.ctas && el_share(total, cta + 1 + others, p.ctas) < block_end) ++others;
            for (int i = threadIdx.x; i < others; i += EL_CONSUMERS) {
              const int o = cta + 1 + i;
              if (el_share(total, o, p.ctas) < el_share(total, o + 1, p.ctas)) el_await(flags + o, 1u, abort_flag);
            }
            __threadfence();
            el_sync();
            for (int i = 0; i < others; ++i) {
              const int o = cta + 1 + i;
              if (el_share(total, o, p.ctas) == el_share(total, o + 1, p.ctas)) continue;
              const float* slot = p.slots + (size_t)o * EL_SLOT + threadIdx.x;
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                if (j * 8 >= n) break;
#pragma unroll
                for (int q = 0; q < 4; ++q) acc[j][q] += __ldcg(slot + (j * 4 + q) * EL_CONSUMERS);
              }
            }
          }
          // the block's sums are whole
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (j * 8 >= n) break;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int token = j * 8 + c * 2 + i;
              if (token >= n) continue;
              if (product == 0) {
                uint16_t* row = p.h + (size_t)(first + token) * p.hidden;
                if (gated) {
                  const int col = w.m * 64 + warp * 8 + g;
                  if (col < p.hidden) row[col] = el_round<BF16>(el_activated(p.activation, acc[j][i]) * acc[j][2 + i]);
                } else {
                  const int col = w.m * 128 + warp * 16 + g;
                  if (col < p.hidden) row[col] = el_round<BF16>(el_activated(p.activation, acc[j][i]));
                  if (col + 8 < p.hidden) row[col + 8] = el_round<BF16>(el_activated(p.activation, acc[j][2 + i]));
                }
              } else {
                const int pair = sh->list[first + token], col = w.m * 128 + warp * 16 + g;
                const float gate = sh->gates[pair];
                float* row = p.part + (size_t)pair * p.out_width;
                if (col < p.out_width) __stcg(row + col, gate * acc[j][i]);
                if (col + 8 < p.out_width) __stcg(row + col + 8, gate * acc[j][2 + i]);
              }
            }
          }
        }
        head = w.at + 1;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
      }
      cp_async_wait_all();
    }
    // ------------------------------------------------------------------ the sum over a token's experts
    el_grid_sync(p.flags + 2 * p.ctas + 1, p.ctas, abort_flag);
    const int per_row = p.out_width / 4;  // the width is a multiple of eight
    for (int i = cta * EL_CONSUMERS + (int)threadIdx.x; i < p.tokens * per_row; i += p.ctas * EL_CONSUMERS) {
      const int t = i / per_row, col = (i - t * per_row) * 4;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int j = 0; j < p.top_k; ++j) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(p.part + (size_t)(t * p.top_k + j) * p.out_width + col));
        sum.x += v.x;
        sum.y += v.y;
        sum.z += v.z;
        sum.w += v.w;
      }
      uint16_t* to = static_cast<uint16_t*>(p.out) + (size_t)t * p.out_pitch + col;
      const uint16_t r[4] = {el_round<BF16>(sum.x), el_round<BF16>(sum.y), el_round<BF16>(sum.z), el_round<BF16>(sum.w)};
      if ((reinterpret_cast<uintptr_t>(to) & 7) == 0) {
        *reinterpret_cast<uint2*>(to) = make_uint2((uint32_t)r[0] | (uint32_t)r[1] << 16, (uint32_t)r[2] | (uint32_t)r[3] << 16);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) to[q] = r[q];
      }
    }
  }
  if (*abort_flag && lane == 0) report_problem();
  if (*abort_flag) {  // copies may still be on their way into this CTA's memory
    const long long start = clock64();
    while (clock64() - start < 2000000) __nanosleep(1000);
  }
}

// Bytes of workspace, and where its parts begin.
struct ExpertSpace {
  size_t logits, flags, slots, h, part, total;
};
inline ExpertSpace expert_space(int tokens, int experts, int top_k, int hidden, int out_width, int ctas) {
  ExpertSpace s;
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  s.logits = take((size_t)tokens * experts * sizeof(double));
  s.flags = take((size_t)(2 * ctas + 3) * sizeof(uint32_t));
  s.slots = take((size_t)ctas * EL_SLOT * sizeof(float));
  s.h = take((size_t)tokens * top_k * hidden * 2);
  s.part = take((size_t)tokens * top_k * out_width * sizeof(float));
  s.total = at;
  return s;
}

template <typename T, typename R>
cudaError_t launch_expert_logits(const ExpertParams& p, cudaStream_t st) {
  return launch_pdl(expert_logits_kernel<T, R>, dim3((unsigned)p.n_experts, (unsigned)((p.tokens + EL_ROUTER_TOKENS - 1) / EL_ROUTER_TOKENS)), EL_ROUTER_THREADS, 0, st, p);
}

template <bool BF16>
int launch_expert_layer(ExpertParams p, const void* w_in, const void* w_out, cudaStream_t st, int max_smem) {
  const int rest = 1024 + EL_X_STAGES * EL_X_BYTES + (int)sizeof(ElShared);
  p.stages = (max_smem - rest) / EL_TILE_BYTES;
  if (p.stages > EL_MAX_STAGES) p.stages = EL_MAX_STAGES;
  if (p.stages < 2) return -1;
  const int smem = rest + p.stages * EL_TILE_BYTES;
  CUtensorMap in, out;
  const int wide = p.gated ? 2 * p.hidden : p.hidden;
  int rc = grouped_tensor_map(&in, w_in, wide, wide, p.width, p.n_experts, EL_K, BF16);
  if (rc == 0) rc = grouped_tensor_map(&out, w_out, p.out_width, p.out_width, p.hidden, p.n_experts, EL_K, BF16);
  if (rc != 0) return rc;
  static std::atomic<int> granted[64];
  if (ensure_smem(expert_layer_kernel<BF16>, max_smem, granted) != 0) return -1;
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3((unsigned)p.ctas);
  lc.blockDim = dim3(EL_THREADS);
  lc.dynamicSmemBytes = (size_t)smem;
  lc.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeCooperative;  // its CTAs wait on one another
  at[0].val.cooperative = 1;
  lc.attrs = at;
  lc.numAttrs = 1;
  return cudaLaunchKernelEx(&lc, expert_layer_kernel<BF16>, p, in, out) == cudaSuccess ? 0 : -1;
}

}  // namespace fgms
