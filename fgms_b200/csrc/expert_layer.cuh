// A whole layer of experts for a few tokens, in two kernels:
//
//   logit[t, e] = x[t] . router[e]                        the top_k largest of a token, the lower index first where two are equal
//   gate[t, j]  = softmax of the chosen logits
//   u = x[t] . W_in[e]      h = act(u), or act(first half of u) * second half where W_in is twice as wide as W_out is high
//   out[t] = sum over j of gate[t, j] (h . W_out[e(t, j)])
//
// expert_choice_kernel has a cluster of up to eight CTAs for a token, a warp for an expert at a time; the logits meet in the first one's shared memory.  A choice
// hangs on the difference of two logits, so they are summed in 64 bits; every expert's in the same order, so that equal rows of the router are equal.
//
// expert_layer_kernel is cooperative, a CTA an SM.  What bounds it is the weights of the experts that some token goes to, each read once.  An item
// is 64 columns of one expert's weight (gated: 32 of either half of u) with the whole contraction, in tiles of 128 rows that come by TMA, a
// ring of them ahead; items go around the CTAs, first those of W_in, then those of W_out, so that neighbours read neighbouring columns at about the same time.  No sum
// crosses CTAs, and the same bits come out on every run: contractions that were shared by CTAs cost 5 us a product in handing sums over, and a barrier of all
// CTAs between the products as much again.  Instead an item of W_out waits for the items of its expert alone, and whoever finishes a
// column block of the output last adds up what the token's experts left there.  The products are mma.sync.m16n8k16 with the columns of the weight as M and an
// expert's tokens as N, eight a step (rows that are no token are computed and thrown away).  h is held as the sum of two values of the type, its rounding
// and what that left, and multiplied twice: rounded once, the output was off by 2^-8.6 in bf16 where its own rounding is 2^-9.2, and the tensor cores have
// nothing else to do.
//
//   warps 0-7   products: 16 rows of every tile each; their sums meet in shared memory at the end of an item
//   warp 8      TMA producer of weights          warp 9   producer of the tokens' rows (cp.async: as a bulk copy a row and tile, 56 ns each, 64 tokens took
//               a tile ten times as long as its weights)
//   warps 10-11 report finished items and add the output up: a report waits until all that was stored is there, a microsecond that the products go on in
//
// All waits are bounded.  bf16: one token, 2 of 8 experts 512 x 1024, 16.4 to 18.2 us, which is latency; 16 tokens, 4 of 64 experts 2048 x 1024 each, 517 MB of weights, 96 to 101 us (79
// at the measured copy rate), 5.6 TB/s between the first tile and the last; 64 tokens, 2 of 32 experts 1024 x 2048 without a gate, 264 MB, 72 us (40).  With 33 tokens an expert and
// more the products take longer than the weights' way: 64 tokens, all of 4 experts 2048 x 1024, 86 us.
#pragma once
#include "grouped_umma.cuh"
#include "row_values.cuh"

namespace fgms {

constexpr int EL_MAX_TOKENS = 64, EL_MAX_TOP_K = 16, EL_MAX_EXPERTS = 512;
constexpr int EL_MAX_PAIRS = EL_MAX_TOKENS * EL_MAX_TOP_K;
constexpr int EL_K = 128, EL_COLUMNS = 64;         // a tile
constexpr int EL_TILE_BYTES = EL_K * EL_COLUMNS * 2;
constexpr int EL_MAX_STAGES = 12;
constexpr int EL_X_PITCH = EL_K * 2 + 16;          // tokens' rows, 16 bytes more apart than they are long so that eight of them lie in all banks
constexpr int EL_CONSUMERS = 256, EL_REPORTERS = 64, EL_THREADS = EL_CONSUMERS + 64 + EL_REPORTERS, EL_WARPS = EL_THREADS / 32;
constexpr int EL_SUMS = 16;                        // of a thread for eight tokens: 64 columns by eight a warp
constexpr int EL_ROUTER_THREADS = 256, EL_ROUTER_AT_ONCE = 4;  // chunks of a row whose loads are on their way together

struct ExpertParams {
  const void *x, *router;
  void* out;
  int32_t* experts;  // [tokens][top_k]
  float* gates;      // [tokens][top_k]
  int tokens, n_experts, top_k, width, hidden, out_width, gated, activation;  // activation: 0 relu, 1 silu
  long long x_pitch, out_pitch;
  // workspace
  uint32_t* flags;   // [experts]: items of W_in that are done, by used expert; [blocks of the output]: items of W_out
  uint16_t* h;       // [tokens top_k][2][hidden], in the order of the experts: rounded, and the remainders
  float* part;       // [tokens top_k][out_width]
  int ctas, n_flags, ring_bytes;  // ring_bytes: of shared memory, for weights and tokens' rows
  int alone;
};

// The top_k largest logits of a token, by a warp: (*expert, *gate) of lane j are the j-th one's.  A logit that is not a number counts as minus infinity (where
// the largest is that, the gates are not numbers).
template <int EACH>
__device__ __forceinline__ void el_choose(const ExpertParams& p, const double* logits, int* expert, float* gate) {
  const int lane = threadIdx.x & 31;
  // as numbers without a sign that are ordered alike; 0 is what has been taken
  unsigned long long v[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    v[i] = 0;
    if (lane + 32 * i < p.n_experts) {
      const double x = logits[lane + 32 * i] + 0.0;  // no minus zero
      const unsigned long long bits = (unsigned long long)__double_as_longlong(x);
      v[i] = x != x ? 0x000fffffffffffffull : bits >> 63 ? ~bits : bits | 0x8000000000000000ull;  // minus infinity is 0x000f...f
    }
  }
  double top = 0.0;
  float mine = 0.f, total = 0.f;
  for (int j = 0; j < p.top_k; ++j) {
    unsigned long long best = v[0];
#pragma unroll
    for (int i = 1; i < EACH; ++i) {
      if (32 * i >= p.n_experts) break;
      best = max(best, v[i]);
    }
    // the largest of the warp's, half by half
    const uint32_t high = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32));
    const uint32_t low = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32) == high ? (uint32_t)best : 0u);
    best = (unsigned long long)high << 32 | low;
    uint32_t at = 0xffffffffu;
#pragma unroll
    for (int i = EACH - 1; i >= 0; --i)
      if (32 * i < p.n_experts && v[i] == best && lane + 32 * i < p.n_experts) at = (uint32_t)(lane + 32 * i);
    at = __reduce_min_sync(0xffffffffu, at);
#pragma unroll
    for (int i = 0; i < EACH; ++i)
      if (at == (uint32_t)(lane + 32 * i)) v[i] = 0;
    const double value = __longlong_as_double((long long)(best >> 63 ? best & 0x7fffffffffffffffull : ~best));
    if (j == 0) top = value;
    const float share = expf((float)(value - top));
    total += share;
    if (lane == j) {
      mine = share;
      *expert = (int)at;
    }
  }
  *gate = mine / total;
}
template <typename T, typename R>
__global__ void __launch_bounds__(EL_ROUTER_THREADS) expert_choice_kernel(const __grid_constant__ ExpertParams p) {
  __shared__ double logits[EL_MAX_EXPERTS];
  umma::cluster_arrive();  // another CTA's shared memory is written only once that CTA is known to run; the kernel before this one is waited for meanwhile
  umma::griddep_wait();
  umma::cluster_wait();
  if (!p.alone) umma::griddep_launch_dependents();
  uint32_t rank, size;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(size));
  const int t = (int)(blockIdx.x / size), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < p.n_flags; i += EL_ROUTER_THREADS) p.flags[i] = 0u;
  const T* x_row = static_cast<const T*>(p.x) + t * p.x_pitch;
  for (int e = (int)rank + (int)size * warp; e < p.n_experts; e += (int)size * (EL_ROUTER_THREADS / 32)) {
    const R* row = static_cast<const R*>(p.router) + (size_t)e * p.width;
    double sum[EL_ROUTER_AT_ONCE] = {};
    for (int col = lane * ROW_CHUNK; col < p.width; col += 32 * ROW_CHUNK * EL_ROUTER_AT_ONCE) {  // the width is a multiple of a chunk
      RowRaw<R> w[EL_ROUTER_AT_ONCE];
      RowRaw<T> x[EL_ROUTER_AT_ONCE];
#pragma unroll
      for (int i = 0; i < EL_ROUTER_AT_ONCE; ++i) {
        const int at = col + i * 32 * ROW_CHUNK;
        w[i] = row_load(row + at, at < p.width ? ROW_CHUNK : 0, true);
        x[i] = row_load(x_row + at, at < p.width ? ROW_CHUNK : 0, true);
      }
#pragma unroll
      for (int k = 0; k < ROW_CHUNK; ++k)
#pragma unroll
        for (int i = 0; i < EL_ROUTER_AT_ONCE; ++i) sum[i] += (double)row_value(x[i], k) * (double)row_value(w[i], k);
    }
    double v = (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) {
      uint32_t there;
      asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(there) : "r"(umma::smem_u32(logits + e)));
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(there), "d"(v) : "memory");
    }
    __syncwarp();
  }
  umma::cluster_sync();
  if (rank != 0 || warp != 0) return;
  int expert = 0;
  float gate = 0.f;
  // few values a lane where there are few experts: code that is not there need not be fetched
  if (p.n_experts <= 64) el_choose<2>(p, logits, &expert, &gate);
  else el_choose<EL_MAX_EXPERTS / 32>(p, logits, &expert, &gate);
  if (lane < p.top_k) {
    p.experts[t * p.top_k + lane] = expert;
    p.gates[t * p.top_k + lane] = gate;
  }
}

struct ElShared {
  uint64_t full[EL_MAX_STAGES], empty[EL_MAX_STAGES], x_full[EL_MAX_STAGES], x_empty[EL_MAX_STAGES], finished[2], reported[2];
  unsigned long long tokens[EL_MAX_EXPERTS];  // of an expert: a bit for each of its tokens
  int abort_flag, used, most, last;  // most: tokens of an expert
  int group_pairs[EL_MAX_EXPERTS / 32], group_used[EL_MAX_EXPERTS / 32];
  float gates[EL_MAX_PAIRS];
  uint16_t chosen[EL_MAX_PAIRS], list[EL_MAX_PAIRS];           // pairs: token * top_k + j; list: in the order of their experts
  uint8_t token[EL_MAX_PAIRS];                                 // of the pairs of the list
  uint16_t place[EL_MAX_EXPERTS];                              // of an expert: its first pair's place in the list
  uint16_t expert[EL_MAX_EXPERTS], first[EL_MAX_EXPERTS + 1];  // of those that are used: which, and the first pair's place
};

// This CTA's items of a product: item i is column block i % blocks of the used expert i / blocks, and the i + skip-th of all go around the CTAs.
struct ElItems {
  int at, total, ctas, blocks;
  __device__ __forceinline__ ElItems(int total_, int skip, int cta, int ctas_, int blocks_) : total(total_), ctas(ctas_), blocks(blocks_) {
    at = cta - skip % ctas;
    if (at < 0) at += ctas;
  }
  __device__ __forceinline__ bool left() const { return at < total; }
  __device__ __forceinline__ void next() { at += ctas; }
  __device__ __forceinline__ int expert() const { return at / blocks; }
  __device__ __forceinline__ int block() const { return at % blocks; }
};

__device__ __forceinline__ void el_sync_reporters() { asm volatile("barrier.cta.sync 2, %0;" ::"n"(EL_REPORTERS) : "memory"); }
__device__ __forceinline__ void el_sync() { asm volatile("barrier.cta.sync 1, %0;" ::"n"(EL_CONSUMERS) : "memory"); }
__device__ __forceinline__ uint32_t el_acquire(const uint32_t* at) {
  uint32_t v;
  asm volatile("ld.acquire.gpu.global.b32 %0, [%1];" : "=r"(v) : "l"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t el_count(uint32_t* at) {
  uint32_t before;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(at) : "memory");
  return before;
}
__device__ __forceinline__ void el_arrive(uint32_t* at) { asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(at) : "memory"); }
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
__device__ __forceinline__ float el_widen(uint16_t h) {
  return BF16 ? __uint_as_float((uint32_t)h << 16) : __half2float(__ushort_as_half(h));
}
template <bool BF16>
__device__ __forceinline__ uint16_t el_round(float v) {
  return BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}

constexpr int EL_FIXED_BYTES = (EL_CONSUMERS * EL_SUMS * (int)sizeof(float) + (int)sizeof(ElShared) + 1023) / 1024 * 1024;

// The pairs in the order of their experts, of an expert in the order of its tokens: a token goes to an expert once at most, so that an expert's
// pairs are a set of tokens, 64 bits.
__device__ __forceinline__ void el_sort(const ExpertParams& p, ElShared* sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pairs = p.tokens * p.top_k, groups = (p.n_experts + 31) / 32;
  if (pairs <= 32) {  // a lane a pair, each counts the ones before it
    if (warp == 0) {
      const int e = lane < pairs ? (int)sh->chosen[lane] : 0x10000;
      const uint32_t peers = __match_any_sync(0xffffffffu, e);  // all lanes take part
      const bool head = lane < pairs && (peers & ((1u << lane) - 1u)) == 0u;
      const int key = e << 1 | (head ? 1 : 0);
      int place = 0, used = 0;
#pragma unroll 8
      for (int i = 0; i < 32; ++i) {
        const int other = __shfl_sync(0xffffffffu, key, i);
        place += (other >> 1) < e || ((other >> 1) == e && i < lane);
        used += (other >> 1) < e && (other & 1);
      }
      if (lane < pairs) {
        sh->list[place] = (uint16_t)lane;
        sh->token[place] = (uint8_t)(lane / p.top_k);
      }
      if (head) {
        sh->expert[used] = (uint16_t)e;
        sh->first[used] = (uint16_t)place;
      }
      const int all = __popc(__ballot_sync(0xffffffffu, head)), most = (int)__reduce_max_sync(0xffffffffu, lane < pairs ? (uint32_t)__popc(peers) : 0u);
      if (lane == 0) {
        sh->most = most;
        sh->used = all;
        sh->first[all] = (uint16_t)pairs;
      }
    }
    __syncthreads();
    return;
  }
  for (int e = threadIdx.x; e < p.n_experts; e += EL_THREADS) sh->tokens[e] = 0ull;
  if (threadIdx.x == 0) sh->most = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < pairs; i += EL_THREADS) atomicOr(&sh->tokens[sh->chosen[i]], 1ull << (i / p.top_k));
  __syncthreads();
  constexpr int ROUNDS = (EL_MAX_EXPERTS / 32 + EL_WARPS - 1) / EL_WARPS;
  int n[ROUNDS], before[ROUNDS];
  uint32_t some[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int group = warp + r * EL_WARPS, e = group * 32 + lane;
    if (group >= groups) break;
    n[r] = e < p.n_experts ? __popcll(sh->tokens[e]) : 0;
    some[r] = __ballot_sync(0xffffffffu, n[r] > 0);
    before[r] = n[r];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, before[r], o);
      if (lane >= o) before[r] += v;
    }
    const uint32_t most = __reduce_max_sync(0xffffffffu, (uint32_t)n[r]);
    if (lane == 31) {
      atomicMax(&sh->most, (int)most);
      sh->group_pairs[group] = before[r];
      sh->group_used[group] = __popc(some[r]);
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int group = warp + r * EL_WARPS, e = group * 32 + lane;
    if (group >= groups) break;
    int first = before[r] - n[r], used = __popc(some[r] & ((1u << lane) - 1u));
    for (int i = 0; i < group; ++i) {
      first += sh->group_pairs[i];
      used += sh->group_used[i];
    }
    if (n[r] > 0) {
      sh->expert[used] = (uint16_t)e;
      sh->first[used] = (uint16_t)first;
      sh->place[e] = (uint16_t)first;
    }
    if (group == groups - 1 && lane == 31) {
      used += some[r] >> 31;
      sh->used = used;
      sh->first[used] = (uint16_t)pairs;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < pairs; i += EL_THREADS) {
    const int e = sh->chosen[i], t = i / p.top_k;
    const int place = sh->place[e] + __popcll(sh->tokens[e] & ((1ull << t) - 1ull));
    sh->list[place] = (uint16_t)i;
    sh->token[place] = (uint8_t)t;
  }
  __syncthreads();
}

// The two rings in `bytes` of shared memory, weights first.  The tokens' rows (`most` of them, with their remainders) get up to twelve tiles but leave six of weights
// at least, two in any case; the weights get the rest.  Fragments are read 16 rows at a time, of which the last ones may be none of the tile's: behind the
// last tile there is room for them (what they hold does not matter).
struct ElRings {
  int x_bytes, x_stages, stages;  // a tile of rows; tiles
};
constexpr int EL_X_ROOM = 16 * EL_X_PITCH;
__host__ __device__ __forceinline__ ElRings el_rings(int bytes, int most) {
  ElRings r;
  r.x_bytes = 2 * most * EL_X_PITCH;  // (W_in's have no remainders and leave half of it)
  const int free = bytes - EL_X_ROOM, x = (free - 6 * EL_TILE_BYTES) / r.x_bytes;
  r.x_stages = x < 2 ? 2 : x < EL_MAX_STAGES ? x : EL_MAX_STAGES;
  const int w = (free - r.x_stages * r.x_bytes) / EL_TILE_BYTES;
  r.stages = w < EL_MAX_STAGES ? w : EL_MAX_STAGES;
  return r;
}

// What every role goes by: the items, and the rings.
struct ElPlan {
  int used, ctas, blocks_in, blocks_out, x_bytes, x_stages, stages;
  __device__ __forceinline__ ElPlan(const ExpertParams& p, const ElShared* sh) {
    const int h_columns = p.gated ? EL_COLUMNS / 2 : EL_COLUMNS;  // that an item of W_in stands for
    used = sh->used;
    ctas = p.ctas;
    blocks_in = (p.hidden + h_columns - 1) / h_columns;
    blocks_out = (p.out_width + EL_COLUMNS - 1) / EL_COLUMNS;
    const ElRings r = el_rings(p.ring_bytes, sh->most);
    x_bytes = r.x_bytes;
    x_stages = r.x_stages;
    stages = r.stages;
  }
  __device__ __forceinline__ ElItems items(int product) const {
    return product == 0 ? ElItems(used * blocks_in, 0, (int)blockIdx.x, ctas, blocks_in) : ElItems(used * blocks_out, used * blocks_in, (int)blockIdx.x, ctas, blocks_out);
  }
};

// ---------------------------------------------------------------------------------------------
// The products, by warps 0-7.  NT: groups of eight tokens that an expert may have.
// ---------------------------------------------------------------------------------------------
template <bool BF16, int NT>
__device__ __forceinline__ void el_products(const ExpertParams& p, ElShared* sh, uint32_t tiles0, uint32_t x0, float* sums) {
  using namespace umma;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &sh->abort_flag;
  const ElPlan plan(p, sh);
  bool ok = true;
  const int g = lane >> 2, c = lane & 3;  // of a fragment: column of the weight; pair of tokens
  const int matrix = lane >> 3, row = lane & 7;
  // this lane's row of the tokens' four 8 x 8 matrices: eight tokens by two of eight of the contraction, and eight tokens more
  const uint32_t rows = x0 + (uint32_t)(((matrix >> 1) * 8 + row) * EL_X_PITCH + warp * 32 + (matrix & 1) * 16);
  int s = 0, x_at = 0;
  uint32_t ph = 0, x_ph = 0, count = 0;
  float acc[NT][4][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[j][i >> 2][i & 3] = 0.f;
  for (int product = 0; product < 2; ++product) {
    const bool gated = product == 0 && p.gated;
    const int length = product == 0 ? p.width : p.hidden, columns = product == 0 ? p.hidden : p.out_width;
    // And of the weight's: two groups of eight columns (side by side, or one of each half of u) by two of eight of the contraction.  Gated, a half has rows of
    // 64 bytes, whose 16-byte chunks are permuted by row / 2 % 4; otherwise rows are 128 bytes and permuted by row % 8.
    const int r = warp * 16 + (matrix >> 1) * 8 + row;
    const uint32_t weights = tiles0 + (uint32_t)(gated ? (matrix & 1) * (EL_TILE_BYTES / 2) + r * 64 : r * 128);
    uint32_t chunk[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) chunk[q] = (uint32_t)((gated ? q ^ (row >> 1) : (2 * q + (matrix & 1)) ^ row) * 16);
    for (ElItems w = plan.items(product); w.left(); w.next()) {
      const int u = w.expert(), m = w.block(), first = sh->first[u], n = sh->first[u + 1] - first;
      for (int k = 0; k < length; k += EL_K) {
        if (ok) ok = mbar_parked_wait(smem_u32(&sh->x_full[x_at]), x_ph, abort_flag) && mbar_parked_wait(smem_u32(&sh->full[s]), ph, abort_flag);
        __syncwarp();
        if (k + warp * 16 < length) {  // (behind the contraction's end both operands are zeros)
          const uint32_t tile = weights + (uint32_t)(s * EL_TILE_BYTES), x = rows + (uint32_t)(x_at * plan.x_bytes);
          uint32_t a[4][4];
#pragma unroll
          for (int q = 0; q < 4; ++q) el_ldmatrix_trans(a[q], tile + chunk[q]);
#pragma unroll
          for (int j = 0; j < NT; j += 2) {
            if (j * 8 < n) {
              uint32_t b[4], rest[4];
              el_ldmatrix(b, x + (uint32_t)(j * 8 * EL_X_PITCH));
              if (product == 1) el_ldmatrix(rest, x + (uint32_t)(plan.x_bytes / 2 + j * 8 * EL_X_PITCH));  // what h's rounding left
#pragma unroll
              for (int q = 0; q < 4; ++q) el_mma<BF16>(acc[j][q], a[q], b[0], b[1]);
              if (j * 8 + 8 < n) {
#pragma unroll
                for (int q = 0; q < 4; ++q) el_mma<BF16>(acc[j + 1][q], a[q], b[2], b[3]);
              }
              if (product == 1) {
#pragma unroll
                for (int q = 0; q < 4; ++q) el_mma<BF16>(acc[j][q], a[q], rest[0], rest[1]);
                if (j * 8 + 8 < n) {
#pragma unroll
                  for (int q = 0; q < 4; ++q) el_mma<BF16>(acc[j + 1][q], a[q], rest[2], rest[3]);
                }
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(&sh->empty[s]));
          mbar_arrive(smem_u32(&sh->x_empty[x_at]));
        }
        if (++s == plan.stages) { s = 0; ph ^= 1u; }
        if (++x_at == plan.x_stages) { x_at = 0; x_ph ^= 1u; }
      }
      // ---------------------------------------------------------------- the item's sums
      // Eight tokens after eight, always from acc[0], the others moving up: the code is there once.  Thread (warp, lane) finishes what lane's fragments hold for
      // 16 columns and one token of a pair.
#pragma unroll 1
      for (int j = 0; j * 8 < n; ++j) {
#pragma unroll
        for (int i = 0; i < EL_SUMS; ++i) sums[(warp * EL_SUMS + i) * 32 + lane] = acc[0][i >> 2][i & 3];
        el_sync();
        const int q = warp >> 1, i = warp & 1, token = j * 8 + c * 2 + i;
        float v0 = 0.f, v1 = 0.f;
#pragma unroll
        for (int o = 0; o < EL_CONSUMERS / 32; ++o) {
          v0 += sums[(o * EL_SUMS + q * 4 + i) * 32 + lane];
          v1 += sums[(o * EL_SUMS + q * 4 + 2 + i) * 32 + lane];
        }
        if (token < n) {
          const int col = m * (gated ? EL_COLUMNS / 2 : EL_COLUMNS) + q * (gated ? 8 : 16) + g;
          if (product == 0) {
            uint16_t* h_row = p.h + (size_t)(first + token) * 2 * p.hidden;
            const auto put = [&](int at, float v) {  // (an h that the type does not hold has no remainder)
              const uint16_t rounded = el_round<BF16>(v);
              const float left = v - el_widen<BF16>(rounded);
              h_row[at] = rounded;
              h_row[p.hidden + at] = el_round<BF16>(fabsf(left) <= fabsf(v) ? left : 0.f);
            };
            v0 = el_activated(p.activation, v0);
            if (gated) {
              if (col < columns) put(col, v0 * v1);
            } else {
              if (col < columns) put(col, v0);
              if (col + 8 < columns) put(col + 8, el_activated(p.activation, v1));
            }
          } else {
            const int pair = sh->list[first + token];
            const float gate = sh->gates[pair];
            float* part_row = p.part + (size_t)pair * p.out_width;
            if (col < columns) __stcg(part_row + col, gate * v0);
            if (col + 8 < columns) __stcg(part_row + col + 8, gate * v1);
          }
        }
        el_sync();  // the sums have been read
#pragma unroll
        for (int o = 0; o < NT; ++o)
#pragma unroll
          for (int t = 0; t < 16; ++t) acc[o][t >> 2][t & 3] = o + 1 < NT ? acc[o + 1 < NT ? o + 1 : o][t >> 2][t & 3] : 0.f;
      }
      // (all that was stored is behind the barriers above)
      if (ok) ok = mbar_parked_wait(smem_u32(&sh->reported[count & 1]), (count >> 1 & 1) ^ 1u, abort_flag);
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh->finished[count & 1]));
      ++count;
    }
  }
}

template <bool BF16>
__global__ void __launch_bounds__(EL_THREADS, 1)
    expert_layer_kernel(const __grid_constant__ ExpertParams p, const __grid_constant__ CUtensorMap map_in, const __grid_constant__ CUtensorMap map_out) {
  using namespace umma;
  extern __shared__ uint8_t el_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(el_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  float* sums = reinterpret_cast<float*>(smem);  // [warps][EL_SUMS][32]
  ElShared* sh = reinterpret_cast<ElShared*>(sums + EL_CONSUMERS * EL_SUMS);
  const uint32_t ring = smem_u32(smem) + EL_FIXED_BYTES;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cta = (int)blockIdx.x;
  volatile int* abort_flag = &sh->abort_flag;
  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_in) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_out) : "memory");
    for (int s = 0; s < EL_MAX_STAGES; ++s) {
      mbar_init(smem_u32(&sh->full[s]), 1);
      mbar_init(smem_u32(&sh->empty[s]), EL_CONSUMERS / 32);
    }
    for (int s = 0; s < EL_MAX_STAGES; ++s) {
      mbar_init(smem_u32(&sh->x_full[s]), 32);
      mbar_init(smem_u32(&sh->x_empty[s]), EL_CONSUMERS / 32);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&sh->finished[i]), EL_CONSUMERS / 32);
      mbar_init(smem_u32(&sh->reported[i]), EL_REPORTERS / 32);
    }
    sh->abort_flag = 0;
    mbar_fence_init();
  }
  for (int i = threadIdx.x; i < p.tokens * p.top_k; i += EL_THREADS) {
    sh->chosen[i] = (uint16_t)__ldcg(p.experts + i);
    sh->gates[i] = __ldcg(p.gates + i);
  }
  __syncthreads();
  el_sort(p, sh);
  const ElPlan plan(p, sh);
  const uint32_t tiles0 = ring, x0 = tiles0 + (uint32_t)(plan.stages * EL_TILE_BYTES);
  uint32_t *done_in = p.flags, *done_out = p.flags + p.n_experts;
  bool ok = true;

  if (warp == EL_CONSUMERS / 32) {
    // ------------------------------------------------------------------ weights
    if (elect_one()) {
      int s = 0;
      uint32_t ph = 1;
      for (int product = 0; product < 2 && ok; ++product) {
        const CUtensorMap* map = product == 0 ? &map_in : &map_out;
        const bool gated = product == 0 && p.gated;
        const int length = product == 0 ? p.width : p.hidden;
        for (ElItems w = plan.items(product); w.left() && ok; w.next()) {
          const int e = sh->expert[w.expert()], col = w.block() * (gated ? EL_COLUMNS / 2 : EL_COLUMNS);
          for (int k = 0; k < length; k += EL_K) {
            ok = mbar_parked_wait(smem_u32(&sh->empty[s]), ph, abort_flag);
            if (!ok) break;
            const uint32_t to = tiles0 + (uint32_t)(s * EL_TILE_BYTES), bar = smem_u32(&sh->full[s]);
            mbar_expect_tx(bar, EL_TILE_BYTES);
            pair_load_3d<1>(to, map, bar, col, k, e);
            if (gated) pair_load_3d<1>(to + EL_TILE_BYTES / 2, map, bar, p.hidden + col, k, e);
            if (++s == plan.stages) { s = 0; ph ^= 1u; }
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == EL_CONSUMERS / 32 + 1) {
    // ------------------------------------------------------------------ tokens' rows
    int s = 0;
    uint32_t ph = 1;
    for (int product = 0; product < 2 && ok; ++product) {
      const int length = product == 0 ? p.width : p.hidden;
      for (ElItems w = plan.items(product); w.left() && ok; w.next()) {
        const int u = w.expert(), first = sh->first[u], n = sh->first[u + 1] - first;
        if (product == 1) {  // all of the expert's h is there
          ok = __all_sync(0xffffffffu, el_await(done_in + u, (uint32_t)plan.blocks_in, abort_flag));
          if (!ok) break;
        }
        for (int k = 0; k < length; k += EL_K) {
          ok = __all_sync(0xffffffffu, mbar_parked_wait(smem_u32(&sh->x_empty[s]), ph, abort_flag));
          if (!ok) break;
          // half a warp a row; zeros behind the contraction's end
          const int at = k + (lane & 15) * 8;
          const uint32_t to = x0 + (uint32_t)(s * plan.x_bytes + (lane & 15) * 16);
#pragma unroll 4
          for (int row = lane >> 4; row < n; row += 2) {
            const uint16_t* src = product == 0 ? static_cast<const uint16_t*>(p.x) + sh->token[first + row] * p.x_pitch : p.h + (size_t)(first + row) * 2 * p.hidden;
            cp_async16(to + (uint32_t)(row * EL_X_PITCH), at < length ? src + at : src, at < length);
            if (product == 1) cp_async16(to + (uint32_t)((sh->most + row) * EL_X_PITCH), at < length ? src + p.hidden + at : src, at < length);
          }
          cp_async_arrive_noinc(smem_u32(&sh->x_full[s]));
          if (++s == plan.x_stages) { s = 0; ph ^= 1u; }
        }
      }
    }
  } else if (warp >= EL_WARPS - EL_REPORTERS / 32) {
    // ------------------------------------------------------------------ reports, and the sum over a token's experts
    const int thread = (int)threadIdx.x - (EL_THREADS - EL_REPORTERS);
    uint32_t count = 0;  // items, of which two may be finished and not reported
    for (int product = 0; product < 2; ++product) {
      for (ElItems w = plan.items(product); w.left(); w.next(), ++count) {
        if (ok) ok = mbar_parked_wait(smem_u32(&sh->finished[count & 1]), count >> 1 & 1, abort_flag);
        __syncwarp();
        if (product == 0) {
          if (thread == 0) el_arrive(done_in + w.expert());
          if (lane == 0) mbar_arrive(smem_u32(&sh->reported[count & 1]));
          continue;
        }
        const int m = w.block(), col = m * EL_COLUMNS + (thread & 15) * 4;  // (the width is a multiple of eight)
        if (thread == 0) sh->last = el_count(done_out + m) + 1u == (uint32_t)plan.used;
        el_sync_reporters();
        if (sh->last && col < p.out_width) {  // the last item of the column block: all of its columns' parts are there
          for (int t0 = thread >> 4; t0 < p.tokens; t0 += 4 * (EL_REPORTERS / 16)) {
            float4 sum[4];  // of four tokens, whose parts are on their way together
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
            for (int j = 0; j < p.top_k; ++j) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int t = min(t0 + i * (EL_REPORTERS / 16), p.tokens - 1);
                const float4 v = __ldcg(reinterpret_cast<const float4*>(p.part + (size_t)(t * p.top_k + j) * p.out_width + col));
                sum[i].x += v.x;
                sum[i].y += v.y;
                sum[i].z += v.z;
                sum[i].w += v.w;
              }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int t = t0 + i * (EL_REPORTERS / 16);
              if (t >= p.tokens) continue;
              uint16_t* to = static_cast<uint16_t*>(p.out) + (size_t)t * p.out_pitch + col;
              const uint16_t b[4] = {el_round<BF16>(sum[i].x), el_round<BF16>(sum[i].y), el_round<BF16>(sum[i].z), el_round<BF16>(sum[i].w)};
              if ((reinterpret_cast<uintptr_t>(to) & 7) == 0) {
                *reinterpret_cast<uint2*>(to) = make_uint2((uint32_t)b[0] | (uint32_t)b[1] << 16, (uint32_t)b[2] | (uint32_t)b[3] << 16);
              } else {
#pragma unroll
                for (int q = 0; q < 4; ++q) to[q] = b[q];
              }
            }
          }
        }
        el_sync_reporters();  // `last` has been read
        if (lane == 0) mbar_arrive(smem_u32(&sh->reported[count & 1]));
      }
    }
  } else {
    if (sh->most <= 16) el_products<BF16, 2>(p, sh, tiles0, x0, sums);
    else if (sh->most <= 32) el_products<BF16, 4>(p, sh, tiles0, x0, sums);
    else el_products<BF16, 8>(p, sh, tiles0, x0, sums);
  }
  if (*abort_flag && lane == 0) report_problem();
  if (*abort_flag) {  // copies may still be on their way into this CTA's memory
    const long long start = clock64();
    while (clock64() - start < 2000000) __nanosleep(1000);
  }
}

// Bytes of workspace, and where its parts begin.
struct ExpertSpace {
  size_t flags, h, part, total;
  int n_flags;
};
inline ExpertSpace expert_space(int tokens, int experts, int top_k, int hidden, int out_width) {
  ExpertSpace s;
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  s.n_flags = experts + (out_width + EL_COLUMNS - 1) / EL_COLUMNS;
  s.flags = take((size_t)s.n_flags * sizeof(uint32_t));
  s.h = take((size_t)tokens * top_k * 2 * hidden * 2);
  s.part = take((size_t)tokens * top_k * out_width * sizeof(float));
  s.total = at;
  return s;
}

// A tensor map of `mats` matrices [rows][cols] of 16-bit values, boxes of 128 rows by `box` columns: 64, or 32 (rows of 64 bytes).
inline int expert_tensor_map(CUtensorMap* map, const void* data, int cols, int rows, int mats, int box, bool bf16) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  const Encode encode = reinterpret_cast<Encode>(tensor_map_encoder());
  if (encode == nullptr) return -1000 - (int)CUDA_ERROR_NOT_FOUND;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)mats}, pitch[2] = {(cuuint64_t)cols * 2, (cuuint64_t)cols * 2 * (cuuint64_t)rows};
  const cuuint32_t boxes[3] = {(cuuint32_t)box, EL_K, 1}, steps[3] = {1, 1, 1};
  const auto made = [&] {
    return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(data), dims, pitch, boxes, steps,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, box == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult rc = made();
  if (rc == CUDA_ERROR_INVALID_CONTEXT) {  // a host thread that has launched nothing yet: see weight_tensor_map
    int dev = 0;
    if (cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) rc = made();
  }
  return rc == CUDA_SUCCESS ? 0 : -1000 - (int)rc;
}

template <typename T, typename R>
cudaError_t launch_expert_choice(const ExpertParams& p, cudaStream_t st) {
  const int size = p.n_experts <= 8 ? 1 : p.n_experts <= 16 ? 2 : p.n_experts <= 32 ? 4 : 8;  // a warp an expert, where eight CTAs have as many
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3((unsigned)(p.tokens * size));
  lc.blockDim = dim3(EL_ROUTER_THREADS);
  lc.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)size;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  lc.attrs = at;
  lc.numAttrs = 2;
  return cudaLaunchKernelEx(&lc, expert_choice_kernel<T, R>, p);
}

template <bool BF16>
int launch_expert_layer(ExpertParams p, const void* w_in, const void* w_out, cudaStream_t st, int max_smem) {
  p.ring_bytes = max_smem - 1024 - EL_FIXED_BYTES;
  if (p.ring_bytes < 6 * EL_TILE_BYTES + 4 * EL_MAX_TOKENS * EL_X_PITCH + EL_X_ROOM) return -1;
  const int smem = max_smem;
  CUtensorMap in, out;
  const int wide = p.gated ? 2 * p.hidden : p.hidden;
  int rc = expert_tensor_map(&in, w_in, wide, p.width, p.n_experts, p.gated ? 32 : 64, BF16);
  if (rc == 0) rc = expert_tensor_map(&out, w_out, p.out_width, p.hidden, p.n_experts, 64, BF16);
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
