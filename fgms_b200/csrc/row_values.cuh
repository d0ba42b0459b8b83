// Rows of values in chunks of eight consecutive ones, and the random lots of dropout: what row_norm.cuh and dropout.cuh share.
#pragma once
#include <type_traits>

#include "grouped.cuh"  // to_f32, from_f32

namespace fgms {

constexpr int ROW_CHUNK = 8;

// Eight values as they lie in memory: 16 bytes, or 32 of fp32.
template <typename T>
struct RowRaw {
  uint32_t w[2 * sizeof(T)];
};
// The bytes from `off` on (0 .. 15, a multiple of the values' size, the same in all lanes) of N words and the four behind them.
template <int N>
__device__ __forceinline__ void row_shift_down(uint32_t (&w)[N + 4], uint32_t off) {
  if (off & 8u) {
#pragma unroll
    for (int i = 0; i < N + 2; ++i) w[i] = w[i + 2];
  }
  if (off & 4u) {
#pragma unroll
    for (int i = 0; i < N + 1; ++i) w[i] = w[i + 1];
  }
  if (off & 2u) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
  }
}
// `there` of the eight values from `p` on (at most eight; none: zeros); vec: rows start on 16-byte boundaries.  Values that are read once pass L1 by.  Off such a
// boundary the 16-byte blocks that the values lie in are read, whose other bytes are a neighbour's (or behind the last row's end, in a block that row is
// in as well), and shifted: 16384 rows of 1001 fp16 values take XXX us so, and YYY a value at a time.
template <typename T>
__device__ __forceinline__ RowRaw<T> row_load(const T* p, int there, bool vec) {
  constexpr int N = 2 * sizeof(T);
  RowRaw<T> r;
  if (vec && there >= ROW_CHUNK) {
    const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p));
    r.w[0] = a.x; r.w[1] = a.y; r.w[2] = a.z; r.w[3] = a.w;
    if constexpr (sizeof(T) == 4) {
      const uint4 b = __ldcs(reinterpret_cast<const uint4*>(p) + 1);
      r.w[4] = b.x; r.w[5] = b.y; r.w[6] = b.z; r.w[7] = b.w;
    }
    return r;
  }
  const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(p) & 15u;
  const uint4* blocks = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)15);
  const int bytes = min(there, ROW_CHUNK) * (int)sizeof(T) + (int)off;  // that are needed, from the first block on
  uint32_t w[N + 4];
#pragma unroll
  for (int i = 0; i < N / 4 + 1; ++i) {
    const uint4 v = there > 0 && bytes > 16 * i ? __ldca(blocks + i) : make_uint4(0, 0, 0, 0);
    w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
  }
  row_shift_down<N>(w, off);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    r.w[i] = w[i];
    if (sizeof(T) == 4) {
      if (i >= there) r.w[i] = 0u;
    } else {
      if (2 * i >= there) r.w[i] = 0u;
      else if (2 * i + 1 >= there) r.w[i] &= 0xffffu;
    }
  }
  return r;
}
template <typename T>
__device__ __forceinline__ float row_value(const RowRaw<T>& r, int e) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(r.w[e]);
  } else {
    const uint16_t h = (uint16_t)(r.w[e / 2] >> (16 * (e % 2)));
    if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half(h));
    else return __uint_as_float((uint32_t)h << 16);
  }
}
// Rounded once to their type.  All lanes of a warp call it (with none there, if it must be); lanes that follow one another hold chunks that do, of the
// same row as long as there are any.  Off 16-byte boundaries (`vec` false) a lane takes the next one's first values and stores the 16-byte blocks that its own
// values end in; what the warp's first and last chunk, or a row's, have beyond such blocks goes value by value.
template <typename T>
__device__ __forceinline__ void row_store(T* p, const float (&x)[ROW_CHUNK], int there, bool vec, bool first_of_row) {
  constexpr int N = 2 * sizeof(T), EACH = 4 / sizeof(T);  // words; values of a word
  __align__(16) T h[ROW_CHUNK];
#pragma unroll
  for (int e = 0; e < ROW_CHUNK; ++e) h[e] = from_f32<T>(x[e]);
  if (vec) {
    if (there >= ROW_CHUNK) {
#pragma unroll
      for (int q = 0; q < (int)sizeof(T) / 2; ++q) reinterpret_cast<uint4*>(p)[q] = reinterpret_cast<const uint4*>(h)[q];
    } else {
#pragma unroll
      for (int e = 0; e < ROW_CHUNK; ++e)
        if (e < there) p[e] = h[e];
    }
    return;
  }
  const int lane = threadIdx.x & 31;
  const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(p) & 15u;
  const int head = (int)((16u - off) & 15u) / (int)sizeof(T);  // values in front of the first block that begins inside this chunk
  uint32_t w[N + 4];
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint32_t*>(h)[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[N + i] = __shfl_down_sync(0xffffffffu, w[i], 1);
  const bool joined = lane < 31 && there - ROW_CHUNK >= head;       // the next chunk has the values that this one's last block lacks
  const bool covered = lane > 0 && !first_of_row && there >= head;  // and the one before has stored this one's head
  const int whole = joined ? N / 4 : there >= ROW_CHUNK ? (ROW_CHUNK - head) * (int)sizeof(T) / 16 : 0;  // blocks that are stored
  row_shift_down<N>(w, (16u - off) & 15u);
  uint4* blocks = reinterpret_cast<uint4*>(p + head);
#pragma unroll
  for (int i = 0; i < N / 4; ++i)
    if (i < whole) blocks[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  const int stored_to = whole > 0 ? head + whole * 4 * EACH : head;  // from `head` on
#pragma unroll
  for (int e = 0; e < ROW_CHUNK; ++e)
    if (e < there && (e < head ? !covered : e >= stored_to)) p[e] = h[e];
}

// ---------------------------------------------------------------------------------------------
// Dropout.  Philox 4x32 with ten rounds (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011): the
// key is the seed, the counter (column / 8, row, call), whose 128 bits are eight lots of 16 bits for the eight columns of a chunk.  A value is dropped
// where its lot is below the threshold, round(p 65536); the others are multiplied by 65536 / (65536 - threshold), so that the mean is kept exactly
// at the probability as it is rounded.  16 bits a lot: 32 would be two evaluations a chunk, 80 wide multiplications instead of 40.
// Nothing is stored: the backward evaluates the same lots again.
//
// State in device memory, [seed, calls made, blocks of this call that have finished]: a call takes the number of calls made as its own number
// and counts it, so that a replayed graph drops other values every time.  What it took is handed on to its backward.
// ---------------------------------------------------------------------------------------------
struct DropParams {
  long long* state;       // forward: [3]
  long long* used;        // forward: null, or [2], where seed and number of the call are left; backward: those
  uint32_t threshold;     // 0: nothing is dropped, 65536: everything
  float factor;           // of what is kept
};
struct DropKey {
  uint32_t key0, key1, call0, call1;
};
__device__ __forceinline__ DropKey drop_key(const long long* at) {
  const long long seed = __ldcg(at), call = __ldcg(at + 1);
  return {(uint32_t)seed, (uint32_t)((unsigned long long)seed >> 32), (uint32_t)call, (uint32_t)((unsigned long long)call >> 32)};
}
// bit e: the chunk's value e is kept
__device__ __forceinline__ uint32_t drop_keep(const DropKey& k, uint32_t chunk, uint32_t row, uint32_t threshold) {
  uint32_t c0 = chunk, c1 = row, c2 = k.call0, c3 = k.call1, k0 = k.key0, k1 = k.key1;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)b;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  const uint32_t w[4] = {c0, c1, c2, c3};
  uint32_t keep = 0;
#pragma unroll
  for (int e = 0; e < ROW_CHUNK; ++e) keep |= ((e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu) >= threshold ? 1u : 0u) << e;
  return keep;
}
// Every thread of the grid has read the state before: the last block counts the call.
__device__ __forceinline__ void drop_count(const DropParams& d) {
  __syncthreads();
  if (threadIdx.x == 0) {
    const long long seed = __ldcg(d.state), call = __ldcg(d.state + 1);
    if (blockIdx.x == 0 && d.used != nullptr) {
      d.used[0] = seed;
      d.used[1] = call;
    }
    __threadfence();
    if (atomicAdd(reinterpret_cast<unsigned long long*>(d.state + 2), 1ull) == gridDim.x - 1) {
      d.state[2] = 0;
      d.state[1] = (long long)((unsigned long long)call + 1ull);
    }
  }
}

}  // namespace fgms
