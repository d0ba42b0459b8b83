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
// `there` of the eight values from `p` on (at most eight; none: zeros); vec: rows start on 16-byte boundaries.  Values that are read once pass L1 by.  Off such a
// boundary they come as words, of which the outer two may hold a neighbour's value as well, and are shifted by a value if need be.
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
  if (there >= ROW_CHUNK) {
    const uint32_t* words = reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)3);
#pragma unroll
    for (int i = 0; i < N; ++i) r.w[i] = __ldca(words + i);
    if (sizeof(T) == 2 && (reinterpret_cast<uintptr_t>(p) & 2)) {
      const uint32_t last = __ldca(words + N);
#pragma unroll
      for (int i = 0; i < N; ++i) r.w[i] = __funnelshift_r(r.w[i], i + 1 < N ? r.w[i + 1 < N ? i + 1 : i] : last, 16);
    }
    return r;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) r.w[i] = 0u;
#pragma unroll
  for (int e = 0; e < ROW_CHUNK; ++e) {
    if (e >= there) continue;
    if constexpr (sizeof(T) == 4) r.w[e] = reinterpret_cast<const uint32_t*>(p)[e];
    else r.w[e / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[e] << (16 * (e % 2));
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
template <typename T>
__device__ __forceinline__ void row_values(const RowRaw<T>& r, float (&x)[ROW_CHUNK]) {
#pragma unroll
  for (int i = 0; i < ROW_CHUNK / 2; ++i) {
    if constexpr (sizeof(T) == 4) {
      x[2 * i] = __uint_as_float(r.w[2 * i]);
      x[2 * i + 1] = __uint_as_float(r.w[2 * i + 1]);
    } else if constexpr (std::is_same<T, __half>::value) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    } else {
      x[2 * i] = __uint_as_float(r.w[i] << 16);
      x[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
    }
  }
}
template <typename T>
__device__ __forceinline__ RowRaw<T> row_rounded(const float (&x)[ROW_CHUNK]) {
  RowRaw<T> r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < ROW_CHUNK; ++i) r.w[i] = __float_as_uint(x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < ROW_CHUNK / 2; ++i) {
      if constexpr (std::is_same<T, __half>::value) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r.w[i]) : "f"(x[2 * i + 1]), "f"(x[2 * i]));
      else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r.w[i]) : "f"(x[2 * i + 1]), "f"(x[2 * i]));
    }
  }
  return r;
}
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
// Rounded once to their type.  All lanes of a warp call it (with none there, if it must be); lanes that follow one another hold chunks that do, of the
// same row as long as there are any.  Off 16-byte boundaries (`vec` false) a lane takes the next one's first values and stores the 16-byte blocks that its own
// values end in; what the warp's first and last chunk, or a row's, have beyond such blocks goes value by value.
template <typename T>
__device__ __forceinline__ void row_store(T* p, const float (&x)[ROW_CHUNK], int there, bool vec, bool first_of_row) {
  constexpr int N = 2 * sizeof(T), EACH = 4 / sizeof(T);  // words; values of a word
  const RowRaw<T> h = row_rounded<T>(x);
  const auto put = [&](int e) {
    if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(p)[e] = h.w[e];
    else reinterpret_cast<uint16_t*>(p)[e] = (uint16_t)(h.w[e / 2] >> (16 * (e % 2)));
  };
  if (vec) {
    if (there >= ROW_CHUNK) {
#pragma unroll
      for (int q = 0; q < N / 4; ++q) reinterpret_cast<uint4*>(p)[q] = make_uint4(h.w[4 * q], h.w[4 * q + 1], h.w[4 * q + 2], h.w[4 * q + 3]);
    } else {
#pragma unroll
      for (int e = 0; e < ROW_CHUNK; ++e)
        if (e < there) put(e);
    }
    return;
  }
  const int lane = threadIdx.x & 31;
  const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(p) & 15u;
  const int head = (int)((16u - off) & 15u) / (int)sizeof(T);  // values in front of the first block that begins inside this chunk
  uint32_t w[N + 4];
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = h.w[i];
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
    if (e < there && (e < head ? !covered : e >= stored_to)) put(e);
}

// ---------------------------------------------------------------------------------------------
// Dropout.  Philox 4x32 with ten rounds (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011): the
// key is the seed, the counter (column / 8, row, call), whose 128 bits are eight lots of 16 bits for the eight columns of a chunk.  A value is dropped
// where its lot is below the threshold, round(p 65536); the others are multiplied by 65536 / (65536 - threshold), so that the mean is kept exactly
// at the probability as it is rounded.  16 bits a lot: 32 would be two evaluations a chunk, 40 wide multiplications instead of 20.
// Nothing is stored: the backward evaluates the same lots again.
//
// State in device memory, [seed, calls made, blocks of this call that have finished]: a call takes the number of calls made as its own number
// and counts it, so that a replayed graph drops other values every time.  What it took is handed on to its backward.
// ---------------------------------------------------------------------------------------------
struct DropParams {
  long long* state;       // forward: [3]
  long long* used;        // forward: null, or [2], where seed and number of the call are left; backward: those
  uint32_t threshold;     // 1 .. 65536 (everything); 0: nothing is dropped, and no lots are drawn
  float factor;           // of what is kept
};
struct DropKey {
  uint32_t key0, key1, call0, call1;
};
__device__ __forceinline__ DropKey drop_key(const long long* at) {
  const long long seed = __ldcg(at), call = __ldcg(at + 1);
  // the same in all lanes, and known to be: what is added to the key round after round is then no lane's work
  const auto one = [](uint32_t v) { return __reduce_or_sync(0xffffffffu, v); };
  return {one((uint32_t)seed), one((uint32_t)((unsigned long long)seed >> 32)), one((uint32_t)call), one((uint32_t)((unsigned long long)call >> 32))};
}
// The lots of a chunk, and whether its value e is kept: lots are compared in the upper halves of words with (threshold << 16) - 1, which they are above where they are
// not below the threshold (which is 1 at least; of 65536 no word is above).
struct DropLots {
  uint32_t w[4];
  __device__ __forceinline__ bool kept(int e, uint32_t below) const { return (e & 1 ? w[e / 2] : w[e / 2] << 16) > below; }
};
__device__ __forceinline__ uint32_t drop_below(uint32_t threshold) { return (threshold << 16) - 1u; }
__device__ __forceinline__ DropLots drop_lots(const DropKey& k, uint32_t chunk, uint32_t row) {
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
  return {{c0, c1, c2, c3}};
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
