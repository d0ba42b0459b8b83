// One AdamW step over many tensors in one launch (fgms_b200_adamw).
//
//   g  = grad / grad_scale
//   m' = b1 m + (1 - b1) g         v' = b2 v + (1 - b2) g^2
//   w' = w (1 - lr decay) - lr / (1 - b1^t)  m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// w is the fp32 master where there is one, else the parameter; the parameter is w' rounded once.  All arithmetic is fp32.  In moments of 8 bits
// every operation is rounded by itself (no contraction), so that codes are the same bits as the formulas evaluated one operation at a time; w'
// takes the approximate root and quotient, 2^-22 of the update.
//
// Moments in 8 bits: e4m3 codes with an fp32 scale (largest value / 448) for each 128 values.  A moving average moves by less than half a
// code per step (v by 0.1 % where codes are 12 % apart) and rounding to the nearest code would leave it where it is, so a value is rounded up with
// the probability of the part that is cut off: the mean is kept, of v down to the smallest code of its block, 1/229376 of the largest value.  The
// random bits are a hash of (seed, step, index), so a step can be repeated bit for bit.  A second moment above zero never becomes zero (its m would
// then be divided by eps alone): below the smallest code it takes that one, which is too large.  So a value whose gradients are more than 479
// times (the root of 229376) smaller than the largest ones of its block takes steps that are smaller by what they are beyond that.  w' is computed from m'
// and v' before they are rounded.
//
// What bounds it is memory with moments in 32 bits (28 bytes a value in fp32, or in 16 bits with masters): 150 M values in fp32 662-668 us, 96 % of the copy
// rate.  With moments in 8 bits (12 or 16 bytes) it is the issue of instructions: 120 M values in fp16 with masters 391-436 us from board to board,
// where their bytes take 295.
#pragma once
#include "grouped.cuh"  // to_f32, from_f32

namespace fgms {

constexpr int ADAMW_THREADS = 256;
constexpr int ADAMW_PER_THREAD = 8;  // consecutive values
constexpr int ADAMW_CHUNK = ADAMW_THREADS * ADAMW_PER_THREAD;
constexpr int ADAMW_BLOCK = 128;  // values that share a scale: 16 lanes
constexpr float ADAMW_E4M3_MAX = 448.0f;
constexpr float ADAMW_SMALLEST = 7.88860905e-31f;      // 2^-100: a block of first moments whose largest value is smaller is held as zeros
constexpr float ADAMW_SCALE_SMALLEST = 1.17549435e-38f;  // 2^-126: of second moments, so that codes stand for multiples of 2^-135, the smallest of them for that

struct AdamwTensor {
  void* param;
  const void* grad;
  float* master;  // or null
  void *m, *v;
  float *m_scale, *v_scale;
  long long count;
  int first_chunk;
  uint8_t param_type, grad_type, aligned, pad;  // aligned: every pointer on a 16-byte boundary (codes: 8)
};

template <int N>
struct AdamwParams {
  double lr, beta1, beta2, decay;
  float b1, c1, b2, c2, eps;  // c = 1 - b
  uint32_t seed, minus_zero;
  const float *lr_device, *grad_scale, *found_inf;
  int* step;  // [2]: steps done, and blocks that have finished this one
  int n, chunks, last;  // last: the launch that counts the step
  int alone;            // see GmsParams
  AdamwTensor t[N];
};

__device__ __forceinline__ uint32_t adamw_mix(uint32_t h) {  // the finalizer of MurmurHash3
  h = (h ^ (h >> 16)) * 0x85EBCA6Bu;
  h = (h ^ (h >> 13)) * 0xC2B2AE35u;
  return h ^ (h >> 16);
}

// Eight values as they lie in memory; `vec`: all there, from a 16-byte boundary.
struct AdamwRaw {
  uint4 part[2];  // 16-bit types: the first one
};
__device__ __forceinline__ AdamwRaw adamw_raw(int type, const void* from, long long i, int there, bool vec) {
  AdamwRaw r;
  if (vec) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(from) + (type == 0 ? i * 4 : i * 2));
    r.part[0] = p[0];
    if (type == 0) r.part[1] = p[1];
    else r.part[1] = make_uint4(0, 0, 0, 0);
    return r;
  }
  uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (e >= there) continue;
    if (type == 0) w[e] = static_cast<const uint32_t*>(from)[i + e];
    else w[e / 2] |= (uint32_t)static_cast<const uint16_t*>(from)[i + e] << (16 * (e % 2));
  }
  r.part[0] = make_uint4(w[0], w[1], w[2], w[3]);
  r.part[1] = make_uint4(w[4], w[5], w[6], w[7]);
  return r;
}
// APART: a loop for each type, else a type for each value.  With 8-bit moments, where instructions are what counts, loops apart: 120 M values 415 -> 390 us;
// with 32-bit ones they cost the values that are on their way their registers: 150 M fp32 values 666 -> 771.
template <bool APART>
__device__ __forceinline__ void adamw_widen(int type, const AdamwRaw& r, float (&x)[8]) {
  const uint32_t w[8] = {r.part[0].x, r.part[0].y, r.part[0].z, r.part[0].w, r.part[1].x, r.part[1].y, r.part[1].z, r.part[1].w};
  const auto one = [&](int type, int e) {
    if (type == 0) return __uint_as_float(w[e]);
    if (type == 1) return __half2float(__ushort_as_half((unsigned short)(w[e / 2] >> (16 * (e % 2)))));
    return __uint_as_float(e % 2 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
  };
  if (!APART) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = one(type, e);
  } else if (type == 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = one(0, e);
  } else if (type == 1) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = one(1, e);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = one(2, e);
  }
}
template <typename T>
__device__ __forceinline__ void adamw_store8(void* to, long long i, int there, bool vec, const float (&x)[8]) {
  T* p = static_cast<T*>(to) + i;
  __align__(16) T h[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = from_f32<T>(x[e]);
  if (vec) {
#pragma unroll
    for (int q = 0; q < (int)sizeof(T) / 2; ++q) reinterpret_cast<uint4*>(p)[q] = reinterpret_cast<const uint4*>(h)[q];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < there) p[e] = h[e];
  }
}
__device__ __forceinline__ void adamw_store(int type, void* to, long long i, int there, bool vec, const float (&x)[8]) {
  if (type == 0) adamw_store8<float>(to, i, there, vec, x);
  else if (type == 1) adamw_store8<__half>(to, i, there, vec, x);
  else adamw_store8<__nv_bfloat16>(to, i, there, vec, x);
}

// Packed operations, two values an instruction, each rounded as it would be by itself.
__device__ __forceinline__ uint64_t adamw_two(float lo, float hi) { return (uint64_t)__float_as_uint(lo) | (uint64_t)__float_as_uint(hi) << 32; }
__device__ __forceinline__ void adamw_part(uint64_t v, float& lo, float& hi) {
  lo = __uint_as_float((uint32_t)v);
  hi = __uint_as_float((uint32_t)(v >> 32));
}
__device__ __forceinline__ uint64_t adamw_mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t adamw_add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t adamw_add2_down(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rz.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t adamw_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
// eight codes
__device__ __forceinline__ uint2 adamw_codes(const void* from, long long i, int there, bool vec) {
  const uint8_t* p = static_cast<const uint8_t*>(from) + i;
  if (vec) return *reinterpret_cast<const uint2*>(p);
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < there) w[e / 4] |= (uint32_t)p[e] << (8 * (e % 4));
  return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void adamw_widen_codes(uint2 codes, float scale, float (&x)[8]) {
  const uint32_t w[2] = {codes.x, codes.y};
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    uint32_t two;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(two) : "h"((unsigned short)(w[e / 4] >> (8 * (e % 4)))));
    const __half2 h = *reinterpret_cast<const __half2*>(&two);
    adamw_part(adamw_mul2(adamw_two(__low2float(h), __high2float(h)), adamw_two(scale, scale)), x[e], x[e + 1]);
  }
}
// the largest of three absolute values; NaN where one of them is
__device__ __forceinline__ float adamw_max3(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Codes of this thread's eight values of a block of 128 (16 lanes), and the block's scale.  lot[e]: 16 random bits.
template <bool FLOOR>
__device__ __forceinline__ void adamw_store_codes(void* to, float* scales, long long i, int there, bool vec, const float (&x)[8], const uint32_t (&lot)[8]) {
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = e < there ? x[e] : 0.f;
  float top = adamw_max3(adamw_max3(y[0], y[1], y[2]), adamw_max3(y[3], y[4], y[5]), adamw_max3(y[6], y[7], 0.f));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) top = adamw_max3(top, __shfl_xor_sync(0xffffffffu, top, o), 0.f);
  const bool finite = top < __uint_as_float(0x7f800000u), held = finite && (FLOOR ? top > 0.f : top >= ADAMW_SMALLEST);
  // a block with a value that is not finite is not held: its scale says so, and its values are NaN from then on
  float scale = held ? __fmul_rn(top, (float)(1.0 / 448.0)) : finite ? 0.f : __uint_as_float(0x7fc00000u);
  if (FLOOR && held) scale = fmaxf(scale, ADAMW_SCALE_SMALLEST);  // (its inverse is finite; a product of a code and it may be subnormal, and is not 0)
  const float inverse = held ? __fdiv_rn(1.f, scale) : 0.f;
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int e = 6; e >= 0; e -= 2) {
    float u[2], whole[2];
    adamw_part(adamw_mul2(adamw_two(x[e], x[e + 1]), adamw_two(inverse, inverse)), u[0], u[1]);
    u[0] = fminf(fabsf(u[0]), ADAMW_E4M3_MAX);
    u[1] = fminf(fabsf(u[1]), ADAMW_E4M3_MAX);
    // From 2^-6 on three bits of the mantissa stay: with the bias taken off the exponent they are the code.  Below, codes are 2^-9 apart: the whole
    // part of 512 u + lot / 2^16.  Both come from the bits of floats, 1 + lot / 2^16 and 2^23 + the sum rounded down: conversions would
    // go through a pipe of a quarter of the rate.
    const uint64_t lots = adamw_add2(adamw_two(__uint_as_float(0x3f800000u | lot[e] << 7), __uint_as_float(0x3f800000u | lot[e + 1] << 7)), adamw_two(-1.f, -1.f));
    adamw_part(adamw_add2_down(adamw_fma2(adamw_two(u[0], u[1]), adamw_two(512.f, 512.f), lots), adamw_two(8388608.f, 8388608.f)), whole[0], whole[1]);
#pragma unroll
    for (int q = 1; q >= 0; --q) {
      const uint32_t normal = (__float_as_uint(u[q]) + (lot[e + q] << 4) - ((127u - 7u) << 23)) >> 20;
      uint32_t code = u[q] < 0.015625f ? __float_as_uint(whole[q]) & 15u : normal;
      if (FLOOR) code = max(code, u[q] > 0.f ? 1u : 0u);
      else code |= (__float_as_uint(x[e + q]) >> 24) & 0x80u;
      w[e / 4] = w[e / 4] * 256u + code;
    }
  }
  uint8_t* p = static_cast<uint8_t*>(to) + i;
  if (vec) {
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < there) p[e] = (uint8_t)(w[e / 4] >> (8 * (e % 4)));
  }
  if (threadIdx.x % 16 == 0 && there > 0) scales[i / ADAMW_BLOCK] = scale;
}

// What a step needs of its numbers.
struct AdamwStep {
  float rate, root, keep, unscale, none;
  uint32_t key;
};

// What a thread reads of its eight values of a chunk, of which `there` are the tensor's.  ALL: all of them, on boundaries, in all threads of the
// block, so that nothing of what follows has a condition.
template <bool EIGHT>
struct AdamwIn {
  AdamwRaw g, w;
  AdamwRaw m, v;      // 32 bits
  uint2 mc, vc;       // 8 bits
  float m_scale, v_scale;
  template <bool ALL>
  __device__ __forceinline__ void read(const AdamwTensor& t, long long i, int there_) {
    const int there = ALL ? 8 : there_;
    const bool vec = ALL || (t.aligned && there == 8);
    g = adamw_raw(t.grad_type, t.grad, i, there, vec);
    if (t.master) w = adamw_raw(0, t.master, i, there, vec);
    else w = adamw_raw(t.param_type, t.param, i, there, vec);
    if (EIGHT) {
      const long long b = i / ADAMW_BLOCK;
      mc = adamw_codes(t.m, i, there, vec);
      vc = adamw_codes(t.v, i, there, vec);
      m_scale = there > 0 ? t.m_scale[b] : 0.f;
      v_scale = there > 0 ? t.v_scale[b] : 0.f;
    } else {
      m = adamw_raw(0, t.m, i, there, vec);
      v = adamw_raw(0, t.v, i, there, vec);
    }
  }
};

template <bool EIGHT, bool ALL, typename P>
__device__ __forceinline__ void adamw_values(const P& p, const AdamwTensor& t, const AdamwStep& now, const AdamwIn<EIGHT>& in, long long i, int there_) {
  const int there = ALL ? 8 : there_;
  const bool vec = ALL || (t.aligned && there == 8);
  float w[8], g[8], m[8], v[8];
  adamw_widen<EIGHT>(t.grad_type, in.g, g);
  adamw_widen<EIGHT>(t.master ? 0 : t.param_type, in.w, w);
  if (EIGHT) {
    adamw_widen_codes(in.mc, in.m_scale, m);
    adamw_widen_codes(in.vc, in.v_scale, v);
  } else {
    adamw_widen<false>(0, in.m, m);
    adamw_widen<false>(0, in.v, v);
  }
  uint32_t lot_m[8], lot_v[8];
  // Products that are to be rounded before they are added: with a -0 that is not known when the kernel is compiled.  A packed product and a sum of its own are made
  // one operation with one rounding, their .rn notwithstanding (one moment in five was off by a step).
  const uint64_t none = adamw_two(now.none, now.none);
  const uint64_t b1 = adamw_two(p.b1, p.b1), c1 = adamw_two(p.c1, p.c1), b2 = adamw_two(p.b2, p.b2), c2 = adamw_two(p.c2, p.c2);
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const uint64_t gg = adamw_mul2(adamw_two(g[e], g[e + 1]), adamw_two(now.unscale, now.unscale));
    if (EIGHT) {
      adamw_part(adamw_add2(adamw_fma2(adamw_two(m[e], m[e + 1]), b1, none), adamw_fma2(gg, c1, none)), m[e], m[e + 1]);
      adamw_part(adamw_add2(adamw_fma2(adamw_two(v[e], v[e + 1]), b2, none), adamw_fma2(adamw_mul2(gg, gg), c2, none)), v[e], v[e + 1]);
    } else {
      adamw_part(adamw_fma2(adamw_two(m[e], m[e + 1]), b1, adamw_mul2(gg, c1)), m[e], m[e + 1]);
      adamw_part(adamw_fma2(adamw_two(v[e], v[e + 1]), b2, adamw_mul2(adamw_mul2(gg, gg), c2)), v[e], v[e + 1]);
    }
    float size[2];  // within 2^-23 of the root, also of a subnormal number
    asm("sqrt.approx.f32 %0, %1;" : "=f"(size[0]) : "f"(v[e]));
    asm("sqrt.approx.f32 %0, %1;" : "=f"(size[1]) : "f"(v[e + 1]));
    float under[2];
    adamw_part(adamw_fma2(adamw_two(size[0], size[1]), adamw_two(now.root, now.root), adamw_two(p.eps, p.eps)), under[0], under[1]);
    // a quotient within two steps of the last place, which the rounding of w hides
    const uint64_t move = adamw_two(__fdividef(m[e], under[0]), __fdividef(m[e + 1], under[1]));
    adamw_part(adamw_fma2(move, adamw_two(-now.rate, -now.rate), adamw_mul2(adamw_two(w[e], w[e + 1]), adamw_two(now.keep, now.keep))), w[e], w[e + 1]);
  }
#pragma unroll
  for (int e = 0; EIGHT && e < 8; ++e) {
    const uint32_t h = adamw_mix((uint32_t)(i + e) * 0x9E3779B1u + now.key);
    lot_m[e] = h & 0xffffu;
    lot_v[e] = h >> 16;
  }
  if (t.master) adamw_store8<float>(t.master, i, there, vec, w);
  adamw_store(t.param_type, t.param, i, there, vec, w);
  if (EIGHT) {
    adamw_store_codes<false>(t.m, t.m_scale, i, there, vec, m, lot_m);
    adamw_store_codes<true>(t.v, t.v_scale, i, there, vec, v, lot_v);
  } else {
    adamw_store8<float>(t.m, i, there, vec, m);
    adamw_store8<float>(t.v, i, there, vec, v);
  }
}

// Where a chunk lies.  Chunks ascend, so its tensor is looked for from the last one's on.
template <typename P>
struct AdamwAt {
  int k = 0;
  long long first = 0;
  bool all = false;
  __device__ __forceinline__ void find(const P& p, int chunk) {
    if (k + 1 < p.n && p.t[k + 1].first_chunk <= chunk) {
      int hi = p.n;
      while (hi - k > 1) {
        const int mid = (k + hi) >> 1;
        if (p.t[mid].first_chunk <= chunk) k = mid; else hi = mid;
      }
    }
    first = (long long)(chunk - p.t[k].first_chunk) * ADAMW_CHUNK;
    all = p.t[k].aligned && first + ADAMW_CHUNK <= p.t[k].count;
  }
};

template <bool EIGHT, int N>
__global__ void __launch_bounds__(ADAMW_THREADS, 3) adamw_kernel(const __grid_constant__ AdamwParams<N> p) {
  __shared__ AdamwStep s_now;
  umma::griddep_wait();
  if (!p.alone) umma::griddep_launch_dependents();
  if (p.found_inf && *p.found_inf != 0.f) return;  // the step is not taken, nor counted
  // a whole chunk's values are read while the one before is worked on
  AdamwAt<AdamwParams<N>> at;
  AdamwIn<EIGHT> in;
  const int mine = threadIdx.x * ADAMW_PER_THREAD;
  if ((int)blockIdx.x < p.chunks) {
    at.find(p, blockIdx.x);
    if (at.all) in.template read<true>(p.t[at.k], at.first + mine, 8);
  }
  // The powers in 64 bits, as 1 - beta^t has few of beta's; what is made of them in 32.  A warp each: they are the longest part of a small step.
  if (threadIdx.x % 32 == 0 && threadIdx.x < 96) {
    const uint32_t t = (uint32_t)p.step[0] + 1u;
    const double lr = p.lr_device ? (double)*p.lr_device : p.lr;
    if (threadIdx.x == 64) {
      s_now.keep = (float)(1.0 - lr * p.decay);
      s_now.unscale = p.grad_scale ? __fdiv_rn(1.f, *p.grad_scale) : 1.f;
      s_now.none = __uint_as_float(p.minus_zero);
      s_now.key = adamw_mix((t * 0x9E3779B9u) ^ p.seed);
    } else {
      double power = 1.0, square = threadIdx.x == 0 ? p.beta1 : p.beta2;
      for (uint32_t e = t; e; e >>= 1) {
        if (e & 1u) power *= square;
        square *= square;
      }
      const float rest = (float)(1.0 - power);
      if (threadIdx.x == 0) s_now.rate = __fdiv_rn((float)lr, rest);
      else s_now.root = __fdiv_rn(1.f, __fsqrt_rn(rest));
    }
  }
  __syncthreads();
  const AdamwStep now = s_now;

  for (int chunk = blockIdx.x; chunk < p.chunks; chunk += gridDim.x) {
    const AdamwAt<AdamwParams<N>> here = at;
    AdamwIn<EIGHT> have = in;
    if (chunk + (int)gridDim.x < p.chunks) {
      at.find(p, chunk + gridDim.x);
      if (at.all) in.template read<true>(p.t[at.k], at.first + mine, 8);
    }
    const AdamwTensor& t = p.t[here.k];
    const long long i = here.first + mine;
    if (here.all) {
      adamw_values<EIGHT, true>(p, t, now, have, i, 8);
    } else {
      const int there = (int)min(max(t.count - i, 0ll), 8ll);
      have.template read<false>(t, i, there);
      adamw_values<EIGHT, false>(p, t, now, have, i, there);
    }
  }
  // the block that finishes last counts the step: by then all have read it
  if (p.last) {
    __syncthreads();
    if (threadIdx.x == 0) {
      if (atomicAdd(p.step + 1, 1) == (int)gridDim.x - 1) {
        p.step[1] = 0;
        p.step[0] += 1;
      }
    }
  }
}

constexpr int ADAMW_FEW = 48, ADAMW_MANY = 400;  // tensors of a launch: 4 KB of arguments, or 32

}  // namespace fgms
