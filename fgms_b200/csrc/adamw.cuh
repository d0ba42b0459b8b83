// One AdamW step over many tensors in one launch (fgms_b200_adamw).
//
//   g  = grad / grad_scale
//   m' = b1 m + (1 - b1) g         v' = b2 v + (1 - b2) g^2
//   w' = w (1 - lr decay) - lr / (1 - b1^t)  m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// w is the fp32 master where there is one, else the parameter; the parameter is w' rounded once.  All arithmetic is fp32 with
// every operation rounded by itself (no contraction): the moments are the same bits as the formulas evaluated one operation at a time.
//
// Moments in 8 bits: e4m3 codes with an fp32 scale (largest value / 448) for each 128 values.  A moving average moves by less than half a
// code per step (v by 0.1 % where codes are 12 % apart) and rounding to the nearest code would leave it where it is, so a value is rounded up with
// the probability of the part that is cut off: the mean is kept.  The random bits are a hash of (seed, step, index), so a step can be
// repeated bit for bit.  A second moment above zero never becomes zero (its m would then be divided by eps alone): it takes the smallest
// code.  w' is computed from m' and v' before they are rounded.
//
// What bounds it is memory: 28 bytes a value with moments in 32 bits (fp32, or 16-bit parameters with masters), 12 or 16 in 8.
#pragma once
#include "grouped.cuh"  // to_f32, from_f32

namespace fgms {

constexpr int ADAMW_THREADS = 256;
constexpr int ADAMW_PER_THREAD = 8;  // consecutive values
constexpr int ADAMW_CHUNK = ADAMW_THREADS * ADAMW_PER_THREAD;
constexpr int ADAMW_BLOCK = 128;  // values that share a scale: 16 lanes
constexpr float ADAMW_E4M3_MAX = 448.0f;
constexpr float ADAMW_SMALLEST = 7.88860905e-31f;  // 2^-100: a block whose largest value is smaller is held as zeros

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
  uint32_t seed;
  const float *lr_device, *grad_scale, *found_inf;
  int* step;  // [2]: steps done, and blocks that have finished this one
  int n, chunks, last;  // last: the launch that counts the step
  AdamwTensor t[N];
};

__device__ __forceinline__ uint32_t adamw_mix(uint32_t h) {  // the finalizer of MurmurHash3
  h = (h ^ (h >> 16)) * 0x85EBCA6Bu;
  h = (h ^ (h >> 13)) * 0xC2B2AE35u;
  return h ^ (h >> 16);
}

template <typename T>
__device__ __forceinline__ void adamw_load8(const void* from, long long i, int there, bool vec, float (&x)[8]) {
  const T* p = static_cast<const T*>(from) + i;
  if (vec) {
    __align__(16) T h[8];
#pragma unroll
    for (int q = 0; q < (int)sizeof(T) / 2; ++q) reinterpret_cast<uint4*>(h)[q] = reinterpret_cast<const uint4*>(p)[q];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = to_f32(h[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = e < there ? to_f32(p[e]) : 0.f;
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
__device__ __forceinline__ void adamw_load(int type, const void* from, long long i, int there, bool vec, float (&x)[8]) {
  if (type == 0) adamw_load8<float>(from, i, there, vec, x);
  else if (type == 1) adamw_load8<__half>(from, i, there, vec, x);
  else adamw_load8<__nv_bfloat16>(from, i, there, vec, x);
}
__device__ __forceinline__ void adamw_store(int type, void* to, long long i, int there, bool vec, const float (&x)[8]) {
  if (type == 0) adamw_store8<float>(to, i, there, vec, x);
  else if (type == 1) adamw_store8<__half>(to, i, there, vec, x);
  else adamw_store8<__nv_bfloat16>(to, i, there, vec, x);
}

// eight codes, widened and scaled
__device__ __forceinline__ void adamw_load_codes(const void* from, long long i, int there, bool vec, float scale, float (&x)[8]) {
  const uint8_t* p = static_cast<const uint8_t*>(from) + i;
  uint32_t w[2] = {0u, 0u};
  if (vec) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    w[0] = u.x;
    w[1] = u.y;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < there) w[e / 4] |= (uint32_t)p[e] << (8 * (e % 4));
  }
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    uint32_t two;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(two) : "h"((unsigned short)(w[e / 4] >> (8 * (e % 4)))));
    const __half2 h = *reinterpret_cast<const __half2*>(&two);
    x[e] = __fmul_rn(__low2float(h), scale);
    x[e + 1] = __fmul_rn(__high2float(h), scale);
  }
}

// Codes of this thread's eight values of a block of 128 (16 lanes), and the block's scale.  lot[e]: 16 random bits.
template <bool FLOOR>
__device__ __forceinline__ void adamw_store_codes(void* to, float* scales, long long i, int there, bool vec, const float (&x)[8], const uint32_t (&lot)[8]) {
  uint32_t largest = 0;  // of the absolute values' bits: a NaN is larger than all else and stays
#pragma unroll
  for (int e = 0; e < 8; ++e) largest = max(largest, e < there ? __float_as_uint(x[e]) & 0x7fffffffu : 0u);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, o));
  const float top = __uint_as_float(largest);
  const bool finite = largest < 0x7f800000u, held = finite && top >= ADAMW_SMALLEST;
  // a block with a value that is not finite is not held: its scale says so, and its values are NaN from then on
  const float scale = held ? __fmul_rn(top, (float)(1.0 / 448.0)) : finite ? 0.f : __uint_as_float(0x7fc00000u);
  const float inverse = held ? __fdiv_rn(1.f, scale) : 0.f;
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float u = held ? fminf(__fmul_rn(fabsf(x[e]), inverse), ADAMW_E4M3_MAX) : 0.f;
    // 2^-6 and more: three bits of the mantissa stay; below, codes are 2^-9 apart
    const uint32_t normal = ((__float_as_uint(u) + (lot[e] << 4)) >> 20) - ((127u - 7u) << 3);
    uint32_t small = (uint32_t)__fadd_rn(__fmul_rn(u, 512.f), __fmul_rn((float)lot[e], 1.f / 65536.f));
    if (FLOOR && u > 0.f) small = max(small, 1u);
    const uint32_t code = (u >= 0.015625f ? normal : small) | (FLOOR ? 0u : (__float_as_uint(x[e]) >> 31) << 7);
    w[e / 4] |= code << (8 * (e % 4));
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

template <bool EIGHT, int N>
__global__ void __launch_bounds__(ADAMW_THREADS, 4) adamw_kernel(const __grid_constant__ AdamwParams<N> p) {
  __shared__ float s_rate, s_root, s_keep, s_unscale;
  __shared__ uint32_t s_key;
  umma::griddep_wait();
  umma::griddep_launch_dependents();
  if (p.found_inf && *p.found_inf != 0.f) return;  // the step is not taken, nor counted
  if (threadIdx.x == 0) {
    const uint32_t t = (uint32_t)p.step[0] + 1u;
    double pow1 = 1.0, pow2 = 1.0, s1 = p.beta1, s2 = p.beta2;
    for (uint32_t e = t; e; e >>= 1) {
      if (e & 1u) { pow1 *= s1; pow2 *= s2; }
      s1 *= s1;
      s2 *= s2;
    }
    const double lr = p.lr_device ? (double)*p.lr_device : p.lr;
    s_rate = (float)(lr / (1.0 - pow1));
    s_root = (float)(1.0 / sqrt(1.0 - pow2));
    s_keep = (float)(1.0 - lr * p.decay);
    s_unscale = p.grad_scale ? __fdiv_rn(1.f, *p.grad_scale) : 1.f;
    s_key = adamw_mix((t * 0x9E3779B9u) ^ p.seed);
  }
  __syncthreads();
  const float rate = s_rate, root = s_root, keep = s_keep, unscale = s_unscale;
  const uint32_t key = s_key;

  int k = 0;  // the tensor of the chunk: chunks ascend, so it is looked for from the last one's on
  for (int chunk = blockIdx.x; chunk < p.chunks; chunk += gridDim.x) {
    if (k + 1 < p.n && p.t[k + 1].first_chunk <= chunk) {
      int hi = p.n;
      while (hi - k > 1) {
        const int mid = (k + hi) >> 1;
        if (p.t[mid].first_chunk <= chunk) k = mid; else hi = mid;
      }
    }
    const AdamwTensor& t = p.t[k];
    const long long i = (long long)(chunk - t.first_chunk) * ADAMW_CHUNK + threadIdx.x * ADAMW_PER_THREAD;
    const int there = (int)min(max(t.count - i, 0ll), 8ll);
    const bool vec = t.aligned && there == 8;
    float w[8], g[8], m[8], v[8];
    adamw_load(t.grad_type, t.grad, i, there, vec, g);
    if (t.master) adamw_load8<float>(t.master, i, there, vec, w);
    else adamw_load(t.param_type, t.param, i, there, vec, w);
    if (EIGHT) {
      const long long b = i / ADAMW_BLOCK;
      adamw_load_codes(t.m, i, there, vec, there > 0 ? t.m_scale[b] : 0.f, m);
      adamw_load_codes(t.v, i, there, vec, there > 0 ? t.v_scale[b] : 0.f, v);
    } else {
      adamw_load8<float>(t.m, i, there, vec, m);
      adamw_load8<float>(t.v, i, there, vec, v);
    }
    uint32_t lot_m[8], lot_v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float ge = p.grad_scale ? __fmul_rn(g[e], unscale) : g[e];
      m[e] = __fadd_rn(__fmul_rn(m[e], p.b1), __fmul_rn(ge, p.c1));
      v[e] = __fadd_rn(__fmul_rn(v[e], p.b2), __fmul_rn(__fmul_rn(ge, ge), p.c2));
      const float denominator = __fadd_rn(__fmul_rn(__fsqrt_rn(v[e]), root), p.eps);
      w[e] = __fsub_rn(__fmul_rn(w[e], keep), __fmul_rn(rate, __fdiv_rn(m[e], denominator)));
      if (EIGHT) {
        const uint32_t h = adamw_mix((uint32_t)(i + e) * 0x9E3779B1u + key);
        lot_m[e] = h & 0xffffu;
        lot_v[e] = h >> 16;
      }
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
  // the block that finishes last counts the step: by then all have read it
  if (p.last) {
    __syncthreads();
    if (threadIdx.x == 0) {
      __threadfence();
      if (atomicAdd(p.step + 1, 1) == (int)gridDim.x - 1) {
        p.step[1] = 0;
        p.step[0] += 1;
      }
    }
  }
}

constexpr int ADAMW_FEW = 48, ADAMW_MANY = 400;  // tensors of a launch: 4 KB of arguments, or 32

}  // namespace fgms
