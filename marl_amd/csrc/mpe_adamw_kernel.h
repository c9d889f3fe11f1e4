// One AdamW step over many tensors, with each gradient's clip before it and the target's polyak step behind it.
//
// For a variable p with gradient g (all in f32, in this order, no fused multiply-add):
//     g' = g * (c / max(|g|, c))                          with max_norm c; |g| summed in 64 bits, rounded once
//     m  = m b1 + g' (1 - b1)
//     v  = v b2 + (g' g') (1 - b2)
//     p  = p (1 - lr wd) - (m / (sqrt(v) / sqrt(1 - b2^t) + eps)) (lr / (1 - b1^t))       rounded to p's type
//     t  = t rho + p (1 - rho)                            with a target; p as it is stored
//
// Moments in 8 bits.  A float's leading bits are a logarithmic code of their own: bits >> 20 counts eighths of a binade.
// A block of 128 consecutive elements of a variable shares a base; an element holds the difference, 7 bits and the sign for
// m (16 binades), 8 bits for v (32 binades, i.e. 16 of sqrt(v)); code 0 is zero, code c > 0 the float (c + base) << 20.  The
// base follows the block's largest element, so that no code overflows.  Rounding is stochastic: random bits below the kept
// ones are added before the cut, which makes the held value right on average.  Rounding to nearest would stop v: with
// b2 = 0.999 a step moves v by 0.1 % of itself, and half a code step is 6 %.  v > 0 is never held as zero (m / eps would be
// a giant step), it becomes the block's smallest value; an m under the block's range becomes zero.
//
// One pass: every value is read and written once (with a clip, gradients of more than one work item are read twice).  Work items
// of 8 192 values: 8 values a thread a turn, 16-byte accesses, no tensor shares an item, so the smallest and the largest tensors
// need one launch together.  Bound by memory: 62 M f32 values with clip and target (2.2 GB) 540 us = 4.2 TB/s, 302 M bf16
// values with 8-bit moments (3.0 GB) 623 us = 4.9 TB/s, the vector units 92 % active; 48 variables of 4 learners 9 us, 28 from
// Python.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mpe {

constexpr int kAdamBlock = 128;    // elements that share a base
constexpr int kAdamItem = 8192;    // elements of a work item (one workgroup)
constexpr int kAdamThreads = 256;
constexpr int kAdamMaxGrads = 448; // gradients (pointers in the kernel's arguments, which end at 4 KiB) per launch

struct AdamTensor {
  void *param, *target, *exp_avg, *exp_avg_base, *exp_avg_sq, *exp_avg_sq_base;
  int64_t count;
  uint32_t first_item, items;
};
struct AdamItem { uint32_t tensor, index; };
struct AdamScalars { float step_size, root, decay; uint32_t key; };  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t), 1 - lr wd
struct AdamClock { int64_t step; AdamScalars s; };                   // device form of the step count
struct AdamArgs {
  const AdamTensor *tensors;
  const AdamItem *items;
  double *norms;  // partial sums of squares, one per item
  const AdamClock *clock;  // NULL: `s`
  AdamScalars s;
  float beta1, beta1c, beta2, beta2c, eps, max_norm, polyak, polyakc;
  uint32_t first_tensor, first_item;  // of this launch
  uint32_t index0;                    // the first tensor's number in the random streams
  const void *grads[kAdamMaxGrads];
};
static_assert(sizeof(AdamArgs) <= 4096, "kernel arguments");

template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Eight { T v[8]; };

template <typename T>
__device__ __forceinline__ void adam_load8(const T *p, int valid, float out[8]) {
  if (valid >= 8) {
    const Eight<T> e = *reinterpret_cast<const Eight<T> *>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = (float)e.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = i < valid ? (float)p[i] : 0.0f;
  }
}
template <typename T>
__device__ __forceinline__ void adam_store8(T *p, int valid, const T in[8]) {
  if (valid >= 8) {
    Eight<T> e;
#pragma unroll
    for (int i = 0; i < 8; ++i) e.v[i] = in[i];
    *reinterpret_cast<Eight<T> *>(p) = e;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < valid) p[i] = in[i];
  }
}

// 32-bit finaliser of MurmurHash3 (A. Appleby, public domain): a bijection whose outputs look random
__device__ __host__ __forceinline__ uint32_t adam_mix(uint32_t h) {
  h ^= h >> 16;
  h *= 0x85EBCA6Bu;
  h ^= h >> 13;
  h *= 0xC2B2AE35u;
  return h ^ (h >> 16);
}
__device__ __host__ __forceinline__ uint32_t adam_step_key(uint64_t seed, int64_t step) {
  return adam_mix((uint32_t)seed + (uint32_t)step * 0x9E3779B9u) ^ (uint32_t)(seed >> 32);
}

__device__ __forceinline__ float adam_decode(uint32_t mag, uint32_t base) {
  return mag ? __uint_as_float((mag + base) << 20) : 0.0f;
}

// maximum over the 16 lanes of a row (the lanes of one 128-element block)
__device__ __forceinline__ uint32_t row_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x128, 0xf, 0xf, false));  // row_ror:8
  x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x124, 0xf, 0xf, false));
  x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x122, 0xf, 0xf, false));
  return max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x121, 0xf, 0xf, false));
}

// codes of eight elements (two words) and the base of their block of 128
template <bool SIGNED>
__device__ __forceinline__ uint2 adam_encode(const float x[8], const uint32_t rnd[8], uint32_t &base) {
  constexpr uint32_t kTop = SIGNED ? 127u : 255u;
  uint32_t bits[8], most = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    bits[i] = __float_as_uint(x[i]) & 0x7FFFFFFFu;
    most = max(most, bits[i]);
  }
  most = row_max(most) >> 20;
  base = most + 1 > kTop ? most + 1 - kTop : 0;  // + 1: rounding may carry
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t up = min(bits[i] + rnd[i], 0x7FFFFFFFu) >> 20;
    uint32_t code = up > base ? up - base : 0;
    if (SIGNED) code |= (__float_as_uint(x[i]) >> 31) << 7;
    else code = max(code, bits[i] ? 1u : 0u);
    w[i >> 2] |= code << (8 * (i & 3));
  }
  return uint2{w[0], w[1]};
}

// Sum over the workgroup in a fixed order; every thread gets it.
__device__ __forceinline__ double adam_block_sum(double s) {
  __shared__ double part[kAdamThreads / 64];
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  return (part[0] + part[1]) + (part[2] + part[3]);
}

// Sum of squares of [begin, end), at most an item, over the workgroup's threads: every load first, then the sums.
template <typename T>
__device__ __forceinline__ double adam_squares(const T *g, int64_t begin, int64_t end) {
  constexpr int kRounds = kAdamItem / (8 * kAdamThreads);
  float x[kRounds][8];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = begin + 8 * (threadIdx.x + r * kAdamThreads);
    adam_load8(g + i, end - i >= 8 ? 8 : (end > i ? (int)(end - i) : 0), x[r]);
  }
  double s = 0.0;
#pragma unroll
  for (int r = 0; r < kRounds; ++r)
#pragma unroll
    for (int e = 0; e < 8; ++e) s = __builtin_fma((double)x[r][e], (double)x[r][e], s);
  return s;
}

// Clip, variables of more than one item: the items' sums of squares.
template <typename T>
__global__ __launch_bounds__(kAdamThreads) void adamw_norm_kernel(const AdamArgs a) {
  const AdamItem it = a.items[a.first_item + blockIdx.x];
  const AdamTensor &t = a.tensors[it.tensor];
  const T *g = static_cast<const T *>(a.grads[it.tensor - a.first_tensor]);
  if (t.items == 1 || g == nullptr) return;
  const int64_t begin = (int64_t)it.index * kAdamItem, end = begin + kAdamItem < t.count ? begin + kAdamItem : t.count;
  const double s = adam_block_sum(adam_squares(g, begin, end));
  if (threadIdx.x == 0) a.norms[a.first_item + blockIdx.x] = s;
}

// FAST: 16-bit parameters with 8-bit moments, 10 bytes a value, leave ~90 vector instructions at the memory's rate, and a correctly
// rounded root and quotient take 20 of them (302 M values bf16: 725 us, 623 without): there the 1-ulp instructions, whose error is
// 2^-12 (f16) or 2^-15 (bf16) of what rounding the parameter brings.  The root's instruction reads subnormal v as zero: the host
// takes FAST only where eps drowns that.  f32 parameters have bytes enough to hide the rounded ones (62 M values: 207 us, 201
// without; with targets 305, 304).
template <typename T, bool EIGHT, bool CLIP, bool FAST>
__global__ __launch_bounds__(kAdamThreads) void adamw_kernel(const AdamArgs a) {
  const AdamItem it = a.items[a.first_item + blockIdx.x];
  const AdamTensor t = a.tensors[it.tensor];
  const T *g = static_cast<const T *>(a.grads[it.tensor - a.first_tensor]);
  T *p = static_cast<T *>(t.param), *target = static_cast<T *>(t.target);
  if (g == nullptr && target == nullptr) return;
  const int64_t begin = (int64_t)it.index * kAdamItem, end = begin + kAdamItem < t.count ? begin + kAdamItem : t.count;
  const AdamScalars s = a.clock ? a.clock->s : a.s;
  float scale = 1.0f;
  if (CLIP && g != nullptr) {
    double sum = 0.0;
    if (t.items == 1) sum = adam_squares(g, begin, end);
    else
      for (uint32_t i = threadIdx.x; i < t.items; i += kAdamThreads) sum += a.norms[t.first_item + i];
    const double root = sqrt(adam_block_sum(sum));
    const float norm = (float)root;
    scale = a.max_norm / (norm < a.max_norm ? a.max_norm : norm);        // NaN stays NaN
    if (norm > 3.4e38f && root < 1e300) scale = (float)(a.max_norm / root);  // finite elements, a norm beyond 32 bits
  }
  const uint32_t key = EIGHT ? adam_mix(s.key + (a.index0 + it.tensor - a.first_tensor) * 0x85EBCA77u) : 0;
  // whole wavefronts run to the end of the last block of 128: its lanes exchange their largest element
  const int64_t stop = (end + kAdamBlock - 1) / kAdamBlock * kAdamBlock;
  for (int64_t i = begin + 8 * threadIdx.x; i < stop; i += 8 * kAdamThreads) {
    const int valid = end - i >= 8 ? 8 : (end > i ? (int)(end - i) : 0);
    float x[8];
    T held[8];
    adam_load8(p + i, valid, x);
    if (g != nullptr) {
      float d[8], m[8], v[8];
      adam_load8(g + i, valid, d);
      if (EIGHT) {
        const uint2 cm = *reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(t.exp_avg) + i);
        const uint2 cv = *reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(t.exp_avg_sq) + i);
        const uint32_t bm = (uint16_t)static_cast<const int16_t *>(t.exp_avg_base)[i / kAdamBlock];
        const uint32_t bv = (uint16_t)static_cast<const int16_t *>(t.exp_avg_sq_base)[i / kAdamBlock];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t c = ((e < 4 ? cm.x : cm.y) >> (8 * (e & 3))) & 255u, w = ((e < 4 ? cv.x : cv.y) >> (8 * (e & 3))) & 255u;
          m[e] = __uint_as_float(__float_as_uint(adam_decode(c & 127u, bm)) | (c >> 7) << 31);
          v[e] = adam_decode(w, bv);
        }
      } else {
        adam_load8(static_cast<const float *>(t.exp_avg) + i, 8, m);
        adam_load8(static_cast<const float *>(t.exp_avg_sq) + i, 8, v);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float gc = CLIP ? d[e] * scale : d[e];
        m[e] = m[e] * a.beta1 + gc * a.beta1c;
        v[e] = v[e] * a.beta2 + (gc * gc) * a.beta2c;
        const float q = FAST ? m[e] * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v[e]) * s.root + a.eps)
                             : m[e] / (sqrtf(v[e]) * s.root + a.eps);
        x[e] = x[e] * s.decay - q * s.step_size;
        held[e] = (T)x[e];
        if (e >= valid) m[e] = v[e] = 0.0f;  // nothing behind the variable's end reaches its block
      }
      if (EIGHT) {
        const uint32_t k2 = key + (uint32_t)(i >> 32) * 0x9E3779B1u;
        uint32_t rm[8], rv[8], base_m, base_v;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t h = adam_mix(((uint32_t)i + e) ^ k2);
          rm[e] = (h >> 16) << 4;
          rv[e] = (h & 0xFFFFu) << 4;
        }
        const uint2 cm = adam_encode<true>(m, rm, base_m), cv = adam_encode<false>(v, rv, base_v);
        *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(t.exp_avg) + i) = cm;
        *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(t.exp_avg_sq) + i) = cv;
        if ((threadIdx.x & 15) == 0) {
          static_cast<int16_t *>(t.exp_avg_base)[i / kAdamBlock] = (int16_t)base_m;
          static_cast<int16_t *>(t.exp_avg_sq_base)[i / kAdamBlock] = (int16_t)base_v;
        }
      } else {
        adam_store8(static_cast<float *>(t.exp_avg) + i, 8, m);
        adam_store8(static_cast<float *>(t.exp_avg_sq) + i, 8, v);
      }
      adam_store8(p + i, valid, held);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (float)held[e];
    }
    if (target != nullptr) {
      float y[8];
      adam_load8(target + i, valid, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) held[e] = (T)(y[e] * a.polyak + x[e] * a.polyakc);
      adam_store8(target + i, valid, held);
    }
  }
}

// Device form of the step count: one more step, and the factors that follow from it (in 64 bits: 1 - b^t cancels).
__global__ void adamw_clock_kernel(AdamClock *c, double lr, double beta1, double beta2, double weight_decay, uint64_t seed) {
  const int64_t t = c->step + 1;
  c->step = t;
  c->s.step_size = (float)(lr / (1.0 - pow(beta1, (double)t)));
  c->s.root = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)t)));
  c->s.decay = (float)(1.0 - lr * weight_decay);
  c->s.key = adam_step_key(seed, t);
}

// 8-bit moments as the values they stand for (four significant bits: exact in T = f32 or bf16); blockIdx.y: first, second
struct AdamMoments { const uint8_t *codes[2]; const int16_t *base[2]; void *out[2]; };
template <typename T>
__global__ __launch_bounds__(256) void adamw_moments_kernel(AdamMoments a, int64_t count) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  const bool first = blockIdx.y == 0;
  const uint8_t *codes = first ? a.codes[0] : a.codes[1];
  if (i >= count || codes == nullptr) return;
  const uint2 c = *reinterpret_cast<const uint2 *>(codes + i);
  const uint32_t b = (uint16_t)(first ? a.base[0] : a.base[1])[i / kAdamBlock];
  T v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t w = ((e < 4 ? c.x : c.y) >> (8 * (e & 3))) & 255u;
    const float x = first ? __uint_as_float(__float_as_uint(adam_decode(w & 127u, b)) | (w >> 7) << 31) : adam_decode(w, b);
    v[e] = (T)x;
  }
  adam_store8(static_cast<T *>(first ? a.out[0] : a.out[1]) + i, 8, v);
}

}  // namespace mpe
