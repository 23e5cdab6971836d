// The activations of zrnn_linear, in 32 bits whatever the operands' type.
#pragma once
#include <cuda_runtime.h>

#include "att_device.cuh"
#include "operators.cuh"

namespace zrnn {
namespace {

__device__ __forceinline__ float linear_act(float x, int act) {
  switch (act) {
    case ACT_TANH: return tanh_f32(x);  // (the gates' functions: within 1.2e-7, in a third of tanhf's and an IEEE division's instructions)
    case ACT_SIGMOID: return sigmoid_f32(x);
    case ACT_RELU: return x > 0.f ? x : (x != x ? x : 0.f);  // (a NaN stays one)
    case ACT_GELU: return 0.5f * x * (1.0f + erff(x * 0.70710678118654752f));
    case ACT_SILU: return x * sigmoid_f32(x);
  }
  return x;
}

// x in 32 bits as two tf32 operands (11 bits of mantissa; the tensor cores ignore what lies below), whose product with another one's leaves out lo lo.
// hi is x rounded to the nearest, so that lo has either sign and is 2^-11 of x at most: what is left out is small and has no side.  (An infinity's hi is the
// largest number, its lo the infinity; a NaN's are both NaN.)
__device__ __forceinline__ uint32_t tf32_near(float x) {
  uint32_t r;
  asm("cvt.rn.satfinite.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return r;
}
// lo has up to 13 bits, of which the tensor cores cut off those below 11: a little more, half a step where the mantissa is 1.5, makes that a rounding,
// off to either side as often.
__device__ __forceinline__ uint32_t tf32_less_cut(float lo) { return __float_as_uint(fmaf(lo, 1.0f / 2048.0f / 1.5f, lo)); }
__device__ __forceinline__ void split_tf32(uint32_t x, uint32_t& hi, uint32_t& lo) {
  hi = tf32_near(__uint_as_float(x));
  lo = tf32_less_cut(__uint_as_float(x) - __uint_as_float(hi));
}
// ... where x stays as it is and hi is what the tensor cores leave of it.  One factor of a product may be split so: its lo is up to 2^-10 of x, with x's
// sign, but what is left out has the other factor's.  (With both hi parts cut off, and lo, sums of positive products came out 2.7e-7 too small, of
// numbers just below 1 + 2^-10 1.3e-6; now 0.5e-7.)  Of an infinity: NaN.
__device__ __forceinline__ uint32_t tf32_rest(uint32_t x) { return tf32_less_cut(__uint_as_float(x) - __uint_as_float(x & 0xffffe000u)); }

// 16 bytes of a row from element k on, zeros from K on.  Rows that lie on 16 bytes with K a multiple of a vector: one load.
template <class T, bool ALIGNED>
__device__ __forceinline__ uint4 load16(const T* row, int k, int K, bool in) {
  constexpr int V = 16 / sizeof(T);
  uint4 r = make_uint4(0u, 0u, 0u, 0u);
  if (!in || k >= K) return r;
  if (ALIGNED) return __ldg(reinterpret_cast<const uint4*>(row + k));
  if constexpr (sizeof(T) == 4) {
    const unsigned* p = reinterpret_cast<const unsigned*>(row + k);
    r.x = __ldg(p);
    if (k + 1 < K) r.y = __ldg(p + 1);
    if (k + 2 < K) r.z = __ldg(p + 2);
    if (k + 3 < K) r.w = __ldg(p + 3);
  } else {
    const unsigned short* p = reinterpret_cast<const unsigned short*>(row + k);
    if (k + V < K) {  // (not the row's last element: the fifth word ends inside the row)
      const unsigned* q = reinterpret_cast<const unsigned*>((uintptr_t)p & ~(uintptr_t)3);
      const unsigned odd = ((uintptr_t)p & 2) * 8;
      unsigned w[5];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __ldg(q + i);
      w[4] = odd ? __ldg(q + 4) : 0u;
      r = make_uint4(__funnelshift_r(w[0], w[1], odd), __funnelshift_r(w[1], w[2], odd), __funnelshift_r(w[2], w[3], odd), __funnelshift_r(w[3], w[4], odd));
    } else {
      unsigned w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (k + i < K) w[i / 2] |= (unsigned)__ldg(p + i) << (16 * (i & 1));
      r = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  return r;
}

// tensor memory for a CTA without a partner, by one warp
__device__ __forceinline__ void lin_tmem_alloc(uint32_t* base, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"((uint32_t)__cvta_generic_to_shared(base)), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void lin_tmem_free(uint32_t base, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
}

}  // namespace
}  // namespace zrnn
