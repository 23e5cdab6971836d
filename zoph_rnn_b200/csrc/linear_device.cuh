// The activations of zrnn_linear, in 32 bits whatever the operands' type.
#pragma once
#include <cuda_runtime.h>

#include "operators.cuh"

namespace zrnn {
namespace {

__device__ __forceinline__ float linear_act(float x, int act) {
  switch (act) {
    case ACT_TANH: return tanhf(x);
    case ACT_SIGMOID: return 1.0f / (1.0f + expf(-x));
    case ACT_RELU: return x > 0.f ? x : (x != x ? x : 0.f);  // (a NaN stays one)
    case ACT_GELU: return 0.5f * x * (1.0f + erff(x * 0.70710678118654752f));
    case ACT_SILU: return x / (1.0f + expf(-x));
  }
  return x;
}

// x in 32 bits as two tf32 operands, of which the tensor cores take the upper 19 bits: hi is x as it is, cut off there; lo what that leaves,
// 13 bits of which 11 count.  What lo loses makes an operand smaller by some 1e-7 of itself; rounding it instead would take three more
// instructions per element, and the splitting of a stage takes as long as its products.  Of an infinity lo is NaN.
__device__ __forceinline__ uint32_t tf32_rest(uint32_t x) { return __float_as_uint(__uint_as_float(x) - __uint_as_float(x & 0xffffe000u)); }
__device__ __forceinline__ void split_tf32(uint32_t x, uint32_t& hi, uint32_t& lo) {
  hi = x;
  lo = tf32_rest(x);
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
