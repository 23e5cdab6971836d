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

}  // namespace
}  // namespace zrnn
