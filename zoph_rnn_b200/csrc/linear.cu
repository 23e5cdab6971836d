// Y = act(W X + bias) + R.
#include <algorithm>
#include <cstring>

#include "kernels.cuh"
#include "linear_device.cuh"
#include "operators.cuh"

namespace zrnn {
namespace {

// 32 outputs x 32 columns per CTA of 256 threads, four columns per thread
template <class T>
__global__ void __launch_bounds__(256) linear_simple_kernel(const LinearArgs a) {
  __shared__ float w[32][33], x[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const long long i0 = (long long)blockIdx.x * 32, c0 = (long long)blockIdx.y * 32;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < a.K; k0 += 32) {
    for (int r = ty; r < 32; r += 8) {
      w[r][tx] = i0 + r < a.n && k0 + tx < a.K ? to_f32(static_cast<const T*>(a.W)[(i0 + r) * a.ldw + k0 + tx]) : 0.f;
      x[r][tx] = c0 + r < a.N && k0 + tx < a.K ? to_f32(static_cast<const T*>(a.X)[(c0 + r) * a.ldx + k0 + tx]) : 0.f;
    }
    __syncthreads();
    for (int k = 0; k < 32; ++k)
      for (int u = 0; u < 4; ++u) acc[u] = fmaf(w[tx][k], x[ty + 8 * u][k], acc[u]);
    __syncthreads();
  }
  const long long i = i0 + tx;
  if (i >= a.n) return;
  const float b = a.bias ? a.bias[i] : 0.f;
  for (int u = 0; u < 4; ++u) {
    const long long c = c0 + ty + 8 * u;
    if (c >= a.N) continue;
    float y = linear_act(acc[u] + b, a.act);
    if (a.R) y += to_f32(static_cast<const T*>(a.R)[c * a.ldr + i]);
    static_cast<T*>(a.Y)[c * a.ldy + i] = from_f32<T>(y);
  }
}

}  // namespace

size_t linear_work(const LinearArgs&, int) { return 0; }
cudaError_t launch_linear(const LinearArgs& a, int elem, cudaStream_t st) {
  if (a.n == 0 || a.N == 0) return cudaSuccess;
  const dim3 grid((a.n + 31) / 32, (a.N + 31) / 32);
  count_launch();
  switch (elem) {
    case ELEM_F32: linear_simple_kernel<float><<<grid, 256, 0, st>>>(a); break;
    case ELEM_BF16: linear_simple_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a); break;
    default: linear_simple_kernel<__half><<<grid, 256, 0, st>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace zrnn
