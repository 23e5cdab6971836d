// The source memory in 4 bits: packing, reading back, and attention over it.
#include <algorithm>
#include <cstring>

#include "kernels.cuh"
#include "operators.cuh"

namespace zrnn {
namespace {

constexpr float kSeventh = 0.14285714924335479736328125f;  // 1/7 rounded to 32 bits
constexpr float kMaxScale = 9352.0f;                       // the largest half that times 7 is finite

// A warp per group, a lane per element.  The scale is fp16(a / 7) of the largest magnitude a (a product with 1/7 in 32 bits).  The code is the
// integer nearest to x / s, ties to even: the rounded quotient can be off by one only where 32 bits end up on the middle between two codes,
// which the remainder x - q s (exact: at most 24 bits) tells apart.
template <class T>
__global__ void __launch_bounds__(256) mem4_pack_kernel(const Mem4Pack a) {
  const int G = mem4_groups(a.d), lane = threadIdx.x & 31;
  const long long total = (long long)a.S * a.B * a.heads * G;
  for (long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); w < total; w += (long long)gridDim.x * 8) {
    const int g = (int)(w % G);
    long long r = w / G;
    const int h = (int)(r % a.heads);
    r /= a.heads;
    const int b = (int)(r % a.B), s = (int)(r / a.B);
    const int i = g * kMem4Group + lane;
    const float x = i < a.d ? to_f32(static_cast<const T*>(a.x)[s * a.ld_slot + b * a.ld_col + (long long)h * a.d + i]) : 0.f;
    unsigned m = __float_as_uint(x) & 0x7fffffffu;  // (as integers: a NaN is the largest)
    m = __reduce_max_sync(0xffffffffu, m);
    const __half sh = m < 0x7f800000u ? __float2half_rn(fminf(__uint_as_float(m) * kSeventh, kMaxScale)) : __ushort_as_half(0x7e00);
    const float sc = __half2float(sh);
    int q = 0;
    if (sc > 0.f) {
      float f = rintf(__fdiv_rn(x, sc));
      const float rem = 2.f * fmaf(-f, sc, x);
      if (fabsf(f) <= 16.f) f += rem > sc ? 1.f : (rem < -sc ? -1.f : 0.f);
      q = (int)fminf(fmaxf(f, -7.f), 7.f);
    }
    const unsigned u = (unsigned)(q + 8);
    const unsigned pair = u | (__shfl_down_sync(0xffffffffu, u, 1) << 4);
    const long long row = (((long long)b * a.S_cap + a.slot0 + s) * a.heads + h) * G + g;
    if ((lane & 1) == 0) a.codes[row * 16 + (lane >> 1)] = (uint8_t)pair;
    if (lane == 0) a.scales[row] = sh;
  }
}

template <class T>
__global__ void __launch_bounds__(256) mem4_unpack_kernel(const Mem4Unpack a) {
  const int G = mem4_groups(a.d);
  const long long total = (long long)a.B * a.S * a.heads * a.d;
  for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long long)gridDim.x * 256) {
    const int i = (int)(e % a.d);
    long long r = e / a.d;
    const int h = (int)(r % a.heads);
    r /= a.heads;
    const int s = (int)(r % a.S), b = (int)(r / a.S);
    const long long row = (((long long)b * a.S_cap + a.slot0 + s) * a.heads + h) * G + i / kMem4Group;
    const unsigned c = a.codes[row * 16 + (i % kMem4Group) / 2];
    const int q = (int)((i & 1) ? c >> 4 : c & 15) - 8;
    static_cast<T*>(a.out)[e] = from_f32<T>(__half2float(__float2half_rn((float)q * __half2float(a.scales[row]))));
  }
}

__device__ __forceinline__ float mem4_value(const Mem4Attend& a, long long row, int i) {
  const unsigned c = a.codes[(row + i / kMem4Group) * 16 + (i % kMem4Group) / 2];
  return __half2float(__float2half_rn((float)((int)((i & 1) ? c >> 4 : c & 15) - 8) * __half2float(a.scales[row + i / kMem4Group])));
}
// A CTA per column and head, a slot after the other.
template <class T>
__global__ void __launch_bounds__(256) mem4_attend_kernel(const Mem4Attend a) {
  __shared__ float red[8];
  const int c = blockIdx.x, h = blockIdx.y, b = c / a.cols, tid = threadIdx.x, G = mem4_groups(a.d);
  const T* q = static_cast<const T*>(a.q) + c * a.ld_q + (long long)h * a.d;
  T* out = static_cast<T*>(a.out) + c * a.ld_out + (long long)h * a.d;
  const long long off = a.offset ? a.offset[b] : 0;
  const int lo = (int)max(off, 0ll), hi = (int)min(off + a.len[b], (long long)a.S_cap);
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f}, qv[4];
  for (int u = 0; u < 4; ++u) qv[u] = tid + 256 * u < a.d ? to_f32(q[tid + 256 * u]) : 0.f;
  if (!a.mask || a.mask[c] != 0)
    for (int s = lo; s < hi; ++s) {
      const long long row = (((long long)b * a.S_cap + s) * a.heads + h) * G;
      float v[4], z = 0.f;
      for (int u = 0; u < 4; ++u) {
        v[u] = tid + 256 * u < a.d ? mem4_value(a, row, tid + 256 * u) : 0.f;
        z += qv[u] * v[u];
      }
      for (int o = 16; o; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
      __syncthreads();
      if ((tid & 31) == 0) red[tid >> 5] = z;
      __syncthreads();
      z = 0.f;
      for (int w = 0; w < 8; ++w) z += red[w];
      z *= a.scale;
      const float mn = fmaxf(m, z), al = m == -INFINITY ? 0.f : expf(m - mn), p = expf(z - mn);
      m = mn;
      l = l * al + p;
      for (int u = 0; u < 4; ++u) acc[u] = acc[u] * al + p * v[u];
    }
  for (int u = 0; u < 4; ++u)
    if (tid + 256 * u < a.d) out[tid + 256 * u] = from_f32<T>(l == 0.f ? 0.f : acc[u] / l);
}

}  // namespace

cudaError_t launch_mem4_pack(const Mem4Pack& a, int elem, cudaStream_t st) {
  const long long warps = (long long)a.S * a.B * a.heads * mem4_groups(a.d);
  if (warps == 0) return cudaSuccess;
  const unsigned grid = (unsigned)std::min<long long>((warps + 7) / 8, 1 << 20);
  count_launch();
  switch (elem) {
    case ELEM_F32: mem4_pack_kernel<float><<<grid, 256, 0, st>>>(a); break;
    case ELEM_BF16: mem4_pack_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a); break;
    default: mem4_pack_kernel<__half><<<grid, 256, 0, st>>>(a);
  }
  return cudaGetLastError();
}
cudaError_t launch_mem4_unpack(const Mem4Unpack& a, int elem, cudaStream_t st) {
  const long long total = (long long)a.B * a.S * a.heads * a.d;
  if (total == 0) return cudaSuccess;
  const unsigned grid = (unsigned)std::min<long long>((total + 255) / 256, 1 << 20);
  count_launch();
  switch (elem) {
    case ELEM_F32: mem4_unpack_kernel<float><<<grid, 256, 0, st>>>(a); break;
    case ELEM_BF16: mem4_unpack_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a); break;
    default: mem4_unpack_kernel<__half><<<grid, 256, 0, st>>>(a);
  }
  return cudaGetLastError();
}
size_t mem4_attend_work(int, int, int, int, int) { return 0; }
cudaError_t launch_mem4_attend(const Mem4Attend& a, int elem, cudaStream_t st) {
  if (a.B == 0 || a.cols == 0) return cudaSuccess;
  const dim3 grid((unsigned)(a.B * a.cols), (unsigned)a.heads);
  count_launch();
  switch (elem) {
    case ELEM_F32: mem4_attend_kernel<float><<<grid, 256, 0, st>>>(a); break;
    case ELEM_BF16: mem4_attend_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a); break;
    default: mem4_attend_kernel<__half><<<grid, 256, 0, st>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace zrnn
