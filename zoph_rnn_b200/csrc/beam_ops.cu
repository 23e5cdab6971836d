// Selection over beams and vocabulary, and the reorder of the states that goes with it.
#include <algorithm>
#include <cstring>

#include "kernels.cuh"
#include "operators.cuh"

namespace zrnn {
namespace {

// A candidate as one whole number: its value in an order-preserving form, then the complement of its index j * V + v, so that the larger number is
// the larger value or, of equal ones, the lower index.  Numbers of different candidates differ.
__device__ __forceinline__ unsigned ordered(float x) {
  const unsigned u = __float_as_uint(x + 0.0f);  // (-0 equals 0)
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(unsigned u) { return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u); }
constexpr unsigned kOrderedMinusInf = 0x007fffffu;
__device__ __forceinline__ unsigned long long candidate_key(float value, unsigned index) {
  return ((unsigned long long)ordered(value) << 32) | (unsigned)~index;
}
// value of word v for hypothesis row r: the two roundings that the definition has
template <class T>
__device__ __forceinline__ float candidate(const BeamSelect& a, long long r, int v) {
  float z;
  if (a.done && a.done[r]) {
    z = v == a.eos ? a.scores[r] : -INFINITY;
  } else {
    z = to_f32(static_cast<const T*>(a.logp)[r * a.ld + v]);
    if (a.lse) z = __fsub_rn(z, a.lse[r]);
    z = __fadd_rn(a.scores[r], z);
  }
  return z != z ? -INFINITY : z;
}

// k passes over a sentence's candidates, each for the best one below the last
template <class T>
__global__ void __launch_bounds__(256) beam_select_simple_kernel(const BeamSelect a) {
  __shared__ unsigned long long red[8];
  const int b = blockIdx.x, tid = threadIdx.x;
  unsigned long long last = ~0ull;
  for (int k = 0; k < a.k; ++k) {
    unsigned long long best = 0;
    for (int j = 0; j < a.beam; ++j)
      for (int v = tid; v < a.V; v += 256) {
        const unsigned long long key = candidate_key(candidate<T>(a, (long long)b * a.beam + j, v), (unsigned)j * a.V + v);
        if (key < last && key > best) best = key;
      }
    for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if ((tid & 31) == 0) red[tid >> 5] = best;
    __syncthreads();
    best = red[0];
    for (int w = 1; w < 8; ++w) best = max(best, red[w]);
    __syncthreads();
    if (tid == 0) {
      const bool some = (unsigned)(best >> 32) > kOrderedMinusInf;
      const unsigned at = ~(unsigned)best;
      const long long o = (long long)b * a.k + k;
      a.score_out[o] = some ? unordered((unsigned)(best >> 32)) : -INFINITY;
      a.word_out[o] = some ? (int)(at % a.V) : -1;
      a.parent_out[o] = some ? (int)(at / a.V) + b * a.beam : -1;
    }
    last = best;
  }
}

// A thread takes one piece of U bytes of the columns of one group (out of place: of one column), all loaded before the first is stored.
template <class U>
__global__ void __launch_bounds__(128) beam_reorder_kernel(const __grid_constant__ BeamReorder a) {
  const int arr = blockIdx.z, first = blockIdx.y * a.group, n = min(a.group, a.n_cols - first);
  const long long pieces = a.bytes[arr] / (long long)sizeof(U), i = (long long)blockIdx.x * 128 + threadIdx.x;
  if (i >= pieces) return;
  const U* src = reinterpret_cast<const U*>(a.src[arr]) + i;
  U* dst = reinterpret_cast<U*>(a.dst[arr]) + i;
  const bool in_place = a.src[arr] == a.dst[arr];
  U v[kReorderGroup];
  for (int c = 0; c < n; ++c) {
    const int p = a.parent[first + c];
    const bool out = in_place ? p >= first + n || (p >= 0 && p < first) : p >= a.n_src_cols;
    if (out) {
      if (a.err) atomicExch(a.err, kErrBadParent);
      if (in_place) v[c] = src[(first + c) * pieces];
      else memset(&v[c], 0, sizeof(U));
    } else if (p < 0) memset(&v[c], 0, sizeof(U));
    else v[c] = src[p * pieces];
  }
  for (int c = 0; c < n; ++c) dst[(first + c) * pieces] = v[c];
}

}  // namespace

size_t beam_select_work(int, int, int, int, int) { return 0; }
cudaError_t launch_beam_select(const BeamSelect& a, int elem, cudaStream_t st) {
  if (a.n_sent == 0) return cudaSuccess;
  count_launch();
  switch (elem) {
    case ELEM_F32: beam_select_simple_kernel<float><<<a.n_sent, 256, 0, st>>>(a); break;
    case ELEM_BF16: beam_select_simple_kernel<__nv_bfloat16><<<a.n_sent, 256, 0, st>>>(a); break;
    default: beam_select_simple_kernel<__half><<<a.n_sent, 256, 0, st>>>(a);
  }
  return cudaGetLastError();
}
cudaError_t launch_beam_reorder(const BeamReorder& a, cudaStream_t st) {
  if (a.n_cols == 0 || a.n_arrays == 0) return cudaSuccess;
  uintptr_t bits = 0;
  long long most = 0;
  for (int i = 0; i < a.n_arrays; ++i) {
    bits |= (uintptr_t)a.src[i] | (uintptr_t)a.dst[i] | (uintptr_t)a.bytes[i];
    most = std::max(most, a.bytes[i]);
  }
  if (most == 0) return cudaSuccess;
  const int unit = bits & 1 ? 1 : bits & 2 ? 2 : bits & 4 ? 4 : bits & 8 ? 8 : 16;
  const dim3 grid((unsigned)((most / unit + 127) / 128), (a.n_cols + a.group - 1) / a.group, a.n_arrays);
  count_launch();
  switch (unit) {
    case 16: beam_reorder_kernel<uint4><<<grid, 128, 0, st>>>(a); break;
    case 8: beam_reorder_kernel<uint2><<<grid, 128, 0, st>>>(a); break;
    case 4: beam_reorder_kernel<unsigned><<<grid, 128, 0, st>>>(a); break;
    case 2: beam_reorder_kernel<unsigned short><<<grid, 128, 0, st>>>(a); break;
    default: beam_reorder_kernel<unsigned char><<<grid, 128, 0, st>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace zrnn
