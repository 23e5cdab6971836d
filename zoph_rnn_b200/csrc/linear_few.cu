// Y = act(W X + bias) + R for few columns or few outputs: the weights stream past the columns through registers, on the warp-level tensor cores.
//
// A CTA computes 16 outputs x up to 32 columns, its eight warps an eighth of the K axis each.  A lane reads 16 consecutive bytes of a weight row and of a
// column: which K indices it holds does not matter as long as both operands agree, so the fragments of a product are what the
// loads bring, without a pass through shared memory (m16n8k16 in 16 bits: 8 elements are two k-steps' halves; m16n8k8 in tf32: 4 elements
// are two k-steps).  32-bit operands are split into tf32 parts, both rounded, for three products; the sums of four chunks (two of
// more than 8 columns) are added in ordinary 32-bit arithmetic, since the tensor core cuts its sums off.  What bounds a call is the latency of a warp's loads, a dozen chunks one
// after the other; where there are few outputs and a long K axis, up to 8 CTAs of a cluster share it (245 x 7429 bf16, 3 columns, rows that
// start anywhere: 27 us on 16 CTAs, so 9).
#include <cooperative_groups.h>

#include <algorithm>
#include <cstring>
#include <type_traits>

#include "kernels.cuh"
#include "linear_device.cuh"
#include "operators.cuh"
#include "tc_gemm.cuh"

namespace zrnn {
namespace {

namespace cg = cooperative_groups;

template <class T> __device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
constexpr int kFewWarps = 8, kFewCut = 8;
template <class T, int NT, bool ALIGNED>
__global__ void __launch_bounds__(kFewWarps * 32) linear_few_kernel(const LinearArgs a) {
  constexpr int V = 16 / sizeof(T), CHUNK = 4 * V, AHEAD = NT == 1 ? 4 : 2;  // K elements of a chunk, chunks in flight
  constexpr bool F32 = sizeof(T) == 4;
  __shared__ float s_sum[kFewWarps][NT * 8][17];
  __shared__ float s_part[kFewCut - 1][16 * NT * 8];  // the first CTA's: sums of the other ones of its cluster
  cg::cluster_group cluster = cg::this_cluster();
  const int cut = cluster.num_blocks(), me = cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const long long i0 = (long long)(blockIdx.x / cut) * 16, c0 = (long long)blockIdx.y * (NT * 8);
  const bool in0 = i0 + g < a.n, in1 = i0 + g + 8 < a.n;
  const T* w0 = static_cast<const T*>(a.W) + (in0 ? i0 + g : 0) * a.ldw;
  const T* w1 = static_cast<const T*>(a.W) + (in1 ? i0 + g + 8 : 0) * a.ldw;
  const T* x[NT];
  bool xin[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    xin[j] = c0 + 8 * j + g < a.N;
    x[j] = static_cast<const T*>(a.X) + (xin[j] ? c0 + 8 * j + g : 0) * a.ldx;
  }
  if (cut > 1) cluster.barrier_arrive();  // (that all of them run is known by the time the sums are there)
  float acc[NT][4], part[NT][4], cross[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int u = 0; u < 4; ++u) acc[j][u] = part[j][u] = cross[j][u] = 0.f;
  const int chunks = (a.K + CHUNK - 1) / CHUNK, walkers = kFewWarps * cut, per = (chunks + walkers - 1) / walkers;
  const int q0 = min((me * kFewWarps + warp) * per, chunks), q1 = min(q0 + per, chunks);
  for (int q = q0; q < q1; q += AHEAD) {
    uint4 wa[AHEAD], wb[AHEAD], xv[AHEAD][NT];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int k = (q + u) * CHUNK + t * V, K = q + u < q1 ? a.K : 0;
      wa[u] = load16<T, ALIGNED>(w0, k, K, in0);
      wb[u] = load16<T, ALIGNED>(w1, k, K, in1);
#pragma unroll
      for (int j = 0; j < NT; ++j) xv[u][j] = load16<T, ALIGNED>(x[j], k, K, xin[j]);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if constexpr (!F32) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          mma16<T>(acc[j], wa[u].x, wb[u].x, wa[u].y, wb[u].y, xv[u][j].x, xv[u][j].y);
          mma16<T>(acc[j], wa[u].z, wb[u].z, wa[u].w, wb[u].w, xv[u][j].z, xv[u][j].w);
        }
      } else {
        uint32_t ah[4], al[4], bh[4], bl[4];
        split_tf32(wa[u].x, ah[0], al[0]); split_tf32(wa[u].y, ah[1], al[1]); split_tf32(wa[u].z, ah[2], al[2]); split_tf32(wa[u].w, ah[3], al[3]);
        split_tf32(wb[u].x, bh[0], bl[0]); split_tf32(wb[u].y, bh[1], bl[1]); split_tf32(wb[u].z, bh[2], bl[2]); split_tf32(wb[u].w, bh[3], bl[3]);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          uint32_t xh[4], xl[4];
          split_tf32(xv[u][j].x, xh[0], xl[0]); split_tf32(xv[u][j].y, xh[1], xl[1]); split_tf32(xv[u][j].z, xh[2], xl[2]); split_tf32(xv[u][j].w, xh[3], xl[3]);
#pragma unroll
          for (int s = 0; s < 4; s += 2) {
            mma8(part[j], ah[s], bh[s], ah[s + 1], bh[s + 1], xh[s], xh[s + 1]);
            mma8(cross[j], al[s], bl[s], al[s + 1], bl[s + 1], xh[s], xh[s + 1]);
            mma8(cross[j], ah[s], bh[s], ah[s + 1], bh[s + 1], xl[s], xl[s + 1]);
          }
        }
      }
    }
    if constexpr (F32) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          acc[j][u] += part[j][u];
          part[j][u] = 0.f;
        }
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int u = 0; u < 4; ++u) s_sum[warp][8 * j + 2 * t + (u & 1)][g + 8 * (u >> 1)] = F32 ? acc[j][u] + cross[j][u] : acc[j][u];
  __syncthreads();
  if (cut > 1) {
    cluster.barrier_wait();
    if (me != 0)
      for (int o = tid; o < 16 * NT * 8; o += kFewWarps * 32) {
        float y = 0.f;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) y += s_sum[w][o >> 4][o & 15];
        *cluster.map_shared_rank(&s_part[me - 1][o], 0) = y;
      }
    cluster.sync();
    if (me != 0) return;
  }
  for (int o = tid; o < 16 * NT * 8; o += kFewWarps * 32) {
    const int r = o & 15, c = o >> 4;
    if (i0 + r >= a.n || c0 + c >= a.N) continue;
    float y = 0.f;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) y += s_sum[w][c][r];
    for (int k = 1; k < cut; ++k) y += s_part[k - 1][o];
    y = linear_act(y + (a.bias ? __ldg(a.bias + i0 + r) : 0.f), a.act);
    if (a.R) y += to_f32(static_cast<const T*>(a.R)[(c0 + c) * a.ldr + i0 + r]);
    static_cast<T*>(a.Y)[(c0 + c) * a.ldy + i0 + r] = from_f32<T>(y);
  }
}

template <class T, int NT>
cudaError_t few_launch(const LinearArgs& all, cudaStream_t st) {
  const auto on16 = [](const void* p, long long ld) { return ((uintptr_t)p & 15) == 0 && (ld * sizeof(T)) % 16 == 0; };
  const bool aligned = all.K % (16 / sizeof(T)) == 0 && on16(all.W, all.ldw) && on16(all.X, all.ldx);
  constexpr long long kMost = 65535ll * NT * 8;  // columns of a launch
  for (long long at = 0; at < all.N; at += kMost) {
    LinearArgs a = all;
    a.N = (int)std::min<long long>(kMost, all.N - at);
    a.X = static_cast<const T*>(a.X) + at * a.ldx;
    a.Y = static_cast<T*>(a.Y) + at * a.ldy;
    if (a.R) a.R = static_cast<const T*>(a.R) + at * a.ldr;
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof(cfg));
    const int cut = few_cut(a.n, a.N, a.K, (int)sizeof(T));
    cfg.gridDim = dim3((a.n + 15) / 16 * cut, (a.N + NT * 8 - 1) / (NT * 8));
    cfg.blockDim = dim3(kFewWarps * 32);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cut;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cut > 1 ? 1 : 0;
    count_launch();
    const cudaError_t e = aligned ? cudaLaunchKernelEx(&cfg, linear_few_kernel<T, NT, true>, a) : cudaLaunchKernelEx(&cfg, linear_few_kernel<T, NT, false>, a);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}
template <class T>
cudaError_t few_type(const LinearArgs& a, cudaStream_t st) {
  return a.N <= 8 ? few_launch<T, 1>(a, st) : a.N <= 16 ? few_launch<T, 2>(a, st) : few_launch<T, 4>(a, st);
}

}  // namespace

// CTAs that share the K axis of 16 outputs: while all of them are resident twice over and a warp keeps four chunks
int few_cut(int n, int N, int K, int eb) {
  const int cols = N <= 8 ? 8 : N <= 16 ? 16 : 32;
  const long long ctas = (long long)((n + 15) / 16) * ((N + cols - 1) / cols), chunks = ((long long)K * eb + 63) / 64;
  int cut = 1;
  while (cut < kFewCut && ctas * cut * 2 <= 2 * device_sms() && chunks / (kFewWarps * cut * 2) >= 4) cut *= 2;
  return cut;
}
cudaError_t launch_linear_few(const LinearArgs& a, int elem, cudaStream_t st) {
  switch (elem) {
    case ELEM_F32: return few_type<float>(a, st);
    case ELEM_BF16: return few_type<__nv_bfloat16>(a, st);
  }
  return few_type<__half>(a, st);
}

}  // namespace zrnn
