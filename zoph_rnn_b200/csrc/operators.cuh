// Launch interfaces of the operators of a decoding step that a host program calls beside the layer objects: the source memory held in 4
// bits (memory4.cu), the product with bias, activation and residual (linear.cu), the selection over beams and vocabulary and the
// reorder of the states (beam_ops.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace zrnn {

enum { ELEM_F32 = 0, ELEM_BF16 = 1, ELEM_F16 = 2 };
inline int elem_bytes(int elem) { return elem == ELEM_F32 ? 4 : 2; }

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <class T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// ---- source memory in 4 bits: vectors of `heads` x d elements per (column, slot).  A head's elements come in groups of 32 (the last one
// filled with zeros): code u = q + 8 with q in -7 .. 7, two per byte, the even element in the low bits, and one half-precision scale
// s per group; the element's value is q * s rounded to half precision.
constexpr int kMem4Group = 32;
inline __host__ __device__ int mem4_groups(int d) { return (d + kMem4Group - 1) / kMem4Group; }
struct Mem4Pack {
  const void* x;               // element i of column b, slot s at x + s * ld_slot + b * ld_col + i
  long long ld_slot, ld_col;
  int S, B, heads, d;
  int slot0, S_cap;            // slots slot0 .. slot0 + S - 1 of S_cap are written
  uint8_t* codes;              // [B][S_cap][heads][groups * 16]
  __half* scales;              // [B][S_cap][heads][groups]
};
cudaError_t launch_mem4_pack(const Mem4Pack& a, int elem, cudaStream_t st);
struct Mem4Unpack {
  const uint8_t* codes;
  const __half* scales;
  int B, S_cap, heads, d, slot0, S;
  void* out;                   // [B][S][heads][d]
};
cudaError_t launch_mem4_unpack(const Mem4Unpack& a, int elem, cudaStream_t st);
struct Mem4Attend {
  const uint8_t* codes;
  const __half* scales;
  int B, S_cap, heads, d;
  const int *len, *offset;     // per sentence; offset may be null (0)
  const void* q;               // column c at q + c * ld_q, B * cols columns; sentence c / cols
  long long ld_q;
  int cols;
  const int* mask;             // per column, may be null; 0: the column's output is zero
  float scale;
  void* out;
  long long ld_out;
  float* work;                 // mem4_attend_work(...) floats
};
constexpr int kMem4MaxHead = 1024;
size_t mem4_attend_work(int B, int cols, int S_cap, int heads, int d);
cudaError_t launch_mem4_attend(const Mem4Attend& a, int elem, cudaStream_t st);

// ---- Y = act(W X + bias) + R
enum { ACT_NONE = 0, ACT_TANH = 1, ACT_SIGMOID = 2, ACT_RELU = 3, ACT_GELU = 4, ACT_SILU = 5 };
struct LinearArgs {
  int n, N, K;                 // outputs, columns, inputs
  const void* W;               // output i's K weights at W + i * ldw
  const void* X;               // column c at X + c * ldx
  long long ldw, ldx;
  const float* bias;           // n, may be null
  const void* R;               // column c at R + c * ldr, may be null, may be Y
  long long ldr;
  void* Y;
  long long ldy;
  int act;
  void* work;
  int* err;                    // device error word
};
size_t linear_work(const LinearArgs& a, int elem);
cudaError_t launch_linear(const LinearArgs& a, int elem, cudaStream_t st);
cudaError_t launch_linear_few(const LinearArgs& a, int elem, cudaStream_t st);  // few columns (linear_few.cu)
int few_cut(int n, int N, int K, int eb);  // ... and how many CTAs share the K axis there

// ---- selection over beams and vocabulary
constexpr int kSelectMax = 64;  // survivors of a sentence
struct BeamSelect {
  const void* logp;            // row r = sentence * beam + j at logp + r * ld
  long long ld;
  const float *lse, *scores;   // per row; lse may be null
  const int* done;             // per row, may be null
  int n_sent, beam, V, k, eos;
  float* score_out;            // [n_sent][k]
  int *word_out, *parent_out;
  unsigned long long* work;    // beam_select_work(...) bytes
  int first_row;               // what is added to the rows in parent_out
};
size_t beam_select_work(int elem, int n_sent, int beam, int V, int k);
cudaError_t launch_beam_select(const BeamSelect& a, int elem, cudaStream_t st);

// ---- dst[:, c] = src[:, parent[c]] for several arrays of columns
struct BeamReorder {
  enum { MAX_ARRAYS = 40 };
  const char* src[MAX_ARRAYS];
  char* dst[MAX_ARRAYS];
  long long bytes[MAX_ARRAYS];  // per column
  int n_arrays;
  const int* parent;           // n_cols; negative: the column becomes zero
  int n_cols, n_src_cols;
  int group;                   // in place (dst == src): columns move within groups of this many
  int* err;
};
constexpr int kReorderGroup = 64;
constexpr int kErrBadParent = 101;
cudaError_t launch_beam_reorder(const BeamReorder& a, cudaStream_t st);

}  // namespace zrnn
