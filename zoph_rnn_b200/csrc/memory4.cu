// The source memory in 4 bits: packing, reading back, and attention over it.
#include <algorithm>
#include <cstring>
#include <type_traits>

#include "kernels.cuh"
#include "operators.cuh"
#include "tc_gemm.cuh"

namespace zrnn {
namespace {

constexpr float kSeventh = 0.14285714924335479736328125f;  // 1/7 rounded to 32 bits
constexpr float kMaxScale = 9352.0f;                       // the largest half that times 7 is finite

// The scale is fp16(a / 7) of the group's largest magnitude a (a product with 1/7 in 32 bits).
__device__ __forceinline__ __half mem4_scale(float a) {
  return a < INFINITY ? __float2half_rn(fminf(a * kSeventh, kMaxScale)) : __ushort_as_half(0x7e00);
}
// Eight codes: the integer nearest to x / s, ties to even, plus 8.  x times an approximate reciprocal, improved by the remainder, is the quotient
// rounded to 32 bits: exact where x / s is half of an odd number v (16-bit states meet these often), and not v where it is not, for x
// and v s differ by no less than x's last place, 2^-23 / m(v s) of it with m the mantissa, and half a place of v is 2^-24 / m(v).  An addition
// of 1.5 * 2^23 then rounds it to a whole number, whose low bits go into the word as they are.
// two 32-bit operations in one instruction
__device__ __forceinline__ unsigned long long pair_of(float x, float y) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void of_pair(unsigned long long p, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p)); }
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float max_abs_nan(float x, float y, float z) {  // the largest magnitude; NaN if one of them is
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}
// most: the group's largest magnitude
__device__ __forceinline__ unsigned mem4_codes(const float (&x)[8], float s, float most) {
  float inv;  // (s is no less than 2^-24)
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  const unsigned long long inv2 = pair_of(inv, inv), minus_s = pair_of(-s, -s), zero = pair_of(0.f, 0.f), one = pair_of(1.f, 1.f), whole = pair_of(12582920.f, 12582920.f);
  float t[8];
#pragma unroll
  for (int u = 0; u < 8; u += 2) {
    const unsigned long long xs = pair_of(x[u], x[u + 1]), near = fma2(xs, inv2, zero);
    of_pair(fma2(fma2(near, minus_s, xs), inv2, near), t[u], t[u + 1]);
  }
  if (most * inv > 7.25f) {  // s was rounded far down, or saturated
#pragma unroll
    for (int u = 0; u < 8; ++u) t[u] = fminf(fmaxf(t[u], -7.f), 7.f);
  }
  unsigned w[8];
#pragma unroll
  for (int u = 0; u < 8; u += 2) {
    float r0, r1;
    of_pair(fma2(pair_of(t[u], t[u + 1]), one, whole), r0, r1);
    w[u] = __float_as_uint(r0);
    w[u + 1] = __float_as_uint(r1);
  }
  return __byte_perm(w[0] + w[1] * 16 + w[2] * 256 + w[3] * 4096, w[4] + w[5] * 16 + w[6] * 256 + w[7] * 4096, 0x5410);
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
// Nibbles 0 .. 3 of each half of x, as pairs (low half, high half) of q * s: 1024 + u and 1024 + 16 u are halves made by or-ing u into a
// mantissa (a well-known way to make numbers of small whole ones), and what follows is exact but for the last product, whose rounding is the definition's.
__device__ __forceinline__ void dequant4(uint32_t x, __half2 s, uint32_t (&v)[4]) {
  const __half2 m1032 = __half2half2(__ushort_as_half(0xe408)), sixteenth = __half2half2(__ushort_as_half(0x2c00)), m72 = __half2half2(__ushort_as_half(0xd480));
  const uint32_t y = x >> 8;
  uint32_t a, b, c, d;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(a) : "r"(x));
  asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(b) : "r"(x));
  asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(c) : "r"(y));
  asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(d) : "r"(y));
  v[0] = h2_bits(__hmul2_rn(__hadd2_rn(bits_h2(a), m1032), s));
  v[1] = h2_bits(__hmul2_rn(__hfma2(bits_h2(b), sixteenth, m72), s));
  v[2] = h2_bits(__hmul2_rn(__hadd2_rn(bits_h2(c), m1032), s));
  v[3] = h2_bits(__hmul2_rn(__hfma2(bits_h2(d), sixteenth, m72), s));
}
template <class T> struct Mem4Vec;  // 8 elements
template <> struct Mem4Vec<float> {
  float4 a, b;
  __device__ void clear() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ void load(const float* p) {
    a = __ldg(reinterpret_cast<const float4*>(p));
    b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  }
  __device__ void get(float (&x)[8]) const { x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w; }
  static __device__ void store(float* p, const float (&x)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  }
};
template <class T> struct Mem4Vec {
  uint4 a;
  __device__ void clear() { a = make_uint4(0u, 0u, 0u, 0u); }
  __device__ void load(const T* p) { a = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ void get(float (&x)[8]) const {
    const unsigned w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        x[2 * i] = __half2float(__ushort_as_half((unsigned short)w[i]));
        x[2 * i + 1] = __half2float(__ushort_as_half((unsigned short)(w[i] >> 16)));
      } else {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
  static __device__ void store(T* p, const float (&x)[8]) {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T a = from_f32<T>(x[2 * i]), b = from_f32<T>(x[2 * i + 1]);
      w[i] = (unsigned)*reinterpret_cast<const unsigned short*>(&a) | (unsigned)*reinterpret_cast<const unsigned short*>(&b) << 16;
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// A lane takes 8 elements, four lanes a group, a team of lanes one source column, whose slots it walks through: all indices are computed once
// per thread (divided per vector, they were two thirds of the instructions).  ALIGNED: vectors lie on 16 bytes and a head is a
// multiple of 8 elements; else a warp's eight groups, all of one vector, go through shared memory, 32 consecutive elements at a time.
constexpr int kMem4PerSm = 6;       // CTAs resident on a multiprocessor
constexpr int kMem4Stage = 8 * 36;  // floats of a warp's groups, four more per group: runs of 8 fall on different banks
template <class T, bool ALIGNED>
__global__ void __launch_bounds__(256, kMem4PerSm) mem4_pack_kernel(const Mem4Pack a, int team) {
  __shared__ __align__(16) float s_stage[ALIGNED ? 1 : 8 * kMem4Stage];
  const int G = mem4_groups(a.d), lane = threadIdx.x % team, sub = threadIdx.x / team, q = blockIdx.z * team + lane, quads = a.heads * G * 4;
  const long long b = (long long)blockIdx.x * (256 / team) + sub;
  const bool mine = q < quads;
  if (sub >= 256 / team || b >= a.B || (ALIGNED && !mine)) return;  // (whole groups of four leave; unaligned: whole warps)
  const int g = q >> 2, h = g / G, i = (q - h * G * 4) * 8;
  const T* row_x = static_cast<const T*>(a.x) + b * a.ld_col + blockIdx.y * a.ld_slot;
  const long long row = (long long)a.heads * G, to = (b * a.S_cap + a.slot0 + blockIdx.y) * row + g;
  unsigned* codes = reinterpret_cast<unsigned*>(a.codes) + to * 4 + (q & 3);
  __half* scales = a.scales + to;
  const unsigned four = 0xfu << (threadIdx.x & 28);
  const long long x_step = gridDim.y * a.ld_slot, step = gridDim.y * row;
  float* stage = s_stage + (ALIGNED ? 0 : (threadIdx.x >> 5) * kMem4Stage);
  const int l32 = threadIdx.x & 31, g0 = (blockIdx.z * team + (lane & ~31)) >> 2;  // the warp's first group
  Mem4Vec<T> next;  // the slot after this one
  next.clear();
  if (ALIGNED) row_x += (long long)h * a.d + i;
  if (ALIGNED && i < a.d && blockIdx.y < a.S) next.load(row_x);
#pragma unroll 2
  for (int s = blockIdx.y; s < a.S; s += gridDim.y, row_x += x_step, codes += step * 4, scales += step) {
    float v[8];
    if (ALIGNED) {
      next.get(v);
      if (i < a.d && s + (int)gridDim.y < a.S) next.load(row_x + x_step);
    } else {
      float x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int gu = g0 + u, hu = a.heads == 1 ? 0 : gu / G, e = (gu - hu * G) * 32 + l32;
        x[u] = hu < a.heads && e < a.d ? to_f32(__ldg(row_x + (long long)hu * a.d + e)) : 0.f;
      }
      __syncwarp();
#pragma unroll
      for (int u = 0; u < 8; ++u) stage[u * 36 + l32] = x[u];
      __syncwarp();
      const float4 lo = *reinterpret_cast<const float4*>(stage + (l32 >> 2) * 36 + (l32 & 3) * 8), hi = *reinterpret_cast<const float4*>(stage + (l32 >> 2) * 36 + (l32 & 3) * 8 + 4);
      v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w; v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
    }
    float m = max_abs_nan(v[0], v[1], v[2]);
    m = max_abs_nan(m, v[3], v[4]);
    m = max_abs_nan(m, v[5], v[6]);
    m = max_abs_nan(m, v[7], __shfl_xor_sync(four, max_abs_nan(m, v[7], 0.f), 1));
    m = max_abs_nan(m, __shfl_xor_sync(four, m, 2), 0.f);
    const __half sh = mem4_scale(m);
    const float sc = __half2float(sh);
    const unsigned w = sc > 0.f ? mem4_codes(v, sc, m) : 0x88888888u;
    if (ALIGNED || mine) {
      *codes = w;
      if ((q & 3) == 0) *scales = sh;
    }
  }
}
// In 32 bits two lanes share two words, each the same half of both, so that what a store writes are whole sectors (a word's 32 bytes by one lane:
// 16 x 8192 vectors of 1024 in 153 us, so 99).
template <class T, bool ALIGNED>
__global__ void __launch_bounds__(256, kMem4PerSm) mem4_unpack_kernel(const Mem4Unpack a, int team) {
  constexpr bool HALVES = ALIGNED && sizeof(T) == 4;
  __shared__ __align__(16) float s_stage[ALIGNED ? 1 : 8 * kMem4Stage];
  const int G = mem4_groups(a.d), lane = threadIdx.x % team, sub = threadIdx.x / team, q = blockIdx.z * team + lane, quads = a.heads * G * 4;
  const long long b = (long long)blockIdx.x * (256 / team) + sub;
  const bool mine = q < quads;
  const int g = q >> 2, h = g / G, i = ((HALVES ? q & ~1 : q) - h * G * 4) * 8;
  if (sub >= 256 / team || b >= a.B || (ALIGNED && (!mine || i >= a.d))) return;
  const long long row = (long long)a.heads * G, from = (b * a.S_cap + a.slot0 + blockIdx.y) * row + g, width = (long long)a.heads * a.d;
  const unsigned* codes = reinterpret_cast<const unsigned*>(a.codes) + from * 4 + (q & 3);
  const __half* scales = a.scales + from;
  T* row_out = static_cast<T*>(a.out) + (b * a.S + blockIdx.y) * width;
  const long long step = gridDim.y * row;
  float* stage = s_stage + (ALIGNED ? 0 : (threadIdx.x >> 5) * kMem4Stage);
  const int l32 = threadIdx.x & 31, g0 = (blockIdx.z * team + (lane & ~31)) >> 2;
  uint2 next[2];  // the words of this slot and the next one; .y: HALVES
  __half next_scale[2];
  auto request = [&](int k, int s, const unsigned* from, const __half* from_scale) {
    next[k] = make_uint2(0u, 0u);
    next_scale[k] = __ushort_as_half(0);
    if (s >= a.S || !mine) return;
    if (HALVES) next[k] = __ldg(reinterpret_cast<const uint2*>(from - (q & 1)));
    else next[k].x = __ldg(from);
    next_scale[k] = __ldg(from_scale);
  };
  request(0, blockIdx.y, codes, scales);
  request(1, blockIdx.y + gridDim.y, codes + step * 4, scales + step);
#pragma unroll 2
  for (int s = blockIdx.y; s < a.S; s += gridDim.y, codes += step * 4, scales += step, row_out += gridDim.y * width) {
    const uint2 w = next[0];
    const __half2 sc = __half2half2(next_scale[0]);
    next[0] = next[1];
    next_scale[0] = next_scale[1];
    request(1, s + 2 * gridDim.y, codes + step * 8, scales + step * 2);
    uint32_t p[4];  // (elements 0, 4), (1, 5), (2, 6), (3, 7)
    dequant4(HALVES ? __byte_perm(w.x, w.y, q & 1 ? 0x7632 : 0x5410) : w.x, sc, p);
    float v[8];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float2 f = __half22float2(bits_h2(p[u]));
      v[u] = f.x;
      v[u + 4] = f.y;
    }
    if constexpr (HALVES) {
      float4* at = reinterpret_cast<float4*>(row_out + (long long)h * a.d + i) + (q & 1);
      at[0] = make_float4(v[0], v[1], v[2], v[3]);
      if (i + 8 < a.d) at[2] = make_float4(v[4], v[5], v[6], v[7]);
    } else if constexpr (ALIGNED) {
      Mem4Vec<T>::store(row_out + (long long)h * a.d + i, v);
    } else {
      __syncwarp();
      float4* at = reinterpret_cast<float4*>(stage + (l32 >> 2) * 36 + (l32 & 3) * 8);
      at[0] = make_float4(v[0], v[1], v[2], v[3]);
      at[1] = make_float4(v[4], v[5], v[6], v[7]);
      __syncwarp();
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int gu = g0 + u, hu = a.heads == 1 ? 0 : gu / G, e = (gu - hu * G) * 32 + l32;
        if (hu < a.heads && e < a.d) row_out[(long long)hu * a.d + e] = from_f32<T>(stage[u * 36 + l32]);
      }
    }
  }
}

// ---- attention
// Per source column b, head and tile of 16 target columns: z = Q V^T and softmax(z) V over the slots, in one pass with a running maximum and
// sum, on the warp-level tensor cores (m16n8k16, half precision in, 32 bits out).  The values q * s are half-precision numbers by
// definition, so they enter a product exactly; in 32 bits Q and the weights are split into a half and a rest (times 2^11) that is another half.
//
// A warp owns NB blocks of 64 elements of the head for the scores and for the output, so that both read the same codes; a team of WT warps
// covers the head and takes tiles of 32 slots, and a CTA has 16 / WT teams, each with slots of its own.  Per tile: the warps'
// partial scores meet in shared memory, each warp finishes 16 / WT rows (a lane per slot: maximum, exponential, weights written as the
// fragments of the second product), and all warps add weights x values to their registers.  Codes come three tiles ahead by
// asynchronous copies.  A warp that has a head to itself (up to 128 elements) keeps scores and weights in registers: they lie there as
// the second product wants them.
//
// Who takes what: ALONE, many short heads: every warp has a column tile and head of its own and all of its slots (481 x 16 heads of 32, one slot: 29 us,
// with a CTA each 200).  WHOLE: a CTA has a source column.  DEALT: where there are fewer of those than multiprocessors, several CTAs, more for
// longer ones, and a second launch that combines them.
//
// What bounds it is the issue of instructions, not memory (16 x 12 columns, 4000 .. 8192 slots of 1024 in bf16: 53 us, 1.1 TB/s; 40 of them the
// slots', the rest the start, the teams' and the parts' sums and the combination).  Per 64 slots x 1024 elements a quarter of a
// multiprocessor has 264 tensor instructions of 8 cycles, 1024 half-precision and some 1300 integer ones of 2 each (a word of 8 codes takes 13
// instructions to become 4 pairs of halves, twice: the scores need pairs of elements, the output pairs of slots; kept between the two, they
// would take 64 registers more), in all some 4000, and takes 5500 cycles: four warps do not fill the rest.
constexpr int kAttWarps = 16, kAttTile = 32, kAttStages = 3, kAttPartLd = 40;
enum { ALONE, WHOLE, DEALT };  // a warp per column tile and head; a CTA; several CTAs
// In 32 bits the weights are a half and 2^11 times the rest as another, in fp16 a half and the rest as it is (the result's 2^-12 would show the half
// alone; 32 x 5 columns, 8 heads of 64, up to 1500 slots: 18.2 us, without the rests 16.0), in bf16 a half, whose 2^-12 is an eighth of the
// result's 2^-9.
template <class T> struct AttParts { static constexpr int Q = 1, W = 1; };
template <> struct AttParts<float> { static constexpr int Q = 2, W = 2; };
template <> struct AttParts<__half> { static constexpr int Q = 1, W = 2; };
template <int PARTS, int W_PARTS, int WT, int NB, bool SOLO>
struct AttShape {
  static constexpr int WARPS = SOLO ? 8 : kAttWarps, TEAMS = WARPS / WT, GP = 2 * NB * WT;  // groups that the team's warps have room for
  static constexpr int ROW = (GP | 1) * 16;                       // bytes of a slot's codes in shared memory: an odd number of 16 spreads them over the banks
  static constexpr int Q = GP * 2 * PARTS * 512;                  // Q as fragments
  static constexpr int STAGE = kAttTile * ROW + GP * kAttTile * 2;
  static constexpr int PART = WT == 1 ? 0 : WT * 16 * kAttPartLd * 4, W = WT == 1 ? 0 : 2 * W_PARTS * 512;  // partial scores, weights: a warp alone keeps them
  static constexpr int TEAM = kAttStages * STAGE + PART + W + 192 + (SOLO ? Q : 0);
  static constexpr int OUT_LD = GP * 32 + 2;                      // floats; the teams' outputs take the place of all that
  static constexpr int RUN = (SOLO ? 0 : Q) + TEAMS * TEAM, OUT = SOLO ? 0 : TEAMS * 16 * OUT_LD * 4;
  static constexpr int ML = (RUN > OUT ? RUN : OUT), SMEM = ML + (SOLO ? 0 : 2 * 16 * 16 * 4);
  static_assert(SMEM <= 227 * 1024 && STAGE % 16 == 0 && TEAM % 16 == 0, "");
};
struct AttPlan {
  int G, warps, blocks;       // groups of a head; WT and NB
  int q_tiles;
  int parts;                  // > 0: CTAs (per column tile and head) that share the source columns; their sums are combined by a second launch
  bool solo;
};

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {  // onto zeros
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ float exp2_approx(float x) {  // within 2 units of the last place
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
// What a row's weights are relative to: a maximum that is followed only once it has risen by 2^8, so that sums are seldom rescaled.  The weights are
// 2^7 times what they are relative to that: of up to 2^15 they use all of half precision, whose steps of 2^-24 are 2^-31 of the reference.
__device__ __forceinline__ float risen(float before, float now) { return now > before + 8.f ? now : before; }
__device__ __forceinline__ float weight(float z, float ref) { return exp2_approx(z - ref + 7.f); }
// x as a half and, times `up`, what that leaves
__device__ __forceinline__ void split_half(float x, float up, __half& hi, __half& lo) {
  hi = __float2half_rn(x);
  lo = __float2half_rn((x - __half2float(hi)) * up);
}
__device__ __forceinline__ uint32_t shared_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared_at(dst)), "l"(src) : "memory");
}

// Tiles t0 .. t1 - 1 of source column b (t1 < 0: all of them) for the columns from c0 on and head h.  w: where the sums go, if the column has others
template <class T, int WT, int NB, bool SOLO>
__device__ __forceinline__ void attend_part(const Mem4Attend& a, const AttPlan& pl, unsigned char* smem, int b, int c0, int h, int t0, int t1, float* w) {
  constexpr int PARTS = AttParts<T>::Q, W_PARTS = AttParts<T>::W, ROWS = 16 / WT;
  constexpr float W_UP = PARTS == 2 ? 2048.f : 1.f;
  using Sh = AttShape<PARTS, W_PARTS, WT, NB, SOLO>;
  static_assert(!SOLO || WT == 1, "");
  constexpr int TEAMS = Sh::TEAMS, GP = Sh::GP, ROW = Sh::ROW;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, team = warp / WT, wt = warp % WT;
  const int g = lane >> 2, t = lane & 3, G = pl.G;
  const int n_cols = min(16, a.cols - c0);
  unsigned char* s_team = smem + (SOLO ? 0 : Sh::Q) + team * Sh::TEAM;
  unsigned char* s_q = SOLO ? s_team + Sh::TEAM - Sh::Q : smem;
  float* s_part = reinterpret_cast<float*>(s_team + kAttStages * Sh::STAGE);
  unsigned char* s_w = s_team + kAttStages * Sh::STAGE + Sh::PART;
  float* s_alpha = reinterpret_cast<float*>(s_w + Sh::W);
  float* s_m = s_alpha + 16;  // running maxima
  float* s_fac = s_m + 16;    // factors of the queries
  float* s_ml = reinterpret_cast<float*>(smem + Sh::ML);  // [team][16]: maxima, sums

  // Q, a row per warp (of a team on its own, one row after the other), a row's elements requested at once
  auto fetch_row = [&](int r, float (&x)[GP]) {
    const bool in = r < n_cols;
    const T* q = static_cast<const T*>(a.q) + ((long long)b * a.cols + c0 + (in ? r : 0)) * a.ld_q + (long long)h * a.d + lane;
#pragma unroll
    for (int k = 0; k < GP; ++k) x[k] = in && k * 32 + lane < a.d ? to_f32(__ldg(q + k * 32)) : 0.f;
  };
  const bool in = SOLO || warp < n_cols;
  constexpr int ROWS_AT_ONCE = SOLO ? 4 : 1;
  float qx[ROWS_AT_ONCE][GP];
#pragma unroll
  for (int r = 0; r < ROWS_AT_ONCE; ++r) fetch_row(SOLO ? r : warp, qx[r]);
  // the slots of this CTA: whole tiles of 32 from the window's first slot on
  const long long off = a.offset ? a.offset[b] : 0;
  const int lo = (int)max(off, 0ll), hi = (int)min(max(off + a.len[b], 0ll), (long long)a.S_cap);
  const int tiles = hi > lo ? (hi - lo + kAttTile - 1) / kAttTile : 0;
  if (t1 < 0) t1 = tiles;
  constexpr int STRIDE = SOLO ? 1 : TEAMS;
  const int tile0 = t0 + (SOLO ? 0 : team), my = t1 > tile0 ? (t1 - tile0 + STRIDE - 1) / STRIDE : 0;  // tiles tile0, + STRIDE, ...

  // a thread copies chunk cq (16 bytes, one group) of the slots cp, cp + 8, .. + 24 of a tile (where the team has 128 threads per NB = 2; half
  // of that: eight slots), and their scales, which lie as [group][slot % 8][slot / 8]
  constexpr int CPY = kAttTile * GP / (WT * 32);  // 2 or 4 slots per thread
  constexpr int STEP = kAttTile / CPY;
  const int tw = wt * 32 + lane, cp = tw / GP, cq = tw % GP;
  const bool copies = cq < G;
  const size_t row_codes = (size_t)a.heads * G * 16, row_scales = (size_t)a.heads * G;
  const uint8_t* codes = a.codes + ((size_t)b * a.S_cap + cp) * row_codes + (size_t)h * G * 16 + cq * 16;
  const unsigned short* scales = reinterpret_cast<const unsigned short*>(a.scales) + ((size_t)b * a.S_cap + cp) * row_scales + (size_t)h * G + cq;
  unsigned short sc_next[CPY];
  auto request = [&](int it) {
    if (it < my && copies) {
      const int p0 = lo + (tile0 + it * STRIDE) * kAttTile, n = hi - p0;
      unsigned char* st = s_team + it % kAttStages * Sh::STAGE + cp * ROW + cq * 16;
      const uint8_t* from = codes + (size_t)p0 * row_codes;
      const unsigned short* sf = scales + (size_t)p0 * row_scales;
#pragma unroll
      for (int u = 0; u < CPY; ++u) {
        if (cp + STEP * u < n) copy16(st + STEP * u * ROW, from + STEP * u * row_codes);
        sc_next[u] = cp + STEP * u < n ? __ldg(sf + STEP * u * row_scales) : (unsigned short)0;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto keep_scales = [&](int it) {  // slots outside the window get 0: their codes, whatever they are, stand for 0
    if (it < my && copies) {
      unsigned short* st = reinterpret_cast<unsigned short*>(s_team + it % kAttStages * Sh::STAGE + kAttTile * ROW) + cq * kAttTile;
#pragma unroll
      for (int u = 0; u < CPY; ++u) {
        const int p = cp + STEP * u;
        st[(p & 7) * 4 + (p >> 3)] = sc_next[u];
      }
    }
  };
  auto team_sync = [&]() {
    if (WT == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(WT * 32) : "memory");
  };
  request(0);
  if (cq >= G)  // groups that the head does not have
    for (int u = 0; u < CPY; ++u)
      for (int k = 0; k < kAttStages; ++k) {
        const int p = cp + STEP * u;
        reinterpret_cast<unsigned short*>(s_team + k * Sh::STAGE + kAttTile * ROW)[cq * kAttTile + (p & 7) * 4 + (p >> 3)] = 0;
      }

  // Q scaled by a power of two to the upper end of half precision, so that elements down to 2^-32 of the row's largest keep all their bits in bf16, and
  // 22 bits down to 2^-28 of it in 32 bits (whose rounding to a half must not reach 2^16); element e of a thread's word of 8 is half e / 4 of register
  // 2 (e % 2) (+ 1: rows 8 .. 15) of k-step (e % 4) / 2, so that a word of codes gives its fragments by masks alone
  auto lay_out_row = [&](int r, const float (&x)[GP]) {
    unsigned m = 0;
#pragma unroll
    for (int k = 0; k < GP; ++k) m = max(m, __float_as_uint(x[k]) & 0x7fffffffu);
    m = __reduce_max_sync(0xffffffffu, m);
    int e = 0;
    if (m - 1u < 0x7f7fffffu) frexpf(__uint_as_float(m), &e);  // (neither zero nor an infinity or NaN)
    e -= PARTS == 2 ? 15 : 16;
    const float down1 = ldexpf(1.f, -(e / 2)), down2 = ldexpf(1.f, -(e - e / 2));
    const int el = lane & 7, tt = lane >> 3;
    // (the fragments of odd k-steps have neighbouring rows exchanged: the two k-steps that a warp writes at once fall on different banks)
    unsigned char* at = s_q + ((el & 3) / 2 * PARTS) * 512 + (((r & 7) * 4 + tt) ^ ((el & 2) * 2)) * 16 + ((el & 1) * 2 + (r >> 3)) * 4 + (el >> 2) * 2;
#pragma unroll
    for (int k = 0; k < GP; ++k) {
      __half x0, x1;
      split_half(x[k] * down1 * down2, 2048.f, x0, x1);
      *reinterpret_cast<__half*>(at + k * 2 * PARTS * 512) = x0;
      if (PARTS == 2) *reinterpret_cast<__half*>(at + k * 2 * PARTS * 512 + 512) = x1;
    }
    // (exponentials are powers of two.)  Beyond the range of 32 bits the largest number does as well: scores that are finite all the same come from sums
    // of less than 1, and two such sums that differ, by 2^-59 at least, are then 2^68 apart.
    float fac = ldexpf(a.scale, e) * 1.44269504f;
    if (fabsf(a.scale) < INFINITY) fac = fminf(fmaxf(fac, -3.4028234663852886e38f), 3.4028234663852886e38f);
    if constexpr (SOLO) {
      if (lane == 0) s_fac[r] = fac;
    } else {  // every team has a copy
      if (lane < TEAMS) s_fac[(lane - team) * (Sh::TEAM / 4) + r] = fac;
    }
  };
  if constexpr (SOLO) {
    for (int r0 = 0; r0 < 16; r0 += ROWS_AT_ONCE) {
#pragma unroll
      for (int r = 0; r < ROWS_AT_ONCE; ++r) lay_out_row(r0 + r, qx[r]);
      if (r0 + ROWS_AT_ONCE < 16)
#pragma unroll
        for (int r = 0; r < ROWS_AT_ONCE; ++r) fetch_row(r0 + ROWS_AT_ONCE + r, qx[r]);
    }
  } else {
    lay_out_row(warp, qx[0]);
  }
  keep_scales(0);
  request(1);
  // rows without a column: weights 0, never rescaled
  for (int i = tw; i < (Sh::W + 64) / 4; i += WT * 32) reinterpret_cast<unsigned*>(s_w)[i] = i < Sh::W / 4 ? 0u : 0x3f800000u;
  if (SOLO) __syncwarp();
  else __syncthreads();

  float acc[NB][8][4], l[4] = {0.f, 0.f, 0.f, 0.f};  // l: the weights' sums, as a product with ones (columns alike)
#pragma unroll
  for (int x = 0; x < NB; ++x)
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int u = 0; u < 4; ++u) acc[x][j][u] = 0.f;
  if (wt == 0 && lane < 16) s_m[lane] = -INFINITY;
  constexpr bool REG = WT == 1;  // the scores are complete in a warp's registers, and so are the maxima of its rows g and g + 8
  float m_run[2] = {-INFINITY, -INFINITY}, fac[2] = {0.f, 0.f};
  if (REG) {
    fac[0] = s_fac[g];
    fac[1] = s_fac[g + 8];
  }
  keep_scales(1);

  auto stage_at = [&](int it) { return s_team + it % kAttStages * Sh::STAGE; };
  auto slots_left = [&](int it) { return hi - (lo + (tile0 + it * STRIDE) * kAttTile); };
  auto scores = [&](int it, float (&z)[PARTS][4][4]) {
    const unsigned char* st = stage_at(it);
    const unsigned char* s_sc = st + kAttTile * ROW;
    // scores of this warp's elements; n-tile j has slot 8 j + c in its column c
    {
      const unsigned char* cw = st + g * ROW + wt * (2 * NB * 16) + t * 4;
#pragma unroll
      for (int k = 0; k < 2 * NB; ++k) {
        uint4 q[2][PARTS];
        const int kg = wt * 2 * NB + k;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int x = 0; x < PARTS; ++x) q[s][x] = *reinterpret_cast<const uint4*>(s_q + ((kg * 2 + s) * PARTS + x) * 512 + (lane ^ (4 * s)) * 16);
        const uint2 sc4 = *reinterpret_cast<const uint2*>(s_sc + kg * (kAttTile * 2) + g * 8);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t w = *reinterpret_cast<const uint32_t*>(cw + 8 * j * ROW + k * 16);
          uint32_t v[4];  // (elements 0, 4), (1, 5), (2, 6), (3, 7) of the word
          dequant4(w, bits_h2(__byte_perm(j < 2 ? sc4.x : sc4.y, 0, j & 1 ? 0x3232 : 0x1010)), v);
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int x = 0; x < PARTS; ++x) {
              if (k == 0 && s == 0) mma_f16_first(z[x][j], q[s][x], v[2 * s], v[2 * s + 1]);
              else mma_f16(z[x][j], q[s][x], v[2 * s], v[2 * s + 1]);
            }
        }
      }
    }
  };
  auto hand_in = [&](const float (&z)[PARTS][4][4]) {  // this warp's share of the scores
      float* at = s_part + (wt * 16 + g) * kAttPartLd + 2 * t;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float y[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) y[u] = PARTS == 2 ? fmaf(z[PARTS - 1][j][u], 1.f / 2048.f, z[0][j][u]) : z[0][j][u];
        *reinterpret_cast<float2*>(at + 8 * j) = make_float2(y[0], y[1]);
        *reinterpret_cast<float2*>(at + 8 * j + 8 * kAttPartLd) = make_float2(y[2], y[3]);
      }
  };
  auto softmax = [&](int n) {
    // softmax: row r of this warp, slot `lane`; as the second product's k, slot 8 j + c is half j % 2 of register 2 (j / 2) (+ 1: rows 8 .. 15) of lane
    // c / 2 (of a row's four), k-step c % 2, so that a thread's four scales lie side by side
    {
      unsigned char* at0 = s_w + (lane & 1) * W_PARTS * 512 + (lane & 7) / 2 * 16 + (lane >> 4) * 8 + (lane >> 3 & 1) * 2;
      constexpr int RC = ROWS < 4 ? ROWS : 4;  // rows side by side: one's latency is another's work
      for (int r0 = wt * ROWS; r0 < (wt + 1) * ROWS && r0 < n_cols; r0 += RC) {
        float z[RC], m_old[RC];
#pragma unroll
        for (int rr = 0; rr < RC; ++rr) {
          z[rr] = 0.f;
#pragma unroll
          for (int w = 0; w < WT; ++w) z[rr] += s_part[(w * 16 + r0 + rr) * kAttPartLd + lane];
          z[rr] = lane < n ? z[rr] * s_fac[r0 + rr] : -INFINITY;
          m_old[rr] = s_m[r0 + rr];
        }
        __syncwarp();
#pragma unroll
        for (int rr = 0; rr < RC; ++rr) {
          const int r = r0 + rr;
          const float m_new = risen(m_old[rr], warp_max(z[rr])), ref = m_new == -INFINITY ? 0.f : m_new;
          const float alpha = exp2_approx(m_old[rr] - ref), p = weight(z[rr], ref);
          if (lane == 0) {
            s_alpha[r] = alpha;
            s_m[r] = m_new;
          }
          __half p0h, p1h;
          split_half(p, W_UP, p0h, p1h);
          unsigned char* at = at0 + (r & 7) * 64 + (r >> 3) * 4;
          *reinterpret_cast<__half*>(at) = p0h;
          if (W_PARTS == 2) *reinterpret_cast<__half*>(at + 512) = p1h;
        }
      }
    }
  };
  // onto the sums with the weights' rests those with their large parts
  auto add_large_parts = [&](float (&y)[4], const uint4 (&w)[2][W_PARTS], uint32_t b0, uint32_t b1, uint32_t b2, uint32_t b3) {
    if (W_PARTS == 1) return;
    if (W_UP != 1.f)
#pragma unroll
      for (int u = 0; u < 4; ++u) y[u] *= 1.f / W_UP;
    mma_f16(y, w[0][0], b0, b1);
    mma_f16(y, w[1][0], b2, b3);
  };
  auto output = [&](int it, const uint4 (&w)[2][W_PARTS], float al0, float al1) {
    const unsigned char* st = stage_at(it);
    const unsigned char* s_sc = st + kAttTile * ROW;
    // weights x values: n-tile j of a block has element 8 c + j of the block in its column c
    {
      // A tile's sums are added to the earlier ones in the ordinary way.  Straight onto the accumulators the tensor core would cut off what is below 2^-24 of
      // them, of every product: a window's many small weights beside a large one would be lost (1 us less of 53).
      {
        constexpr uint32_t ones = 0x3c003c00u;
        float y[4];
        mma_f16_first(y, w[0][W_PARTS - 1], ones, ones);
        mma_f16(y, w[1][W_PARTS - 1], ones, ones);
        add_large_parts(y, w, ones, ones, ones, ones);
#pragma unroll
        for (int u = 0; u < 4; ++u) l[u] = fmaf(l[u], u < 2 ? al0 : al1, y[u]);
      }
#pragma unroll
      for (int x = 0; x < NB; ++x) {
        const int blk = wt * NB + x;
        const unsigned char* at = st + 2 * t * ROW + blk * 32 + g * 4;
        uint32_t cw[2][4];
        uint2 sc[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
          for (int u = 0; u < 4; ++u) cw[s][u] = *reinterpret_cast<const uint32_t*>(at + (REG ? 16 * s + 8 * (u >> 1) + (u & 1) : s + 8 * u) * ROW);
          const unsigned char* sc_at = s_sc + (2 * blk + (g >> 2)) * (kAttTile * 2) + (2 * t + (REG ? 0 : s)) * 8;
          if (REG) {  // slots 16 s + 2 t, + 1 and + 8, + 9
            const uint32_t even = *reinterpret_cast<const uint32_t*>(sc_at + 4 * s), odd = *reinterpret_cast<const uint32_t*>(sc_at + 8 + 4 * s);
            sc[s] = make_uint2(__byte_perm(even, odd, 0x5410), __byte_perm(even, odd, 0x7632));
          } else {
            sc[s] = *reinterpret_cast<const uint2*>(sc_at);
          }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t v[2][2][4];
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            dequant4(__byte_perm(cw[s][0], cw[s][1], half ? 0x7632 : 0x5410), bits_h2(sc[s].x), v[s][0]);
            dequant4(__byte_perm(cw[s][2], cw[s][3], half ? 0x7632 : 0x5410), bits_h2(sc[s].y), v[s][1]);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float (&o)[4] = acc[x][half * 4 + j];
            float y[4];
            mma_f16_first(y, w[0][W_PARTS - 1], v[0][0][j], v[0][1][j]);
            mma_f16(y, w[1][W_PARTS - 1], v[1][0][j], v[1][1][j]);
            add_large_parts(y, w, v[0][0][j], v[0][1][j], v[1][0][j], v[1][1][j]);
#pragma unroll
            for (int u = 0; u < 4; ++u) o[u] = fmaf(o[u], u < 2 ? al0 : al1, y[u]);
          }
        }
      }
    }
  };
  // w: the weights as fragments of the second product; al0, al1: what the rows' earlier sums are worth now
  if constexpr (REG) {
    for (int it = 0; it < my; ++it) {
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      team_sync();  // the tile is there for all, and all are done with the one before
      request(it + 2);
      const int n = slots_left(it);
      float z[PARTS][4][4];
      scores(it, z);
      uint4 w[2][W_PARTS];
      float al0, al1;
      // The scores lie as the weights have to: half u % 2 of register 2 (j % 2) (+ 1: rows 8 .. 15) of k-step j / 2 is slot 8 j + 2 t + u % 2
      float m[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float y = PARTS == 2 ? fmaf(z[PARTS - 1][j][u], 1.f / 2048.f, z[0][j][u]) : z[0][j][u];
          z[0][j][u] = 8 * j + 2 * t + (u & 1) < n ? y * fac[u >> 1] : -INFINITY;
          m[u >> 1] = fmaxf(m[u >> 1], z[0][j][u]);
        }
      float ref[2], al[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        m[r] = fmaxf(m[r], __shfl_xor_sync(0xffffffffu, m[r], 1));
        m[r] = risen(m_run[r], fmaxf(m[r], __shfl_xor_sync(0xffffffffu, m[r], 2)));
        ref[r] = m[r] == -INFINITY ? 0.f : m[r];
        al[r] = exp2_approx(m_run[r] - ref[r]);
        m_run[r] = m[r];
      }
      al0 = al[0];
      al1 = al[1];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // register k: n-tile 2 s + k / 2, rows of half k % 2
          const int j = 2 * s + (k >> 1), r = k & 1;
          const float p0 = weight(z[0][j][2 * r], ref[r]), p1 = weight(z[0][j][2 * r + 1], ref[r]);
          const __half2 h = __floats2half2_rn(p0, p1);
          hi[k] = h2_bits(h);
          if (W_PARTS == 2) {
            const float2 f = __half22float2(h);
            lo[k] = h2_bits(__floats2half2_rn((p0 - f.x) * W_UP, (p1 - f.y) * W_UP));
          }
        }
        w[s][0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if (W_PARTS == 2) w[s][W_PARTS - 1] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
      output(it, w, al0, al1);
      keep_scales(it + 2);
    }
  } else if (my > 0) {
    // A tile's scores before the output of the one ahead of it: between two barriers lies the work of both products, and the softmax after them is
    // the other teams' time.
    auto next_scores = [&](int it) {
      float z[PARTS][4][4];
      scores(it, z);
      hand_in(z);
    };
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    team_sync();  // tile 0 is there for all
    next_scores(0);
    team_sync();
    request(2);
    softmax(slots_left(0));
    for (int it = 0; it < my; ++it) {
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      team_sync();  // tile it + 1 is there for all, and tile it's weights
      if (it + 1 < my) next_scores(it + 1);
      {
        uint4 w[2][W_PARTS];
        float al0, al1;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int x = 0; x < W_PARTS; ++x) w[s][x] = *reinterpret_cast<const uint4*>(s_w + (s * W_PARTS + x) * 512 + lane * 16);
      al0 = s_alpha[g];
      al1 = s_alpha[g + 8];
        output(it, w, al0, al1);
      }
      keep_scales(it + 2);
      if (it + 1 == my) break;
      team_sync();  // all are done with tile it, and their scores are there
      request(it + 3);
      softmax(slots_left(it + 1));
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");

  if constexpr (SOLO) {  // each lane has runs of 8 elements of two rows
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = g + 8 * half;
      if (r >= n_cols) break;
      const long long c = (long long)b * a.cols + c0 + r;
      // (a column with slots, whatever its sum: one whose scores are all -inf has weights of 0 and gets 0 / 0)
      const bool on = hi > lo && (!a.mask || a.mask[c] != 0);
      const float inv = 1.f / l[2 * half];
      T* o = static_cast<T*>(a.out) + c * a.ld_out + (long long)h * a.d;
      const bool vec = ((uintptr_t)o & 15) == 0;
#pragma unroll
      for (int x = 0; x < NB; ++x)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int i = x * 64 + 8 * (2 * t + u);
          float y[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = on ? acc[x][j][2 * half + u] * inv : 0.f;
          if (vec && i + 8 <= a.d) {
            Mem4Vec<T>::store(o + i, y);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (i + j < a.d) o[i + j] = from_f32<T>(y[j]);
          }
        }
    }
    return;
  }
  // the teams' maxima and sums, then their outputs side by side
  team_sync();
  if (wt == 0) {
    if (REG) {
      if (t == 0) {
        s_ml[team * 16 + g] = m_run[0];
        s_ml[team * 16 + g + 8] = m_run[1];
      }
    } else if (lane < 16) {
      s_ml[team * 16 + lane] = s_m[lane];
    }
    if (t == 0) {
      s_ml[256 + team * 16 + g] = l[0];
      s_ml[256 + team * 16 + g + 8] = l[2];
    }
  }
  __syncthreads();  // (also: nobody reads the fragments and stages any more)
  float* s_out = reinterpret_cast<float*>(smem);
  const int busy = min(TEAMS, t1 - t0);
  if (team < busy) {
    float* o = s_out + (team * 16 + g) * Sh::OUT_LD + 16 * t;
#pragma unroll
    for (int x = 0; x < NB; ++x)
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int u = 0; u < 4; ++u) o[(u >> 1) * 8 * Sh::OUT_LD + (wt * NB + x) * 64 + 8 * (u & 1) + j] = acc[x][j][u];
  }
  __syncthreads();
  // row r: warp r
  if (!in) return;
  float m = -INFINITY, sum = 0.f, f[TEAMS];
#pragma unroll
  for (int k = 0; k < TEAMS; ++k) m = fmaxf(m, s_ml[k * 16 + warp]);
#pragma unroll
  for (int k = 0; k < TEAMS; ++k) {
    f[k] = k < busy ? exp2f(s_ml[k * 16 + warp] - (m == -INFINITY ? 0.f : m)) : 0.f;
    if (k < busy) sum += s_ml[256 + k * 16 + warp] * f[k];
  }
  const long long c = (long long)b * a.cols + c0 + warp;
  const bool part = w != nullptr, on = hi > lo && (!a.mask || a.mask[c] != 0);
  const int dp = G * 32;
  w += part ? warp * (dp + 2) : 0;
  T* out = static_cast<T*>(a.out) + c * a.ld_out + (long long)h * a.d;
  if (part && lane == 0) { w[0] = m; w[1] = sum; }
  const float inv = on ? 1.f / sum : 0.f;
  constexpr int AT_ONCE = GP < 8 ? GP : 8;
  for (int k0 = 0; k0 < GP; k0 += AT_ONCE) {
    float y[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) y[u] = 0.f;
#pragma unroll
    for (int k = 0; k < TEAMS; ++k) {
      if (k >= busy) break;
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) y[u] = fmaf(s_out[(k * 16 + warp) * Sh::OUT_LD + (k0 + u) * 32 + lane], f[k], y[u]);
    }
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int i = (k0 + u) * 32 + lane;
      if (part) {
        if (i < dp) w[2 + i] = y[u];
      } else if (i < a.d) {
        out[i] = from_f32<T>(on ? y[u] * inv : 0.f);
      }
    }
  }
}
// `parts` CTAs are dealt out to the source columns: at least one each, and so many that none has more tiles than the least number with which they
// suffice.  (16 columns of 4000 .. 8192 slots: 9 CTAs each: the multiprocessors were at work 70 % of the time; one each and the others by
// tiles, rounded down: 90 %, 54 us, so 52.5.)  The first CTA of column b, for b = 0 .. B (B <= kMostColumns), and its tiles.  By one warp.
constexpr int kMostColumns = 256;
__device__ __forceinline__ void deal_out(const Mem4Attend& a, int parts, int* first, int* tiles) {
  const int lane = threadIdx.x & 31;
  int total = 0, before = 0;
  const auto per_column = [](int tiles, int most) { return max(1, (tiles + most - 1) / most); };
  for (int b = lane; b < a.B; b += 32) {
    const long long off = a.offset ? a.offset[b] : 0;
    const int lo = (int)max(off, 0ll), hi = (int)min(max(off + a.len[b], 0ll), (long long)a.S_cap);
    const int n = hi > lo ? (hi - lo + kAttTile - 1) / kAttTile : 0;
    tiles[b] = n;
    total += n;
  }
  total = __reduce_add_sync(0xffffffffu, total);
  int low = max(1, (total + parts - 1) / parts), most = max(1, (total + parts - a.B - 1) / (parts - a.B));  // (with `most` they suffice: parts > B)
  while (low < most) {
    const int mid = (low + most) / 2;
    int n = 0;
    for (int b = lane; b < a.B; b += 32) n += per_column(tiles[b], mid);
    if ((int)__reduce_add_sync(0xffffffffu, n) <= parts) most = mid;
    else low = mid + 1;
  }
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const int b = b0 + lane, n = b < a.B ? per_column(tiles[b], most) : 0;
    int up = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += x;
    }
    if (b < a.B) first[b] = before + up - n;
    before += __shfl_sync(0xffffffffu, up, 31);
  }
  if (lane == 0) first[a.B] = before;
  __syncwarp();
}
template <class T, int WT, int NB, int HOW>  // HOW: ALONE, WHOLE, DEALT
__global__ void __launch_bounds__((HOW == ALONE ? 8 : kAttWarps) * 32, HOW == ALONE && NB == 1 ? 2 : 1) mem4_attend_kernel(const Mem4Attend a, const AttPlan pl) {
  constexpr bool SOLO = HOW == ALONE;
  extern __shared__ __align__(16) unsigned char smem[];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // (the combination waits for this launch's end before it reads anything)
  if constexpr (SOLO) {
    const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (unit >= (long long)a.B * pl.q_tiles * a.heads) return;  // (teams of one warp: no barrier is missed)
    const int bq = (int)(unit / a.heads), b = bq / pl.q_tiles;
    attend_part<T, WT, NB, SOLO>(a, pl, smem, b, (bq - b * pl.q_tiles) * 16, (int)(unit - (long long)bq * a.heads), 0, -1, nullptr);
  } else if constexpr (HOW == DEALT) {
    __shared__ int s_first[kMostColumns + 1], s_tiles[kMostColumns];
    if (threadIdx.x < 32) deal_out(a, pl.parts, s_first, s_tiles);
    __syncthreads();
    const int p = blockIdx.x;
    if (p >= s_first[a.B]) return;  // (the whole CTA)
    int b = 0, hi = a.B;
    while (hi - b > 1) {
      const int mid = (b + hi) / 2;
      if (s_first[mid] <= p) b = mid;
      else hi = mid;
    }
    const int n = s_first[b + 1] - s_first[b], k = p - s_first[b], share = s_tiles[b] / n, more = s_tiles[b] - share * n, t0 = k * share + min(k, more);
    attend_part<T, WT, NB, SOLO>(a, pl, smem, b, blockIdx.y * 16, blockIdx.z, t0, t0 + share + (k < more),
                                 a.work + (((long long)blockIdx.z * pl.q_tiles + blockIdx.y) * pl.parts + p) * 16 * (pl.G * 32 + 2));
  } else {
    const int b = blockIdx.y / pl.q_tiles;
    attend_part<T, WT, NB, SOLO>(a, pl, smem, b, (blockIdx.y - b * pl.q_tiles) * 16, blockIdx.z, 0, -1, nullptr);
  }
}
// The parts of a column and head: their weights first, then a thread per element
template <class T>
__global__ void __launch_bounds__(256) mem4_combine_kernel(const __grid_constant__ Mem4Attend a, const AttPlan pl) {
  __shared__ int s_first[kMostColumns + 1], s_tiles[kMostColumns];
  __shared__ float s_f[kMostColumns], s_red[8];
  const int pieces = (a.d + 255) / 256;  // of 256 elements, a CTA each
  const long long c = blockIdx.x / pieces, b = c / a.cols;
  const int tid = threadIdx.x, h = blockIdx.y, dp = pl.G * 32, at = (int)(c - b * a.cols);
  if (tid < 32) deal_out(a, pl.parts, s_first, s_tiles);  // (the lengths are not the launch's ahead)
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long step = 16ll * (dp + 2);
  const int n = s_first[b + 1] - s_first[b];
  const float* w = a.work + (((long long)h * pl.q_tiles + at / 16) * pl.parts + s_first[b]) * step + (at % 16) * (dp + 2);
  float m = -INFINITY;
  for (int s = tid; s < n; s += 256) {
    const float x = __ldcg(w + s * step);
    s_f[s] = x;
    m = fmaxf(m, x);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((tid & 31) == 0) s_red[tid >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 8; ++k) m = fmaxf(m, s_red[k]);
  __syncthreads();
  float l = 0.f;
  for (int s = tid; s < n; s += 256) {
    const float f = exp2f(s_f[s] - (m == -INFINITY ? 0.f : m));
    s_f[s] = f;
    l += __ldcg(w + s * step + 1) * f;  // (also where f is 0: a part whose scores are all NaN has no maximum, but its sum is NaN)
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  if ((tid & 31) == 0) s_red[tid >> 5] = l;
  __syncthreads();
  l = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) l += s_red[k];
  const bool on = s_tiles[b] > 0 && (!a.mask || a.mask[c] != 0);
  T* out = static_cast<T*>(a.out) + c * a.ld_out + (long long)h * a.d;
  const int i = (int)(blockIdx.x - c * pieces) * 256 + tid;
  if (i < a.d) {
    float y = 0.f;
#pragma unroll 8
    for (int s = 0; s < n; ++s) {
      const float x = __ldcg(w + s * step + 2 + i), f = s_f[s];
      y = fmaf(x, f, y);
    }
    out[i] = from_f32<T>(on ? y / l : 0.f);
  }
}

}  // namespace

namespace {

// Teams of as many lanes as a vector has (256 at most, then several CTAs share it).  CTAs along the slots: the six per multiprocessor that are resident
// at once (with eight, 16 x 8192 vectors of 1024 in bf16 are packed in 78 us, not 64); of longer memories in unpacking, whose stores like
// to lie together, up to 32 with 16 slots each (61 -> 59 us, fp32 115 -> 99).
dim3 mem4_grid(int B, int S, int heads, int d, bool aligned, bool unpack, int* team) {
  const int quads = heads * mem4_groups(d) * 4;
  *team = std::min(aligned ? quads : (quads + 31) / 32 * 32, 256);  // (unaligned: whole warps)
  const long long x = (B + 256 / *team - 1) / (256 / *team), z = (quads + *team - 1) / *team;
  const auto along = [&](long long per_sm) { return (per_sm * device_sms() + x * z - 1) / (x * z); };
  const long long want = unpack ? std::max(along(kMem4PerSm), std::min<long long>(S / 16, along(32))) : along(kMem4PerSm);
  const long long y = std::max<long long>(1, std::min<long long>(S, want));
  return dim3((unsigned)x, (unsigned)std::min<long long>(y, 65535), (unsigned)z);
}
template <class T>
cudaError_t pack_type(const Mem4Pack& a, cudaStream_t st) {
  int team;
  const bool aligned = ((uintptr_t)a.x & 15) == 0 && a.ld_slot * sizeof(T) % 16 == 0 && a.ld_col * sizeof(T) % 16 == 0 && a.d % 8 == 0;
  const dim3 grid = mem4_grid(a.B, a.S, a.heads, a.d, aligned, false, &team);
  if (aligned) mem4_pack_kernel<T, true><<<grid, 256, 0, st>>>(a, team);
  else mem4_pack_kernel<T, false><<<grid, 256, 0, st>>>(a, team);
  return cudaGetLastError();
}
template <class T>
cudaError_t unpack_type(const Mem4Unpack& a, cudaStream_t st) {
  int team;
  const bool aligned = ((uintptr_t)a.out & 15) == 0 && a.d % 8 == 0;
  const dim3 grid = mem4_grid(a.B, a.S, a.heads, a.d, aligned, true, &team);
  if (aligned) mem4_unpack_kernel<T, true><<<grid, 256, 0, st>>>(a, team);
  else mem4_unpack_kernel<T, false><<<grid, 256, 0, st>>>(a, team);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_mem4_pack(const Mem4Pack& a, int elem, cudaStream_t st) {
  if (a.S == 0) return cudaSuccess;
  count_launch();
  return elem == ELEM_F32 ? pack_type<float>(a, st) : elem == ELEM_BF16 ? pack_type<__nv_bfloat16>(a, st) : pack_type<__half>(a, st);
}
cudaError_t launch_mem4_unpack(const Mem4Unpack& a, int elem, cudaStream_t st) {
  if (a.S == 0) return cudaSuccess;
  count_launch();
  return elem == ELEM_F32 ? unpack_type<float>(a, st) : elem == ELEM_BF16 ? unpack_type<__nv_bfloat16>(a, st) : unpack_type<__half>(a, st);
}
namespace {

AttPlan att_plan(int B, int cols, int S_cap, int heads, int d) {
  AttPlan pl;
  pl.G = mem4_groups(d);
  pl.warps = pl.G <= 4 ? 1 : pl.G <= 8 ? 2 : pl.G <= 16 ? 4 : 8;
  pl.blocks = pl.G <= 2 ? 1 : 2;
  pl.q_tiles = (cols + 15) / 16;
  const long long units = (long long)B * pl.q_tiles * heads, sms = device_sms(), tiles = (S_cap + kAttTile - 1) / kAttTile;
  // Parts: no more than the multiprocessors, nor than leave each team of a part two tiles; only where there are twice as many of them as source
  // columns (100 columns of up to 1000 slots on 148 CTAs: 65 us, on 100 53)
  const long long parts = std::min<long long>(sms / ((long long)pl.q_tiles * heads), B * tiles / (2 * (kAttWarps / pl.warps)));
  pl.parts = parts >= 2ll * B && parts > 1 && parts <= kMostColumns ? (int)parts : 0;
  // a team on its own: as long as the tiles of all units take its multiprocessor no longer than the CTAs that a unit each would need (in tiles'
  // times: two for the start and the end of a CTA)
  const long long per_sm = pl.blocks == 1 ? 16 : 8;
  const long long alone = (units + per_sm * sms - 1) / (per_sm * sms) * (2 + tiles), shared = (units + sms - 1) / sms * (2 + (tiles + 15) / 16);
  pl.solo = pl.warps == 1 && pl.parts == 0 && alone <= shared;
  return pl;
}
template <class T, int WT, int NB, int HOW>
cudaError_t attend_launch(const Mem4Attend& a, const AttPlan& pl, cudaStream_t st) {
  constexpr bool SOLO = HOW == ALONE;
  using Sh = AttShape<AttParts<T>::Q, AttParts<T>::W, WT, NB, SOLO>;
  constexpr int smem = Sh::SMEM;
  static bool configured[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(mem4_attend_kernel<T, WT, NB, HOW>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  const long long units = (long long)a.B * pl.q_tiles * a.heads;
  const dim3 grid = SOLO ? dim3((unsigned)((units + Sh::TEAMS - 1) / Sh::TEAMS)) : pl.parts ? dim3(pl.parts, pl.q_tiles, (unsigned)a.heads) : dim3(1, (unsigned)(a.B * pl.q_tiles), (unsigned)a.heads);
  mem4_attend_kernel<T, WT, NB, HOW><<<grid, Sh::WARPS * 32, smem, st>>>(a, pl);
  return cudaGetLastError();
}
template <class T, int WT, int NB>
cudaError_t attend_how(const Mem4Attend& a, const AttPlan& pl, cudaStream_t st) {
  if constexpr (WT == 1)
    if (pl.solo) return attend_launch<T, WT, NB, ALONE>(a, pl, st);
  return pl.parts ? attend_launch<T, WT, NB, DEALT>(a, pl, st) : attend_launch<T, WT, NB, WHOLE>(a, pl, st);
}
template <class T>
cudaError_t attend_type(const Mem4Attend& all, cudaStream_t st) {
  const AttPlan pl = att_plan(all.B, all.cols, all.S_cap, all.heads, all.d);
  const int most = 65535 / pl.q_tiles;  // source columns of a launch
  if (most < 1) return cudaErrorInvalidValue;
  for (int at = 0; at < all.B; at += most) {
    Mem4Attend a = all;
    a.B = std::min(most, all.B - at);
    const size_t rows = (size_t)at * a.S_cap * a.heads * pl.G;
    const long long cols = (long long)at * a.cols;
    a.codes += rows * 16;
    a.scales += rows;
    a.len += at;
    if (a.offset) a.offset += at;
    if (a.mask) a.mask += cols;
    a.q = static_cast<const T*>(a.q) + cols * a.ld_q;
    a.out = static_cast<T*>(a.out) + cols * a.ld_out;
    count_launch();
    const cudaError_t e = pl.blocks == 1   ? attend_how<T, 1, 1>(a, pl, st)
                          : pl.warps == 1 ? attend_how<T, 1, 2>(a, pl, st)
                          : pl.warps == 2 ? attend_how<T, 2, 2>(a, pl, st)
                          : pl.warps == 4 ? attend_how<T, 4, 2>(a, pl, st)
                                          : attend_how<T, 8, 2>(a, pl, st);
    if (e != cudaSuccess) return e;
    if (pl.parts == 0) continue;
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)((long long)a.B * a.cols * ((a.d + 255) / 256)), a.heads);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    count_launch();
    const cudaError_t e2 = cudaLaunchKernelEx(&cfg, mem4_combine_kernel<T>, a, pl);
    if (e2 != cudaSuccess) return e2;
  }
  return cudaSuccess;
}

}  // namespace

size_t mem4_attend_work(int B, int cols, int S_cap, int heads, int d) {
  const AttPlan pl = att_plan(B, cols, S_cap, heads, d);
  return pl.parts ? (size_t)heads * pl.q_tiles * pl.parts * 16 * (pl.G * 32 + 2) : 0;
}
cudaError_t launch_mem4_attend(const Mem4Attend& a, int elem, cudaStream_t st) {
  if (a.B == 0 || a.cols == 0) return cudaSuccess;
  switch (elem) {
    case ELEM_F32: return attend_type<float>(a, st);
    case ELEM_BF16: return attend_type<__nv_bfloat16>(a, st);
  }
  return attend_type<__half>(a, st);
}

}  // namespace zrnn
