// Selection over beams and vocabulary, and the reorder of the states that goes with it.
#include <cooperative_groups.h>

#include <algorithm>
#include <cstring>
#include <type_traits>

#include "kernels.cuh"
#include "operators.cuh"
#include "tc_gemm.cuh"

namespace zrnn {
namespace {

namespace cg = cooperative_groups;

// A candidate as one whole number: its value in an order-preserving form, then the complement of its index j * V + v, so that the larger number is
// the larger value or, of equal ones, the lower index.  Numbers of different candidates differ.
__device__ __forceinline__ unsigned ordered(float x) {
  const unsigned u = __float_as_uint(x + 0.0f);  // (-0 equals 0)
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(unsigned u) { return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u); }
constexpr unsigned kOrderedMinusInf = 0x007fffffu;

// Outcome `rank` of a sentence; key 0: there is none
__device__ __forceinline__ void write_choice(const BeamSelect& a, int sent, int rank, unsigned long long key) {
  const bool some = (unsigned)(key >> 32) > kOrderedMinusInf;
  const unsigned at = ~(unsigned)key;
  const long long o = (long long)sent * a.k + rank;
  a.score_out[o] = some ? unordered((unsigned)(key >> 32)) : -INFINITY;
  a.word_out[o] = some ? (int)(at % (unsigned)a.V) : -1;
  a.parent_out[o] = some ? a.first_row + (int)(at / (unsigned)a.V) + sent * a.beam : -1;
}
// largest of the block's numbers; `slot` alternates between consecutive calls
__device__ __forceinline__ unsigned long long block_max(unsigned long long x, int slot) {
  __shared__ unsigned long long s_red[2][32];
  const int lane = threadIdx.x & 31;
  const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned)(x >> 32));
  const unsigned lo = __reduce_max_sync(0xffffffffu, (unsigned)(x >> 32) == hi ? (unsigned)x : 0u);
  if (lane == 0) s_red[slot][threadIdx.x >> 5] = ((unsigned long long)hi << 32) | lo;
  __syncthreads();
  x = lane < (int)blockDim.x / 32 ? s_red[slot][lane] : 0ull;
  const unsigned h = __reduce_max_sync(0xffffffffu, (unsigned)(x >> 32));
  return ((unsigned long long)h << 32) | __reduce_max_sync(0xffffffffu, (unsigned)(x >> 32) == h ? (unsigned)x : 0u);
}
// A number that at least k of the block's threads reach, where k are above -inf, else the least one above that: the smallest of the W warps'
// ceil(k / W)-th largest.  Some 50 of 256 random numbers reach that of k = 12, and ranking 50 is cheaper than 12 rounds for the largest (2400
// cycles).
__device__ __forceinline__ unsigned common_bound(unsigned v, int k) {
  __shared__ unsigned s_nth[32];
  const int lane = threadIdx.x & 31, W = blockDim.x / 32;
  unsigned nth = 0;
  for (int r = (k + W - 1) / W; r > 0; --r) {
    nth = __reduce_max_sync(0xffffffffu, v);
    const unsigned who = __ballot_sync(0xffffffffu, v == nth);
    if (lane == __ffs(who) - 1) v = 0;
  }
  if (lane == 0) s_nth[threadIdx.x >> 5] = nth;
  __syncthreads();
  return max(__reduce_min_sync(0xffffffffu, s_nth[lane & (W - 1)]), kOrderedMinusInf + 1);
}
// The selection reads every value once and compares maxima.  With the row's score and normaliser the candidate's value is a monotone function of
// the value read, so a segment (E = 32 lanes x 16 bytes x U consecutive values of a row) needs one maximum of raw values: one
// instruction per value in 32 bits, half of one in 16.  The CTAs of a cluster share a sentence's segments; then
//   1. they agree on the k segments of largest (maximum, lowest index): each of these holds a candidate that beats all of any other segment,
//      so the k best candidates lie in them; the least of the k maxima is a bound for the k-th best;
//   2. each reads its own ones of those segments again and takes what reaches the bound, at most k of a segment, largest first;
//   3. the first CTA ranks these (a dozen or two unless values tie or ascend).
// Steps 1 to 3 are some 5000 cycles of latency; the rest is the stream of the values: 64 x 12 x 50000 fp32 35 us (4.4 TB/s over all), 128 x 8 x
// 200000 bf16 73 (5.6 TB/s), 12 x 40000 fp32 11.  As separate CTAs, each with k segments of its own to read again and its k best to be merged
// by a second launch, a batch of 64 x 12 x 50000 fp32 took 40 us (26 of them the stream of the values, at 6 TB/s) and a sentence of 12 x
// 40000 11.7.  Sentences too long for a cluster (8 x 1024 segments) still go that way.
constexpr int kSelSegs = 1024, kSelCluster = 8;

template <class T> struct Raw;
template <> struct Raw<float> {
  static constexpr int VEC = 4;
  float m;
  __device__ void init() { m = -INFINITY; }
  __device__ void take(uint4 v) {
    m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w))));
  }
  __device__ void take1(unsigned x) { m = fmaxf(m, __uint_as_float(x)); }
  __device__ float value() const { return m; }
};
template <bool HALF>
struct Raw16 {  // two maxima side by side; a NaN loses against a number
  static constexpr int VEC = 8;
  uint32_t m;
  __device__ static uint32_t max2(uint32_t x, uint32_t y) {
    uint32_t r;
    if (HALF) asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
    else asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
    return r;
  }
  __device__ static float f32(uint32_t bits) { return HALF ? __half2float(__ushort_as_half((unsigned short)bits)) : __uint_as_float(bits << 16); }
  __device__ void init() { m = HALF ? 0xfc00fc00u : 0xff80ff80u; }
  __device__ void take(uint4 v) { m = max2(m, max2(max2(v.x, v.y), max2(v.z, v.w))); }
  __device__ void take1(unsigned x) { m = max2(m, (m & 0xffff0000u) | x); }
  __device__ float value() const { return fmaxf(f32(m & 0xffffu), f32(m >> 16)); }
};
template <> struct Raw<__half> : Raw16<true> {};
template <> struct Raw<__nv_bfloat16> : Raw16<false> {};

struct SelectPlan {
  int segs_row, n_seg;  // segments of a row, of a sentence
  int ctas, per;        // CTAs of a sentence, segments of a CTA
  int parts;            // > 1: lists that a second launch merges; 1: the CTAs are a cluster
  int U, NT;
};

template <class T> __device__ __forceinline__ float bits_f32(unsigned x) {
  if constexpr (std::is_same<T, float>::value) return __uint_as_float(x);
  else if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)x));
  else return __uint_as_float(x << 16);
}
// what makes a row's raw value a candidate's value
struct RowForm {
  float score, lse;
  bool has_lse, done;
  __device__ float operator()(float z) const {
    if (has_lse) z = __fsub_rn(z, lse);
    return __fadd_rn(score, z);
  }
};
__device__ __forceinline__ RowForm row_form(const BeamSelect& a, long long r) {
  return RowForm{a.scores[r], a.lse ? a.lse[r] : 0.f, a.lse != nullptr, a.done && a.done[r] != 0};
}
__device__ __forceinline__ unsigned ordered_or_none(float x) { return x != x ? 0u : ordered(x); }

template <class T, int U, int NT>
__global__ void __launch_bounds__(NT, NT == 256 ? 4 : 1) beam_select_kernel(const BeamSelect a, const SelectPlan pl) {
  constexpr int VEC = Raw<T>::VEC, E = 32 * VEC * U, W = NT / 32;
  using Bits = typename std::conditional<sizeof(T) == 4, unsigned, unsigned short>::type;
  extern __shared__ __align__(16) unsigned long long s_list[];  // k * k, the first CTA's
  __shared__ unsigned s_max[kSelSegs];
  __shared__ unsigned long long s_seg[kSelSegs];                  // segments that reach the CTA's bound
  __shared__ unsigned long long s_all[kSelCluster * kSelectMax];  // the CTAs' k best segments
  __shared__ int s_chosen[kSelectMax];
  __shared__ unsigned s_bound;
  __shared__ int s_n, s_left, s_chosen_n;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), me = cluster.block_rank();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // (a merge waits for this launch's end before it reads anything)
  const int sent = blockIdx.y, part = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int first = min(part * pl.per, pl.n_seg), n = min(pl.per, pl.n_seg - first);
  const T* base = static_cast<const T*>(a.logp) + (long long)sent * a.beam * a.ld;
  for (int i = tid; i < kSelSegs; i += NT) s_max[i] = 0;
  for (int i = tid; i < kSelCluster * kSelectMax; i += NT) s_all[i] = 0;
  if (tid == 0) {
    s_n = s_left = s_chosen_n = 0;
    s_bound = kOrderedMinusInf + 1;
  }
  __syncthreads();  // (the words are zero before any warp stores a maximum there)
  __syncwarp();
  if (C > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  // segment q of a row holds the values [q * E - lead, (q + 1) * E - lead): its vectors lie on 16 bytes
  auto lead_of = [&](const T* row) { return (int)(((uintptr_t)row & 15) / sizeof(T)); };
  // A warp walks over consecutive segments, the next one's vectors requested before it looks at the present one's.
  struct Cursor {
    int j, q;  // row of the sentence, segment of the row
  };
  const int each = (n + W - 1) / W, i0 = min(warp * each, n), i1 = min(i0 + each, n);
  int form_row = -1;
  RowForm form;
  auto enter = [&](int j) {  // (a warp stays in a row for tens of segments, mostly)
    if (j != form_row) {
      form = row_form(a, (long long)sent * a.beam + j);
      form_row = j;
    }
  };
  auto whole = [&](const Cursor& c) {
    const int from = c.q * E - lead_of(base + c.j * a.ld);
    return from >= 0 && from + E <= a.V;
  };
  auto request = [&](const Cursor& c, uint4 (&v)[U]) {
    if (!whole(c) || (a.done && __ldg(a.done + (long long)sent * a.beam + c.j))) return;
    const T* row = base + c.j * a.ld;
    const uint4* p = reinterpret_cast<const uint4*>(row + (c.q * E - lead_of(row))) + lane;
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = __ldg(p + 32 * u);
  };
  auto look = [&](const Cursor& c, const uint4 (&v)[U], int i) {
    enter(c.j);
    float best = -INFINITY;
    Raw<T> m;
    m.init();
    const T* row = base + c.j * a.ld;
    const int from = c.q * E - lead_of(row);
    if (form.done) {
      if (a.eos >= from && a.eos < from + E) best = form.score;
    } else {
      if (whole(c)) {
#pragma unroll
        for (int u = 0; u < U; ++u) m.take(v[u]);
      } else {
        for (int e = from + lane; e < from + E; e += 32)
          if (e >= 0 && e < a.V) m.take1(reinterpret_cast<const Bits*>(row)[e]);
      }
      best = form(m.value());
    }
    const unsigned o = __reduce_max_sync(0xffffffffu, ordered_or_none(best));
    if (lane == 0) s_max[i] = o;
  };
  auto step = [&](Cursor& c) {
    if (++c.q == pl.segs_row) { c.q = 0; ++c.j; }
  };
  if (i0 < i1) {
    uint4 v0[U], v1[U];
    Cursor c{(first + i0) / pl.segs_row, (first + i0) % pl.segs_row};
    request(c, v0);
    for (int i = i0; i < i1; i += 2) {
      Cursor d = c;
      step(d);
      if (i + 1 < i1) request(d, v1);
      look(c, v0, i);
      if (i + 1 == i1) break;
      c = d;
      step(c);
      if (i + 2 < i1) request(c, v0);
      look(d, v1, i + 1);
    }
  }
  __syncthreads();
  // 1. the CTA's best segments, ties to the lower one, then the cluster's
  {
    unsigned v[kSelSegs / NT], most = 0;
#pragma unroll
    for (int u = 0; u < kSelSegs / NT; ++u) {
      v[u] = s_max[u * NT + lane * W + warp];  // (every warp sees segments of all places)
      most = max(most, v[u]);
    }
    const unsigned floor = common_bound(most, a.k);
#pragma unroll
    for (int u = 0; u < kSelSegs / NT; ++u)
      if (v[u] >= floor) s_seg[atomicAdd(&s_left, 1)] = ((unsigned long long)v[u] << 32) | (unsigned)~(first + u * NT + lane * W + warp);
    __syncwarp();
    if (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // (the others' arrays are in place)
    __syncthreads();
    const int left = s_left;
    for (int i = tid; i < left; i += NT) {
      const unsigned long long key = s_seg[i];
      int rank = 0;
      for (int o = 0; o < left; ++o) rank += s_seg[o] > key;
      if (rank < a.k)
        for (int r = 0; r < C; ++r) *cluster.map_shared_rank(&s_all[me * a.k + rank], r) = key;
    }
    if (C > 1) cluster.sync();
    else __syncthreads();
    for (int i = tid; i < C * a.k; i += NT) {
      const unsigned long long key = s_all[i];
      int rank = 0;
      for (int o = 0; o < C * a.k; ++o) rank += s_all[o] > key;
      if (key == 0 || rank >= a.k) continue;
      if (i / a.k == me) s_chosen[atomicAdd(&s_chosen_n, 1)] = (int)~(unsigned)key;
      if (rank == a.k - 1) s_bound = (unsigned)(key >> 32);
    }
  }
  __syncthreads();
  // 2. what reaches the bound in them
  const unsigned bound = s_bound;
  const int chosen = s_chosen_n;
  unsigned long long* list = cluster.map_shared_rank(s_list, 0);
  int* list_n = cluster.map_shared_rank(&s_n, 0);
  for (int c = warp; c < chosen; c += W) {
    const int at = s_chosen[c], j = at / pl.segs_row, q = at - j * pl.segs_row;
    const T* row = base + j * a.ld;
    const RowForm f = row_form(a, (long long)sent * a.beam + j);
    const int from = q * E - lead_of(row);
    unsigned raw[E / 32];  // value from + 32 i + lane; all requested before the first is looked at (in a branch each they took turns: 14 us)
#pragma unroll
    for (int i = 0; i < E / 32; ++i) raw[i] = __ldg(reinterpret_cast<const Bits*>(row) + min(max(from + 32 * i + lane, 0), a.V - 1));
    unsigned v[E / 32];
    unsigned mine = 0;
    int where = 0;
#pragma unroll
    for (int i = 0; i < E / 32; ++i) {
      const int e = from + 32 * i + lane;
      const float x = f.done ? (e == a.eos ? f.score : -INFINITY) : f(bits_f32<T>(raw[i]));
      v[i] = e >= 0 && e < a.V ? ordered_or_none(x) : 0u;
      if (v[i] > mine) { mine = v[i]; where = i; }
    }
    for (int taken = 0; taken < a.k; ++taken) {
      const unsigned top = __reduce_max_sync(0xffffffffu, mine);
      if (top < bound) break;
      const unsigned off = __reduce_min_sync(0xffffffffu, mine == top ? (unsigned)(32 * where + lane) : ~0u);
      if ((off & 31) == (unsigned)lane) {
        list[atomicAdd(list_n, 1)] = ((unsigned long long)top << 32) | ~((unsigned)j * (unsigned)a.V + (unsigned)(from + (int)off));
        mine = 0;
#pragma unroll
        for (int i = 0; i < E / 32; ++i) {
          if (i == (int)(off >> 5)) v[i] = 0;
          if (v[i] > mine) { mine = v[i]; where = i; }
        }
      }
    }
  }
  if (C > 1) cluster.sync();
  else __syncthreads();
  // 3. their order
  if (me != 0) return;
  const int m = s_n;
  auto put = [&](int rank, unsigned long long key) {
    if (pl.parts > 1) a.work[((long long)sent * pl.parts + part) * a.k + rank] = key;
    else write_choice(a, sent, rank, key);
  };
  if (m <= 512) {
    for (int i = tid; i < m; i += NT) {
      const unsigned long long key = s_list[i];
      int rank = 0;
      for (int o = 0; o < m; ++o) rank += s_list[o] > key;
      if (rank < a.k) put(rank, key);
    }
  } else {
    unsigned long long last = ~0ull;
    for (int rank = 0; rank < a.k; ++rank) {
      unsigned long long best = 0;
      for (int i = tid; i < m; i += NT) best = s_list[i] < last ? max(best, s_list[i]) : best;
      last = block_max(best, rank & 1);
      if (tid == 0) put(rank, last);
    }
  }
  for (int rank = m + tid; rank < a.k; rank += NT) put(rank, 0);
}

// The parts' lists, each sorted, of a sentence.  What fits into shared memory is brought there; the keys that reach a bound for the k-th best (at
// least k heads do) are ranked.  Where there are too many of those (ties), or the lists are too long: k rounds for the largest head.
// (A byte per list as well: both fit into the 48 KB that need no asking, 2^15 lists, of 2^25 rows of a segment each, without the keys.)
constexpr int kMergeThreads = 256, kMergeKeys = 4800, kMergeRank = 512;
static_assert(kMergeKeys * 9 + kMergeRank * 8 + 1024 <= 48 * 1024 && (1 << 15) + kMergeRank * 8 + 1024 <= 48 * 1024, "");
__global__ void __launch_bounds__(kMergeThreads) beam_select_merge_kernel(const BeamSelect a, int parts) {
  extern __shared__ __align__(16) unsigned long long s_keys[];  // the keys, if they fit; then per list how many are gone
  __shared__ unsigned long long s_cand[kMergeRank];
  __shared__ int s_n;
  const int sent = blockIdx.x, tid = threadIdx.x, total = parts * a.k;
  const bool near = total <= kMergeKeys;
  unsigned char* s_gone = reinterpret_cast<unsigned char*>(s_keys + (near ? total : 0));
  for (int p = tid; p < parts; p += kMergeThreads) s_gone[p] = 0;
  if (tid == 0) s_n = 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const unsigned long long* lists = a.work + (long long)sent * total;
  if (near) {
#pragma unroll 4
    for (int i = tid; i < total; i += kMergeThreads) s_keys[i] = __ldcg(lists + i);
    __syncthreads();
    const int list = (tid & 31) * 8 + (tid >> 5);
    unsigned head = 0;
    for (int p = list; p < parts; p += kMergeThreads) head = max(head, (unsigned)(s_keys[p * a.k] >> 32));
    const unsigned floor = common_bound(head, a.k);
    for (int p = list; p < parts; p += kMergeThreads)
      for (int i = p * a.k; i < (p + 1) * a.k; ++i) {
        const unsigned long long key = s_keys[i];
        if ((unsigned)(key >> 32) < floor) break;
        const int at = atomicAdd(&s_n, 1);
        if (at < kMergeRank) s_cand[at] = key;
      }
    __syncthreads();
    const int m = s_n;
    if (m <= kMergeRank) {
      for (int i = tid; i < m; i += kMergeThreads) {
        const unsigned long long key = s_cand[i];
        int rank = 0;
        for (int o = 0; o < m; ++o) rank += s_cand[o] > key;
        if (rank < a.k) write_choice(a, sent, rank, key);
      }
      for (int rank = m + tid; rank < a.k; rank += kMergeThreads) write_choice(a, sent, rank, 0);
      return;
    }
  }
  unsigned long long mine = 0, won = 0;
  int from = 0;
  auto look = [&]() {
    mine = 0;
    for (int p = tid; p < parts; p += kMergeThreads) {
      const int at = p * a.k + s_gone[p];
      const unsigned long long head = s_gone[p] >= a.k ? 0ull : near ? s_keys[at] : __ldcg(lists + at);
      if (head > mine) { mine = head; from = p; }
    }
  };
  look();
  for (int rank = 0; rank < a.k; ++rank) {
    const unsigned long long top = block_max(mine, rank & 1);
    if (tid == rank) won = top;
    if (mine == top && top) {
      ++s_gone[from];
      look();
    }
  }
  if (tid < a.k) write_choice(a, sent, tid, won);
}

// A thread takes one piece (a U) of the columns of one group, at most NG of them, and has all loaded before it stores the first, so that a
// group can be reordered in place; out of place a group is whatever four columns follow one another.
template <class U, int NG>
__global__ void __launch_bounds__(128) beam_reorder_kernel(const __grid_constant__ BeamReorder a) {
  const int arr = blockIdx.z;
  const long long pieces = a.bytes[arr] / (long long)sizeof(U), i = (long long)blockIdx.x * 128 + threadIdx.x;
  if (i >= pieces) return;
  const U* src = reinterpret_cast<const U*>(a.src[arr]) + i;
  U* dst = reinterpret_cast<U*>(a.dst[arr]) + i;
  const bool in_place = a.src[arr] == a.dst[arr];
  for (int first = blockIdx.y * a.group; first < a.n_cols; first += gridDim.y * a.group) {
    const int n = min(a.group, a.n_cols - first);
    U v[NG];
#pragma unroll
    for (int c = 0; c < NG; ++c) {
      v[c] = U{};
      if (c >= n) continue;
      int p = __ldg(a.parent + first + c);
      if (in_place ? p >= first + n || (p >= 0 && p < first) : p >= a.n_src_cols) {
        if (a.err) atomicExch(a.err, kErrBadParent);
        p = in_place ? first + c : -1;
      }
      if (p >= 0) v[c] = src[p * pieces];
    }
#pragma unroll
    for (int c = 0; c < NG; ++c)
      if (c < n) dst[(first + c) * pieces] = v[c];
  }
}
template <class U, int NG>
cudaError_t reorder_launch(const BeamReorder& a, long long most, cudaStream_t st) {
  const long long groups = (a.n_cols + a.group - 1) / a.group;
  beam_reorder_kernel<U, NG><<<dim3((unsigned)((most / (long long)sizeof(U) + 127) / 128), (unsigned)std::min<long long>(groups, 32768), a.n_arrays), 128, 0, st>>>(a);
  return cudaGetLastError();
}
template <class U>
cudaError_t reorder_unit(const BeamReorder& a, long long most, cudaStream_t st) {
  if (a.group <= 4) return reorder_launch<U, 4>(a, most, st);
  if (a.group <= 16) return reorder_launch<U, 16>(a, most, st);
  if constexpr (sizeof(U) <= 4) return reorder_launch<U, 64>(a, most, st);
  return cudaErrorInvalidValue;
}

}  // namespace

namespace {

// A sentence's CTAs: as many as let all CTAs be resident at once (4 of 256 threads per multiprocessor, or one of 1024 where there are few
// sentences: what a multiprocessor has in flight bounds its share of the stream).  U: as many as leave a warp two segments.
void select_plan(int elem, int n_sent, int beam, int V, int k, SelectPlan* pl) {
  const int vec = 32 * 16 / elem_bytes(elem), sms = device_sms();
  auto segs = [&](int u) { return (long long)(V + 16 / elem_bytes(elem) - 2) / (vec * u) + 1; };
  int C = 1;
  pl->NT = (long long)n_sent * kSelCluster * 2 > sms * 4 ? 256 : 1024;
  const int slots = pl->NT == 256 ? 4 * sms : sms;
  while (C < kSelCluster && (long long)n_sent * 2 * C <= slots) C *= 2;
  while (C < kSelCluster && segs(4) * beam > (long long)C * kSelSegs) C *= 2;
  pl->parts = 1;
  pl->U = 4;
  if (segs(4) * beam > (long long)C * kSelSegs) {  // too long for a cluster
    pl->NT = 256;
    pl->segs_row = (int)segs(4);
    pl->n_seg = beam * pl->segs_row;
    // (a part with fewer than k segments would have no bound in step 1, and k candidates of each)
    const long long parts = std::max<long long>((pl->n_seg + kSelSegs - 1) / kSelSegs, std::min(4 * sms / n_sent, pl->n_seg / k));
    pl->per = (int)((pl->n_seg + parts - 1) / parts);
    pl->ctas = pl->parts = (pl->n_seg + pl->per - 1) / pl->per;
    return;
  }
  while (pl->U > 1 && segs(pl->U) * beam < 2ll * C * pl->NT / 32) pl->U /= 2;
  pl->segs_row = (int)segs(pl->U);
  pl->n_seg = beam * pl->segs_row;
  pl->ctas = C;
  pl->per = (pl->n_seg + C - 1) / C;
}
template <class T, int U, int NT>
cudaError_t select_launch(const BeamSelect& a, const SelectPlan& pl, cudaStream_t st) {
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(pl.ctas, a.n_sent);
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = (size_t)a.k * a.k * 8;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = pl.parts > 1 ? 1 : pl.ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  static bool configured[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(beam_select_kernel<T, U, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSelectMax * kSelectMax * 8);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  return cudaLaunchKernelEx(&cfg, beam_select_kernel<T, U, NT>, a, pl);
}
template <class T, int U>
cudaError_t select_threads(const BeamSelect& a, const SelectPlan& pl, cudaStream_t st) {
  return pl.NT == 256 ? select_launch<T, U, 256>(a, pl, st) : select_launch<T, U, 1024>(a, pl, st);
}
template <class T>
cudaError_t select_type(const BeamSelect& a, const SelectPlan& pl, cudaStream_t st) {
  return pl.U == 4 ? select_threads<T, 4>(a, pl, st) : pl.U == 2 ? select_threads<T, 2>(a, pl, st) : select_threads<T, 1>(a, pl, st);
}

}  // namespace

size_t beam_select_work(int elem, int n_sent, int beam, int V, int k) {
  SelectPlan pl;
  select_plan(elem, n_sent, beam, V, k, &pl);
  return pl.parts > 1 ? (size_t)n_sent * pl.parts * k * 8 : 0;
}
cudaError_t launch_beam_select(const BeamSelect& all, int elem, cudaStream_t st) {
  SelectPlan pl;
  select_plan(elem, all.n_sent, all.beam, all.V, all.k, &pl);
  constexpr int kMost = 65535;  // sentences of a launch
  for (int at = 0; at < all.n_sent; at += kMost) {
    BeamSelect a = all;
    const long long rows = (long long)at * a.beam, outs = (long long)at * a.k;
    a.n_sent = std::min(kMost, all.n_sent - at);
    a.logp = static_cast<const char*>(a.logp) + rows * a.ld * elem_bytes(elem);
    a.scores += rows;
    if (a.lse) a.lse += rows;
    if (a.done) a.done += rows;
    a.score_out += outs; a.word_out += outs; a.parent_out += outs;
    a.first_row = (int)rows;
    if (pl.parts > 1) a.work += outs * pl.parts;
    count_launch();
    cudaError_t e = elem == ELEM_F32 ? select_type<float>(a, pl, st) : elem == ELEM_BF16 ? select_type<__nv_bfloat16>(a, pl, st) : select_type<__half>(a, pl, st);
    if (e != cudaSuccess) return e;
    if (pl.parts == 1) continue;
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(a.n_sent);
    cfg.blockDim = dim3(kMergeThreads);
    cfg.dynamicSmemBytes = (size_t)(pl.parts * a.k <= kMergeKeys ? pl.parts * a.k * 8 : 0) + pl.parts;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    count_launch();
    e = cudaLaunchKernelEx(&cfg, beam_select_merge_kernel, a, pl.parts);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}
cudaError_t launch_beam_reorder(const BeamReorder& all, cudaStream_t st) {
  if (all.n_cols == 0 || all.n_arrays == 0) return cudaSuccess;
  BeamReorder a = all;
  uintptr_t bits = 0;
  long long most = 0;
  bool in_place = false;
  for (int i = 0; i < a.n_arrays; ++i) {
    bits |= (uintptr_t)a.src[i] | (uintptr_t)a.dst[i] | (uintptr_t)a.bytes[i];
    most = std::max(most, a.bytes[i]);
    in_place = in_place || a.src[i] == a.dst[i];
  }
  if (most == 0) return cudaSuccess;
  if (!in_place) a.group = 4;
  int unit = bits & 1 ? 1 : bits & 2 ? 2 : bits & 4 ? 4 : bits & 8 ? 8 : 16;
  if (a.group > 16) unit = std::min(unit, 4);  // (64 pieces in registers)
  count_launch();
  switch (unit) {
    case 16: return reorder_unit<uint4>(a, most, st);
    case 8: return reorder_unit<uint2>(a, most, st);
    case 4: return reorder_unit<unsigned>(a, most, st);
    case 2: return reorder_unit<unsigned short>(a, most, st);
  }
  return reorder_unit<unsigned char>(a, most, st);
}

}  // namespace zrnn
