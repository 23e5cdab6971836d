// Y = act(W X + bias) + R for more than a few columns, on tcgen05.
//
// A tile is 128 outputs (the M side: a lane of tensor memory per output, so that a warp stores 32 consecutive ones of a column) x nb columns, on one
// CTA; of 16-bit operands, where there are enough of them, 256 x nb on a pair of CTAs that share the MMAs and hold half of the columns' operand
// each (tc_pair_device.cuh).  One warp brings the k-blocks of 128 bytes by TMA, one issues the MMAs, sixteen take the accumulators
// through bias, activation and residual while the next tile's MMAs run; persistent.
//
// 32-bit operands go as two tf32 parts each and three products (hi hi; hi lo and lo hi into an accumulator of their own).  The tensor cores
// ignore the bits below tf32, so the outputs' tile that TMA brought is their hi part as it is; three teams of four warps make the rest of the stages
// (one team alone: a product took 1.7 times as long): the columns' hi, rounded, in the tile's place and lo beside it in shared memory, so that W's hi part is
// read once for both, the outputs' lo in tensor memory, which is an operand as well.  Rounding hi of one of the factors is what keeps the left-out lo lo
// without a side (linear_device.cuh); it costs 8 % (1000 x 2000 x 768: 23.6 us, with both cut off 21.9), lo lo as a fourth product 18 %.  A
// tensor-core accumulator cuts its sums off, so the products of four k-blocks (16 additions) go into a fresh pair, two pairs in turn, and the
// sixteen warps add those up in ordinary 32-bit arithmetic: sums of positive products come out 6e-7 of themselves too small (fresh pairs every two
// k-blocks: 2.2e-7, for 4 to 13 % more time).
// What bounds it is shared memory: per k-block of 128 x 96 the TMA writes, the splitting's reads and writes and the MMAs' reads are 132 KB,
// 1060 cycles at 128 bytes each, of 1110 measured (with both lo parts in shared memory, or with pairs of CTAs, 170 to 250 more), for MMAs of
// 580.
//
// Long products of few tiles: 2, 4 or 8 CTAs of a cluster share a tile's K axis and exchange their sums through distributed shared memory.
// 16-bit outputs and residuals of whole tiles go through shared memory and TMA.  us, this kernel / the library's product alone: bf16 16384 x
// 4096 x 4096 350 / 337, 4096 x 4096 x 512 18.5 / 15.2, 512 x 8192 x 512 18 / 17, 1000 x 1000 x 64 6.5 / 3.9; fp32 16384 x 4096 x 4096
// 2850 / 8400 (FMA), 1000 x 2000 x 768 23.6 / 83.
//
// A CTA asks for all of an SM's shared memory, so that a pair's allocation of tensor memory waits for nobody that could wait for it in turn.
#include <algorithm>
#include <cstdint>
#include <cstring>

#include "kernels.cuh"
#include "linear_device.cuh"
#include "operators.cuh"
#include "tc_pair_device.cuh"

namespace zrnn {
namespace {

enum { LIN_F32 = ELEM_F32, LIN_BF16 = ELEM_BF16, LIN_F16 = ELEM_F16 };
constexpr int kEpiWarps = 16, kLoadWarp = 16, kMmaWarp = 17, kSplitWarp0 = 18, kSplitWarps = 4, kSplitTeams = 3;
constexpr int kSmem = 227 * 1024, kMaxStages = 8, kRound = 4;  // kRound: k-blocks per fresh accumulator (32 bits)
static_assert(fills_sm(kSmem), "both CTAs of a pair hold all of the tensor memory");
__host__ __device__ constexpr int lin_threads(int mode) { return mode == LIN_F32 ? 32 * (kSplitWarp0 + kSplitTeams * kSplitWarps) : 32 * kSplitWarp0; }
__host__ __device__ constexpr int lin_max_nb(int mode, bool cut) { return mode == LIN_F32 ? 96 : cut ? 128 : 256; }
__host__ __device__ constexpr uint32_t lin_fmt(int mode) { return mode == LIN_BF16 ? 1u : mode == LIN_F16 ? 0u : 2u; }
struct LinParams {
  CUtensorMap w, x;  // boxes of 128 rows and of nb / CG columns
  CUtensorMap y, r;  // bulk: 128 outputs x nb columns
  int bulk;          // outputs and residual go through shared memory, as whole tiles
  LinearArgs a;
  int nb, n_ct, r_tiles, kb, stages;
  int cut_log2;  // 2^cut_log2 CTAs of a cluster share a tile's K axis (0: none; not with pairs)
};
struct alignas(16) LinCtrl {
  uint64_t full[kMaxStages], split[kMaxStages], empty[kMaxStages];
  uint64_t acc_full[2], acc_empty[2], res_full;
  uint32_t tmem_base;
  int abort;
};
template <int MODE> struct LinElem { using T = float; };
template <> struct LinElem<LIN_BF16> { using T = __nv_bfloat16; };
template <> struct LinElem<LIN_F16> { using T = __half; };

template <int CG>
__device__ __forceinline__ void lin_tma(void* dst, const CUtensorMap* map, uint32_t bar, int k, int row) {
  if constexpr (CG == 2)
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 :: "r"(smem_u32(dst)), "l"(map), "r"(bar), "r"(k), "r"(row) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 :: "r"(smem_u32(dst)), "l"(map), "r"(bar), "r"(k), "r"(row) : "memory");
}
template <int CG, int TF32>
__device__ __forceinline__ void lin_mma(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 2) umma_pair<TF32>(d, da, db, idesc, accumulate);
  else umma<TF32>(d, da, db, idesc, accumulate);
}
// the same with the outputs' operand in tensor memory (a: its first column there), tf32
__device__ __forceinline__ void lin_mma_ts(uint32_t d, uint32_t a, uint64_t db, uint32_t idesc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(db), "r"(idesc),
               "r"(1u)
               : "memory");
}
// a lane's 16 words into 16 columns of tensor memory
__device__ __forceinline__ void lin_tmem_st16(uint32_t at, const uint32_t (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
               "r"(v[13]), "r"(v[14]), "r"(v[15])
               : "memory");
}
template <int CG>
__device__ __forceinline__ void lin_commit(uint64_t* bar) {
  if constexpr (CG == 2) umma_commit_pair(bar);
  else umma_commit(bar);
}
// arrival on the leader's barrier (a CTA alone leads itself)
template <int CG>
__device__ __forceinline__ void lin_arrive(uint64_t* bar) {
  if constexpr (CG == 2) mbar_arrive_leader(bar);
  else mbar_arrive(bar);
}

template <int MODE, int CG, int ACT, bool CUT>
__global__ void __launch_bounds__(lin_threads(MODE), 1) linear_tc_kernel(const __grid_constant__ LinParams p) {
  using T = typename LinElem<MODE>::T;
  constexpr bool F32 = MODE == LIN_F32;
  constexpr int EPK = 128 / (int)sizeof(T), GROUPS = lin_max_nb(MODE, CUT) / 32;
  static_assert(CG == 1 || (!CUT && !F32), "a pair's tiles are of 16-bit operands and not cut");
  extern __shared__ __align__(1024) uint8_t lin_smem[];
  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  const int rank = CG == 2 ? (int)(blockIdx.x & 1) : 0, cut = CUT ? 1 << p.cut_log2 : 1, unit = blockIdx.x / CG >> (CUT ? p.cut_log2 : 0), n_units = gridDim.x / CG >> (CUT ? p.cut_log2 : 0);
  const int part = CUT ? (int)blockIdx.x & (cut - 1) : 0;
  const int kb0 = CUT ? (int)((long long)p.kb * part >> p.cut_log2) : 0, kb = CUT ? (int)((long long)p.kb * (part + 1) >> p.cut_log2) - kb0 : p.kb;  // this CTA's k-blocks
  const int nb = p.nb, x_rows = nb / CG, w_bytes = 128 * 128, x_bytes = x_rows * 128, raw = w_bytes + x_bytes, stage = raw + (F32 ? x_bytes : 0);
  // a stage: W, X; in 32 bits also X lo: X and its rest are one operand of twice the columns.  W lo lies in tensor memory, 32 columns per stage
  // behind the accumulators.
  const int acc = nb * (F32 ? 2 : 1);
  LinCtrl& ct = *reinterpret_cast<LinCtrl*>(lin_smem + (size_t)p.stages * stage);
  const int n_tiles = p.r_tiles * p.n_ct, rounds = F32 ? (kb + kRound - 1) / kRound : 1;
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&ct.full[s], 1);                       // the stage's bytes; the leader's, of both CTAs
      mbar_init(&ct.split[s], kSplitWarps);            // the lo parts are written
      mbar_init(&ct.empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&ct.acc_full[b], 1);
      mbar_init(&ct.acc_empty[b], CG * kEpiWarps);
    }
    mbar_init(&ct.res_full, 1);
    ct.abort = (smem_u32(lin_smem) & 1023) ? 1 : 0;
    if (ct.abort && p.a.err) atomicExch(p.a.err, 8);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    if constexpr (CG == 2) tmem_alloc_pair(&ct.tmem_base, 512);
    else lin_tmem_alloc(&ct.tmem_base, 512);
  }
  tc_fence_before();
  __syncthreads();
  if (CG == 2 || CUT) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = ct.tmem_base;
  const bool sound = __all_sync(0xffffffffu, ct.abort == 0);

  if (warp == kLoadWarp) {
    // ------------------------------------------------------------ loads
    const bool one = elect_one();
    bool ok = sound;
    int st = 0, it = 0;
    uint32_t ph = 0;
    for (int tile = unit; tile < n_tiles && ok; tile += n_units) {
      const int col = tile % p.n_ct * nb + rank * x_rows, row = (tile / p.n_ct * CG + rank) * 128;
      for (int k = kb0; k < kb0 + kb; ++k, ++it) {
        if (it >= p.stages && !mbar_wait_warp(&ct.empty[st], ph ^ 1u, &ct.abort, p.a.err, 1)) { ok = false; break; }
        uint8_t* dst = lin_smem + (size_t)st * stage;
        if (one) {
          const uint32_t bar = CG == 2 ? cluster_map(smem_u32(&ct.full[st]), 0) : smem_u32(&ct.full[st]);
          if (rank == 0) mbar_expect_tx(&ct.full[st], (uint32_t)(CG * raw));
          lin_tma<CG>(dst, &p.w, bar, k * EPK, row);
          lin_tma<CG>(dst + w_bytes, &p.x, bar, k * EPK, col);
        }
        __syncwarp();
        if (++st == p.stages) { st = 0; ph ^= 1u; }
      }
    }
    if (sound && !ok) settle_copies();
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------ MMAs
    if (rank == 0 && sound) {
      const bool one = elect_one();
      const uint32_t idesc = CG == 2 ? make_idesc_pair(lin_fmt(MODE), (uint32_t)nb) : make_idesc(lin_fmt(MODE), (uint32_t)nb);
      const uint32_t w_lo = tmem_base + 2u * acc;
      const uint32_t idesc2 = make_idesc(lin_fmt(MODE), 2u * nb);
      int st = 0, use = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int tile = unit; tile < n_tiles && ok; tile += n_units) {
        uint32_t d = 0;
        for (int k = 0; k < kb; ++k) {
          const bool fresh = F32 ? k % kRound == 0 : k == 0;
          if (fresh) {
            if (!mbar_wait_warp(&ct.acc_empty[use & 1], (uint32_t)(((use >> 1) & 1) ^ 1), &ct.abort, p.a.err, 4)) { ok = false; break; }
            d = tmem_base + (uint32_t)((use & 1) * acc);
          }
          if (!mbar_wait_warp(F32 ? &ct.split[st] : &ct.full[st], ph, &ct.abort, p.a.err, 2)) { ok = false; break; }
          tc_fence_after();
          const uint32_t w_addr = smem_u32(lin_smem + (size_t)st * stage), x_addr = w_addr + w_bytes;
          const uint64_t dw = make_smem_desc(w_addr), dx = make_smem_desc(x_addr);
          if (one) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t more = !fresh || i > 0 ? 1u : 0u;
              if constexpr (F32) {  // hi times [hi lo] of the columns, twice as wide; lo times hi
                lin_mma<CG, 1>(d, dw + 2 * i, dx + 2 * i, idesc2, more);
                lin_mma_ts(d + nb, w_lo + (uint32_t)(32 * st + 8 * i), dx + 2 * i, idesc);
              } else {
                lin_mma<CG, 0>(d, dw + 2 * i, dx + 2 * i, idesc, more);
              }
            }
            lin_commit<CG>(&ct.empty[st]);
          }
          __syncwarp();
          if (++st == p.stages) { st = 0; ph ^= 1u; }
          if (F32 ? (k % kRound == kRound - 1 || k == kb - 1) : k == kb - 1) {
            if (one) lin_commit<CG>(&ct.acc_full[use & 1]);
            __syncwarp();
            ++use;
          }
        }
      }
      if (!ok) settle_copies();
    }
  } else if (warp < kEpiWarps) {
    // ------------------------------------------------------------ epilogue: outputs 32 quad .. +31 of the CTA's 128, every fourth group of 8 columns
    const int quad = warp & 3, cg = warp >> 2;
    const LinearArgs& a = p.a;
    int use = 0;
    bool ready = sound;
    // bulk: one thread brings a tile's residual and takes its outputs away; both lie at `out`, 128 outputs per column
    constexpr bool BULK = !F32 && !CUT;
    T* out = reinterpret_cast<T*>(lin_smem + (size_t)p.stages * stage + ((sizeof(LinCtrl) + 127) / 128) * 128);
    const bool one = BULK && threadIdx.x == 0;
    uint32_t res_ph = 0;
    auto bring_residual = [&](int tile) {
      const int row = (tile / p.n_ct * CG + rank) * 128;
      if (tile >= n_tiles || row >= a.n) return;
      mbar_expect_tx(&ct.res_full, (uint32_t)(128 * nb * sizeof(T)));
      tma_load_2d(out, &p.r, &ct.res_full, row, tile % p.n_ct * nb);
    };
    if (BULK && p.bulk && a.R && one && sound) bring_residual(unit);
    for (int tile = unit; tile < n_tiles && (ready || CUT || (BULK && p.bulk)); tile += n_units) {  // (to the end even after a wait that gave up: barriers)
      const int col = tile % p.n_ct * nb, cols = min(nb, a.N - col), i = (tile / p.n_ct * CG + rank) * 128 + quad * 32 + lane;
      const bool in = i < a.n;
      const float bias = in && a.bias ? __ldg(a.bias + i) : 0.f;
      float z[GROUPS][8];
      const uint32_t lanes = tmem_base + ((uint32_t)(quad * 32) << 16) + 8u * cg;
      for (int r = 0; r < rounds && ready; ++r, ++use) {
        ready = __all_sync(0xffffffffu, mbar_wait(&ct.acc_full[use & 1], (uint32_t)((use >> 1) & 1), &ct.abort, a.err, 3));
        if (!ready) break;
        tc_fence_after();
        const uint32_t at = lanes + (uint32_t)((use & 1) * acc);
        if (!F32) {
#pragma unroll
          for (int j = 0; j < GROUPS; ++j)
            if (32 * j + 8 * cg < nb) tmem_ld8(at + 32 * j, z[j]);
          tmem_wait_ld();
        } else {  // this round's sums and, beside them, the cross products
#pragma unroll
          for (int j = 0; j < GROUPS; ++j) {
            if (32 * j + 8 * cg < nb) {
              float y[2][8];
              tmem_ld8(at + 32 * j, y[0]);
              tmem_ld8(at + nb + 32 * j, y[1]);
              tmem_wait_ld();
#pragma unroll
              for (int u = 0; u < 8; ++u) z[j][u] = r == 0 ? y[0][u] + y[1][u] : z[j][u] + (y[0][u] + y[1][u]);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) lin_arrive<CG>(&ct.acc_empty[use & 1]);
      }
      if (CUT) {
        // The CTAs of the cluster each finish every cut-th group of 8 columns: the other ones' sums of it go into that CTA's shared memory, where
        // the operands were (one tile per cluster), and are added to its own in the order of the CTAs.
        __syncwarp();
        cluster_sync_all();  // all MMAs of all of them are over
        const int per = (nb / 8 + cut - 1) >> p.cut_log2;
        auto slot = [&](int from, int group) { return (uint32_t)((((from * 4 + quad) * per + (group >> p.cut_log2)) * 64 + lane) * 16); };
        if (ready) {
#pragma unroll
          for (int j = 0; j < GROUPS; ++j) {
            const int group = cg * (nb / 32) + j, to = group & (cut - 1);  // (a warp's groups go to different CTAs)
            if (32 * j >= nb || to == part) continue;
            const uint32_t at = cluster_map(smem_u32(lin_smem) + slot(part, group), (uint32_t)to);
            st_cluster_v4(at, z[j][0], z[j][1], z[j][2], z[j][3]);
            st_cluster_v4(at + 512, z[j][4], z[j][5], z[j][6], z[j][7]);
          }
        }
        __syncwarp();
        cluster_sync_all();
        if (ready) {
#pragma unroll
          for (int j = 0; j < GROUPS; ++j) {
            const int group = cg * (nb / 32) + j;
            if (32 * j >= nb || (group & (cut - 1)) != part) continue;
            for (int from = 0; from < cut; ++from) {
              if (from == part) continue;
              const float4* got = reinterpret_cast<const float4*>(lin_smem + slot(from, group));
              const float4 lo = got[0], hi = got[32];
              z[j][0] += lo.x; z[j][1] += lo.y; z[j][2] += lo.z; z[j][3] += lo.w;
              z[j][4] += hi.x; z[j][5] += hi.y; z[j][6] += hi.z; z[j][7] += hi.w;
            }
          }
        }
      }
      if (BULK && p.bulk) {
        const int row = (tile / p.n_ct * CG + rank) * 128;
        if (row < a.n) {  // (the same for the whole CTA)
          if (a.R && ready) {
            ready = __all_sync(0xffffffffu, mbar_wait(&ct.res_full, res_ph, &ct.abort, a.err, 7));
            res_ph ^= 1u;
          }
          T* o = out + quad * 32 + lane;
#pragma unroll
          for (int j = 0; j < GROUPS; ++j) {
            const int c0 = 32 * j + 8 * cg;
            if (c0 >= nb || !ready) break;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              float v = linear_act(z[j][u] + bias, ACT);
              if (a.R) v += to_f32(o[(c0 + u) * 128]);
              o[(c0 + u) * 128] = from_f32<T>(v);
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          asm volatile("bar.sync 1, %0;" ::"n"(kEpiWarps * 32) : "memory");
          if (one && ready) {
            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(&p.y), "r"(smem_u32(out)), "r"(row), "r"(col) : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            if (a.R) bring_residual(tile + n_units);
          }
          asm volatile("bar.sync 1, %0;" ::"n"(kEpiWarps * 32) : "memory");  // the tile's place is free again
        }
        continue;
      }
      if (!ready) break;
      if (in) {
#pragma unroll
        for (int j = 0; j < GROUPS; ++j) {
          const int c0 = 32 * j + 8 * cg;
          if (c0 >= cols) break;
          if (CUT && ((cg * (nb / 32) + j) & (cut - 1)) != part) continue;
          const long long c = col + c0;
          T* y = static_cast<T*>(a.Y) + c * a.ldy + i;
          const T* res = static_cast<const T*>(a.R) + c * a.ldr + i;
          float rv[8];
          if (a.R) {
#pragma unroll
            for (int u = 0; u < 8; ++u) rv[u] = c0 + u < cols ? to_f32(res[u * a.ldr]) : 0.f;
          }
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            float v = linear_act(z[j][u] + bias, ACT);
            if (a.R) v += rv[u];
            if (c0 + u < cols) y[u * a.ldy] = from_f32<T>(v);
          }
        }
      }
      __syncwarp();
    }
    if (BULK && p.bulk && one) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    if (BULK && p.bulk && a.R && one && sound && !ready) settle_copies();  // (a residual may still be on its way)
  } else if (F32) {
    // ------------------------------------------------------------ the lo parts of a stage: what tf32 cuts off of the tile beside it
    // Teams of four warps take the k-blocks in turn: one's waits are filled by the others.  A stage's next user may be another team, and copies may arrive out
    // of order: a team waits until the MMAs have used up the stage's last round before it asks for its own copy.  (While that copy ahead is still on its way,
    // the barrier would answer the question for the next one's parity with yes.  The round before that is used up: the team has seen the copy
    // of kSplitTeams k-blocks ago, and copies are requested in order, the stage's last one when the round before it was used up.)
    const int team = (warp - kSplitWarp0) / kSplitWarps, me = (warp - kSplitWarp0) % kSplitWarps * 32 + lane;
    const int wv = w_bytes / 16, xv = x_bytes / 16, row = 32 * (warp & 3) + lane;  // (a warp reaches the lanes of tensor memory that its number gives)
    const uint32_t w_lo = tmem_base + 2u * acc + ((uint32_t)(row & ~31) << 16);
    long long its = 0;
    for (int tile = unit; tile < n_tiles; tile += n_units) its += kb;
    int st = team % p.stages;
    uint32_t ph = (uint32_t)(team / p.stages) & 1u;
    for (long long it = team; it < its && sound; it += kSplitTeams) {
      if (!mbar_wait_warp(&ct.empty[st], ph ^ 1u, &ct.abort, p.a.err, 6)) break;
      if (!mbar_wait_warp(&ct.full[st], ph, &ct.abort, p.a.err, 6)) break;
      uint4* tiles = reinterpret_cast<uint4*>(lin_smem + (size_t)st * stage);
      tc_fence_after();
#pragma unroll
      for (int half = 0; half < 2; ++half) {  // a lane has a row; piece q of it lies at q ^ (row % 8)
        uint32_t lo[16];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint4 x = tiles[row * 8 + ((4 * half + q) ^ (row & 7))];
          lo[4 * q] = tf32_rest(x.x); lo[4 * q + 1] = tf32_rest(x.y); lo[4 * q + 2] = tf32_rest(x.z); lo[4 * q + 3] = tf32_rest(x.w);
        }
        lin_tmem_st16(w_lo + (uint32_t)(32 * st + 16 * half), lo);
      }
#pragma unroll 2
      for (int e = wv + me; e < wv + xv; e += kSplitWarps * 32) {
        const uint4 x = tiles[e];
        uint4 hi, lo;
        split_tf32(x.x, hi.x, lo.x); split_tf32(x.y, hi.y, lo.y); split_tf32(x.z, hi.z, lo.z); split_tf32(x.w, hi.w, lo.w);
        tiles[e] = hi;
        tiles[xv + e] = lo;
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ct.split[st]);
      st += kSplitTeams;
      while (st >= p.stages) { st -= p.stages; ph ^= 1u; }
    }
  }
  __syncwarp();
  if (CUT && warp >= kEpiWarps) {  // (the epilogue's two cluster barriers are everybody's)
    cluster_sync_all();
    cluster_sync_all();
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync_all();  // neither CTA ends while the other one's MMAs read its tiles or its arrivals come in
  if (warp == kMmaWarp) {
    tc_fence_after();
    if constexpr (CG == 2) tmem_free_pair(tmem_base, 512);
    else lin_tmem_free(tmem_base, 512);
  }
}

// Rows that no 16-byte copy can start at, moved to where one can: 16 bytes of the new row per thread, from the words that hold them
template <class T>
__global__ void __launch_bounds__(256) linear_align_kernel(const T* src, long long ld, int rows, int K, T* dst, long long ld_dst) {
  constexpr int V = 16 / (int)sizeof(T);
  const int vecs = (K + V - 1) / V, lanes = min(vecs, 256), per = 256 / lanes, lane = threadIdx.x % lanes, sub = threadIdx.x / lanes;
  if (sub >= per) return;
  for (long long r = (long long)blockIdx.x * per + sub; r < rows; r += (long long)gridDim.x * per)
    for (int q = blockIdx.y * lanes + lane; q < vecs; q += gridDim.y * lanes)
      reinterpret_cast<uint4*>(dst + r * ld_dst)[q] = load16<T, false>(src + r * ld, q * V, K, true);
}

struct LinPlan {
  bool few;
  int cg, nb, n_ct, cut;
  bool align_w, align_x;
  long long ld_pad;         // elements of a row that was moved
  size_t w_bytes, x_bytes;  // of the workspace
};
LinPlan lin_plan(const LinearArgs& a, int elem) {
  LinPlan pl;
  std::memset(&pl, 0, sizeof(pl));
  const int eb = elem_bytes(elem), sms = device_sms(), kb = (a.K * eb + 127) / 128;
  const long long rows1 = (a.n + 127) / 128, rows2 = (a.n + 255) / 256;
  // The time of a launch in ns, as measured with all multiprocessors at work: a start and an end (4 us, with a cut 6), and for the busiest unit's
  // tiles the k-blocks or the epilogue, whichever takes longer.  A k-block of 16-bit operands takes a pair the MMAs' time, a CTA that of
  // its shared memory (450 ns with 224 columns), but no less than 200 ns (its way from the L2); of 32 bits what shared memory lets through: 583 ns
  // with 96 columns, 3.5 less per column (a pair, with twice the rows on two multiprocessors, took some 90 ns more than a CTA, so there are none).
  double best = 0;
  const bool f32 = elem == ELEM_F32;
  for (int cg = 1; cg <= (f32 ? 1 : 2); ++cg)
    for (int w = lin_max_nb(elem, false); w >= 32; w -= 32) {
      const int n_ct = (a.N - 1) / w + 1, nb = ((a.N - 1) / n_ct + 32) / 32 * 32;
      if ((long long)nb * (n_ct - 1) >= a.N) continue;
      const long long tiles = (cg == 2 ? rows2 : rows1) * n_ct;
      const double block = f32 ? 250 + 3.5 * nb : cg == 2 ? std::max(200.0, 1.1 * nb) : std::max(200.0, 140 + 1.4 * nb), end = 14.0 * nb;
      for (int cut = 1; cut <= 8; cut *= 2) {
        if (cut > 1 && (cg == 2 || kb < 4 * cut || nb / 8 < cut || nb > lin_max_nb(elem, true))) break;
        // clusters of 4 and 8 CTAs that take whole multiprocessors do not fill the processing clusters: 33 and 15 of them on 148
        const long long units = cut == 1 ? sms / cg : cut == 2 ? sms / 2 : cut == 4 ? sms * 33 / 148 : sms * 15 / 148, waves = (tiles + units - 1) / units;
        if (cut > 1 && waves > 1) break;
        const double cost = waves * std::max(block * ((kb + cut - 1) / cut), end) + end / cut + (cut > 1 ? 6000 : 4000);
        if (pl.nb == 0 || cost < best) {
          best = cost;
          pl.cg = cg; pl.nb = nb; pl.n_ct = n_ct; pl.cut = cut;
        }
      }
    }
  const auto off16 = [&](const void* p, long long ld) { return ((uintptr_t)p & 15) != 0 || (ld * eb) % 16 != 0; };
  pl.align_w = off16(a.W, a.ldw);
  pl.align_x = off16(a.X, a.ldx);
  if (pl.align_w) best += 2000 + (double)a.n * a.K * eb / 3000;
  if (pl.align_x) best += 2000 + (double)a.N * a.K * eb / 3000;
  // The kernel for few columns: 2.7 us, and per chunk of a warp (64 bytes of K) its latency or its share of a multiprocessor that has many CTAs (both
  // in ns, with tiles of 8, 16 and 32 columns), 1.6 times that, in 16 bits 2.3 times, on rows that would have to be moved first.  Up to 8
  // columns it is ahead, up to 32 with few weights or such rows (us, few / tcgen05: fp32 4000 x 1001 x 20 11.7 / 15.8, 212 x 559 x 1668
  // 27 / 14, 1000 x 1000 x 48 7.1 / 8.8; bf16 4000 x 1001 x 20 8.8 / 12.1, 1000 x 2001 x 40 15.5 / 12.0, 512 x 512 x 64 3.9 / 5.6).
  static const double lat[2][3] = {{300, 460, 550}, {270, 460, 840}}, thr[2][3] = {{232, 390, 520}, {154, 230, 380}};
  const int t = a.N <= 8 ? 0 : a.N <= 16 ? 1 : 2, cols = 8 << t;
  const int shared = few_cut(a.n, a.N, a.K, eb);
  const double ctas = (double)((a.n + 15) / 16) * ((a.N + cols - 1) / cols) * shared, chunks = (((long long)a.K * eb + 63) / 64 + 8 * shared - 1) / (8 * shared);
  const double anywhere = !(pl.align_w || pl.align_x || a.K * eb % 16) ? 1.0 : f32 ? 1.6 : 2.3;
  pl.few = 2700 + (shared > 1 ? 1500 : 0) + anywhere * chunks * std::max(lat[!f32][t], thr[!f32][t] * ctas / sms) <= best;
  if (pl.few) {
    pl.align_w = pl.align_x = false;
    return pl;
  }
  pl.ld_pad = (a.K * eb + 15) / 16 * 16 / eb;
  const auto whole = [](size_t b) { return (b + 255) / 256 * 256; };
  pl.w_bytes = pl.align_w ? whole((size_t)a.n * pl.ld_pad * eb) : 0;
  pl.x_bytes = pl.align_x ? whole((size_t)a.N * pl.ld_pad * eb) : 0;
  return pl;
}

template <int MODE, int CG, int ACT, bool CUT>
cudaError_t lin_launch(LinParams& p, cudaStream_t st) {
  const int raw = (128 + p.nb / CG) * 128, stage = raw + (MODE == LIN_F32 ? p.nb * 128 : 0);
  const int out = p.bulk ? 128 * p.nb * 2 : 0;
  p.stages = std::min((kSmem - ((int)sizeof(LinCtrl) + 127) / 128 * 128 - out) / stage, (int)kMaxStages);
  if (MODE == LIN_F32) p.stages = std::min(p.stages, (512 - 4 * p.nb) / 32);  // (what the accumulators leave of tensor memory)
  static bool configured[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(linear_tc_kernel<MODE, CG, ACT, CUT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)((CG << p.cut_log2) * std::min<long long>((long long)p.r_tiles * p.n_ct, CUT ? (1ll << 30) : device_sms() / CG)));
  cfg.blockDim = dim3(lin_threads(MODE));
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CG << p.cut_log2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CG == 2 || CUT ? 1 : 0;
  count_launch();
  return cudaLaunchKernelEx(&cfg, linear_tc_kernel<MODE, CG, ACT, CUT>, p);
}
template <int MODE, int CG, bool CUT>
cudaError_t lin_act(LinParams& p, cudaStream_t st) {
  switch (p.a.act) {
    case ACT_TANH: return lin_launch<MODE, CG, ACT_TANH, CUT>(p, st);
    case ACT_SIGMOID: return lin_launch<MODE, CG, ACT_SIGMOID, CUT>(p, st);
    case ACT_RELU: return lin_launch<MODE, CG, ACT_RELU, CUT>(p, st);
    case ACT_GELU: return lin_launch<MODE, CG, ACT_GELU, CUT>(p, st);
    case ACT_SILU: return lin_launch<MODE, CG, ACT_SILU, CUT>(p, st);
  }
  return lin_launch<MODE, CG, ACT_NONE, CUT>(p, st);
}
template <int MODE>
cudaError_t lin_type(const LinearArgs& all, const LinPlan& pl, cudaStream_t st) {
  using T = typename LinElem<MODE>::T;
  LinParams p;
  std::memset(&p, 0, sizeof(p));
  p.a = all;
  char* work = static_cast<char*>(all.work);
  const auto move = [&](const void* src, long long ld, int rows, char* dst) {
    count_launch();
    const int vecs = (int)((all.K * (long long)sizeof(T) + 15) / 16), lanes = std::min(vecs, 256), per = 256 / lanes;
    linear_align_kernel<T><<<dim3((unsigned)std::min((rows + per - 1) / per, 16 * device_sms()), (unsigned)((vecs + lanes - 1) / lanes)), 256, 0, st>>>(
        static_cast<const T*>(src), ld, rows, all.K, reinterpret_cast<T*>(dst), pl.ld_pad);
    return cudaGetLastError();
  };
  if (pl.align_w) {
    const cudaError_t e = move(all.W, all.ldw, all.n, work);
    if (e != cudaSuccess) return e;
    p.a.W = work;
    p.a.ldw = pl.ld_pad;
  }
  if (pl.align_x) {
    const cudaError_t e = move(all.X, all.ldx, all.N, work + pl.w_bytes);
    if (e != cudaSuccess) return e;
    p.a.X = work + pl.w_bytes;
    p.a.ldx = pl.ld_pad;
  }
  p.nb = pl.nb;
  p.n_ct = pl.n_ct;
  while (1 << p.cut_log2 < pl.cut) ++p.cut_log2;
  p.r_tiles = (all.n + 128 * pl.cg - 1) / (128 * pl.cg);
  p.kb = (int)((all.K * (long long)sizeof(T) + 127) / 128);
  // Whole tiles of 16-bit outputs through shared memory, where TMA can address them and the residual and the product is no shorter than a ring:
  // with stores of 64 bytes per warp and a residual that a warp waits for, 8192 x 2048 x 16384 took 574 us.
  p.bulk = sizeof(T) == 2 && pl.cut == 1 && p.kb >= 8 && make_plain_map(&p.y, all.Y, 2, all.n, all.N, all.ldy, 128, pl.nb) &&
           (!all.R || make_plain_map(&p.r, all.R, 2, all.n, all.N, all.ldr, 128, pl.nb));
  if (!make_kmajor_map(&p.w, p.a.W, sizeof(T), all.K, all.n, p.a.ldw, 128) || !make_kmajor_map(&p.x, p.a.X, sizeof(T), all.K, all.N, p.a.ldx, pl.nb / pl.cg))
    return cudaErrorInvalidValue;
  if constexpr (MODE != LIN_F32)
    if (pl.cg == 2) return lin_act<MODE, 2, false>(p, st);
  return pl.cut > 1 ? lin_act<MODE, 1, true>(p, st) : lin_act<MODE, 1, false>(p, st);
}

}  // namespace

size_t linear_work(const LinearArgs& a, int elem) {
  const LinPlan pl = lin_plan(a, elem);
  return pl.w_bytes + pl.x_bytes;
}
cudaError_t launch_linear(const LinearArgs& a, int elem, cudaStream_t st) {
  if (a.n == 0 || a.N == 0) return cudaSuccess;
  const LinPlan pl = lin_plan(a, elem);
  if (pl.few) return launch_linear_few(a, elem, st);
  switch (elem) {
    case ELEM_F32: return lin_type<LIN_F32>(a, pl, st);
    case ELEM_BF16: return lin_type<LIN_BF16>(a, pl, st);
  }
  return lin_type<LIN_F16>(a, pl, st);
}

}  // namespace zrnn
