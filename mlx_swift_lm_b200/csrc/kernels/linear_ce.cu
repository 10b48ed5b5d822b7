// Softmax cross entropy of a linear head, without the logits:
//
//   u = h . W^T,  z = cap > 0 ? cap * tanh(u / cap) : u          (T x V, never stored)
//   d = log sum_{v != y} exp z_v - z_y,  loss = log(1 + exp d)
//   G[t, v] = dloss_t * (p_v - [v = y]) * dz/du,  p_v = exp(z_v - lse), lse = log sum exp z
//   (dloss_t in dh and dW instead where it is the same for all t)
//   dh = G . W,  dW = G^T . h
//
// The target's logit stands apart from the sum over the others, so a loss near
// zero (and p_y - 1 = expm1(-loss)) keeps its digits. It is a dot product in
// fp32 of its own; the others come from the tensor cores, in chunks (kChunk).
//
// Forward: one product whose tiles leave a (max, sum of exp) pair per row and
// 256 columns. Backward: the vocabulary in pieces; each forms its logits again
// and turns them into G in bf16 (at most 2^-8 of each entry, as any bf16 product
// of gradients rounds its operands), which two products with fp32 accumulators
// contract with W and h. So the work is 2 T V K forward and 6 backward, 4 of
// them the gradients' own; the memory is one piece of G.
//
// Only scored rows take part: they are gathered first (stable order) and their
// count stays on the device, so padding costs nothing and whatever ignored rows
// hold (NaN included) reaches no gradient.
//
// One kernel does the four products (Op): persistent pairs of CTAs on neighbouring
// SMs walk 256 x 256 output tiles (tcgen05.mma.cta_group::2: each CTA holds half of
// either operand's rows and half of the accumulator's). Per CTA, warp 0 fetches its
// operand halves by TMA into a ring of 64-deep stages, one thread of the pair issues
// the MMAs into one of two accumulators in tensor memory (2 x 256 columns), and warps
// 4 - 11 work on the other one's finished tile, half a row of it per thread: the softmax
// arithmetic and the stores run under the next tile's product. Tiles leave through
// shared memory by TMA; the fp32 sums of dh are added up in L2 by its reduction.
//
// Bound by the tensor cores and, in a loop, by the power cap that slows their clock.
// 4096 rows, 32768 x 4096 head, single passes: statistics 745 us, G 757, dh 724, dW 754
// (1.45 - 1.52 PFLOP/s); 151936 x 4096 head: 14.7 - 15.9 ms in all when repeated (1.28 -
// 1.39 PFLOP/s over the four products). With one CTA per 128 x 256 tile and stores from
// registers the step took 21.8 ms (dW's part alone 10).
#include "b200_common.cuh"
#include "b200_train.h"

namespace b200 {

bool make_tmap_2d(CUtensorMap* out, const void* ptr, int64_t rows, int64_t cols, int64_t ld_elems, int box_rows,
                  int box_cols, int dtype_bytes);

namespace lce {

constexpr float kLog2e = 1.4426950408889634f;

enum Op : int {
  kStats = 0,  // A = h rows, B = W rows; out: (max, sum exp) of each row's 256 columns
  kGrad = 1,   // A = h rows, B = W rows of a piece; out: G
  kDh = 2,     // A = G (vocabulary inner), B = W columns; out: fp32 dh, added piece by piece
  kDw = 3,     // A = G columns, B = h columns (rows contracted); out: bf16 dW
};

struct Args {
  const int* count;      // [1] scored rows n
  const int* target;     // [T] target of each scored row (-1: out of range)
  const int* token;      // [T] the scored row's index in the batch
  const float* zt;       // [T] target logits (capped)
  const float* loss;     // [T] losses of the scored rows
  const float* lse;      // [T] logarithms of their sums of exp
  const float* dloss;    // incoming gradient, element token * dloss_stride
  int64_t dloss_stride;
  int mean;              // dloss is of the mean: divide by n
  const float* lost;     // kDw: [T][Kp] sums of what the targets' entries of G lost, times h
  const int* lost_of;    // kDw: [V] their rows, by vocabulary row
  int Kp;
  float2* part;          // kStats: [tiles of 256 columns][T]
  int acc_rows;          // kDh: rows of one part of the fp32 sums (whole half tiles, so that none reaches into the next)
  int T, V, K;
  int v0, nv;            // the piece's first column and columns
  int piece, pairs;      // kDh: columns of a whole piece and CTA pairs (choose_parts)
  int most_parts, first;  // kDh: parts the sums have room for; first piece stores, others add
  float cap, inv_cap;    // cap 0: none
};

constexpr int kTileM = 256, kTileN = 256, kStages = 6;  // of a pair of CTAs
constexpr int kRowsM = kTileM / 2, kRowsN = kTileN / 2;   // a CTA's share of either operand
constexpr int kABytes = kRowsM * 128, kBBytes = kRowsN * 128, kStageBytes = kABytes + kBBytes;
constexpr int kOutBytes = kRowsM * 128;  // a staging buffer for each half of the columns: 128 rows of 128 bytes
constexpr int kBars = 2 * kStages + 4;
constexpr int kBarOffset = kStages * kStageBytes + 2 * kOutBytes;
constexpr int kSmem = kBarOffset + kBars * 8 + 16 + 1024;  // kStats keeps its pairs in the staging buffers
constexpr int kThreads = 384;
// Epilogue: two warps for each quarter of the lanes, one for the left half of the columns, one for
// the right (with four warps the capped G of 901 x 50257 x 2560 took 312 us for 254).
constexpr int kEpiWarps = 8;
constexpr int kHalfN = kTileN / 2;
constexpr int kGroupM = 16;  // row tiles walked per column tile before the next: W is read once per 16 x 256 rows, h stays in L2
static_assert(kSmem <= 227 * 1024, "shared memory plan exceeds the per-CTA limit");

// The tensor cores add each 16-deep step into the fp32 accumulator by truncation, so a sum
// comes out too small by up to half a step of what it had reached, each time: without more the
// loss of logits up to 20 at K = 4096 is off by 6.7e-6 on normal operands and 2.9e-4 where all
// products are positive (fp32 sums rounded to nearest: 9e-7 and 2e-5), and not at all where the
// sums are exact. So the logits are summed a chunk of blocks of 64 at a time, and the chunks
// added up, rounded to nearest, in the registers of the epilogue's threads, half a row of a
// tile each. Reading the accumulators more often costs the products their time: statistics of
// 512 rows of 151936 x 4096 457 us in one chunk, 472 in chunks 1024 deep, 490 in 512 (which
// brings the errors to those of rounded sums), 540 in 256. G is rounded to bf16: 1024 there
// (a full step of 4096 rows 14.9 ms in one chunk, 15.5 as it is, 15.8 with 512 for both).
template <int OP>
constexpr int kChunk = OP == 0 ? 8 : OP == 1 ? 16 : 1 << 30;  // kStats, kGrad; the others' results are rounded to bf16
// Those threads need more registers than 168, the share of 384: the other four warps give some of
// theirs (what is left to spill are 28 - 32 bytes a thread).
constexpr int kRegsMax = 168, kRegsRest = 56, kRegsEpi = 224;
static_assert(128 * kRegsRest + 256 * kRegsEpi <= kThreads * kRegsMax, "more registers than the block is launched with");

// --- tcgen05 on a pair of CTAs ---
__device__ __forceinline__ void tmem_alloc2(uint32_t dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tmem_relinquish2() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc2(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void mma2_f16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrive on the barrier at this shared-memory offset in both CTAs once all MMAs issued so far are complete.
__device__ __forceinline__ void commit2(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"((uint16_t)3)
      : "memory");
}
// Address of a shared-memory variable of the pair's first CTA.
__device__ __forceinline__ uint32_t in_leader(uint32_t addr) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void arrive_cluster(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
// Load into this CTA's shared memory, counted on a barrier of the pair's first CTA.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* m, uint32_t cluster_bar, int c0, int c1,
                                              uint64_t hint) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%2, %3}], [%4], %5;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(c0), "r"(c1), "r"(cluster_bar), "l"(hint)
      : "memory");
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// --- tiles to global memory ---
__device__ __forceinline__ void tma_store(const CUtensorMap* m, uint32_t src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(m)),
               "r"(src), "r"(c0), "r"(c1)
               : "memory");
}
__device__ __forceinline__ void tma_add_f32(const CUtensorMap* m, uint32_t src, int c0, int c1) {
  asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(m)),
               "r"(src), "r"(c0), "r"(c1)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
// Barrier of the four warps of one half of the columns (ids 1 and 2), and of all eight (3).
__device__ __forceinline__ void half_barrier(int half) { asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory"); }
__device__ __forceinline__ void epi_barrier() { asm volatile("bar.sync 3, %0;" ::"n"(32 * kEpiWarps) : "memory"); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Parts of dh's contraction of `kb` blocks of 64 over `tiles` output tiles: the
// fewest that minimise the rounds of the CTA pairs times their length, so that few
// rows still fill the machine and the last round is not half empty. A part's tile
// costs about kPartBlocks blocks on its way out, and its fp32 sums are written and
// read once (512 KB a tile at 5 TB/s are kPartTraffic of the 0.37 us of a block).
// Chosen on the device, where the number of scored rows is known, by a whole warp: a
// lane weighs two of the at most kMostParts choices.
constexpr int kPartBlocks = 6, kMostParts = 64;
constexpr float kPartTraffic = 0.28f;
__device__ __forceinline__ int choose_parts(int tiles, int kb, int pairs, int most) {
  unsigned best = 0xFFFFFFFFu;
#pragma unroll
  for (int i = 0; i < kMostParts / 32; ++i) {
    const int s = (threadIdx.x & 31) + 32 * i + 1;
    if (s <= most && (s == 1 || kb >= 16 * s)) {
      const float rounds = ceilf((float)tiles * (float)s / (float)pairs);
      const float cost = rounds * (float)((kb + s - 1) / s + kPartBlocks) + kPartTraffic * (float)tiles * (float)s;
      best = min(best, (unsigned)fminf(cost, 6e7f) * kMostParts + (unsigned)(s - 1));  // the fewer win a tie
    }
  }
  return (int)(__reduce_min_sync(0xffffffffu, best) % kMostParts) + 1;
}

// 1 - 2 / (1 + e^2x): off by at most 2^-22 of one; 5 instructions for tanhf's 20 or so. The cap
// multiplies that error in the exponent of G's entries, which are rounded to bf16 (2^-8 at
// most): up to kFastTanhCap it stays below 2^-14 of an entry. Larger caps and the losses take
// tanhf, whose error is relative.
constexpr float kFastTanhCap = 256.f;
__device__ __forceinline__ float tanh_fast(float x) {
  return 1.f - __fdividef(2.f, 1.f + ex2(2.f * kLog2e * x));
}

// (max, sum of exp) of two sets of logits as one.
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2);
  if (top > -INFINITY) {
    s = s * (m > -INFINITY ? ex2((m - top) * kLog2e) : 1.f) + s2 * (m2 > -INFINITY ? ex2((m2 - top) * kLog2e) : 1.f);
    m = top;
  } else {
    s += s2;
  }
}

// The tile walk of one launch: `mt` x `nt` tiles (times `splits` of the
// contraction), columns of kGroupM row tiles.
struct Walk {
  int mt, nt, splits, total;
  __device__ __forceinline__ void at(int t, int& m, int& n, int& s) const {
    s = t / (mt * nt);
    t -= s * mt * nt;
    const int per = kGroupM * nt;
    const int g = t / per, r = t - g * per;
    const int gm = min(kGroupM, mt - g * kGroupM);
    n = r / gm;
    m = g * kGroupM + r - n * gm;
  }
};

// What an upstream gradient multiplies: each row of G where every token has its own;
// a common one (of a sum or mean) multiplies dh and dW in fp32 instead. The target's
// entry, the largest of a row by far, is then 1 - p, and not a constant whose rounding
// to bf16 would be the same for all rows and would not average out in dW.
__device__ __forceinline__ float row_factor(const Args& a, int row) {
  return a.dloss_stride ? a.dloss[a.dloss_stride * a.token[row]] : 1.f;
}
__device__ __forceinline__ float common_factor(const Args& a, int n) {
  return (a.dloss_stride ? 1.f : *a.dloss) * (a.mean ? 1.f / (float)max(n, 1) : 1.f);
}
// The target's entry of G before it is rounded.
__device__ __forceinline__ float target_grad(const Args& a, int row) {
  const float q = a.zt[row] * a.inv_cap;  // inv_cap 0: no cap
  return expm1f(-a.loss[row]) * (1.f - q * q) * row_factor(a, row);
}

// Row of `lost` (lost_targets_kernel) that belongs to vocabulary row `col`, or -1. The map is
// written for targets only: elsewhere it holds anything, and no row has that target.
__device__ __forceinline__ int lost_row(const Args& a, int n, int col) {
  const int r = a.lost_of[col];
  return (unsigned)r < (unsigned)n && a.target[r] == col ? r : -1;
}
// Added to 32 columns (from k0) of dW's row.
__device__ __forceinline__ void add_lost(const Args& a, int r, int k0, uint32_t (&v)[32]) {
  const float* p = a.lost + (int64_t)r * a.Kp + k0;
#pragma unroll
  for (int j = 0; j < 32; j += 4)
    if (k0 + j < a.Kp) {
      const float4 x = *reinterpret_cast<const float4*>(p + j);
      v[j] = __float_as_uint(__uint_as_float(v[j]) + x.x), v[j + 1] = __float_as_uint(__uint_as_float(v[j + 1]) + x.y);
      v[j + 2] = __float_as_uint(__uint_as_float(v[j + 2]) + x.z), v[j + 3] = __float_as_uint(__uint_as_float(v[j + 3]) + x.w);
    }
}

// All pieces (the last may be shorter) and the final sum use the same parts.
__device__ __forceinline__ int dh_parts(const Args& a, int n) {
  const int tiles = ((n + kTileM - 1) / kTileM) * ((a.K + kTileN - 1) / kTileN);
  return choose_parts(tiles, min(a.piece, a.V) / 64, a.pairs, a.most_parts);
}

template <int REGS>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS)); }
template <int REGS>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS)); }

template <int OP>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                const __grid_constant__ CUtensorMap tmO, const Args a) {
  constexpr bool A_MN = OP == kDw, B_MN = OP == kDh || OP == kDw;
  constexpr bool kLogits = OP == kStats || OP == kGrad;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t out_smem = sbase + kStages * kStageBytes;
  const uint32_t bar_full = sbase + kBarOffset;        // the first CTA's: both CTAs' operands in place
  const uint32_t bar_empty = bar_full + kStages * 8;   // each CTA's: stage consumed
  const uint32_t bar_tfull = bar_empty + kStages * 8;  // [2] each CTA's: accumulator complete
  const uint32_t bar_tempty = bar_tfull + 16;          // [2] the first CTA's: accumulator read by both
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kBarOffset + kBars * 8);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar_tfull + 8 * s, 1);
      mbar_init(bar_tempty + 8 * s, 2 * kEpiWarps);
    }
    fence_barrier_init();
  }
  if (warp == 2) {
    tmem_alloc2(smem_u32(tmem_slot), 512);
    tmem_relinquish2();
  }
  tc_fence_before();
  __syncthreads();
  cluster_barrier();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  const int n = *a.count;
  Walk w;
  int kb_total;
  if constexpr (OP == kStats || OP == kGrad) {
    w.mt = (n + kTileM - 1) / kTileM;
    w.nt = (a.nv + kTileN - 1) / kTileN;
    kb_total = (a.K + 63) / 64;
  } else if constexpr (OP == kDh) {
    w.mt = (n + kTileM - 1) / kTileM;
    w.nt = (a.K + kTileN - 1) / kTileN;
    kb_total = (a.nv + 63) / 64;
  } else {
    w.mt = (a.nv + kTileM - 1) / kTileM;
    w.nt = (a.K + kTileN - 1) / kTileN;
    kb_total = (n + 63) / 64;
  }
  w.splits = OP == kDh ? dh_parts(a, n) : 1;
  w.total = w.mt * w.nt * w.splits;
  const int kb_per = (kb_total + w.splits - 1) / w.splits;

  if (warp < 4) {
    if constexpr (kLogits) regs_down<kRegsRest>();
    if (warp == 0) {
      if (lane == 0) {
        // both operands are read by several pairs and rounds (4096 rows: 15.9 ms a step; 16.2 with W
        // evict-normal, 16.3 evict-first)
        const uint64_t pol = l2_policy_evict_last();
        int it = 0;
        bool ok = true;
        for (int t = pair; ok && t < w.total; t += pairs) {
          int m, nn, s;
          w.at(t, m, nn, s);
          const int m0 = m * kTileM + rank * kRowsM, n0 = nn * kTileN + rank * kRowsN;
          const int kb0 = s * kb_per, kb1 = min(kb_total, kb0 + kb_per);
          for (int kb = kb0; kb < kb1; ++kb, ++it) {
            const int st = it % kStages, r = it / kStages;
            if (r > 0 && !mbar_wait(bar_empty + 8 * st, (r - 1) & 1, kErrGemmWait)) {
              ok = false;
              break;
            }
            const uint32_t sa = sbase + st * kStageBytes, sb = sa + kABytes;
            const uint32_t bar = in_leader(bar_full + 8 * st);
            if (rank == 0) mbar_arrive_expect_tx(bar_full + 8 * st, 2 * kStageBytes);
            const int kc = kb * 64;
            if constexpr (A_MN) {
#pragma unroll
              for (int j = 0; j < kRowsM / 64; ++j) tma_load_pair(sa + j * 8192, &tmA, bar, m0 + 64 * j, kc, pol);
            } else {
              tma_load_pair(sa, &tmA, bar, kc, m0, pol);
            }
            if constexpr (B_MN) {
              const int row = OP == kDh ? a.v0 + kc : kc;
#pragma unroll
              for (int j = 0; j < kRowsN / 64; ++j) tma_load_pair(sb + j * 8192, &tmB, bar, n0 + 64 * j, row, pol);
            } else {
              tma_load_pair(sb, &tmB, bar, kc, a.v0 + n0, pol);
            }
          }
        }
        // every stage filled here has been consumed before the CTA leaves, so that no copy
        // and no arrival on its barriers is still under way
        for (int i = max(0, it - kStages); i < it; ++i)
          mbar_wait(bar_empty + 8 * (i % kStages), (i / kStages) & 1, kErrGemmWait);
      }
    } else if (warp == 1) {
      if (lane == 0 && rank == 0) {
        constexpr uint32_t idesc = umma_idesc_bf16(kTileM, kTileN, A_MN, B_MN);
        int it = 0, fill = 0;  // fill: chunks into an accumulator
        bool ok = true;
        for (int t = pair; ok && t < w.total; t += pairs) {
          int m, nn, s;
          w.at(t, m, nn, s);
          const int kb0 = s * kb_per, kb1 = min(kb_total, kb0 + kb_per);
          int kb = kb0;
          do {  // once where nothing is contracted
            const int first = kb, last = kb1 - kb > kChunk<OP> ? kb + kChunk<OP> : kb1, buf = fill & 1;
            if (!mbar_wait(bar_tempty + 8 * buf, ((fill >> 1) & 1) ^ 1, kErrTmemWait)) {
              ok = false;
              break;
            }
            tc_fence_after();
            for (; kb < last; ++kb, ++it) {
              const int st = it % kStages, r = it / kStages;
              if (!mbar_wait(bar_full + 8 * st, r & 1, kErrGemmWait)) {
                ok = false;
                break;
              }
              tc_fence_after();
              const uint32_t sa = sbase + st * kStageBytes, sb = sa + kABytes;
              // 16 deep per instruction: K-major tiles step 32 bytes along their rows, MN-major ones 16
              // rows of 128 bytes
              const uint64_t ad = A_MN ? umma_desc_mn_sw128(sa, 8192, 1024) : umma_desc_k_sw128(sa, 1024);
              const uint64_t bd = B_MN ? umma_desc_mn_sw128(sb, 8192, 1024) : umma_desc_k_sw128(sb, 1024);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                mma2_f16(tmem + buf * kTileN, ad + (A_MN ? 128 : 2) * k, bd + (B_MN ? 128 : 2) * k, idesc,
                         (kb > first || k > 0) ? 1u : 0u);
              commit2(bar_empty + 8 * st);
            }
            commit2(bar_tfull + 8 * buf);
            ++fill;
          } while (ok && kb < kb1);
        }
      }
    }
  } else {
    if constexpr (kLogits) regs_up<kRegsEpi>();
    const int r = (warp & 3) * 32 + lane;  // row of the CTA's half tile = tensor-memory lane
    const int half = (warp - 4) >> 2, left = half * kHalfN;
    const bool first_thread = (threadIdx.x & 127) == 0;  // of the half
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const float factor = OP == kDw ? common_factor(a, n) : 1.f;
    const uint32_t release = in_leader(bar_tempty);
    int tile = 0, fill = 0;
    bool dead = false;
    // The next full accumulator (its left column of this half). After a wait that ran out (the
    // status word says so) the warp goes on without waiting, so that the barriers among the
    // warps are all met and the kernel ends.
    auto filled = [&]() -> uint32_t {
      const int buf = fill & 1;
      if (!dead) dead = __any_sync(0xffffffffu, !mbar_wait(bar_tfull + 8 * buf, (fill >> 1) & 1, kErrTmemWait));
      tc_fence_after();
      return tmem + lanes + buf * kTileN + left;
    };
    auto emptied = [&] {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_cluster(release + 8 * (fill & 1));
      ++fill;
    };
    // 128 bytes of a row (64 bf16 or 32 fp32) through the half's staging buffer in the 128-byte
    // swizzle, stored by one thread while the next ones are formed. c: first column in the
    // tile; row0: first row; a box that starts outside is not stored, what reaches past the
    // end of another is not written.
    auto put = [&](const uint32_t (&o)[32], int col, int row0, bool any_row) {
      const uint32_t stage = out_smem + half * kOutBytes;
      if (first_thread) bulk_wait_read<0>();  // the last store has left the buffer
      half_barrier(half);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + sw128_offset(r, 16 * j)), "r"(o[4 * j]),
                     "r"(o[4 * j + 1]), "r"(o[4 * j + 2]), "r"(o[4 * j + 3])
                     : "memory");
      fence_proxy_async_smem();
      half_barrier(half);
      if (first_thread) {
        if (any_row) {
          if (OP != kDh || a.first) tma_store(&tmO, stage, col, row0);
          else tma_add_f32(&tmO, stage, col, row0);
        }
        bulk_commit();
      }
    };
    for (int t = pair; t < w.total; t += pairs, ++tile) {
      int m, nn, s;
      w.at(t, m, nn, s);
      const int m0 = m * kTileM + rank * kRowsM, row = m0 + r, n0 = nn * kTileN;
      const int cols = min(kTileN, (kLogits ? a.nv : a.K) - n0);
      const int end = min(left + kHalfN, cols);  // this half: columns left .. end - 1 of the tile, or none
      if constexpr (kLogits) {
        int target = -1;
        float shift = 0.f, dl = 0.f, at_target = 0.f;
        if (row < n) {
          target = a.target[row] - (a.v0 + n0);  // its column in this tile, if within 0 .. 255
          if constexpr (OP == kGrad) {
            shift = a.lse[row] * kLog2e;
            dl = row_factor(a, row);
            at_target = target_grad(a, row);
          }
        }
        // this half row of the tile: the chunks' sums
        uint32_t z[kHalfN];
        {
          const uint32_t acc = filled();
#pragma unroll
          for (int i = 0; i < kHalfN; i += 32) tmem_ld32(acc + i, z + i);
          tc_wait_ld();
          emptied();
        }
        for (int kb = kChunk<OP>; kb < kb_total; kb += kChunk<OP>) {
          const uint32_t acc = filled();
#pragma unroll
          for (int i = 0; i < kHalfN; i += 32) {
            uint32_t v[32];
            tmem_ld32(acc + i, v);
            tc_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; ++j) z[i + j] = __float_as_uint(__uint_as_float(z[i + j]) + __uint_as_float(v[j]));
          }
          emptied();
        }
        if constexpr (OP == kStats) {
          float mx = -INFINITY, sum = 0.f;
#pragma unroll
          for (int i = 0; i < kHalfN; i += 32) {
            const int c = left + i;
            uint32_t* v = z + i;
            if (c >= end) continue;
            if (a.cap > 0.f) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(a.cap * tanhf(__uint_as_float(v[j]) * a.inv_cap));
            }
            // columns past the vocabulary and the target's take no part
            if (c + 32 > cols || (unsigned)(target - c) < 32u) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (c + j >= cols || c + j == target) v[j] = 0xff800000u;
            }
            float cm = __uint_as_float(v[0]);
#pragma unroll
            for (int j = 1; j < 32; ++j) cm = fmaxf(cm, __uint_as_float(v[j]));
            const float m2 = fmaxf(mx, cm);
            if (m2 > -INFINITY) {
              const float off = m2 * kLog2e;
              sum = mx > -INFINITY ? sum * ex2(mx * kLog2e - off) : sum;  // 0, or NaN that stays
              float s0 = 0.f, s1 = 0.f;
#pragma unroll
              for (int j = 0; j < 32; j += 2) {
                s0 += ex2(fmaf(__uint_as_float(v[j]), kLog2e, -off));
                s1 += ex2(fmaf(__uint_as_float(v[j + 1]), kLog2e, -off));
              }
              sum += s0 + s1;
              mx = m2;
            } else {
              // only -inf or NaN so far: NaN has to reach the sum
#pragma unroll
              for (int j = 0; j < 32; ++j) sum += __uint_as_float(v[j]) == -INFINITY ? 0.f : __uint_as_float(v[j]);
            }
          }
          // the right half's pair joins the left's; the buffers alternate between tiles, and the barrier
          // of the next tile is passed before one is written again
          float2* pairs_smem = reinterpret_cast<float2*>(smem + kStages * kStageBytes) + (tile & 1) * kRowsM;
          if (half) pairs_smem[r] = make_float2(mx, sum);
          epi_barrier();
          if (!half && row < n) {
            const float2 p = pairs_smem[r];
            join(mx, sum, p.x, p.y);
            a.part[(int64_t)nn * a.T + row] = make_float2(mx, sum);
          }
        } else {
#pragma unroll
          for (int i = 0; i < kHalfN; i += 64) {
            const int c = left + i;
            uint32_t* v = z + i;
            if (c >= end) continue;
            if (a.cap > kFastTanhCap) {
#pragma unroll
              for (int j = 0; j < 64; ++j) v[j] = __float_as_uint(tanhf(__uint_as_float(v[j]) * a.inv_cap));
            } else if (a.cap > 0.f) {
#pragma unroll
              for (int j = 0; j < 64; ++j) v[j] = __float_as_uint(tanh_fast(__uint_as_float(v[j]) * a.inv_cap));
            }
            const int rel = target - c;
            uint32_t o[32];
#pragma unroll
            for (int j = 0; j < 64; j += 2) {
              float p[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float u = __uint_as_float(v[j + e]), slope = dl;
                if (a.cap > 0.f) {  // u is the tanh
                  slope *= 1.f - u * u;
                  u *= a.cap;
                }
                p[e] = ex2(fmaf(u, kLog2e, -shift)) * slope;
                if (rel == j + e) p[e] = at_target;
                if (row >= n || c + j + e >= cols) p[e] = 0.f;
              }
              o[j / 2] = pack_bf16x2(p[0], p[1]);
            }
            put(o, n0 + c, m0, m0 < n);
          }
        }
      } else {
        const bool empty = s * kb_per >= kb_total;  // nothing contracted: the product is zero
        int lost = -1;
        if (OP == kDw && row < a.nv) lost = lost_row(a, n, a.v0 + row);
        const uint32_t acc = filled() - left;
        constexpr int kStep = OP == kDh ? 32 : 64;
#pragma unroll 1
        for (int c = left; c < end; c += kStep) {
          uint32_t o[32];
          if constexpr (OP == kDh) {
            tmem_ld32(acc + c, o);
            tc_wait_ld();
          } else {
#pragma unroll
            for (int hh = 0; hh < 64; hh += 32) {
              uint32_t v[32];
              tmem_ld32(acc + c + hh, v);
              tc_wait_ld();
              if (lost >= 0) add_lost(a, lost, n0 + c + hh, v);
#pragma unroll
              for (int j = 0; j < 32; j += 2)
                o[(hh + j) / 2] = pack_bf16x2(__uint_as_float(v[j]) * factor, __uint_as_float(v[j + 1]) * factor);
            }
          }
          if (empty) {
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = 0u;
          }
          if constexpr (OP == kDh) put(o, n0 + c, s * a.acc_rows + m0, m0 < n);
          else put(o, n0 + c, a.v0 + m0, m0 < a.nv);
        }
        emptied();
      }
    }
    if (OP != kStats && first_thread) bulk_wait_all();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_barrier();
  tc_fence_after();
  if (warp == 2) tmem_dealloc2(tmem, 512);
}

// ---------------------------------------------------------------------------
// Gather of the scored rows. A CTA owns `rows` consecutive rows of the batch: it
// counts the scored ones before them (every CTA reads the targets itself: no
// second pass, no waiting), then a warp copies a row and takes its target logit.
// ---------------------------------------------------------------------------
struct PrepArgs {
  const __nv_bfloat16* h;
  const __nv_bfloat16* w;
  const int64_t* targets;
  int64_t ldh, ldw;
  int64_t ignore;
  __nv_bfloat16* hc;  // [T][Kp] scored rows; Kp a multiple of 8, zero past K
  int *count, *target, *token, *place;  // place: [T] row of hc, or -1
  float *zt, *loss;                     // loss: [T] by token (ignored rows: 0)
  unsigned* ticket;
  int T, V, K, Kp, rows, vec;  // vec: rows of h in whole 16-byte vectors (W's and hc's are)
  float cap, inv_cap;
};

__global__ void __launch_bounds__(256) prep_kernel(PrepArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  extern __shared__ int dest[];  // [rows]
  __shared__ int warp_n[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row0 = blockIdx.x * a.rows, row1 = min(a.T, row0 + a.rows);
  int before = 0;
  for (int t = threadIdx.x; t < row0; t += 256) before += a.targets[t] != a.ignore;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if (lane == 0) warp_n[warp] = before;
  __syncthreads();
  int base = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) base += warp_n[i];
  if (warp == 0) {
    for (int t = row0; t < row1; t += 32) {
      const bool scored = t + lane < row1 && a.targets[t + lane] != a.ignore;
      const unsigned b = __ballot_sync(0xffffffffu, scored);
      if (t + lane < row1) dest[t + lane - row0] = scored ? base + __popc(b & ((1u << lane) - 1)) : -1;
      base += __popc(b);
    }
    if (row1 == a.T) {
      if (lane == 0) {
        *a.count = base;
        *a.ticket = 0;
        dest[a.rows] = base;
      }
    }
  }
  __syncthreads();
  for (int t = row0 + warp; t < row1; t += 8) {
    const int d = dest[t - row0];
    if (lane == 0) a.place[t] = d;
    if (d < 0) {
      if (lane == 0) a.loss[t] = 0.f;
      continue;
    }
    const int64_t y = a.targets[t];
    const bool valid = y >= 0 && y < a.V;
    const __nv_bfloat16* hr = a.h + (int64_t)t * a.ldh;
    const __nv_bfloat16* wr = a.w + (valid ? y : 0) * a.ldw;
    __nv_bfloat16* o = a.hc + (int64_t)d * a.Kp;
    float s = 0.f;
    if (a.vec) {
#pragma unroll 4
      for (int c = lane * 8; c < a.K; c += 256) {
        const uint4 hv = *reinterpret_cast<const uint4*>(hr + c), wv = *reinterpret_cast<const uint4*>(wr + c);
        *reinterpret_cast<uint4*>(o + c) = hv;
        const __nv_bfloat16 *he = reinterpret_cast<const __nv_bfloat16*>(&hv), *we = reinterpret_cast<const __nv_bfloat16*>(&wv);
#pragma unroll
        for (int j = 0; j < 8; ++j) s = fmaf(bf2f(he[j]), bf2f(we[j]), s);
      }
    } else {
      for (int c = lane; c < a.Kp; c += 32) {
        const __nv_bfloat16 x = c < a.K ? hr[c] : f2bf(0.f);
        o[c] = x;
        if (c < a.K) s = fmaf(bf2f(x), bf2f(wr[c]), s);
      }
    }
    s = warp_sum(s);
    if (lane == 0) {
      if (a.cap > 0.f) s = a.cap * tanhf(s * a.inv_cap);
      if (!valid) {
        set_status(kErrBounds);
        s = NAN;
      }
      a.zt[d] = s;
      a.target[d] = valid ? (int)y : -1;
      a.token[d] = t;
    }
  }
  // rows up to the contraction's next block of 64 take part in dW: zeros
  if (row1 == a.T) {
    const int n = dest[a.rows];
    const int end = min(a.T, (n + 63) / 64 * 64);
    for (int64_t i = (int64_t)n * a.Kp + threadIdx.x; i < (int64_t)end * a.Kp; i += 256) a.hc[i] = f2bf(0.f);
  }
}

// ---------------------------------------------------------------------------
// Merge of the (max, sum) pairs: 32 rows a CTA (lanes), the column tiles dealt to
// its warps; then each row's loss. The last CTA adds the rows' losses in order.
// ---------------------------------------------------------------------------
struct MergeArgs {
  const float2* part;  // [nt][T]
  const int *count, *token;
  const float* zt;
  float* row_loss;  // [T] by scored row
  float* lse;       // [T] by scored row (not zt + loss: a target far below the others would leave none of its digits)
  float* loss;      // [T] by token
  float* total;     // [1] sum or mean, or null
  unsigned* ticket;
  int T, nt, mean;
};
constexpr int kMergeWarps = 32;

__global__ void __launch_bounds__(32 * kMergeWarps) merge_kernel(MergeArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float2 sh[kMergeWarps][32];
  __shared__ float red[32];
  __shared__ bool last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = *a.count;
  const int row = blockIdx.x * 32 + lane;
  float m = -INFINITY, s = 0.f;
  if (row < n)
    for (int t = warp; t < a.nt; t += 8 * kMergeWarps) {  // eight loads in flight
      float2 p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int q = t + i * kMergeWarps;
        p[i] = q < a.nt ? a.part[(int64_t)q * a.T + row] : make_float2(-INFINITY, 0.f);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) join(m, s, p[i].x, p[i].y);
    }
  sh[warp][lane] = make_float2(m, s);
  __syncthreads();
  if (warp == 0 && row < n) {
    for (int i = 1; i < kMergeWarps; ++i) join(m, s, sh[i][lane].x, sh[i][lane].y);
    // s = 0 (a vocabulary of one): d = -inf, loss 0
    const float zt = a.zt[row], others = m + logf(s), d = others - zt;
    const float more = d == -INFINITY ? 0.f : log1pf(expf(-fabsf(d)));
    const float loss = d != d ? d : fmaxf(d, 0.f) + more;
    a.row_loss[row] = loss;
    a.lse[row] = d != d ? d : fmaxf(others, zt) + more;
    a.loss[a.token[row]] = loss;
  }
  if (a.total == nullptr) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  float acc = 0.f;
  for (int i = threadIdx.x; i < n; i += 32 * kMergeWarps) acc += __ldcg(a.row_loss + i);
  acc = block_sum(acc, red);
  if (threadIdx.x == 0) *a.total = a.mean ? acc / (float)max(n, 1) : acc;
}

// What the targets' entries of G lose when they are rounded to bf16, as dW misses it: for each
// target the sum of e_t h_t over its rows in order, e_t = g_t - bf16(g_t). A target's row of dW
// consists mostly of those entries, however many rows the batch has, so without it their rounding
// shows beside dW's own (error against 64 bits, 1001 rows with weights, 50257 x 2560: 2.24e-3
// without, 1.7e-3 with, the output's own rounding; 20 us of 950).
// CTA (r, y): scored row r, which does the work of its target if it is the first row that has it,
// and 2048 columns. Finding the rows reads at most n targets for each different one.
struct LostArgs {
  Args g;
  const __nv_bfloat16* hc;  // [T][Kp] scored rows
  float* lost;              // [T][Kp]: row r for the target that row r is the first of
  int* lost_of;             // [V]
};
constexpr int kLostThreads = 256;
__global__ void __launch_bounds__(kLostThreads) lost_targets_kernel(const LostArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ int found[kLostThreads];
  __shared__ int warp_n[kLostThreads / 32];
  const int r = blockIdx.x, n = *a.g.count, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (r >= n) return;
  const int y = a.g.target[r];
  if (y < 0) return;
  // later rows of a frequent target find an earlier one soon
  for (int t0 = 0; t0 < r; t0 += 4 * kLostThreads) {
    bool seen = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = t0 + i * kLostThreads + (int)threadIdx.x;
      seen |= t < r && a.g.target[t] == y;
    }
    if (__syncthreads_or(seen)) return;
  }
  const int c = (blockIdx.y * kLostThreads + threadIdx.x) * 8;
  float s[8] = {};
  for (int t0 = r; t0 < n; t0 += kLostThreads) {
    const int t = t0 + threadIdx.x;
    const bool mine = t < n && a.g.target[t] == y;
    const unsigned b = __ballot_sync(0xffffffffu, mine);
    if (!__syncthreads_or(mine)) continue;  // also: the list of the rows before has been read
    if (lane == 0) warp_n[warp] = __popc(b);
    __syncthreads();
    int at = __popc(b & ((1u << lane) - 1)), total = 0;
#pragma unroll
    for (int i = 0; i < kLostThreads / 32; ++i) {
      at += i < warp ? warp_n[i] : 0;
      total += warp_n[i];
    }
    if (mine) found[at] = t;
    __syncthreads();
    if (c < a.g.Kp)
      for (int i = 0; i < total; ++i) {
        const int row = found[i];
        const float g = target_grad(a.g, row), e = g - bf2f(f2bf(g));
        const uint4 hv = *reinterpret_cast<const uint4*>(a.hc + (int64_t)row * a.g.Kp + c);
        const __nv_bfloat16* he = reinterpret_cast<const __nv_bfloat16*>(&hv);
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] = fmaf(e, bf2f(he[j]), s[j]);
      }
  }
  if (c < a.g.Kp) {
    float4* o = reinterpret_cast<float4*>(a.lost + (int64_t)r * a.g.Kp + c);
    o[0] = make_float4(s[0], s[1], s[2], s[3]);
    o[1] = make_float4(s[4], s[5], s[6], s[7]);
  }
  if (blockIdx.y == 0 && threadIdx.x == 0) a.lost_of[y] = r;
}

// dh[t] = (sum over the contraction's parts of acc[.][place[t]] + e W[y]) * factor, 0
// for ignored rows. e is what the target's entry of G lost when it was rounded to bf16:
// that entry alone is of the size of the whole row, the others are far below it, so
// with it added back the rounding of G hardly shows in dh (measured against 64 bits:
// 2.7e-3 -> 1.7e-3, the output's own rounding). A thread takes E columns of a row.
struct FinishArgs {
  Args g;
  const float* acc;
  const int* place;
  const __nv_bfloat16* w;
  __nv_bfloat16* dh;
  int64_t ldw;
  int lda;       // row stride of acc
  int per_row;   // threads a row
};
template <int E>
__global__ void __launch_bounds__(256) finish_dh_kernel(const FinishArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int n = *a.g.count;
  const int parts = dh_parts(a.g, n);
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int t = (int)(i / a.per_row);
  if (t >= a.g.T) return;
  const int c = (int)(i - (int64_t)t * a.per_row) * E;
  const int p = a.place[t];
  __nv_bfloat16* o = a.dh + (int64_t)t * a.g.K + c;
  float s[E] = {};
  if (p >= 0) {
    const float g = target_grad(a.g, p);
    const float e = g - bf2f(f2bf(g));
    const __nv_bfloat16* wr = a.w + (int64_t)max(a.g.target[p], 0) * a.ldw + c;
    const float* row = a.acc + (int64_t)p * a.lda + c;
    const int64_t part = (int64_t)a.g.acc_rows * a.lda;
    if constexpr (E == 8) {
      const uint4 wv = *reinterpret_cast<const uint4*>(wr);
      const __nv_bfloat16* we = reinterpret_cast<const __nv_bfloat16*>(&wv);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] = e * bf2f(we[j]);
#pragma unroll 4
      for (int k = 0; k < parts; ++k) {
        const float4 x = *reinterpret_cast<const float4*>(row + k * part);
        const float4 y = *reinterpret_cast<const float4*>(row + k * part + 4);
        s[0] += x.x, s[1] += x.y, s[2] += x.z, s[3] += x.w;
        s[4] += y.x, s[5] += y.y, s[6] += y.z, s[7] += y.w;
      }
    } else {
      s[0] = e * bf2f(*wr);
      for (int k = 0; k < parts; ++k) s[0] += row[k * part];
    }
    const float factor = common_factor(a.g, n);
#pragma unroll
    for (int j = 0; j < E; ++j) s[j] *= factor;
  }
  if constexpr (E == 8)
    *reinterpret_cast<uint4*>(o) =
        make_uint4(pack_bf16x2(s[0], s[1]), pack_bf16x2(s[2], s[3]), pack_bf16x2(s[4], s[5]), pack_bf16x2(s[6], s[7]));
  else
    *o = f2bf(s[0]);
}

// setmaxnreg.inc would wait for good for registers that the block was not launched with.
template <int OP>
static int split_fits() {
  static const int rc = [] {
    cudaFuncAttributes f;
    const cudaError_t e = cudaFuncGetAttributes(&f, gemm_kernel<OP>);
    return e != cudaSuccess ? (int)e : f.numRegs < kRegsMax ? (int)cudaErrorInvalidKernelImage : 0;
  }();
  return rc;
}

template <int OP>
static int launch_gemm(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& to, const Args& a, int64_t tiles,
                       int num_sms, cudaStream_t st) {
  if (tiles <= 0) return 0;
  if (tiles > 0x7FFFFFFFll - 1024) return -1;
  if (int e = smem_attr_once<gemm_kernel<OP>>(kSmem)) return e;
  if (OP == kStats || OP == kGrad)
    if (int e = split_fits<OP>()) return e;
  const int grid = (int)(tiles < num_sms / 2 ? tiles : num_sms / 2);
  cudaError_t e = launch_k(gemm_kernel<OP>, dim3(2 * grid), dim3(kThreads), kSmem, st, 1, ta, tb, to, a);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

static inline int64_t tiles_of(int64_t n, int tile) { return (n + tile - 1) / tile; }

}  // namespace lce
}  // namespace b200

using namespace b200;
using namespace b200::lce;

extern "C" {

// What a forward pass leaves for its backward pass, in one buffer of
// b200_lce_saved_bytes: hc [T, Kp] bf16, then zt, row loss and lse fp32 [T] each, then
// int32 count, ticket, target [T], token [T], place [T].
int64_t b200_lce_saved_bytes(int T, int Kp) { return (int64_t)T * Kp * 2 + ((int64_t)6 * T + 2) * 4; }

// Scratch of the forward pass: a (max, sum) pair per row and column tile.
int64_t b200_lce_forward_bytes(int T, int V) { return (int64_t)T * tiles_of(V, kTileN) * 8; }

// Parts of dh's sums there is room for with up to T scored rows: eight rounds of tiles
// of all CTA pairs, at most 155 MB, and always one.
static int most_parts(int T, int K, int num_sms) {
  const int64_t s = 8 * (num_sms / 2) / (tiles_of(T, kTileM) * tiles_of(K, kTileN));
  return (int)(s > kMostParts ? kMostParts : s < 1 ? 1 : s);
}
// Rows and row stride (elements) of one part of dh's sums.
static int acc_rows(int T) { return (int)(tiles_of(T, kRowsM) * kRowsM); }
static int acc_cols(int K) { return (K + 3) / 4 * 4; }

// Scratch of the backward pass: one piece of G (bf16 [T, piece]), dh's sums, and for dW what
// the targets' entries lost (fp32 [T, Kp]) with its map (int32 [V]).
static int64_t dh_bytes(int T, int K, int num_sms) { return (int64_t)most_parts(T, K, num_sms) * acc_rows(T) * acc_cols(K) * 4; }
int64_t b200_lce_backward_bytes(int T, int V, int K, int Kp, int piece, int want_dh, int want_dw, int num_sms) {
  return (int64_t)T * piece * 2 + (want_dh ? dh_bytes(T, K, num_sms) : 0) + (want_dw ? (int64_t)T * Kp * 4 + (int64_t)V * 4 : 0);
}

struct Saved {
  uint8_t* hc;
  float *zt, *loss, *lse;
  int *count, *target, *token, *place;
  Saved(void* p, int T, int Kp) {
    hc = reinterpret_cast<uint8_t*>(p);
    zt = reinterpret_cast<float*>(hc + (int64_t)T * Kp * 2);
    loss = zt + T;
    lse = loss + T;
    count = reinterpret_cast<int*>(lse + T);
    target = count + 2;
    token = target + T;
    place = token + T;
  }
};

// Forward. h [T, K] and W [V, K] bf16 (strides in elements; W 16-byte aligned with
// ldw % 8 == 0), targets int64. loss fp32 [T]; total [1] or null (mean: divided by
// the scored rows, at least 1). Returns 0, a CUDA error code, or -1 for arguments
// out of range.
int b200_lce_forward(const void* h, int64_t ldh, const void* W, int64_t ldw, const int64_t* targets, int64_t ignore,
                     int T, int V, int K, int Kp, float cap, void* saved, void* part, float* loss, float* total,
                     int mean, int num_sms, cudaStream_t st) {
  if (T <= 0 || V <= 0 || K <= 0 || Kp < K || (Kp % 8) || (ldw % 8) || ((uintptr_t)W & 15) || ((uintptr_t)saved & 15))
    return -1;
  const Saved f(saved, T, Kp);
  PrepArgs p = {};
  p.h = reinterpret_cast<const __nv_bfloat16*>(h);
  p.w = reinterpret_cast<const __nv_bfloat16*>(W);
  p.targets = targets;
  p.ldh = ldh;
  p.ldw = ldw;
  p.ignore = ignore;
  p.hc = reinterpret_cast<__nv_bfloat16*>(f.hc);
  p.count = f.count;
  p.ticket = reinterpret_cast<unsigned*>(f.count + 1);
  p.target = f.target;
  p.token = f.token;
  p.place = f.place;
  p.zt = f.zt;
  p.loss = loss;
  p.T = T;
  p.V = V;
  p.K = K;
  p.Kp = Kp;
  p.cap = cap;
  p.inv_cap = cap > 0.f ? 1.f / cap : 0.f;
  p.vec = K % 8 == 0 && ldh % 8 == 0 && ((uintptr_t)h & 15) == 0;
  // eight rows a CTA (one a warp) while that is at most four CTAs an SM
  const int64_t want = tiles_of(T, 4 * num_sms);
  p.rows = (int)(want < 8 ? 8 : want > 8192 ? 8192 : (want + 7) / 8 * 8);
  cudaError_t e = launch_k(prep_kernel, dim3((unsigned)tiles_of(T, p.rows)), dim3(256), (p.rows + 1) * sizeof(int), st, 1, p);
  if (e != cudaSuccess) return (int)e;
  Args a = {};
  a.count = f.count;
  a.target = f.target;
  a.token = f.token;
  a.zt = f.zt;
  a.part = reinterpret_cast<float2*>(part);
  a.T = T;
  a.V = V;
  a.K = K;
  a.nv = V;
  a.cap = p.cap;
  a.inv_cap = p.inv_cap;
  CUtensorMap ta, tb;
  if (!make_tmap_2d(&ta, f.hc, T, Kp, Kp, kRowsM, 64, 2) || !make_tmap_2d(&tb, W, V, K, ldw, kRowsN, 64, 2)) return -1;
  if (int r = launch_gemm<kStats>(ta, tb, ta, a, tiles_of(T, kTileM) * tiles_of(V, kTileN), num_sms, st)) return r;
  MergeArgs g = {};
  g.part = a.part;
  g.count = f.count;
  g.token = f.token;
  g.zt = f.zt;
  g.row_loss = f.loss;
  g.lse = f.lse;
  g.loss = loss;
  g.total = total;
  g.ticket = p.ticket;
  g.T = T;
  g.nt = (int)tiles_of(V, kTileN);
  g.mean = mean;
  e = launch_k(merge_kernel, dim3((unsigned)tiles_of(T, 32)), dim3(32 * kMergeWarps), 0, st, 1, g);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

// Backward from what the forward pass saved. dloss: element token * dloss_stride.
// dh [T, K] contiguous and dW [V, K] (row stride lddw, a multiple of 8) are null
// where not wanted. piece: columns of the vocabulary at a time, a multiple of 256.
int b200_lce_backward(void* saved, const void* W, int64_t ldw, const float* dloss, int64_t dloss_stride, int mean, int T,
                      int V, int K, int Kp, float cap, int piece, void* scratch, void* dh, void* dW, int64_t lddw,
                      int num_sms, cudaStream_t st) {
  if (T <= 0 || V <= 0 || K <= 0 || Kp < K || (Kp % 8) || (ldw % 8) || ((uintptr_t)W & 15) || piece <= 0 ||
      (piece % kTileN) || (((uintptr_t)saved | (uintptr_t)scratch | (uintptr_t)dh | (uintptr_t)dW) & 15) ||
      (dW && ((lddw % 8) || lddw < K)))
    return -1;
  const Saved f(saved, T, Kp);
  Args a = {};
  a.count = f.count;
  a.target = f.target;
  a.token = f.token;
  a.zt = f.zt;
  a.loss = f.loss;
  a.lse = f.lse;
  a.dloss = dloss;
  a.dloss_stride = dloss_stride;
  a.mean = mean;
  a.acc_rows = acc_rows(T);
  a.T = T;
  a.V = V;
  a.K = K;
  a.piece = piece;
  a.pairs = num_sms / 2;
  a.most_parts = most_parts(T, K, num_sms);
  a.cap = cap;
  a.inv_cap = cap > 0.f ? 1.f / cap : 0.f;
  a.Kp = Kp;
  void* G = scratch;
  float* acc = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(scratch) + (int64_t)T * piece * 2);
  const int lda = acc_cols(K);
  if ((int64_t)a.most_parts * a.acc_rows > 0x7FFFFFFFll) return -1;
  CUtensorMap h_rows, w_rows, g_rows, w_cols, g_cols, h_cols, o_dh, o_dw;
  if (!make_tmap_2d(&h_rows, f.hc, T, Kp, Kp, kRowsM, 64, 2) || !make_tmap_2d(&w_rows, W, V, K, ldw, kRowsN, 64, 2) ||
      !make_tmap_2d(&g_rows, G, T, piece, piece, kRowsM, 64, 2))
    return -1;
  if (dh && (!make_tmap_2d(&w_cols, W, V, K, ldw, 64, 64, 2) ||
             !make_tmap_2d(&o_dh, acc, (int64_t)a.most_parts * a.acc_rows, K, lda, kRowsM, 32, 4)))
    return -1;
  if (dW && (!make_tmap_2d(&g_cols, G, T, piece, piece, 64, 64, 2) || !make_tmap_2d(&h_cols, f.hc, T, Kp, Kp, 64, 64, 2) ||
             !make_tmap_2d(&o_dw, dW, V, K, lddw, kRowsM, 64, 2)))
    return -1;
  if (dW) {
    LostArgs l = {};
    l.lost = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(acc) + (dh ? dh_bytes(T, K, num_sms) : 0));
    l.lost_of = reinterpret_cast<int*>(l.lost + (int64_t)T * Kp);
    a.lost = l.lost;
    a.lost_of = l.lost_of;
    l.g = a;
    l.hc = reinterpret_cast<const __nv_bfloat16*>(f.hc);
    const dim3 grid((unsigned)T, (unsigned)tiles_of(Kp, 8 * kLostThreads));
    const cudaError_t e = launch_k(lost_targets_kernel, grid, dim3(kLostThreads), 0, st, 1, l);
    if (e != cudaSuccess) return (int)e;
  }
  for (int64_t v0 = 0; v0 < V; v0 += piece) {
    a.v0 = (int)v0;
    a.nv = (int)(V - v0 < piece ? V - v0 : piece);
    a.first = v0 == 0;
    const int64_t rows = tiles_of(T, kTileM);
    if (int r = launch_gemm<kGrad>(h_rows, w_rows, g_rows, a, rows * tiles_of(a.nv, kTileN), num_sms, st)) return r;
    if (dh)
      if (int r = launch_gemm<kDh>(g_rows, w_cols, o_dh, a, rows * tiles_of(K, kTileN) * a.most_parts, num_sms, st)) return r;
    if (dW)
      if (int r = launch_gemm<kDw>(g_cols, h_cols, o_dw, a, tiles_of(a.nv, kTileM) * tiles_of(K, kTileN), num_sms, st)) return r;
  }
  if (dh) {
    FinishArgs q = {};
    q.g = a;
    q.acc = acc;
    q.place = f.place;
    q.w = reinterpret_cast<const __nv_bfloat16*>(W);
    q.ldw = ldw;
    q.dh = reinterpret_cast<__nv_bfloat16*>(dh);
    q.lda = lda;
    // vectors of eight where rows are whole ones (W's and the sums' rows are aligned whatever K is)
    q.per_row = K % 8 == 0 ? K / 8 : K;
    const int64_t blocks = tiles_of((int64_t)T * q.per_row, 256);
    if (blocks > 0x7FFFFFFFll) return -1;
    cudaError_t e = launch_k(K % 8 == 0 ? finish_dh_kernel<8> : finish_dh_kernel<1>, dim3((unsigned)blocks), dim3(256), 0, st, 1, q);
    if (e != cudaSuccess) return (int)e;
  }
  return (int)cudaGetLastError();
}

}  // extern "C"

B200_STATUS_ACCESSORS(linear_ce)
