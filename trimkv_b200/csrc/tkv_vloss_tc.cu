// Cross entropy against a vocabulary (tkv_vloss.cuh) on tcgen05 + TMEM:
//   kVtStats  : logits of 256 tokens x up to 256 words -> largest logit and sum of weights of every token, logit of its label;
//   kVtLogits : the same logits again -> a tile of dL in the type of the operands;
//   kVtGrads  : dx shares (dL w, both read along the vocabulary) and dw (dL^T x, both read along the tokens) of a piece, one launch.
//
// Bound by the tensor cores.  A tile belongs to a pair of CTAs (cta_group::2): each holds 128 of its 256 rows and, of every stage of 64
// along the inner axis, its rows of A and half of B, 32 KB; the products read the other half from the neighbour, so that a CTA fetches
// 32 KB for the work for which a CTA alone fetches 48.  Six stages; two accumulators of 256 TMEM columns, so that a tile's epilogue runs
// beside the next tile's products.  One pair per two SMs, tiles in turn: row tiles innermost, in groups whose rows stay in L2, so that a
// tile of w comes from HBM once per group.
// What is stored along the inner axis (x, w in the logits; dL for dx) is read K-major, what is stored across it MN-major: nothing is
// transposed in memory.
// fp32 operands are three bf16 numbers each (x = a + b + c, each the rounding of what the ones before leave: 24 bits together), stored as
// three matrices one below the other, and a product is the six products of parts down to 2^-16 of the first, the smallest ones first; what
// is left out is below 2^-24 of a product.  w is taken apart a piece of the vocabulary at a time, so that its parts stay in L2.
//
// Copies of both CTAs complete on the even CTA's barriers; it issues the products; their completion is told to both.  Every wait is
// bounded; a CTA whose wait runs out records TKV_DEV_TIMEOUT, in the plan too (losses, dx and dw become NaN), and tells its neighbour; both
// drain and free their TMEM.
#include <cuda.h>
#include "tkv_vloss.cuh"
#include "tkv_tc.cuh"

namespace tkv {

constexpr int kVtThreads = 320;                            // warp 0: copies, warp 1: products, warps 2-9: epilogue
constexpr int kVtK = 64, kVtRows = 256, kVtCols = 256, kVtStages = 6;
constexpr int kVtABytes = 128 * kVtK * 2, kVtBBytes = 128 * kVtK * 2, kVtStage = kVtABytes + kVtBBytes;
constexpr int kVtGroup = 32;                               // row tiles that share a pass over w
constexpr int kVtPairs = 74;
constexpr int kVtHalf = kVtCols / 2;                       // columns of a warp of the epilogue
// Stages that are added up in TMEM (1024 of the inner axis): the tensor cores cut what they add to an accumulator.  Relative error of a
// logit of 40 whose products are all positive, width 4096, bf16: one sum -5.4e-6; sums of 16 stages -1.3e-6, of 8 -5.6e-7, of 4 -2.8e-7
// (before vt_up puts the mean of that back).
// ms of 8192 x 151936 x 2048 with both gradients: 14.6, 14.7, 15.2, 16.4; us of 1500 tokens scored: 600, 620, 655, 710.
constexpr int kVtSum = 16;
// In fp32 half as many.  RMS error of the gradients of 300 tokens, width 1024, 32768 words, with 16 stages: 8.4e-7 (dx) and 8.9e-7 (dw), with 8
// 4.6e-7 and 3.3e-7 (fp32 products on the CUDA cores: 1.0e-6 and 5.4e-7); us of the pass's kernels 620 and 636.
constexpr int kVtSum32 = 8;
// Gradients in 16 bits: sums of 4096 of the tokens or words.  In one sum of any length, whose products come to be far below it, dw of 32768, 2^17
// and 2^21 tokens with products of one sign was -2.0e-4, -8.3e-4 and -1.3e-2 of itself off in the mean, all of it to one side (rounding to fp16
// is 2.4e-4 in the mean, either way); with 256 stages -8e-5, 128 -4e-5, 64 -2e-5 at every length.  us of dx and dw of 4096 x 30000 x 2048:
// 1008, 1010, 1011, 1011; of 8192 x 151936 x 2048 10.8 ms with any.
constexpr int kVtSumGrad = 64;
// The label's entry of dL, g (p - 1), is most of its row, and what rounding it to 16 bits takes away does not average out: all of a row of
// dx, and of dw's row of the label, is off by it.  It is kept (Vloss::rest) and goes back in where those rows are finished, w[label] rest into
// dx, x rest into dw.  For dw every warp of 32 rows looks through the tokens' labels, up to kVtExact tokens and the first kVtExactHits of them:
// RMS error of dw of 256 tokens, bf16, with a gradient for each token 1.7e-3 (the rounding of dw itself) for 168 us, without it 2.3e-3; 4096
// tokens would take 1600 us for 1330.  A word that is many tokens' label averages their roundings (256 tokens of one word, all put back: 590 us).
constexpr int kVtExact = 256, kVtExactHits = 8;

enum { kVtStats, kVtLogits, kVtGrads };

struct VtSmem {
  uint64_t full[kVtStages], empty[kVtStages], acc_full[2], acc_empty[2];
  uint32_t tmem_base;
  int abort_flag;
};
constexpr int kVtOut = 4096;                               // 32 rows of 128 bytes on their way out, for every warp of the epilogue
constexpr int kVtSmemBytes = kVtStages * kVtStage + 8 * kVtOut + (int)sizeof(VtSmem);
static_assert(kVtSmemBytes <= 232448, "shared memory");

struct VtParams {
  Vloss l;
  int cols;                                                // of a tile (a multiple of 16)
  int a_box, a_ranks;                                      // rows of x or dL that a CTA fetches, CTAs of a pair that have any (few tokens)
  int64_t v0, piece_cols;                                  // the vocabulary from v0
  int tile0;                                               // kVtStats: tiles of the pieces before
  int parts, rows, w_rows, w0;                             // of an operand (1 or 3), rows of a part of x and dL, and of w; the piece's first row there
  int want_dx, want_dw, more;                              // kVtGrads
  int64_t piece_steps;                                     // stages of a whole piece
  int sum_steps;                                           // stages that are added up in TMEM
  const void* xc;                                          // the rows of x that count
};

// What a sum of so many stages is multiplied by.  Each of its 4 additions a stage cuts half a unit of what is there on average, 2^-24 / m of a
// number of mantissa m, in the mean over m 2^-24 / (2 ln 2), and over a sum that grows evenly half of that for every addition.  The sum
// of the means is known, so it is put back: it is the same for all tokens, and a mean over them would keep it.  Mean loss of 300 tokens of random
// rows, widths 512 to 4096, off by 2 to 8e-7 of itself without, by 0.1 to 2e-7 with it; a token's loss by 1.1 to 2.3e-7 RMS, as with fp32
// products (0.7 to 3.5e-7).  It is a mean: a logit whose products are few and leave nothing to cut (a row with one element) becomes up to
// 1.4e-6 of itself larger (16 stages), and where a thousand products of one sign lose more, a logit stays 4.5e-6 too small in fp16, whose products
// are longer (5.9e-6 without), and becomes 4e-7 too large in bf16 (1.0e-6 too small without).
__device__ __forceinline__ float vt_up(int stages) { return 1.f + (float)(4 * stages) * (0.36067376f / 16777216.f); }

// The parts that product c takes of A and of B; with one part there is product 5 alone.
constexpr int kVtProducts = 6;
__device__ __forceinline__ int vt_part_a(int c) { return (0x052 >> (2 * c)) & 3; }   // 2 0 1 1 0 0
__device__ __forceinline__ int vt_part_b(int c) { return (0x118 >> (2 * c)) & 3; }   // 0 2 1 0 1 0

// ---- instructions for pairs of CTAs
__device__ __forceinline__ uint32_t vt_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t vt_of_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void vt_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void vt_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void vt_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accum) : "memory");
}
__device__ __forceinline__ void vt_commit(uint64_t* bar) {  // to both CTAs
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void vt_arrive(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void vt_raise(uint32_t cluster_addr) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(1) : "memory");
}
__device__ __forceinline__ float vt_max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// kind::f16 of a pair: D fp32, M = 256, N = n; which operands lie across the inner axis.
__device__ __forceinline__ uint32_t vt_idesc(int bf16, int a_mn, int b_mn, int n) {
  return (1u << 4) | ((uint32_t)bf16 << 7) | ((uint32_t)bf16 << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | (16u << 24);
}

// A pair's tiles in order; every role keeps its own.
struct VtTile {
  int dx;                                                  // kVtGrads: 1 for a share of dx, 0 for dw
  int row0, col0, slot, step0, steps;                      // of 256 rows and `cols` columns; stages of the inner axis
};
template <int kMode> struct VtTiles {
  const VtParams& p;
  int n, tile, count, mt, nt;
  int pair, turn, dx_count, dw_count, ht, slots, split, more, extra;   // kVtGrads: see vloss_rows_grad_kernel
  __device__ __forceinline__ VtTiles(const VtParams& q, int at) : p(q), pair(at) {
    n = q.l.plan.head[0];
    tile = pair - kVtPairs;
    mt = (n + kVtRows - 1) / kVtRows;
    if (kMode == kVtGrads) {
      ht = (q.l.width + kVtCols - 1) / kVtCols;
      slots = q.l.slots[0];
      split = ((int)q.piece_steps + slots - 1) / slots;
      dx_count = q.want_dx ? mt * ht * slots : 0;
      dw_count = q.want_dw ? (int)((q.piece_cols + kVtRows - 1) / kVtRows) * ht : 0;
      more = dx_count % kVtPairs;
      extra = more ? min(q.l.slots[1], dw_count / (kVtPairs - more)) : 0;   // (a last piece has fewer tiles)
      turn = 0;
    } else {
      nt = (int)((q.piece_cols + q.cols - 1) / q.cols);
      count = mt * nt;
    }
  }
  // The next tile of dx, or of dw from dx_count on; -1 after the last.
  __device__ __forceinline__ int next_grad() {
    if (tile + kVtPairs < dx_count) return tile += kVtPairs;
    tile = dx_count;
    const int fewer = kVtPairs - more, mine = pair < more ? 0 : extra, j = turn++;
    const int i = j < mine ? pair - more + fewer * j : extra * fewer + (pair + kVtPairs - more) % kVtPairs + kVtPairs * (j - mine);
    return i < dw_count ? dx_count + i : -1;
  }
  __device__ __forceinline__ bool next(VtTile& t) {
    if (kMode == kVtGrads) {
      const int at = next_grad();
      if (at < 0) return false;
      t.dx = at < dx_count;
      const int i = t.dx ? at : at - dx_count;
      t.col0 = i % ht * kVtCols;
      const int r = i / ht;
      if (t.dx) {
        t.row0 = r / slots * kVtRows;
        t.slot = r % slots;
        t.step0 = t.slot * split;
        t.steps = max(0, min(split, (int)((p.piece_cols + kVtK - 1) / kVtK) - t.step0));
      } else {
        t.row0 = r * kVtRows;
        t.slot = t.step0 = 0;
        t.steps = (n + kVtK - 1) / kVtK;
      }
    } else {
      tile += kVtPairs;
      if (tile >= count) return false;
      const int per = kVtGroup * nt, g = tile / per, r = tile - g * per, rows = min(kVtGroup, mt - g * kVtGroup);
      t.dx = t.slot = t.step0 = 0;
      t.row0 = (g * kVtGroup + r % rows) * kVtRows;
      t.col0 = r / rows * p.cols;
      t.steps = (p.l.width + kVtK - 1) / kVtK;
    }
    return true;
  }
};

template <typename T> __device__ __forceinline__ uint32_t vt_pack(float a, float b) {
  if constexpr (sizeof(T) == 2 && __is_same(T, __half)) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// Maps: a, b of the logits (x, w, K-major), c: dL; of the gradients dL along and across (a, a2), w across (b), x across (b2), shares of dx
// (c), dw (d).
// kDirect: a tile is one sum (no more than sum_steps stages).
template <int kMode, typename T, bool kDirect>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kVtThreads, 1)
vloss_tc_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_a2,
                const __grid_constant__ CUtensorMap map_b2, const __grid_constant__ CUtensorMap map_c, const __grid_constant__ CUtensorMap map_d,
                const __grid_constant__ VtParams p) {
  extern __shared__ __align__(1024) uint8_t base[];
  VtSmem* sm = reinterpret_cast<VtSmem*>(base + kVtStages * kVtStage + 8 * kVtOut);
  const int tid = threadIdx.x, warp = warp_uniform(tid >> 5), lane = tid & 31;
  const int rank = (int)vt_rank(), pair = blockIdx.x >> 1;
  volatile int* abort_flag = &sm->abort_flag;
  const uint32_t peer_abort = vt_of_rank(smem_u32(&sm->abort_flag), rank ^ 1);
  if (tid == 0) {
    for (int s = 0; s < kVtStages; ++s) { mbar_init(&sm->full[s], 1); mbar_init(&sm->empty[s], 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(&sm->acc_full[s], 1); mbar_init(&sm->acc_empty[s], 16); }
    sm->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm->tmem_base)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
  }
  if (kMode != kVtGrads || p.want_dx) {                    // rows of A that no copy fills: zeros cost the products least power (us of 5 tokens of 151936 x 2048 scored: 122, so 118)
    const int kept = rank < p.a_ranks ? p.a_box * 128 : 0;
    for (int i = kept + tid * 16; i < kVtABytes; i += kVtThreads * 16)
      for (int st = 0; st < kVtStages; ++st) st16(base + st * kVtStage + i, make_uint4(0, 0, 0, 0));
    fence_async_smem();
  }
  grid_dependency_wait();
  grid_launch_dependents();
  tc_fence_before();
  __syncthreads();
  vt_cluster_sync();                                       // both CTAs' barriers are there
  tc_fence_after();
  const uint32_t tmem = sm->tmem_base;
  auto give_up = [&]() {
    if (*abort_flag == 0) { report(p.l.status, TKV_DEV_TIMEOUT); p.l.plan.head[2] = 1; }
    *abort_flag = 1;
    vt_raise(peer_abort);
  };
  if ((smem_u32(base) & 1023u) != 0 && tid == 0) give_up();   // the swizzled tiles need the alignment; the launch gives it
  __syncthreads();
  VtTiles<kMode> tiles(p, pair);
  VtTile t;
  int copies = 0;                                          // stages whose copies this CTA has started

  if (warp == 0) {
    bool ok = (bool)__all_sync(0xffffffffu, *abort_flag == 0);
    int it = 0;
    while (ok && tiles.next(t)) {
      const bool a_mn = kMode == kVtGrads && !t.dx, b_mn = kMode == kVtGrads;
      const int half = kMode == kVtGrads ? kVtCols / 2 : p.cols / 2;
      const int box = a_mn ? 128 : p.a_box, ranks = a_mn ? 2 : p.a_ranks;
      const uint32_t bytes = (ranks * box + 2 * half) * kVtK * 2;        // of both CTAs
      const int arow = t.row0 + rank * 128, brow = t.col0 + rank * half;
      for (int c = p.parts == 1 ? kVtProducts - 1 : 0; ok && c < kVtProducts; ++c)
      for (int k = t.step0; k < t.step0 + t.steps; ++k, ++it) {
        const int s = it % kVtStages;
        const int a_at = vt_part_a(c) * p.rows, x_at = vt_part_b(c) * p.rows, w_at = p.w0 + vt_part_b(c) * p.w_rows;
        ok = warp_wait(&sm->empty[s], ((it / kVtStages) & 1) ^ 1, abort_flag);
        if (!ok) break;
        if (elect_one()) {
          const uint32_t bar = vt_of_rank(smem_u32(&sm->full[s]), 0), a = smem_u32(base + s * kVtStage), b = a + kVtABytes;
          if (rank == 0) mbar_expect_tx(&sm->full[s], bytes);
          if (a_mn) {
            vt_load(a, &map_a2, bar, arow, a_at + k * kVtK);
            vt_load(a + kVtABytes / 2, &map_a2, bar, arow + 64, a_at + k * kVtK);
          } else if (rank < ranks) {                       // rows beyond the box hold what was there: rows of D that nobody reads
            vt_load(a, &map_a, bar, k * kVtK, a_at + arow);
          }
          if (b_mn) {
            const CUtensorMap* mb = t.dx ? &map_b : &map_b2;
            const int y = k * kVtK + (t.dx ? w_at : x_at);
            vt_load(b, mb, bar, brow, y);
            vt_load(b + kVtBBytes / 2, mb, bar, brow + 64, y);
          } else {
            vt_load(b, &map_b, bar, k * kVtK, w_at + brow);
          }
        }
        __syncwarp();
      }
    }
    // the last stages' products are told to this CTA before it may leave
    for (int i = max(0, it - kVtStages); ok && i < it; ++i) ok = warp_wait(&sm->empty[i % kVtStages], (i / kVtStages) & 1, abort_flag);
    if (!ok && lane == 0) give_up();
    copies = it;
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t tm = warp_uniform(tmem);
      const int bf16 = !__is_same(T, __half);
      const uint64_t k_desc = make_desc(smem_u32(base), 16, 1024, 2), mn_desc = make_desc(smem_u32(base), kVtABytes / 2, 1024, 2);
      int it = 0, acc = 0;
      bool ok = (bool)__all_sync(0xffffffffu, *abort_flag == 0);
      while (ok && tiles.next(t)) {
        const bool a_mn = kMode == kVtGrads && !t.dx, b_mn = kMode == kVtGrads;
        const uint32_t idesc = vt_idesc(bf16, a_mn, b_mn, kMode == kVtGrads ? kVtCols : p.cols);
        const int steps = t.steps * (p.parts == 1 ? 1 : kVtProducts);
        for (int k = 0, in_sum = 0; ok && k < max(steps, 1); ++k) {      // (a share without stages: its epilogue writes zeros)
          const int buf = acc & 1;
          if (in_sum == 0) {
            ok = warp_wait(&sm->acc_empty[buf], ((acc >> 1) & 1) ^ 1, abort_flag);
            tc_fence_after();
          }
          const int s = it % kVtStages;
          if (ok && steps > 0) ok = warp_wait(&sm->full[s], (it / kVtStages) & 1, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const bool last = in_sum == p.sum_steps - 1 || k >= steps - 1;
          if (elect_one()) {
            if (steps > 0) {
              const uint64_t at = (uint32_t)s * (kVtStage >> 4);
              const uint64_t a = (a_mn ? mn_desc : k_desc) + at, b = (b_mn ? mn_desc : k_desc) + at + (kVtABytes >> 4);
              const uint32_t da = a_mn ? 128 : 2, db = b_mn ? 128 : 2;
#pragma unroll
              for (int q = 0; q < 4; ++q) vt_mma(tm + buf * kVtCols, a + q * da, b + q * db, idesc, (in_sum > 0 || q > 0));
              vt_commit(&sm->empty[s]);
            }
            if (last) vt_commit(&sm->acc_full[buf]);
          }
          __syncwarp();
          if (steps > 0) ++it;
          ++in_sum;
          if (last) { in_sum = 0; ++acc; }
        }
      }
      if (!ok && lane == 0) give_up();
    }
    __syncwarp();
  } else {
    // ---- epilogue: thread = row of the CTA's half of the tile, and half of its columns; the sums of kVtSum stages are added up here, where
    // additions round.
    const int quarter = warp & 3, row_in = quarter * 32 + lane, c0 = warp >= 6 ? kVtHalf : 0;
    const uint32_t acc_empty0 = vt_of_rank(smem_u32(&sm->acc_empty[0]), 0);
    int acc = 0;
    uint8_t* box = base + kVtStages * kVtStage + (warp - 2) * kVtOut;
    // 32 rows of 128 bytes by a bulk copy: a lane puts the eight 16-byte pieces of its row in the swizzled places.
    auto put = [&](const uint32_t* w) {
      if (lane == 0) tma_store_read();
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i)
        *reinterpret_cast<uint4*>(box + lane * 128 + ((i ^ (lane & 7)) << 4)) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
      fence_async_smem();
      __syncwarp();
    };
    bool ok = *abort_flag == 0;
    while (ok && tiles.next(t)) {
      const int row = t.row0 + rank * 128 + row_in, first = t.row0 + rank * 128 + quarter * 32;
      // columns of this warp that exist, and whether any of its rows is wanted (dL: the products to come read whole steps of rows)
      const int left = (int)min((int64_t)(kMode == kVtGrads ? kVtCols : p.cols), kMode == kVtGrads ? (int64_t)p.l.width - t.col0 : p.piece_cols - t.col0) - c0;
      const bool wanted = left > 0 && first < (kMode == kVtStats || t.dx ? tiles.n : kMode == kVtLogits ? (tiles.n + kVtK - 1) / kVtK * kVtK : (int)p.piece_cols);
      const int steps = t.steps * (p.parts == 1 ? 1 : kVtProducts);
      float v[kVtHalf];
      if (!kDirect || steps == 0) {
#pragma unroll
        for (int i = 0; i < kVtHalf; ++i) v[i] = 0.f;
      }
      for (int k = 0; k < (kDirect ? 1 : max(steps, 1)); k += p.sum_steps) {
        const int buf = acc & 1;
        ok = (bool)__all_sync(0xffffffffu, mbar_wait_or_abort(&sm->acc_full[buf], (acc >> 1) & 1, abort_flag));
        if (!ok) break;
        tc_fence_after();
        const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + buf * kVtCols + c0;
        if (wanted && steps > 0) {                         // (columns beyond the last hold what was there: nobody reads them)
          if constexpr (kDirect) {
#pragma unroll
            for (int c = 0; c < kVtHalf; c += 32) tmem_ld32(from + c, v + c);
          } else {
            const float up = vt_up(min(p.sum_steps, steps - k));
#pragma unroll
            for (int c = 0; c < kVtHalf; c += 16) {
              float u[16];
              tmem_ld16(from + c, u);
#pragma unroll
              for (int i = 0; i < 16; ++i) v[c + i] = fmaf(u[i], up, v[c + i]);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) vt_arrive(acc_empty0 + buf * 8);
        ++acc;
      }
      if (!ok) break;
      if (!wanted) {
        // a half without columns has nothing to say of its rows
        if (kMode == kVtStats && row < tiles.n) p.l.part[(int64_t)row * p.l.tiles + 2 * (p.tile0 + t.col0 / p.cols) + (c0 > 0)] = make_float2(-INFINITY, 0.f);
        continue;
      }
      const float up = kDirect ? vt_up(steps) : 1.f;       // (other sums have it already)
      if constexpr (kMode == kVtStats) {
        const bool live = row < tiles.n;
        const int label = live ? (int)(p.l.plan.label[row] - p.v0 - t.col0) - c0 : -1;
        if ((unsigned)label < (unsigned)min(left, kVtHalf)) {
          float mine = 0.f;
#pragma unroll
          for (int i = 0; i < kVtHalf; ++i) mine = i == label ? v[i] : mine;
          p.l.mine[row] = mine * up;
        }
        __syncwarp();
        if (left < kVtHalf) {
#pragma unroll
          for (int i = 0; i < kVtHalf; ++i) v[i] = i < left ? v[i] : -INFINITY;
        }
        float top[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
        for (int i = 4; i < kVtHalf; i += 8) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            top[j] = i + 4 + j < kVtHalf ? vt_max3(top[j], v[i + j], v[i + 4 + j]) : fmaxf(top[j], v[i + j]);
        }
        top[0] = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        top[0] *= up;
        const float at = top[0] == -INFINITY ? 0.f : top[0];
        const float2 below = make_float2(-at, -at), one = make_float2(1.f, 1.f), ups = make_float2(up, up), by = make_float2(kLog2e, kLog2e), none = make_float2(-0.f, -0.f);
        float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int i = 0; i < kVtHalf; i += 2) {
          const float2 d = fma2(fma2(make_float2(v[i], v[i + 1]), ups, below), by, none);
          sums[(i >> 1) & 1] = fma2(make_float2(exp2_weight(d.x), exp2_weight(d.y)), one, sums[(i >> 1) & 1]);
        }
        if (live) p.l.part[(int64_t)row * p.l.tiles + 2 * (p.tile0 + t.col0 / p.cols) + (c0 > 0)] = make_float2(top[0], (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y));
      } else if constexpr (kMode == kVtLogits) {
        const bool live = row < tiles.n;
        const int label = live ? (int)(p.l.plan.label[row] - p.v0 - t.col0) - c0 : -1;
        const float2 lse = live ? p.l.plan.lse[row] : make_float2(0.f, 0.f);
        const float g = live ? p.l.g[row] : 0.f;
        const float2 below = make_float2(-lse.x, -lse.x), ups = make_float2(up, up), by = make_float2(kLog2e, kLog2e), less = make_float2(-lse.y, -lse.y),
                     gg = make_float2(g, g), none = make_float2(-0.f, -0.f);
        const bool whole = (bool)__all_sync(0xffffffffu, live) && left >= kVtHalf, label_here = (bool)__any_sync(0xffffffffu, (unsigned)label < (unsigned)kVtHalf);
#pragma unroll
        for (int c = 0; c < kVtHalf; c += 64) {            // (the second half is made while the first leaves)
          if (c0 + c >= p.cols) break;
#pragma unroll
          for (int i = c; i < c + 64; i += 2) {
            const float2 d = fma2(fma2(make_float2(v[i], v[i + 1]), ups, below), by, less);
            const float2 e = fma2(make_float2(exp2_weight(d.x), exp2_weight(d.y)), gg, none);
            v[i] = e.x;
            v[i + 1] = e.y;
          }
          if (label_here) {
            const float mine = live ? g * p.l.plan.own[row] : 0.f;
#pragma unroll
            for (int i = c; i < c + 64; ++i) v[i] = i == label ? mine : v[i];
            if (sizeof(T) == 2 && (unsigned)(label - c) < 64u && label < left) p.l.rest[row] = mine - round_as<T>(mine);
          }
          if (!whole) {
#pragma unroll
            for (int i = c; i < c + 64; ++i) v[i] = live && i < left ? v[i] : 0.f;   // rows and columns that do not exist are zeros for the products to come
          }
#pragma unroll
          for (int part = 0; part < (sizeof(T) == 4 ? 3 : 1); ++part) {
            uint32_t w[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              w[i] = vt_pack<T>(v[c + 2 * i], v[c + 2 * i + 1]);
              if (sizeof(T) == 4) { v[c + 2 * i] -= __uint_as_float(w[i] << 16); v[c + 2 * i + 1] -= __uint_as_float(w[i] & 0xffff0000u); }
            }
            put(w);
            if (lane == 0) tma_store_2d(&map_c, box, t.col0 + c0 + c, part * p.rows + first);
          }
        }
      } else {
        const float back = t.dx ? 1.f : p.l.g_scale[1];
        if constexpr (sizeof(T) == 2) {
          if (!t.dx && tiles.n <= kVtExact) {
            int room = kVtExactHits;
            for (int i0 = 0; i0 < tiles.n && room > 0; i0 += 32) {
              const int y = i0 + lane < tiles.n ? (int)(p.l.plan.label[i0 + lane] - p.v0 - first) : -1;
              for (unsigned hits = __ballot_sync(0xffffffffu, (unsigned)y < 32u); hits != 0 && room > 0; hits &= hits - 1, --room) {
                const int j = __ffs(hits) - 1, i = i0 + j, who = __shfl_sync(0xffffffffu, y, j);
                const T* x = reinterpret_cast<const T*>(p.xc) + (int64_t)i * p.l.width + t.col0 + c0;
                if (lane == who) {
                  const float r = p.l.rest[i];
#pragma unroll
                  for (int c = 0; c < kVtHalf; c += 8) {
                    if (c >= left) break;
                    float u[8];
                    load_vec<8>(x + c, u);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[c + e] += r * u[e];
                  }
                }
                __syncwarp();
              }
            }
          }
        }
        if (t.dx || sizeof(T) == 4) {                      // a share's rows are whole tiles
#pragma unroll
          for (int c = 0; c < kVtHalf; c += 32) {
            if (c >= left) break;
            if (!t.dx) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[c + i] *= back;
            }
            put(reinterpret_cast<const uint32_t*>(v + c));
            if (lane == 0) {
              const int y = t.slot * tiles.mt * kVtRows + first;
              if (!t.dx) tma_store_2d(&map_d, box, t.col0 + c0 + c, (int)p.v0 + first);
              else if (p.more) tma_add_2d(&map_c, box, t.col0 + c0 + c, y);
              else tma_store_2d(&map_c, box, t.col0 + c0 + c, y);
            }
          }
        } else {
#pragma unroll
          for (int c = 0; c < kVtHalf; c += 64) {
            if (c >= left) break;
            uint32_t w[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) w[i] = vt_pack<T>(v[c + 2 * i] * back, v[c + 2 * i + 1] * back);
            put(w);
            if (lane == 0) tma_store_2d(&map_d, box, t.col0 + c0 + c, (int)p.v0 + first);
          }
        }
      }
    }
    if (lane == 0 && kMode != kVtStats) tma_store_done();
    if (!ok && lane == 0) give_up();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && rank == 0 && *abort_flag != 0)           // copies in flight, the neighbour's too, land before the shared memory is released
    for (int i = max(0, copies - kVtStages); i < copies; ++i) mbar_wait(&sm->full[i % kVtStages], (i / kVtStages) & 1);
  __syncthreads();
  vt_cluster_sync();                                       // nobody reads or signals a CTA that has left
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

// -------------------------------------------------------------------------------------------------- rows that count, together
constexpr int kVtGatherThreads = 256;

// Eight elements as they are stored for the products: themselves, or (fp32) their three parts.
template <typename T, bool kVec> __device__ __forceinline__ void vt_take(const T* in, uint16_t* out, int64_t part) {
  if constexpr (sizeof(T) == 2) {
    if (kVec) st16(out, ld16_stream(in));
    else
      for (int e = 0; e < 8; ++e) out[e] = in[e];
  } else {
    float v[8];
    if (kVec) load_vec<8>(in, v);
    else
      for (int e = 0; e < 8; ++e) v[e] = in[e];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = vt_pack<float>(v[2 * i], v[2 * i + 1]);
        v[2 * i] -= __uint_as_float(w[i] << 16);
        v[2 * i + 1] -= __uint_as_float(w[i] & 0xffff0000u);
      }
      st16(out + k * part, make_uint4(w[0], w[1], w[2], w[3]));
    }
  }
}
template <typename T> __device__ __forceinline__ void vt_zero(uint16_t* out, int64_t part) {
  for (int k = 0; k < (sizeof(T) == 4 ? 3 : 1); ++k) st16(out + k * part, make_uint4(0, 0, 0, 0));
}

// Row i of xc is the row of the i-th token that counts; zeros up to the end of the last tile of rows.  T: uint16_t or float.
template <typename T, bool kVec> __global__ void __launch_bounds__(kVtGatherThreads) vloss_gather_kernel(const T* x, int64_t x_stride, VlossPlan plan, int width, uint16_t* xc, int64_t part) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int n = plan.head[0];
  const int64_t i = blockIdx.x;
  if (i >= ((int64_t)n + kVtRows - 1) / kVtRows * kVtRows) return;
  uint16_t* out = xc + i * width;
  const T* in = x + (i < n ? (int64_t)plan.rows[i] : 0) * x_stride;
  for (int c = threadIdx.x * 8; c < width; c += kVtGatherThreads * 8) {
    if (i < n) vt_take<T, kVec>(in + c, out + c, part);
    else vt_zero<T>(out + c, part);
  }
}

// The three parts of a piece of w (fp32), zeros behind its last row up to a whole step.
__global__ void __launch_bounds__(kVtGatherThreads) vloss_parts_kernel(const float* w, int64_t n, int64_t whole, uint16_t* out, int64_t part) {
  grid_dependency_wait();
  grid_launch_dependents();
  for (int64_t i = ((int64_t)blockIdx.x * kVtGatherThreads + threadIdx.x) * 8; i < whole; i += (int64_t)gridDim.x * kVtGatherThreads * 8) {
    if (i < n) vt_take<float, true>(w + i, out + i, part);
    else vt_zero<float>(out + i, part);
  }
}

constexpr int kVtFirst = 1024;                             // most tokens for which every CTA can look through the labels itself

// vloss_plan_kernel and vloss_gather_kernel in one launch, for few tokens: every CTA finds its row among the labels.  The grid is the rows
// that the logits' boxes reach.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kVtGatherThreads) vloss_first_kernel(const int64_t* labels, int64_t ignore, int tokens, int64_t vocab, VlossPlan plan, float* loss,
                                                                     int32_t* status, const T* x, int64_t x_stride, int width, uint16_t* xc, int64_t part) {
  constexpr int kPer = kVtFirst / kVtGatherThreads;
  __shared__ int sums[kVtGatherThreads / 32 + 1], token, bad_any;
  grid_dependency_wait();
  grid_launch_dependents();
  if (threadIdx.x == 0) bad_any = 0;
  int64_t y[kPer];
  int n = 0;
  bool bad = false;
  const int t1 = threadIdx.x * kPer;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    y[i] = t1 + i < tokens ? labels[t1 + i] : ignore;
    const bool off = y[i] != ignore && (y[i] < 0 || y[i] >= vocab);
    if (blockIdx.x == 0 && t1 + i < tokens && (off || y[i] == ignore)) loss[t1 + i] = off ? __int_as_float(0x7fffffff) : 0.f;
    bad |= off;
    if (off) y[i] = ignore;
    n += y[i] != ignore;
  }
  if (bad) bad_any = 1;
  int total;
  int at = block_exclusive_scan<kVtGatherThreads>(n, sums, &total);
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (y[i] != ignore) {
      if (at == (int)blockIdx.x) token = t1 + i;
      if (blockIdx.x == 0) { plan.rows[at] = t1 + i; plan.label[at] = (int32_t)y[i]; }
      ++at;
    }
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    plan.head[0] = total; plan.head[1] = bad_any; plan.head[2] = plan.head[3] = 0;
    if (bad_any) report(status, TKV_DEV_BAD_INDEX);
  }
  if ((int)blockIdx.x >= (total + kVtRows - 1) / kVtRows * kVtRows) return;
  uint16_t* out = xc + (int64_t)blockIdx.x * width;
  const bool live = (int)blockIdx.x < total;
  const T* in = x + (live ? token : 0) * x_stride;
  for (int c = threadIdx.x * 8; c < width; c += kVtGatherThreads * 8) {
    if (live) vt_take<T, kVec>(in + c, out + c, part);
    else vt_zero<T>(out + c, part);
  }
}

// ------------------------------------------------------------------------------------------------------------------ the host
bool vloss_tc_shape(int tokens, int64_t vocab, int width, int dtype) { return elem_size(dtype) != 0 && width % 8 == 0 && tokens > 0; }
static int vt_parts(int dtype) { return dtype == TKV_F32 ? 3 : 1; }

// ---------------------------------------------------------------------------------------------- a handful of tokens, CUDA cores
// Logits of up to four tokens in 16 bits, bound by the weight's bytes: a warp takes four words at a time, a lane eight columns of every 256 of
// each, and keeps the largest logit and the sum of one of the 4 kR (word, token) pairs while it goes through the vocabulary, so that a CTA
// writes one pair of numbers for a token.  us of 151936 words, width 2048, 1, 2 and 4 tokens: 96, 98, 110; on the tensor cores,
// where these few no longer go, 113, 116, 121.  8 tokens would take 273 here for 118 there: 8 x 311e6 products are more than the bytes.
// One run of columns requested ahead 117 (1 token), two 98, three 96; three CTAs an SM, with fewer registers, 103 to 227.
constexpr int kVwThreads = 256, kVwWords = 4, kVwCols = 256, kVwCtas = 2, kVwGrid = 148 * kVwCtas, kVwTokens = 4;
constexpr int kVwValues = 16384, kVwBytes = 2 * kVwValues * 4;   // x in shared memory: tokens up to a power of two, whole runs of 256 columns

static int64_t vt_rows(int tokens) { return vl_round(tokens, kVtRows); }
// Columns of a tile: what a pair does in its rounds is rounds x columns, and a little per round; few rounds make it matter that the last
// one is full.  us of 5 tokens scored, 151936 words, width 2048: 256 columns 120.3, by this rule (208) 118.3.
static int vt_tile_cols(int tokens, int64_t vocab, int step) {
  const int64_t mt = vt_rows(tokens) / kVtRows;
  if (mt * ((vocab + kVtCols - 1) / kVtCols) > 20 * kVtPairs) return kVtCols;
  int best = kVtCols;
  int64_t least = INT64_MAX;
  for (int cols = kVtCols; cols >= 64; cols -= step) {
    const int64_t rounds = (mt * ((vocab + cols - 1) / cols) + kVtPairs - 1) / kVtPairs;
    if (rounds * (cols + 16) < least) { least = rounds * (cols + 16); best = cols; }
  }
  return best;
}
static int vt_a_box(int tokens) { return tokens >= 128 ? 128 : (int)vl_round(tokens, 8); }
// The vocabulary in equal pieces: of at most 256 MB of dL where that is not fewer than 8192 words (so from 16385 tokens on dL is larger, 16 KB a
// token); fp32: of at most 96 MB of parts of w too, and not fewer than 2048 words (from 21846 tokens on dL is 12 KB a token).
static int64_t vt_piece(int tokens, int64_t vocab, int width, int dtype) {
  int64_t n = ((int64_t)256 << 20) / (2 * vt_parts(dtype) * vt_rows(tokens));
  int64_t least = 8192;
  if (dtype == TKV_F32) {
    const int64_t w = ((int64_t)96 << 20) / (6 * (int64_t)width);
    if (n > w) n = w;
    least = 2048;
  }
  n = n / kVtCols * kVtCols;
  if (n < least) n = least;
  const int64_t pieces = (vocab + n - 1) / n;
  return vl_round((vocab + pieces - 1) / pieces, kVtCols);
}
// Room for shares of dx.  How many there are is decided on the device, where the number of tokens that count is known (vloss_rows_grad_kernel):
// a tile of dx is as long as the piece, and its few tiles rarely fill whole rounds of the pairs.
static int vt_slots(int tokens, int width) {
  const int64_t tiles = vt_rows(tokens) / kVtRows * ((width + kVtCols - 1) / kVtCols);
  const int64_t s = (8 * kVtPairs + tiles - 1) / tiles;
  return (int)(s > kVlMaxSlots ? kVlMaxSlots : s < 1 ? 1 : s);
}
VlossWork vloss_tc_work(int tokens, int64_t vocab, int width, int dtype, bool want_dx, bool want_dw) {
  const int64_t piece = vt_piece(tokens, vocab, width, dtype);
  return {kVtPairs, kVtRows, kVtRows, (width + kVtCols - 1) / kVtCols, (int)((piece + kVtRows - 1) / kVtRows), (int)(piece / kVtK), kVtK, vt_slots(tokens, width), (int)vt_rows(tokens),
          kVlMaxSlots, want_dx, want_dw};
}

static bool vw_shape(int tokens, int width, int dtype) { return dtype != TKV_F32 && tokens <= kVwTokens && (int64_t)tokens * width <= kVwValues; }

// What lies where in a workspace.
struct VtRoom {
  int64_t rows, piece, xc, w, dl, acc, part, bytes;        // bytes from the start
  int cols, tiles;                                         // columns of a tile; halves of tiles
  VtRoom(int tokens, int64_t vocab, int width, int dtype, bool backward, bool dx) {
    const int64_t parts = vt_parts(dtype);
    auto pad = [](int64_t n) { return vl_round(n, 1024); };
    rows = vt_rows(tokens);
    piece = backward || parts == 3 ? vt_piece(tokens, vocab, width, dtype) : vocab;
    cols = vt_tile_cols(tokens, piece, backward ? 64 : 16);   // dL leaves in boxes of 64 columns
    const int64_t before = (vocab - 1) / piece;              // whole pieces before the last
    tiles = (int)(before * ((piece + cols - 1) / cols) + (vocab - before * piece + cols - 1) / cols) * 2;
    xc = 0;
    w = xc + pad(parts * rows * width * 2);
    dl = w + (parts == 3 ? pad(3 * piece * width * 2) : 0);
    acc = dl + (backward ? pad(parts * rows * piece * 2) : 0);
    part = acc + (backward && dx ? pad((int64_t)vt_slots(tokens, width) * rows * width * 4) : 0);
    bytes = part + (backward ? 0 : pad((int64_t)tokens * (vw_shape(tokens, width, dtype) && kVwGrid > tiles ? kVwGrid : tiles) * 8));
  }
};
int64_t vloss_tc_bytes(int tokens, int64_t vocab, int width, int dtype, bool backward, bool dx) { return 1024 + VtRoom(tokens, vocab, width, dtype, backward, dx).bytes; }

static int vt_check(cudaError_t e) { return e == cudaSuccess ? check_launch("tkv_vloss") : fail(TKV_ERR_LAUNCH, "tkv_vloss: %s", cudaGetErrorString(e)); }

template <typename T> static int vt_gather(const Vloss& p, void* xc, cudaStream_t st) {
  const bool vec = aligned16(p.x) && p.x_stride % (16 / (int64_t)sizeof(T)) == 0;
  return vt_check(launch_pdl(vec ? vloss_gather_kernel<T, true> : vloss_gather_kernel<T, false>, dim3((unsigned)vt_rows(p.tokens)), dim3(kVtGatherThreads), 0, st,
                             reinterpret_cast<const T*>(p.x), p.x_stride, p.plan, p.width, reinterpret_cast<uint16_t*>(xc), vt_rows(p.tokens) * p.width));
}
template <typename T> static int vt_first(const Vloss& p, const int64_t* labels, int64_t ignore, float* loss, void* xc, cudaStream_t st) {
  const bool vec = aligned16(p.x) && p.x_stride % (16 / (int64_t)sizeof(T)) == 0;
  return vt_check(launch_pdl(vec ? vloss_first_kernel<T, true> : vloss_first_kernel<T, false>, dim3((unsigned)(p.tokens > 128 ? vt_rows(p.tokens) : vt_a_box(p.tokens))),
                             dim3(kVtGatherThreads), 0, st, labels, ignore, p.tokens, p.vocab, p.plan, loss, p.status, reinterpret_cast<const T*>(p.x), p.x_stride, p.width,
                             reinterpret_cast<uint16_t*>(xc), vt_rows(p.tokens) * p.width));
}
// fp32: the parts of the piece of w at v0.
static int vt_parts_of(const VtParams& p, const VtRoom& room, void* w, cudaStream_t st) {
  if (p.parts == 1) return TKV_OK;
  const int64_t whole = vl_round(p.piece_cols, kVtK) * p.l.width;
  const int64_t blocks = (whole + kVtGatherThreads * 8 - 1) / (kVtGatherThreads * 8);
  return vt_check(launch_pdl(vloss_parts_kernel, dim3((unsigned)(blocks < 148 * 16 ? blocks : 148 * 16)), dim3(kVtGatherThreads), 0, st,
                             reinterpret_cast<const float*>(p.l.w) + p.v0 * p.l.width, p.piece_cols * p.l.width, whole, reinterpret_cast<uint16_t*>(w), room.piece * p.l.width));
}

template <int kMode, typename T, bool kDirect> static int vt_launch(const CUtensorMap* m, const VtParams& p, cudaStream_t st) {
  static bool allowed[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev < 0 || dev >= 64 || !allowed[dev])) {
    e = cudaFuncSetAttribute(vloss_tc_kernel<kMode, T, kDirect>, cudaFuncAttributeMaxDynamicSharedMemorySize, kVtSmemBytes);
    if (e == cudaSuccess && dev >= 0 && dev < 64) allowed[dev] = true;
  }
  if (e == cudaSuccess) e = launch_pdl(vloss_tc_kernel<kMode, T, kDirect>, dim3(2 * kVtPairs), dim3(kVtThreads), (size_t)kVtSmemBytes, st, m[0], m[1], m[2], m[3], m[4], m[5], p);
  return vt_check(e);
}
template <int kMode, typename T> static int vt_launch(const CUtensorMap* m, const VtParams& p, cudaStream_t st) {
  // the longest tile: the width (logits), the piece and the tokens (gradients)
  const int64_t inner = kMode == kVtGrads ? (p.piece_steps > vt_rows(p.l.tokens) / kVtK ? p.piece_steps : vt_rows(p.l.tokens) / kVtK) : (p.l.width + kVtK - 1) / kVtK;
  return inner * (p.parts == 1 ? 1 : kVtProducts) <= p.sum_steps ? vt_launch<kMode, T, true>(m, p, st) : vt_launch<kMode, T, false>(m, p, st);
}
template <int kMode> static int vt_launch(const CUtensorMap* m, const VtParams& p, cudaStream_t st) {
  return p.l.dtype == TKV_BF16 ? vt_launch<kMode, __nv_bfloat16>(m, p, st) : p.l.dtype == TKV_F16 ? vt_launch<kMode, __half>(m, p, st) : vt_launch<kMode, float>(m, p, st);
}

// Sums over the lanes of N values a lane, in lane l that of value l N / 32: every exchange over O lanes halves what is left to a lane.
template <int N, int O = 16> __device__ __forceinline__ float vw_sums(float (&v)[N], int lane) {
  if constexpr (N == 1) {
    float s = v[0];
#pragma unroll
    for (int o = O; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
  } else {
    float u[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float mine = lane & O ? v[N / 2 + i] : v[i], other = lane & O ? v[i] : v[N / 2 + i];
      u[i] = mine + __shfl_xor_sync(0xffffffffu, other, O);
    }
    return vw_sums<N / 2, O / 2>(u, lane);
  }
}
__device__ __forceinline__ void vw_floats(const uint4& r, float2* v, __nv_bfloat16) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
__device__ __forceinline__ void vw_floats(const uint4& r, float2* v, __half) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
}
// A largest value and the sum of the weights beside it, joined with another's.
__device__ __forceinline__ float2 vw_join(float2 a, float2 b) {
  const float top = fmaxf(a.x, b.x);
  return make_float2(top, a.y * vl_weight(a.x, top) + b.y * vl_weight(b.x, top));
}

template <typename T, int kR> __global__ void __launch_bounds__(kVwThreads, kVwCtas) vloss_words_kernel(const __grid_constant__ Vloss p, const T* xc) {
  extern __shared__ __align__(16) float4 vw_x[];            // [token][half of eight columns][eight columns], zeros behind the last
  __shared__ float2 join[kVwThreads];
  grid_dependency_wait();
  grid_launch_dependents();
  const int n = p.plan.head[0], lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (n == 0) return;                                      // nothing counts: nobody reads the parts
  const int chunks = (p.width + kVwCols - 1) / kVwCols, eights = chunks * 32;
  for (int i = threadIdx.x; i < kR * eights; i += kVwThreads) {
    const int r = i / eights, c = i - r * eights;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (r < n && c * 8 < p.width) load_vec<8>(xc + (int64_t)r * p.width + c * 8, v);
    vw_x[(r * 2 + 0) * eights + c] = make_float4(v[0], v[1], v[2], v[3]);
    vw_x[(r * 2 + 1) * eights + c] = make_float4(v[4], v[5], v[6], v[7]);
  }
  __syncthreads();
  constexpr int kEach = 32 / (kVwWords * kR);              // lanes with the same word and token
  const int at = lane / kEach, r = at % kR, j = at / kR;
  const int64_t label = r < n ? p.plan.label[r] : -1;
  float2 mine = make_float2(-INFINITY, 0.f);
  const T* w = reinterpret_cast<const T*>(p.w);
  constexpr int kVwAhead = kR <= 2 ? 3 : 2;
  // Eight columns of four words, kVwAhead of them requested before they are used: across the end of a row too.
  const int64_t step = (int64_t)gridDim.x * (kVwThreads / 32) * kVwWords;
  int64_t v0 = ((int64_t)blockIdx.x * (kVwThreads / 32) + warp) * kVwWords, v_in = v0;
  const T* row[kVwWords];
  int c_in = 0, c = 0;
  auto rows = [&]() {
#pragma unroll
    for (int i = 0; i < kVwWords; ++i) row[i] = w + min(v_in + i, p.vocab - 1) * p.width + lane * 8;
  };
  rows();
  uint4 ahead[kVwAhead][kVwWords];
  auto fetch = [&](uint4 (&to)[kVwWords]) {
    const bool in = v_in < p.vocab && c_in * kVwCols + lane * 8 < p.width;
#pragma unroll
    for (int i = 0; i < kVwWords; ++i) to[i] = in ? ld16_stream(row[i] + c_in * kVwCols) : make_uint4(0, 0, 0, 0);
    if (++c_in == chunks) { c_in = 0; v_in += step; rows(); }
  };
#pragma unroll
  for (int b = 0; b < kVwAhead; ++b) fetch(ahead[b]);
  float2 acc[kVwWords * kR];
#pragma unroll
  for (int i = 0; i < kVwWords * kR; ++i) acc[i] = make_float2(0.f, 0.f);
  while (v0 < p.vocab) {
#pragma unroll
    for (int b = 0; b < kVwAhead; ++b) {
      if (v0 >= p.vocab) break;
      float2 f[kVwWords][4];
#pragma unroll
      for (int i = 0; i < kVwWords; ++i) vw_floats(ahead[b][i], f[i], T());
      fetch(ahead[b]);
#pragma unroll
      for (int t = 0; t < kR; ++t) {
        const float4 x0 = vw_x[(t * 2 + 0) * eights + c * 32 + lane], x1 = vw_x[(t * 2 + 1) * eights + c * 32 + lane];
#pragma unroll
        for (int i = 0; i < kVwWords; ++i) {
          float2& s = acc[i * kR + t];
          s = fma2(make_float2(x0.x, x0.y), f[i][0], s);
          s = fma2(make_float2(x0.z, x0.w), f[i][1], s);
          s = fma2(make_float2(x1.x, x1.y), f[i][2], s);
          s = fma2(make_float2(x1.z, x1.w), f[i][3], s);
        }
      }
      if (++c < chunks) continue;
      float sums[kVwWords * kR];
#pragma unroll
      for (int i = 0; i < kVwWords * kR; ++i) {
        sums[i] = acc[i].x + acc[i].y;
        acc[i] = make_float2(0.f, 0.f);
      }
      const float s = vw_sums(sums, lane);
      if (v0 + j < p.vocab) {
        if (v0 + j == label && lane % kEach == 0) p.mine[r] = s;
        mine = vw_join(mine, make_float2(s, 1.f));
      }
      c = 0;
      v0 += step;
    }
  }
  join[threadIdx.x] = mine;
  __syncthreads();
  if (threadIdx.x < n) {                                   // (n <= kR)
    float2 all = make_float2(-INFINITY, 0.f);
    for (int i = 0; i < kVwThreads / 32 * kVwWords; ++i) all = vw_join(all, join[(i / kVwWords) * 32 + ((i % kVwWords) * kR + threadIdx.x) * kEach]);
    p.part[(int64_t)threadIdx.x * p.tiles + blockIdx.x] = all;
  }
}

template <typename T, int kR> static int vw_launch(const Vloss& p, const void* xc, cudaStream_t st) {
  const int bytes = kR * ((p.width + kVwCols - 1) / kVwCols) * kVwCols * 4;
  cudaError_t e = cudaFuncSetAttribute(vloss_words_kernel<T, kR>, cudaFuncAttributeMaxDynamicSharedMemorySize, kVwBytes);
  if (e == cudaSuccess) e = launch_pdl(vloss_words_kernel<T, kR>, dim3((unsigned)p.tiles), dim3(kVwThreads), (size_t)bytes, st, p, reinterpret_cast<const T*>(xc));
  return vt_check(e);
}
template <typename T> static int vw_launch(const Vloss& p, const void* xc, cudaStream_t st) {
  return p.tokens == 1 ? vw_launch<T, 1>(p, xc, st) : p.tokens == 2 ? vw_launch<T, 2>(p, xc, st) : vw_launch<T, 4>(p, xc, st);
}

static char* vt_align(void* p) { return reinterpret_cast<char*>(((uintptr_t)p + 1023) & ~(uintptr_t)1023); }

static VtParams vt_params(const Vloss& l, const VtRoom& room, const void* base) {
  VtParams p = {};
  p.l = l;
  p.cols = room.cols;
  p.a_box = vt_a_box(l.tokens);
  p.a_ranks = l.tokens > 128 ? 2 : 1;
  p.parts = vt_parts(l.dtype);
  p.rows = (int)room.rows;
  p.w_rows = (int)room.piece;
  p.sum_steps = p.parts == 1 ? kVtSum : kVtSum32;
  p.xc = base;
  return p;
}
static void vt_piece_at(VtParams* p, const VtRoom& room, int64_t v0) {
  p->v0 = v0;
  p->piece_cols = p->l.vocab - v0 < room.piece ? p->l.vocab - v0 : room.piece;
  p->w0 = p->parts == 1 ? (int)v0 : 0;
  p->tile0 = (int)(v0 / room.piece * ((room.piece + room.cols - 1) / room.cols));
  p->more = v0 > 0;
}

int vloss_tc_forward(Vloss& l, const int64_t* labels, int64_t ignore, float* loss, void* ws, cudaStream_t st) {
  const VtRoom room(l.tokens, l.vocab, l.width, l.dtype, false, false);
  char* base = vt_align(ws);
  const bool f32 = l.dtype == TKV_F32;
  int rc;
  if (l.tokens <= kVtFirst) {
    rc = f32 ? vt_first<float>(l, labels, ignore, loss, base, st) : vt_first<uint16_t>(l, labels, ignore, loss, base, st);
  } else {
    rc = vloss_plan_rows(l, labels, ignore, loss, st);
    if (rc == TKV_OK) rc = f32 ? vt_gather<float>(l, base, st) : vt_gather<uint16_t>(l, base, st);
  }
  l.part = reinterpret_cast<float2*>(base + room.part);
  if (vw_shape(l.tokens, l.width, l.dtype)) {
    const int64_t groups = (l.vocab + kVwThreads / 32 * kVwWords - 1) / (kVwThreads / 32 * kVwWords);
    l.tiles = (int)(groups < kVwGrid ? groups : kVwGrid);
    return rc != TKV_OK ? rc : l.dtype == TKV_BF16 ? vw_launch<__nv_bfloat16>(l, base, st) : vw_launch<__half>(l, base, st);
  }
  l.tiles = room.tiles;
  VtParams p = vt_params(l, room, base);
  const int type = f32 ? TKV_BF16 : l.dtype;
  const void* w = f32 ? (const void*)(base + room.w) : l.w;
  CUtensorMap m[6];
  if (rc == TKV_OK) rc = make_map_wide(&m[0], base, l.width, p.parts * room.rows, kVtK, p.a_box, type);
  if (rc == TKV_OK) rc = make_map_wide(&m[1], w, l.width, f32 ? 3 * room.piece : l.vocab, kVtK, p.cols / 2, type);
  if (rc != TKV_OK) return rc;
  m[2] = m[3] = m[4] = m[5] = m[0];
  for (int64_t v0 = 0; v0 < l.vocab && rc == TKV_OK; v0 += room.piece) {
    vt_piece_at(&p, room, v0);
    rc = vt_parts_of(p, room, base + room.w, st);
    if (rc == TKV_OK) rc = vt_launch<kVtStats>(m, p, st);
  }
  return rc;
}

int vloss_tc_backward(Vloss& l, void* ws, bool want_dx, cudaStream_t st) {
  const VtRoom room(l.tokens, l.vocab, l.width, l.dtype, true, want_dx);
  char* base = vt_align(ws);
  const bool f32 = l.dtype == TKV_F32;
  l.dl = base + room.dl;
  l.acc = reinterpret_cast<float*>(base + room.acc);
  VtParams p = vt_params(l, room, base);
  p.want_dx = want_dx;
  p.want_dw = l.dw != nullptr;
  p.piece_steps = room.piece / kVtK;
  const int type = f32 ? TKV_BF16 : l.dtype;
  const void* w = f32 ? (const void*)(base + room.w) : l.w;
  const int64_t rows = p.parts * room.rows, w_rows = f32 ? 3 * room.piece : l.vocab;
  CUtensorMap a[6], g[6];
  int rc = f32 ? vt_gather<float>(l, base, st) : vt_gather<uint16_t>(l, base, st);
  if (rc == TKV_OK) rc = make_map_wide(&a[0], base, l.width, rows, kVtK, p.a_box, type);
  if (rc == TKV_OK) rc = make_map_wide(&a[1], w, l.width, w_rows, kVtK, p.cols / 2, type);
  if (rc == TKV_OK) rc = make_map_wide(&a[4], l.dl, room.piece, rows, 64, 32, type);
  if (rc == TKV_OK) rc = make_map_wide(&g[0], l.dl, room.piece, rows, kVtK, p.a_box, type);
  if (rc == TKV_OK) rc = make_map_wide(&g[1], w, l.width, w_rows, 64, kVtK, type);
  if (rc == TKV_OK) rc = make_map_wide(&g[2], l.dl, room.piece, rows, 64, kVtK, type);
  if (rc == TKV_OK) rc = make_map_wide(&g[3], base, l.width, rows, 64, kVtK, type);
  if (rc == TKV_OK && want_dx) rc = make_map_wide(&g[4], l.acc, l.width, (int64_t)vt_slots(l.tokens, l.width) * room.rows, 32, 32, TKV_F32);
  if (rc == TKV_OK && l.dw) rc = make_map_wide(&g[5], l.dw, l.width, l.vocab, f32 ? 32 : 64, 32, l.dtype);
  if (rc != TKV_OK) return rc;
  a[2] = a[3] = a[5] = a[0];
  if (!want_dx) g[4] = g[0];
  if (l.dw == nullptr) g[5] = g[0];
  for (int64_t v0 = 0; v0 < l.vocab && rc == TKV_OK; v0 += room.piece) {
    vt_piece_at(&p, room, v0);
    rc = vt_parts_of(p, room, base + room.w, st);
    p.sum_steps = f32 ? kVtSum32 : kVtSum;
    if (rc == TKV_OK) rc = vt_launch<kVtLogits>(a, p, st);
    if (!f32) p.sum_steps = kVtSumGrad;
    if (rc == TKV_OK) rc = vt_launch<kVtGrads>(g, p, st);
  }
  return rc;
}

}  // namespace tkv
