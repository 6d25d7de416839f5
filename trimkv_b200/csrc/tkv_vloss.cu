// Cross entropy against a vocabulary (tkv_vloss.cuh): the plan, the joining of the tiles' shares, the gradients of the rows, the entry
// points, and the form for every type, width and alignment, on the CUDA cores.
//
// The CUDA-core products take tiles of 128 x 128 over steps of 16 of the inner axis, 8 x 8 results a thread, the next step's operands in
// registers meanwhile: bound by the fp32 multiply-adds.
#include "tkv_vloss.cuh"

namespace tkv {

// ------------------------------------------------------------------------------------------------------------------ the plan
constexpr int kPlanThreads = 1024, kPlanPer = 8;

// Rows and labels of the tokens that count, in order; loss 0 for ignored ones, NaN for labels out of range (they do not count).
__global__ void __launch_bounds__(kPlanThreads) vloss_plan_kernel(const int64_t* labels, int64_t ignore, int tokens, int64_t vocab, VlossPlan plan,
                                                                  float* loss, int32_t* status) {
  __shared__ int sums[kPlanThreads / 32 + 1];
  __shared__ int bad_any;
  grid_dependency_wait();
  grid_launch_dependents();
  if (threadIdx.x == 0) bad_any = 0;
  int base = 0;
  bool bad = false;
  __syncthreads();
  for (int64_t t0 = 0; t0 < tokens; t0 += kPlanThreads * kPlanPer) {
    int64_t y[kPlanPer];
    int n = 0;
    const int64_t t1 = t0 + (int64_t)threadIdx.x * kPlanPer;
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i) {
      y[i] = t1 + i < tokens ? labels[t1 + i] : ignore;
      const bool off = y[i] != ignore && (y[i] < 0 || y[i] >= vocab);
      if (t1 + i < tokens && (off || y[i] == ignore)) loss[t1 + i] = off ? __int_as_float(0x7fffffff) : 0.f;
      bad |= off;
      if (off) y[i] = ignore;
      n += y[i] != ignore;
    }
    int total;
    int at = base + block_exclusive_scan<kPlanThreads>(n, sums, &total);
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i)
      if (y[i] != ignore) { plan.rows[at] = (int32_t)(t1 + i); plan.label[at] = (int32_t)y[i]; ++at; }
    base += total;
  }
  if (bad) { bad_any = 1; report(status, TKV_DEV_BAD_INDEX); }
  __syncthreads();
  if (threadIdx.x == 0) { plan.head[0] = base; plan.head[1] = bad_any; plan.head[2] = plan.head[3] = 0; }
}

// --------------------------------------------------------------------------------------------------------------- the products
constexpr int kVgThreads = 256, kVgTile = 128, kVgK = 16, kVgPitch = kVgTile + 4;

enum { kVgStats, kVgLogitGrad, kVgShare, kVgOut };

struct VgOperand {                                         // element (i, k): K-major p[row(i) * ld + k], else p[row(k) * ld + i]
  const void* p; int64_t ld;
  const int32_t* rows;                                     // of the axis that steps by ld, or NULL
  int vec;                                                 // four elements may be read at once
};
struct VgProduct {
  VgOperand a, b;
  int64_t m, n, k;                                         // where the token axis is one of them, at most *count of it
  const int32_t* count;
  int token_axis;                                          // 0: m, 2: k
  int mt;                                                  // tiles along m; blockIdx.x goes through them, then along n
  int64_t col0;                                            // column 0 is this of the vocabulary
  int split; int64_t split_len;                            // kVgShare: most shares; the whole of k
  int more;                                                // shares are added to what is there
  Vloss l;
};

template <typename T> __device__ __forceinline__ void vg_load4(const T* p, int64_t left, bool vec, float* v) {
  if (vec && left >= 4) {
    if constexpr (sizeof(T) == 4) {
      const float4 x = *reinterpret_cast<const float4*>(p);
      v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    } else {
      alignas(8) T e[4];
      *reinterpret_cast<uint2*>(e) = *reinterpret_cast<const uint2*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = to_f32<T>(e[i]);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = i < left ? to_f32<T>(p[i]) : 0.f;
}
// This thread's 8 of the 128 x 16 elements of a step.
template <typename T, bool kKMajor> __device__ __forceinline__ void vg_fetch(const VgOperand& o, int64_t i0, int64_t ni, int64_t k0, int64_t k1, float* v) {
  const T* base = reinterpret_cast<const T*>(o.p);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float* u = v + 4 * h;
    if constexpr (kKMajor) {
      const int64_t i = i0 + (threadIdx.x >> 2) + 64 * h, k = k0 + (threadIdx.x & 3) * 4;
      if (i < ni && k < k1) vg_load4(base + (o.rows ? (int64_t)o.rows[i] : i) * o.ld + k, k1 - k, o.vec, u);
      else u[0] = u[1] = u[2] = u[3] = 0.f;
    } else {
      const int64_t k = k0 + (threadIdx.x >> 4), i = i0 + (threadIdx.x & 15) * 4 + 64 * h;
      if (k < k1 && i < ni) vg_load4(base + (o.rows ? (int64_t)o.rows[k] : k) * o.ld + i, ni - i, o.vec, u);
      else u[0] = u[1] = u[2] = u[3] = 0.f;
    }
  }
}
template <bool kKMajor> __device__ __forceinline__ void vg_put(float (*s)[kVgPitch], const float* v) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if constexpr (kKMajor) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[(threadIdx.x & 3) * 4 + e][(threadIdx.x >> 2) + 64 * h] = v[4 * h + e];
    } else {
      *reinterpret_cast<float4*>(&s[threadIdx.x >> 4][(threadIdx.x & 15) * 4 + 64 * h]) = make_float4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
    }
  }
}

template <typename TA, bool kAK, typename TB, bool kBK, int kMode, typename TOut>
__global__ void __launch_bounds__(kVgThreads, 2) vloss_any_kernel(const __grid_constant__ VgProduct p) {
  __shared__ __align__(16) float a_s[2][kVgK][kVgPitch], b_s[2][kVgK][kVgPitch];
  grid_dependency_wait();
  grid_launch_dependents();
  const int64_t count = *p.count;
  const int64_t m = p.token_axis == 0 ? min(p.m, count) : p.m, kend = p.token_axis == 2 ? min(p.k, count) : p.k;
  const int n_tile = (int)blockIdx.x / p.mt;
  const int64_t m0 = (int64_t)((int)blockIdx.x - n_tile * p.mt) * kVgTile, n0 = (int64_t)n_tile * kVgTile;
  int64_t split_len = p.split_len;
  if (kMode == kVgShare) {                                 // as many shares as the device chose, of the grid's
    const int64_t slots = *p.l.slots;
    if ((int64_t)blockIdx.z >= slots) return;
    split_len = ((p.split_len + slots - 1) / slots + kVgK - 1) / kVgK * kVgK;
  }
  const int64_t k_first = (int64_t)blockIdx.z * split_len, k_last = min(kend, k_first + split_len);
  if (m0 >= m) return;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float2 acc[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = make_float2(0.f, 0.f);
  float fa[8], fb[8];
  if (k_first < k_last) {
    vg_fetch<TA, kAK>(p.a, m0, m, k_first, k_last, fa);
    vg_fetch<TB, kBK>(p.b, n0, p.n, k_first, k_last, fb);
    vg_put<kAK>(a_s[0], fa);
    vg_put<kBK>(b_s[0], fb);
  }
  __syncthreads();
  int buf = 0;
  for (int64_t k0 = k_first; k0 < k_last; k0 += kVgK, buf ^= 1) {
    const bool next = k0 + kVgK < k_last;
    if (next) {
      vg_fetch<TA, kAK>(p.a, m0, m, k0 + kVgK, k_last, fa);
      vg_fetch<TB, kBK>(p.b, n0, p.n, k0 + kVgK, k_last, fb);
    }
#pragma unroll
    for (int k = 0; k < kVgK; ++k) {
      const float4 a0 = *reinterpret_cast<const float4*>(&a_s[buf][k][ty * 4]), a1 = *reinterpret_cast<const float4*>(&a_s[buf][k][64 + ty * 4]);
      const float4 b0 = *reinterpret_cast<const float4*>(&b_s[buf][k][tx * 4]), b1 = *reinterpret_cast<const float4*>(&b_s[buf][k][64 + tx * 4]);
      const float av[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
      const float2 bv[4] = {make_float2(b0.x, b0.y), make_float2(b0.z, b0.w), make_float2(b1.x, b1.y), make_float2(b1.z, b1.w)};
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fma2(make_float2(av[i], av[i]), bv[j], acc[i][j]);
    }
    if (next) {
      vg_put<kAK>(a_s[buf ^ 1], fa);
      vg_put<kBK>(b_s[buf ^ 1], fb);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = m0 + (i < 4 ? ty * 4 + i : 64 + ty * 4 + i - 4);
    const bool live = row < m;
    float v[8];
    int64_t col[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = j & 1 ? acc[i][j >> 1].y : acc[i][j >> 1].x;
      col[j] = n0 + (j < 4 ? tx * 4 + j : 64 + tx * 4 + j - 4);
    }
    if constexpr (kMode == kVgStats) {
      const int64_t label = live ? (int64_t)p.l.plan.label[row] : -1;
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (live && col[j] == label) p.l.mine[row] = v[j];
        if (col[j] < p.n) top = fmaxf(top, v[j]);
      }
#pragma unroll
      for (int o = 8; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += col[j] < p.n ? vl_weight(v[j], top) : 0.f;
#pragma unroll
      for (int o = 8; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (live && tx == 0) p.l.part[row * p.l.tiles + n_tile] = make_float2(top, sum);
    } else if (live) {
      if constexpr (kMode == kVgLogitGrad) {
        const float2 lse = p.l.plan.lse[row];
        const float g = p.l.g[row], own = p.l.plan.own[row];
        const int64_t label = (int64_t)p.l.plan.label[row] - p.col0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (col[j] < p.n) reinterpret_cast<float*>(p.l.dl)[row * p.l.piece + col[j]] = g * (col[j] == label ? own : exp2f(fmaf(v[j] - lse.x, kLog2e, -lse.y)));
      } else if constexpr (kMode == kVgShare) {
        float* out = p.l.acc + ((int64_t)blockIdx.z * count + row) * p.n;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (col[j] < p.n) out[col[j]] = p.more ? out[col[j]] + v[j] : v[j];
      } else {
        const float back = p.l.g_scale[1];
        TOut* out = reinterpret_cast<TOut*>(p.l.dw) + (p.col0 + row) * p.n;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (col[j] < p.n) out[col[j]] = from_f32<TOut>(v[j] * back);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ few tokens, fp32, CUDA cores
// Bound by the weight's bytes: tiles of 64 words x 64 of the inner axis come by cp.async, kFewStages of them ahead, and are multiplied with
// up to 32 tokens.  us of 8 tokens, 162637 words, width 3488, loss and both gradients: as three parts on the tensor cores 9200, so 1750;
// scoring 3600 and 430 (5.3 TB/s).  32 tokens, bound by the products: 4230 and 1155.
constexpr int kFewThreads = 256, kFewCols = 64, kFewK = 64, kFewPitch = kFewK + 4, kFewStages = 4;

// 64 words a CTA: a warp has all of them, two a lane, up to 16 tokens and a part of every 64 of the inner axis.  (Every value of a token
// that comes out of shared memory is used for two words; with one word a lane those loads took as long as the products.)
template <int kR, int kMode> __global__ void __launch_bounds__(kFewThreads) vloss_few_kernel(const __grid_constant__ Vloss p, const float* w, int64_t col0, int64_t cols) {
  extern __shared__ __align__(16) float few_s[];
  constexpr int kStage = (kFewCols + kR) * kFewPitch;
  grid_dependency_wait();
  grid_launch_dependents();
  const int n = p.plan.head[0], r0 = blockIdx.y * kR, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (r0 >= n) return;
  constexpr int kRows = kR > 8 ? kR / 2 : kR, kSplit = kFewThreads / 32 * kRows / kR, kPart = kFewK / kSplit;
  const int part = warp % kSplit, first = warp / kSplit * kRows, steps = (p.width + kFewK - 1) / kFewK;
  float* join = few_s;                                     // [part][token][word], when the stages are done with
  // A thread fetches the same four columns of the same rows of every stage: words i0 + 16 i, then tokens.
  const int i0 = threadIdx.x >> 4, k0 = 4 * (threadIdx.x & 15);
  constexpr int kMine = kFewCols / 16 + (kR + 15) / 16;
  const float* from[kMine];
  bool there[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int r = i0 + 16 * i, x_row = r - kFewCols;
    const int64_t v = (int64_t)blockIdx.x * kFewCols + r;
    there[i] = x_row < 0 ? v < cols : x_row < kR && r0 + x_row < n;
    from[i] = (!there[i] ? w : x_row < 0 ? w + v * p.width : reinterpret_cast<const float*>(p.x) + (int64_t)p.plan.rows[r0 + x_row] * p.x_stride) + k0;
  }
  const uint32_t to0 = (uint32_t)__cvta_generic_to_shared(few_s + i0 * kFewPitch + k0);
  int step_in = 0, slot_in = 0;
  auto fetch = [&]() {                                     // words and tokens that do not exist, and columns beyond the last: zeros
    if (step_in < steps) {
      const bool in = step_in * kFewK + k0 < p.width;
      const uint32_t to = to0 + (uint32_t)(slot_in * kStage) * 4;
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        if (i < kFewCols / 16 || i0 + 16 * i < kFewCols + kR)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + i * 16 * kFewPitch * 4), "l"(in ? from[i] : w), "r"(in && there[i] ? 16 : 0) : "memory");
        from[i] += kFewK;
      }
      ++step_in;
      slot_in = slot_in + 1 == kFewStages ? 0 : slot_in + 1;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int i = 0; i < kFewStages - 1; ++i) fetch();
  int slot = 0;
  {
    float2 acc[kRows][2];
#pragma unroll
    for (int r = 0; r < kRows; ++r) acc[r][0] = acc[r][1] = make_float2(0.f, 0.f);
    for (int step = 0; step < steps; ++step) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kFewStages - 2) : "memory");
      __syncthreads();                                     // this stage is there, and everyone is done with the one that is fetched into
      fetch();
      const float* stage = few_s + slot * kStage + part * kPart;
      slot = slot + 1 == kFewStages ? 0 : slot + 1;
#pragma unroll
      for (int k = 0; k < kPart; k += 4) {
        const float4 f0 = *reinterpret_cast<const float4*>(stage + lane * kFewPitch + k), f1 = *reinterpret_cast<const float4*>(stage + (lane + 32) * kFewPitch + k);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const float4 y = *reinterpret_cast<const float4*>(stage + (kFewCols + first + r) * kFewPitch + k);
          acc[r][0] = fma2(make_float2(y.x, y.y), make_float2(f0.x, f0.y), acc[r][0]);
          acc[r][1] = fma2(make_float2(y.x, y.y), make_float2(f1.x, f1.y), acc[r][1]);
          acc[r][0] = fma2(make_float2(y.z, y.w), make_float2(f0.z, f0.w), acc[r][0]);
          acc[r][1] = fma2(make_float2(y.z, y.w), make_float2(f1.z, f1.w), acc[r][1]);
        }
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) join[(part * kR + first + r) * kFewCols + lane + 32 * h] = acc[r][h].x + acc[r][h].y;
    __syncthreads();
    for (int r = warp; r < kR && r0 + r < n; r += kFewThreads / 32) {
      const int t = r0 + r;
      float s[2];
      int64_t c[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = lane + 32 * h;
        c[h] = (int64_t)blockIdx.x * kFewCols + at;
        s[h] = join[r * kFewCols + at];
#pragma unroll
        for (int i = 1; i < kSplit; ++i) s[h] += join[(i * kR + r) * kFewCols + at];
      }
      const int64_t label = p.plan.label[t] - col0;
      if constexpr (kMode == kVgStats) {
        float top = -INFINITY;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (c[h] == label) p.mine[t] = s[h];
          if (c[h] < cols) top = fmaxf(top, s[h]);
        }
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float sum = warp_add((c[0] < cols ? vl_weight(s[0], top) : 0.f) + (c[1] < cols ? vl_weight(s[1], top) : 0.f));
        if (lane == 0) p.part[(int64_t)t * p.tiles + blockIdx.x] = make_float2(top, sum);
      } else {
        const float2 lse = p.plan.lse[t];
        const float g = p.g[t], own = p.plan.own[t];
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (c[h] < cols) reinterpret_cast<float*>(p.dl)[t * p.piece + c[h]] = g * (c[h] == label ? own : exp2f(fmaf(s[h] - lse.x, kLog2e, -lse.y)));
      }
    }
  }
}

// Shares of dx of kR tokens and 512 columns: 4 columns a thread, every fourth run of 64 words of the share to each quarter of the CTA.
constexpr int kFewShareThreads = 512, kFewShareCols = 512, kFewWords = 64;

template <int kR> __global__ void __launch_bounds__(kFewShareThreads) vloss_few_share_kernel(const __grid_constant__ Vloss p, const float* w, int64_t words, int more) {
  __shared__ __align__(16) float ds[4][kFewWords][kR];
  __shared__ __align__(16) float join[kR][kFewShareCols / 4];          // a quarter of the columns at a time
  grid_dependency_wait();
  grid_launch_dependents();
  const int n = p.plan.head[0], slots = *p.slots, r0 = blockIdx.y * kR, quarter = threadIdx.x >> 7, t = threadIdx.x & 127;
  if (r0 >= n || (int)blockIdx.z >= slots) return;
  const int64_t each = ((words + slots - 1) / slots + 3) / 4 * 4, first = blockIdx.z * each, last = min(words, first + each);
  const int c = blockIdx.x * kFewShareCols + 4 * t;
  const bool mine = c < p.width;
  float2 acc[kR / 2][4];                                   // tokens in pairs: their dL comes out of shared memory as the instruction wants it
#pragma unroll
  for (int r = 0; r < kR / 2; ++r)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[r][e] = make_float2(0.f, 0.f);
  for (int64_t v0 = first; v0 < last; v0 += 4 * kFewWords) {
    __syncthreads();
    for (int i = threadIdx.x; i < 4 * kFewWords * kR; i += kFewShareThreads) {
      const int r = i / (4 * kFewWords), k = i - r * (4 * kFewWords);
      ds[k / kFewWords][k % kFewWords][r] = r0 + r < n && v0 + k < last ? reinterpret_cast<const float*>(p.dl)[(int64_t)(r0 + r) * p.piece + v0 + k] : 0.f;
    }
    __syncthreads();
    const int64_t v1 = v0 + quarter * kFewWords;
    const int left = mine ? (int)min((int64_t)kFewWords, last - v1) : 0;
    const float* at = w + v1 * p.width + c;
    for (int k = 0; k < left; k += 8) {
      float4 f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = k + i < left ? *reinterpret_cast<const float4*>(at + (int64_t)(k + i) * p.width) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 fx = make_float2(f[i].x, f[i].x), fy = make_float2(f[i].y, f[i].y), fz = make_float2(f[i].z, f[i].z), fw = make_float2(f[i].w, f[i].w);
#pragma unroll
        for (int r = 0; r < kR / 2; ++r) {
          const float2 d = *reinterpret_cast<const float2*>(&ds[quarter][k + i][2 * r]);
          acc[r][0] = fma2(fx, d, acc[r][0]);
          acc[r][1] = fma2(fy, d, acc[r][1]);
          acc[r][2] = fma2(fz, d, acc[r][2]);
          acc[r][3] = fma2(fw, d, acc[r][3]);
        }
      }
    }
  }
  for (int part = 0; part < 4; ++part) {                   // threads 32 part .. + 31 of every quarter, the quarters in order
    const bool in = (t >> 5) == part;
    for (int q = 0; q < 4; ++q) {
      __syncthreads();
      if (in && quarter == q)
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          float4* to = reinterpret_cast<float4*>(&join[r][4 * (t & 31)]);
          const float2* a = acc[r / 2];
          float4 s = r % 2 == 0 ? make_float4(a[0].x, a[1].x, a[2].x, a[3].x) : make_float4(a[0].y, a[1].y, a[2].y, a[3].y);
          if (q > 0) { s.x += to->x; s.y += to->y; s.z += to->z; s.w += to->w; }
          if (q < 3) { *to = s; continue; }
          if (!mine || r0 + r >= n) continue;
          float4* out = reinterpret_cast<float4*>(p.acc + ((int64_t)blockIdx.z * n + r0 + r) * p.width + c);
          if (more) { const float4 o = *out; s.x += o.x; s.y += o.y; s.z += o.z; s.w += o.w; }
          *out = s;
        }
    }
  }
}

// dw of up to kR tokens: a thread has four columns of all of them in registers and writes those of 64 words.
constexpr int kFewOutThreads = 128;

template <int kR> __global__ void __launch_bounds__(kFewOutThreads) vloss_few_out_kernel(const __grid_constant__ Vloss p, int64_t v0, int64_t words) {
  __shared__ __align__(16) float ds[kFewWords][kR];
  grid_dependency_wait();
  grid_launch_dependents();
  const int n = p.plan.head[0];
  const int64_t first = (int64_t)blockIdx.x * kFewWords;
  const int c = (blockIdx.y * kFewOutThreads + threadIdx.x) * 4, left = (int)min((int64_t)kFewWords, words - first);
  for (int i = threadIdx.x; i < kR * kFewWords; i += kFewOutThreads) {
    const int r = i / kFewWords, k = i - r * kFewWords;
    ds[k][r] = r < n && k < left ? reinterpret_cast<const float*>(p.dl)[r * p.piece + first + k] : 0.f;
  }
  float2 x[kR / 2][4];                                     // tokens in pairs
#pragma unroll
  for (int r = 0; r < kR; r += 2) {
    float4 a[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      a[i] = r + i < n && c < p.width ? *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.x) + (int64_t)p.plan.rows[r + i] * p.x_stride + c) : make_float4(0.f, 0.f, 0.f, 0.f);
    x[r / 2][0] = make_float2(a[0].x, a[1].x);
    x[r / 2][1] = make_float2(a[0].y, a[1].y);
    x[r / 2][2] = make_float2(a[0].z, a[1].z);
    x[r / 2][3] = make_float2(a[0].w, a[1].w);
  }
  __syncthreads();
  if (c >= p.width) return;
  const float back = p.g_scale[1];
  float* out = reinterpret_cast<float*>(p.dw) + (v0 + first) * p.width + c;
  for (int k = 0; k < left; ++k) {
    float2 a[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = make_float2(0.f, 0.f);
#pragma unroll
    for (int r = 0; r < kR / 2; ++r) {
      const float2 d = *reinterpret_cast<const float2*>(&ds[k][2 * r]);
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] = fma2(x[r][e], d, a[e]);
    }
    *reinterpret_cast<float4*>(out + (int64_t)k * p.width) = make_float4((a[0].x + a[0].y) * back, (a[1].x + a[1].y) * back, (a[2].x + a[2].y) * back, (a[3].x + a[3].y) * back);
  }
}

// Where they are used (see use_few_forward too): fp32, rows of x and w in vectors of 16 bytes, few enough tokens that a pass over w for each 32 of them costs less
// than what taking w apart does.
static bool few_shape(int tokens, int width, int dtype) { return dtype == TKV_F32 && width % 8 == 0 && tokens > 0 && tokens <= 32; }
static int few_rows(int tokens) { return tokens <= 8 ? 8 : tokens <= 16 ? 16 : 32; }
template <int kR, int kMode> static int few_launch(const Vloss& p, const float* w, int64_t col0, int64_t cols, cudaStream_t st) {
  constexpr int kBytes = kFewStages * (kFewCols + kR) * kFewPitch * 4;
  static_assert(8 * kR * kFewCols * 4 <= kBytes, "the parts are joined where the stages were");
  const int64_t tiles = (cols + kFewCols - 1) / kFewCols;
  static bool allowed[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev < 0 || dev >= 64 || !allowed[dev])) {
    e = cudaFuncSetAttribute(vloss_few_kernel<kR, kMode>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (e == cudaSuccess && dev >= 0 && dev < 64) allowed[dev] = true;
  }
  if (e == cudaSuccess)
    e = launch_pdl(vloss_few_kernel<kR, kMode>, dim3((unsigned)tiles, (p.tokens + kR - 1) / kR), dim3(kFewThreads), (size_t)kBytes, st, p, w, col0, cols);
  return e == cudaSuccess ? check_launch("tkv_vloss") : fail(TKV_ERR_LAUNCH, "tkv_vloss: %s", cudaGetErrorString(e));
}
template <int kMode> static int few_launch(const Vloss& p, const float* w, int64_t col0, int64_t cols, cudaStream_t st) {
  switch (few_rows(p.tokens)) {
    case 8: return few_launch<8, kMode>(p, w, col0, cols, st);
    case 16: return few_launch<16, kMode>(p, w, col0, cols, st);
    default: return few_launch<32, kMode>(p, w, col0, cols, st);
  }
}
static int few_out_launch(const Vloss& p, int64_t v0, int64_t words, cudaStream_t st) {
  const int r = few_rows(p.tokens);
  const int64_t blocks = (words + kFewWords - 1) / kFewWords;
  cudaError_t e = launch_pdl(r == 8 ? vloss_few_out_kernel<8> : r == 16 ? vloss_few_out_kernel<16> : vloss_few_out_kernel<32>,
                             dim3((unsigned)blocks, (p.width + 4 * kFewOutThreads - 1) / (4 * kFewOutThreads)), dim3(kFewOutThreads), 0, st, p, v0, words);
  return e == cudaSuccess ? check_launch("tkv_vloss") : fail(TKV_ERR_LAUNCH, "tkv_vloss: %s", cudaGetErrorString(e));
}
static int few_share_launch(const Vloss& p, const float* w, int64_t words, int room, int more, cudaStream_t st) {
  const int r = p.tokens <= 8 ? 8 : 16;
  cudaError_t e = launch_pdl(r == 8 ? vloss_few_share_kernel<8> : vloss_few_share_kernel<16>, dim3((p.width + kFewShareCols - 1) / kFewShareCols, (p.tokens + r - 1) / r, room),
                             dim3(kFewShareThreads), 0, st, p, w, words, more);
  return e == cudaSuccess ? check_launch("tkv_vloss") : fail(TKV_ERR_LAUNCH, "tkv_vloss: %s", cudaGetErrorString(e));
}

template <typename TA, bool kAK, typename TB, bool kBK, int kMode, typename TOut> static int vg_launch(VgProduct p, cudaStream_t st) {
  // (2^43 logits are below 2^30 tiles; the other products have fewer)
  const int64_t mt = (p.m + kVgTile - 1) / kVgTile, nt = (p.n + kVgTile - 1) / kVgTile;
  if (mt * nt > INT32_MAX) return fail(TKV_ERR_UNSUPPORTED, "tkv_vloss: %lld x %lld tiles", (long long)mt, (long long)nt);
  p.mt = (int)mt;
  cudaError_t e = launch_pdl(vloss_any_kernel<TA, kAK, TB, kBK, kMode, TOut>, dim3((unsigned)(mt * nt), 1, p.split), dim3(kVgThreads), 0, st, p);
  if (e != cudaSuccess) return fail(TKV_ERR_LAUNCH, "tkv_vloss: %s", cudaGetErrorString(e));
  return check_launch("tkv_vloss");
}

static bool vec4(const void* p, int64_t ld, int size) { return ((uintptr_t)p | (uintptr_t)(ld * size)) % (size * 4) == 0; }

template <typename T> static int vloss_any_forward(Vloss l, cudaStream_t st) {
  VgProduct p = {};
  p.a = {l.x, l.x_stride, l.plan.rows, vec4(l.x, l.x_stride, sizeof(T))};
  p.b = {l.w, l.width, nullptr, vec4(l.w, l.width, sizeof(T))};
  p.m = l.tokens; p.n = l.vocab; p.k = l.width; p.count = l.plan.head; p.token_axis = 0;
  p.split = 1; p.split_len = l.width; p.l = l;
  return vg_launch<T, true, T, true, kVgStats, T>(p, st);
}

// Pieces of the vocabulary: up to 64 MB of dL, whole tiles.
static int64_t any_piece(int tokens, int64_t vocab) {
  int64_t n = ((int64_t)64 << 20) / (4 * (int64_t)(tokens > 0 ? tokens : 1)) / kVgTile * kVgTile;
  if (n < 1024) n = 1024;
  return n < vocab ? n : vl_round(vocab, 4);
}
// Room for shares of dx, whose few tiles of [tokens, width] are as long as the piece (the device chooses how many it uses).
static int any_slots(int tokens, int width) {
  const int64_t tiles = ((tokens + kVgTile - 1) / kVgTile) * (int64_t)((width + kVgTile - 1) / kVgTile);
  const int64_t s = (8 * 148 + tiles - 1) / (tiles > 0 ? tiles : 1);
  return (int)(s < 1 ? 1 : s > kVlMaxSlots ? kVlMaxSlots : s);
}

template <typename T> static int vloss_any_backward(Vloss l, bool want_dx, int most_slots, bool few, cudaStream_t st) {
  for (int64_t v0 = 0; v0 < l.vocab; v0 += l.piece) {
    const int64_t n = l.vocab - v0 < l.piece ? l.vocab - v0 : l.piece;
    const T* w = reinterpret_cast<const T*>(l.w) + v0 * l.width;
    VgProduct p = {};
    p.count = l.plan.head; p.col0 = v0; p.l = l; p.split = 1;
    const VgOperand x = {l.x, l.x_stride, l.plan.rows, vec4(l.x, l.x_stride, sizeof(T))}, wk = {w, l.width, nullptr, vec4(w, l.width, sizeof(T))},
                    dl = {l.dl, l.piece, nullptr, vec4(l.dl, l.piece, 4)};
    p.a = x; p.b = wk; p.m = l.tokens; p.n = n; p.k = p.split_len = l.width; p.token_axis = 0;
    int rc = few ? few_launch<kVgLogitGrad>(l, reinterpret_cast<const float*>(w), v0, n, st) : vg_launch<T, true, T, true, kVgLogitGrad, T>(p, st);
    if (rc == TKV_OK && want_dx && few) {
      rc = few_share_launch(l, reinterpret_cast<const float*>(w), n, most_slots, v0 > 0, st);
    } else if (rc == TKV_OK && want_dx) {
      p.a = dl; p.b = wk; p.m = l.tokens; p.n = l.width; p.k = n; p.token_axis = 0;
      p.split = most_slots; p.split_len = l.piece; p.more = v0 > 0;
      rc = vg_launch<float, true, T, false, kVgShare, T>(p, st);
    }
    if (rc == TKV_OK && l.dw && few) {
      rc = few_out_launch(l, v0, n, st);
    } else if (rc == TKV_OK && l.dw) {
      p.a = dl; p.b = x; p.m = n; p.n = l.width; p.k = p.split_len = l.tokens; p.token_axis = 2; p.split = 1;
      rc = vg_launch<float, false, T, false, kVgOut, T>(p, st);
    }
    if (rc != TKV_OK) return rc;
  }
  return TKV_OK;
}

// ---------------------------------------------------------------------------------------------- joining, gradients of the rows
constexpr int kJoinThreads = 128;

// A CTA per token that counts: lse from the tiles' maxima and sums, loss.
__global__ void __launch_bounds__(kJoinThreads) vloss_join_kernel(Vloss p, float* loss) {
  __shared__ float red[2][kJoinThreads / 32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int row = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (row >= p.plan.head[0]) return;
  const float2* part = p.part + (int64_t)row * p.tiles;
  float top = -INFINITY, sum = 0.f;
  for (int i = threadIdx.x; i < p.tiles; i += kJoinThreads) {
    const float2 x = part[i];
    const float next = fmaxf(top, x.x);
    sum = sum * vl_weight(top, next) + x.y * vl_weight(x.x, next);
    top = next;
  }
  float all = top;
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
  if (lane == 0) red[0][warp] = all;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoinThreads / 32; ++w) all = fmaxf(all, red[0][w]);
  sum = warp_add(sum * vl_weight(top, all));
  if (lane == 0) red[1][warp] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinThreads / 32; ++w) sum += red[1][w];
    p.plan.lse[row] = make_float2(all, log2f(sum));
    const float l = (all - p.mine[row]) + logf(sum);       // maximum and label first: they are often the same number
    p.plan.own[row] = expm1f(-l);
    loss[p.plan.rows[row]] = p.plan.head[2] ? __int_as_float(0x7fffffff) : l;
  }
}

constexpr int kSumThreads = 1024;

// Sum (reduction 2) or mean (1) of the losses, in fp64, in a fixed order.
__global__ void __launch_bounds__(kSumThreads) vloss_sum_kernel(const float* loss, int tokens, VlossPlan plan, int reduction, float* out) {
  __shared__ double red[kSumThreads / 32];
  grid_dependency_wait();
  grid_launch_dependents();
  double s = 0.0;
  for (int t = threadIdx.x; t < tokens; t += kSumThreads) s += (double)loss[t];
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int w = 0; w < kSumThreads / 32; ++w) s += red[w];
    *out = (float)(reduction == 1 ? s / (double)plan.head[0] : s);
  }
}

// Gradient of every counting row's loss, times a power of two that brings the largest to about 2^14: fp16 keeps what is small beside it
// (a mean over many tokens makes all of them small), and exponents of bf16 and fp32 are only shifted.
// And how the gradients' tiles are dealt out: those of dx in turn; to the workers that got one fewer, x tiles of dw each that make up for it;
// the others of dw in turn.  With s shares a tile of dx takes steps / s (and a little for what it writes), one of dw the tokens' steps: the s
// that makes the busiest worker's work least.
__global__ void __launch_bounds__(kSumThreads) vloss_rows_grad_kernel(const float* grad, int64_t stride, int reduction, VlossPlan plan, VlossWork work, float* g,
                                                                      float* scale, int* slots) {
  __shared__ float red[kSumThreads / 32];
  __shared__ int cost[kVlMaxSlots], extra[kVlMaxSlots];
  grid_dependency_wait();
  grid_launch_dependents();
  const int n = plan.head[0], lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float by = reduction == 1 ? 1.0f / (float)n : 1.0f;
  float top = 0.f;
  for (int i = threadIdx.x; i < n; i += kSumThreads) top = fmaxf(top, fabsf(grad[(int64_t)plan.rows[i] * stride] * by));
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) red[warp] = top;
  if (lane == 0) {
    const int s = warp + 1, mt = (n + work.rows - 1) / work.rows, W = work.workers;  // this warp looks at s shares
    const int dx = work.dx ? mt * work.ht * s : 0, dw = work.dw ? work.vt * work.ht : 0;
    const int dx_cost = (work.steps + s - 1) / s + 12, dw_cost = (n + work.step - 1) / work.step + 4;
    const int more = dx % W, fewer = W - more;                                       // workers with a tile of dx more than the others
    const int x = more ? min(dx_cost / dw_cost, dw / fewer) : 0, rest = dw - x * fewer, last = rest % W;
    const int with = more ? (dx / W + 1) * dx_cost + (rest / W + (last > fewer)) * dw_cost : 0;
    const int without = dx / W * dx_cost + (x + rest / W + (last > 0)) * dw_cost;
    const bool fits = s == 1 || (s <= work.most && (int64_t)s * ((n + work.acc_rows - 1) / work.acc_rows * work.acc_rows) <= (int64_t)work.room * work.tokens && work.steps >= 8 * s);
    cost[warp] = fits ? max(with, without) : INT32_MAX;
    extra[warp] = x;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSumThreads / 32; ++w) top = fmaxf(top, red[w]);
  int e = 0;
  if (top > 0.f && top < INFINITY) e = min(max(14 - ilogbf(top), -100), 100);
  const float s = ldexpf(1.f, e);
  float same = 1.f;                                        // a gradient that all tokens share is multiplied in at the end: g is then a power of two
  if (stride == 0 && top > 0.f && top < INFINITY) same = ldexpf(top, -ilogbf(top));
  for (int i = threadIdx.x; i < n; i += kSumThreads) {
    const float v = grad[(int64_t)plan.rows[i] * stride] * by * s;
    g[i] = same == 1.f ? v : copysignf(ldexpf(1.f, ilogbf(v)), v);
  }
  if (threadIdx.x == 0) {
    scale[0] = s; scale[1] = ldexpf(same, -e);
    int best = 0;
    for (int i = 1; i < kVlMaxSlots; ++i)
      if (cost[i] < cost[best]) best = i;
    slots[0] = best + 1;
    slots[1] = extra[best];
  }
}
static_assert(kSumThreads / 32 == kVlMaxSlots, "a warp for every number of shares");

constexpr int kDxThreads = 256;

// Where a wait ran out, tiles of dw are missing: all of it becomes NaN.
template <typename T> __device__ __forceinline__ void vl_spoil(const VlossPlan& plan, T* dw, int64_t n) {
  if (dw == nullptr || plan.head[2] == 0) return;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) dw[i] = from_f32<T>(__int_as_float(0x7fffffff));
}
template <typename T> __global__ void __launch_bounds__(kDxThreads) vloss_spoil_kernel(Vloss p) {
  grid_dependency_wait();
  grid_launch_dependents();
  vl_spoil(p.plan, reinterpret_cast<T*>(p.dw), p.vocab * p.width);
}

// dx: the shares of a row added up in order, in the caller's type and place; zeros for tokens that do not count.  The rows of the plan are
// in order, so a token finds itself there by halving.
template <typename T> __global__ void __launch_bounds__(kDxThreads) vloss_dx_kernel(Vloss p, T* dx) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int t = blockIdx.x, n = p.plan.head[0];
  vl_spoil(p.plan, reinterpret_cast<T*>(p.dw), p.vocab * p.width);
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (p.plan.rows[mid] < t) lo = mid + 1; else hi = mid;
  }
  const bool live = lo < n && p.plan.rows[lo] == t;
  const int slots = *p.slots;
  const int64_t each = ((int64_t)n + p.acc_rows - 1) / p.acc_rows * p.acc_rows;
  const float back = p.plan.head[2] ? __int_as_float(0x7fffffff) : p.g_scale[1];
  T* out = dx + (int64_t)t * p.width;
  if (p.width % 8 == 0) {
    const float rest = live && p.rest ? p.rest[lo] : 0.f;
    const T* w = reinterpret_cast<const T*>(p.w) + (int64_t)(live ? p.plan.label[lo] : 0) * p.width;
    for (int c = threadIdx.x * 8; c < p.width; c += kDxThreads * 8) {
      float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (live)
        for (int i = 0; i < slots; ++i) {
          float v[8];
          load_vec<8>(p.acc + (i * each + lo) * p.width + c, v);
#pragma unroll
          for (int e = 0; e < 8; ++e) s[e] += v[e];
        }
      if (rest != 0.f) {
        float v[8];
        load_vec<8>(w + c, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] += rest * v[e];
      }
      alignas(16) T e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(s[i] * back);
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) st16(reinterpret_cast<char*>(out + c) + 16 * i, *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(e) + 16 * i));
    }
    return;
  }
  for (int c = threadIdx.x; c < p.width; c += kDxThreads) {
    float s = 0.f;
    if (live)
      for (int i = 0; i < slots; ++i) s += p.acc[(i * each + lo) * p.width + c];
    out[c] = from_f32<T>(s * back);
  }
}

template <typename... A> static int vl_launch(const char* what, void (*kernel)(A...), dim3 grid, int threads, cudaStream_t st, A... args) {
  cudaError_t e = launch_pdl(kernel, grid, dim3(threads), 0, st, args...);
  if (e != cudaSuccess) return fail(TKV_ERR_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
  return check_launch(what);
}

template <typename T> static int vloss_finish(const Vloss& p, void* dx, cudaStream_t st) {
  if (dx) return vl_launch("tkv_vloss_backward", vloss_dx_kernel<T>, dim3((unsigned)p.tokens), kDxThreads, st, p, (T*)dx);
  return vl_launch("tkv_vloss_backward", vloss_spoil_kernel<T>, dim3(148), kDxThreads, st, p);
}

int vloss_plan_rows(const Vloss& p, const int64_t* labels, int64_t ignore, float* loss, cudaStream_t st) {
  return vl_launch("tkv_vloss_forward", vloss_plan_kernel, dim3(1), kPlanThreads, st, labels, ignore, p.tokens, p.vocab, p.plan, loss, p.status);
}
static bool use_few(const Vloss& p) { return few_shape(p.tokens, p.width, p.dtype) && aligned16(p.w) && aligned16(p.x) && p.x_stride % 4 == 0 && (p.dw == nullptr || aligned16(p.dw)); }
// Scoring of up to 64 tokens in two passes over a large w: us of 64 tokens, 162637 words, width 3488, in two passes 2230, on the tensor cores
// 3600; of 60000 words, width 2048, 540 and 590; of 32768, width 1024, whose parts stay in L2, 186 and 135.
constexpr int kFewForward = 64;
static bool use_few_forward(const Vloss& p) {
  return use_few(p) || (p.dtype == TKV_F32 && p.width % 8 == 0 && p.tokens <= kFewForward && p.vocab * p.width >= (int64_t)1 << 27 && aligned16(p.w) && aligned16(p.x) && p.x_stride % 4 == 0);
}
static bool use_tc(const Vloss& p) { return !use_few(p) && vloss_tc_shape(p.tokens, p.vocab, p.width, p.dtype) && aligned16(p.w) && (p.dw == nullptr || aligned16(p.dw)); }
static int64_t pad256(int64_t bytes) { return vl_round(bytes, 256); }
static int64_t any_forward_bytes(int tokens, int64_t vocab, int dtype) {
  const int tile = dtype == TKV_F32 && tokens <= kFewForward ? kFewCols : kVgTile;   // the narrower tiles where they may run
  return (int64_t)tokens * ((vocab + tile - 1) / tile) * 8;
}
static int64_t any_backward_bytes(int tokens, int64_t vocab, int width, bool dx) {
  const int64_t piece = any_piece(tokens, vocab);
  return pad256((int64_t)tokens * piece * 4) + (dx ? (int64_t)any_slots(tokens, width) * tokens * width * 4 : 0);
}
static int check_sizes(const char* what, int64_t tokens, int64_t vocab, int width, int64_t x_stride, int dtype) {
  if (tokens < 0 || vocab < 1 || width < 1 || elem_size(dtype) == 0 || (tokens > 1 && x_stride < width))
    return fail(TKV_ERR_ARG, "%s: tokens=%lld vocab=%lld width=%d rows %lld apart dtype=%d", what, (long long)tokens, (long long)vocab, width, (long long)x_stride, dtype);
  if (tokens > (1 << 24) || vocab > (1 << 23) || width > 65536 || tokens * vocab > ((int64_t)1 << 43))
    return fail(TKV_ERR_UNSUPPORTED, "%s: tokens=%lld (at most 2^24) vocab=%lld (2^23; together 2^43) width=%d (65536)", what, (long long)tokens, (long long)vocab, width);
  return TKV_OK;
}

}  // namespace tkv

extern "C" int64_t tkv_vloss_plan_words(int64_t tokens) { return 4 + 5 * (tokens > 0 ? tokens : 0); }

extern "C" int64_t tkv_vloss_workspace_bytes(int64_t tokens, int64_t vocab, int width, int dtype, int backward, int want_dx) {
  using namespace tkv;
  if (check_sizes("tkv_vloss_workspace_bytes", tokens, vocab, width, width, dtype) != TKV_OK) return -1;
  const int t = (int)tokens;
  int64_t n = backward ? any_backward_bytes(t, vocab, width, want_dx != 0) : any_forward_bytes(t, vocab, dtype);
  if (vloss_tc_shape(t, vocab, width, dtype)) {            // which form runs is known with the addresses: room for either
    const int64_t tc = vloss_tc_bytes(t, vocab, width, dtype, backward != 0, want_dx != 0);
    n = n > tc ? n : tc;
  }
  return 512 + (backward ? 2 : 1) * pad256((int64_t)t * 4) + n;
}

extern "C" int tkv_vloss_forward(const void* x, int64_t x_stride, const void* w, const int64_t* labels, int64_t ignore, int64_t tokens,
                                 int64_t vocab, int width, int reduction, float* loss, float* reduced, int32_t* plan, void* workspace,
                                 int64_t workspace_bytes, int dtype, int32_t* status, tkv_stream_t stream) {
  using namespace tkv;
  const int rc0 = check_sizes("tkv_vloss_forward", tokens, vocab, width, x_stride, dtype);
  if (rc0 != TKV_OK) return rc0;
  if (reduction < 0 || reduction > 2) return fail(TKV_ERR_ARG, "tkv_vloss_forward: reduction=%d", reduction);
  if (!plan || !workspace || (reduction && !reduced) || (tokens && (!x || !w || !labels || !loss))) return fail(TKV_ERR_ARG, "tkv_vloss_forward: NULL pointer argument");
  if (((uintptr_t)plan & 7) != 0) return fail(TKV_ERR_ARG, "tkv_vloss_forward: the plan must be 8-byte aligned");
  if (!aligned16(workspace) || workspace_bytes < tkv_vloss_workspace_bytes(tokens, vocab, width, dtype, 0, 0))
    return fail(TKV_ERR_ARG, "tkv_vloss_forward: workspace of %lld bytes", (long long)workspace_bytes);
  cudaStream_t st = (cudaStream_t)stream;
  Vloss p = {};
  p.x = x; p.x_stride = x_stride; p.w = w; p.vocab = vocab; p.tokens = (int)tokens; p.width = width; p.dtype = dtype;
  p.plan = vloss_plan(plan, tokens); p.status = status;
  p.mine = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + 512);
  void* rest = reinterpret_cast<char*>(p.mine) + pad256(tokens * 4);
  int rc;
  if (tokens && !use_few_forward(p) && use_tc(p)) {
    rc = vloss_tc_forward(p, labels, ignore, loss, rest, st);
  } else {
    rc = vloss_plan_rows(p, labels, ignore, loss, st);
    p.part = reinterpret_cast<float2*>(rest);
    const bool few = use_few_forward(p);
    const int tile = few ? kFewCols : kVgTile;
    p.tiles = (int)((vocab + tile - 1) / tile);
    if (rc == TKV_OK && tokens)
      rc = few ? few_launch<kVgStats>(p, reinterpret_cast<const float*>(w), 0, vocab, st) : dtype == TKV_F32 ? vloss_any_forward<float>(p, st) : dtype == TKV_BF16 ? vloss_any_forward<__nv_bfloat16>(p, st) : vloss_any_forward<__half>(p, st);
  }
  if (rc == TKV_OK && tokens) rc = vl_launch("tkv_vloss_forward", vloss_join_kernel, dim3((unsigned)tokens), kJoinThreads, st, p, loss);
  if (rc == TKV_OK && reduction) rc = vl_launch("tkv_vloss_forward", vloss_sum_kernel, dim3(1), kSumThreads, st, (const float*)loss, p.tokens, p.plan, reduction, reduced);
  return rc;
}

extern "C" int tkv_vloss_backward(const void* x, int64_t x_stride, const void* w, const int32_t* plan, const float* grad, int64_t grad_stride,
                                  int reduction, int64_t tokens, int64_t vocab, int width, void* dx, void* dw, void* workspace,
                                  int64_t workspace_bytes, int dtype, int32_t* status, tkv_stream_t stream) {
  using namespace tkv;
  const int rc0 = check_sizes("tkv_vloss_backward", tokens, vocab, width, x_stride, dtype);
  if (rc0 != TKV_OK) return rc0;
  if (reduction < 0 || reduction > 2) return fail(TKV_ERR_ARG, "tkv_vloss_backward: reduction=%d", reduction);
  cudaStream_t st = (cudaStream_t)stream;
  if (tokens == 0) {
    if (dw && cudaMemsetAsync(dw, 0, (size_t)vocab * width * elem_size(dtype), st) != cudaSuccess) return check_launch("tkv_vloss_backward");
    return TKV_OK;
  }
  if (!plan || !workspace || !w || !grad || (!dx && !dw) || !x) return fail(TKV_ERR_ARG, "tkv_vloss_backward: NULL pointer argument");
  if (((uintptr_t)plan & 7) != 0) return fail(TKV_ERR_ARG, "tkv_vloss_backward: the plan must be 8-byte aligned");
  if (!aligned16(workspace) || workspace_bytes < tkv_vloss_workspace_bytes(tokens, vocab, width, dtype, 1, dx != nullptr))
    return fail(TKV_ERR_ARG, "tkv_vloss_backward: workspace of %lld bytes", (long long)workspace_bytes);
  if (dx && width % 8 == 0 && !aligned16(dx)) return fail(TKV_ERR_ARG, "tkv_vloss_backward: dx must be 16-byte aligned");
  Vloss p = {};
  p.x = x; p.x_stride = x_stride; p.w = w; p.vocab = vocab; p.tokens = (int)tokens; p.width = width; p.dtype = dtype;
  p.plan = vloss_plan(const_cast<int32_t*>(plan), tokens); p.status = status; p.dw = dw;
  float* scale = reinterpret_cast<float*>(workspace);
  float* g = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + 512);
  char* rest = reinterpret_cast<char*>(g) + 2 * pad256(tokens * 4);
  p.g = g; p.g_scale = scale; p.slots = reinterpret_cast<int*>(scale) + 2;
  const bool tc = use_tc(p);
  if (tc && dtype != TKV_F32) p.rest = reinterpret_cast<float*>(reinterpret_cast<char*>(g) + pad256(tokens * 4));
  const int64_t piece = any_piece(p.tokens, vocab);
  const int room = any_slots(p.tokens, width);
  const bool few = use_few(p);
  const VlossWork work = few ? VlossWork{148, p.tokens <= 8 ? 8 : 16, 1, (width + kFewShareCols - 1) / kFewShareCols, 0, (int)((piece + kFewWords - 1) / kFewWords), kFewWords, room, p.tokens, room, dx != nullptr, false}
                       : tc ? vloss_tc_work(p.tokens, vocab, width, dtype, dx != nullptr, dw != nullptr)
                            : VlossWork{2 * 148, kVgTile, 1, (width + kVgTile - 1) / kVgTile, 0, (int)((piece + kVgK - 1) / kVgK), kVgK, room, p.tokens, room, dx != nullptr, false};
  int rc = vl_launch("tkv_vloss_backward", vloss_rows_grad_kernel, dim3(1), kSumThreads, st, grad, grad_stride, reduction, p.plan, work, g, scale,
                     reinterpret_cast<int*>(scale) + 2);
  if (rc != TKV_OK) return rc;
  p.acc_rows = work.acc_rows;
  if (tc) {
    rc = vloss_tc_backward(p, rest, dx != nullptr, st);
  } else {
    p.piece = piece;
    p.dl = rest;
    p.acc = reinterpret_cast<float*>(rest + pad256(tokens * piece * 4));
    rc = dtype == TKV_F32 ? vloss_any_backward<float>(p, dx != nullptr, room, few, st)
                          : dtype == TKV_BF16 ? vloss_any_backward<__nv_bfloat16>(p, dx != nullptr, room, false, st) : vloss_any_backward<__half>(p, dx != nullptr, room, false, st);
  }
  if (rc != TKV_OK) return rc;
  if (dtype == TKV_F32) return vloss_finish<float>(p, dx, st);
  return dtype == TKV_BF16 ? vloss_finish<__nv_bfloat16>(p, dx, st) : vloss_finish<__half>(p, dx, st);
}
