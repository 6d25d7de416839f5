// How evenly a router spreads its tokens over the experts.  Of n valid tokens with k choices each and p_t = softmax(z_t):
//   c_e = choices of expert e,  f_e = c_e / (n k),  P_e = sum_t p_te / n,  loss = E sum_e f_e P_e
//   d loss / d z_te = (E / n) p_te (f_e - sum_j p_tj f_j)          (the counts have no gradient)
// Both passes read the logits once and recompute the softmax: a few lanes or a warp per token, its experts in their registers, so HBM (or,
// for few tokens, the launches) is the bound.  The sums over tokens stay in registers, lane by lane, and are added up in a fixed order:
// first the warps of a CTA, then the CTAs.  No atomics on floating point: equal inputs give equal bits.
#include "tkv_elem.cuh"

namespace tkv {

constexpr int kBalThreads = 1024, kBalWarps = kBalThreads / 32, kBalCtas = 148, kBalExperts = 1024;
#define bal_threads(per) ((per) <= 4 ? kBalThreads : kBalThreads / 2)   // many experts a lane: their registers

struct Balance {
  const void* z; int64_t stride;                           // [tokens, experts]
  const void* choice; int64_t choice_stride;               // [tokens, top]
  const uint8_t* valid; int64_t valid_stride;              // [tokens], or NULL: all
  int64_t tokens;
  int experts, top, choice64;
  float* sums;                                             // [ctas, experts] sums of p
  int32_t* hits;                                           // [ctas, experts + 1] choices of each expert, and valid tokens
  int32_t* counts;                                         // [experts]
  float* load;                                             // [experts + 1] f_e, and E / n
  float* loss;
  const float* grad;                                       // backward: gradient of the loss
  void* dz; int64_t dz_stride;
};

// A token belongs to kLanes lanes, 32 / kLanes tokens to a warp.  kVec: lane l holds experts 4 (l + kLanes i) .. + 3 (four at a time from
// memory; experts and strides are multiples of four), else l + kLanes i; kPer values a lane.
template <typename T, int kLanes, int kPer, bool kVec> struct BalRow {
  alignas(16) T raw[kPer];
  __device__ __forceinline__ static int expert(int l, int i) { return kVec ? 4 * (l + kLanes * (i / 4)) + (i & 3) : l + kLanes * i; }
  __device__ __forceinline__ void load(const T* z, int experts, int l) {
    if constexpr (kVec) {
#pragma unroll
      for (int i = 0; i < kPer; i += 4) {
        if (expert(l, i) >= experts) continue;
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(raw + i) = ld16_stream(z + expert(l, i));
        else *reinterpret_cast<uint2*>(raw + i) = *reinterpret_cast<const uint2*>(z + expert(l, i));
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (expert(l, i) < experts) raw[i] = z[expert(l, i)];
    }
  }
  __device__ __forceinline__ void softmax(int experts, int l, float* p) const {
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      p[i] = expert(l, i) < experts ? to_f32<T>(raw[i]) : -INFINITY;
      top = fmaxf(top, p[i]);
    }
#pragma unroll
    for (int o = kLanes / 2; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p[i]) : "f"((p[i] - top) * 1.4426950408889634f));   // 0 beyond the last
      sum += p[i];
    }
#pragma unroll
    for (int o = kLanes / 2; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float inv = 1.0f / sum;
#pragma unroll
    for (int i = 0; i < kPer; ++i) p[i] *= inv;
  }
};

// Adds up the CTAs' shares; one CTA of kThreads.  A column of the shares (an expert, and the valid tokens) to every thread, several threads
// to a column where there are fewer columns, 16 CTAs' shares requested at a time.
struct BalFinish { double part[kBalWarps]; float sums[kBalThreads]; int32_t hits[kBalThreads]; int32_t n; };

template <int kThreads> __device__ __forceinline__ void balance_finish(const Balance& p, int ctas, BalFinish* sm) {
  const int E = p.experts, wide = min((E + 1 + 31) / 32 * 32, kThreads), slices = kThreads / wide;
  const int slice = threadIdx.x / wide, at = threadIdx.x - slice * wide;
  double part = 0.0;
  for (int e0 = E / wide * wide; e0 >= 0; e0 -= wide) {    // the last columns first: the valid tokens are among them
    const int e = e0 + at;
    float s = 0.f;
    int c = 0;
    if (slice < slices && e <= E)
      for (int b0 = slice; b0 < ctas; b0 += 16 * slices) {
        float v[16];
        int h[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int b = b0 + i * slices;
          v[i] = b < ctas && e < E ? p.sums[(int64_t)b * E + e] : 0.f;
          h[i] = b < ctas ? p.hits[(int64_t)b * (E + 1) + e] : 0;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) { s += v[i]; c += h[i]; }
      }
    sm->sums[threadIdx.x] = s;
    sm->hits[threadIdx.x] = c;
    __syncthreads();
    if (slice == 0 && e <= E) {
      for (int k = 1; k < slices; ++k) { s += sm->sums[k * wide + at]; c += sm->hits[k * wide + at]; }
      if (e == E) sm->n = c;
    }
    __syncthreads();
    if (slice == 0 && e < E) {
      const int n = sm->n;
      const float f = n > 0 && p.top > 0 ? (float)c / ((float)n * (float)p.top) : 0.f;
      p.counts[e] = c;
      p.load[e] = f;
      part += (double)f * (double)s;
    }
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
  if ((threadIdx.x & 31) == 0) sm->part[threadIdx.x >> 5] = part;
  __syncthreads();
  if (threadIdx.x == 0) {
    double sum = 0.0;
    for (int w = 0; w < kThreads / 32; ++w) sum += sm->part[w];
    const float scale = sm->n > 0 ? (float)E / (float)sm->n : 0.f;
    *p.loss = (float)sum * scale;
    p.load[E] = scale;
  }
}

constexpr int kBalChunk = 128;                             // experts whose sums of all warps are in shared memory at a time

template <typename T, int kLanes, int kPer, bool kVec> __global__ void __launch_bounds__(bal_threads(kPer), 1) balance_sum_kernel(const __grid_constant__ Balance p) {
  extern __shared__ float sums[];                          // [warps][min(experts, kBalChunk)]
  __shared__ BalFinish finish;
  __shared__ int32_t hits[kBalExperts + 1];
  constexpr int kRows = 32 / kLanes, kWarps = bal_threads(kPer) / 32, kBatch = kPer <= 4 ? 4 : kPer <= 16 ? 3 : 1;   // tokens of a warp whose logits are requested together
  using Row = BalRow<T, kLanes, kPer, kVec>;
  const int E = p.experts, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % kLanes, mine = lane / kLanes;
  grid_dependency_wait();
  for (int e = threadIdx.x; e <= E; e += blockDim.x) hits[e] = 0;
  __syncthreads();
  float acc[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) acc[i] = 0.f;
  int seen = 0;
  const int64_t step = (int64_t)gridDim.x * kWarps * kRows;
  Row row[kBatch];
  bool live[kBatch];
  auto request = [&](int64_t t0) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int64_t t = t0 + i * step;
      live[i] = t < p.tokens && (p.valid == nullptr || p.valid[t * p.valid_stride] != 0);
      if (live[i]) row[i].load(reinterpret_cast<const T*>(p.z) + t * p.stride, E, l);
      seen += live[i] && l == 0;
    }
  };
  int64_t t0 = ((int64_t)blockIdx.x * kWarps + warp) * kRows + mine;
  request(t0);
  // While the first rows come, the choices, a thread each, wherever their tokens' logits are read (tokens * top is below 2^31).
  const uint32_t all = (uint32_t)p.tokens * (uint32_t)p.top, threads = gridDim.x * blockDim.x;
#pragma unroll 4
  for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i < all; i += threads) {
    const uint32_t t = i / (uint32_t)p.top;
    const int64_t at = t * p.choice_stride + (i - t * (uint32_t)p.top);
    const int64_t e = p.choice64 ? reinterpret_cast<const int64_t*>(p.choice)[at] : (int64_t)reinterpret_cast<const int32_t*>(p.choice)[at];
    if (e >= 0 && e < E && (p.valid == nullptr || p.valid[t * p.valid_stride] != 0)) atomicAdd(&hits[e], 1);
  }
  while (t0 - mine < p.tokens) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      float s[kPer];
      row[i].softmax(E, l, s);                             // shuffles: every lane takes part
#pragma unroll
      for (int k = 0; k < kPer; ++k) acc[k] += live[i] ? s[k] : 0.f;
    }
    t0 += kBatch * step;
    if (t0 - mine < p.tokens) request(t0);
  }
#pragma unroll
  for (int o = kLanes; o < 32; o <<= 1) {                  // the tokens of a warp
    seen += __shfl_xor_sync(0xffffffffu, seen, o);
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
  }
  if (lane == 0) atomicAdd(&hits[E], seen);
  const int wide = min(E, kBalChunk);
  for (int e0 = 0; e0 < E; e0 += wide) {                   // the warps of the CTA, in order
    if (mine == 0) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int e = Row::expert(l, i) - e0;
        if (e >= 0 && e < wide) sums[warp * wide + e] = acc[i];
      }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < wide && e0 + e < E; e += blockDim.x) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) s += sums[w * wide + e];
      p.sums[(int64_t)blockIdx.x * E + e0 + e] = s;
    }
    __syncthreads();
  }
  for (int e = threadIdx.x; e <= E; e += blockDim.x) p.hits[(int64_t)blockIdx.x * (E + 1) + e] = hits[e];
  grid_launch_dependents();
  if (gridDim.x == 1) {
    __syncthreads();
    balance_finish<bal_threads(kPer)>(p, 1, &finish);
  }
}

__global__ void __launch_bounds__(kBalThreads) balance_finish_kernel(const __grid_constant__ Balance p, int ctas) {
  __shared__ BalFinish finish;
  grid_dependency_wait();
  grid_launch_dependents();
  balance_finish<kBalThreads>(p, ctas, &finish);
}

template <typename T, int kLanes, int kPer, bool kVec> __global__ void __launch_bounds__(bal_threads(kPer), 1) balance_grad_kernel(const __grid_constant__ Balance p) {
  constexpr int kRows = 32 / kLanes, kBatch = kPer <= 16 ? 2 : 1;
  using Row = BalRow<T, kLanes, kPer, kVec>;
  const int E = p.experts, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % kLanes, mine = lane / kLanes;
  grid_dependency_wait();
  grid_launch_dependents();
  const float g = p.grad[0] * p.load[E];
  float f[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) f[i] = Row::expert(l, i) < E ? p.load[Row::expert(l, i)] : 0.f;
  const int64_t step = (int64_t)gridDim.x * (bal_threads(kPer) / 32) * kRows;
  for (int64_t t0 = ((int64_t)blockIdx.x * (bal_threads(kPer) / 32) + warp) * kRows + mine; t0 - mine < p.tokens; t0 += kBatch * step) {
    Row row[kBatch];
    bool live[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int64_t t = t0 + i * step;
      live[i] = t < p.tokens && (p.valid == nullptr || p.valid[t * p.valid_stride] != 0);
      if (live[i]) row[i].load(reinterpret_cast<const T*>(p.z) + t * p.stride, E, l);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      float s[kPer], dot = 0.f;
      row[i].softmax(E, l, s);
#pragma unroll
      for (int k = 0; k < kPer; ++k) dot = fmaf(s[k], f[k], dot);
#pragma unroll
      for (int o = kLanes / 2; o >= 1; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
      const int64_t t = t0 + i * step;
      if (t >= p.tokens) continue;
      T* out = reinterpret_cast<T*>(p.dz) + t * p.dz_stride;
      alignas(16) T d[kPer];
#pragma unroll
      for (int k = 0; k < kPer; ++k) d[k] = from_f32<T>(live[i] ? g * s[k] * (f[k] - dot) : 0.f);
      if constexpr (kVec) {
#pragma unroll
        for (int k = 0; k < kPer; k += 4) {
          if (Row::expert(l, k) >= E) continue;
          if constexpr (sizeof(T) == 4) st16(out + Row::expert(l, k), *reinterpret_cast<const uint4*>(d + k));
          else *reinterpret_cast<uint2*>(out + Row::expert(l, k)) = *reinterpret_cast<const uint2*>(d + k);
        }
      } else {
#pragma unroll
        for (int k = 0; k < kPer; ++k)
          if (Row::expert(l, k) < E) out[Row::expert(l, k)] = d[k];
      }
    }
  }
}

// One CTA where its warps take a token or a few each, so that nothing has to be joined by a second launch; else up to a CTA per SM.
static int balance_ctas(int64_t tokens) {
  if (tokens <= 4 * kBalWarps) return 1;
  const int64_t need = (tokens + 4 * kBalWarps - 1) / (4 * kBalWarps);
  return need < kBalCtas ? (int)need : kBalCtas;
}

template <typename T, int kLanes, int kPer, bool kVec> static int balance_launch(const Balance& p, bool grad, cudaStream_t st) {
  cudaError_t e;
  if (grad) {
    const int64_t need = (p.tokens * kLanes + bal_threads(kPer) - 1) / bal_threads(kPer);
    e = launch_pdl(balance_grad_kernel<T, kLanes, kPer, kVec>, dim3((unsigned)(need < 2 * kBalCtas ? need : 2 * kBalCtas)), dim3(bal_threads(kPer)), 0, st, p);
  } else {
    const int ctas = balance_ctas(p.tokens);
    e = launch_pdl(balance_sum_kernel<T, kLanes, kPer, kVec>, dim3(ctas), dim3(bal_threads(kPer)),
                   (size_t)bal_threads(kPer) / 32 * (p.experts < kBalChunk ? p.experts : kBalChunk) * 4, st, p);
    if (e == cudaSuccess && ctas > 1) e = launch_pdl(balance_finish_kernel, dim3(1), dim3(kBalThreads), 0, st, p, ctas);
  }
  const char* what = grad ? "tkv_moe_balance_grad" : "tkv_moe_balance";
  return e == cudaSuccess ? check_launch(what) : fail(TKV_ERR_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
}
template <typename T> static int balance_run(const Balance& p, bool grad, cudaStream_t st) {
  const uintptr_t bytes = 4 * sizeof(T);
  const bool vec = p.experts % 4 == 0 && p.stride % 4 == 0 && (uintptr_t)p.z % bytes == 0 && (!grad || (p.dz_stride % 4 == 0 && (uintptr_t)p.dz % bytes == 0));
  const int E = p.experts;
  // Few lanes a token, each with 16 of its experts: what a reduction over lanes costs is shared by the tokens of a warp.  us of 65536
  // tokens, 128 experts, forward and gradient: a warp a token 24.7 and 20.2, 8 lanes a token 19.6 and 13.2
  // (a device copy of as many bytes as the gradient moves takes about 12).
  if (vec) {
    if (E <= 8) return balance_launch<T, 2, 4, true>(p, grad, st);
    if (E <= 16) return balance_launch<T, 4, 4, true>(p, grad, st);
    if (E <= 32) return balance_launch<T, 2, 16, true>(p, grad, st);
    if (E <= 64) return balance_launch<T, 4, 16, true>(p, grad, st);
    if (E <= 128) return balance_launch<T, 8, 16, true>(p, grad, st);
    if (E <= 256) return balance_launch<T, 16, 16, true>(p, grad, st);
    if (E <= 512) return balance_launch<T, 32, 16, true>(p, grad, st);
    return balance_launch<T, 32, 32, true>(p, grad, st);
  }
  if (E <= 32) return balance_launch<T, 32, 1, false>(p, grad, st);
  if (E <= 128) return balance_launch<T, 32, 4, false>(p, grad, st);
  return balance_launch<T, 32, 32, false>(p, grad, st);
}
static int balance_any(const Balance& p, int dtype, bool grad, cudaStream_t st) {
  if (dtype == TKV_BF16) return balance_run<__nv_bfloat16>(p, grad, st);
  if (dtype == TKV_F16) return balance_run<__half>(p, grad, st);
  return balance_run<float>(p, grad, st);
}

}  // namespace tkv

extern "C" int64_t tkv_moe_balance_workspace_bytes(int64_t tokens, int experts) {
  if (tokens < 0 || experts < 1) return 0;
  return (int64_t)tkv::balance_ctas(tokens) * (2 * (int64_t)experts + 1) * 4;
}

extern "C" int tkv_moe_balance(const void* logits, int64_t logit_stride, const void* choice, int64_t choice_stride, int choice_bits,
                               const uint8_t* valid, int64_t valid_stride, int64_t tokens, int experts, int top, float* loss,
                               int32_t* counts, float* load, void* workspace, int64_t workspace_bytes, int dtype, tkv_stream_t stream) {
  using namespace tkv;
  if (tokens < 0 || tokens > INT32_MAX || experts < 1 || top < 0 || elem_size(dtype) == 0 || (choice_bits != 32 && choice_bits != 64))
    return fail(TKV_ERR_ARG, "tkv_moe_balance: tokens=%lld experts=%d top=%d dtype=%d, choices of %d bits", (long long)tokens, experts, top, dtype, choice_bits);
  if (experts > kBalExperts || top > 1024 || tokens * top > INT32_MAX)
    return fail(TKV_ERR_UNSUPPORTED, "tkv_moe_balance: %d of %d experts (at most 1024), %lld tokens (at most 2^31 choices)", top, experts, (long long)tokens);
  if ((tokens && (!logits || (top && !choice))) || !loss || !counts || !load || !workspace) return fail(TKV_ERR_ARG, "tkv_moe_balance: NULL pointer argument");
  if (workspace_bytes < tkv_moe_balance_workspace_bytes(tokens, experts)) return fail(TKV_ERR_ARG, "tkv_moe_balance: workspace too small");
  Balance p = {};
  p.z = logits; p.stride = logit_stride; p.choice = choice; p.choice_stride = choice_stride; p.choice64 = choice_bits == 64;
  p.valid = valid; p.valid_stride = valid_stride; p.tokens = tokens; p.experts = experts; p.top = top;
  p.loss = loss; p.counts = counts; p.load = load;
  p.sums = reinterpret_cast<float*>(workspace);
  p.hits = reinterpret_cast<int32_t*>(p.sums + (int64_t)balance_ctas(tokens) * experts);
  return balance_any(p, dtype, false, (cudaStream_t)stream);
}

extern "C" int tkv_moe_balance_grad(const void* logits, int64_t logit_stride, const uint8_t* valid, int64_t valid_stride, const float* load,
                                    const float* grad, int64_t tokens, int experts, void* dlogits, int64_t dlogit_stride, int dtype,
                                    tkv_stream_t stream) {
  using namespace tkv;
  if (tokens < 0 || tokens > INT32_MAX || experts < 1 || elem_size(dtype) == 0)
    return fail(TKV_ERR_ARG, "tkv_moe_balance_grad: tokens=%lld experts=%d dtype=%d", (long long)tokens, experts, dtype);
  if (experts > kBalExperts) return fail(TKV_ERR_UNSUPPORTED, "tkv_moe_balance_grad: %d experts (at most 1024)", experts);
  if (tokens == 0) return TKV_OK;
  if (!logits || !load || !grad || !dlogits) return fail(TKV_ERR_ARG, "tkv_moe_balance_grad: NULL pointer argument");
  Balance p = {};
  p.z = logits; p.stride = logit_stride; p.valid = valid; p.valid_stride = valid_stride; p.tokens = tokens; p.experts = experts;
  p.load = const_cast<float*>(load); p.grad = grad; p.dz = dlogits; p.dz_stride = dlogit_stride;
  return balance_any(p, dtype, true, (cudaStream_t)stream);
}
