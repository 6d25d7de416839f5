// How evenly a router spreads its tokens over the experts.  Of n valid tokens with k choices each and p_t = softmax(z_t):
//   c_e = choices of expert e,  f_e = c_e / (n k),  P_e = sum_t p_te / n,  loss = E sum_e f_e P_e
//   d loss / d z_te = (E / n) p_te (f_e - sum_j p_tj f_j)          (the counts have no gradient)
// Both passes read the logits once and recompute the softmax: a warp per token, its experts in the lanes' registers, so HBM (or, for
// few tokens, the launches) is the bound.  The sums over tokens stay in registers, lane by lane, and are added up in a fixed order:
// first the warps of a CTA, then the CTAs.  No atomics on floating point: equal inputs give equal bits.
#include "tkv_elem.cuh"

namespace tkv {

constexpr int kBalThreads = 512, kBalWarps = kBalThreads / 32, kBalCtas = 148;

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

// Softmax of a token's logits, expert lane + 32 i in p[i] (0 beyond the last).
template <typename T, int kPer> __device__ __forceinline__ void balance_softmax(const T* z, int experts, int lane, float* p) {
  float top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    p[i] = lane + 32 * i < experts ? to_f32<T>(z[lane + 32 * i]) : -INFINITY;
    top = fmaxf(top, p[i]);
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    p[i] = lane + 32 * i < experts ? expf(p[i] - top) : 0.f;
    sum += p[i];
  }
  const float inv = 1.0f / warp_add(sum);
#pragma unroll
  for (int i = 0; i < kPer; ++i) p[i] *= inv;
}

// Adds up the CTAs' shares; one CTA.
__device__ __forceinline__ void balance_finish(const Balance& p, int ctas, double* red /* [kBalWarps + 1] */) {
  const int E = p.experts;
  int mine = 0;
  for (int c = threadIdx.x; c < ctas; c += kBalThreads) mine += p.hits[(int64_t)c * (E + 1) + E];
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  int* whole = reinterpret_cast<int*>(red);
  if ((threadIdx.x & 31) == 0) whole[threadIdx.x >> 5] = mine;
  __syncthreads();
  int64_t n = 0;
  for (int w = 0; w < kBalWarps; ++w) n += whole[w];
  __syncthreads();
  const double inv = n > 0 ? 1.0 / (double)n : 0.0;
  double part = 0.0;
  const int lane = threadIdx.x & 31;
  for (int e0 = (threadIdx.x >> 5) * 8; e0 < E; e0 += kBalWarps * 8) {      // a warp takes 8 experts, 4 CTAs' shares at a time
    const int e = e0 + (lane & 7);
    double s = 0.0;
    int64_t c = 0;
    if (e < E)
      for (int b = lane >> 3; b < ctas; b += 4) {
        s += (double)p.sums[(int64_t)b * E + e];
        c += p.hits[(int64_t)b * (E + 1) + e];
      }
#pragma unroll
    for (int o = 8; o <= 16; o <<= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      c += __shfl_xor_sync(0xffffffffu, c, o);
    }
    if (e < E && lane < 8) {
      const double f = (double)c * inv / (double)(p.top > 0 ? p.top : 1);
      p.counts[e] = (int32_t)c;
      p.load[e] = (float)f;
      part += f * s * inv;
    }
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
  if (lane == 0) red[threadIdx.x >> 5] = part;
  __syncthreads();
  if (threadIdx.x == 0) {
    double sum = 0.0;
    for (int w = 0; w < kBalWarps; ++w) sum += red[w];
    *p.loss = (float)(sum * (double)E);
    p.load[E] = (float)((double)E * inv);
  }
}

template <typename T, int kPer> __global__ void __launch_bounds__(kBalThreads) balance_sum_kernel(const __grid_constant__ Balance p) {
  extern __shared__ float sm[];                            // [experts] sums, [experts + 1] hits
  __shared__ double red[kBalWarps + 1];
  float* sums = sm;
  int32_t* hits = reinterpret_cast<int32_t*>(sm + p.experts);
  const int E = p.experts, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  grid_dependency_wait();
  for (int e = threadIdx.x; e <= E; e += kBalThreads) { hits[e] = 0; if (e < E) sums[e] = 0.f; }
  __syncthreads();
  float acc[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) acc[i] = 0.f;
  int seen = 0;
  for (int64_t t = (int64_t)blockIdx.x * kBalWarps + warp; t < p.tokens; t += (int64_t)gridDim.x * kBalWarps) {
    if (p.valid != nullptr && p.valid[t * p.valid_stride] == 0) continue;
    ++seen;
    for (int c = lane; c < p.top; c += 32) {
      const int64_t at = t * p.choice_stride + c;
      const int64_t e = p.choice64 ? reinterpret_cast<const int64_t*>(p.choice)[at] : (int64_t) reinterpret_cast<const int32_t*>(p.choice)[at];
      if (e >= 0 && e < E) atomicAdd(&hits[e], 1);
    }
    float s[kPer];
    balance_softmax<T, kPer>(reinterpret_cast<const T*>(p.z) + t * p.stride, E, lane, s);
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] += s[i];
  }
  for (int w = 0; w < kBalWarps; ++w) {                    // the warps' sums, one warp after the other
    if (warp == w) {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (lane + 32 * i < E) sums[lane + 32 * i] += acc[i];
      if (lane == 0) hits[E] += seen;
    }
    __syncthreads();
  }
  for (int e = threadIdx.x; e <= E; e += kBalThreads) {
    p.hits[(int64_t)blockIdx.x * (E + 1) + e] = hits[e];
    if (e < E) p.sums[(int64_t)blockIdx.x * E + e] = sums[e];
  }
  grid_launch_dependents();
  if (gridDim.x == 1) {
    __syncthreads();
    balance_finish(p, 1, red);
  }
}

__global__ void __launch_bounds__(kBalThreads) balance_finish_kernel(const __grid_constant__ Balance p, int ctas) {
  __shared__ double red[kBalWarps + 1];
  grid_dependency_wait();
  grid_launch_dependents();
  balance_finish(p, ctas, red);
}

template <typename T, int kPer> __global__ void __launch_bounds__(kBalThreads) balance_grad_kernel(const __grid_constant__ Balance p) {
  const int E = p.experts, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  grid_dependency_wait();
  grid_launch_dependents();
  const float g = p.grad[0] * p.load[E];
  float f[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) f[i] = lane + 32 * i < E ? p.load[lane + 32 * i] : 0.f;
  for (int64_t t = (int64_t)blockIdx.x * kBalWarps + warp; t < p.tokens; t += (int64_t)gridDim.x * kBalWarps) {
    T* out = reinterpret_cast<T*>(p.dz) + t * p.dz_stride;
    if (p.valid != nullptr && p.valid[t * p.valid_stride] == 0) {
      for (int e = lane; e < E; e += 32) out[e] = from_f32<T>(0.f);
      continue;
    }
    float s[kPer], dot = 0.f;
    balance_softmax<T, kPer>(reinterpret_cast<const T*>(p.z) + t * p.stride, E, lane, s);
#pragma unroll
    for (int i = 0; i < kPer; ++i) dot = fmaf(s[i], f[i], dot);
    dot = warp_add(dot);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (lane + 32 * i < E) out[lane + 32 * i] = from_f32<T>(g * s[i] * (f[i] - dot));
  }
}

// Tokens of a CTA where there are fewer than one per warp of every SM; beyond, a CTA per SM (the sums of a CTA are read again).
static int balance_ctas(int64_t tokens) {
  const int64_t need = (tokens + 2 * kBalWarps - 1) / (2 * kBalWarps);
  return need < 1 ? 1 : need < kBalCtas ? (int)need : kBalCtas;
}

template <typename T, int kPer> static int balance_forward(const Balance& p, cudaStream_t st) {
  const int ctas = balance_ctas(p.tokens);
  cudaError_t e = launch_pdl(balance_sum_kernel<T, kPer>, dim3(ctas), dim3(kBalThreads), (size_t)(2 * p.experts + 1) * 4, st, p);
  if (e == cudaSuccess && ctas > 1) e = launch_pdl(balance_finish_kernel, dim3(1), dim3(kBalThreads), 0, st, p, ctas);
  if (e != cudaSuccess) return fail(TKV_ERR_LAUNCH, "tkv_moe_balance: %s", cudaGetErrorString(e));
  return check_launch("tkv_moe_balance");
}
template <typename T, int kPer> static int balance_backward(const Balance& p, cudaStream_t st) {
  const int64_t need = (p.tokens + kBalWarps - 1) / kBalWarps;
  cudaError_t e = launch_pdl(balance_grad_kernel<T, kPer>, dim3((unsigned)(need < 4 * kBalCtas ? need : 4 * kBalCtas)), dim3(kBalThreads), 0, st, p);
  if (e != cudaSuccess) return fail(TKV_ERR_LAUNCH, "tkv_moe_balance_grad: %s", cudaGetErrorString(e));
  return check_launch("tkv_moe_balance_grad");
}
template <typename T> static int balance_run(const Balance& p, bool grad, cudaStream_t st) {
  const int per = (p.experts + 31) / 32;
  if (per <= 1) return grad ? balance_backward<T, 1>(p, st) : balance_forward<T, 1>(p, st);
  if (per <= 2) return grad ? balance_backward<T, 2>(p, st) : balance_forward<T, 2>(p, st);
  if (per <= 4) return grad ? balance_backward<T, 4>(p, st) : balance_forward<T, 4>(p, st);
  if (per <= 8) return grad ? balance_backward<T, 8>(p, st) : balance_forward<T, 8>(p, st);
  return grad ? balance_backward<T, 32>(p, st) : balance_forward<T, 32>(p, st);
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
  if (experts > 1024 || top > 1024 || tokens * top > INT32_MAX)
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
  if (experts > 1024) return fail(TKV_ERR_UNSUPPORTED, "tkv_moe_balance_grad: %d experts (at most 1024)", experts);
  if (tokens == 0) return TKV_OK;
  if (!logits || !load || !grad || !dlogits) return fail(TKV_ERR_ARG, "tkv_moe_balance_grad: NULL pointer argument");
  Balance p = {};
  p.z = logits; p.stride = logit_stride; p.valid = valid; p.valid_stride = valid_stride; p.tokens = tokens; p.experts = experts;
  p.load = const_cast<float*>(load); p.grad = grad; p.dz = dlogits; p.dz_stride = dlogit_stride;
  return balance_any(p, dtype, true, (cudaStream_t)stream);
}
