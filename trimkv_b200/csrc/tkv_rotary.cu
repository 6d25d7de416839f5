// Rotary positions of queries and keys, one launch, out of place:
//   (a, b) -> scale (a cos(theta) - b sin(theta), b cos(theta) + a sin(theta)),   theta = +-position * f_i
// on the first 2 * pairs elements of every head (a = x[i], b = x[pairs + i], or a = x[2i], b = x[2i + 1]); the rest is copied.  The
// inverse turn is also the gradient: the transpose of a turn is the turn back.
//
// Bound by HBM: a head is read once and written once.  What does not depend on the head is done once per token: a CTA takes a few
// tokens, puts scale * cos and scale * sin of their angles into shared memory and then streams all heads past them.
// An angle is reduced in fp64 (position * f in turns minus the nearest whole number), so that only the sine and cosine of the
// remaining part of a turn are taken in fp32: a position of 2^31 loses no more than a position of 1.
#include "tkv_elem.cuh"

namespace tkv {

constexpr int kRotThreads = 256;

struct RotaryHeads {                                       // x [batch, heads, tokens, dim]: element strides, elements of a head consecutive
  const void* x; int64_t xb, xh, xs;
  void* y; int64_t yb, yh, ys;
  int heads;
};
struct Rotary {
  RotaryHeads part[2];                                     // queries, keys (heads 0: none)
  const void* pos; int64_t pb, ps;                         // [batch, tokens], strides in elements
  const float* freq;                                       // [pairs, 2]
  int64_t rows;                                            // batch * tokens
  int tokens, dim, pairs, tile, pos64;
  float scale, sign;
};

template <typename T, int V> struct RotVec {               // V elements as fp32; V * sizeof(T) up to 32 bytes, in words of at most 16
  static constexpr int kBytes = V * (int)sizeof(T), kWord = kBytes >= 16 ? 16 : kBytes;
  __device__ __forceinline__ static void load(const T* p, float* v) {
    alignas(16) T e[V];
#pragma unroll
    for (int i = 0; i < kBytes / kWord; ++i) {
      if constexpr (kWord == 16) *reinterpret_cast<uint4*>(reinterpret_cast<char*>(e) + 16 * i) = ld16_stream(reinterpret_cast<const char*>(p) + 16 * i);
      else if constexpr (kWord == 8) *reinterpret_cast<uint2*>(e) = *reinterpret_cast<const uint2*>(p);
      else if constexpr (kWord == 4) *reinterpret_cast<uint32_t*>(e) = *reinterpret_cast<const uint32_t*>(p);
      else e[0] = p[0];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = to_f32<T>(e[i]);
  }
  __device__ __forceinline__ static void store(T* p, const float* v) {
    alignas(16) T e[V];
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = from_f32<T>(v[i]);
#pragma unroll
    for (int i = 0; i < kBytes / kWord; ++i) {
      if constexpr (kWord == 16) st16(reinterpret_cast<char*>(p) + 16 * i, *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(e) + 16 * i));
      else if constexpr (kWord == 8) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(e);
      else if constexpr (kWord == 4) *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(e);
      else p[0] = e[0];
    }
  }
};

// A unit is V pairs, or 2 V elements behind the turned part.
template <typename T, int V, bool kHalf>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const __grid_constant__ Rotary p) {
  extern __shared__ float2 table[];                        // [tile][pairs] scale * (cos, sin)
  grid_dependency_wait();
  grid_launch_dependents();
  const int64_t row0 = (int64_t)blockIdx.x * p.tile;
  const int rows = (int)min((int64_t)p.tile, p.rows - row0);
  for (int i = threadIdx.x; i < rows * p.pairs; i += kRotThreads) {
    const int r = i / p.pairs, j = i - r * p.pairs;
    const int64_t row = row0 + r, b = row / p.tokens, s = row - b * p.tokens, at = b * p.pb + s * p.ps;
    const double where = p.pos64 ? (double)reinterpret_cast<const int64_t*>(p.pos)[at] : (double)reinterpret_cast<const int32_t*>(p.pos)[at];
    const double turns = where * (((double)p.freq[2 * j] + (double)p.freq[2 * j + 1]) * 0.15915494309189533577);
    float sn, cs;
    sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
    table[i] = make_float2(p.scale * cs, p.scale * p.sign * sn);
  }
  __syncthreads();
  const int turned = p.pairs / V, units = turned + (p.dim - 2 * p.pairs + 2 * V - 1) / (2 * V);
  const int heads = p.part[0].heads + p.part[1].heads, per_row = heads * units;
  for (int i = threadIdx.x; i < rows * per_row; i += kRotThreads) {
    const int r = i / per_row, in_row = i - r * per_row;
    int h = in_row / units;
    const int u = in_row - h * units;
    const int64_t row = row0 + r, b = row / p.tokens, s = row - b * p.tokens;
    const int which = h >= p.part[0].heads;
    const RotaryHeads& part = p.part[which];
    if (which) h -= p.part[0].heads;
    const T* x = reinterpret_cast<const T*>(part.x) + b * part.xb + h * part.xh + s * part.xs;
    T* y = reinterpret_cast<T*>(part.y) + b * part.yb + h * part.yh + s * part.ys;
    float a[V], c[V];
    const int at0 = u < turned ? (kHalf ? u * V : 2 * u * V) : 2 * p.pairs + 2 * (u - turned) * V;
    const int at1 = u < turned && kHalf ? p.pairs + u * V : at0 + V;
    RotVec<T, V>::load(x + at0, a);
    const bool both = V > 1 || at1 < p.dim;                // an odd number of elements behind the turned part: V is 1
    if (both) RotVec<T, V>::load(x + at1, c);
    if (u < turned) {
      const float2* t = table + r * p.pairs + u * V;
      if constexpr (kHalf) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float2 w = t[e];
          const float x0 = a[e], x1 = c[e];
          a[e] = fmaf(x0, w.x, -x1 * w.y);
          c[e] = fmaf(x1, w.x, x0 * w.y);
        }
      } else if constexpr (V == 1) {
        const float2 w = t[0];
        const float x0 = a[0], x1 = c[0];
        a[0] = fmaf(x0, w.x, -x1 * w.y);
        c[0] = fmaf(x1, w.x, x0 * w.y);
      } else {
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          const float2 w = t[e / 2], z = t[V / 2 + e / 2];
          const float x0 = a[e], x1 = a[e + 1], x2 = c[e], x3 = c[e + 1];
          a[e] = fmaf(x0, w.x, -x1 * w.y);
          a[e + 1] = fmaf(x1, w.x, x0 * w.y);
          c[e] = fmaf(x2, z.x, -x3 * z.y);
          c[e + 1] = fmaf(x3, z.x, x2 * z.y);
        }
      }
    }
    RotVec<T, V>::store(y + at0, a);
    if (both) RotVec<T, V>::store(y + at1, c);
  }
}

template <typename T, int V, bool kHalf> static int launch_rotary(const Rotary& p, cudaStream_t st) {
  const int64_t blocks = (p.rows + p.tile - 1) / p.tile;
  const size_t bytes = (size_t)p.tile * p.pairs * sizeof(float2);
  cudaError_t e = launch_pdl(rotary_kernel<T, V, kHalf>, dim3((unsigned)blocks), dim3(kRotThreads), bytes, st, p);
  if (e != cudaSuccess) return fail(TKV_ERR_LAUNCH, "tkv_rotary: %s", cudaGetErrorString(e));
  return check_launch("tkv_rotary");
}
template <typename T, bool kHalf> static int launch_rotary(const Rotary& p, int v, cudaStream_t st) {
  switch (v) {
    case 8: return launch_rotary<T, 8, kHalf>(p, st);
    case 4: return launch_rotary<T, 4, kHalf>(p, st);
    case 2: return launch_rotary<T, 2, kHalf>(p, st);
    default: return launch_rotary<T, 1, kHalf>(p, st);
  }
}

}  // namespace tkv

extern "C" int tkv_rotary(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_ss, void* q_out, int q_heads, const void* k, int64_t k_sb,
                          int64_t k_sh, int64_t k_ss, void* k_out, int k_heads, const void* pos, int pos_bits, int64_t pos_sb,
                          int64_t pos_ss, const float* freq_hi_lo, int batch, int tokens, int dim, int pairs, int layout, int inverse,
                          float scale, int dtype, tkv_stream_t stream) {
  using namespace tkv;
  if (batch < 0 || tokens < 0 || q_heads < 0 || k_heads < 0 || dim < 0 || pairs < 0 || (int64_t)2 * pairs > dim)
    return fail(TKV_ERR_ARG, "tkv_rotary: batch=%d tokens=%d heads=%d, %d dim=%d pairs=%d", batch, tokens, q_heads, k_heads, dim, pairs);
  if (elem_size(dtype) == 0 || (pos_bits != 32 && pos_bits != 64) || (layout != 0 && layout != 1))
    return fail(TKV_ERR_ARG, "tkv_rotary: dtype=%d, positions of %d bits, layout=%d", dtype, pos_bits, layout);
  if ((int64_t)batch * tokens == 0 || q_heads + k_heads == 0 || dim == 0) return TKV_OK;
  if ((q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out)) || !pos || (pairs && !freq_hi_lo))
    return fail(TKV_ERR_ARG, "tkv_rotary: NULL pointer argument");
  if (pairs > 4096 || dim > 65536 || q_heads + k_heads > 16384)
    return fail(TKV_ERR_UNSUPPORTED, "tkv_rotary: %d heads of %d, %d pairs", q_heads + k_heads, dim, pairs);
  Rotary p;
  const int64_t qt = (int64_t)q_heads * dim, kt = (int64_t)k_heads * dim;       // outputs: [batch, tokens, heads, dim]
  p.part[0] = {q, q_sb, q_sh, q_ss, q_out, qt * tokens, dim, qt, q_heads};
  p.part[1] = {k, k_sb, k_sh, k_ss, k_out, kt * tokens, dim, kt, k_heads};
  p.pos = pos; p.pb = pos_sb; p.ps = pos_ss; p.pos64 = pos_bits == 64;
  p.freq = freq_hi_lo;
  p.rows = (int64_t)batch * tokens;
  p.tokens = tokens; p.dim = dim; p.pairs = pairs;
  p.scale = scale; p.sign = inverse ? -1.f : 1.f;
  // The widest vectors that the sizes, strides and addresses allow.
  const int size = elem_size(dtype);
  int v = 8;
  auto fits = [&](int n) {
    const int64_t bytes = n * size < 16 ? n * size : 16;
    if (pairs % n || (dim - 2 * pairs) % (2 * n) || ((int64_t)dim * size) % bytes) return false;
    for (const RotaryHeads& h : p.part)
      if (h.heads && ((uintptr_t)h.x % bytes || (uintptr_t)h.y % bytes || (h.xb * size) % bytes || (h.xh * size) % bytes || (h.xs * size) % bytes))
        return false;
    return true;
  };
  while (v > 1 && !fits(v)) v >>= 1;
  // Tokens per CTA: several where there are enough of them for every SM's resident CTAs, so that the units of a head that do not
  // fill the last round of threads count less; one where tokens are few.  The table stays within 32 KB.
  p.tile = p.rows >= 148 * 32 ? 4 : p.rows >= 148 * 16 ? 2 : 1;
  while (p.tile > 1 && (int64_t)p.tile * pairs * 8 > 32768) p.tile >>= 1;
  if ((p.rows + p.tile - 1) / p.tile > INT32_MAX) return fail(TKV_ERR_UNSUPPORTED, "tkv_rotary: %lld tokens", (long long)p.rows);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == TKV_BF16) return layout == 0 ? launch_rotary<__nv_bfloat16, true>(p, v, st) : launch_rotary<__nv_bfloat16, false>(p, v, st);
  if (dtype == TKV_F16) return layout == 0 ? launch_rotary<__half, true>(p, v, st) : launch_rotary<__half, false>(p, v, st);
  return layout == 0 ? launch_rotary<float, true>(p, v, st) : launch_rotary<float, false>(p, v, st);
}
