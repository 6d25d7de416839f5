// Rotary positions of queries and keys, one launch, out of place:
//   (a, b) -> scale (a cos(theta) - b sin(theta), b cos(theta) + a sin(theta)),   theta = +-position * f_i
// on the first 2 * pairs elements of every head (a = x[i], b = x[pairs + i], or a = x[2i], b = x[2i + 1]); the rest is copied.  The
// inverse turn is also the gradient: the transpose of a turn is the turn back.
//
// Bound by HBM in bytes (a head is read once and written once), and near it in instructions.  What does not depend on the head is done
// once per token: a CTA takes a run of tokens, puts scale * cos and scale * sin of all their angles into shared memory and then walks the
// tokens, every thread with the same 8 pairs of the same head each time: its addresses advance by one stride, the next token's vectors are
// requested before this one's are turned, and two pairs go through the multiply-adds at a time.
// An angle is reduced in fp64 (position * f in turns minus the nearest whole number), so that only the sine and cosine of the
// remaining part of a turn are taken in fp32: a position of 2^31 loses no more than a position of 1.
#include "tkv_elem.cuh"

namespace tkv {

// Most threads of a CTA, CTAs of that size an SM; most angles and tokens of a run.  us of 8192 tokens of 40 heads of 128 in bf16, halves
// (a device copy of the same bytes: 28.8), by threads, tokens requested ahead and tokens of a run: 320, 2, 4: 29.7; 1: 33.8; 4: 42; runs
// of 2: 34, 6: 32, 64: 32.6; 512 threads: 37.  One CTA for a whole token's heads, angles and rows one after the other: 35.
constexpr int kRotThreads = 320, kRotCtas = 4, kRotTable = 4096, kRotRun = 4, kRotAhead = 2;

struct RotaryHeads {                                       // x [batch, heads, tokens, dim]: element strides, elements of a head consecutive
  const void* x; int64_t xb, xh, xs;
  void* y; int64_t yb, yh, ys;
  int heads;
};
struct Rotary {
  RotaryHeads part[2];                                     // queries, keys (heads 0: none)
  const void* pos; int64_t pb, ps;                         // [batch, tokens], strides in elements
  const float* freq;                                       // [pairs, 2]
  int64_t rows;                                            // batch * tokens (32 bits)
  int tokens, dim, pairs, run, pos64;                      // run: tokens of a CTA
  int units, lanes, side;                                  // of a head; threads of a token; tokens side by side
  float scale, sign;
};

// V elements as they are in memory, in words of at most 16 bytes: requested together, well before they are used.
template <typename T, int V> struct RotVec {
  static constexpr int kBytes = V * (int)sizeof(T), kWord = kBytes >= 16 ? 16 : kBytes;
  alignas(16) T e[V];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kBytes / kWord; ++i) {
      if constexpr (kWord == 16) *reinterpret_cast<uint4*>(reinterpret_cast<char*>(e) + 16 * i) = ld16_stream(reinterpret_cast<const char*>(p) + 16 * i);
      else if constexpr (kWord == 8) *reinterpret_cast<uint2*>(e) = *reinterpret_cast<const uint2*>(p);
      else if constexpr (kWord == 4) *reinterpret_cast<uint32_t*>(e) = *reinterpret_cast<const uint32_t*>(p);
      else e[0] = p[0];
    }
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kBytes / kWord; ++i) {
      if constexpr (kWord == 16) st16(reinterpret_cast<char*>(p) + 16 * i, *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(e) + 16 * i));
      else if constexpr (kWord == 8) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(e);
      else if constexpr (kWord == 4) *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(e);
      else p[0] = e[0];
    }
  }
};
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return fma2(a, b, make_float2(-0.f, -0.f)); }
template <typename T> __device__ __forceinline__ float2 rot_two(const T* e) { return make_float2(to_f32<T>(e[0]), to_f32<T>(e[1])); }
template <> __device__ __forceinline__ float2 rot_two<__nv_bfloat16>(const __nv_bfloat16* e) {
  const uint32_t w = *reinterpret_cast<const uint32_t*>(e);
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 rot_two<__half>(const __half* e) { return __half22float2(*reinterpret_cast<const __half2*>(e)); }
template <typename T> __device__ __forceinline__ void rot_put(T* e, float2 v) {
  if constexpr (sizeof(T) == 4) { e[0] = v.x; e[1] = v.y; }
  else if constexpr (__is_same(T, __half)) *reinterpret_cast<__half2*>(e) = __floats2half2_rn(v.x, v.y);
  else *reinterpret_cast<__nv_bfloat162*>(e) = __floats2bfloat162_rn(v.x, v.y);
}
// Turns a unit: halves hold the pairs' first and second elements, else a and c hold pair after pair.  cs, sn: of its pairs.
template <typename T, int V, bool kHalf> __device__ __forceinline__ void rot_unit(RotVec<T, V>& a, RotVec<T, V>& c, const float* cs, const float* sn) {
  if constexpr (V == 1) {
    const float x = to_f32<T>(a.e[0]), y = to_f32<T>(c.e[0]);
    a.e[0] = from_f32<T>(fmaf(x, cs[0], -y * sn[0]));
    c.e[0] = from_f32<T>(fmaf(y, cs[0], x * sn[0]));
  } else if constexpr (kHalf) {
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const float2 x = rot_two<T>(a.e + e), y = rot_two<T>(c.e + e), w = *reinterpret_cast<const float2*>(cs + e), z = *reinterpret_cast<const float2*>(sn + e);
      rot_put<T>(a.e + e, fma2(y, make_float2(-z.x, -z.y), mul2(x, w)));
      rot_put<T>(c.e + e, fma2(x, z, mul2(y, w)));
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; e += 2) {                       // (x, y) cos + (-y, x) sin
      const float2 p = rot_two<T>(a.e + e), q = rot_two<T>(c.e + e);
      const float w0 = cs[e / 2], z0 = sn[e / 2], w1 = cs[V / 2 + e / 2], z1 = sn[V / 2 + e / 2];
      rot_put<T>(a.e + e, fma2(make_float2(p.y, p.x), make_float2(-z0, z0), mul2(p, make_float2(w0, w0))));
      rot_put<T>(c.e + e, fma2(make_float2(q.y, q.x), make_float2(-z1, z1), mul2(q, make_float2(w1, w1))));
    }
  }
}

// A unit is V pairs, or 2 V elements behind the turned part.
template <typename T, int V, bool kHalf>
__global__ void __launch_bounds__(kRotThreads, kRotCtas) rotary_kernel(const __grid_constant__ Rotary p) {
  extern __shared__ __align__(16) float table[];           // [run][2][pairs]: scale * cos, scale * sin
  grid_dependency_wait();
  grid_launch_dependents();
  const int row0 = blockIdx.x * p.run, run = min(p.run, (int)p.rows - row0);
  const int b0 = row0 / p.tokens, s0 = row0 - b0 * p.tokens;
  const int heads = p.part[0].heads + p.part[1].heads, per_token = heads * p.units, turned = p.pairs / V;
  const int slot = threadIdx.x / p.lanes;
  bool made = false;
  for (int w = threadIdx.x - slot * p.lanes; ; w += p.lanes) {          // more units than threads: the run again with the next ones
    const bool mine = slot < p.side && w < per_token;
    const int head = mine ? w / p.units : 0, u = mine ? w - head * p.units : 0;
    const bool second = head >= p.part[0].heads, turns = u < turned;
    const RotaryHeads& part = p.part[second];
    const int64_t h = second ? head - p.part[0].heads : head;
    const int at0 = turns ? (kHalf ? u * V : 2 * u * V) : 2 * p.pairs + 2 * (u - turned) * V;
    const int at1 = turns && kHalf ? p.pairs + u * V : at0 + V;
    const bool both = V > 1 || at1 < p.dim;                // an odd number of elements behind the turned part: V is 1
    const T* x = reinterpret_cast<const T*>(part.x) + h * part.xh + at0;
    T* y = reinterpret_cast<T*>(part.y) + h * part.yh + (int64_t)row0 * part.ys + at0;
    const int gap = at1 - at0;
    const float* cs = table + u * V;
    int b = b0, s = s0 + slot, next = slot;                // the next token to request
    RotVec<T, V> a[kRotAhead], c[kRotAhead];
    auto request = [&](RotVec<T, V>& va, RotVec<T, V>& vc) {
      if (mine && next < run) {
        if (s >= p.tokens) { b += s / p.tokens; s %= p.tokens; }
        const T* from = x + b * part.xb + s * part.xs;
        va.load(from);
        if (both) vc.load(from + gap);
      }
      s += p.side;
      next += p.side;
    };
#pragma unroll
    for (int i = 0; i < kRotAhead; ++i) request(a[i], c[i]);
    if (!made) {
      made = true;
      for (int i = threadIdx.x; i < run * p.pairs; i += blockDim.x) {
        const int t = i / p.pairs, j = i - t * p.pairs;
        int bt = b0, st = s0 + t;
        if (st >= p.tokens) { bt += st / p.tokens; st %= p.tokens; }
        const int64_t at = bt * p.pb + st * p.ps;
        const double where = p.pos64 ? (double)reinterpret_cast<const int64_t*>(p.pos)[at] : (double)reinterpret_cast<const int32_t*>(p.pos)[at];
        const double turned_by = where * (((double)p.freq[2 * j] + (double)p.freq[2 * j + 1]) * 0.15915494309189533577);
        float sn, cn;
        sincospif(2.0f * (float)(turned_by - rint(turned_by)), &sn, &cn);
        table[2 * t * p.pairs + j] = p.scale * cn;
        table[(2 * t + 1) * p.pairs + j] = p.scale * p.sign * sn;
      }
      __syncthreads();
    }
    for (int t = slot; mine && t < run;) {
#pragma unroll
      for (int i = 0; i < kRotAhead; ++i) {
        if (t < run) {
          if (turns) rot_unit<T, V, kHalf>(a[i], c[i], cs + 2 * t * p.pairs, cs + (2 * t + 1) * p.pairs);
          T* to = y + t * part.ys;
          a[i].store(to);
          if (both) c[i].store(to + gap);
          request(a[i], c[i]);
          t += p.side;
        }
      }
    }
    if (w - (int)threadIdx.x + slot * p.lanes + p.lanes >= per_token) break;   // the same for all threads
  }
}

template <typename T, int V, bool kHalf> static int launch_rotary(const Rotary& p, cudaStream_t st) {
  const int threads = (p.lanes * p.side + 31) / 32 * 32;
  cudaError_t e = launch_pdl(rotary_kernel<T, V, kHalf>, dim3((unsigned)((p.rows + p.run - 1) / p.run)), dim3(threads),
                             (size_t)p.run * p.pairs * 8, st, p);
  if (e != cudaSuccess) return fail(TKV_ERR_LAUNCH, "tkv_rotary: %s", cudaGetErrorString(e));
  return check_launch("tkv_rotary");
}
template <typename T, bool kHalf> static int launch_rotary(const Rotary& p, int v, cudaStream_t st) {
  switch (v) {
    case 8:
      if constexpr (sizeof(T) == 2) return launch_rotary<T, 8, kHalf>(p, st);
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
  if (pairs > kRotTable || dim > 65536 || q_heads + k_heads > 16384)
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
  int v = 16 / size;                   // 16 bytes
  auto fits = [&](int n) {
    const int64_t bytes = n * size < 16 ? n * size : 16;
    if (pairs % n || (dim - 2 * pairs) % (2 * n) || ((int64_t)dim * size) % bytes) return false;
    for (const RotaryHeads& h : p.part)
      if (h.heads && ((uintptr_t)h.x % bytes || (uintptr_t)h.y % bytes || (h.xb * size) % bytes || (h.xh * size) % bytes || (h.xs * size) % bytes))
        return false;
    return true;
  };
  while (v > 1 && !fits(v)) v >>= 1;
  if (p.rows > INT32_MAX / 2) return fail(TKV_ERR_UNSUPPORTED, "tkv_rotary: %lld tokens", (long long)p.rows);
  p.units = pairs / v + (dim - 2 * pairs + 2 * v - 1) / (2 * v);
  // Threads of a token: one per unit up to kRotThreads; beyond, as many rounds over the run as that takes.  Few units: tokens side by side.
  const int64_t per_token = (int64_t)(q_heads + k_heads) * p.units;
  const int64_t rounds = (per_token + kRotThreads - 1) / kRotThreads;
  p.lanes = (int)((per_token + rounds - 1) / rounds);
  p.side = p.lanes >= 128 ? 1 : 256 / p.lanes;
  const int64_t wave = 148 * (kRotThreads * kRotCtas / ((p.lanes * p.side + 31) / 32 * 32));     // CTAs that run at once
  int64_t run = (p.rows + wave - 1) / wave;
  if (run > kRotRun * p.side) run = kRotRun * p.side;
  if (run < p.side) run = p.side;
  if (pairs && run > kRotTable / pairs) run = kRotTable / pairs;
  p.run = (int)(run < 1 ? 1 : run);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == TKV_BF16) return layout == 0 ? launch_rotary<__nv_bfloat16, true>(p, v, st) : launch_rotary<__nv_bfloat16, false>(p, v, st);
  if (dtype == TKV_F16) return layout == 0 ? launch_rotary<__half, true>(p, v, st) : launch_rotary<__half, false>(p, v, st);
  return layout == 0 ? launch_rotary<float, true>(p, v, st) : launch_rotary<float, false>(p, v, st);
}
