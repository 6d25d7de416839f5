// Cross entropy of hidden rows x [tokens, width] against the vocabulary of w [vocab, width], without keeping the logits.
//   s = x w^T,  lse_t = log sum_v exp(s_tv),  loss_t = lse_t - s_t,label
//   dL_tv = g_t (exp(s_tv - lse_t) - [v = label_t]),  dx = dL w,  dw = dL^T x
// The tokens that count are moved together first (their places, labels and lse are the "plan" that the backward pass starts from), so
// that ignored ones cost nothing and nothing of them, NaN included, gets anywhere.  Then the vocabulary goes by in tiles: the forward pass
// keeps a maximum and a sum per (token, tile), the backward pass computes the logits of a piece of the vocabulary again, turns them into
// the piece of dL, and multiplies that with w and x.  lse is kept as the largest logit and the base-2 logarithm of the sum of the weights
// beside it: their sum in fp32 would lose the digits that a nearly certain token's loss and gradient consist of.
#pragma once
#include "tkv_elem.cuh"

namespace tkv {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kVlRowTile = 256;                            // workspaces hold whole tiles of rows

// int32 words: [0] tokens that count, [1] is 1 if a label was out of range, [2] if a wait ran out, then of the tokens that count lse (two fp32), rows,
// labels, and p - 1 of the label (fp32), which the gradients take from here: near 1 - p = 0 it is lost in a logit made again by another form.
struct VlossPlan {
  int32_t* head; float2* lse; int32_t* rows; int32_t* label; float* own;
};
inline __host__ __device__ VlossPlan vloss_plan(int32_t* p, int64_t tokens) {
  return {p, reinterpret_cast<float2*>(p + 4), p + 4 + 2 * tokens, p + 4 + 3 * tokens, reinterpret_cast<float*>(p + 4 + 4 * tokens)};
}

// exp(x - top) of a logit or a maximum x <= top; nothing counts for nothing where there is no maximum yet.
__device__ __forceinline__ float vl_weight(float x, float top) { return x == -INFINITY ? 0.f : exp2f((x - top) * kLog2e); }

struct Vloss {
  const void* x; int64_t x_stride;                         // rows of the caller
  const void* w;
  int64_t vocab;
  int tokens, width, dtype;
  VlossPlan plan;
  int32_t* status;
  // forward
  float2* part; int tiles;                                 // [tokens][tiles] largest logit of a tile, sum of the weights beside it
  float* mine;                                             // [tokens] logit of the label
  // backward
  const float* g;                                          // [tokens] gradient of each counting row's loss, times g_scale
  const float* g_scale;                                    // [2] scale and its inverse
  const int* slots;                                        // [2] shares of dx; tiles of dw that make up for a tile of dx fewer
  void* dl; int64_t piece;                                 // [tokens][piece]
  float* rest;                                             // [tokens] what rounding dL to 16 bits took from the label's entry (vloss_tc_backward)
  float* acc;                                              // [*slots][tokens that count, whole tiles of acc_rows][width] shares of dx
  int acc_rows;
  void* dw;
};

inline int64_t vl_round(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

constexpr int kVlMaxSlots = 32;
// What a launch of the gradients has to share out, for the choice of the shares of dx: workers, rows of a tile and what rows
// of a share are rounded to, tiles of the width and of a piece, steps of a piece, elements of a step, room for shares of `tokens` rows (fewer
// rows that count leave room for more shares), and the most shares that the launches compute: the grid's, where it has a block for each.
struct VlossWork { int workers, rows, acc_rows, ht, vt, steps, step, room, tokens, most; bool dx, dw; };

int vloss_plan_rows(const Vloss& p, const int64_t* labels, int64_t ignore, float* loss, cudaStream_t st);

// The form on the tensor cores (tkv_vloss_tc.cu): widths of multiples of 8, w and dw on 16 bytes; x of any alignment.
bool vloss_tc_shape(int tokens, int64_t vocab, int width, int dtype);
int64_t vloss_tc_bytes(int tokens, int64_t vocab, int width, int dtype, bool backward, bool dx);
VlossWork vloss_tc_work(int tokens, int64_t vocab, int width, int dtype, bool want_dx, bool want_dw);
int vloss_tc_forward(Vloss& p, const int64_t* labels, int64_t ignore, float* loss, void* ws, cudaStream_t st);   // the plan, part and mine; sets tiles
int vloss_tc_backward(Vloss& p, void* ws, bool want_dx, cudaStream_t st);                                        // dw and acc

}  // namespace tkv
