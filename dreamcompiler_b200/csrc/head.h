// Internal interface of the vocabulary-head kernels (linear + softmax losses
// that never keep the logits): head.cu runs what head_api.cu has validated.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "common.h"

namespace dgx {

constexpr int kHeadMaxK = 256;          // teacher entries per row
constexpr int kHeadSlot = 64;          // columns per entry of a target list's start table
constexpr int kHeadMaxDim = 1 << 23;    // R, V and d: tile and fragment counts fit 32 bits

// One problem: logits z = (H . W^T + bias) / T of R rows over V columns, and a
// sparse target per row: K ids with K probabilities. The hard target is K = 1
// with probability 1 and teacher == nullptr.
struct HeadArgs {
  const void* H;       // [R][ldh] bf16
  const void* W;       // [V][ldw] bf16
  const float* bias;   // [V] or null
  const int* idx;      // [R][K]; an id outside [0, V) is an absent entry
  const float* teacher;  // [R][K] teacher logits, or null (hard target)
  int ldh, ldw, R, V, d, K;
  float t, inv_t;      // temperature and its reciprocal
  // forward results (inputs of the backward)
  float* loss;         // [R]
  float* lse;          // [R] log-sum-exp of z
  float* mean;         // sum of loss / R, or null
  // backward
  const float* dloss;  // [R] weight per row, or null (1)
  float scale;
  void* dH;            // [R][lddh] or null
  void* dW;            // [V][lddw] or null
  float* db;           // [V] or null
  int dh_bf16, lddh, dw_bf16, lddw;
  int add_w, add_h;    // dW (fp32) and db, dH (fp32) are added to
  uint32_t* err;
};

// One launch of the tensor-core logits kernel (head_tc.cu): columns
// [c0, c0 + n) of the vocabulary, c0 a multiple of 256.
struct HeadTcArgs {
  int R, V, d, K, c0, n;
  int tiles_m, tiles_n, group_m;  // filled by the launcher
  float inv_t, k;           // 1 / T, log2(e) / T
  const float* bias;        // [V] or null
  const int* sid;           // [R][K] target ids, ascending when K > 1
  const float* sq;          // [R][K] their probabilities, or null (1)
  const uint16_t* start;    // [R][slots] first entry with id >= kHeadSlot * (slot0 + slot), or null (K = 1)
  int slots, slot0;
  float* zs;                // [R][K] out: raw logits at the ids (statistics)
                            // (a hard target's is left out of the row's statistics)
  float2* part;             // [ceil(n / head_stat_cols())][R] out: (max, sum) per slot of the piece's columns (statistics)
  float *loss, *lse_out;    // [R] out: a hard target's results where one tile holds every column
                            // (n = V <= 256; zs and part are not written then), or null (statistics)
  const float* live;        // [R] 0 where the row has no target, or null (id in [0, V))
  const float* dloss;       // [R] or null
  const float* lse;         // [R]
  float* dbp;               // [ceil(R / 32)][n] out: column sums per 32 rows, or null (gradient)
  uint32_t* err;
};
int head_stat_cols(int d, bool bias);  // columns per statistics slot: 64 or 128
cudaError_t head_logits_tc(HeadTcArgs a, const void* H, int ldh, const void* W, int ldw, bool grad, void* g, int ldg,
                           cudaStream_t s);

// The forward's statistics for up to 16 rows and a hard target (head_small.cu):
// part [slots][R] and zs [R], with slots = head_small_slots() (0: not for these
// sizes; 1: loss and lse are written at once and part is not).
int head_small_slots(int R, int V, int d);
cudaError_t head_small(const HeadTcArgs& a, const void* H, int ldh, const void* W, int ldw, int slots, float* loss,
                       float* lse, cudaStream_t s);

// Both gradient products of one piece (head_grads.cu). out[0] is dH [R][ld],
// out[1] dW [n][ld]; with splits > 1 the output is fp32 partial sums
// [splits][rows][ld]. ptr null: the product is skipped.
constexpr int kMaxSplits = 32;
struct GradOut {
  void* ptr;
  int bf16, add, ld, splits;
  float alpha;
};
struct HeadGradTc {
  const void *G, *W, *H;  // [R][ldg], [n][ldw], [R][ldh] bf16
  int ldg, ldw, ldh, R, n, d;
  GradOut out[2];
  uint32_t* err;
};
struct GradSplits {
  int dh, dw;
};
GradSplits head_grad_splits(int R, int n, int d, bool want_dh, bool want_dw);
cudaError_t head_grads_tc(const HeadGradTc& g, cudaStream_t s);

size_t head_fwd_scratch_bytes(int R, int V, int d, int K, bool lists);
size_t head_bwd_scratch_bytes(int R, int V, int d, int K, bool lists);
dgx_status head_fwd(const HeadArgs& a, void* ws, cudaStream_t s);
dgx_status head_bwd(const HeadArgs& a, void* ws, cudaStream_t s);

// lse and loss of one row with a hard target, from the statistics (m, s) of the
// OTHER columns (max of the raw logits, sum of exp((z - m) / T)) and the
// target's raw logit zt (has = false: the row has none, (m, s) are all columns).
// With the target left out of the sum a small loss, log(1 + sum / exp(zt)),
// keeps its relative precision; log of a sum near 1 would lose it.
__device__ __forceinline__ void nll_row(float m, float s, float zt, bool has, float inv_t, float& loss, float& lse) {
  loss = 0.f;
  const float mx = has ? fmaxf(m, zt) : m;
  if (!has || isinf(mx)) {  // every column masked, or an overflow: loss NaN or inf as inf - inf gives it
    lse = mx * inv_t + logf(s);
    if (has) loss = lse - zt * inv_t;
    return;
  }
  const float delta = (m - zt) * inv_t;
  if (delta <= 0.f) {
    loss = log1pf(s * expf(delta));
    lse = zt * inv_t + loss;
  } else {
    const float log_s = logf(s + expf(-delta));
    loss = delta + log_s;
    lse = m * inv_t + log_s;
  }
}

}  // namespace dgx
