// Vocabulary head: linear layer + softmax + loss with a sparse target, forward
// and backward, in pieces of the vocabulary. The logits of one piece at a time
// exist in scratch; what is kept between forward and backward is the row
// log-sum-exp.
//
//   z = (H W^T + b) / T        lse_r = log sum_j exp(z_rj)
//   hard target t_r:           loss_r = lse_r - z_{r,t}
//   soft target (ids i_k, probabilities q_k = softmax(teacher_k / T)):
//                              loss_r = T^2 sum_k q_k (log q_k - z_{r,i_k} + lse_r)
//   G_rj = w_r (exp(z_rj - lse_r) - q_rj)    dH = s G W    dW = s G^T H    db = s sum_r G
// with s the caller's scale (times T for the soft target) and w_r the row's
// weight, 0 for a row without a target.
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>

#include "gemm.h"
#include "head.h"
#include "sm100.cuh"

namespace dgx {
namespace {

constexpr int kNoId = 0x7fffffff;  // absent entry of a sorted target list

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// ---------------------------------------------------------------- target lists
// One warp per row: q = softmax(teacher / T) over the entries whose id lies in
// [0, V), and the entries in ascending order of (id, position), absent ones
// last (id kNoId, q 0). A teacher logit of -inf has q = 0; a row whose entries
// are all absent or -inf has live = 0. The rank of an entry is the number of
// entries before it (K <= 256: at most 8 x 256 comparisons per lane).
__global__ void head_lists_kernel(const int* __restrict__ idx, const float* __restrict__ teacher, int R, int V, int K,
                                  float inv_t, int* __restrict__ sid, float* __restrict__ sq,
                                  float* __restrict__ live) {
  __shared__ int ids_s[4][kHeadMaxK];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.x * 4 + w;
  if (row >= R) return;
  int* ids = ids_s[w];
  const int* ir = idx + (size_t)row * K;
  const float* tr = teacher + (size_t)row * K;
  float mx = -INFINITY;
  for (int k = lane; k < K; k += 32) {
    const int id = ir[k];
    const bool ok = id >= 0 && id < V;
    ids[k] = ok ? id : kNoId;
    if (ok) mx = fmaxf(mx, tr[k]);
  }
  mx = warp_max(mx);
  float s = 0.f;
  if (mx != -INFINITY)
    for (int k = lane; k < K; k += 32)
      if (ids[k] != kNoId) s += expf((tr[k] - mx) * inv_t);
  s = warp_sum(s);
  __syncwarp();
  const bool any = mx != -INFINITY;
  const float inv_s = any ? 1.f / s : 0.f;
  for (int k = lane; k < K; k += 32) {
    const int id = ids[k];
    int rank = 0;
    for (int j = 0; j < K; ++j) rank += (ids[j] < id || (ids[j] == id && j < k)) ? 1 : 0;
    const float q = (any && id != kNoId) ? expf((tr[k] - mx) * inv_t) * inv_s : 0.f;
    sid[(size_t)row * K + rank] = id;
    sq[(size_t)row * K + rank] = q;
  }
  if (lane == 0) live[row] = any ? 1.f : 0.f;
}

// ---------------------------------------------------------------- forward
// Row statistics of one piece of logits z [R][ldz] (columns c0 .. c0 + n of
// the vocabulary): (max, sum of exp((z - max) / T)) into part[row], and the
// raw logits at the target's ids into zs. One warp per row.
__global__ void head_stats_kernel(const float* __restrict__ z, int ldz, int c0, int n, int R, float inv_t,
                                  const int* __restrict__ sid, int K, float* __restrict__ zs,
                                  float2* __restrict__ part) {
  const int row = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= R) return;
  const float* zr = z + (size_t)row * ldz;
  float mx = -INFINITY;
  for (int j = lane; j < n; j += 32) mx = fmaxf(mx, zr[j]);
  mx = warp_max(mx);
  const float base = mx == -INFINITY ? 0.f : mx;
  float s = 0.f;
  for (int j = lane; j < n; j += 32) s += expf((zr[j] - base) * inv_t);
  s = warp_sum(s);
  if (lane == 0) part[row] = make_float2(mx, s);
  for (int k = lane; k < K; k += 32) {
    const int id = sid[(size_t)row * K + k];
    if (id >= c0 && id < c0 + n) zs[(size_t)row * K + k] = zr[id - c0];
  }
}

// lse and loss from the partial statistics part[t][R] of `nt` pieces. One warp
// per row. Hard target: sq == null.
__global__ void head_finish_kernel(const float2* __restrict__ part, int nt, int R, int V, float t, float inv_t,
                                   const int* __restrict__ sid, const float* __restrict__ sq, int K,
                                   const float* __restrict__ zs, float* __restrict__ loss, float* __restrict__ lse) {
  const int row = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= R) return;
  float m = -INFINITY, s = 0.f;
  for (int i = lane; i < nt; i += 32) {
    const float2 p = part[(size_t)i * R + row];
    const float mn = fmaxf(m, p.x), base = mn == -INFINITY ? 0.f : mn;
    s = s * expf((m - base) * inv_t) + p.y * expf((p.x - base) * inv_t);
    m = mn;
  }
  const float mr = warp_max(m), base = mr == -INFINITY ? 0.f : mr;
  s = warp_sum(s * expf((m - base) * inv_t));
  const float log_s = logf(s);
  // z - lse = (raw - max)/T - log s: the subtraction of the maximum first
  // keeps the loss accurate when the logits are large
  float l = 0.f;
  for (int k = lane; k < K; k += 32) {
    const int id = sid[(size_t)row * K + k];
    if (id < 0 || id >= V) continue;
    const float q = sq ? sq[(size_t)row * K + k] : 1.f;
    if (q == 0.f) continue;
    const float lp = (zs[(size_t)row * K + k] - base) * inv_t - log_s;
    l += sq ? q * (logf(q) - lp) : -lp;
  }
  l = warp_sum(l);
  if (lane == 0) {
    lse[row] = base * inv_t + log_s;
    loss[row] = t * t * l;
  }
}

// *mean = sum(loss) / R in a fixed order (one block).
__global__ void head_mean_kernel(const float* __restrict__ loss, int R, float* __restrict__ mean) {
  __shared__ float red[32];
  float s = 0.f;
  for (int i = threadIdx.x; i < R; i += blockDim.x) s += loss[i];
  s = warp_sum(s);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x < 32) {
    s = warp_sum(threadIdx.x < (blockDim.x >> 5) ? red[threadIdx.x] : 0.f);
    if (threadIdx.x == 0) *mean = s / R;
  }
}

// ---------------------------------------------------------------- backward
constexpr int kSlabRows = 32;  // rows per partial column sum

// G of one piece from its logits: a block owns kSlabRows rows and 256 columns,
// one column per thread. G is rounded to bf16 (the operand of the gradient
// GEMMs); the column sums are taken before the rounding.
__global__ void head_grad_kernel(const float* __restrict__ z, int ldz, int c0, int n, int R, int V, float inv_t,
                                 const float* __restrict__ lse, const float* __restrict__ dloss,
                                 const float* __restrict__ live, const int* __restrict__ sid,
                                 const float* __restrict__ sq, int K, __nv_bfloat16* __restrict__ g, int ldg,
                                 float* __restrict__ dbp) {
  const int j = blockIdx.x * 256 + threadIdx.x;
  const int r0 = blockIdx.y * kSlabRows, r1 = min(R, r0 + kSlabRows);
  if (j >= ldg) return;
  float col = 0.f;
  for (int r = r0; r < r1; ++r) {
    float w;
    if (live) {
      w = live[r];
    } else {
      const int t = sid[r];
      w = (t >= 0 && t < V) ? 1.f : 0.f;
    }
    float v = 0.f;
    if (w != 0.f && j < n) {
      if (dloss) w = dloss[r];
      v = expf(z[(size_t)r * ldz + j] * inv_t - lse[r]);
      for (int k = 0; k < K; ++k)
        if (sid[(size_t)r * K + k] == c0 + j) v -= sq ? sq[(size_t)r * K + k] : 1.f;
      v *= w;
    }
    g[(size_t)r * ldg + j] = __float2bfloat16_rn(v);
    col += v;
  }
  if (dbp && j < n) dbp[(size_t)blockIdx.y * n + j] = col;
}

// db[j] (+)= scale * sum over slabs of dbp[slab][j], in order.
__global__ void head_db_kernel(const float* __restrict__ dbp, int slabs, int n, float scale, int accumulate,
                               float* __restrict__ db) {
  const int j = blockIdx.x * blockDim.x + threadIdx.x;
  if (j >= n) return;
  float s = 0.f;
  for (int i = 0; i < slabs; ++i) s += dbp[(size_t)i * n + j];
  db[j] = (accumulate ? db[j] : 0.f) + scale * s;
}

// out[r][j] (+)= scale * acc[r][j], rounded once to bf16 where asked.
__global__ void head_out_kernel(const float* __restrict__ acc, int rows, int d, float scale, int bf16_out,
                                int accumulate, void* __restrict__ out, int ldo) {
  const long long total = (long long)rows * d;
  for (long long e = blockIdx.x * (long long)blockDim.x + threadIdx.x; e < total;
       e += (long long)gridDim.x * blockDim.x) {
    const long long r = e / d, j = e % d;
    const float v = scale * acc[e];
    if (bf16_out) {
      reinterpret_cast<__nv_bfloat16*>(out)[r * ldo + j] = __float2bfloat16_rn(v);
    } else {
      float* o = reinterpret_cast<float*>(out) + r * ldo + j;
      *o = accumulate ? *o + v : v;
    }
  }
}

constexpr size_t kPieceBytes = 256u << 20;  // fp32 logits of one piece

size_t align128(size_t b) { return (b + 127) & ~size_t(127); }

// Columns of one piece: as many as keep R x columns fp32 logits within
// kPieceBytes, a multiple of 256.
int piece_cols(int R, int V) {
  const long long c = (long long)(kPieceBytes / 4 / (size_t)R) / 256 * 256;
  return (int)std::min<long long>(std::max<long long>(c, 256), (V + 255) / 256 * 256);
}

dgx_status piece_logits(const HeadArgs& a, int c0, int n, float* z, int ldz, cudaStream_t s) {
  GemmArgs g{};
  g.M = a.R;
  g.N = n;
  g.K = a.d;
  g.lda = a.ldh;
  g.ldb = a.ldw;
  g.ldc = ldz;
  g.transB = 1;
  g.C = z;
  g.bias = a.bias ? a.bias + c0 : nullptr;
  g.err = a.err;
  return gemm_run(g, a.H, (const __nv_bfloat16*)a.W + (size_t)c0 * a.ldw, DGX_BF16, 0, nullptr, 0, s);
}

struct Carve {
  char* p;
  template <typename T>
  T* take(size_t n) {
    T* r = reinterpret_cast<T*>(p);
    p += align128(n * sizeof(T));
    return r;
  }
};

}  // namespace

size_t head_fwd_scratch_bytes(int R, int V, int d, int K, bool lists) {
  const int pc = piece_cols(R, V), nt = (V + pc - 1) / pc;
  size_t b = align128((size_t)R * pc * 4) + align128((size_t)nt * R * 8) + align128((size_t)R * K * 4);
  if (lists) b += 2 * align128((size_t)R * K * 4) + align128((size_t)R * 4);
  return b;
}

size_t head_bwd_scratch_bytes(int R, int V, int d, int K, bool lists) {
  const int pc = piece_cols(R, V);
  size_t b = align128((size_t)R * pc * 4) + align128((size_t)R * pc * 2) +
             align128((size_t)((R + kSlabRows - 1) / kSlabRows) * pc * 4) + align128((size_t)R * d * 4) +
             align128((size_t)pc * d * 4);
  if (lists) b += 2 * align128((size_t)R * K * 4) + align128((size_t)R * 4);
  return b;
}

dgx_status head_fwd(const HeadArgs& a, void* ws, cudaStream_t s) {
  const int pc = piece_cols(a.R, a.V), nt = (a.V + pc - 1) / pc;
  Carve c{(char*)ws};
  float* z = c.take<float>((size_t)a.R * pc);
  float2* part = c.take<float2>((size_t)nt * a.R);
  float* zs = c.take<float>((size_t)a.R * a.K);
  const int* sid = a.idx;
  const float* sq = nullptr;
  if (a.teacher) {
    int* si = c.take<int>((size_t)a.R * a.K);
    float* q = c.take<float>((size_t)a.R * a.K);
    float* live = c.take<float>(a.R);
    head_lists_kernel<<<(a.R + 3) / 4, 128, 0, s>>>(a.idx, a.teacher, a.R, a.V, a.K, a.inv_t, si, q, live);
    sid = si;
    sq = q;
  }
  for (int t = 0; t < nt; ++t) {
    const int c0 = t * pc, n = std::min(pc, a.V - c0);
    const dgx_status st = piece_logits(a, c0, n, z, pc, s);
    if (st != DGX_OK) return st;
    head_stats_kernel<<<(a.R + 7) / 8, 256, 0, s>>>(z, pc, c0, n, a.R, a.inv_t, sid, a.K, zs, part + (size_t)t * a.R);
  }
  head_finish_kernel<<<(a.R + 7) / 8, 256, 0, s>>>(part, nt, a.R, a.V, a.t, a.inv_t, sid, sq, a.K, zs, a.loss, a.lse);
  if (a.mean) head_mean_kernel<<<1, 1024, 0, s>>>(a.loss, a.R, a.mean);
  return cuda_status(cudaGetLastError(), "head forward");
}

dgx_status head_bwd(const HeadArgs& a, void* ws, cudaStream_t s) {
  const int pc = piece_cols(a.R, a.V), slabs = (a.R + kSlabRows - 1) / kSlabRows;
  Carve c{(char*)ws};
  float* z = c.take<float>((size_t)a.R * pc);
  __nv_bfloat16* g = c.take<__nv_bfloat16>((size_t)a.R * pc);
  float* dbp = c.take<float>((size_t)slabs * pc);
  float* dh = c.take<float>((size_t)a.R * a.d);
  float* dw = c.take<float>((size_t)pc * a.d);
  const int* sid = a.idx;
  const float *sq = nullptr, *live = nullptr;
  if (a.teacher) {
    int* si = c.take<int>((size_t)a.R * a.K);
    float* q = c.take<float>((size_t)a.R * a.K);
    float* lv = c.take<float>(a.R);
    head_lists_kernel<<<(a.R + 3) / 4, 128, 0, s>>>(a.idx, a.teacher, a.R, a.V, a.K, a.inv_t, si, q, lv);
    sid = si;
    sq = q;
    live = lv;
  }
  const int grid_out = num_sms() * 8;
  for (int c0 = 0; c0 < a.V; c0 += pc) {
    const int n = std::min(pc, a.V - c0);
    dgx_status st = piece_logits(a, c0, n, z, pc, s);
    if (st != DGX_OK) return st;
    head_grad_kernel<<<dim3(pc / 256, slabs), 256, 0, s>>>(z, pc, c0, n, a.R, a.V, a.inv_t, a.lse, a.dloss, live, sid,
                                                           sq, a.K, g, pc, a.db ? dbp : nullptr);
    if (a.db) head_db_kernel<<<(n + 255) / 256, 256, 0, s>>>(dbp, slabs, n, a.scale, a.accumulate, a.db + c0);
    if (a.dH) {  // dh += G W
      GemmArgs m{};
      m.M = a.R;
      m.N = a.d;
      m.K = n;
      m.lda = pc;
      m.ldb = a.ldw;
      m.ldc = a.d;
      m.C = dh;
      m.beta = c0 ? 1.f : 0.f;
      m.err = a.err;
      st = gemm_run(m, g, (const __nv_bfloat16*)a.W + (size_t)c0 * a.ldw, DGX_BF16, 0, nullptr, 0, s);
      if (st != DGX_OK) return st;
    }
    if (a.dW) {  // dw = G^T H
      GemmArgs m{};
      m.M = n;
      m.N = a.d;
      m.K = a.R;
      m.lda = pc;
      m.ldb = a.ldh;
      m.ldc = a.d;
      m.transA = 1;
      m.C = dw;
      m.err = a.err;
      st = gemm_run(m, g, a.H, DGX_BF16, 0, nullptr, 0, s);
      if (st != DGX_OK) return st;
      void* out = (char*)a.dW + (size_t)c0 * a.lddw * (a.dw_bf16 ? 2 : 4);
      head_out_kernel<<<grid_out, 256, 0, s>>>(dw, n, a.d, a.scale, a.dw_bf16, a.accumulate, out, a.lddw);
    }
  }
  if (a.dH) head_out_kernel<<<grid_out, 256, 0, s>>>(dh, a.R, a.d, a.scale, a.dh_bf16, 0, a.dH, a.lddh);
  return cuda_status(cudaGetLastError(), "head backward");
}

}  // namespace dgx
