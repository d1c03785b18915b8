// Vocabulary head: linear layer + softmax + loss with a sparse target, forward
// and backward, in pieces of the vocabulary. No logit is written to memory: the
// forward leaves (max, sum) of 64 or 128 columns of a row in scratch, the
// backward the bf16 gradient G of a piece; what is kept between the two is the
// row log-sum-exp.
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
#include "launch.h"
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

// Every kernel here is launched as its predecessor's programmatic dependent.
// The ones that another kernel of the same call follows let it start early;
// the last one of a call does not, so that what the caller issues next starts
// with the whole call done.
__device__ __forceinline__ void dependents_may_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void wait_for_predecessor() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---------------------------------------------------------------- target lists
// One warp per row: q = softmax(teacher / T) over the entries whose id lies in
// [0, V), and the entries in ascending order of (id, position), absent ones
// last (id kNoId, q 0). A teacher logit of -inf has q = 0; a row whose entries
// are all absent or -inf has live = 0 (a NaN entry is neither: its row has a
// target, and NaN results). The rank of an entry is the number of
// entries before it, counted four ids per shared-memory load. start[row][s] is
// the first entry whose id is at least kHeadSlot (slot0 + s). KI: entries per lane.
// Latency of two dependent loads and the ranking: 5 us at 333 rows of 17.
template <int KI>
__global__ void __launch_bounds__(128) head_lists_kernel(const int* __restrict__ idx, const float* __restrict__ teacher,
                                                         int R, int V, int K, float inv_t, int* __restrict__ sid,
                                                         float* __restrict__ sq, float* __restrict__ live,
                                                         uint16_t* __restrict__ start, int slots, int slot0) {
  __shared__ __align__(16) int ids_s[4][KI * 32], sorted_s[4][KI * 32];
  dependents_may_start();
  wait_for_predecessor();
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.x * 4 + w;
  if (row >= R) return;
  int* ids = ids_s[w];
  int* sorted = sorted_s[w];
  int id[KI];
  float q[KI];
  float mx = -INFINITY;
  bool some = false;
#pragma unroll
  for (int i = 0; i < KI; ++i) {
    const int k = lane + 32 * i;
    id[i] = kNoId;
    q[i] = -INFINITY;
    if (k < K) {
      const int v = idx[(size_t)row * K + k];
      const float l = teacher[(size_t)row * K + k];
      if (v >= 0 && v < V) {
        id[i] = v;
        q[i] = l;
        mx = fmaxf(mx, l);  // drops a NaN
        some |= l != -INFINITY;
      }
    }
    ids[k] = id[i];
  }
  mx = warp_max(mx);
  const bool any = __any_sync(0xffffffffu, some);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < KI; ++i) {
    q[i] = any && id[i] != kNoId ? expf((q[i] - mx) * inv_t) : 0.f;
    s += q[i];
  }
  s = warp_sum(s);
  const float inv_s = any ? 1.f / s : 0.f;
  __syncwarp();
  int rank[KI] = {};
#pragma unroll 4
  for (int j = 0; j < KI * 32; j += 4) {
    const int4 o = *reinterpret_cast<const int4*>(ids + j);
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      const int k = lane + 32 * i;
      rank[i] += (o.x < id[i] || (o.x == id[i] && j < k)) + (o.y < id[i] || (o.y == id[i] && j + 1 < k)) +
                 (o.z < id[i] || (o.z == id[i] && j + 2 < k)) + (o.w < id[i] || (o.w == id[i] && j + 3 < k));
    }
  }
#pragma unroll
  for (int i = 0; i < KI; ++i) {
    sorted[rank[i]] = id[i];
    if (rank[i] < K) {
      sid[(size_t)row * K + rank[i]] = id[i];
      sq[(size_t)row * K + rank[i]] = q[i] * inv_s;
    }
  }
  if (lane == 0) live[row] = any ? 1.f : 0.f;
  __syncwarp();
  for (int t = lane; t < slots; t += 32) {
    int lo = 0;  // entries below kHeadSlot t: a binary descent over KI * 32 entries
#pragma unroll
    for (int step = KI * 32; step; step >>= 1)
      if (lo + step <= KI * 32 && sorted[lo + step - 1] < (slot0 + t) * kHeadSlot) lo += step;
    start[(size_t)row * slots + t] = (uint16_t)min(lo, K);
  }
}

// ---------------------------------------------------------------- forward
// The statistics of a block's 32 rows over `slots` slots part[slot][R] (max of
// the raw logits and sum of exp((z - max) / T) over the slot's columns; without
// a hard target's column, which nll_row adds), one row per lane: the NW warps
// walk the slots, eight loads in flight, and their results are joined in warp
// order. Valid in warp 0.
template <int NW>
__device__ __forceinline__ void join_slots(const float2* part, int slots, int R, float inv_t,
                                           float2 (&ms)[NW][32], float& m, float& s, float& base) {
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.x * 32 + lane;
  m = -INFINITY;
  s = 0.f;
  if (row < R)
    for (int i = w; i < slots; i += 8 * NW) {
      float2 p[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        p[u] = i + u * NW < slots ? part[(size_t)(i + u * NW) * R + row] : make_float2(-INFINITY, 0.f);
      float mn = m;
#pragma unroll
      for (int u = 0; u < 8; ++u) mn = fmaxf(mn, p[u].x);
      const float b = mn == -INFINITY ? 0.f : mn;
      s *= expf((m - b) * inv_t);
#pragma unroll
      for (int u = 0; u < 8; ++u) s += p[u].y * expf((p[u].x - b) * inv_t);
      m = mn;
    }
  ms[w][lane] = make_float2(m, s);
  __syncthreads();
  if (w) return;
#pragma unroll
  for (int i = 1; i < NW; ++i) m = fmaxf(m, ms[i][lane].x);
  base = m == -INFINITY ? 0.f : m;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < NW; ++i) s += ms[i][lane].y * expf((ms[i][lane].x - base) * inv_t);
}

// One slot out[R] of the statistics in place of `slots` of them: between the
// pieces of a forward that has several. out may be the first of them.
__global__ void __launch_bounds__(1024) head_join_kernel(const float2* part, int slots, int R, float inv_t, float2* out) {
  __shared__ float2 ms[32][32];
  wait_for_predecessor();
  float m, s, base;
  join_slots<32>(part, slots, R, inv_t, ms, m, s, base);
  const int row = blockIdx.x * 32 + threadIdx.x;
  if (threadIdx.x < 32 && row < R) out[row] = make_float2(m, s);
}

// lse and loss of 32 rows per block from the statistics. Hard target: sq ==
// null. Latency: 4 us past the logits kernel at 512 rows of 256 slots, 8 us at
// 333 rows of 786.
template <int NW>
__global__ void __launch_bounds__(NW * 32) head_finish_kernel(
    const float2* __restrict__ part, int slots, int R, int V, float t, float inv_t, const int* __restrict__ sid,
    const float* __restrict__ sq, int K, const float* __restrict__ zs, float* __restrict__ loss,
    float* __restrict__ lse) {
  __shared__ float2 ms[NW][32];
  __shared__ float base_s[32], logs_s[32];
  wait_for_predecessor();
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row0 = blockIdx.x * 32, row = row0 + lane;
  float m, s, base;
  join_slots<NW>(part, slots, R, inv_t, ms, m, s, base);
  if (w == 0) {
    if (!sq) {
      if (row < R) {
        const int id = sid[row];
        const bool has = id >= 0 && id < V;
        nll_row(m, s, has ? zs[row] : 0.f, has, inv_t, loss[row], lse[row]);
      }
    } else {
      // z - lse = (raw - max)/T - log s: subtracting the maximum first keeps
      // the loss accurate when the logits are large
      const float log_s = logf(s);
      if (row < R) lse[row] = base * inv_t + log_s;
      base_s[lane] = base;
      logs_s[lane] = log_s;
    }
  }
  if (!sq) return;
  __syncthreads();
  for (int r = w; r < 32 && row0 + r < R; r += NW) {
    const size_t at = (size_t)(row0 + r) * K;
    float l = 0.f;
    for (int k = lane; k < K; k += 32) {
      const float q = sq[at + k];
      if (sid[at + k] == kNoId || q == 0.f) continue;
      l += q * (logf(q) - ((zs[at + k] - base_s[r]) * inv_t - logs_s[r]));
    }
    l = warp_sum(l);
    if (lane == 0) loss[row0 + r] = t * t * l;
  }
}

// *mean = sum(loss) / R in a fixed order (one block).
__global__ void head_mean_kernel(const float* __restrict__ loss, int R, float* __restrict__ mean) {
  __shared__ float red[32];
  wait_for_predecessor();
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

// What is left after the gradient products of a piece, in one launch: the first
// blocks sum db, the others the slices of a product.
struct SliceSum {  // out[r][j] (+)= scale * sum over slices of acc[slice][r][j], in order
  const float* acc;
  void* out;
  int slices, rows, d, lda, bf16_out, add, ldo;  // pitches are multiples of four elements
};
struct BiasSum {  // db[j] (+)= scale * sum over slabs of dbp[slab][j]
  const float* dbp;
  float* db;
  int slabs, n, add, blocks;
};

// A block owns 32 columns; its 8 warps take the slabs in turn and are joined in
// warp order.
__device__ __forceinline__ void bias_sum(const BiasSum& b, float scale, float (*red)[32]) {
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int j = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (j < b.n) {
#pragma unroll 8
    for (int i = w; i < b.slabs; i += 8) s += b.dbp[(size_t)i * b.n + j];
  }
  red[w][lane] = s;
  __syncthreads();
  if (w == 0 && j < b.n) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += red[i][lane];
    b.db[j] = (b.add ? b.db[j] : 0.f) + scale * s;
  }
}

// Rounded once to bf16 where asked; four columns per thread.
__global__ void __launch_bounds__(256) head_sums_kernel(SliceSum a, BiasSum b, float scale) {
  __shared__ float red[8][32];
  wait_for_predecessor();
  if (blockIdx.x < b.blocks) {
    bias_sum(b, scale, red);
    return;
  }
  const int dq = (a.d + 3) >> 2;
  const long long total = (long long)a.rows * dq;
  const size_t slice = (size_t)a.rows * a.lda;
  for (long long e = (blockIdx.x - b.blocks) * (long long)blockDim.x + threadIdx.x; e < total;
       e += (long long)(gridDim.x - b.blocks) * blockDim.x) {
    const long long r = e / dq;
    const int j = (int)(e - r * dq) * 4;
    const float* p = a.acc + (size_t)r * a.lda + j;
    float4 v = *reinterpret_cast<const float4*>(p);
#pragma unroll 4
    for (int i = 1; i < a.slices; ++i) {
      const float4 u = *reinterpret_cast<const float4*>(p + i * slice);
      v.x += u.x;
      v.y += u.y;
      v.z += u.z;
      v.w += u.w;
    }
    const float f[4] = {scale * v.x, scale * v.y, scale * v.z, scale * v.w};
    if (a.bf16_out) {
      __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(a.out) + r * a.ldo + j;
      if (j + 4 <= a.d)
        *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
      else
        for (int i = 0; j + i < a.d; ++i) o[i] = __float2bfloat16_rn(f[i]);
    } else {
      float* o = reinterpret_cast<float*>(a.out) + r * a.ldo + j;
      for (int i = 0; i < 4 && j + i < a.d; ++i) o[i] = a.add ? o[i] + f[i] : f[i];
    }
  }
}

// Columns of one piece of the vocabulary in the backward: G (bf16, R rows) of
// about 256 MB, so that its buffer stays far below the logits while the two
// gradient products get a long enough piece to fill the GPU.
constexpr size_t kPieceBytes = 256u << 20;

size_t align128(size_t b) { return (b + 127) & ~size_t(127); }

int piece_cols(int R, int V) {
  const long long c = (long long)(kPieceBytes / 2 / (size_t)R) / 256 * 256;
  return (int)std::min<long long>(std::max<long long>(c, 256), ((long long)V + 255) / 256 * 256);
}

// Columns of one piece of the forward: statistics of at most 256 MB (64-column
// slots), so that they stay a fixed amount of scratch whatever R V is. One piece
// up to 2^31 logits; a further one costs a join and, for a soft target, a
// launch of the lists.
int stat_piece_cols(int R, int V) {
  const long long c = (1ll << 31) / R / 256 * 256;  // 256 at the largest R
  return (int)std::min<long long>(c, ((long long)V + 255) / 256 * 256);
}

// The start table of the target lists covers this many columns of the vocabulary
// at a time (64 MB at most): whole pieces of the backward.
int list_cols(int R, int V, bool backward) {
  const int c = stat_piece_cols(R, V);
  return backward ? c / piece_cols(R, V) * piece_cols(R, V) : c;
}

int num_slots(int V) { return (int)(((long long)V + 255) / 256 * (256 / kHeadSlot)); }

struct Carve {
  char* p;
  template <typename T>
  T* take(size_t n) {
    T* r = reinterpret_cast<T*>(p);
    p += align128(n * sizeof(T));
    return r;
  }
};

size_t list_bytes(int R, int K, int cols) {
  return 2 * align128((size_t)R * K * 4) + align128((size_t)R * 4) + align128((size_t)R * num_slots(cols) * 2);
}

// Sorted target lists of the soft target (the hard one is its own list), with
// the start table of the columns [c0, c0 + cols).
struct Lists {
  int *sid, cols;
  float *q, *live;
  uint16_t* start;
};
Lists carve_lists(const HeadArgs& a, Carve& c, int cols) {
  Lists l{};
  l.cols = cols;
  if (!a.teacher) return l;
  l.sid = c.take<int>((size_t)a.R * a.K);
  l.q = c.take<float>((size_t)a.R * a.K);
  l.live = c.take<float>(a.R);
  l.start = c.take<uint16_t>((size_t)a.R * num_slots(cols));
  return l;
}
cudaError_t target_lists(const HeadArgs& a, const Lists& l, int c0, HeadTcArgs& t, cudaStream_t s) {
  t.sid = a.idx;
  t.K = a.K;
  if (!a.teacher) return cudaSuccess;
  t.slots = num_slots(l.cols);
  t.slot0 = c0 / kHeadSlot;
  t.sid = l.sid;
  t.sq = l.q;
  t.live = l.live;
  t.start = l.start;
  auto kern = a.K <= 32    ? head_lists_kernel<1>
              : a.K <= 64  ? head_lists_kernel<2>
              : a.K <= 128 ? head_lists_kernel<4>
                           : head_lists_kernel<8>;
  return launch_dependent(kern, (a.R + 3) / 4, 128, 0, 1, s, a.idx, a.teacher, a.R, a.V, a.K, a.inv_t, l.sid, l.q, l.live,
                          l.start, t.slots, t.slot0);
}

HeadTcArgs tc_args(const HeadArgs& a) {
  HeadTcArgs t{};
  t.R = a.R;
  t.V = a.V;
  t.d = a.d;
  t.inv_t = a.inv_t;
  t.k = a.inv_t * 1.4426950408889634f;
  t.bias = a.bias;
  t.err = a.err;
  return t;
}

}  // namespace

size_t head_fwd_scratch_bytes(int R, int V, int d, int K, bool lists) {
  const int pc = stat_piece_cols(R, V), cols = head_stat_cols(d, true);  // a bias never widens the slots
  const int slots = std::max((std::min(pc, V) + cols - 1) / cols + (pc < V), lists ? 0 : head_small_slots(R, V, d));
  return align128((size_t)slots * R * 8) + align128((size_t)R * K * 4) +
         (lists ? list_bytes(R, K, list_cols(R, V, false)) : 0);
}

// How the backward of one problem is cut: columns per piece, the slices of the
// gradient sums and the scratch they need. Sized for dH and dW both wanted.
struct Plan {
  int pc, pieces, slabs, dp;
  GradSplits sp;
  bool dh_scratch;  // dH goes through fp32 scratch (several pieces, or slices)
};
static Plan make_plan(int R, int V, int d) {
  Plan p;
  p.pc = piece_cols(R, V);
  p.pieces = (V + p.pc - 1) / p.pc;
  p.slabs = (R + kSlabRows - 1) / kSlabRows;
  p.dp = (d + 3) / 4 * 4;
  p.sp = head_grad_splits(R, std::min(p.pc, V), d, true, true);
  p.dh_scratch = p.pieces > 1 || p.sp.dh > 1;
  return p;
}

size_t head_bwd_scratch_bytes(int R, int V, int d, int K, bool lists) {
  const Plan p = make_plan(R, V, d);
  return align128((size_t)R * p.pc * 2) + align128((size_t)p.slabs * p.pc * 4) +
         align128(p.dh_scratch ? (size_t)p.sp.dh * R * p.dp * 4 : 0) +
         align128(p.sp.dw > 1 ? (size_t)p.sp.dw * std::min(p.pc, V) * p.dp * 4 : 0) +
         (lists ? list_bytes(R, K, list_cols(R, V, true)) : 0);
}

dgx_status head_fwd(const HeadArgs& a, void* ws, cudaStream_t s) {
  Carve c{(char*)ws};
  HeadTcArgs t = tc_args(a);
  const int small = a.teacher ? 0 : head_small_slots(a.R, a.V, a.d);
  const int cols = head_stat_cols(a.d, a.bias != nullptr);
  const int pc = small ? a.V : stat_piece_cols(a.R, a.V);
  const int first = pc < a.V;  // several pieces: slot 0 holds the joined earlier ones
  const int max_slots = small ? small : (std::min(pc, a.V) + cols - 1) / cols + first;
  float2* part = c.take<float2>((size_t)max_slots * a.R);
  t.zs = c.take<float>((size_t)a.R * a.K);
  const Lists lists = carve_lists(a, c, list_cols(a.R, a.V, false));
  const bool whole = !a.teacher && !small && a.V <= 256;  // one tile holds a row: finished in the tile's epilogue
  if (whole) {
    t.loss = a.loss;
    t.lse_out = a.lse;
  }
  cudaError_t e = cudaSuccess;
  for (int c0 = 0; c0 < a.V && e == cudaSuccess; c0 += pc) {
    t.c0 = c0;
    t.n = std::min(pc, a.V - c0);
    t.part = part + (size_t)first * a.R;
    e = target_lists(a, lists, c0, t, s);
    if (e == cudaSuccess)
      e = small ? head_small(t, a.H, a.ldh, a.W, a.ldw, small, a.loss, a.lse, s)
                : head_logits_tc(t, a.H, a.ldh, a.W, a.ldw, false, nullptr, 0, s);
    if (e != cudaSuccess || small == 1 || whole) break;
    const bool earlier = c0 > 0;
    const float2* from = earlier ? part : t.part;
    const int slots = (small ? small : (t.n + cols - 1) / cols) + earlier;
    const unsigned blocks = (a.R + 31) / 32;
    if (t.n < a.V - c0) {
      e = launch_dependent(head_join_kernel, blocks, 1024, 0, 1, s, from, slots, a.R, a.inv_t, part);
      continue;
    }
    // few slots: few warps, so that many rows do not pay for idle ones
    const bool wide = slots > 32;
    e = launch_dependent(wide ? head_finish_kernel<32> : head_finish_kernel<4>, blocks, wide ? 1024 : 128, 0, 1, s, from,
                         slots, a.R, a.V, a.t, a.inv_t, t.sid, t.sq, a.K, t.zs, a.loss, a.lse);
  }
  if (e == cudaSuccess && a.mean) e = launch_dependent(head_mean_kernel, 1, 1024, 0, 1, s, a.loss, a.R, a.mean);
  return cuda_status(e, "head forward");
}

static cudaError_t launch_sums(const SliceSum& a, const BiasSum& b, float scale, cudaStream_t s) {
  const long long quads = a.acc ? (long long)a.rows * ((a.d + 3) / 4) : 0;
  const unsigned blocks = (unsigned)std::min<long long>((quads + 255) / 256, num_sms() * 8ll) + b.blocks;
  return blocks ? launch_dependent(head_sums_kernel, blocks, 256, 0, 1, s, a, b, scale) : cudaSuccess;
}

dgx_status head_bwd(const HeadArgs& a, void* ws, cudaStream_t s) {
  const Plan p = make_plan(a.R, a.V, a.d);
  Carve c{(char*)ws};
  HeadTcArgs t = tc_args(a);
  __nv_bfloat16* g = c.take<__nv_bfloat16>((size_t)a.R * p.pc);
  float* dbp = c.take<float>((size_t)p.slabs * p.pc);
  float* dh = p.dh_scratch ? c.take<float>((size_t)p.sp.dh * a.R * p.dp) : nullptr;
  float* dw = p.sp.dw > 1 ? c.take<float>((size_t)p.sp.dw * std::min(p.pc, a.V) * p.dp) : nullptr;
  const int lc = list_cols(a.R, a.V, true);
  const Lists lists = carve_lists(a, c, lc);
  cudaError_t e = cudaSuccess;
  t.dbp = a.db ? dbp : nullptr;
  t.dloss = a.dloss;
  t.lse = a.lse;
  for (int c0 = 0; c0 < a.V; c0 += p.pc) {
    const int n = std::min(p.pc, a.V - c0);
    t.c0 = c0;
    t.n = n;
    if (c0 % lc == 0) e = target_lists(a, lists, c0, t, s);
    if (e == cudaSuccess) e = head_logits_tc(t, a.H, a.ldh, a.W, a.ldw, true, g, p.pc, s);
    if (e != cudaSuccess) return cuda_status(e, "head backward");
    HeadGradTc m{};
    m.G = g;
    m.ldg = p.pc;
    m.W = (const __nv_bfloat16*)a.W + (size_t)c0 * a.ldw;
    m.ldw = a.ldw;
    m.H = a.H;
    m.ldh = a.ldh;
    m.R = a.R;
    m.n = n;
    m.d = a.d;
    m.err = a.err;
    void* dw_out = a.dW ? (char*)a.dW + (size_t)c0 * a.lddw * (a.dw_bf16 ? 2 : 4) : nullptr;
    if (a.dH) m.out[0] = dh ? GradOut{dh, 0, c0 > 0, p.dp, p.sp.dh, 1.f} : GradOut{a.dH, a.dh_bf16, a.add_h, a.lddh, 1, a.scale};
    if (a.dW) m.out[1] = dw ? GradOut{dw, 0, 0, p.dp, p.sp.dw, 1.f} : GradOut{dw_out, a.dw_bf16, a.add_w, a.lddw, 1, a.scale};
    e = head_grads_tc(m, s);
    if (e == cudaSuccess) {
      SliceSum w{};
      BiasSum b{};
      if (a.dW && dw) w = SliceSum{dw, dw_out, p.sp.dw, n, a.d, p.dp, a.dw_bf16, a.add_w, a.lddw};
      if (a.db) b = BiasSum{dbp, a.db + c0, p.slabs, n, a.add_w, (n + 31) / 32};
      e = launch_sums(w, b, a.scale, s);
    }
    if (e != cudaSuccess) return cuda_status(e, "head backward");
  }
  if (a.dH && dh)
    e = launch_sums(SliceSum{dh, a.dH, p.sp.dh, a.R, a.d, p.dp, a.dh_bf16, a.add_h, a.lddh}, BiasSum{}, a.scale, s);
  return cuda_status(e, "head backward");
}

}  // namespace dgx
