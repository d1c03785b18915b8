// Token embedding with a scale, and its table gradient summed in token order.
//
//   x_i  = s * W[tok_i] (+ P[i mod S])          an id outside [0, V): zero (+ P)
//   dW_t (+)= s * sum over i with tok_i = t of dx_i, in ascending i
//
// Tables, activations and gradients in fp32 or bf16; sums in fp32 in a fixed
// order (no atomics on values), rounded once. All passes are bound by HBM: the
// gather reads the touched rows and writes x, the gradient reads dx once and
// writes dW once. The order of the sums comes from a stable radix sort of the
// token ids, which one cluster of 8 CTAs runs in its own shared memory.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>

#include "common.h"
#include "sm100.cuh"

namespace dgx {
namespace {

namespace cg = cooperative_groups;

// ---------------------------------------------------------------- rows of 8 elements
// Eight consecutive elements per lane (VEC: 16-byte accesses), or eight
// elements 32 columns apart (any pitch and alignment). col(k) is the column of
// element k within a 256-column slab.
template <bool VEC>
struct Lane8 {
  static __device__ __forceinline__ int col(int lane, int k) { return VEC ? lane * 8 + k : lane + 32 * k; }
};

__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b) {
  a = __uint_as_float(w << 16);
  b = __uint_as_float(w & 0xFFFF0000u);
}

template <bool VEC>
__device__ __forceinline__ void load8(const float* p, int lane, int left, float (&v)[8]) {
  if constexpr (VEC) {
    if (lane * 8 < left) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(p + lane * 8));
      const float4 b = __ldg(reinterpret_cast<const float4*>(p + lane * 8 + 4));
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = 0.f;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = lane + 32 * k < left ? __ldg(p + lane + 32 * k) : 0.f;
  }
}
template <bool VEC>
__device__ __forceinline__ void load8(const __nv_bfloat16* p, int lane, int left, float (&v)[8]) {
  if constexpr (VEC) {
    uint4 a = make_uint4(0, 0, 0, 0);
    if (lane * 8 < left) a = __ldg(reinterpret_cast<const uint4*>(p + lane * 8));
    unpack2(a.x, v[0], v[1]);
    unpack2(a.y, v[2], v[3]);
    unpack2(a.z, v[4], v[5]);
    unpack2(a.w, v[6], v[7]);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = lane + 32 * k < left ? __bfloat162float(p[lane + 32 * k]) : 0.f;
  }
}
template <bool VEC>
__device__ __forceinline__ void store8(float* p, int lane, int left, const float (&v)[8]) {
  if constexpr (VEC) {
    if (lane * 8 < left) {
      *reinterpret_cast<float4*>(p + lane * 8) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(p + lane * 8 + 4) = make_float4(v[4], v[5], v[6], v[7]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (lane + 32 * k < left) p[lane + 32 * k] = v[k];
  }
}
template <bool VEC>
__device__ __forceinline__ void store8(__nv_bfloat16* p, int lane, int left, const float (&v)[8]) {
  if constexpr (VEC) {
    if (lane * 8 < left)
      *reinterpret_cast<uint4*>(p + lane * 8) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                                           pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (lane + 32 * k < left) p[lane + 32 * k] = __float2bfloat16_rn(v[k]);
  }
}

constexpr int kSlab = 256;  // columns per warp

// ---------------------------------------------------------------- forward
// One warp per (token, 256 columns); kRows tokens per warp, all their loads in
// flight before the first store.
constexpr int kFwdRows = 2;

template <typename TW, typename TX, bool VEC>
__global__ void __launch_bounds__(256) embed_fwd_kernel(const int* __restrict__ tok, const TW* __restrict__ W, int ldw,
                                                        const float* __restrict__ P, int S, float scale,
                                                        TX* __restrict__ x, int ldx, int n, int d, int V, int slabs) {
  const int lane = threadIdx.x & 31;
  const long long item = blockIdx.x * 8ll + (threadIdx.x >> 5);
  const int slab = (int)(item % slabs);
  const long long i0 = item / slabs * kFwdRows;
  const int c0 = slab * kSlab, left = d - c0;
  float v[kFwdRows][8];
#pragma unroll
  for (int r = 0; r < kFwdRows; ++r) {
    const int t = i0 + r < n ? tok[i0 + r] : -1;
    if (t >= 0 && t < V) {
      load8<VEC>(W + (size_t)t * ldw + c0, lane, left, v[r]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[r][k] = 0.f;
    }
  }
#pragma unroll
  for (int r = 0; r < kFwdRows; ++r) {
    if (i0 + r >= n) break;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[r][k] *= scale;
    if (P) {
      float p[8];
      load8<VEC>(P + (size_t)((int)(i0 + r) % S) * d + c0, lane, left, p);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[r][k] += p[k];
    }
    store8<VEC>(x + (size_t)(i0 + r) * ldx + c0, lane, left, v[r]);
  }
}

// ---------------------------------------------------------------- token sort
// Stable LSD radix sort of (token, position) by one cluster: every warp owns a
// contiguous range of the input. Per pass each warp counts its digits
// (match-any gives equal digits of 32 keys one representative), the counts are
// scanned over warps, over the cluster's CTAs (through distributed shared
// memory) and over digits, and each warp scatters its keys in order. Ids
// outside [0, V) get the key V and end up last. Afterwards seg[t] is the range
// of token t in the sorted order (0, 0 where it does not occur).
constexpr int kSortThreads = 1024, kSortWarps = 32, kMaxDigitBits = 10;

struct SortArgs {
  const int* tok;
  int n, V, passes, bits;  // digit bits per pass
  int2* a;                 // [n] (key, position) ping-pong buffers
  int2* b;
  int2* seg;               // [V]
  int* counters;           // [ncounters] cleared for the summing kernel
  int ncounters;
};

__device__ __forceinline__ int sort_key(const int* tok, int i, int V) {
  const int t = tok[i];
  return t >= 0 && t < V ? t : V;
}

__global__ void __launch_bounds__(kSortThreads) embed_sort_kernel(SortArgs a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  cg::cluster_group cluster = cg::this_cluster();
  const int ncta = (int)cluster.num_blocks(), cta = (int)cluster.block_rank();
  extern __shared__ int hist[];  // [kSortWarps][bins]
  __shared__ int total[1 << kMaxDigitBits];  // this CTA's keys per digit (read by the cluster)
  __shared__ int warp_sums[kSortWarps];
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const int bins = 1 << a.bits;
  const int gt = cta * kSortThreads + tid, nthreads = ncta * kSortThreads;
  for (int i = gt; i < a.V; i += nthreads) a.seg[i] = make_int2(0, 0);
  for (int i = gt; i < a.ncounters; i += nthreads) a.counters[i] = 0;

  // this warp's range, a multiple of 32 keys long
  const int warps = ncta * kSortWarps;
  const int per = ((a.n + warps - 1) / warps + 31) & ~31;
  const int lo = min((long long)a.n, (long long)(cta * kSortWarps + w) * per), hi = min((long long)a.n, (long long)lo + per);
  int* wh = hist + w * bins;
  const int2* src = nullptr;  // null: the token ids themselves
  for (int pass = 0; pass < a.passes; ++pass) {
    const int shift = pass * a.bits;
    int2* dst = pass & 1 ? a.b : a.a;
    for (int i = lane; i < bins; i += 32) wh[i] = 0;
    __syncwarp();
    for (int i0 = lo; i0 < hi; i0 += 32) {
      const bool in = i0 + lane < hi;
      const int key = in ? (src ? src[i0 + lane].x : sort_key(a.tok, i0 + lane, a.V)) : 0;
      const int digit = in ? (key >> shift) & (bins - 1) : bins;
      const unsigned same = __match_any_sync(0xffffffffu, digit);
      if (in && (same & ((1u << lane) - 1)) == 0) wh[digit] += __popc(same);
      __syncwarp();
    }
    __syncthreads();
    // counts of one digit: exclusive over the warps, total for the CTA
    if (tid < bins) {
      int s = 0;
#pragma unroll 8
      for (int i = 0; i < kSortWarps; ++i) {
        const int c = hist[i * bins + tid];
        hist[i * bins + tid] = s;
        s += c;
      }
      total[tid] = s;
    }
    cluster.sync();
    // first place of this CTA's keys of digit `tid`: keys of smaller digits
    // in the whole cluster, then of the same digit in earlier CTAs
    int all = 0, before = 0;
    if (tid < bins)
      for (int c = 0; c < ncta; ++c) {
        const int v = cluster.map_shared_rank(total, c)[tid];
        all += v;
        before += c < cta ? v : 0;
      }
    int incl = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) warp_sums[w] = incl;
    __syncthreads();
    if (w == 0) {
      int v = warp_sums[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      warp_sums[lane] = v;
    }
    __syncthreads();
    if (tid < bins) {
      const int base = incl - all + (w ? warp_sums[w - 1] : 0) + before;
#pragma unroll 8
      for (int i = 0; i < kSortWarps; ++i) hist[i * bins + tid] += base;
    }
    __syncthreads();
    for (int i0 = lo; i0 < hi; i0 += 32) {
      const bool in = i0 + lane < hi;
      int2 kv = make_int2(0, i0 + lane);
      if (in) {
        if (src)
          kv = src[i0 + lane];
        else
          kv.x = sort_key(a.tok, i0 + lane, a.V);
      }
      const int digit = in ? (kv.x >> shift) & (bins - 1) : bins;
      const unsigned same = __match_any_sync(0xffffffffu, digit);
      const unsigned below = same & ((1u << lane) - 1);
      const int at = in ? wh[digit] + __popc(below) : 0;
      __syncwarp();
      if (in) {
        dst[at] = kv;
        if (below == 0) wh[digit] += __popc(same);
      }
      __syncwarp();
    }
    cluster.sync();  // dst complete; nobody reads `total` any more
    src = dst;
  }
  for (int i = gt; i < a.n; i += nthreads) {
    const int key = src[i].x;
    if (key >= a.V) continue;
    if (i == 0 || src[i - 1].x != key) a.seg[key].x = i;
    if (i + 1 == a.n || src[i + 1].x != key) a.seg[key].y = i + 1;
  }
}

// ---------------------------------------------------------------- sums
// A warp owns 256 columns of one table row and adds the token's rows of dx in
// order. A token that occurs more than 2C times is split at multiples of C in
// the sorted order: one warp per chunk of C positions sums its part into
// scratch, and the warp that finishes a token's last outstanding part adds the
// parts in order. (A chunk touches at most two such tokens: the one its first
// position belongs to and the one its last position belongs to.)
struct SumArgs {
  const int2* sorted;  // (token, position)
  const int2* seg;
  int* counters;       // [chunks][slabs] parts finished of the split token that starts in the chunk
  float* parts;        // [chunks][2][slabs * kSlab]
  int n, d, V, C, chunks, slabs;
  int lddx, lddw, accumulate;
  float scale;
};

// acc += rows of positions [p0, p1), in order; kUnroll rows in flight.
template <typename TG, bool VEC>
__device__ __forceinline__ void add_rows(const SumArgs& a, const TG* dx, int c0, int p0, int p1, int lane,
                                         float (&acc)[8]) {
  constexpr int kUnroll = 4;
  const int left = a.d - c0;
  for (int q0 = p0; q0 < p1; q0 += 32) {
    const int mine = q0 + lane < p1 ? a.sorted[q0 + lane].y : 0;
    const int cnt = min(32, p1 - q0);
    int j = 0;
    for (; j + kUnroll <= cnt; j += kUnroll) {
      float v[kUnroll][8];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int i = __shfl_sync(0xffffffffu, mine, j + u);
        load8<VEC>(dx + (size_t)i * a.lddx + c0, lane, left, v[u]);
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] += v[u][k];
    }
    for (; j < cnt; ++j) {
      float v[8];
      const int i = __shfl_sync(0xffffffffu, mine, j);
      load8<VEC>(dx + (size_t)i * a.lddx + c0, lane, left, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[k] += v[k];
    }
  }
}

template <typename TW, bool VEC>
__device__ __forceinline__ void finish_row(const SumArgs& a, TW* dW, int t, int c0, int lane, float (&acc)[8]) {
  TW* o = dW + (size_t)t * a.lddw + c0;
#pragma unroll
  for (int k = 0; k < 8; ++k) acc[k] *= a.scale;
  if constexpr (sizeof(TW) == 4) {
    if (a.accumulate) {
      const int left = a.d - c0;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int j = Lane8<VEC>::col(lane, k);
        if (j < left) acc[k] += o[j];
      }
    }
  }
  store8<VEC>(o, lane, a.d - c0, acc);
}

template <typename TG, typename TW, bool VEC>
__global__ void __launch_bounds__(256) embed_sum_kernel(const TG* __restrict__ dx, TW* __restrict__ dW, SumArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  long long item = blockIdx.x * 8ll + (threadIdx.x >> 5);
  const long long nchunk_items = (long long)a.chunks * 2 * a.slabs;
  float acc[8] = {};
  if (item < nchunk_items) {  // part of a split token
    const int slab = (int)(item % a.slabs);
    item /= a.slabs;
    const int side = (int)(item & 1), c = (int)(item >> 1);
    const int first = c * a.C, last = min(a.n, first + a.C) - 1;
    const int t0 = a.sorted[first].x, t = side ? a.sorted[last].x : t0;
    if (t >= a.V || (side && t == t0)) return;
    const int2 sg = a.seg[t];
    if (sg.y - sg.x <= 2 * a.C) return;
    const int c0 = slab * kSlab, width = a.slabs * kSlab;
    add_rows<TG, VEC>(a, dx, c0, max(first, sg.x), min(last + 1, sg.y), lane, acc);
    float* part = a.parts + ((size_t)c * 2 + side) * width + c0;
#pragma unroll
    for (int k = 0; k < 8; ++k) part[Lane8<VEC>::col(lane, k)] = acc[k];
    __threadfence();
    __syncwarp();
    const int cs = sg.x / a.C, ce = (sg.y - 1) / a.C;
    int done = 0;
    if (lane == 0) done = atomicAdd(&a.counters[(size_t)cs * a.slabs + slab], 1);
    done = __shfl_sync(0xffffffffu, done, 0);
    if (done != ce - cs) return;
    __threadfence();
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k] = 0.f;
#pragma unroll 4
    for (int i = cs; i <= ce; ++i) {
      // side 1 where the token starts inside the chunk
      const float* p = a.parts + ((size_t)i * 2 + (i == cs && sg.x > cs * a.C ? 1 : 0)) * width + c0;
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[k] += __ldcg(p + Lane8<VEC>::col(lane, k));
    }
    finish_row<TW, VEC>(a, dW, t, c0, lane, acc);
    return;
  }
  item -= nchunk_items;
  const long long t = item / a.slabs;
  if (t >= a.V) return;
  const int c0 = (int)(item % a.slabs) * kSlab;
  const int2 sg = a.seg[t];
  const int len = sg.y - sg.x;
  if (len > 2 * a.C || (a.accumulate && len == 0)) return;
  add_rows<TG, VEC>(a, dx, c0, sg.x, sg.y, lane, acc);
  finish_row<TW, VEC>(a, dW, (int)t, c0, lane, acc);
}

bool type_ok(int t) { return t == DGX_F32 || t == DGX_BF16; }
int type_size(int t) { return t == DGX_F32 ? 4 : 2; }

// 16-byte accesses of 8 elements: every row starts on 16 bytes and holds whole groups of 8.
bool vec_ok(const void* p, int type, int ld, int d) {
  return d % 8 == 0 && ((uintptr_t)p & 15) == 0 && ((long long)ld * type_size(type)) % 16 == 0;
}

size_t align16(size_t b) { return (b + 15) & ~size_t(15); }

// Positions per chunk of a split token: about half of sqrt(n), so that neither
// one chunk's rows nor one token's parts make a long serial sum.
int chunk_len(int n) {
  int c = 32;
  while (c < 512 && (long long)c * c * 4 < n) c *= 2;
  return c;
}

struct Layout {
  int C, chunks, slabs;
  size_t a, b, seg, counters, parts, bytes;
};
Layout layout(int n, int d, int V) {
  Layout l;
  l.C = chunk_len(n);
  l.chunks = (n + l.C - 1) / l.C;
  l.slabs = (d + kSlab - 1) / kSlab;
  size_t o = 0;
  l.a = o, o += align16((size_t)n * 8);
  l.b = o, o += align16((size_t)n * 8);
  l.seg = o, o += align16((size_t)V * 8);
  l.counters = o, o += align16((size_t)l.chunks * l.slabs * 4);
  l.parts = o, o += (size_t)l.chunks * 2 * l.slabs * kSlab * 4;
  l.bytes = o;
  return l;
}

cudaError_t launch_sort(const SortArgs& a, cudaStream_t s) {
  const int smem = kSortWarps * (1 << a.bits) * 4;
  cudaError_t e =
      cudaFuncSetAttribute(embed_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortWarps * 4 << kMaxDigitBits);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  // up to 4096 tokens one CTA sorts without leaving its SM
  const int ncta = a.n <= 4096 ? 1 : 8;
  cfg.gridDim = dim3(ncta);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ncta;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, embed_sort_kernel, a);
}

template <typename TG, typename TW, bool VEC>
cudaError_t launch_sum(const void* dx, void* dW, const SumArgs& a, cudaStream_t s) {
  const long long items = ((long long)a.chunks * 2 + a.V) * a.slabs;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((items + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, embed_sum_kernel<TG, TW, VEC>, (const TG*)dx, (TW*)dW, a);
}

}  // namespace
}  // namespace dgx

using namespace dgx;

extern "C" {

dgx_status dgx_embed_fwd(const int* tok, const void* W, dgx_dtype w_type, int ldw, const float* P, int S, float scale,
                         void* x, dgx_dtype x_type, int ldx, int n, int d, int V, void* stream) {
  DGX_FAULT_POINT("dgx_embed_fwd");
  if (n < 0 || d <= 0 || V <= 0 || (P && S <= 0))
    return set_error(DGX_EINVAL, "dgx_embed_fwd: bad size n=%d d=%d V=%d S=%d", n, d, V, S);
  if (!type_ok(w_type) || !type_ok(x_type)) return set_error(DGX_EINVAL, "dgx_embed_fwd: types %d %d", w_type, x_type);
  if (ldw < d || ldx < d) return set_error(DGX_EINVAL, "dgx_embed_fwd: row pitch %d or %d < d=%d", ldw, ldx, d);
  if (n == 0) return DGX_OK;
  if (!tok || !W || !x) return set_error(DGX_EINVAL, "dgx_embed_fwd: null pointer");
  cudaStream_t s = (cudaStream_t)stream;
  const int slabs = (d + kSlab - 1) / kSlab;
  const long long blocks = (((long long)n + kFwdRows - 1) / kFwdRows * slabs + 7) / 8;
  if (blocks > 0x7fffffffll) return set_error(DGX_EINVAL, "dgx_embed_fwd: n=%d d=%d too large", n, d);
  const bool vec = vec_ok(W, w_type, ldw, d) && vec_ok(x, x_type, ldx, d) && (!P || vec_ok(P, DGX_F32, d, d));
  auto run = [&](auto* w, auto* o) {
    using TW = std::remove_const_t<std::remove_pointer_t<decltype(w)>>;
    using TX = std::remove_pointer_t<decltype(o)>;
    if (vec)
      embed_fwd_kernel<TW, TX, true><<<(unsigned)blocks, 256, 0, s>>>(tok, w, ldw, P, P ? S : 1, scale, o, ldx, n, d, V,
                                                                      slabs);
    else
      embed_fwd_kernel<TW, TX, false><<<(unsigned)blocks, 256, 0, s>>>(tok, w, ldw, P, P ? S : 1, scale, o, ldx, n, d,
                                                                       V, slabs);
  };
  if (w_type == DGX_F32 && x_type == DGX_F32) run((const float*)W, (float*)x);
  else if (w_type == DGX_F32) run((const float*)W, (__nv_bfloat16*)x);
  else if (x_type == DGX_F32) run((const __nv_bfloat16*)W, (float*)x);
  else run((const __nv_bfloat16*)W, (__nv_bfloat16*)x);
  return cuda_status(cudaGetLastError(), "dgx_embed_fwd");
}

size_t dgx_embed_bwd_workspace_size(int n, int d, int V) {
  if (n <= 0 || d <= 0 || V <= 0) return 0;
  return layout(n, d, V).bytes;
}

dgx_status dgx_embed_bwd(const int* tok, const void* dx, dgx_dtype dx_type, int lddx, float scale, void* dW,
                         dgx_dtype dw_type, int lddw, int n, int d, int V, int accumulate, void* workspace,
                         size_t workspace_bytes, void* stream) {
  DGX_FAULT_POINT("dgx_embed_bwd");
  if (n < 0 || d <= 0 || V <= 0 || V == 0x7fffffff)
    return set_error(DGX_EINVAL, "dgx_embed_bwd: bad size n=%d d=%d V=%d", n, d, V);
  if (!type_ok(dx_type) || !type_ok(dw_type))
    return set_error(DGX_EINVAL, "dgx_embed_bwd: types %d %d", dx_type, dw_type);
  if (lddx < d || lddw < d) return set_error(DGX_EINVAL, "dgx_embed_bwd: row pitch %d or %d < d=%d", lddx, lddw, d);
  if (accumulate && dw_type != DGX_F32) return set_error(DGX_EUNSUPPORTED, "dgx_embed_bwd: accumulate needs an fp32 dW");
  if (!dW || (n > 0 && (!tok || !dx))) return set_error(DGX_EINVAL, "dgx_embed_bwd: null pointer");
  cudaStream_t s = (cudaStream_t)stream;
  if (n == 0) {
    if (accumulate) return DGX_OK;
    const size_t es = type_size(dw_type);
    return cuda_status(cudaMemset2DAsync(dW, lddw * es, 0, d * es, V, s), "dgx_embed_bwd");
  }
  const Layout l = layout(n, d, V);
  if ((((long long)l.chunks * 2 + V) * l.slabs + 7) / 8 > 0x7fffffffll)
    return set_error(DGX_EINVAL, "dgx_embed_bwd: V=%d d=%d too large", V, d);
  char* ws = (char*)workspace;
  if (ws && workspace_bytes < l.bytes)
    return set_error(DGX_ENOMEM, "dgx_embed_bwd: workspace %zu bytes < %zu", workspace_bytes, l.bytes);
  if (ws && ((uintptr_t)ws & 15)) return set_error(DGX_EINVAL, "dgx_embed_bwd: workspace must be 16-byte aligned");
  if (!ws) ws = (char*)library_scratch(l.bytes, s);
  if (!ws) return set_error(DGX_ENOMEM, "dgx_embed_bwd: cannot allocate %zu bytes of scratch", l.bytes);
  SortArgs so{};
  so.tok = tok;
  so.n = n;
  so.V = V;
  int kb = 1;
  while (kb < 31 && (V >> kb)) ++kb;  // keys 0 .. V
  so.passes = (kb + kMaxDigitBits - 1) / kMaxDigitBits;
  so.bits = (kb + so.passes - 1) / so.passes;
  so.a = (int2*)(ws + l.a);
  so.b = (int2*)(ws + l.b);
  so.seg = (int2*)(ws + l.seg);
  so.counters = (int*)(ws + l.counters);
  so.ncounters = l.chunks * l.slabs;
  cudaError_t e = launch_sort(so, s);
  if (e != cudaSuccess) return cuda_status(e, "dgx_embed_bwd");
  SumArgs a{};
  a.sorted = so.passes & 1 ? so.a : so.b;
  a.seg = so.seg;
  a.counters = so.counters;
  a.parts = (float*)(ws + l.parts);
  a.n = n;
  a.d = d;
  a.V = V;
  a.C = l.C;
  a.chunks = l.chunks;
  a.slabs = l.slabs;
  a.lddx = lddx;
  a.lddw = lddw;
  a.accumulate = accumulate ? 1 : 0;
  a.scale = scale;
  const bool vec = vec_ok(dx, dx_type, lddx, d) && vec_ok(dW, dw_type, lddw, d);
  const bool g32 = dx_type == DGX_F32, w32 = dw_type == DGX_F32;
  if (g32 && w32)
    e = vec ? launch_sum<float, float, true>(dx, dW, a, s) : launch_sum<float, float, false>(dx, dW, a, s);
  else if (g32)
    e = vec ? launch_sum<float, __nv_bfloat16, true>(dx, dW, a, s) : launch_sum<float, __nv_bfloat16, false>(dx, dW, a, s);
  else if (w32)
    e = vec ? launch_sum<__nv_bfloat16, float, true>(dx, dW, a, s) : launch_sum<__nv_bfloat16, float, false>(dx, dW, a, s);
  else
    e = vec ? launch_sum<__nv_bfloat16, __nv_bfloat16, true>(dx, dW, a, s)
            : launch_sum<__nv_bfloat16, __nv_bfloat16, false>(dx, dW, a, s);
  return cuda_status(e, "dgx_embed_bwd");
}

}  // extern "C"
