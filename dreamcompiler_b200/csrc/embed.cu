// Token embedding with a scale, and its table gradient summed in token order.
//
//   x_i  = s * W[tok_i] (+ P[i mod S])          an id outside [0, V): zero (+ P)
//   dW_t (+)= s * sum over i with tok_i = t of dx_i, in ascending i
//
// Tables, activations and gradients in fp32 or bf16; sums in fp32 in a fixed
// order (no atomics on values), rounded once. All passes are bound by HBM: the
// gather reads the touched rows and writes x, the gradient reads dx once and
// writes dW once. The order of the sums comes from a stable radix sort of the
// token ids, which one cluster of CTAs runs in its own shared memory.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.h"
#include "launch.h"
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

// A lane's 8 elements of a row as loaded (bf16 stays packed until it is used,
// so that twice the rows fit in the same registers).
template <typename T, bool VEC>
struct Row8 {
  static constexpr bool kPacked = VEC && sizeof(T) == 2;
  static constexpr int kRegs = kPacked ? 4 : 8;
  uint32_t r[kRegs];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int k = 0; k < kRegs; ++k) r[k] = 0;
  }
  // p: the lane's slab of the row, `left` columns wide
  __device__ __forceinline__ void load(const T* p, int lane, int left) {
    if constexpr (VEC) {
      if (lane * 8 < left) {
        const uint4* q = reinterpret_cast<const uint4*>(p + lane * 8);
#pragma unroll
        for (int k = 0; k < kRegs / 4; ++k) {
          const uint4 a = __ldg(q + k);
          r[4 * k] = a.x, r[4 * k + 1] = a.y, r[4 * k + 2] = a.z, r[4 * k + 3] = a.w;
        }
      } else {
        zero();
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float v = 0.f;
        if (lane + 32 * k < left) {
          if constexpr (sizeof(T) == 2)
            v = __bfloat162float(p[lane + 32 * k]);
          else
            v = __ldg(p + lane + 32 * k);
        }
        r[k] = __float_as_uint(v);
      }
    }
  }
  __device__ __forceinline__ float get(int k) const {
    if constexpr (kPacked)
      return __uint_as_float(k & 1 ? r[k >> 1] & 0xFFFF0000u : r[k >> 1] << 16);
    else
      return __uint_as_float(r[k]);
  }
};
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
// One warp per (token rows, 256 columns), all its loads in flight before the
// first store: as many rows as 16 registers hold, 4 of a bf16 table (65536 x
// 2048 bf16 70 -> 61 us against 2), 2 of an fp32 one (16384 x 384 9.0 us; 4 rows
// leave too few warps, 11.2).
template <typename TW, bool VEC>
constexpr int fwd_rows() {
  return 16 / Row8<TW, VEC>::kRegs;
}

template <typename TW, typename TX, bool VEC, bool POS>
__global__ void __launch_bounds__(256) embed_fwd_kernel(const int* __restrict__ tok, const TW* __restrict__ W, int ldw,
                                                        const float* __restrict__ P, int S, float scale,
                                                        TX* __restrict__ x, int ldx, int n, int d, int V, int slabs) {
  constexpr int kRows = fwd_rows<TW, VEC>();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const unsigned item = blockIdx.x * 8u + (threadIdx.x >> 5);
  const unsigned group = item / (unsigned)slabs;
  const int c0 = (int)(item - group * slabs) * kSlab, left = d - c0;
  const long long i0 = (long long)group * kRows;
  if (i0 >= n) return;
  Row8<TW, VEC> w[kRows];
  Row8<float, VEC> p[POS ? kRows : 1];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int t = i0 + r < n ? __ldg(tok + i0 + r) : -1;
    if (POS) p[r].load(P + (size_t)((int)min(i0 + r, n - 1ll) % S) * d + c0, lane, left);
    if (t >= 0 && t < V)
      w[r].load(W + (size_t)t * ldw + c0, lane, left);
    else
      w[r].zero();
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    if (i0 + r >= n) break;
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = POS ? fmaf(scale, w[r].get(k), p[r].get(k)) : scale * w[r].get(k);
    store8<VEC>(x + (size_t)(i0 + r) * ldx + c0, lane, left, v);
  }
}

// ---------------------------------------------------------------- token sort
// Stable LSD radix sort of (token, position) by one cluster: every warp owns a
// contiguous range of the input. Per pass each warp ranks its keys among the
// equal digits before them (ballots over the digit's bits give the lanes with
// the same digit), the counts are scanned over warps, over the cluster's CTAs
// (through distributed shared memory) and over digits, and every key goes to
// digit base + warp base + rank. Ids outside [0, V) get the key V and end up
// last. Bound by latency and by the scatter of 8-byte items, about 1.4 cycles
// per item and SM: 65536 ids of 18 bits (two passes) take 26 us on 16 CTAs, 41
// on 8; 16384 ids of 7 bits (one pass) 7 us.
constexpr int kSortThreads = 1024, kSortWarps = 32, kMaxDigitBits = 9, kMaxCluster = 16;
// Keys per lane in registers: 65536 keys in 16 CTAs. Beyond, keys are read twice
// and ranks go through memory (whole gradient on 1000 x 64: 65536 tokens 29.4
// us, 65537 34.3, 131072 51.6).
constexpr int kBatch = 4;

struct SortArgs {
  const int* tok;
  int n, V, passes, bits;  // digit bits per pass
  int2* a;                 // [n] (key, position) ping-pong buffers
  int2* b;
  int* rank;               // [n] scratch when a warp's range exceeds one batch
  int* counters;           // [ncounters] cleared for the summing kernel
  int ncounters;
};

__global__ void __launch_bounds__(kSortThreads) embed_sort_kernel(SortArgs a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  extern __shared__ int hist[];              // [kSortWarps][bins]
  cg::cluster_group cluster = cg::this_cluster();
  const int ncta = (int)cluster.num_blocks(), cta = (int)cluster.block_rank();
  __shared__ int total[1 << kMaxDigitBits];  // this CTA's keys per digit (read by the cluster)
  __shared__ int base[1 << kMaxDigitBits];   // first place of this CTA's keys per digit
  __shared__ int warp_sums[kSortWarps];
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const int bins = 1 << a.bits;
  const int gt = cta * kSortThreads + tid, nthreads = ncta * kSortThreads;

  // this warp's range, a multiple of 32 keys long
  const int warps = ncta * kSortWarps;
  const int per = ((a.n + warps - 1) / warps + 31) & ~31;
  const long long lo = min((long long)a.n, (long long)(cta * kSortWarps + w) * per), hi = min((long long)a.n, lo + per);
  const bool one_batch = per <= 32 * kBatch;
  int* wh = hist + w * bins;
  const unsigned lt = (1u << lane) - 1;
  const int2* src = nullptr;  // null: the token ids themselves
  int2 kv[kBatch];
  int rank[kBatch];
  auto load = [&](long long i0) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const long long i = i0 + 32 * u + lane;
      kv[u] = make_int2(0, (int)i);
      if (i < hi) {
        if (src) {
          kv[u] = src[i];
        } else {
          const int t = a.tok[i];
          kv[u].x = t >= 0 && t < a.V ? t : a.V;
        }
      }
    }
  };
  for (int pass = 0; pass < a.passes; ++pass) {
    const int shift = pass * a.bits;
    int2* dst = pass & 1 ? a.b : a.a;
    for (int i = lane; i < bins; i += 32) wh[i] = 0;
    __syncwarp();
    for (long long i0 = lo; i0 < hi; i0 += 32 * kBatch) {
      load(i0);
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const long long first = i0 + 32 * u;
        if (first >= hi) break;
        const bool in = first + lane < hi;
        const int digit = (kv[u].x >> shift) & (bins - 1);
        unsigned same = __ballot_sync(0xffffffffu, in);
        for (int k = 0; k < a.bits; ++k) {
          const unsigned v = __ballot_sync(0xffffffffu, (digit >> k) & 1);
          same &= (digit >> k) & 1 ? v : ~v;
        }
        if (in) rank[u] = wh[digit] + __popc(same & lt);
        __syncwarp();
        if (in && (same & lt) == 0) wh[digit] += __popc(same);
        __syncwarp();
        if (!one_batch && in) a.rank[first + lane] = rank[u];
      }
    }
    if (pass == 0)  // off the critical path of the loads above
      for (int i = gt; i < a.ncounters; i += nthreads) a.counters[i] = 0;
    __syncthreads();
    // counts of one digit: exclusive over the warps, total for the CTA
    if (tid < bins) {
      int s = 0;
#pragma unroll
      for (int i0 = 0; i0 < kSortWarps; i0 += 8) {
        int c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = hist[(i0 + i) * bins + tid];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          hist[(i0 + i) * bins + tid] = s;
          s += c[i];
        }
      }
      total[tid] = s;
    }
    cluster.sync();
    // first place of this CTA's keys of digit `tid`: keys of smaller digits
    // in the whole cluster, then of the same digit in earlier CTAs
    int all = 0, before = 0;
    if (tid < bins) {
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c)
        if (c < ncta) {
          const int v = cluster.map_shared_rank(total, c)[tid];
          all += v;
          before += c < cta ? v : 0;
        }
    }
    int incl = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) warp_sums[w] = incl;
    __syncthreads();
    int earlier = lane < w ? warp_sums[lane] : 0;
#pragma unroll
    for (int o = 16; o; o >>= 1) earlier += __shfl_xor_sync(0xffffffffu, earlier, o);
    if (tid < bins) base[tid] = earlier + incl - all + before;
    __syncthreads();
    for (long long i0 = lo; i0 < hi; i0 += 32 * kBatch) {
      if (!one_batch) {
        load(i0);
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
          if (i0 + 32 * u + lane < hi) rank[u] = a.rank[i0 + 32 * u + lane];
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (i0 + 32 * u + lane < hi) {
          const int digit = (kv[u].x >> shift) & (bins - 1);
          dst[base[digit] + wh[digit] + rank[u]] = kv[u];
        }
    }
    cluster.sync();  // dst complete; nobody reads `total` any more
    src = dst;
  }
}

// ---------------------------------------------------------------- sums
// The sorted positions are cut evenly, whatever the tokens: a block owns 128
// positions and 256 columns, each of its 8 warps 16 positions, so no token's
// frequency makes a long serial sum. Within its 16 positions a warp adds rows
// in order and writes the tokens that begin and end there. A token that runs
// on into the next warp is joined through shared memory, one that runs on into
// the next block through scratch: the block that finishes the token's last
// outstanding part adds the parts, all in position order. (A block holds at
// most two such tokens, one coming in and one going out.) Bound by HBM where
// dx is large; 16384 rows of 384 fp32 columns (25 MB) take 13 us, most of it
// the latency of four batches of rows and of the joins. Twice the rows in flight
// at half the blocks per SM: 12 us there, but 65536 x 2048 bf16 20 us more.
constexpr int kWarpPos = 16, kBlockPos = 8 * kWarpPos;

struct SumArgs {
  const int2* sorted;  // (token, position)
  int* counters;       // [blocks][slabs] parts finished of the token that runs out of the block it began in
  float* parts;        // [blocks][2][slabs * kSlab]: of the token coming in, of the one beginning and going out
  int n, d, V, slabs, blocks;
  int lddx, lddw, accumulate;
  float scale;
  int zero_blocks, zero_rows;  // blocks that zero rows, and rows for each
  int bulk;                    // rows of dW are whole aligned 16-byte units
};

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

struct SumShared {
  float head[8][kSlab];  // element k of lane l at [l + 32 k] (a block that zeroes rows: the zeros)
  int through[8];                        // the warp's positions are one token that comes in and goes on
  int last_token[2], last_block[2], last_parts[2];  // token whose parts are complete (or -1), its blocks
};

__device__ __forceinline__ void put(float (&row)[kSlab], int lane, const float (&acc)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) row[lane + 32 * k] = acc[k];
}
__device__ __forceinline__ void add(const float (&row)[kSlab], int lane, float (&acc)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) acc[k] += row[lane + 32 * k];
}

// First block b in [lo, hi) whose position `at` (the last one of the order
// where the block is short) holds a token >= t, or hi. The warp probes 32
// blocks at a time: the last of each of 32 equal shares.
__device__ __forceinline__ int search(const SumArgs& a, int lo, int hi, int at, int t, int lane) {
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32, b = lo + (lane + 1) * step - 1;
    const bool ge = b >= hi || a.sorted[min((long long)a.n - 1, (long long)b * kBlockPos + at)].x >= t;
    const unsigned m = __ballot_sync(0xffffffffu, ge);
    if (!m) return hi;
    lo += (__ffs(m) - 1) * step;
    hi = min(hi, lo + step - 1);
  }
  return lo;
}

// Writes the block's part of token t and notes the token if that was the last part.
__device__ __forceinline__ void put_part(const SumArgs& a, SumShared& sh, int blk, int slab, int side, int t, int lane,
                                         const float (&acc)[8]) {
  // the token's blocks: from the one it runs out of (its last position's
  // token) to the last one whose first position has it; the 32 neighbours on
  // either side first (one round trip), then a search
  const bool fwd = blk + 1 + lane < a.blocks && a.sorted[(size_t)(blk + 1 + lane) * kBlockPos].x == t;
  const bool back = !side && lane < blk && a.sorted[(size_t)(blk - lane) * kBlockPos - 1].x == t;
  float* p = a.parts + ((size_t)blk * 2 + side) * a.slabs * kSlab + slab * kSlab;
#pragma unroll
  for (int k = 0; k < 8; ++k) p[lane + 32 * k] = acc[k];
  __threadfence();
  const int nf = __popc(__ballot_sync(0xffffffffu, fwd)), nb = __popc(__ballot_sync(0xffffffffu, back));
  const int b0 = nb < 32 ? blk - nb : search(a, 0, blk - 32, kBlockPos - 1, t, lane);
  const int b1 = nf < 32 ? blk + nf : search(a, blk + 33, a.blocks, 0, t + 1, lane) - 1;
  __syncwarp();
  if (lane == 0 && atomicAdd(&a.counters[(size_t)b0 * a.slabs + slab], 1) == b1 - b0) {
    sh.last_token[side] = t;
    sh.last_block[side] = b0;
    sh.last_parts[side] = b1 - b0 + 1;
  }
}

// ---------------------------------------------------------------- rows without a token
// Blocks of the summing launch zero the rows of dW whose token does not occur,
// up to 256 rows at a time: a lane looks its row up in the sorted tokens (all
// rows at once, so the search's dependent loads cost a few us in all) and sends
// it out as bulk copies of a zeroed piece of shared memory. These blocks come
// first: the sums' latency hides behind their writes (gradient of 16381 tokens
// on 50257 x 1024 fp32 59 us, 62 with them last; 4096 on 32768 x 1024 47 against
// 53; 65536 on 131072 x 2048 bf16 161.5 against 160). A launch of its own beside
// the sort took 52, but would have to read the ids and write dW without having
// waited for the work before the call.
constexpr int kZeroRows = 128, kZeroBytes = 64 << 10;

template <typename TW>
__device__ __forceinline__ void zero_rows(const SumArgs& a, SumShared& sh, TW* dW, unsigned group) {
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (a.bulk) {
    for (int i = threadIdx.x; i < 8 * kSlab; i += 256) (&sh.head[0][0])[i] = 0.f;
    fence_proxy_async_smem();
  }
  __syncthreads();
  const int each = min(a.zero_rows, 256) / 8;  // rows per warp and pass
  for (int r = 0; r < a.zero_rows; r += 256) {
    const unsigned t = group * a.zero_rows + r + w * each + lane;
    bool absent = lane < each && t < (unsigned)a.V;
    if (absent) {
      int lo = 0, hi = a.n;  // first position whose token is t or above
      while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;
        if ((unsigned)a.sorted[mid].x < t)
          lo = mid + 1;
        else
          hi = mid;
      }
      absent = lo == a.n || (unsigned)a.sorted[lo].x != t;
    }
    if (a.bulk) {
      const int bytes = a.d * (int)sizeof(TW);
      char* row = reinterpret_cast<char*>(dW + (size_t)t * a.lddw);
      if (absent)
        for (int j = 0; j < bytes; j += (int)sizeof(sh.head))
          bulk_store(row + j, sh.head, (uint32_t)min((int)sizeof(sh.head), bytes - j));
    } else {
      for (unsigned m = __ballot_sync(0xffffffffu, absent); m; m &= m - 1) {
        TW* row = dW + (size_t)(t - lane + __ffs(m) - 1) * a.lddw;
        for (int j = lane; j < a.d; j += 32) row[j] = TW(0.f);
      }
    }
  }
  if (a.bulk) {
    bulk_commit();
    bulk_wait0();
  }
}

template <typename TG, typename TW, bool VEC>
__global__ void __launch_bounds__(256, 4) embed_sum_kernel(const TG* __restrict__ dx, TW* __restrict__ dW, SumArgs a) {
  __shared__ __align__(16) SumShared sh;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (blockIdx.x < (unsigned)a.zero_blocks) {
    zero_rows(a, sh, dW, blockIdx.x);
    return;
  }
  const unsigned b = blockIdx.x - a.zero_blocks;
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int blk = b / a.slabs, slab = b % a.slabs;
  const int c0 = slab * kSlab, left = a.d - c0;
  if (threadIdx.x < 2) sh.last_token[threadIdx.x] = -1;
  // lanes 0..15: this warp's positions, 16: the one after them, 17: the one before
  const int p0 = blk * kBlockPos + w * kWarpPos;
  const int pl = lane <= kWarpPos ? p0 + lane : p0 - 1;
  int2 kv = make_int2(a.V, 0);
  if (lane <= kWarpPos + 1 && pl >= 0 && pl < a.n) kv = a.sorted[pl];
  if (lane == kWarpPos + 1 && pl < 0) kv.x = -1;
  const int cnt = __popc(__ballot_sync(0xffffffffu, lane < kWarpPos && kv.x < a.V));
  const int before = __shfl_sync(0xffffffffu, kv.x, kWarpPos + 1), after = __shfl_sync(0xffffffffu, kv.x, kWarpPos);
  int cur = __shfl_sync(0xffffffffu, kv.x, 0);
  bool coming = before == cur;  // the current token began before this warp's positions
  bool through = false, tail = false;
  float acc[8] = {};
  if (cnt) {
    // as many rows in flight as 32 registers hold: 8 of bf16, 4 of fp32
    using Row = Row8<TG, VEC>;
    constexpr int kUnroll = 32 / Row::kRegs;
#pragma unroll 1
    for (int j = 0; j < cnt; j += kUnroll) {
      Row v[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int i = __shfl_sync(0xffffffffu, kv.y, j + u);
        if (j + u < cnt) v[u].load(dx + (size_t)i * a.lddx + c0, lane, left);
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int t = __shfl_sync(0xffffffffu, kv.x, j + u);
        if (j + u >= cnt) break;
        if (t != cur) {
          if (coming)
            put(sh.head[w], lane, acc);
          else
            finish_row<TW, VEC>(a, dW, cur, c0, lane, acc);
          coming = false;
          cur = t;
#pragma unroll
          for (int k = 0; k < 8; ++k) acc[k] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] += v[u].get(k);
      }
    }
    const bool going = cnt == kWarpPos && after == cur;
    if (coming) {
      put(sh.head[w], lane, acc);
      through = going;
    } else if (going) {
      tail = true;  // stays in acc: this warp joins the token
    } else {
      finish_row<TW, VEC>(a, dW, cur, c0, lane, acc);
    }
  }
  if (lane == 0) sh.through[w] = through;
  __syncthreads();
  if (w == 0 && cnt && before == __shfl_sync(0xffffffffu, kv.x, 0)) {  // the token that comes into the block
    float in[8] = {};
    add(sh.head[0], lane, in);
    for (int i = 0; i < 7 && sh.through[i]; ++i) add(sh.head[i + 1], lane, in);
    put_part(a, sh, blk, slab, 0, before, lane, in);
  }
  if (tail) {  // a token that begins in this warp and goes on
    int i = w + 1;
    for (; i < 8; ++i) {
      add(sh.head[i], lane, acc);
      if (!sh.through[i]) break;
    }
    if (i < 8)
      finish_row<TW, VEC>(a, dW, cur, c0, lane, acc);
    else
      put_part(a, sh, blk, slab, 1, cur, lane, acc);
  }
  __syncthreads();
#pragma unroll 1
  for (int side = 0; side < 2; ++side) {
    const int t = sh.last_token[side];
    if (t < 0) continue;
    // every part of the token is written: its blocks, split over the warps
    __threadfence();
    const int b0 = sh.last_block[side], parts = sh.last_parts[side], per = (parts + 7) / 8;
    const int i1 = min(parts, (w + 1) * per);
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k] = 0.f;
#pragma unroll 4
    for (int i = w * per; i < i1; ++i) {
      // where the token began it is that block's outgoing part
      const float* p = a.parts + ((size_t)(b0 + i) * 2 + (i == 0)) * a.slabs * kSlab + c0;
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[k] += __ldcg(p + lane + 32 * k);
    }
    __syncthreads();
    put(sh.head[w], lane, acc);
    __syncthreads();
    if (w == 0) {
      for (int i = 1; i < 8; ++i) add(sh.head[i], lane, acc);
      finish_row<TW, VEC>(a, dW, t, c0, lane, acc);
    }
  }
}

// ---------------------------------------------------------------- few tokens
// Up to kFew tokens need no sort: a block owns 32 table rows, reads all ids,
// keeps those of its rows in order, and each warp sums and writes (or zeroes)
// 256 columns of four rows. One launch instead of two: 128 ids on 5000 x 1024
// fp32 7 us instead of 17. The rows of one token are added by one warp, which
// bounds kFew, and kFewBytes lies where equal ids begin to lose what spread ones
// gain (128 ids, this against the sorted form, us: spread and all equal, 20 MB
// of table 7.3 / 17.2 and 18.9 / 17.5; 29 MB 9.6 / 17.7 and 26 / 17.9; 49 MB 14.5
// / 18.2 and 38 / 18.4; 154 MB 40 / 35 and 63 / 35).
constexpr int kFew = 128;
constexpr long long kFewBytes = 32ll << 20;

template <typename TG, typename TW, bool VEC>
__global__ void __launch_bounds__(256, 4) embed_few_kernel(const int* __restrict__ tok, const TG* __restrict__ dx,
                                                        TW* __restrict__ dW, SumArgs a) {
  __shared__ int pos_s[kFew], row_s[kFew], mine_s[8][kFew], count_s[4];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t0 = blockIdx.x * 32, c0 = blockIdx.y * kSlab, left = a.d - c0;
  const unsigned lt = (1u << lane) - 1;
  unsigned hits = 0;
  int row = -1;
  if (w < kFew / 32) {
    const unsigned t = threadIdx.x < a.n ? (unsigned)tok[threadIdx.x] : 0xffffffffu;
    if (t < (unsigned)a.V && t - (unsigned)t0 < 32u) row = (int)(t - t0);
    hits = __ballot_sync(0xffffffffu, row >= 0);
    if (lane == 0) count_s[w] = __popc(hits);
  }
  __syncthreads();
  int total = 0, at = 0;
#pragma unroll
  for (int i = 0; i < kFew / 32; ++i) {
    if (i < w) at += count_s[i];
    total += count_s[i];
  }
  if (row >= 0) {
    pos_s[at + __popc(hits & lt)] = threadIdx.x;
    row_s[at + __popc(hits & lt)] = row;
  }
  __syncthreads();
  for (int r = w; r < 32 && t0 + r < a.V; r += 8) {
    int cnt = 0;
    for (int c = 0; c < total; c += 32) {
      const bool is = c + lane < total && row_s[c + lane] == r;
      const unsigned m = __ballot_sync(0xffffffffu, is);
      if (is) mine_s[w][cnt + __popc(m & lt)] = pos_s[c + lane];
      cnt += __popc(m);
    }
    __syncwarp();
    if (a.accumulate && !cnt) continue;
    using Row = Row8<TG, VEC>;
    constexpr int kUnroll = 32 / Row::kRegs;
    float acc[8] = {};
    for (int j = 0; j < cnt; j += kUnroll) {
      Row v[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (j + u < cnt) v[u].load(dx + (size_t)mine_s[w][j + u] * a.lddx + c0, lane, left);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (j + u < cnt) {
#pragma unroll
          for (int k = 0; k < 8; ++k) acc[k] += v[u].get(k);
        }
    }
    finish_row<TW, VEC>(a, dW, t0 + r, c0, lane, acc);
    __syncwarp();  // mine_s is reused
  }
}

bool type_ok(int t) { return t == DGX_F32 || t == DGX_BF16; }
int type_size(int t) { return t == DGX_F32 ? 4 : 2; }

// 16-byte accesses of 8 elements: every row starts on 16 bytes and holds whole groups of 8.
bool vec_ok(const void* p, int type, int ld, int d) {
  return d % 8 == 0 && ((uintptr_t)p & 15) == 0 && ((long long)ld * type_size(type)) % 16 == 0;
}

size_t align16(size_t b) { return (b + 15) & ~size_t(15); }

// Tokens of one gradient call. The sort and the sums count positions in 32
// bits and step past the last one by up to a cluster's stride (16 x 1024).
constexpr int kMaxTokens = 0x7fffffff - 0xffff;

struct Layout {
  bool few;           // the one-launch form (by the table's fp32 size, whatever its type)
  int blocks, slabs;  // blocks of kBlockPos positions
  size_t a, b, rank, counters, parts, bytes;
};
Layout layout(int n, int d, int V) {
  Layout l{};
  l.few = n <= kFew && (long long)V * d <= kFewBytes / 4;
  l.blocks = (int)(((long long)n + kBlockPos - 1) / kBlockPos);
  l.slabs = (d - 1) / kSlab + 1;
  size_t o = 0;
  if (l.few) {  // no sort, no parts
    l.bytes = 0;
    return l;
  }
  l.a = o, o += align16((size_t)n * 8);
  l.b = o, o += align16((size_t)n * 8);
  l.rank = o, o += align16((size_t)n * 4);
  l.counters = o, o += align16((size_t)l.blocks * l.slabs * 4);
  l.parts = o, o += (size_t)l.blocks * 2 * l.slabs * kSlab * 4;
  l.bytes = o;
  return l;
}

// CTAs of the sorting cluster: 16 where the device can place such a cluster
// (more than the portable 8), looked up once per device.
int wide_cluster() {
  static std::atomic<int> cache[64];
  int dev = 0;
  cudaGetDevice(&dev);
  int c = cache[dev & 63].load(std::memory_order_relaxed);
  if (c) return c;
  const int smem = kSortWarps * 4 << kMaxDigitBits;
  c = 8;
  int placed = 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(kMaxCluster);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kMaxCluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaFuncSetAttribute(embed_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) == cudaSuccess &&
      cudaFuncSetAttribute(embed_sort_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
      cudaOccupancyMaxActiveClusters(&placed, embed_sort_kernel, &cfg) == cudaSuccess && placed > 0)
    c = kMaxCluster;
  cudaGetLastError();
  cache[dev & 63].store(c, std::memory_order_relaxed);
  return c;
}

cudaError_t launch_sort(const SortArgs& a, cudaStream_t s) {
  const int wide = wide_cluster();
  // Up to 2048 tokens one CTA sorts without leaving its SM, up to 8192 a cluster
  // of 8. The whole gradient with 1, 8 and 16 CTAs, tables of 1000 x 64 and
  // 50257 x 64 (us): 1000 tokens 14.7, 16.7, 16.8 and 14.9, 17.5, 18.5; 2048
  // tokens 17.0, 17.0, 17.3 and 18.3, 18.2, 19.3; 4096 tokens 21.8, 17.5, 17.9 and
  // 24.3, 19.1, 19.9; 8192 tokens 32.7, 17.5, 17.8 and 39.1, 20.9, 21.5; 8193
  // tokens 34.4, 19.7, 17.9 and 40.9, 23.3, 21.6.
  const int cluster = a.n <= 2048 ? 1 : a.n <= 8192 ? 8 : wide;
  return launch_dependent(embed_sort_kernel, cluster, kSortThreads, kSortWarps * 4 << a.bits, cluster, s, a);
}

// Rows of dW for one block to look up and zero: three blocks for an SM, which
// leaves room for the sums, but not more rows than 128 or 64 KB. Whole gradient
// (us) by rows per block: 16381 tokens on 50257 x 1024 fp32 61 at 32, 64 at 64, 59
// at 128 and 63 at 256; 200 on 5000 x 1024 17.2 at 16 and 18.6 at 128; 1000 on
// 20000 x 1024 27.9 at 64 and 31.4 at 128; 300 on 1000000 x 16 49 at 128, 36.6 at
// 256 and 31.7 at 1024.
int zero_rows_per_block(int V, size_t row_bytes) {
  const long long most = std::max<long long>(kZeroRows, kZeroBytes / (long long)row_bytes);
  int rows = 16;
  while (2ll * rows <= most && V > 3ll * num_sms() * rows) rows *= 2;
  return rows;
}

template <typename TG, typename TW, bool VEC>
cudaError_t launch_sum(const int* tok, const void* dx, void* dW, const SumArgs& a, int blocks, bool few, cudaStream_t s) {
  if (few) {
    return launch_dependent(embed_few_kernel<TG, TW, VEC>, dim3((a.V + 31) / 32, a.slabs), 256, 0, 1, s, tok,
                            (const TG*)dx, (TW*)dW, a);
  }
  return launch_dependent(embed_sum_kernel<TG, TW, VEC>, blocks, 256, 0, 1, s, (const TG*)dx, (TW*)dW, a);
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
  const bool vec = vec_ok(W, w_type, ldw, d) && vec_ok(x, x_type, ldx, d) && (!P || vec_ok(P, DGX_F32, d, d));
  const int slabs = (d - 1) / kSlab + 1;
  const int rows = vec && w_type == DGX_BF16 ? fwd_rows<__nv_bfloat16, true>() : fwd_rows<float, true>();
  const long long items = ((long long)n + rows - 1) / rows * slabs;
  if (items > 0x7fffffffll) return set_error(DGX_EINVAL, "dgx_embed_fwd: n=%d d=%d too large", n, d);
  cudaError_t e = cudaSuccess;
  auto run = [&](auto* w, auto* o) {
    using TW = std::remove_const_t<std::remove_pointer_t<decltype(w)>>;
    using TX = std::remove_pointer_t<decltype(o)>;
    auto k = vec ? (P ? embed_fwd_kernel<TW, TX, true, true> : embed_fwd_kernel<TW, TX, true, false>)
                 : (P ? embed_fwd_kernel<TW, TX, false, true> : embed_fwd_kernel<TW, TX, false, false>);
    e = launch_dependent(k, (unsigned)((items + 7) / 8), 256, 0, 1, s, tok, w, ldw, P, P ? S : 1, scale, o, ldx, n, d, V,
                         slabs);
  };
  if (w_type == DGX_F32 && x_type == DGX_F32) run((const float*)W, (float*)x);
  else if (w_type == DGX_F32) run((const float*)W, (__nv_bfloat16*)x);
  else if (x_type == DGX_F32) run((const __nv_bfloat16*)W, (float*)x);
  else run((const __nv_bfloat16*)W, (__nv_bfloat16*)x);
  return cuda_status(e, "dgx_embed_fwd");
}

size_t dgx_embed_bwd_workspace_size(int n, int d, int V) {
  if (n <= 0 || n > kMaxTokens || d <= 0 || V <= 0) return 0;
  return layout(n, d, V).bytes;
}

dgx_status dgx_embed_bwd(const int* tok, const void* dx, dgx_dtype dx_type, int lddx, float scale, void* dW,
                         dgx_dtype dw_type, int lddw, int n, int d, int V, int accumulate, void* workspace,
                         size_t workspace_bytes, void* stream) {
  DGX_FAULT_POINT("dgx_embed_bwd");
  if (n < 0 || d <= 0 || V <= 0 || V == 0x7fffffff)
    return set_error(DGX_EINVAL, "dgx_embed_bwd: bad size n=%d d=%d V=%d", n, d, V);
  if (n > kMaxTokens) return set_error(DGX_EINVAL, "dgx_embed_bwd: n=%d above %d", n, kMaxTokens);
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
  const int zero_rows = zero_rows_per_block(V, (size_t)d * type_size(dw_type));
  const long long zero_blocks = ((long long)V + zero_rows - 1) / zero_rows;
  if ((long long)l.blocks * l.slabs + zero_blocks > 0x7fffffffll || l.slabs > 65535)
    return set_error(DGX_EINVAL, "dgx_embed_bwd: n=%d V=%d d=%d too large", n, V, d);
  char* ws = (char*)workspace;
  if (ws && workspace_bytes < l.bytes)
    return set_error(DGX_ENOMEM, "dgx_embed_bwd: workspace %zu bytes < %zu", workspace_bytes, l.bytes);
  if (ws && ((uintptr_t)ws & 15)) return set_error(DGX_EINVAL, "dgx_embed_bwd: workspace must be 16-byte aligned");
  SumArgs a{};
  a.n = n;
  a.d = d;
  a.V = V;
  a.slabs = l.slabs;
  a.blocks = l.blocks;
  a.lddx = lddx;
  a.lddw = lddw;
  a.accumulate = accumulate ? 1 : 0;
  a.scale = scale;
  cudaError_t e = cudaSuccess;
  if (!l.few) {
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
    so.rank = (int*)(ws + l.rank);
    so.counters = (int*)(ws + l.counters);
    so.ncounters = l.blocks * l.slabs;
    e = launch_sort(so, s);
    if (e != cudaSuccess) return cuda_status(e, "dgx_embed_bwd");
    a.sorted = so.passes & 1 ? so.a : so.b;
    a.counters = so.counters;
    a.parts = (float*)(ws + l.parts);
    const size_t ts = type_size(dw_type);
    a.zero_blocks = accumulate ? 0 : (int)zero_blocks;
    a.zero_rows = zero_rows;
    a.bulk = (((uintptr_t)dW | lddw * ts | d * ts) & 15) == 0;
  }
  const int blocks = l.blocks * l.slabs + a.zero_blocks;
  const bool vec = vec_ok(dx, dx_type, lddx, d) && vec_ok(dW, dw_type, lddw, d);
  const bool g32 = dx_type == DGX_F32, w32 = dw_type == DGX_F32;
  if (g32 && w32)
    e = vec ? launch_sum<float, float, true>(tok, dx, dW, a, blocks, l.few, s) : launch_sum<float, float, false>(tok, dx, dW, a, blocks, l.few, s);
  else if (g32)
    e = vec ? launch_sum<float, __nv_bfloat16, true>(tok, dx, dW, a, blocks, l.few, s) : launch_sum<float, __nv_bfloat16, false>(tok, dx, dW, a, blocks, l.few, s);
  else if (w32)
    e = vec ? launch_sum<__nv_bfloat16, float, true>(tok, dx, dW, a, blocks, l.few, s) : launch_sum<__nv_bfloat16, float, false>(tok, dx, dW, a, blocks, l.few, s);
  else
    e = vec ? launch_sum<__nv_bfloat16, __nv_bfloat16, true>(tok, dx, dW, a, blocks, l.few, s)
            : launch_sum<__nv_bfloat16, __nv_bfloat16, false>(tok, dx, dW, a, blocks, l.few, s);
  return cuda_status(e, "dgx_embed_bwd");
}

}  // extern "C"
