// Forward of the vocabulary head for a few rows (a decoded token, a short
// prompt): the logits of R <= 16 rows against every row of W, with a hard
// target. What counts is the stream of W (V x d bf16, read once); the products
// are a thin tensor-core contraction on warp-level MMAs, 16 rows of W by 8 or
// 16 rows of H, whose operand fragments the lanes load straight from
// global memory: a lane's 16 bytes of a W row are four consecutive k pairs, and
// H is laid out in shared memory in the same order (the order of a sum's terms
// is free), so nothing is staged or transposed.
//
// Bound by the stream of W where W is large: 131072 x 2048 (537 MB) takes 96 us
// for one row, 5.6 TB/s. 32768 x 1024 (67 MB) takes 18.4 us, 3.6 TB/s: 256 blocks
// of one tile per warp, unevenly on 148 SMs, then the kernel that joins their
// statistics. The tcgen05 kernel, whose 256-row tiles keep a few stages of loads
// in flight on 74 SM pairs, takes 149 and 28 us.
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>

#include "head.h"
#include "launch.h"
#include "sm100.cuh"

namespace dgx {
namespace {

constexpr int kWarps = 8, kTileRows = 16;  // W rows per warp and step
constexpr int kInFlight = 8;               // 32-wide k chunks of loads in flight per lane
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Elements k .. k + 7 of a row of `d`, zero past its end (the row may end
// anywhere; its memory past d is not touched).
__device__ __forceinline__ uint4 load_k8(const __nv_bfloat16* row, int k, int d) {
  if (k + 8 <= d) return __ldg(reinterpret_cast<const uint4*>(row + k));
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (k + i < d) w[i >> 1] |= (uint32_t)__bfloat16_as_ushort(row[k + i]) << (16 * (i & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// (m, s) of two disjoint sets of logits
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float mn = fmaxf(m, m2), base = mn == -INFINITY ? 0.f : mn;
  s = s * ex2((m - base) * kLog2e) + s2 * ex2((m2 - base) * kLog2e);
  m = mn;
}

// NT: groups of 8 rows of H. part[block][R] gets the statistics of the block's
// columns but the target's, zs[r] the target's logit; a single block holds all columns and writes
// loss and lse itself.
template <int NT>
__global__ void __launch_bounds__(kWarps * 32) head_small_kernel(const __nv_bfloat16* __restrict__ H, int ldh,
                                                                 const __nv_bfloat16* __restrict__ W, int ldw,
                                                                 const float* __restrict__ bias,
                                                                 const int* __restrict__ target, int R, int V, int d,
                                                                 float* __restrict__ zs, float2* __restrict__ part,
                                                                 float* __restrict__ loss, float* __restrict__ lse) {
  if (gridDim.x > 1) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the finish kernel follows
  extern __shared__ uint4 hs[];  // [chunks][NT][32 lanes]
  __shared__ float2 ms[kWarps][NT * 8];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int chunks = (d + 31) / 32;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int i = threadIdx.x; i < chunks * NT * 32; i += kWarps * 32) {
    const int l = i & 31, nt = (i >> 5) % NT, c = (i >> 5) / NT;
    const int r = nt * 8 + (l >> 2);
    hs[i] = r < R ? load_k8(H + (size_t)r * ldh, c * 32 + (l & 3) * 8, d) : make_uint4(0, 0, 0, 0);
  }
  int tg[NT][2];  // targets of this lane's rows of H
  float m[NT][2], s[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int r = nt * 8 + 2 * t + c;
      tg[nt][c] = r < R ? target[r] : -1;
      m[nt][c] = -INFINITY;
      s[nt][c] = 0.f;
    }
  __syncthreads();

  const int tiles = (V + kTileRows - 1) / kTileRows;
  for (int tile = blockIdx.x * kWarps + w; tile < tiles; tile += gridDim.x * kWarps) {
    const int v0 = tile * kTileRows + g, v1 = v0 + 8;
    const __nv_bfloat16* w0 = W + (size_t)min(v0, V - 1) * ldw;
    const __nv_bfloat16* w1 = W + (size_t)min(v1, V - 1) * ldw;
    float c[NT][4] = {};
    for (int k0 = 0; k0 < chunks; k0 += kInFlight) {
      uint4 a0[kInFlight], a1[kInFlight];
#pragma unroll
      for (int u = 0; u < kInFlight; ++u)
        if (k0 + u < chunks) {
          a0[u] = load_k8(w0, (k0 + u) * 32 + t * 8, d);
          a1[u] = load_k8(w1, (k0 + u) * 32 + t * 8, d);
        }
#pragma unroll
      for (int u = 0; u < kInFlight; ++u)
        if (k0 + u < chunks) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint4 b = hs[((k0 + u) * NT + nt) * 32 + lane];
            mma_bf16(c[nt], a0[u].x, a1[u].x, a0[u].y, a1[u].y, b.x, b.y);
            mma_bf16(c[nt], a0[u].z, a1[u].z, a0[u].w, a1[u].w, b.z, b.w);
          }
        }
    }
    const float b0 = bias && v0 < V ? bias[v0] : 0.f, b1 = bias && v1 < V ? bias[v1] : 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float z0 = c[nt][k] + b0, z1 = c[nt][2 + k] + b1;
        if (v0 >= V) z0 = -INFINITY;
        if (v1 >= V) z1 = -INFINITY;
        const int id = tg[nt][k];
        if (id == v0 && v0 < V) {
          zs[nt * 8 + 2 * t + k] = z0;
          z0 = -INFINITY;
        }
        if (id == v1 && v1 < V) {
          zs[nt * 8 + 2 * t + k] = z1;
          z1 = -INFINITY;
        }
        const float mn = max3f(m[nt][k], z0, z1), base = mn == -INFINITY ? 0.f : mn;
        s[nt][k] = s[nt][k] * ex2((m[nt][k] - base) * kLog2e) + (ex2((z0 - base) * kLog2e) + ex2((z1 - base) * kLog2e));
        m[nt][k] = mn;
      }
  }
  // over the 8 row groups of the warp, then over the warps
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m[nt][k], o), s2 = __shfl_xor_sync(0xffffffffu, s[nt][k], o);
        join(m[nt][k], s[nt][k], m2, s2);
      }
      if (g == 0) ms[w][nt * 8 + 2 * t + k] = make_float2(m[nt][k], s[nt][k]);
    }
  __syncthreads();
  if (threadIdx.x < R) {
    float mm = ms[0][threadIdx.x].x, ss = ms[0][threadIdx.x].y;
    for (int i = 1; i < kWarps; ++i) join(mm, ss, ms[i][threadIdx.x].x, ms[i][threadIdx.x].y);
    if (gridDim.x > 1) {
      part[(size_t)blockIdx.x * R + threadIdx.x] = make_float2(mm, ss);
    } else {
      const int id = target[threadIdx.x];
      const bool has = id >= 0 && id < V;
      // zs[row] was written by this block before the barrier
      nll_row(mm, ss, has ? __ldcg(zs + threadIdx.x) : 0.f, has, 1.f, loss[threadIdx.x], lse[threadIdx.x]);
    }
  }
}

int small_smem(int R, int d) { return (d + 31) / 32 * ((R + 7) / 8) * 512; }

}  // namespace

// Statistics slots (blocks) of the small kernel, 0 where it does not apply: up
// to 16 rows whose fragments fit 96 KB of shared memory (two blocks per SM).
// Small against tcgen05 kernel, whole forward (us), at 8, 16 and, by the latter
// alone, 17 rows: 32768 x 1024 19.2 / 25.3, 22.6 / 23.5, 23.7; 131072 x 2048
// 98 / 138, 103 / 133, 133; 5000 x 512 7.2 / 10.7, 8.4 / 11.0, 10.9; 65 x 384
// 4.0 / 7.4, 4.7 / 7.4, 7.4.
int head_small_slots(int R, int V, int d) {
  if (R > 16 || small_smem(R, d) > 96 * 1024) return 0;
  const int tiles = (V + kTileRows - 1) / kTileRows;
  return std::min((tiles + kWarps - 1) / kWarps, 2 * num_sms());
}

cudaError_t head_small(const HeadTcArgs& a, const void* H, int ldh, const void* W, int ldw, int slots, float* loss,
                       float* lse, cudaStream_t s) {
  const int smem = small_smem(a.R, a.d);
  auto run = [&](auto kern, std::atomic<unsigned long long>& done) {
    const cudaError_t e = allow_smem(kern, 96 * 1024, done);
    if (e != cudaSuccess) return e;
    return launch_dependent(kern, slots, kWarps * 32, smem, 1, s, (const __nv_bfloat16*)H, ldh, (const __nv_bfloat16*)W,
                            ldw, a.bias, a.sid, a.R, a.V, a.d, a.zs, a.part, loss, lse);
  };
  static std::atomic<unsigned long long> done[2];
  return a.R <= 8 ? run(head_small_kernel<1>, done[0]) : run(head_small_kernel<2>, done[1]);
}

}  // namespace dgx
