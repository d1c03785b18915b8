// Token embedding with a scale, and its table gradient summed in token order.
//
//   x_i  = s * W[tok_i] (+ P[i mod S])          an id outside [0, V): zero (+ P)
//   dW_t (+)= s * sum over i with tok_i = t of dx_i, in ascending i
//
// Tables, activations and gradients in fp32 or bf16; sums in fp32 in a fixed
// order (no atomics on values), rounded once.
#include <cuda_bf16.h>

#include <algorithm>

#include "common.h"
#include "sm100.cuh"

namespace dgx {
namespace {

__device__ __forceinline__ float ldf(const float* p) { return *p; }
__device__ __forceinline__ float ldf(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void stf(float* p, float v) { *p = v; }
__device__ __forceinline__ void stf(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <typename TW, typename TX>
__global__ void embed_fwd_kernel(const int* __restrict__ tok, const TW* __restrict__ W, int ldw,
                                 const float* __restrict__ P, int S, float scale, TX* __restrict__ x, int ldx, int n,
                                 int d, int V) {
  const long long total = (long long)n * d;
  for (long long e = blockIdx.x * (long long)blockDim.x + threadIdx.x; e < total;
       e += (long long)gridDim.x * blockDim.x) {
    const int i = (int)(e / d), j = (int)(e % d);
    const int t = tok[i];
    float v = (t >= 0 && t < V) ? scale * ldf(W + (size_t)t * ldw + j) : 0.f;
    if (P) v += P[(size_t)(i % S) * d + j];
    stf(x + (size_t)i * ldx + j, v);
  }
}

// One warp per (table row, 128 columns): the lanes scan the tokens 32 at a
// time and add the matching rows in order.
template <typename TG, typename TW>
__global__ void embed_bwd_scan_kernel(const int* __restrict__ tok, const TG* __restrict__ dx, int lddx, float scale,
                                      TW* __restrict__ dW, int lddw, int n, int d, int V, int accumulate) {
  const int t = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (t >= V) return;
  for (int c0 = blockIdx.y * 128; c0 < d; c0 += gridDim.y * 128) {
    float acc[4] = {};
    bool hit = false;
    for (int i0 = 0; i0 < n; i0 += 32) {
      unsigned m = __ballot_sync(0xffffffffu, i0 + lane < n && tok[i0 + lane] == t);
      while (m) {
        const int i = i0 + __ffs(m) - 1;
        m &= m - 1;
        hit = true;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int j = c0 + k * 32 + lane;
          if (j < d) acc[k] += ldf(dx + (size_t)i * lddx + j);
        }
      }
    }
    if (accumulate && !hit) continue;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int j = c0 + k * 32 + lane;
      if (j >= d) continue;
      TW* o = dW + (size_t)t * lddw + j;
      stf(o, (accumulate ? ldf(o) : 0.f) + scale * acc[k]);
    }
  }
}

bool type_ok(int t) { return t == DGX_F32 || t == DGX_BF16; }

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
  const long long total = (long long)n * d;
  const int grid = (int)std::min<long long>((total + 255) / 256, num_sms() * 8ll);
  auto run = [&](auto* w, auto* o) {
    embed_fwd_kernel<<<grid, 256, 0, s>>>(tok, w, ldw, P, P ? S : 1, scale, o, ldx, n, d, V);
  };
  if (w_type == DGX_F32 && x_type == DGX_F32) run((const float*)W, (float*)x);
  else if (w_type == DGX_F32) run((const float*)W, (__nv_bfloat16*)x);
  else if (x_type == DGX_F32) run((const __nv_bfloat16*)W, (float*)x);
  else run((const __nv_bfloat16*)W, (__nv_bfloat16*)x);
  return cuda_status(cudaGetLastError(), "dgx_embed_fwd");
}

size_t dgx_embed_bwd_workspace_size(int n, int d, int V) {
  (void)n;
  (void)d;
  (void)V;
  return 0;
}

dgx_status dgx_embed_bwd(const int* tok, const void* dx, dgx_dtype dx_type, int lddx, float scale, void* dW,
                         dgx_dtype dw_type, int lddw, int n, int d, int V, int accumulate, void* workspace,
                         size_t workspace_bytes, void* stream) {
  DGX_FAULT_POINT("dgx_embed_bwd");
  if (n < 0 || d <= 0 || V <= 0) return set_error(DGX_EINVAL, "dgx_embed_bwd: bad size n=%d d=%d V=%d", n, d, V);
  if (!type_ok(dx_type) || !type_ok(dw_type))
    return set_error(DGX_EINVAL, "dgx_embed_bwd: types %d %d", dx_type, dw_type);
  if (lddx < d || lddw < d) return set_error(DGX_EINVAL, "dgx_embed_bwd: row pitch %d or %d < d=%d", lddx, lddw, d);
  if (accumulate && dw_type != DGX_F32) return set_error(DGX_EUNSUPPORTED, "dgx_embed_bwd: accumulate needs an fp32 dW");
  if (!dW || (n > 0 && (!tok || !dx))) return set_error(DGX_EINVAL, "dgx_embed_bwd: null pointer");
  (void)workspace;
  (void)workspace_bytes;
  cudaStream_t s = (cudaStream_t)stream;
  const dim3 grid((V + 7) / 8, std::min((d + 127) / 128, 64));
  auto run = [&](auto* g, auto* o) {
    embed_bwd_scan_kernel<<<grid, 256, 0, s>>>(tok, g, lddx, scale, o, lddw, n, d, V, accumulate);
  };
  if (dx_type == DGX_F32 && dw_type == DGX_F32) run((const float*)dx, (float*)dW);
  else if (dx_type == DGX_F32) run((const float*)dx, (__nv_bfloat16*)dW);
  else if (dw_type == DGX_F32) run((const __nv_bfloat16*)dx, (float*)dW);
  else run((const __nv_bfloat16*)dx, (__nv_bfloat16*)dW);
  return cuda_status(cudaGetLastError(), "dgx_embed_bwd");
}

}  // extern "C"
