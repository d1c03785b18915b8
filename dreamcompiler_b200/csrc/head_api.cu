// C ABI entry points of the vocabulary head (include/dgx.h): the linear
// layer, softmax and loss of a language model in one operator, for a hard
// target (dgx_linear_nll_*) and for a teacher's largest logits
// (dgx_linear_distill_*). Argument checks and workspace handling; the work is
// in head.cu.
#include <algorithm>
#include <cmath>

#include "common.h"
#include "head.h"

using namespace dgx;

namespace {

dgx_status head_check(const char* op, const void* H, int ldh, const void* W, int ldw, int R, int V, int d, int K) {
  if (R < 0 || V <= 0 || d <= 0) return set_error(DGX_EINVAL, "%s: bad size R=%d V=%d d=%d", op, R, V, d);
  if (R > kHeadMaxDim || V > kHeadMaxDim || d > kHeadMaxDim)
    return set_error(DGX_EINVAL, "%s: R=%d, V=%d or d=%d above %d", op, R, V, d, kHeadMaxDim);
  if (K < 1 || K > kHeadMaxK) return set_error(DGX_EINVAL, "%s: K=%d (1..%d entries per row)", op, K, kHeadMaxK);
  if (ldh < d || ldw < d || ldh % 8 || ldw % 8)
    return set_error(DGX_EINVAL, "%s: row pitch ldh=%d ldw=%d (>= d=%d and a multiple of 8)", op, ldh, ldw, d);
  if (R > 0 && (!H || !W)) return set_error(DGX_EINVAL, "%s: null operand", op);
  if (((uintptr_t)H | (uintptr_t)W) & 15) return set_error(DGX_EINVAL, "%s: H and W must be 16-byte aligned", op);
  return DGX_OK;
}

// The workspace of a call: the caller's when given (checked), else the library's.
dgx_status head_workspace(const char* op, void*& ws, size_t bytes, size_t need, cudaStream_t s) {
  if (ws) {
    if (bytes < need) return set_error(DGX_ENOMEM, "%s: workspace %zu bytes < %zu", op, bytes, need);
    if ((uintptr_t)ws & 127) return set_error(DGX_EINVAL, "%s: workspace must be 128-byte aligned", op);
    return DGX_OK;
  }
  ws = library_scratch_slot(kScratchHead, need, s);
  if (!ws) return set_error(DGX_ENOMEM, "%s: cannot allocate %zu bytes of scratch", op, need);
  return DGX_OK;
}

dgx_status run_fwd(const char* op, HeadArgs& a, void* ws, size_t ws_bytes, cudaStream_t s) {
  dgx_status st = head_check(op, a.H, a.ldh, a.W, a.ldw, a.R, a.V, a.d, a.K);
  if (st != DGX_OK) return st;
  if (a.R == 0) {
    if (a.mean) return cuda_status(cudaMemsetAsync(a.mean, 0, sizeof(float), s), op);
    return DGX_OK;
  }
  if (!a.idx || !a.loss || !a.lse) return set_error(DGX_EINVAL, "%s: null pointer", op);
  st = head_workspace(op, ws, ws_bytes, head_fwd_scratch_bytes(a.R, a.V, a.d, a.K, a.teacher != nullptr), s);
  if (st != DGX_OK) return st;
  a.err = device_error_word();
  return head_fwd(a, ws, s);
}

dgx_status run_bwd(const char* op, HeadArgs& a, int dh_type, int dw_type, int accumulate, void* ws, size_t ws_bytes, cudaStream_t s) {
  dgx_status st = head_check(op, a.H, a.ldh, a.W, a.ldw, a.R, a.V, a.d, a.K);
  if (st != DGX_OK) return st;
  if (a.dH && dh_type != DGX_F32 && dh_type != DGX_BF16) return set_error(DGX_EINVAL, "%s: dH type %d", op, dh_type);
  if (a.dW && dw_type != DGX_F32 && dw_type != DGX_BF16) return set_error(DGX_EINVAL, "%s: dW type %d", op, dw_type);
  a.dh_bf16 = dh_type == DGX_BF16;
  a.dw_bf16 = dw_type == DGX_BF16;
  const int hq = a.dh_bf16 ? 8 : 4, wq = a.dw_bf16 ? 8 : 4;  // elements in 16 bytes
  if (a.dH && (a.lddh < a.d || a.lddh % hq || ((uintptr_t)a.dH & 15)))
    return set_error(DGX_EINVAL, "%s: dH needs 16-byte aligned rows of at least d=%d elements (lddh=%d)", op, a.d, a.lddh);
  if (a.dW && (a.lddw < a.d || a.lddw % wq || ((uintptr_t)a.dW & 15)))
    return set_error(DGX_EINVAL, "%s: dW needs 16-byte aligned rows of at least d=%d elements (lddw=%d)", op, a.d, a.lddw);
  if (accumulate & ~(DGX_ACC_W | DGX_ACC_H)) return set_error(DGX_EINVAL, "%s: accumulate %d", op, accumulate);
  a.add_w = (accumulate & DGX_ACC_W) != 0;
  a.add_h = (accumulate & DGX_ACC_H) != 0;
  if ((a.add_w && a.dW && a.dw_bf16) || (a.add_h && a.dH && a.dh_bf16))
    return set_error(DGX_EUNSUPPORTED, "%s: accumulate needs an fp32 %s", op, a.add_w && a.dw_bf16 ? "dW" : "dH");
  if (a.R == 0) {  // a sum over no rows
    cudaError_t e = cudaSuccess;
    if (!a.add_w && a.dW)
      e = cudaMemset2DAsync(a.dW, (size_t)a.lddw * (a.dw_bf16 ? 2 : 4), 0, (size_t)a.d * (a.dw_bf16 ? 2 : 4), a.V, s);
    if (e == cudaSuccess && !a.add_w && a.db) e = cudaMemsetAsync(a.db, 0, (size_t)a.V * sizeof(float), s);
    return cuda_status(e, op);
  }
  if (!a.idx || !a.lse) return set_error(DGX_EINVAL, "%s: null pointer", op);
  if (!a.dH && !a.dW && !a.db) return DGX_OK;
  st = head_workspace(op, ws, ws_bytes, head_bwd_scratch_bytes(a.R, a.V, a.d, a.K, a.teacher != nullptr), s);
  if (st != DGX_OK) return st;
  a.err = device_error_word();
  return head_bwd(a, ws, s);
}

dgx_status check_temperature(const char* op, float t) {
  // T^2 and the scaled logits' factor log2(e) / T have to be finite too
  if (!(t > 0.f) || !std::isfinite(t * t) || !std::isfinite(2.f / t))
    return set_error(DGX_EINVAL, "%s: temperature %g", op, (double)t);
  return DGX_OK;
}

}  // namespace

extern "C" {

size_t dgx_linear_nll_workspace_size(int R, int V, int d, int backward) {
  if (R <= 0 || V <= 0 || d <= 0 || std::max({R, V, d}) > kHeadMaxDim) return 0;
  return backward ? head_bwd_scratch_bytes(R, V, d, 1, false) : head_fwd_scratch_bytes(R, V, d, 1, false);
}

size_t dgx_linear_distill_workspace_size(int R, int V, int d, int K, int backward) {
  if (R <= 0 || V <= 0 || d <= 0 || std::max({R, V, d}) > kHeadMaxDim || K < 1 || K > kHeadMaxK) return 0;
  return backward ? head_bwd_scratch_bytes(R, V, d, K, true) : head_fwd_scratch_bytes(R, V, d, K, true);
}

dgx_status dgx_linear_nll_fwd(const void* H, int ldh, const void* W, int ldw, const float* bias, const int* target,
                              int R, int V, int d, float* loss, float* lse, float* mean, void* workspace,
                              size_t workspace_bytes, void* stream) {
  DGX_FAULT_POINT("dgx_linear_nll_fwd");
  HeadArgs a{};
  a.H = H;
  a.W = W;
  a.bias = bias;
  a.idx = target;
  a.ldh = ldh;
  a.ldw = ldw;
  a.R = R;
  a.V = V;
  a.d = d;
  a.K = 1;
  a.t = a.inv_t = 1.f;
  a.loss = loss;
  a.lse = lse;
  a.mean = mean;
  return run_fwd("dgx_linear_nll_fwd", a, workspace, workspace_bytes, (cudaStream_t)stream);
}

dgx_status dgx_linear_nll_bwd(const void* H, int ldh, const void* W, int ldw, const float* bias, const int* target,
                              const float* lse, const float* dloss, float scale, int R, int V, int d, void* dH,
                              dgx_dtype dh_type, int lddh, void* dW, dgx_dtype dw_type, int lddw, float* db,
                              int accumulate, void* workspace, size_t workspace_bytes, void* stream) {
  DGX_FAULT_POINT("dgx_linear_nll_bwd");
  HeadArgs a{};
  a.H = H;
  a.W = W;
  a.bias = bias;
  a.idx = target;
  a.ldh = ldh;
  a.ldw = ldw;
  a.R = R;
  a.V = V;
  a.d = d;
  a.K = 1;
  a.t = a.inv_t = 1.f;
  a.lse = const_cast<float*>(lse);
  a.dloss = dloss;
  a.scale = scale;
  a.dH = dH;
  a.lddh = lddh;
  a.dW = dW;
  a.lddw = lddw;
  a.db = db;
  return run_bwd("dgx_linear_nll_bwd", a, dh_type, dw_type, accumulate, workspace, workspace_bytes, (cudaStream_t)stream);
}

dgx_status dgx_linear_distill_fwd(const void* H, int ldh, const void* W, int ldw, const float* bias, const int* idx,
                                  const float* teacher, int K, float temperature, int R, int V, int d, float* loss,
                                  float* lse, float* mean, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  DGX_FAULT_POINT("dgx_linear_distill_fwd");
  dgx_status st = check_temperature("dgx_linear_distill_fwd", temperature);
  if (st != DGX_OK) return st;
  if (R > 0 && (!teacher)) return set_error(DGX_EINVAL, "dgx_linear_distill_fwd: null pointer");
  HeadArgs a{};
  a.H = H;
  a.W = W;
  a.bias = bias;
  a.idx = idx;
  a.teacher = teacher;
  a.ldh = ldh;
  a.ldw = ldw;
  a.R = R;
  a.V = V;
  a.d = d;
  a.K = K;
  a.t = temperature;
  a.inv_t = 1.f / temperature;
  a.loss = loss;
  a.lse = lse;
  a.mean = mean;
  return run_fwd("dgx_linear_distill_fwd", a, workspace, workspace_bytes, (cudaStream_t)stream);
}

dgx_status dgx_linear_distill_bwd(const void* H, int ldh, const void* W, int ldw, const float* bias, const int* idx,
                                  const float* teacher, int K, float temperature, const float* lse,
                                  const float* dloss, float scale, int R, int V, int d, void* dH, dgx_dtype dh_type,
                                  int lddh, void* dW, dgx_dtype dw_type, int lddw, float* db, int accumulate,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  DGX_FAULT_POINT("dgx_linear_distill_bwd");
  dgx_status st = check_temperature("dgx_linear_distill_bwd", temperature);
  if (st != DGX_OK) return st;
  if (R > 0 && !teacher) return set_error(DGX_EINVAL, "dgx_linear_distill_bwd: null pointer");
  HeadArgs a{};
  a.H = H;
  a.W = W;
  a.bias = bias;
  a.idx = idx;
  a.teacher = teacher;
  a.ldh = ldh;
  a.ldw = ldw;
  a.R = R;
  a.V = V;
  a.d = d;
  a.K = K;
  a.t = temperature;
  a.inv_t = 1.f / temperature;
  a.lse = const_cast<float*>(lse);
  a.dloss = dloss;
  a.scale = scale * temperature;  // T^2 of the loss times 1/T of the logits
  a.dH = dH;
  a.lddh = lddh;
  a.dW = dW;
  a.lddw = lddw;
  a.db = db;
  return run_bwd("dgx_linear_distill_bwd", a, dh_type, dw_type, accumulate, workspace, workspace_bytes, (cudaStream_t)stream);
}

}  // extern "C"
