// Both gradient products of one piece of the vocabulary in one launch:
//   dH (+)= G W     [R, d], summed over the n columns of the piece
//   dW    = G^T H   [n, d], summed over the R rows
// G [R, n] bf16 is read as it stands by both: K-major for dH, MN-major for dW
// (the tcgen05 operand descriptors transpose). Output tiles of 256 x BN over a
// CTA pair with the main loop of gemm2_kernel.
//
// One launch rather than two GEMMs: 256 x 256 tiles quantise badly over 74 SM
// pairs (R = 8192, n = 16384, d = 1024: 128 dH tiles are 1.7 waves, 256 dW
// tiles 3.5). The tiles of the two products differ in length (n / 64 or R / 64
// steps), so the longer ones go out first, one round over the pairs at a time,
// and the pairs that got one fewer start on the shorter ones meanwhile; every
// pair ends within about one short tile of the mean. Where a tile alone would
// take longer than the mean load of a pair, its sum is split into slices that
// go to fp32 scratch [slice][rows][d] and head_sums_kernel adds them in order.
// Bound by the tensor pipe: 344 us, 1.60 PFLOP/s, at R = 4096, n = 32768,
// d = 1024. Short tiles wait for operand loads: a sixth stage is worth 1-2 %,
// sixteen epilogue warps (and five stages) cost 1-3 %.
#include <algorithm>

#include "gemm.h"
#include "head.h"
#include "launch.h"
#include "pair.cuh"
#include "sm100.cuh"

namespace dgx {
namespace {

constexpr int HG_BM = 128;  // rows per CTA (256 per pair)
constexpr int HG_BK = 64;
constexpr int HG_STAGES = 6;
constexpr int HG_EPI_WARPS = 8;
constexpr int HG_THREADS = 64 + 32 * HG_EPI_WARPS;
constexpr uint32_t HG_TMEM_COLS = 512;

template <int BN>
struct HgCfg {
  static constexpr int A_BYTES = HG_BM * HG_BK * 2;
  static constexpr int B_BYTES = (BN / 2) * HG_BK * 2;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int SMEM = HG_STAGES * STAGE + HG_EPI_WARPS * 4096 + 1024 + 256;
};

struct GradProblem {
  int rows, tiles_m, nk, splits, kper, units;
  int out;      // 0 bf16 store, 1 fp32 store, 2 fp32 reduce-add
  float alpha;
};

struct GradArgs {
  GradProblem p[2];  // dH, dW
  int tiles_n, d;
  int heavy, nh, nl, r, x;  // schedule (see unit_at)
  uint32_t* err;
};

struct Unit {
  int prob, tm, tn, kb0, kb1, slice;
};

// The i-th unit of pair `p` of P; false past the last. The nh heavy units go
// round-robin; r = nh % P pairs have one more than the others, which take x
// light units each first; the remaining light units go round-robin too, so
// that the pairs running together share operand tiles in L2.
__device__ __forceinline__ bool unit_at(const GradArgs& a, int i, int p, int P, Unit& u) {
  const int mine = a.nh > p ? (a.nh - p - 1) / P + 1 : 0;
  int idx;
  if (i < mine) {
    u.prob = a.heavy;
    idx = p + i * P;
  } else {
    u.prob = 1 - a.heavy;
    const int j = i - mine;
    if (p >= a.r)
      idx = j < a.x ? j * (P - a.r) + (p - a.r) : a.x * (P - a.r) + (j - a.x) * P + (p - a.r);
    else
      idx = a.x * (P - a.r) + j * P + (P - a.r) + p;
    if (idx >= a.nl) return false;
  }
  const GradProblem& g = a.p[u.prob];
  u.tn = idx % a.tiles_n;
  idx /= a.tiles_n;
  u.slice = idx % g.splits;
  u.tm = idx / g.splits;
  u.kb0 = u.slice * g.kper;
  u.kb1 = min(g.nk, u.kb0 + g.kper);
  return true;
}

template <int BN>
__global__ void __launch_bounds__(HG_THREADS, 1)
    head_grads_kernel(const __grid_constant__ CUtensorMap tmGk, const __grid_constant__ CUtensorMap tmGm,
                      const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmH,
                      const __grid_constant__ CUtensorMap tmO0, const __grid_constant__ CUtensorMap tmO1, GradArgs a) {
  using Cfg = HgCfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* out_stage = smem + HG_STAGES * Cfg::STAGE;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(out_stage + HG_EPI_WARPS * 4096);
  uint64_t* empty_bar = full_bar + HG_STAGES;
  uint64_t* accf_bar = empty_bar + HG_STAGES;  // [2]
  uint64_t* acce_bar = accf_bar + 2;           // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acce_bar + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank_u32();
  const bool leader = rank == 0;
  WaitCtx wc{abort_flag, a.err};

  if (threadIdx.x == 0) {
    for (int s = 0; s < HG_STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&accf_bar[b], 1);
      mbar_init(&acce_bar[b], 2 * HG_EPI_WARPS);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmGk);
    tma_prefetch_desc(&tmGm);
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmH);
  }
  if (warp == 1) {
    tmem_alloc2(tmem_slot, HG_TMEM_COLS);
    tmem_relinquish2();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all2();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs)
    if (elect_one_lane()) {
      uint32_t fill = 0;
      Unit u;
      for (int i = 0; unit_at(a, i, pair, npairs, u) && !*abort_flag; ++i) {
        const int m0 = u.tm * 2 * HG_BM + (int)rank * HG_BM;
        const int n0 = u.tn * BN + (int)rank * (BN / 2);
        const CUtensorMap* mb = u.prob ? &tmH : &tmW;
        for (int kb = u.kb0; kb < u.kb1; ++kb, ++fill) {
          const int s = fill % HG_STAGES;
          if (!mbar_wait(&empty_bar[s], ((fill / HG_STAGES) & 1) ^ 1, wc)) break;
          uint8_t* sa = smem + s * Cfg::STAGE;
          uint8_t* sb = sa + Cfg::A_BYTES;
          if (leader) mbar_arrive_expect_tx(&full_bar[s], 2 * Cfg::STAGE);
          const int k0 = kb * HG_BK;
          if (u.prob) {
#pragma unroll
            for (int c = 0; c < 2; ++c) tma_load_2d_pair(sa + c * HG_BK * 128, &tmGm, &full_bar[s], m0 + c * 64, k0);
          } else {
            tma_load_2d_pair(sa, &tmGk, &full_bar[s], k0, m0);
          }
#pragma unroll
          for (int c = 0; c < BN / 128; ++c) tma_load_2d_pair(sb + c * HG_BK * 128, mb, &full_bar[s], n0 + c * 64, k0);
        }
      }
      const uint32_t first = fill > (uint32_t)HG_STAGES ? fill - HG_STAGES : 0;
      for (uint32_t f = first; f < fill; ++f) mbar_drain(&empty_bar[f % HG_STAGES], (f / HG_STAGES) & 1);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader only)
    if (leader && elect_one_lane()) {
      constexpr uint32_t idesc_k = make_idesc(1, 0, 1, 2 * HG_BM, BN), idesc_m = make_idesc(1, 1, 1, 2 * HG_BM, BN);
      uint32_t fill = 0, use = 0;
      Unit u;
      bool ok = true;
      for (int i = 0; ok && unit_at(a, i, pair, npairs, u); ++i) {
        if (u.kb0 >= u.kb1) continue;
        const int buf = use & 1;
        if (!mbar_wait(&acce_bar[buf], ((use >> 1) & 1) ^ 1, wc)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * BN;
        for (int kb = u.kb0; kb < u.kb1; ++kb, ++fill) {
          const int s = fill % HG_STAGES;
          if (!mbar_wait(&full_bar[s], (fill / HG_STAGES) & 1, wc)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + s * Cfg::STAGE), sb = sa + Cfg::A_BYTES;
#pragma unroll
          for (int kk = 0; kk < HG_BK / 16; ++kk) {
            const uint64_t adesc = u.prob ? sw128_desc(sa + kk * 16 * 128, HG_BK * 128, 1024)
                                          : sw128_desc(sa + kk * 32, 16, 1024);
            const uint64_t bdesc = sw128_desc(sb + kk * 16 * 128, HG_BK * 128, 1024);
            mma2_f16_ss(d_tmem, adesc, bdesc, u.prob ? idesc_m : idesc_k, (kb > u.kb0 || kk > 0) ? 1u : 0u);
          }
          tc_commit2_mc(&empty_bar[s], 0x3);
        }
        if (!ok) break;
        tc_commit2_mc(&accf_bar[buf], 0x3);
        ++use;
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue (warps 2..9, both CTAs)
    // Two warps per TMEM lane quarter take the column chunks in turn: a tile of
    // few K steps lasts as long as its epilogue.
    const int q = warp & 3, half = (warp - 2) >> 2;
    uint8_t* st = out_stage + (warp - 2) * 4096;
    uint32_t issued = 0, use = 0;
    Unit u;
    for (int i = 0; unit_at(a, i, pair, npairs, u); ++i) {
      if (u.kb0 >= u.kb1) continue;
      const int buf = use & 1;
      const GradProblem& g = a.p[u.prob];
      if (!mbar_wait(&accf_bar[buf], (use >> 1) & 1, wc)) break;
      tc_fence_after();
      const int row0 = u.tm * 2 * HG_BM + (int)rank * HG_BM + q * 32;
      const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + buf * BN;
      const CUtensorMap* mo = u.prob ? &tmO1 : &tmO0;
      const int cw = g.out == 0 ? 64 : 32;
#pragma unroll 1
      for (int c = half * cw; c < BN; c += 2 * cw) {
        uint32_t r[64];
        tmem_ld32(taddr + c, *reinterpret_cast<uint32_t(*)[32]>(&r[0]));
        if (cw == 64) tmem_ld32(taddr + c + 32, *reinterpret_cast<uint32_t(*)[32]>(&r[32]));
        tmem_ld_wait();
        if (c + 2 * cw >= BN) {  // this warp's last read of the accumulator
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (leader)
              mbar_arrive(&acce_bar[buf]);
            else
              mbar_arrive_remote_relaxed(&acce_bar[buf], 0);
          }
        }
        if (u.tn * BN + c >= a.d || row0 >= g.rows) continue;  // uniform: past the last column or row
        if (lane == 0 && issued) bulk_wait_read0();
        __syncwarp();
        uint32_t w[32];
        if (cw == 64) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            w[j] = pack_bf16x2(g.alpha * __uint_as_float(r[2 * j]), g.alpha * __uint_as_float(r[2 * j + 1]));
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) w[j] = __float_as_uint(g.alpha * __uint_as_float(r[j]));
        }
#pragma unroll
        for (int v = 0; v < 8; ++v)
          *reinterpret_cast<uint4*>(st + lane * 128 + ((v ^ (lane & 7)) << 4)) =
              make_uint4(w[4 * v], w[4 * v + 1], w[4 * v + 2], w[4 * v + 3]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (g.out == 2)
            tma_reduce_add_3d(mo, st, u.tn * BN + c, row0, u.slice);
          else
            tma_store_3d(mo, st, u.tn * BN + c, row0, u.slice);
          bulk_commit();
        }
        ++issued;
      }
      ++use;
    }
    if (lane == 0) bulk_wait0();
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all2();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc2(tmem_base, HG_TMEM_COLS);
  }
}

bool encode_out(CUtensorMap* map, void* base, bool bf16, uint64_t d, uint64_t rows, uint64_t slices, uint64_t ld) {
  auto enc = get_tensor_map_encoder();
  if (!enc) return false;
  const int es = bf16 ? 2 : 4;
  const cuuint64_t dims[3] = {d, rows, slices};
  const cuuint64_t strides[2] = {ld * es, rows * ld * es};
  const cuuint32_t box[3] = {(cuuint32_t)(128 / es), 32, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  return enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, base, dims, strides, box,
             estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BN>
cudaError_t launch(const CUtensorMap (&m)[6], const GradArgs& a, int pairs, cudaStream_t s) {
  static std::atomic<unsigned long long> done;
  const cudaError_t e = allow_smem(head_grads_kernel<BN>, HgCfg<BN>::SMEM, done);
  if (e != cudaSuccess) return e;
  return launch_dependent(head_grads_kernel<BN>, 2 * pairs, HG_THREADS, HgCfg<BN>::SMEM, 2, s, m[0], m[1], m[2], m[3],
                          m[4], m[5], a);
}

}  // namespace

// K steps that a tile costs at least: its epilogue and the latency of its first
// loads (4 / 7 / 10 / 14 / 20: 60 x 32000 x 1024 training 89 / 81 / 83 / 87 / 96
// us, 333 x 50257 x 512 distillation 139 / 136 / 132 / 135 / 140, 16384 x 65 x 384
// training 44 / 41 / 41 / 43 / 44).
constexpr int kMinCost = 10;

// Slices of the two products' sums so that no tile takes longer than the mean
// load of an SM pair (at most kMaxSplits; the scratch is sized by the same rule).
GradSplits head_grad_splits(int R, int n, int d, bool want_dh, bool want_dw) {
  const long long tn = (d + 255) / 256, pairs = std::max(1, num_sms() / 2);
  const long long kp[2] = {(n + 63) / 64, (R + 63) / 64};
  const long long tiles[2] = {want_dh ? (R + 255) / 256 * tn : 0, want_dw ? (n + 255) / 256 * tn : 0};
  const long long work = tiles[0] * std::max<long long>(kp[0], kMinCost) + tiles[1] * std::max<long long>(kp[1], kMinCost);
  const long long mean = std::max<long long>(8, (work + pairs - 1) / pairs);
  GradSplits sp;
  int* out[2] = {&sp.dh, &sp.dw};
  for (int i = 0; i < 2; ++i) {
    long long s = std::min<long long>((kp[i] + mean - 1) / mean, kMaxSplits);
    const long long kper = (kp[i] + s - 1) / s;
    *out[i] = (int)((kp[i] + kper - 1) / kper);  // no empty slice
  }
  return sp;
}

cudaError_t head_grads_tc(const HeadGradTc& g, cudaStream_t s) {
  GradArgs a{};
  a.err = g.err;
  constexpr int BN = 256;
  a.tiles_n = (g.d + BN - 1) / BN;
  a.d = g.d;
  CUtensorMap m[6]{};
  if (!encode_2d_bf16(&m[0], g.G, g.n, g.R, (uint64_t)g.ldg * 2, HG_BK, HG_BM) ||
      !encode_2d_bf16(&m[1], g.G, g.n, g.R, (uint64_t)g.ldg * 2, 64, HG_BK) ||
      !encode_2d_bf16(&m[2], g.W, g.d, g.n, (uint64_t)g.ldw * 2, 64, HG_BK) ||
      !encode_2d_bf16(&m[3], g.H, g.d, g.R, (uint64_t)g.ldh * 2, 64, HG_BK))
    return cudaErrorInvalidValue;
  m[4] = m[5] = m[0];
  const int rows[2] = {g.R, g.n}, k[2] = {g.n, g.R};
  for (int i = 0; i < 2; ++i) {
    const GradOut& o = g.out[i];
    GradProblem& p = a.p[i];
    p.nk = (k[i] + HG_BK - 1) / HG_BK;
    p.splits = std::max(1, o.splits);
    p.kper = (p.nk + p.splits - 1) / p.splits;
    if (!o.ptr) continue;
    p.rows = rows[i];
    p.tiles_m = (rows[i] + 2 * HG_BM - 1) / (2 * HG_BM);
    p.units = p.tiles_m * a.tiles_n * p.splits;
    p.out = o.bf16 ? 0 : o.add ? 2 : 1;
    p.alpha = o.alpha;
    if (!encode_out(&m[4 + i], o.ptr, o.bf16, g.d, rows[i], p.splits, o.ld)) return cudaErrorInvalidValue;
  }
  const int total = a.p[0].units + a.p[1].units;
  if (!total) return cudaSuccess;
  const int P = std::min(total, std::max(1, num_sms() / 2));
  a.heavy = a.p[1].units && (!a.p[0].units || a.p[1].kper > a.p[0].kper) ? 1 : 0;
  a.nh = a.p[a.heavy].units;
  a.nl = a.p[1 - a.heavy].units;
  a.r = a.nh % P;
  if (a.r && a.nl) {
    const int ch = std::max(a.p[a.heavy].kper, kMinCost), cl = std::max(a.p[1 - a.heavy].kper, kMinCost);
    a.x = std::min((ch + cl / 2) / cl, a.nl / (P - a.r));
  }
  return launch<BN>(m, a, P, s);
}

}  // namespace dgx
