// Tensor-core kernels of the vocabulary head (head.cu drives them): the logits
// of 256 rows x 256 columns of the vocabulary are one tcgen05 accumulator
// tile over a CTA pair (cta_group::2, each SM its own 128 rows), consumed by
// the epilogue where they stand. No logit is written to memory.
//
//   head_logits_kernel<kStats>   per row and warp: max and sum of
//                                exp((z - max) / T), and z at the target's ids
//   head_logits_kernel<kGrad>    G = w (exp(z/T - lse) - q) as bf16, and its
//                                column sums before the rounding
//
// Both run the main loop of gemm2_kernel (TMA operand ring, one MMA-issuing
// thread in the leader, two TMEM accumulators) with eight or sixteen epilogue
// warps. Bound by the tensor pipe from d = 1024 on (4096 x 32768 x 1024: 170 us
// and 175 us, 1.61 and 1.57 PFLOP/s), by the epilogue for short contractions.
#include <algorithm>

#include "gemm.h"
#include "head.h"
#include "launch.h"
#include "pair.cuh"
#include "sm100.cuh"

namespace dgx {
namespace {

constexpr int HD_BM = 128;  // rows per CTA (256 per pair)
constexpr int HD_BN = 256;  // vocabulary columns per tile (128 W rows loaded per CTA)
constexpr int HD_BK = 64;   // one 128-byte swizzled row of bf16
constexpr int HD_STAGE = 2 * HD_BM * HD_BK * 2;  // 16 KB of H and 16 KB of W
constexpr uint32_t HD_TMEM_COLS = 512;

constexpr int kStats = 0, kGrad = 1;
// EW epilogue warps; a TMEM lane quarter's 256 columns are split over the
// quarter's warps. After the operand stages: a 4 KB staging box for G per
// warp (the gradient), each warp's columns of the bias, and its rows' results
// of a tile (statistics; twice, for alternate tiles).
template <int MODE, bool BIAS, int EW>
struct HdCfg {
  static constexpr int COLS = 4 * HD_BN / EW;
  static constexpr int THREADS = 64 + 32 * EW;
  static constexpr int OUT = MODE == kGrad ? EW * 4096 : 0;
  static constexpr int BIAS_BYTES = BIAS ? 4 * HD_BN * 4 : 0;
  static constexpr int ROWS = MODE == kStats ? 2 * EW * 32 * 3 * 4 : 0;
  static constexpr int TAIL = OUT + BIAS_BYTES + ROWS + 1024 + 256;
  static constexpr int FIT = (232448 - TAIL) / HD_STAGE;
  static constexpr int STAGES = FIT < 6 ? FIT : 6;
  static constexpr int SMEM = STAGES * HD_STAGE + TAIL;
};
// How many: the exponentials, sums and moves of a 256 x 256 tile take eight
// warps about 4100 cycles (statistics) to 7000 (gradient with bias sums), mostly
// waiting for one another's results; sixteen, with half the registers each,
// need about two thirds of that. A tile's MMAs take 8 d cycles, so sixteen are
// faster up to d = 640, or 768 with a bias (whole training pass, 8 against 16
// warps: 333 x 50257 x 512 129 / 121 us, 8192 x 4000 x 256 101 / 96,
// 2000 x 20000 x 640 with bias 189 / 183, 1537 x 50257 x 768 with bias 405 /
// 400), and beyond that eight, whose smaller staging leaves an operand stage
// more (1000 x 32000 x 768 157 / 160, 2000 x 20000 x 896 with bias 236 / 237,
// 4096 x 32768 x 1024 742 / 753).
constexpr int kManyWarps = 16, kFewWarps = 8;
bool many_warps(int d, bool bias) { return d <= (bias ? 768 : 640); }

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// One row's sparse target: the entries of its sorted list from a tile's first
// column on. The entry after the current one is already loaded when the current
// one is used, so a hit does not wait for memory.
struct Target {
  const int* ids;   // [K] ascending
  const float* qs;  // [K], or null: every q is 1
  int k, K;         // current entry
  int nid, pid;     // its id and the following one's (kNone: none)
  float nq, pq;     // their probabilities
  static constexpr int kNone = 0x7fffffff;
  __device__ __forceinline__ void fetch(int i, int& id, float& q) const {
    id = i < K ? __ldg(ids + i) : kNone;
    q = i < K && qs ? __ldg(qs + i) : 1.f;
  }
  __device__ __forceinline__ void start(int first) {
    k = first;
    fetch(k, nid, nq);
    fetch(k + 1, pid, pq);
  }
  __device__ __forceinline__ void next() {
    ++k;
    nid = pid;
    nq = pq;
    fetch(k + 1, pid, pq);
  }
};

// Row statistics of 32 logits of one row: the target's logits to zs (or zt),
// the running maximum and sum. n0: column within the piece, j0: its vocabulary id.
__device__ __forceinline__ void stats32(float (&z)[32], int n0, int j0, int row, const HeadTcArgs& a, Target& tg,
                                        float& m, float& s, float& zt) {
  if (n0 + 32 > a.n) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (n0 + j >= a.n) z[j] = -INFINITY;
  }
  while (__any_sync(0xffffffffu, (unsigned)tg.nid - (unsigned)j0 < 32u)) {
    const int at = (int)((unsigned)tg.nid - (unsigned)j0);
    float v = 0.f;
#pragma unroll
    for (int j = 0; j < 32; ++j) v = at == j ? z[j] : v;
    if (!a.sq) {  // a hard target stays out of the sum
#pragma unroll
      for (int j = 0; j < 32; ++j) z[j] = at == j ? -INFINITY : z[j];
    }
    if ((unsigned)at < 32u) {
      zt = v;
      if (!a.loss) a.zs[(size_t)row * a.K + tg.k] = v;
      tg.next();
    }
  }
  float cm = max3f(z[0], z[1], z[2]);
#pragma unroll
  for (int j = 3; j < 31; j += 2) cm = max3f(cm, z[j], z[j + 1]);
  cm = fmaxf(cm, z[31]);
  const float mn = fmaxf(m, cm);
  const float base = mn == -INFINITY ? 0.f : mn;
  float2 s0 = make_float2(s * ex2((m - base) * a.k), 0.f), s1 = make_float2(0.f, 0.f);
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    // subtract before scaling: exact for equal logits of any size
    const float2 x = fsubmul2(z[j], z[j + 1], base, base, a.k, a.k);
    const float2 y = fsubmul2(z[j + 2], z[j + 3], base, base, a.k, a.k);
    s0 = fadd2(s0, ex2(x.x), ex2(x.y));
    s1 = fadd2(s1, ex2(y.x), ex2(y.y));
  }
  s = (s0.x + s0.y) + (s1.x + s1.y);
  m = mn;
}

// 32 logits of one row to w (exp(z / T - lse) - q). A row without a target
// (w = 0) is exactly zero, whatever its logits hold.
__device__ __forceinline__ void grad32(float (&z)[32], int j0, const HeadTcArgs& a, Target& tg, float w, float lse) {
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    const float2 x = ffma2(z[j], z[j + 1], a.inv_t, -lse);
    z[j] = ex2(x.x * kLog2e) * w;
    z[j + 1] = ex2(x.y * kLog2e) * w;
  }
  if (w == 0.f) {
#pragma unroll
    for (int j = 0; j < 32; ++j) z[j] = 0.f;
  }
  while (__any_sync(0xffffffffu, (unsigned)tg.nid - (unsigned)j0 < 32u)) {
    const int at = (int)((unsigned)tg.nid - (unsigned)j0);
    const bool hit = (unsigned)at < 32u;
    const float qw = hit ? tg.nq * w : 0.f;
#pragma unroll
    for (int j = 0; j < 32; ++j) z[j] -= at == j ? qw : 0.f;
    if (hit) tg.next();
  }
}

// Column sums over the warp's 32 rows: 32 x 32 values, each step exchanging
// half of what is left with the lane 16, 8, ... away; lane j ends with column j
// in z[0] (31 shuffles instead of 160).
__device__ __forceinline__ void column_sums(float (&z)[32], int lane) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int j = 0; j < o; ++j) {
      const float mine = up ? z[j + o] : z[j], give = up ? z[j] : z[j + o];
      z[j] = mine + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
}

template <int MODE, bool BIAS, int HD_EPI_WARPS>
__global__ void __launch_bounds__(64 + 32 * HD_EPI_WARPS, 1)
    head_logits_kernel(const __grid_constant__ CUtensorMap tmH, const __grid_constant__ CUtensorMap tmW,
                       const __grid_constant__ CUtensorMap tmG, HeadTcArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  using Cfg = HdCfg<MODE, BIAS, HD_EPI_WARPS>;
  constexpr int COLS = Cfg::COLS;
  constexpr int HD_STAGES = Cfg::STAGES;
  uint8_t* out_stage = smem + HD_STAGES * HD_STAGE;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(out_stage + Cfg::OUT + Cfg::BIAS_BYTES + Cfg::ROWS);
  uint64_t* empty_bar = full_bar + HD_STAGES;
  uint64_t* accf_bar = empty_bar + HD_STAGES;  // [2]
  uint64_t* acce_bar = accf_bar + 2;           // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acce_bar + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank_u32();
  const bool leader = rank == 0;
  WaitCtx wc{abort_flag, a.err};

  if (threadIdx.x == 0) {
    for (int s = 0; s < HD_STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&accf_bar[b], 1);
      mbar_init(&acce_bar[b], 2 * HD_EPI_WARPS);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmH);
    tma_prefetch_desc(&tmW);
    if (MODE == kGrad) tma_prefetch_desc(&tmG);
  }
  if (warp == 1) {  // same warp in both CTAs, same destination offset
    tmem_alloc2(tmem_slot, HD_TMEM_COLS);
    tmem_relinquish2();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all2();  // both CTAs' barriers are initialised before any cross-CTA traffic
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  if (MODE == kGrad || !a.loss) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // not the last kernel
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const int num_tiles = a.tiles_m * a.tiles_n;
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  const int nk = (a.d + HD_BK - 1) / HD_BK;
  const int kGroup = a.group_m;
  auto coords = [&](int t, int& tm, int& tn) {
    const int per_group = kGroup * a.tiles_n;
    const int g = t / per_group, r = t - g * per_group;
    const int gsize = min(a.tiles_m - g * kGroup, kGroup);
    tm = g * kGroup + r % gsize;
    tn = r / gsize;
  };

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs)
    if (elect_one_lane()) {
      uint32_t fill = 0;
      for (int t = pair; t < num_tiles && !*abort_flag; t += npairs) {
        int tm, tn;
        coords(t, tm, tn);
        const int m0 = tm * 2 * HD_BM + (int)rank * HD_BM;        // this CTA's 128 rows of H
        const int n0 = tn * HD_BN + (int)rank * (HD_BN / 2);      // this CTA's 128 rows of W
        for (int kb = 0; kb < nk; ++kb, ++fill) {
          const int s = fill % HD_STAGES;
          if (!mbar_wait(&empty_bar[s], ((fill / HD_STAGES) & 1) ^ 1, wc)) break;
          uint8_t* sa = smem + s * HD_STAGE;
          if (leader) mbar_arrive_expect_tx(&full_bar[s], 2 * HD_STAGE);
          tma_load_2d_pair(sa, &tmH, &full_bar[s], kb * HD_BK, m0);
          tma_load_2d_pair(sa + HD_STAGE / 2, &tmW, &full_bar[s], kb * HD_BK, n0);
        }
        if (*abort_flag) break;
      }
      // This CTA's copies have landed once the MMAs that read them are done.
      const uint32_t first = fill > (uint32_t)HD_STAGES ? fill - HD_STAGES : 0;
      for (uint32_t f = first; f < fill; ++f) mbar_drain(&empty_bar[f % HD_STAGES], (f / HD_STAGES) & 1);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader only)
    if (leader && elect_one_lane()) {
      constexpr uint32_t idesc = make_idesc(1, 0, 0, 2 * HD_BM, HD_BN);
      uint32_t fill = 0, use = 0;
      for (int t = pair; t < num_tiles; t += npairs, ++use) {
        const int buf = use & 1;
        if (!mbar_wait(&acce_bar[buf], ((use >> 1) & 1) ^ 1, wc)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * HD_BN;
        bool ok = true;
        for (int kb = 0; kb < nk; ++kb, ++fill) {
          const int s = fill % HD_STAGES;
          if (!mbar_wait(&full_bar[s], (fill / HD_STAGES) & 1, wc)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + s * HD_STAGE), sb = sa + HD_STAGE / 2;
#pragma unroll
          for (int kk = 0; kk < HD_BK / 16; ++kk)
            mma2_f16_ss(d_tmem, sw128_desc(sa + kk * 32, 16, 1024), sw128_desc(sb + kk * 32, 16, 1024), idesc,
                        (kb > 0 || kk > 0) ? 1u : 0u);
          tc_commit2_mc(&empty_bar[s], 0x3);
        }
        if (!ok) break;
        tc_commit2_mc(&accf_bar[buf], 0x3);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue (the other warps, both CTAs)
    const int q = warp & 3;              // TMEM lane quarter this warp may access
    const int part = (warp - 2) >> 2;    // its columns of the tile
    uint8_t* st = out_stage + (warp - 2) * 4096;
    float* bias_s = reinterpret_cast<float*>(out_stage + Cfg::OUT) + (warp - 2) * COLS;
    float* rows_s = reinterpret_cast<float*>(out_stage + Cfg::OUT + Cfg::BIAS_BYTES);
    const bool whole = MODE == kStats && a.loss;  // this tile finishes its rows
    uint32_t issued = 0, use = 0;
    for (int t = pair; t < num_tiles; t += npairs, ++use) {
      const int buf = use & 1;
      int tm, tn;
      coords(t, tm, tn);
      const int row0 = tm * 2 * HD_BM + (int)rank * HD_BM + q * 32, row = row0 + lane;
      const int nbase = tn * HD_BN + part * COLS;  // first column of this warp, within the piece
      const bool row_ok = row < a.R;
      // the row's target entries from this warp's columns on
      Target tg{nullptr, nullptr, 0, 0, Target::kNone, Target::kNone, 0.f, 0.f};
      float w = 1.f, lse = 0.f;
      if (row_ok) {
        tg.ids = a.sid + (size_t)row * a.K;
        tg.qs = a.sq ? a.sq + (size_t)row * a.K : nullptr;
        tg.K = a.K;
        tg.start(a.start ? a.start[(size_t)row * a.slots + (a.c0 + nbase) / kHeadSlot - a.slot0] : 0);
        if (MODE == kGrad) {
          const bool live = a.live ? a.live[row] != 0.f : (tg.nid >= 0 && tg.nid < a.V);
          w = live ? (a.dloss ? a.dloss[row] : 1.f) : 0.f;
          lse = a.lse[row];
        }
      } else if (MODE == kGrad) {
        w = 0.f;
      }
      if constexpr (BIAS) {  // loaded while the accumulator is still being filled
#pragma unroll
        for (int j = lane; j < COLS; j += 32) bias_s[j] = nbase + j < a.n ? __ldg(a.bias + a.c0 + nbase + j) : 0.f;
        __syncwarp();
      }
      // where the quarter's warps meet below, one that gave up still comes
      const bool ok = mbar_wait(&accf_bar[buf], (use >> 1) & 1, wc);
      if (!ok && !whole) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + buf * HD_BN + part * COLS;
      float m = -INFINITY, s = 0.f, zt = 0.f;
#pragma unroll 1
      for (int c = ok ? 0 : COLS; c < COLS; c += 32) {
        float z[32];
        {
          uint32_t r[32];
          tmem_ld32(taddr + c, r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) z[j] = __uint_as_float(r[j]);
        }
        if (c + 32 == COLS) {  // this warp's last read of the accumulator
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (leader)
              mbar_arrive(&acce_bar[buf]);
            else
              mbar_arrive_remote_relaxed(&acce_bar[buf], 0);
          }
        }
        const int n0 = nbase + c;   // column within the piece
        const int j0 = a.c0 + n0;   // vocabulary id of column 0
        if (n0 >= a.n) continue;    // uniform: nothing of the piece in this chunk
        if constexpr (BIAS) {
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 b = *reinterpret_cast<const float4*>(bias_s + c + j);
            z[j] += b.x;
            z[j + 1] += b.y;
            z[j + 2] += b.z;
            z[j + 3] += b.w;
          }
        }
        if constexpr (MODE == kStats) {
          stats32(z, n0, j0, row, a, tg, m, s, zt);
        } else {
          grad32(z, j0, a, tg, w, lse);
          // 64 columns to a box; a half past the piece is not stored
          if (!(c & 32)) {  // the box staged before has left
            if (lane == 0 && issued) bulk_wait_read0();
            __syncwarp();
          }
#pragma unroll
          for (int u = 0; u < 4; ++u)
            *reinterpret_cast<uint4*>(st + lane * 128 + (((u + (c >> 3 & 4)) ^ (lane & 7)) << 4)) =
                make_uint4(pack_bf16x2(z[8 * u], z[8 * u + 1]), pack_bf16x2(z[8 * u + 2], z[8 * u + 3]),
                           pack_bf16x2(z[8 * u + 4], z[8 * u + 5]), pack_bf16x2(z[8 * u + 6], z[8 * u + 7]));
          if ((c & 32) || n0 + 32 >= a.n) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&tmG, st, nbase + (c & 64), row0);
              bulk_commit();
            }
            ++issued;
          }
          if (a.dbp) {
            column_sums(z, lane);
            if (row0 < a.R && n0 + lane < a.n) a.dbp[(size_t)(row0 >> 5) * a.n + n0 + lane] = z[0];
          }
        }
      }
      if (whole) {
        float* mine = rows_s + ((buf * HD_EPI_WARPS + warp - 2) * 32 + lane) * 3;
        mine[0] = m;
        mine[1] = s;
        mine[2] = zt;
        asm volatile("bar.sync %0, %1;" ::"r"(1 + q), "n"(8 * HD_EPI_WARPS) : "memory");
        if (part == 0 && row_ok) {  // joins the quarter's warps in column order
          constexpr int NEXT = 4 * 32 * 3;
#pragma unroll
          for (int i = 1; i < HD_EPI_WARPS / 4; ++i) m = fmaxf(m, mine[i * NEXT]);
          const float base = m == -INFINITY ? 0.f : m;
          s = 0.f;
#pragma unroll
          for (int i = 0; i < HD_EPI_WARPS / 4; ++i) s += mine[i * NEXT + 1] * expf((mine[i * NEXT] - base) * a.inv_t);
          const int id = a.sid[row];
          const bool has = id >= 0 && id < a.V;
          nll_row(m, s, has ? mine[id / COLS * NEXT + 2] : 0.f, has, a.inv_t, a.loss[row], a.lse_out[row]);
        }
      } else if (MODE == kStats && row_ok && nbase < a.n) a.part[(size_t)(nbase / COLS) * a.R + row] = make_float2(m, s);
    }
    if (MODE == kGrad && lane == 0) bulk_wait0();
  }

  // Neither CTA leaves (or frees TMEM) while its pair may still use its
  // shared memory or TMEM.
  tc_fence_before();
  __syncthreads();
  cluster_sync_all2();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc2(tmem_base, HD_TMEM_COLS);
  }
}

}  // namespace

int head_stat_cols(int d, bool bias) { return 4 * HD_BN / (many_warps(d, bias) ? kManyWarps : kFewWarps); }

// Logits of the piece [c0, c0 + n) of the vocabulary: row statistics
// (grad = false) or G (grad = true, into g with pitch ldg).
cudaError_t head_logits_tc(HeadTcArgs a, const void* H, int ldh, const void* W, int ldw, bool grad, void* g, int ldg,
                           cudaStream_t s) {
  CUtensorMap mh{}, mw{}, mg{};
  const __nv_bfloat16* wp = (const __nv_bfloat16*)W + (size_t)a.c0 * ldw;
  if (!encode_2d_bf16(&mh, H, a.d, a.R, (uint64_t)ldh * 2, HD_BK, HD_BM)) return cudaErrorInvalidValue;
  if (!encode_2d_bf16(&mw, wp, a.d, a.n, (uint64_t)ldw * 2, HD_BK, HD_BN / 2)) return cudaErrorInvalidValue;
  mg = mh;
  if (grad && !encode_2d_bf16(&mg, g, a.n, a.R, (uint64_t)ldg * 2, 64, 32)) return cudaErrorInvalidValue;
  a.tiles_m = (a.R + 2 * HD_BM - 1) / (2 * HD_BM);
  a.tiles_n = (a.n + HD_BN - 1) / HD_BN;
  // Row tiles are innermost, in groups as large as keep their rows of H (48 MB)
  // in L2 while the W tiles stream by: W is read from HBM once per group
  // (groups of 8 read it four times at R = 8192: 8192 x 65536 x 2048 training
  // 6.74 -> 6.58 ms, 4096 x 32768 x 1024 874 -> 863 us with one group).
  a.group_m = (int)std::min<long long>(a.tiles_m, std::max<long long>(8, (48ll << 20) / (2ll * HD_BM * 2 * a.d)));
  const int pairs = (int)std::min<long long>((long long)a.tiles_m * a.tiles_n, num_sms() / 2);
  auto run = [&](auto mode, auto bias, auto warps) {
    constexpr int M = decltype(mode)::value, EW = decltype(warps)::value;
    constexpr bool B = decltype(bias)::value != 0;
    using Cfg = HdCfg<M, B, EW>;
    static std::atomic<unsigned long long> done;
    const cudaError_t e = allow_smem(head_logits_kernel<M, B, EW>, Cfg::SMEM, done);
    if (e != cudaSuccess) return e;
    return launch_dependent(head_logits_kernel<M, B, EW>, 2 * pairs, Cfg::THREADS, Cfg::SMEM, 2, s, mh, mw, mg, a);
  };
  auto with_warps = [&](auto mode, auto bias) {
    return many_warps(a.d, a.bias != nullptr) ? run(mode, bias, IntC<kManyWarps>{}) : run(mode, bias, IntC<kFewWarps>{});
  };
  if (grad) return a.bias ? with_warps(IntC<kGrad>{}, IntC<1>{}) : with_warps(IntC<kGrad>{}, IntC<0>{});
  return a.bias ? with_warps(IntC<kStats>{}, IntC<1>{}) : with_warps(IntC<kStats>{}, IntC<0>{});
}

}  // namespace dgx
