// Block-scaled e4m3 GEMM for middling numbers of tokens:
//   out[m, n] = sum_kb a_s[m, kb] * w_s[n / 128, kb] * D_kb[m, n] (+ bias[n]),
//   D_kb[m, n] = sum_{k in block kb} a[m, k] * w[n, k]
//
// tcgen05.mma kind::f8f6f4 forms each block's D_kb as a fresh fp32 accumulator in
// tensor memory; the epilogue warps read it while the next blocks' MMAs run, and add
// it, times its scales, to fp32 totals in their registers. Tokens are the MMA's
// M = 128 rows (a TMEM lane, so an epilogue thread, is one token: its factor
// a_s * w_s is one scalar per block, one FMA per element), 128 output channels (one
// weight-scale block) its columns, 64 per epilogue warpgroup.
//
// Bound: a block's 32 KB of operands take 340 to 840 clocks to come from HBM or L2,
// its MMAs 256, but a wait on shared memory costs 270 to 340 while the tensor cores
// and TMA use it, and a fence 150. So four warps issue MMAs, each with its own
// accumulator, two produce and two wait for accumulators, all on alternate blocks.
//
// CTAs take whole tiles, or, where that leaves SMs idle, the k-blocks of all tiles end
// to end in one contiguous range per CTA (cb_gemm_common.cuh), as many CTAs as pay for
// the join (plan_split): parts of a cut tile are published as they end, and the tile's
// first contributor adds them in CTA order after a short bounded poll, else the last to
// arrive does. No CTA waits for one that may not run, and the bits do not depend on who
// adds.
//
// Warps: 0, 12 TMA producers; 1-3, 13 MMA issuers; 14-15 accumulator waiters; 4-11
// epilogue.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "cb_gemm_common.cuh"
#include "cb_internal.h"
#include "cb_ptx.cuh"
#include "fp8_block_out.cuh"

namespace cb {
namespace {

constexpr int kBM = 128, kBN = 128, kBK = 128;
constexpr int kStages = 6;
constexpr int kAcc = 4;  // accumulators in tensor memory, one per MMA issuer
constexpr int kThreads = 512;
// Registers: 512 x 128 at launch = 256 x 80 + 256 x 176. The epilogue holds 64 totals and
// an accumulator's 64 columns, or two parts' quarters in flight.
constexpr int kRegsLaunch = 128, kRegsFirst = 80, kRegsEpi = 176;
constexpr int kTC = 64;  // channels per epilogue warpgroup
constexpr int kHandBar = 2, kHandThreads = 32 + 256;
constexpr int kGroupM = 16;  // m-tiles that neighbouring CTAs share weight tiles over
constexpr uint32_t kTileBytes = 128 * kBK, kStageBytes = 2 * kTileBytes;

struct TcParams {
  int M, N, KB;
  int m_tiles, n_tiles;
  long long tiles;
  StreamK sk;
  const float* a_scale;
  long long as_sb, as_sm;
  const float* w_scale;
  long long ws_sb, ws_sn;
  const void* bias;
  int bias_dtype;
  long long bias_sb;
  void* out;
  int out_dtype;
  long long out_sb, out_sm;
  int unit;  // bytes of an output store
  float* partials;  // [grid][2][kBN][kBM]
  int* counters;
  int* status;
  unsigned long long dbg_wait_ns;  // failure-detection test hook: limit of a wait that expires (0: off)
};

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}

// (batch, m-tile, n-tile) of a tile: n fastest within groups of kGroupM m-tiles, so
// the tiles in flight together share both operands in L2.
__device__ __forceinline__ void tile_of(const TcParams& p, long long tile, int& b, int& mt, int& nt) {
  const long long per = static_cast<long long>(p.m_tiles) * p.n_tiles;
  b = static_cast<int>(tile / per);
  const int r = static_cast<int>(tile - b * per);
  const int span = kGroupM * p.n_tiles;
  const int grp = r / span, in = r - grp * span;
  const int rows = p.m_tiles - grp * kGroupM < kGroupM ? p.m_tiles - grp * kGroupM : kGroupM;
  nt = in / rows;
  mt = grp * kGroupM + (in - nt * rows);
}

// A unit (tile, k-block) of this CTA, advanced one or several at a time.
template <bool SPLIT>
struct Unit {
  long long tile;
  int kb, b, mt, nt;
  __device__ __forceinline__ Unit(const TcParams& p, int skip) {
    if (!SPLIT) {
      tile = blockIdx.x;
      kb = 0;
    } else {
      const long long g = p.sk.start(blockIdx.x);
      tile = g / p.KB;
      kb = static_cast<int>(g - tile * p.KB);
    }
    tile_of(p, tile, b, mt, nt);
    advance(p, skip);
  }
  __device__ __forceinline__ void advance(const TcParams& p, int n) {
    kb += n;
    if (kb < p.KB) return;
    do {
      kb -= p.KB;
      tile += SPLIT ? 1 : static_cast<int>(gridDim.x);
    } while (kb >= p.KB);
    if (tile < p.tiles) tile_of(p, tile, b, mt, nt);  // (past the CTA's last unit it is not used)
  }
};

// SPLIT: a contiguous range of k-blocks per CTA; else whole tiles cta, cta + grid, ...
template <bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
    block_gemm_tc_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                         const TcParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[kStages], empty_bar[kStages];
  __shared__ __align__(8) uint64_t tfull_bar[kAcc], tempty_bar[kAcc], drain_bar[kAcc];
  __shared__ uint32_t tmem_base_sh;
  __shared__ int abort_flag, sh_issued[2], sh_consumed[kAcc], sh_last[2];
  volatile int* abort_ptr = &abort_flag;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int units = SPLIT ? static_cast<int>(p.sk.start(blockIdx.x + 1) - p.sk.start(blockIdx.x))
                          : static_cast<int>(((p.tiles - 1 - blockIdx.x) / gridDim.x + 1) * p.KB);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < kAcc; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], 8);
      mbar_init(&drain_bar[a], 1);
      sh_consumed[a] = a;
    }
    sh_issued[0] = sh_issued[1] = 0;
    abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmap_a);
    prefetch_tmap(&tmap_w);
  }
  __syncwarp();
  if (warp == 1) {
    tmem_alloc(&tmem_base_sh, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_sh;

  if (warp < 4 || warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsFirst));
    if (warp == 0 || warp == 12) {
      // ---------------- TMA producers: the first ring pass by the lanes of warp 0, then units j, j + 2, ... ----------------
      const int j = warp == 0 ? 0 : 1;
      const uint64_t pol = policy_evict_normal();
      auto fill = [&](const Unit<SPLIT>& u, int stage) {
        mbar_arrive_expect_tx(&full_bar[stage], kStageBytes);
        uint8_t* dst = smem + stage * kStageBytes;
        tma_load_3d(dst, &tmap_a, &full_bar[stage], u.kb * kBK, u.mt * kBM, u.b, pol);
        tma_load_3d(dst + kTileBytes, &tmap_w, &full_bar[stage], u.kb * kBK, u.nt * kBN, u.b, pol);
      };
      const Unit<SPLIT> first(p, j == 0 && lane < kStages && lane < units ? lane : 0);
      Unit<SPLIT> u(p, kStages + j < units ? kStages + j : 0);
      pdl_wait_primary();
      if (threadIdx.x == 0) pdl_launch_dependents();
      __syncwarp();
      if (j == 0 && lane < kStages && lane < units) fill(first, lane);
      __syncwarp();
      if (lane == 0) {
        int i = kStages + j;
        for (; i < units; i += 2) {
          const int stage = i % kStages;
          if (!mbar_wait_quick(&empty_bar[stage], static_cast<uint32_t>((i / kStages - 1) & 1), abort_ptr, p.status)) break;
          fill(u, stage);
          u.advance(p, 2);
        }
        sh_issued[j] = i < units ? i : units;  // this warp's units below that are issued
      }
      __syncwarp();
    } else if (warp < 4 || warp == 13) {
      // ---------------- MMA issuers: accumulator j, units j, j + 4, ... ----------------
      const int j = warp == 13 ? 3 : warp - 1;
      pdl_wait_primary();
      int i = j;
      if (lane == 0) {
        const uint32_t idesc = idesc_e4m3_f32(kBM, kBN);
        const bool dead = j == 0 && p.dbg_wait_ns != 0 && !wait_counter(p.status + 1, 1, abort_ptr, p.status, p.dbg_wait_ns);
        for (; i < units && !dead; i += kAcc) {
          const int stage = i % kStages;
          if (!mbar_wait_quick(&tempty_bar[j], static_cast<uint32_t>((i / kAcc) & 1) ^ 1u, abort_ptr, p.status) ||
              !mbar_wait_quick(&full_bar[stage], static_cast<uint32_t>((i / kStages) & 1), abort_ptr, p.status))
            break;
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * kStageBytes), sw = sa + kTileBytes;
#pragma unroll
          for (int kk = 0; kk < kBK / 32; ++kk)
            mma_f8_ss(tmem + j * kBN, smem_desc_sw128(sa + kk * 32), smem_desc_sw128(sw + kk * 32), idesc, kk != 0);
          mma_commit(&tfull_bar[j]);
          mma_commit(&empty_bar[stage]);
        }
        sh_consumed[j] = i;  // first unit of this warp's that was not issued
        mma_commit(&drain_bar[j]);
      }
      // Every commit's arrival must land before the CTA exits: the MMAs' end, the last
      // use of each stage (waited for by the warp that issued it; after an expired wait at
      // the end, when all know what was issued) and the last hand-off.
      i = __shfl_sync(0xffffffffu, i, 0);
      if (lane == 31) mbar_wait_quick(&drain_bar[j], 0, nullptr, p.status);
      const int js = i - kAcc - kAcc * lane;
      if (lane < 2 && js >= 0 && js + kStages >= units)
        mbar_wait_quick(&empty_bar[js % kStages], static_cast<uint32_t>((js / kStages) & 1), nullptr, p.status);
      if (lane == 16 && i >= kAcc) mbar_wait_quick(&tfull_bar[j], static_cast<uint32_t>(((i - kAcc) / kAcc) & 1), nullptr, p.status);
      __syncwarp();
    } else if (warp >= 14) {
      // ---------------- accumulator waiters: hand over the units j, j + 2, ... ----------------
      const int j = warp - 14;
      pdl_wait_primary();
      for (int i = j; i < units; i += 2) {
        bool ok = true;
        if (lane == 0) ok = mbar_wait_quick(&tfull_bar[i % kAcc], static_cast<uint32_t>((i / kAcc) & 1), abort_ptr, p.status);
        ok = __all_sync(0xffffffffu, ok);
        if (named_bar_or(kHandBar + j, kHandThreads, !ok)) break;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpi));
    // ---------------- epilogue: one token per thread, 64 channels per warpgroup ----------------
    const int group = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const int leader = 128 + group * 128, ebar = 4 + group;
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + group * kTC;
    int* const counters = p.counters + group * (kMaxGrid / 2);  // one counter per group: groups finish on their own
    Unit<SPLIT> u(p, 0);
    // contributors of the tiles that this CTA's range begins and ends in
    long long cc_a = 0, cc_z = 0;
    if (SPLIT) {
      cc_a = cut_contributors(p.sk.total, p.sk.grid, p.KB, u.tile);
      cc_z = cut_contributors(p.sk.total, p.sk.grid, p.KB, (p.sk.start(blockIdx.x + 1) - 1) / p.KB);
    }
    pdl_wait_primary();
    uint8_t* const stg = smem + kStages * kStageBytes + (warp - 4) * kOutBytes;
    float sum[kTC];
    // Part of CTA c of a cut tile: slot 1 where the tile is cut by the end of c's range
    // (its first contributor), 0 where c's range began inside it. Token fastest.
    auto slot = [&](int c, int c_first) {
      return p.partials + (static_cast<long long>(c) * 2 + (c == c_first ? 1 : 0)) * (kBN * kBM) + group * kTC * kBM + row;
    };
    // sum = the parts of c_first .. c_last in order; the first is in sum if `held`. A
    // quarter of the channels at a time, each part's requested two ahead of its addition.
    auto add_parts = [&](int c_first, int c_last, bool held, bool row_live) {
      constexpr int kAt = 16, kParts = 2;
      const int from = held ? c_first + 1 : c_first;
#pragma unroll
      for (int x0 = 0; x0 < kTC; x0 += kAt) {
        float v[kAt], buf[kParts][kAt];
#pragma unroll
        for (int x = 0; x < kAt; ++x) v[x] = 0.0f + (held ? sum[x0 + x] : 0.0f);
        auto load = [&](int c, float (&to)[kAt]) {
          const float* src = slot(c, c_first) + x0 * kBM;
          const bool on = row_live && c <= c_last;
#pragma unroll
          for (int x = 0; x < kAt; ++x) to[x] = on ? __ldcg(src + x * kBM) : 0.0f;
        };
#pragma unroll
        for (int q = 0; q < kParts; ++q) load(from + q, buf[q]);
        for (int c = from; c <= c_last; c += kParts) {
#pragma unroll
          for (int q = 0; q < kParts; ++q) {
#pragma unroll
            for (int x = 0; x < kAt; ++x) v[x] += buf[q][x];
            load(c + q + kParts, buf[q]);
          }
        }
#pragma unroll
        for (int x = 0; x < kAt; ++x) sum[x0 + x] = v[x];
      }
    };
    auto store_out = [&](int b, int mt, int nt) {
      const int m0 = mt * kBM + quarter * 32, n0 = nt * kBN + group * kTC;
      if (m0 >= p.M || n0 >= p.N) return;
      if (p.bias) add_bias(sum, p.bias, p.bias_dtype, b * p.bias_sb + n0, p.N - n0, lane);
      const int es = p.out_dtype == CB_DTYPE_F32 ? 4 : 2;
      store_rows(stg, sum, static_cast<char*>(p.out) + (b * p.out_sb + static_cast<long long>(m0) * p.out_sm + n0) * es, p.out_sm * es,
                 p.M - m0, p.N - n0, p.out_dtype, p.unit, lane);
    };
    // After an expired wait the work is skipped, but every named barrier of a group is
    // still reached by all of its warps, and the hand-over barriers until both waiters
    // have left.
    bool live = true;
    // Stores this CTA's part; after the barrier the leader's fence covers all of them.
    auto publish = [&](int c_first, bool row_live) {
      if (live && row_live) {
        float* dst = slot(blockIdx.x, c_first);
#pragma unroll
        for (int c = 0; c < kTC; ++c) dst[c * kBM] = sum[c];
      }
      named_bar_sync(ebar, 128);
      if (threadIdx.x == leader) __threadfence();
    };
    long long pend_tile = -1;  // cut tile whose count this CTA bumped without looking at the result
    int pend_old = 0, pend_first = 0, pend_last = 0;
    int i = 0;
    while (i < units) {
      const int kb0 = u.kb;
      const int here = p.KB - kb0 < units - i ? p.KB - kb0 : units - i;  // units of this segment
      const int m = u.mt * kBM + row;
      const bool row_live = m < p.M;
      const bool some = u.mt * kBM + quarter * 32 < p.M && u.nt * kBN + group * kTC < p.N;
      const float* as = p.a_scale + u.b * p.as_sb + (row_live ? static_cast<long long>(m) * p.as_sm : 0) + kb0;
      const float* ws = p.w_scale + u.b * p.ws_sb + u.nt * p.ws_sn + kb0;
#pragma unroll
      for (int c = 0; c < kTC; ++c) sum[c] = 0.0f;
      float next = __ldg(as) * __ldg(ws);
      for (int k = 0; k < here && live; ++k) {
        const int n = i + k, acc = n % kAcc;
        const float f = row_live ? next : 0.0f;
        if (k + 1 < here) next = __ldg(as + k + 1) * __ldg(ws + k + 1);
        live = !named_bar_or(kHandBar + (n & 1), kHandThreads, false);
        if (!live) {
          // the other waiter comes to the next unit's barrier, whatever it has seen: it leaves from there
          if (n + 1 < units) named_bar_or(kHandBar + ((n + 1) & 1), kHandThreads, true);
          break;
        }
        if (some) {
          tc_fence_after();
          uint32_t r[2][32];
          tmem_ld32(lane_addr + acc * kBN, r[0]);
          tmem_ld32(lane_addr + acc * kBN + 32, r[1]);
          tmem_ld_wait();
#pragma unroll
          for (int x = 0; x < kTC; ++x) sum[x] = fmaf(__uint_as_float(r[x / 32][x % 32]), f, sum[x]);
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty_bar[acc]);
      }
      bool emit = live;
      if (SPLIT && here != p.KB) {
        const long long cc = i == 0 ? cc_a : cc_z;
        const int c_first = static_cast<int>(cc & 0xffffffffLL), c_last = static_cast<int>(cc >> 32);
        const int n_parts = c_last - c_first + 1, me = static_cast<int>(blockIdx.x);
        if (me != c_first) {
          // looked at again at the end
          publish(c_first, row_live);
          if (threadIdx.x == leader && !*abort_ptr) pend_old = atomicAdd(&counters[c_first], 1);
          pend_tile = u.tile, pend_first = c_first, pend_last = c_last;
          emit = false;
        } else {
          // every warp looks first (usually all parts are there); the leader polls on
          bool last = p.sk.first_poll_ns && ld_acquire_gpu(&counters[c_first]) == n_parts - 1;
          last = !named_bar_or(ebar, 128, !last);
          if (!last && p.sk.first_poll_ns) {
            if (threadIdx.x == leader) sh_last[group] = poll_counter(&counters[c_first], n_parts - 1, abort_ptr, p.sk.first_poll_ns);
            named_bar_sync(ebar, 128);
            last = sh_last[group] != 0;
            if (last) __threadfence();
          }
          if (!last) {
            publish(c_first, row_live);
            if (threadIdx.x == leader) sh_last[group] = !*abort_ptr && atomicAdd(&counters[c_first], 1) == n_parts - 1;
            named_bar_sync(ebar, 128);
            last = sh_last[group] != 0;
            if (last) __threadfence();
          }
          if (last) {
            if (live) add_parts(c_first, c_last, true, row_live);
            if (threadIdx.x == leader) counters[c_first] = 0;  // the next launch starts from zero
          }
          emit = emit && last;
          named_bar_sync(ebar, 128);  // sh_last is read by all before it is written again
        }
      }
      if (emit) store_out(u.b, u.mt, u.nt);
      i += here;
      u.advance(p, here);
    }
    // The part published without looking: if it was the tile's last to arrive (the
    // first contributor gave up its poll), the tile is reduced here.
    if (SPLIT && pend_tile >= 0) {
      if (threadIdx.x == leader) sh_last[group] = !*abort_ptr && pend_old == pend_last - pend_first;
      named_bar_sync(ebar, 128);
      if (sh_last[group]) {
        __threadfence();
        int b, mt, nt;
        tile_of(p, pend_tile, b, mt, nt);
        add_parts(pend_first, pend_last, false, mt * kBM + row < p.M);
        if (threadIdx.x == leader) counters[pend_first] = 0;
        store_out(b, mt, nt);
      }
    }
  }

  __syncthreads();
  if (warp == 0) {
    if (abort_flag && lane < kStages) {
      // the last use of stage `lane`: unit k of issuer j, the stage again every 3 of its units
      int last = -1;
      for (int j = 0; j < kAcc; ++j)
        for (int x = 1, k = sh_consumed[j] - kAcc; x <= kStages / 2 && k >= 0; ++x, k -= kAcc)
          if (k % kStages == lane && k > last) last = k;
      if (last >= 0) mbar_wait_quick(&empty_bar[lane], static_cast<uint32_t>((last / kStages) & 1), nullptr, p.status);
    }
    __syncwarp();
    if (lane == 0 && abort_flag) {
      // loads issued but never consumed must land before the CTA exits
      for (int j = 0; j < kAcc; ++j)
        for (int k = sh_consumed[j]; k < sh_issued[k & 1] || k < (kStages < units ? kStages : units); k += kAcc)
          mbar_wait_quick(&full_bar[k % kStages], (k / kStages) & 1, nullptr, p.status);
    }
    __syncwarp();
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Blocks per CTA with whole tiles, and with a split. A join takes as long as 14 blocks
// (0.3 us each) and 3 more for a third part on: with K = 8192, 128 x 1024 takes 27.1 us
// whole, 20.7 / 17.0 / 17.4 / 18.5 in 2 / 4 / 6 / 8 parts a tile and 28.2 on all SMs;
// 1000 x 1000 27.9 whole, 23.1 in two, 23.8 on all; with K = 2048, 100 x 2000 9.5 whole
// and 12.0 in two.
constexpr JoinCost kJoin = {11, 1, 3};
long long tiles_of(const BlockGemmArgs& L) { return L.batch * ((L.M + kBM - 1) / kBM) * ((L.N + kBN - 1) / kBN); }
long long whole_blocks(const BlockGemmArgs& L, int sms) { return (tiles_of(L) + sms - 1) / sms * ((L.K + kBK - 1) / kBK); }
SplitPlan split_plan(const BlockGemmArgs& L, int sms) { return plan_split(tiles_of(L), (L.K + kBK - 1) / kBK, sms, kJoin); }

}  // namespace

long long block_gemm_tc_blocks(const BlockGemmArgs& L) {
  const int sms = sm_count();
  if (sms <= 0) return 0;
  const long long w = whole_blocks(L, sms), s = split_plan(L, sms).cost;
  return w < s ? w : s;
}

size_t block_gemm_tc_workspace() {
  int sms = sm_count();
  if (sms <= 0) sms = 148;
  return workspace_need(sms, static_cast<size_t>(kBM) * kBN * sizeof(float));
}

int launch_block_gemm_tc(const BlockGemmArgs& L, cudaStream_t stream) {
  int sms = sm_count();
  if (sms <= 0) return CB_ERR_CUDA;
  if (sms > kMaxGrid / 2) sms = kMaxGrid / 2;  // two counters a CTA
  TcParams p = {};
  p.M = static_cast<int>(L.M), p.N = static_cast<int>(L.N), p.KB = static_cast<int>((L.K + kBK - 1) / kBK);
  p.m_tiles = (p.M + kBM - 1) / kBM;
  p.n_tiles = (p.N + kBN - 1) / kBN;
  p.tiles = L.batch * static_cast<long long>(p.m_tiles) * p.n_tiles;
  const long long total = p.tiles * p.KB;
  const SplitPlan split = split_plan(L, sms);
  const bool whole = whole_blocks(L, sms) <= split.cost;
  const int grid = !whole ? split.grid : p.tiles < sms ? static_cast<int>(p.tiles) : sms;
  p.sk.total = total;
  p.sk.grid = grid;
  p.sk.kb_per_tile = p.KB;
  p.sk.first_poll_ns = debug_force_last_arriver() ? 0 : kFirstPollNs;
  p.dbg_wait_ns = debug_wait_ns();
  p.a_scale = L.a_scale, p.as_sb = L.as_sb, p.as_sm = L.as_sm;
  p.w_scale = L.w_scale, p.ws_sb = L.ws_sb, p.ws_sn = L.ws_sn;
  p.bias = L.bias, p.bias_dtype = L.bias_dtype, p.bias_sb = L.b_sb;
  p.out = L.out, p.out_dtype = L.out_dtype, p.out_sb = L.o_sb, p.out_sm = L.o_sm;
  p.unit = out_unit(L);
  Workspace ws = carve_workspace(L.workspace, grid);
  p.partials = static_cast<float*>(ws.partials);
  p.counters = ws.counters;
  p.status = ws.status;
  CUtensorMap ta, tw;
  int st = encode_tmap_3d(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, L.a, L.K, L.M, L.batch, L.a_sm, L.a_sb, kBK, kBM,
                          CU_TENSOR_MAP_SWIZZLE_128B);
  if (st != CB_OK) return st;
  st = encode_tmap_3d(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, L.w, L.K, L.N, L.batch, L.w_sn, L.w_sb, kBK, kBN,
                      CU_TENSOR_MAP_SWIZZLE_128B);
  if (st != CB_OK) return st;
  constexpr size_t smem = kStages * kStageBytes + 8 * kOutBytes + 1024;
  const auto kernel = whole ? block_gemm_tc_kernel<false> : block_gemm_tc_kernel<true>;
  static thread_local int configured_dev[2] = {-1, -1};
  int dev = 0;
  cudaGetDevice(&dev);
  if (configured_dev[whole] != dev) {
    // the warpgroups' register exchange counts on the launch's registers
    cudaFuncAttributes attr;
    if (cudaFuncGetAttributes(&attr, kernel) != cudaSuccess) return CB_ERR_CUDA;
    if (attr.numRegs != kRegsLaunch) return CB_ERR_UNSUPPORTED;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess)
      return CB_ERR_CUDA;
    configured_dev[whole] = dev;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, ta, tw, p));
}

}  // namespace cb
