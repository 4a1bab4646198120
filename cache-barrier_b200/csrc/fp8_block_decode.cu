// Block-scaled e4m3 GEMM for few tokens (decode): out[m, n], M <= 64.
//
// Bound: HBM on the weights (1 byte a weight, 2 M flops). The weight tile is the
// MMA's M = 128 operand (a TMEM lane, so an epilogue thread, is one output channel)
// and the tokens are its TN columns, so a 128-element block of K is one 16 KB TMA
// tile of weights and a fresh accumulator of only TN columns; eight of those form a
// ring in tensor memory, deep enough that the round trip MMA -> epilogue -> MMA never
// stops the weight stream. The epilogue adds each, times a_s[m, kb] * w_s[n / 128, kb],
// to fp32 totals in registers.
//
// The (128 channels, k-block) units of all tiles are laid end to end and dealt to the
// CTAs (at most one per SM, as many as pay for the join: plan_split) in equal contiguous
// ranges; cut tiles are reduced as
// cb_gemm_common.cuh describes (parts published early, the first contributor adds
// them in CTA order after a short bounded poll, else the last to arrive does), so no
// CTA waits for one that may not run, and the bits do not depend on who adds.
//
// What a block costs each role is latency: 340 clocks for an mbarrier wait and about
// 100 for each other step on shared memory while the tensor cores and TMA use it (so
// 650 for the producer's step, 760 for waiting and laying out a block's factors),
// against 700 clocks of HBM time per 16 KB. So each role that touches shared memory
// has two warps on alternate blocks, and the epilogue warps, which only meet the
// accumulator waiters at a named barrier, read tensor memory and add.
//
// Streaming the weights into mma.sync fragments instead (registers, f16 conversion,
// two CTAs of eight warps per SM) took 22 us at K = N = 8192, M = 1 and 53 us at
// M = 32: conversions, addresses and fragment loads cost 240 instructions per warp
// and 2 KB.
//
// Warps: 0 and the last but one TMA producers, 1-2 MMA issuers, 3 and the last
// accumulator waiters, 4.. epilogue: four warps up to 16 tokens, two groups of four, each
// with half of the tokens, above.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "cb_gemm_common.cuh"
#include "cb_internal.h"
#include "cb_ptx.cuh"
#include "fp8_block.h"

namespace cb {
namespace {

constexpr int kBlk = 128;
constexpr int kAcc = 8;                    // accumulator ring
constexpr int kHandBar = 2;                // named barriers 2, 3: the block's accumulator and factors are ready
template <int TN>
constexpr int kGroups = TN > 16 ? 2 : 1;
template <int TN>
constexpr int kThreads = 192 + 128 * kGroups<TN>;
// Up to 16 tokens a CTA takes half an SM's shared memory and registers, so that the
// next kernel's CTAs (one per SM here too) can start under programmatic dependent
// launch: their set-up and first L2 prefetches run while this kernel ends.
template <int TN>
constexpr int kPerSm = TN > 16 ? 1 : 2;
constexpr uint32_t kWBytes = kBlk * kBlk;  // weight tile of a unit

struct DecodeParams {
  int M, N, KB, n_tiles;
  int stages;
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
  float* partials;    // [grid][2][TN][128]
  int* counters;
  int* status;
  unsigned long long dbg_wait_ns;  // failure-detection test hook: limit of a wait that expires (0: off)
};

// A unit's place, advanced without division.
struct Unit {
  int kb, nt, b;
  __device__ __forceinline__ Unit(const DecodeParams& p, long long u) {
    const long long tile = u / p.KB;
    kb = static_cast<int>(u - tile * p.KB);
    b = static_cast<int>(tile / p.n_tiles);
    nt = static_cast<int>(tile - static_cast<long long>(b) * p.n_tiles);
  }
  __device__ __forceinline__ void next(const DecodeParams& p) {
    if (++kb == p.KB) {
      kb = 0;
      if (++nt == p.n_tiles) nt = 0, ++b;
    }
  }
};

__device__ __forceinline__ void tma_prefetch_3d(const CUtensorMap* map, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}

template <int TN>
__global__ void __launch_bounds__(kThreads<TN>, kPerSm<TN>)
    block_gemm_decode_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_a,
                             const DecodeParams p) {
  constexpr uint32_t kABytes = TN * kBlk, kStage = kWBytes + kABytes;
  constexpr int kHandThreads = 32 + 128 * kGroups<TN>;  // an accumulator waiter and the epilogue
  constexpr int kWarp1 = kThreads<TN> / 32 - 2;         // the second producer; kWarp1 + 1 the second waiter
  constexpr uint32_t kCols = kAcc * TN < 32 ? 32 : kAcc * TN;
  static_assert(kCols <= 512 && (kCols & (kCols - 1)) == 0, "the ring must fit tensor memory");

  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[kMaxStages], empty_bar[kMaxStages];
  __shared__ __align__(8) uint64_t tfull_bar[kAcc], tempty_bar[kAcc], drain_bar[2];
  __shared__ uint32_t tmem_base_sh;
  __shared__ int abort_flag, sh_issued[2], sh_consumed[2], sh_last[kGroups<TN>];
  __shared__ __align__(16) float sh_factor[4][TN];  // a_s * w_s of a unit's tokens
  volatile int* abort_ptr = &abort_flag;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = p.stages;
  const long long u0 = p.sk.start(blockIdx.x);
  const int units = static_cast<int>(p.sk.start(blockIdx.x + 1) - u0);
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < kAcc; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], 4 * kGroups<TN>);
    }
    for (int j = 0; j < 2; ++j) {
      mbar_init(&drain_bar[j], 1);
      sh_consumed[j] = j;
      sh_issued[j] = j;
    }
    abort_flag = 0;
    fence_mbar_init();
  }
  // Places of each role's units (64-bit divisions) before the wait for the kernel
  // before this one. The first weight tiles may go to L2 meanwhile (a hint: nothing is
  // read yet, so that kernel may still write them).
  const uint64_t pol_w = policy_evict_first(), pol_a = policy_evict_last();
  const Unit first(p, u0 + (warp == 0 && lane < units ? lane : 0));
  Unit steady(p, u0);
  if (warp == 0 || warp == kWarp1) steady = Unit(p, u0 + S + (warp == 0 ? 0 : 1));
  if (warp == 0 && lane < S && lane < units) tma_prefetch_3d(&tmap_w, first.kb * kBlk, first.nt * kBlk, first.b);
  __syncwarp();
  if (warp == 1) {
    tmem_alloc(&tmem_base_sh, kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_sh;
  if (warp < 4 || warp >= kWarp1) pdl_wait_primary();  // the epilogue warps have more to do first
  if (threadIdx.x == 0) pdl_launch_dependents();
  __syncwarp();

  if (warp == 0 || warp == kWarp1) {
    // ---------------- TMA producers: the first ring pass by the lanes of warp 0, then units j, j + 2, ... ----------------
    const int j = warp == 0 ? 0 : 1;
    auto fill = [&](const Unit& u, int stage) {
      mbar_arrive_expect_tx(&full_bar[stage], kStage);
      uint8_t* dst = smem + stage * kStage;
      tma_load_3d(dst, &tmap_w, &full_bar[stage], u.kb * kBlk, u.nt * kBlk, u.b, pol_w);
      tma_load_3d(dst + kWBytes, &tmap_a, &full_bar[stage], u.kb * kBlk, 0, u.b, pol_a);
    };
    if (j == 0 && lane < S && lane < units) fill(first, lane);
    __syncwarp();
    if (lane == 0) {
      // S is even, so each stage belongs to one producer and one MMA issuer
      int i = S + j, stage = j;
      uint32_t phase = 0;
      for (; i < units; i += 2) {
        if (!mbar_wait_quick(&empty_bar[stage], phase, abort_ptr, p.status)) break;
        fill(steady, stage);
        steady.next(p);
        steady.next(p);
        stage += 2;
        if (stage >= S) stage -= S, phase ^= 1u;
      }
      sh_issued[j] = i < units ? i : units;  // this warp's units below that are issued
    }
    __syncwarp();
  } else if (warp < 3) {
    // ---------------- MMA issuers: warp 1 + j takes the units j, j + 2, ... ----------------
    const int j = warp - 1;
    int i = j;
    if (lane == 0) {
      const uint32_t idesc = idesc_e4m3_f32(kBlk, TN);
      int stage = j;
      uint32_t phase = 0;
      const bool dead = j == 0 && p.dbg_wait_ns != 0 && !wait_counter(p.status + 1, 1, abort_ptr, p.status, p.dbg_wait_ns);
      for (; i < units && !dead; i += 2) {
        const int acc = i % kAcc;
        if (!mbar_wait_quick(&tempty_bar[acc], static_cast<uint32_t>((i / kAcc) & 1) ^ 1u, abort_ptr, p.status) ||
            !mbar_wait_quick(&full_bar[stage], phase, abort_ptr, p.status))
          break;
        tc_fence_after();
        const uint32_t sw = smem_u32(smem + stage * kStage), sa = sw + kWBytes;
#pragma unroll
        for (int kk = 0; kk < kBlk / 32; ++kk)
          mma_f8_ss(tmem + acc * TN, smem_desc_sw128(sw + kk * 32), smem_desc_sw128(sa + kk * 32), idesc, kk != 0);
        mma_commit(&tfull_bar[acc]);
        mma_commit(&empty_bar[stage]);
        stage += 2;
        if (stage >= S) stage -= S, phase ^= 1u;
      }
      sh_consumed[j] = i;  // first unit of this warp's that was not issued
      mma_commit(&drain_bar[j]);
    }
    // Every commit's arrival must land before the CTA exits: the MMAs' end, this
    // warp's last stage releases and its last accumulator hand-offs.
    i = __shfl_sync(0xffffffffu, i, 0);
    if (lane == 31) mbar_wait_quick(&drain_bar[j], 0, nullptr, p.status);
    const int js = i - 2 - 2 * lane;
    if (2 * lane < S && js >= 0) mbar_wait_quick(&empty_bar[js % S], static_cast<uint32_t>((js / S) & 1), nullptr, p.status);
    const int ja = i - 2 - 2 * (lane - 16);
    if (lane >= 16 && lane < 16 + kAcc / 2 && ja >= 0)
      mbar_wait_quick(&tfull_bar[ja % kAcc], static_cast<uint32_t>((ja / kAcc) & 1), nullptr, p.status);
    __syncwarp();
  } else if (warp == 3 || warp == kWarp1 + 1) {
    // ---------------- accumulator waiters: factors and hand-over of units j, j + 2, ... ----------------
    constexpr int kPer = (TN + 31) / 32;  // tokens per lane
    const int j = warp == 3 ? 0 : 1;
    Unit u = steady;
    if (j) u.next(p);
    float next[kPer];
    auto load = [&] {
      const float w = __ldg(p.w_scale + u.b * p.ws_sb + u.nt * p.ws_sn + u.kb);
#pragma unroll
      for (int x = 0; x < kPer; ++x) {
        const int m = x * 32 + lane;
        next[x] = m < p.M ? __ldg(p.a_scale + u.b * p.as_sb + m * p.as_sm + u.kb) * w : 0.0f;
      }
    };
    if (j < units) load();
    for (int i = j; i < units; i += 2) {
      // slot i & 3 was last read for unit i - 4, before its readers came to the barrier of unit i - 2
#pragma unroll
      for (int x = 0; x < kPer; ++x)
        if (x * 32 + lane < TN) sh_factor[i & 3][x * 32 + lane] = next[x];
      u.next(p);
      u.next(p);
      if (i + 2 < units) load();
      bool ok = true;
      if (lane == 0)
        ok = mbar_wait_quick(&tfull_bar[i % kAcc], static_cast<uint32_t>((i / kAcc) & 1), abort_ptr, p.status);
      ok = __all_sync(0xffffffffu, ok);
      if (named_bar_or(kHandBar + j, kHandThreads, !ok)) break;
    }
  } else if (warp >= 4) {
    // ---------------- epilogue: one output channel per thread, TC tokens per group ----------------
    constexpr int TC = TN / kGroups<TN>;
    const int group = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const int leader = 128 + group * 128, ebar = 4 + group;
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + group * TC;
    const int M = p.M - group * TC < TC ? p.M - group * TC : TC;  // this group's tokens (none: it only keeps the barriers)
    // After an expired wait the work is skipped, but every named barrier of a group is
    // still reached by all of its warps, and the hand-over barriers until both waiters
    // have left.
    bool live = true;
    Unit u = steady;
    int i = 0;
    long long pend_tile = -1;  // cut tile whose count this CTA bumped without looking at the result
    int pend_old = 0, pend_first = 0, pend_last = 0;
    // contributors of the tiles that this CTA's range begins and ends in
    const long long tile_a = static_cast<long long>(steady.b) * p.n_tiles + steady.nt;
    const long long tile_z = (u0 + units - 1) / p.KB;
    const long long cc_a = cut_contributors(p.sk.total, p.sk.grid, p.KB, tile_a);
    const long long cc_z = cut_contributors(p.sk.total, p.sk.grid, p.KB, tile_z);
    pdl_wait_primary();
    float sum[TC];
    auto store_out = [&](int b, int nt) {
      const int ch = nt * kBlk + row;
      if (ch >= p.N) return;
      const float bias = p.bias ? load_elem(p.bias, p.bias_dtype, b * p.bias_sb + ch) : 0.0f;
      const long long base = b * p.out_sb + ch + static_cast<long long>(group * TC) * p.out_sm;
      auto put = [&](auto* out, auto cvt) {
        out += base;
#pragma unroll
        for (int m = 0; m < TC; ++m)
          if (m < M) out[m * p.out_sm] = cvt(p.bias ? sum[m] + bias : sum[m]);
      };
      if (p.out_dtype == CB_DTYPE_BF16)
        put(static_cast<__nv_bfloat16*>(p.out), [](float v) { return __float2bfloat16_rn(v); });
      else if (p.out_dtype == CB_DTYPE_F16)
        put(static_cast<__half*>(p.out), [](float v) { return __float2half_rn(v); });
      else
        put(static_cast<float*>(p.out), [](float v) { return v; });
    };
    // Part of CTA c of a cut tile: slot 1 where the tile is cut by the end of c's
    // range (its first contributor), 0 where c's range began inside it.
    auto slot = [&](int c, int c_first) {
      return p.partials + (static_cast<long long>(c) * 2 + (c == c_first ? 1 : 0)) * (TN * kBlk) + group * TC * kBlk + row;
    };
    // sum = the parts of c_first .. c_last in order; the first is in sum if `held`
    auto add_parts = [&](int c_first, int c_last, bool held) {
      constexpr int kStep = 8, kAhead = 4;  // tokens and parts whose loads are in flight together
#pragma unroll
      for (int c = 0; c < TC; c += kStep) {
        if (c >= M) break;
        float v[kStep];
#pragma unroll
        for (int x = 0; x < kStep; ++x) v[x] = 0.0f + (held ? sum[c + x] : 0.0f);
        for (int q0 = held ? c_first + 1 : c_first; q0 <= c_last; q0 += kAhead) {
          float part[kAhead][kStep];
#pragma unroll
          for (int q = 0; q < kAhead; ++q) {
            const float* src = slot(q0 + q <= c_last ? q0 + q : c_last, c_first) + c * kBlk;
#pragma unroll
            for (int x = 0; x < kStep; ++x) part[q][x] = c + x < M ? __ldcg(src + x * kBlk) : 0.0f;
          }
#pragma unroll
          for (int q = 0; q < kAhead; ++q)
            if (q0 + q <= c_last) {
#pragma unroll
              for (int x = 0; x < kStep; ++x) v[x] += part[q][x];
            }
        }
#pragma unroll
        for (int x = 0; x < kStep; ++x) sum[c + x] = v[x];
      }
    };
    // Stores this CTA's part; after the barrier the leader's fence covers all of them.
    auto publish = [&](int c_first) {
      if (live) {
        float* dst = slot(blockIdx.x, c_first);
#pragma unroll
        for (int c = 0; c < TC; ++c)
          if (c < M) dst[c * kBlk] = sum[c];
      }
      named_bar_sync(ebar, 128);
      if (threadIdx.x == leader) __threadfence();
    };
    // one counter per group: groups finish on their own
    int* const counters = p.counters + group * kMaxGrid / 2;
    while (i < units) {
      const int kb0 = u.kb;
      const int here = p.KB - kb0 < units - i ? p.KB - kb0 : units - i;  // units of this segment
#pragma unroll
      for (int c = 0; c < TC; ++c) sum[c] = 0.0f;
      for (int k = 0; k < here && live; ++k) {
        const int n = i + k, acc = n % kAcc;
        live = !named_bar_or(kHandBar + (n & 1), kHandThreads, false);
        if (!live) {
          // the other waiter comes to the next unit's barrier, whatever it has seen: it leaves from there
          if (n + 1 < units) named_bar_or(kHandBar + ((n + 1) & 1), kHandThreads, true);
          break;
        }
        tc_fence_after();
        uint32_t r[TC / 16][16];
#pragma unroll
        for (int c = 0; c < TC / 16; ++c)
          if (c * 16 < M) tmem_ld16(lane_addr + acc * TN + c * 16, r[c]);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty_bar[acc]);
        const float* factor = sh_factor[n & 3] + group * TC;
#pragma unroll
        for (int c = 0; c < TC; c += 4) {
          if (c < M) {
            const float4 f = *reinterpret_cast<const float4*>(factor + c);
            sum[c] = fmaf(__uint_as_float(r[c / 16][c % 16]), f.x, sum[c]);
            sum[c + 1] = fmaf(__uint_as_float(r[c / 16][c % 16 + 1]), f.y, sum[c + 1]);
            sum[c + 2] = fmaf(__uint_as_float(r[c / 16][c % 16 + 2]), f.z, sum[c + 2]);
            sum[c + 3] = fmaf(__uint_as_float(r[c / 16][c % 16 + 3]), f.w, sum[c + 3]);
          }
        }
      }
      bool emit = live;
      if (here != p.KB) {
        const long long tile = static_cast<long long>(u.b) * p.n_tiles + u.nt;
        const long long cc = i == 0 ? cc_a : cc_z;
        const int c_first = static_cast<int>(cc & 0xffffffffLL), c_last = static_cast<int>(cc >> 32);
        const int n_parts = c_last - c_first + 1, me = static_cast<int>(blockIdx.x);
        if (me != c_first) {
          // published at the start or the middle of the tile's work; looked at again at the end
          publish(c_first);
          if (threadIdx.x == leader && !*abort_ptr) pend_old = atomicAdd(&counters[c_first], 1);
          pend_tile = tile, pend_first = c_first, pend_last = c_last;
          emit = false;
        } else {
          // every warp looks first (usually all parts are there); the leader polls on
          bool last = p.sk.first_poll_ns && ld_acquire_gpu(&counters[c_first]) == n_parts - 1;
          last = named_bar_or(ebar, 128, !last) == false;
          if (!last && p.sk.first_poll_ns) {
            if (threadIdx.x == leader) sh_last[group] = poll_counter(&counters[c_first], n_parts - 1, abort_ptr, p.sk.first_poll_ns);
            named_bar_sync(ebar, 128);
            last = sh_last[group] != 0;
            if (last) __threadfence();
          }
          if (!last) {
            publish(c_first);
            if (threadIdx.x == leader)
              sh_last[group] = !*abort_ptr && atomicAdd(&counters[c_first], 1) == n_parts - 1;
            named_bar_sync(ebar, 128);
            last = sh_last[group] != 0;
            if (last) __threadfence();
          }
          if (last) {
            if (live) add_parts(c_first, c_last, true);
            if (threadIdx.x == leader) counters[c_first] = 0;  // the next launch starts from zero
          }
          emit = emit && last;
          named_bar_sync(ebar, 128);  // sh_last is read by all before it is written again
        }
      }
      if (emit) store_out(u.b, u.nt);
      i += here;
      u.kb += here - 1;
      u.next(p);
    }
    // The part published without looking: if it was the tile's last to arrive (the
    // first contributor gave up its poll), the tile is reduced here.
    if (pend_tile >= 0) {
      if (threadIdx.x == leader) sh_last[group] = !*abort_ptr && pend_old == pend_last - pend_first;
      named_bar_sync(ebar, 128);
      if (sh_last[group]) {
        __threadfence();
        add_parts(pend_first, pend_last, false);
        if (threadIdx.x == leader) counters[pend_first] = 0;
        store_out(static_cast<int>(pend_tile / p.n_tiles), static_cast<int>(pend_tile % p.n_tiles));
      }
    }
  }

  __syncthreads();
  if (warp == 0) {
    if (lane == 0 && abort_flag) {
      // loads issued but never consumed must land before the CTA exits
      for (int j = 0; j < 2; ++j)
        for (int k = sh_consumed[j]; k < sh_issued[j]; k += 2) mbar_wait_quick(&full_bar[k % S], (k / S) & 1, nullptr, p.status);
    }
    __syncwarp();
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kCols);
  }
}

template <int TN>
int launch_tn(const BlockGemmArgs& L, DecodeParams& p, cudaStream_t stream) {
  CUtensorMap tw, ta;
  int st = encode_tmap_3d(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, L.w, L.K, L.N, L.batch, L.w_sn, L.w_sb, kBlk, kBlk,
                          CU_TENSOR_MAP_SWIZZLE_128B);
  if (st != CB_OK) return st;
  st = encode_tmap_3d(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, L.a, L.K, L.M, L.batch, L.a_sm, L.a_sb, kBlk, TN,
                      CU_TENSOR_MAP_SWIZZLE_128B);
  if (st != CB_OK) return st;
  // even, so that a stage always belongs to one producer and one MMA issuer
  constexpr int kStages = (kPerSm<TN> == 2 ? 110 : 200) * 1024 / (kWBytes + TN * kBlk) / 2 * 2;
  static_assert(kStages <= kMaxStages, "barriers");
  p.stages = kStages;
  constexpr size_t smem = static_cast<size_t>(kStages) * (kWBytes + TN * kBlk) + 1024;
  static thread_local int configured_dev = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (configured_dev != dev) {
    if (cudaFuncSetAttribute(block_gemm_decode_kernel<TN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(smem)) != cudaSuccess)
      return CB_ERR_CUDA;
    configured_dev = dev;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.sk.grid);
  cfg.blockDim = dim3(kThreads<TN>);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, block_gemm_decode_kernel<TN>, tw, ta, p));
}

}  // namespace

size_t block_gemm_decode_workspace() {
  int sms = sm_count();
  if (sms <= 0) sms = 148;
  return workspace_need(sms, static_cast<size_t>(64) * kBlk * sizeof(float));
}

int launch_block_gemm_decode(const BlockGemmArgs& L, cudaStream_t stream) {
  const int sms = sm_count();
  if (sms <= 0) return CB_ERR_CUDA;
  DecodeParams p = {};
  p.M = static_cast<int>(L.M), p.N = static_cast<int>(L.N);
  p.KB = static_cast<int>((L.K + kBlk - 1) / kBlk);
  p.n_tiles = static_cast<int>((L.N + kBlk - 1) / kBlk);
  p.sk.total = L.batch * static_cast<long long>(p.n_tiles) * p.KB;
  // A join takes as long as 8 blocks (0.28 us each) and, for every four parts, 1 to 4
  // more. With K = 4096, N = 4096 and one token: 13.4 us whole, 8.7 in four parts a
  // tile, 9.0 on all SMs; 64 tokens 16.8, 12.7, 14.3. With K = 1024, N = 9000: 6.0
  // whole and 7.8 on all SMs. With K = 17408, N = 256 and 64 tokens 16.7 in nine parts
  // a tile, 46.3 on all SMs.
  const SplitPlan split = plan_split(L.batch * p.n_tiles, p.KB, sms < kMaxGrid / 2 ? sms : kMaxGrid / 2,  // two counters a CTA
                                     {8, 4, L.M <= 16 ? 1 : L.M <= 32 ? 2 : 4});
  const int grid = split.grid;
  p.sk.grid = grid;
  p.sk.kb_per_tile = p.KB;
  p.a_scale = L.a_scale, p.as_sb = L.as_sb, p.as_sm = L.as_sm;
  p.w_scale = L.w_scale, p.ws_sb = L.ws_sb, p.ws_sn = L.ws_sn;
  p.bias = L.bias, p.bias_dtype = L.bias_dtype, p.bias_sb = L.b_sb;
  p.out = L.out, p.out_dtype = L.out_dtype, p.out_sb = L.o_sb, p.out_sm = L.o_sm;
  p.sk.first_poll_ns = debug_force_last_arriver() ? 0 : kFirstPollNs;
  p.dbg_wait_ns = debug_wait_ns();
  Workspace ws = carve_workspace(L.workspace, grid);
  p.partials = static_cast<float*>(ws.partials);
  p.counters = ws.counters;
  p.status = ws.status;
  if (p.M <= 16) return launch_tn<16>(L, p, stream);
  if (p.M <= 32) return launch_tn<32>(L, p, stream);
  return launch_tn<64>(L, p, stream);
}

}  // namespace cb
