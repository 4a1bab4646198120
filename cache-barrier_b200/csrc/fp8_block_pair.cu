// Block-scaled e4m3 GEMM for problems with many tiles: 256 tokens x 256 output
// channels per pair of CTAs (tcgen05.mma cta_group::2).
//
// The arithmetic is that of fp8_block_tc.cu: each 128-element block of K is a fresh
// fp32 accumulator in tensor memory, which the epilogue warps scale and add to their
// registers while the tensor cores form the next one. What changes is the operand
// traffic. One SM's shared memory delivers about 128 bytes a clock, and a 128 x 256
// tile of one CTA moves 96 KB through it (TMA writes + MMA reads) per block, which
// its MMAs would take 512 clocks for: 188 bytes a clock. In a pair each CTA holds
// its own 128 tokens and half of the 256 channels, and the tensor cores of both read
// both halves: 64 KB per 512 clocks.
//
// CTA 0 of the pair issues the MMAs; both load their own tiles, with the transaction
// count on CTA 0's barriers. Commits arrive at both CTAs; epilogue warps of both
// release an accumulator at CTA 0.
//
// Warps: 0 TMA producer, 1-2 MMA issuers (CTA 0), 3 idle, 4-11 epilogue: warp w holds
// tokens 32 (w % 4) .., channels 128 ((w - 4) / 4) ..: 128 fp32 sums a thread, for
// which the epilogue's warpgroups take over registers of the first one.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "cb_gemm_common.cuh"
#include "cb_internal.h"
#include "cb_ptx.cuh"
#include "fp8_block_out.cuh"

namespace cb {
namespace {

constexpr int kBM = 128;   // tokens per CTA
constexpr int kBN = 256;   // channels per pair
constexpr int kBK = 128;
constexpr int kStages = 6;
constexpr int kThreads = 384;
constexpr int kEpiWarps = 8;
constexpr int kGroupM = 8;  // 256-token tiles that neighbouring pairs share weight tiles over
constexpr int kAcc = 2;
static_assert(kStages % 2 == 0, "the two MMA issuers take alternate stages");
constexpr uint32_t kTileBytes = 128 * kBK;            // one operand tile of one CTA
constexpr uint32_t kStageBytes = 2 * kTileBytes;
// Registers per thread at launch, and after the warpgroups' exchange:
// 128 x 88 + 256 x 208 = 384 x 168.
constexpr int kRegsLaunch = 168, kRegsFirst = 88, kRegsEpi = 208;
static_assert(128 * kRegsFirst + 256 * kRegsEpi <= kThreads * kRegsLaunch, "the exchange must not exceed the launch's registers");

struct PairParams {
  int M, N, KB;
  int m_tiles, n_tiles;
  long long tiles;
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
  int* status;
};

__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Shared-memory address of the same variable in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t peer_addr(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
// What it hands over is tensor memory, ordered by tcgen05.wait::ld and the tcgen05
// fences; release.cluster here would also flush this warp's other accesses, about
// 1000 clocks a block.
__device__ __forceinline__ void arrive_remote(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Tile load into this CTA's shared memory whose bytes count on a barrier of the pair.
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2,
                                              uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5}], [%2], %6;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void mma_f8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives once at this barrier in both CTAs when the MMAs issued so far are done.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}
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

// (batch, m-tile, n-tile): n fastest within groups of kGroupM m-tiles.
__device__ __forceinline__ void tile_of(const PairParams& p, long long tile, int& b, int& mt, int& nt) {
  const long long per = static_cast<long long>(p.m_tiles) * p.n_tiles;
  b = static_cast<int>(tile / per);
  const int r = static_cast<int>(tile - b * per);
  const int span = kGroupM * p.n_tiles;
  const int grp = r / span, in = r - grp * span;
  const int rows = p.m_tiles - grp * kGroupM < kGroupM ? p.m_tiles - grp * kGroupM : kGroupM;
  nt = in / rows;
  mt = grp * kGroupM + (in - nt * rows);
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    block_gemm_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                           const PairParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[kStages], empty_bar[kStages];
  __shared__ __align__(8) uint64_t tfull_bar[kAcc], tempty_bar[kAcc], drain_bar[kAcc];
  __shared__ uint32_t tmem_base_sh;
  __shared__ int abort_flag, sh_issued, sh_consumed[kAcc];
  volatile int* abort_ptr = &abort_flag;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cta_rank();
  const long long pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < kAcc; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], 2 * kEpiWarps);
      mbar_init(&drain_bar[a], 1);
      sh_consumed[a] = 0;
    }
    abort_flag = 0;
    sh_issued = 0;
    fence_mbar_init();
    prefetch_tmap(&tmap_a);
    prefetch_tmap(&tmap_w);
  }
  __syncwarp();
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_sh)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the barriers of both CTAs exist
  tc_fence_after();
  const uint32_t tmem = tmem_base_sh;
  pdl_wait_primary();
  if (threadIdx.x == 0) pdl_launch_dependents();
  __syncwarp();
  const long long blocks_total = pair < p.tiles ? ((p.tiles - 1 - pair) / pairs + 1) * p.KB : 0;  // k-blocks of this pair

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsFirst));
    if (warp == 0) {
      // ---------------- TMA producer (both CTAs) ----------------
      if (lane == 0) {
        const uint64_t pol = policy_evict_normal();
        int stage = 0, issued = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (long long t = pair; t < p.tiles && ok; t += pairs) {
          int b, mt, nt;
          tile_of(p, t, b, mt, nt);
          const int m0 = mt * 2 * kBM + static_cast<int>(rank) * kBM, n0 = nt * kBN + static_cast<int>(rank) * 128;
          for (int kb = 0; kb < p.KB; ++kb) {
            if (!mbar_wait_quick(&empty_bar[stage], phase ^ 1u, abort_ptr, p.status)) {
              ok = false;
              break;
            }
            if (rank == 0) mbar_arrive_expect_tx(&full_bar[stage], 2 * kStageBytes);
            uint8_t* dst = smem + stage * kStageBytes;
            const uint32_t bar = peer_addr(&full_bar[stage], 0);
            tma_load_pair(dst, &tmap_a, bar, kb * kBK, m0, b, pol);
            tma_load_pair(dst + kTileBytes, &tmap_w, bar, kb * kBK, n0, b, pol);
            ++issued;
            if (++stage == kStages) stage = 0, phase ^= 1u;
          }
        }
        sh_issued = issued;
      }
      __syncwarp();
    } else if (warp < 3) {
      // ---------------- MMA issuers (CTA 0): warp 1 + j takes the blocks j, j + 2, ... ----------------
      // A wait on shared memory takes its thread some 270 clocks while the tensor
      // cores read operands, and the fence another 150: two issuers overlap them.
      // Blocks are independent (each has a fresh accumulator), so they need no order.
      const int acc = warp - 1;
      long long consumed = blocks_total;
      if (rank == 0) {
        if (lane == 0) {
          const uint32_t idesc = idesc_e4m3_f32(256, kBN);
          int stage = acc;
          uint32_t phase = 0;
          for (consumed = acc; consumed < blocks_total; consumed += 2) {
            if (!mbar_wait_quick(&full_bar[stage], phase, abort_ptr, p.status) ||
                !mbar_wait_quick(&tempty_bar[acc], static_cast<uint32_t>((consumed >> 1) & 1) ^ 1u, abort_ptr, p.status))
              break;
            tc_fence_after();
            const uint32_t sa = smem_u32(smem + stage * kStageBytes), sw = sa + kTileBytes;
#pragma unroll
            for (int kk = 0; kk < kBK / 32; ++kk)
              mma_f8_pair(tmem + acc * kBN, smem_desc_sw128(sa + kk * 32), smem_desc_sw128(sw + kk * 32), idesc, kk != 0);
            commit_pair(&tfull_bar[acc]);
            commit_pair(&empty_bar[stage]);
            stage += 2;
            if (stage >= kStages) stage -= kStages, phase ^= 1u;
          }
          sh_consumed[acc] = static_cast<int>(consumed);  // first block of this warp's that was not issued
          commit_pair(&drain_bar[acc]);
        }
        consumed = __shfl_sync(0xffffffffu, consumed, 0);
      }
      // Every commit's arrival must land in both CTAs before they exit: the MMAs'
      // end, this warp's last stage releases and its last accumulator hand-off.
      // (After an abort CTA 1 does not know the count: its waits then run out.)
      const long long mine = rank == 0 ? consumed : blocks_total + ((blocks_total ^ acc) & 1);
      if (lane == 31) mbar_wait_quick(&drain_bar[acc], 0, nullptr, p.status);
      const long long js = mine - 2 - 2 * lane;
      if (lane < kStages / 2 && js >= 0)
        mbar_wait_quick(&empty_bar[js % kStages], static_cast<uint32_t>((js / kStages) & 1), nullptr, p.status);
      const long long ja = mine - 2;
      if (lane == 16 && ja >= 0) mbar_wait_quick(&tfull_bar[acc], static_cast<uint32_t>((ja >> 1) & 1), nullptr, p.status);
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpi));
    // ---------------- epilogue: one token per thread, 128 channels per warpgroup ----------------
    const int group = (warp - 4) >> 2, quarter = warp & 3;
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + group * 128;
    uint8_t* stg = smem + kStages * kStageBytes + (warp - 4) * kOutBytes;
    const uint32_t tempty = peer_addr(tempty_bar, 0);
    uint32_t it = 0;
    bool live = true;
    for (long long t = pair; t < p.tiles && live; t += pairs) {
      int b, mt, nt;
      tile_of(p, t, b, mt, nt);
      const int m_warp = mt * 2 * kBM + static_cast<int>(rank) * kBM + quarter * 32;
      const int m = m_warp + lane;
      const int nb = nt * 2 + group;  // 128-channel block
      const bool some = m_warp < p.M && nb * 128 < p.N;
      const float* as = p.a_scale + b * p.as_sb + static_cast<long long>(m < p.M ? m : 0) * p.as_sm;
      const float* ws = p.w_scale + b * p.ws_sb + static_cast<long long>(nb * 128 < p.N ? nb : 0) * p.ws_sn;
      float sum[128];
#pragma unroll
      for (int i = 0; i < 128; ++i) sum[i] = 0.0f;
      float sa = __ldg(as), sw = __ldg(ws);
      for (int kb = 0; kb < p.KB; ++kb, ++it) {
        const float s = m < p.M ? sa * sw : 0.0f;
        if (kb + 1 < p.KB) sa = __ldg(as + kb + 1), sw = __ldg(ws + kb + 1);
        const uint32_t acc = it & 1;
        live = __all_sync(0xffffffffu, mbar_wait_quick(&tfull_bar[acc], (it >> 1) & 1, abort_ptr, p.status));
        if (!live) break;
        if (some) {
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t r[32];
            tmem_ld32(lane_addr + acc * kBN + c * 32, r);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) sum[c * 32 + i] = fmaf(__uint_as_float(r[i]), s, sum[c * 32 + i]);
          }
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) arrive_remote(tempty + acc * sizeof(uint64_t));
      }
      if (!live || !some) continue;
      const int n0 = nb * 128;
      if (p.bias) add_bias(sum, p.bias, p.bias_dtype, b * p.bias_sb + n0, p.N - n0, lane);
      const int es = p.out_dtype == CB_DTYPE_F32 ? 4 : 2;
      store_rows(stg, sum, static_cast<char*>(p.out) + (b * p.out_sb + static_cast<long long>(m_warp) * p.out_sm + n0) * es,
                 p.out_sm * es, p.M - m_warp, p.N - n0, p.out_dtype, p.unit, lane);
    }
  }

  __syncthreads();
  cluster_sync();
  if (warp == 0) {
    if (lane == 0 && rank == 0 && abort_flag) {
      // loads issued but never consumed must land before the CTAs exit
      const int from = sh_consumed[0] < sh_consumed[1] ? sh_consumed[0] : sh_consumed[1];
      for (int j = from; j < sh_issued; ++j) mbar_wait_quick(&full_bar[j % kStages], (j / kStages) & 1, nullptr, p.status);
    }
    __syncwarp();
  }
  __syncthreads();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

}  // namespace

long long block_gemm_pair_blocks(const BlockGemmArgs& L) {
  const int pairs = sm_count() / 2;
  const long long tiles = L.batch * ((L.M + 255) / 256) * ((L.N + 255) / 256);
  return pairs > 0 ? (tiles + pairs - 1) / pairs * ((L.K + kBK - 1) / kBK) : 0;
}

int launch_block_gemm_pair(const BlockGemmArgs& L, cudaStream_t stream) {
  const int sms = sm_count();
  if (sms <= 0) return CB_ERR_CUDA;
  PairParams p = {};
  p.M = static_cast<int>(L.M), p.N = static_cast<int>(L.N), p.KB = static_cast<int>((L.K + kBK - 1) / kBK);
  p.m_tiles = (p.M + 255) / 256, p.n_tiles = (p.N + kBN - 1) / kBN;
  p.tiles = L.batch * static_cast<long long>(p.m_tiles) * p.n_tiles;
  p.a_scale = L.a_scale, p.as_sb = L.as_sb, p.as_sm = L.as_sm;
  p.w_scale = L.w_scale, p.ws_sb = L.ws_sb, p.ws_sn = L.ws_sn;
  p.bias = L.bias, p.bias_dtype = L.bias_dtype, p.bias_sb = L.b_sb;
  p.out = L.out, p.out_dtype = L.out_dtype, p.out_sb = L.o_sb, p.out_sm = L.o_sm;
  p.unit = out_unit(L);
  p.status = static_cast<int*>(L.workspace);
  CUtensorMap ta, tw;
  int st = encode_tmap_3d(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, L.a, L.K, L.M, L.batch, L.a_sm, L.a_sb, kBK, kBM,
                          CU_TENSOR_MAP_SWIZZLE_128B);
  if (st != CB_OK) return st;
  st = encode_tmap_3d(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, L.w, L.K, L.N, L.batch, L.w_sn, L.w_sb, kBK, 128,
                      CU_TENSOR_MAP_SWIZZLE_128B);
  if (st != CB_OK) return st;
  constexpr size_t smem = kStages * kStageBytes + kEpiWarps * kOutBytes + 1024;
  static thread_local int configured_dev = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (configured_dev != dev) {
    // the warpgroups' register exchange counts on the launch's registers
    cudaFuncAttributes attr;
    if (cudaFuncGetAttributes(&attr, block_gemm_pair_kernel) != cudaSuccess) return CB_ERR_CUDA;
    if (attr.numRegs != kRegsLaunch) return CB_ERR_UNSUPPORTED;
    if (cudaFuncSetAttribute(block_gemm_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) !=
        cudaSuccess)
      return CB_ERR_CUDA;
    configured_dev = dev;
  }
  long long pairs = sms / 2;
  if (p.tiles < pairs) pairs = p.tiles;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, block_gemm_pair_kernel, ta, tw, p));
}

}  // namespace cb
