// Block-scaled e4m3 GEMM on the tensor cores:
//   out[m, n] = sum_kb a_s[m, kb] * w_s[n / 128, kb] * D_kb[m, n] (+ bias[n]),
//   D_kb[m, n] = sum_{k in block kb} a[m, k] * w[n, k]
//
// tcgen05.mma kind::f8f6f4 forms each block's D_kb as a fresh fp32 accumulator in
// tensor memory; the epilogue warps read it while the next block's MMAs run, and
// add it, times its scales, to fp32 totals in their registers. Tokens are the
// MMA's M = 128 rows (a TMEM lane, so one thread, is one token: its factor a_s * w_s
// is one scalar per block, one FMA per element) and BN output channels are its
// columns, 128 per epilogue warpgroup, so w_s is uniform there.
//
// Work is cut stream-K (cb_gemm_common.cuh) when tiles do not fill the SMs evenly:
// the k-blocks of all tiles end to end in one contiguous range per CTA. Every part
// of a cut tile goes to the workspace, and the CTA whose atomic completes the
// tile's count adds them in CTA order: no CTA waits on another, and the bits do not
// depend on who adds. Otherwise CTAs take whole tiles.
//
// Warps: 0 TMA producer, 1 MMA issuer, 2-3 idle (they complete a warpgroup),
// 4.. BN / 128 epilogue warpgroups.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "cb_gemm_common.cuh"
#include "cb_internal.h"
#include "cb_ptx.cuh"
#include "fp8_block.h"

namespace cb {
namespace {

constexpr int kBM = 128;
constexpr int kBK = 128;
constexpr int kGroupM = 16;  // m-tiles that neighbouring CTAs share weight tiles over

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

struct TcParams {
  int M, N, KB;
  int m_tiles, n_tiles;
  long long tiles;
  int whole;  // CTAs take whole tiles cta, cta + grid, ... ; else stream-K ranges
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
  int vec_out;  // 16-bit output with 16-byte aligned rows, N % 8 == 0
  float* partials;  // [grid][2][kBM][BN]
  int* counters;
  int* status;
};

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

// The CTA's segments: (tile, first and last k-block).
struct Segments {
  long long g, g1, tile, step;
  int whole;
  __device__ __forceinline__ Segments(const TcParams& p) {
    whole = p.whole;
    if (whole) {
      tile = blockIdx.x;
      g1 = p.tiles;
      step = gridDim.x;
      g = 0;
    } else {
      g = p.sk.start(blockIdx.x);
      g1 = p.sk.start(blockIdx.x + 1);
      tile = g / p.KB;
      step = 1;
    }
  }
  __device__ __forceinline__ bool next(const TcParams& p, long long& t, int& kb0, int& kb1) {
    if (whole) {
      if (tile >= g1) return false;
      t = tile, kb0 = 0, kb1 = p.KB;
      tile += step;
      return true;
    }
    if (g >= g1) return false;
    t = tile;
    kb0 = static_cast<int>(g - tile * p.KB);
    const long long left = g1 - g;
    kb1 = p.KB - kb0 < left ? p.KB : kb0 + static_cast<int>(left);
    g += kb1 - kb0;
    ++tile;
    return true;
  }
};

template <int BN>
constexpr int threads_of() { return 128 + BN; }

template <int BN>
__global__ void __launch_bounds__(threads_of<BN>(), 1)
    block_gemm_tc_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                         const TcParams p) {
  constexpr uint32_t kABytes = kBM * kBK, kWBytes = BN * kBK, kStage = kABytes + kWBytes;
  constexpr int kAcc = 512 / BN;  // accumulator ring in TMEM
  constexpr int kEpiWarps = BN / 32;

  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[kMaxStages], empty_bar[kMaxStages];
  __shared__ __align__(8) uint64_t tfull_bar[kAcc], tempty_bar[kAcc], drain_bar;
  __shared__ uint32_t tmem_base_sh;
  __shared__ int abort_flag, sh_issued, sh_consumed, sh_last;
  volatile int* abort_ptr = &abort_flag;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = p.stages;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < kAcc; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], kEpiWarps);
    }
    mbar_init(&drain_bar, 1);
    abort_flag = 0;
    sh_issued = 0;
    sh_consumed = 0;
    sh_last = 0;
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
  pdl_wait_primary();
  if (threadIdx.x == 0) pdl_launch_dependents();
  __syncwarp();

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      const uint64_t pol = policy_evict_normal();
      Segments seg(p);
      long long t;
      int kb0, kb1, stage = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      while (ok && seg.next(p, t, kb0, kb1)) {
        int b, mt, nt;
        tile_of(p, t, b, mt, nt);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait_quick(&empty_bar[stage], phase ^ 1u, abort_ptr, p.status)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full_bar[stage], kStage);
          uint8_t* dst = smem + stage * kStage;
          tma_load_3d(dst, &tmap_a, &full_bar[stage], kb * kBK, mt * kBM, b, pol);
          tma_load_3d(dst + kABytes, &tmap_w, &full_bar[stage], kb * kBK, nt * BN, b, pol);
          ++issued;
          if (++stage == S) stage = 0, phase ^= 1u;
        }
      }
      sh_issued = issued;
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    int consumed = 0;
    if (lane == 0) {
      const uint32_t idesc = idesc_e4m3_f32(kBM, BN);
      Segments seg(p);
      long long t;
      int kb0, kb1, stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      while (ok && seg.next(p, t, kb0, kb1)) {
        for (int kb = kb0; kb < kb1; ++kb, ++consumed) {
          const int acc = consumed % kAcc;
          if (!mbar_wait_quick(&tempty_bar[acc], ((consumed / kAcc) & 1) ^ 1u, abort_ptr, p.status) ||
              !mbar_wait_quick(&full_bar[stage], phase, abort_ptr, p.status)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * kStage), sw = sa + kABytes;
#pragma unroll
          for (int kk = 0; kk < kBK / 32; ++kk)
            mma_f8_ss(tmem + acc * BN, smem_desc_sw128(sa + kk * 32), smem_desc_sw128(sw + kk * 32), idesc, kk != 0);
          mma_commit(&empty_bar[stage]);
          mma_commit(&tfull_bar[acc]);
          if (++stage == S) stage = 0, phase ^= 1u;
        }
      }
      sh_consumed = consumed;
      mma_commit(&drain_bar);
      mbar_wait_quick(&drain_bar, 0, nullptr, p.status);
    }
    // Every commit's arrival must land before the CTA exits: the last S stage
    // releases (lanes 0..) and the last kAcc accumulator hand-offs (lanes 16..).
    consumed = __shfl_sync(0xffffffffu, consumed, 0);
    const int js = consumed - 1 - lane;
    if (lane < S && js >= 0) mbar_wait_quick(&empty_bar[js % S], static_cast<uint32_t>((js / S) & 1), nullptr, p.status);
    const int ja = consumed - 1 - (lane - 16);
    if (lane >= 16 && lane < 16 + kAcc && ja >= 0)
      mbar_wait_quick(&tfull_bar[ja % kAcc], static_cast<uint32_t>((ja / kAcc) & 1), nullptr, p.status);
    __syncwarp();
  } else if (warp >= 4) {
    // ---------------- epilogue: one token per thread, 128 channels per warpgroup ----------------
    const int epi = warp - 4, group = epi >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + group * 128;
    const int etid = threadIdx.x - 128;  // thread among the epilogue's BN
    Segments seg(p);
    long long t;
    int kb0, kb1, it = 0;
    // After an expired wait a warp skips its work but still reaches every named
    // barrier, so no other warp is left waiting on it.
    bool live = true;
    while (seg.next(p, t, kb0, kb1)) {
      int b, mt, nt;
      tile_of(p, t, b, mt, nt);
      const int m = mt * kBM + row;
      const int nb = nt * (BN / 128) + group;  // 128-channel block
      const bool rows_live = mt * kBM + quarter * 32 < p.M && nb * 128 < p.N;
      const float* as = p.a_scale + b * p.as_sb + static_cast<long long>(m < p.M ? m : 0) * p.as_sm;
      const float* ws = p.w_scale + b * p.ws_sb + static_cast<long long>(nb * 128 < p.N ? nb : 0) * p.ws_sn;
      float sum[128];
#pragma unroll
      for (int i = 0; i < 128; ++i) sum[i] = 0.0f;
      float sa = __ldg(as + kb0), sw = __ldg(ws + kb0);
      for (int kb = kb0; kb < kb1 && live; ++kb, ++it) {
        const float s = m < p.M ? sa * sw : 0.0f;
        if (kb + 1 < kb1) sa = __ldg(as + kb + 1), sw = __ldg(ws + kb + 1);
        const int acc = it % kAcc;
        live = __all_sync(0xffffffffu, mbar_wait_quick(&tfull_bar[acc], (it / kAcc) & 1, abort_ptr, p.status));
        if (!live) break;
        if (rows_live) {
          tc_fence_after();
          uint32_t r[2][32];
          tmem_ld32(lane_addr + acc * BN, r[0]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            tmem_ld_wait();
            if (c < 3) tmem_ld32(lane_addr + acc * BN + (c + 1) * 32, r[(c + 1) & 1]);
#pragma unroll
            for (int i = 0; i < 32; ++i) sum[c * 32 + i] = fmaf(__uint_as_float(r[c & 1][i]), s, sum[c * 32 + i]);
          }
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty_bar[acc]);
      }
      const int n0 = nb * 128;
      const bool whole = kb0 == 0 && kb1 == p.KB;
      if (whole) {
        if (live && m < p.M) {
          const long long orow = b * p.out_sb + static_cast<long long>(m) * p.out_sm;
          if (p.bias) {
#pragma unroll
            for (int i = 0; i < 128; ++i)
              if (n0 + i < p.N) sum[i] += load_elem(p.bias, p.bias_dtype, b * p.bias_sb + n0 + i);
          }
          if (p.vec_out) {
#pragma unroll
            for (int i = 0; i < 128; i += 8) {
              if (n0 + i < p.N) {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  if (p.out_dtype == CB_DTYPE_BF16) {
                    const __nv_bfloat162 v = __floats2bfloat162_rn(sum[i + 2 * j], sum[i + 2 * j + 1]);
                    w[j] = *reinterpret_cast<const uint32_t*>(&v);
                  } else {
                    const __half2 v = __floats2half2_rn(sum[i + 2 * j], sum[i + 2 * j + 1]);
                    w[j] = *reinterpret_cast<const uint32_t*>(&v);
                  }
                }
                *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + orow + n0 + i) = make_uint4(w[0], w[1], w[2], w[3]);
              }
            }
          } else {
#pragma unroll
            for (int i = 0; i < 128; ++i)
              if (n0 + i < p.N) store_elem(p.out, p.out_dtype, orow + n0 + i, sum[i]);
          }
        }
      } else {
        // part of a cut tile, token-major
        const long long cc = cut_contributors(p.sk.total, p.sk.grid, p.KB, t);
        const int c_first = static_cast<int>(cc & 0xffffffffLL), c_last = static_cast<int>(cc >> 32);
        const int live_rows = p.M - mt * kBM < kBM ? p.M - mt * kBM : kBM;
        auto slot = [&](int c) { return p.partials + (static_cast<long long>(c) * 2 + p.sk.kind(c, t)) * (kBM * BN); };
        if (live && row < live_rows) {
          float4* dst = reinterpret_cast<float4*>(slot(blockIdx.x) + row * BN + group * 128);
#pragma unroll
          for (int i = 0; i < 32; ++i) dst[i] = make_float4(sum[4 * i], sum[4 * i + 1], sum[4 * i + 2], sum[4 * i + 3]);
        }
        __threadfence();
        named_bar_sync(1, BN);
        if (etid == 0) sh_last = !*abort_ptr && atomicAdd(&p.counters[c_first], 1) == c_last - c_first;
        named_bar_sync(1, BN);
        if (sh_last) {
          __threadfence();
          // 4 positions x 4 parts of loads in flight per thread
          for (int base = etid; base < live_rows * (BN / 4); base += BN * 4) {
            float4 v[4] = {};
            for (int c0 = c_first; c0 <= c_last; c0 += 4) {
              float4 u[4][4];
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const float* part = slot(c0 + c <= c_last ? c0 + c : c_last);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                  const int i = base + x * BN;
                  u[x][c] = c0 + c <= c_last && i < live_rows * (BN / 4)
                                ? __ldcg(reinterpret_cast<const float4*>(part) + i)
                                : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
              }
#pragma unroll
              for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                  v[x].x += u[x][c].x, v[x].y += u[x][c].y, v[x].z += u[x][c].z, v[x].w += u[x][c].w;
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int i = base + x * BN;
              if (i >= live_rows * (BN / 4)) break;
              const int r = i / (BN / 4), n = (i - r * (BN / 4)) * 4;
              const float f[4] = {v[x].x, v[x].y, v[x].z, v[x].w};
              const long long orow = b * p.out_sb + static_cast<long long>(mt * kBM + r) * p.out_sm;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int col = nt * BN + n + j;
                if (col < p.N)
                  store_elem(p.out, p.out_dtype, orow + col,
                             p.bias ? f[j] + load_elem(p.bias, p.bias_dtype, b * p.bias_sb + col) : f[j]);
              }
            }
          }
          if (etid == 0) p.counters[c_first] = 0;  // the next launch starts from zero
        }
        named_bar_sync(1, BN);  // sh_last is read by all before the next cut tile writes it
      }
    }
  }

  __syncthreads();
  if (warp == 0) {
    if (lane == 0 && abort_flag) {
      // loads issued but never consumed must land before the CTA exits
      for (int j = sh_consumed; j < sh_issued; ++j) mbar_wait_quick(&full_bar[j % S], (j / S) & 1, nullptr, p.status);
    }
    __syncwarp();
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int BN>
int launch_bn(const BlockGemmArgs& L, const TcParams& p, int grid, cudaStream_t stream) {
  CUtensorMap ta, tw;
  int st = encode_tmap_3d(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, L.a, L.K, L.M, L.batch, L.a_sm, L.a_sb, kBK, kBM,
                          CU_TENSOR_MAP_SWIZZLE_128B);
  if (st != CB_OK) return st;
  st = encode_tmap_3d(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, L.w, L.K, L.N, L.batch, L.w_sn, L.w_sb, kBK, BN,
                      CU_TENSOR_MAP_SWIZZLE_128B);
  if (st != CB_OK) return st;
  const size_t smem = static_cast<size_t>(p.stages) * (kBM + BN) * kBK + 1024;
  static thread_local int configured_dev = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (configured_dev != dev) {
    if (cudaFuncSetAttribute(block_gemm_tc_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024) != cudaSuccess)
      return CB_ERR_CUDA;
    configured_dev = dev;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads_of<BN>());
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, block_gemm_tc_kernel<BN>, ta, tw, p));
}

}  // namespace

size_t block_gemm_tc_workspace() {
  int sms = sm_count();
  if (sms <= 0) sms = 148;
  return workspace_need(sms, static_cast<size_t>(kBM) * 128 * sizeof(float));
}

int launch_block_gemm_tc(const BlockGemmArgs& L, cudaStream_t stream) {
  int sms = sm_count();
  if (sms <= 0) return CB_ERR_CUDA;
  TcParams p = {};
  p.M = static_cast<int>(L.M), p.N = static_cast<int>(L.N), p.KB = static_cast<int>((L.K + kBK - 1) / kBK);
  p.m_tiles = (p.M + kBM - 1) / kBM;
  constexpr int BN = 128;
  p.n_tiles = (p.N + BN - 1) / BN;
  p.tiles = L.batch * static_cast<long long>(p.m_tiles) * p.n_tiles;
  const long long total = p.tiles * p.KB;
  p.whole = 0;
  // at least 4 k-blocks per CTA of a split problem (fewer, larger parts)
  int grid = sms;
  if (p.whole) {
    if (p.tiles < grid) grid = static_cast<int>(p.tiles);
  } else {
    const int per = p.KB < 4 ? p.KB : 4;
    if (total < static_cast<long long>(grid) * per) grid = static_cast<int>((total + per - 1) / per);
  }
  p.sk.total = total;
  p.sk.grid = grid;
  p.sk.kb_per_tile = p.KB;
  p.stages = 6;
  p.a_scale = L.a_scale, p.as_sb = L.as_sb, p.as_sm = L.as_sm;
  p.w_scale = L.w_scale, p.ws_sb = L.ws_sb, p.ws_sn = L.ws_sn;
  p.bias = L.bias, p.bias_dtype = L.bias_dtype, p.bias_sb = L.b_sb;
  p.out = L.out, p.out_dtype = L.out_dtype, p.out_sb = L.o_sb, p.out_sm = L.o_sm;
  p.vec_out = (L.out_dtype == CB_DTYPE_BF16 || L.out_dtype == CB_DTYPE_F16) && L.N % 8 == 0 && aligned16(L.out) &&
              L.o_sm % 8 == 0 && (L.batch == 1 || L.o_sb % 8 == 0);
  Workspace ws = carve_workspace(L.workspace, grid);
  p.partials = static_cast<float*>(ws.partials);
  p.counters = ws.counters;
  p.status = ws.status;
  return launch_bn<128>(L, p, grid, stream);
}

}  // namespace cb
