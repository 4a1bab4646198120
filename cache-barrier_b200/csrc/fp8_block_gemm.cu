// e4m3 GEMM with one scale per 128 elements of K (activations: per token and
// block; weights: per 128 x 128 block):
//   out[m, n] = sum_kb a_s[m, kb] * w_s[n / 128, kb] * (sum_{k in kb} a[m, k] * w[n, k]) (+ bias[n])
// The inner sums run on the tensor cores with fp32 accumulators; each block's sum
// is scaled and added to an fp32 total, so the scales never touch the 8-bit
// operands.
//
// Simple form: one CTA per 128 output channels x 16 tokens, one warp per 16
// channels, mma.sync m16n8k32 with the weights as the 16-row operand. A lane's
// 16-byte loads are fragments as they are: the order of k inside a block is free
// as long as both operands share it.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "cb_gemm_common.cuh"
#include "cb_internal.h"
#include "cb_ptx.cuh"
#include "fp8_block.h"

namespace cb {
namespace {

constexpr int kBlk = 128;

struct BlockGemmParams {
  const uint8_t* a;
  const float* a_scale;
  const uint8_t* w;
  const float* w_scale;
  const void* bias;
  int bias_dtype;
  void* out;
  int out_dtype;
  int M, N, K, KB;
  long long a_sb, a_sm, w_sb, w_sn, o_sb, o_sm, as_sb, as_sm, ws_sb, ws_sn, b_sb;
};

__device__ __forceinline__ void mma_e4m3(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__global__ void __launch_bounds__(256) block_gemm_simple_kernel(const BlockGemmParams p) {
  pdl_wait_primary();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * kBlk + warp * 16, m0 = blockIdx.y * 16;
  const long long b = blockIdx.z;
  const uint8_t* w = p.w + b * p.w_sb;
  const uint8_t* a = p.a + b * p.a_sb;
  const float* ws = p.w_scale + b * p.ws_sb + static_cast<long long>(blockIdx.x) * p.ws_sn;
  const float* as = p.a_scale + b * p.as_sb;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  float total[2][4] = {};
  for (int kb = 0; kb < p.KB; ++kb) {
    float acc[2][4] = {};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int k = kb * kBlk + half * 64 + t * 16;
      const bool in = k < p.K;  // K is a multiple of 16
      uint4 wr[2], ar[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int n = n0 + g + 8 * r, m = m0 + g + 8 * r;
        wr[r] = in && n < p.N ? *reinterpret_cast<const uint4*>(w + n * p.w_sn + k) : zero;
        ar[r] = in && m < p.M ? *reinterpret_cast<const uint4*>(a + m * p.a_sm + k) : zero;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        mma_e4m3(acc[j], wr[0].x, wr[1].x, wr[0].y, wr[1].y, ar[j].x, ar[j].y);
        mma_e4m3(acc[j], wr[0].z, wr[1].z, wr[0].w, wr[1].w, ar[j].z, ar[j].w);
      }
    }
    const float sw = ws[kb];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int m = m0 + j * 8 + 2 * t + c;
        const float s = m < p.M ? as[m * p.as_sm + kb] * sw : 0.0f;
        total[j][c] = fmaf(acc[j][c], s, total[j][c]);
        total[j][2 + c] = fmaf(acc[j][2 + c], s, total[j][2 + c]);
      }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int m = m0 + j * 8 + 2 * t + (c & 1), n = n0 + g + 8 * (c >> 1);
      if (m >= p.M || n >= p.N) continue;
      float v = total[j][c];
      if (p.bias) v += load_elem(p.bias, p.bias_dtype, b * p.b_sb + n);
      store_elem(p.out, p.out_dtype, b * p.o_sb + m * p.o_sm + n, v);
    }
}

int launch_block_gemm(const BlockGemmParams& p, int64_t batch, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.N + kBlk - 1) / kBlk, (p.M + 15) / 16, static_cast<unsigned>(batch));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, block_gemm_simple_kernel, p));
}

}  // namespace

size_t fp8_block_workspace_bytes(int64_t M) {
  (void)M;
  return block_gemm_tc_workspace();
}

}  // namespace cb

using namespace cb;

extern "C" CB_API int cb_fp8_block_gemm(const uint8_t* aq, const float* a_scale, const uint8_t* w,
                                        const float* w_scale, const void* bias, int bias_dtype, void* out,
                                        int out_dtype, int64_t batch, int64_t M, int64_t N, int64_t K,
                                        const int64_t* strides, void* workspace, size_t workspace_bytes,
                                        cb_stream_t stream) {
  if (batch < 0 || M < 0 || N < 0 || K < 0) return CB_ERR_INVALID_ARG;
  if (batch == 0 || M == 0 || N == 0) return CB_OK;
  if (K == 0 || K % 16 != 0) return CB_ERR_SHAPE;
  if (!aq || !a_scale || !w || !w_scale || !out || !strides) return CB_ERR_INVALID_ARG;
  if (out_dtype != CB_DTYPE_BF16 && out_dtype != CB_DTYPE_F16 && out_dtype != CB_DTYPE_F32) return CB_ERR_DTYPE;
  if (bias && bias_dtype != CB_DTYPE_BF16 && bias_dtype != CB_DTYPE_F16 && bias_dtype != CB_DTYPE_F32)
    return CB_ERR_DTYPE;
  if (batch > 65535 || M > (1 << 20) - 16 || N > (1LL << 30) || K > (1LL << 30)) return CB_ERR_TOO_LARGE;
  const int64_t KB = (K + kBlk - 1) / kBlk;
  for (int i = 0; i < 11; ++i)
    if (strides[i] < 0) return CB_ERR_STRIDE;
  // a row may be shorter than its stride, never longer (a single row has none)
  if ((M > 1 && (strides[1] < K || strides[5] < N || strides[7] < KB)) || (N > 1 && strides[3] < K) ||
      (N > kBlk && strides[9] < KB))
    return CB_ERR_STRIDE;
  if (!aligned16(aq) || !aligned16(w) || (M > 1 && strides[1] % 16) || (N > 1 && strides[3] % 16) ||
      (batch > 1 && (strides[0] % 16 || strides[2] % 16)))
    return CB_ERR_ALIGNMENT;
  if (!workspace || workspace_bytes < fp8_block_workspace_bytes(M)) return CB_ERR_WORKSPACE;
  cudaStream_t cs = reinterpret_cast<cudaStream_t>(stream);
  if (M > 16) {
    BlockGemmArgs L = {};
    L.a = aq, L.a_scale = a_scale, L.w = w, L.w_scale = w_scale, L.bias = bias, L.bias_dtype = bias_dtype;
    L.out = out, L.out_dtype = out_dtype, L.batch = batch, L.M = M, L.N = N, L.K = K;
    L.a_sb = strides[0], L.a_sm = strides[1], L.w_sb = strides[2], L.w_sn = strides[3], L.o_sb = strides[4];
    L.o_sm = strides[5], L.as_sb = strides[6], L.as_sm = strides[7], L.ws_sb = strides[8], L.ws_sn = strides[9];
    L.b_sb = strides[10];
    L.workspace = workspace;
    return block_gemm_pair_eligible(L) ? launch_block_gemm_pair(L, cs) : launch_block_gemm_tc(L, cs);
  }
  BlockGemmParams p = {};
  p.a = aq, p.a_scale = a_scale, p.w = w, p.w_scale = w_scale, p.bias = bias, p.bias_dtype = bias_dtype;
  p.out = out, p.out_dtype = out_dtype;
  p.M = static_cast<int>(M), p.N = static_cast<int>(N), p.K = static_cast<int>(K), p.KB = static_cast<int>(KB);
  p.a_sb = strides[0], p.a_sm = strides[1], p.w_sb = strides[2], p.w_sn = strides[3], p.o_sb = strides[4];
  p.o_sm = strides[5], p.as_sb = strides[6], p.as_sm = strides[7], p.ws_sb = strides[8], p.ws_sn = strides[9];
  p.b_sb = strides[10];
  return launch_block_gemm(p, batch, cs);
}

extern "C" CB_API int cb_fp8_block_gemm_dynamic(const void* a, int a_dtype, int64_t a_sb, int64_t a_sm, uint8_t* q,
                                                float* scale, const uint8_t* w, const float* w_scale, const void* bias,
                                                int bias_dtype, void* out, int out_dtype, int64_t batch, int64_t M,
                                                int64_t N, int64_t K, const int64_t* strides, void* workspace,
                                                size_t workspace_bytes, cb_stream_t stream) {
  if (batch < 0 || M < 0 || N < 0 || K < 0) return CB_ERR_INVALID_ARG;
  if (batch == 0 || M == 0 || N == 0) return CB_OK;
  if (!strides) return CB_ERR_INVALID_ARG;
  const int rc = cb_quant_act_fp8_block(a, a_dtype, batch, M, K, a_sb, a_sm, q, strides[0], strides[1], scale,
                                        strides[6], strides[7], stream);
  if (rc != CB_OK) return rc;
  return cb_fp8_block_gemm(q, scale, w, w_scale, bias, bias_dtype, out, out_dtype, batch, M, N, K, strides, workspace,
                           workspace_bytes, stream);
}
