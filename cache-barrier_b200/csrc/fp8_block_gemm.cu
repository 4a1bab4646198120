// e4m3 GEMM with one scale per 128 elements of K (activations: per token and
// block; weights: per 128 x 128 block):
//   out[m, n] = sum_kb a_s[m, kb] * w_s[n / 128, kb] * (sum_{k in kb} a[m, k] * w[n, k]) (+ bias[n])
// The inner sums run on the tensor cores with fp32 accumulators; each block's sum
// is scaled and added to an fp32 total, so the scales never touch the 8-bit
// operands.
//
// Three kernels, by the number of tokens (launch_block_gemm):
//   fp8_block_decode.cu  tcgen05, 128 channels x up to 64 tokens, split over K
//   fp8_block_tc.cu      tcgen05, 128 x 128 tiles, split over K
//   fp8_block_pair.cu    tcgen05 on CTA pairs, 256 x 256 tiles
#include <initializer_list>

#include "cb_internal.h"
#include "fp8_block.h"

namespace cb {
namespace {

constexpr int kBlk = 128;

int launch_block_gemm(const BlockGemmArgs& L, cudaStream_t stream) {
  if (L.M <= 64) return launch_block_gemm_decode(L, stream);
  // A 256 x 256 block of a pair takes about 0.65 us, a 128 x 128 block of a CTA 0.45 us
  // when all SMs are busy (M x N x K = 512 x 8192 x 8192: 45 us against 58 us; 1500 x
  // 3000 x 6000: 38 against 66; 300 x 17408 x 5120: 56 against 54; 256 x 8192 x 8192:
  // 43 against 33).
  if (3 * block_gemm_pair_blocks(L) < 2 * block_gemm_tc_blocks(L)) return launch_block_gemm_pair(L, stream);
  return launch_block_gemm_tc(L, stream);
}

// Checks the arguments of both entries and fills L. A dimension of one has no stride: what
// the caller gives there (frameworks give anything) is not looked at.
int check_block_gemm(BlockGemmArgs& L, const uint8_t* aq, const float* a_scale, const uint8_t* w, const float* w_scale,
                     const void* bias, int bias_dtype, void* out, int out_dtype, int64_t batch, int64_t M, int64_t N, int64_t K,
                     const int64_t* strides, void* workspace, size_t workspace_bytes) {
  if (K == 0 || K % 16 != 0) return CB_ERR_SHAPE;
  if (!aq || !a_scale || !w || !w_scale || !out || !strides) return CB_ERR_INVALID_ARG;
  if (out_dtype != CB_DTYPE_BF16 && out_dtype != CB_DTYPE_F16 && out_dtype != CB_DTYPE_F32) return CB_ERR_DTYPE;
  if (bias && bias_dtype != CB_DTYPE_BF16 && bias_dtype != CB_DTYPE_F16 && bias_dtype != CB_DTYPE_F32)
    return CB_ERR_DTYPE;
  if (batch > 65535 || M > (1 << 20) - 16 || N > (1LL << 30) || K > (1LL << 30)) return CB_ERR_TOO_LARGE;
  const int64_t KB = (K + kBlk - 1) / kBlk;
  L = {};
  L.a_sb = strides[0], L.a_sm = strides[1], L.w_sb = strides[2], L.w_sn = strides[3], L.o_sb = strides[4];
  L.o_sm = strides[5], L.as_sb = strides[6], L.as_sm = strides[7], L.ws_sb = strides[8], L.ws_sn = strides[9];
  L.b_sb = strides[10];
  if (M == 1) L.a_sm = K, L.o_sm = N, L.as_sm = KB;
  if (N == 1) L.w_sn = K;
  if (N <= kBlk) L.ws_sn = KB;
  if (batch == 1) L.a_sb = L.w_sb = L.o_sb = L.as_sb = L.ws_sb = L.b_sb = 0;
  for (const int64_t s : {L.a_sb, L.a_sm, L.w_sb, L.w_sn, L.o_sb, L.o_sm, L.as_sb, L.as_sm, L.ws_sb, L.ws_sn, L.b_sb})
    if (s < 0) return CB_ERR_STRIDE;
  // a row may be shorter than its stride, never longer
  if (L.a_sm < K || L.w_sn < K || L.o_sm < N || L.as_sm < KB || L.ws_sn < KB) return CB_ERR_STRIDE;
  if (!aligned16(aq) || !aligned16(w) || L.a_sm % 16 || L.w_sn % 16 || L.a_sb % 16 || L.w_sb % 16) return CB_ERR_ALIGNMENT;
  if (!workspace || workspace_bytes < fp8_block_workspace_bytes(M)) return CB_ERR_WORKSPACE;
  L.a = aq, L.a_scale = a_scale, L.w = w, L.w_scale = w_scale, L.bias = bias, L.bias_dtype = bias_dtype;
  L.out = out, L.out_dtype = out_dtype, L.batch = batch, L.M = M, L.N = N, L.K = K;
  L.workspace = workspace;
  return CB_OK;
}

}  // namespace

size_t fp8_block_workspace_bytes(int64_t M) {
  return M <= 64 ? block_gemm_decode_workspace() : block_gemm_tc_workspace();
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
  BlockGemmArgs L;
  const int rc = check_block_gemm(L, aq, a_scale, w, w_scale, bias, bias_dtype, out, out_dtype, batch, M, N, K, strides, workspace,
                                  workspace_bytes);
  return rc != CB_OK ? rc : launch_block_gemm(L, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" CB_API int cb_fp8_block_gemm_dynamic(const void* a, int a_dtype, int64_t a_sb, int64_t a_sm, uint8_t* q,
                                                float* scale, const uint8_t* w, const float* w_scale, const void* bias,
                                                int bias_dtype, void* out, int out_dtype, int64_t batch, int64_t M,
                                                int64_t N, int64_t K, const int64_t* strides, void* workspace,
                                                size_t workspace_bytes, cb_stream_t stream) {
  if (batch < 0 || M < 0 || N < 0 || K < 0) return CB_ERR_INVALID_ARG;
  if (batch == 0 || M == 0 || N == 0) return CB_OK;
  BlockGemmArgs L;
  int rc = check_block_gemm(L, q, scale, w, w_scale, bias, bias_dtype, out, out_dtype, batch, M, N, K, strides, workspace,
                            workspace_bytes);
  if (rc != CB_OK) return rc;  // before anything is written
  rc = cb_quant_act_fp8_block(a, a_dtype, batch, M, K, a_sb, a_sm, q, L.a_sb, L.a_sm, scale, L.as_sb, L.as_sm, stream);
  return rc != CB_OK ? rc : launch_block_gemm(L, reinterpret_cast<cudaStream_t>(stream));
}
