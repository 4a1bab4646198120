// The block-scaled FP8 GEMM's launchers (validated arguments; strides in elements).
#pragma once

#include "cb_internal.h"

namespace cb {

struct BlockGemmArgs {
  const uint8_t* a;
  const float* a_scale;
  const uint8_t* w;
  const float* w_scale;
  const void* bias;
  int bias_dtype;
  void* out;
  int out_dtype;
  int64_t batch, M, N, K;
  int64_t a_sb, a_sm, w_sb, w_sn, o_sb, o_sm, as_sb, as_sm, ws_sb, ws_sn, b_sb;
  void* workspace;
};

// 128-element blocks of K that the busiest CTA (pair) works through.
long long block_gemm_pair_blocks(const BlockGemmArgs& L);
long long block_gemm_tc_blocks(const BlockGemmArgs& L);
int launch_block_gemm_pair(const BlockGemmArgs& L, cudaStream_t stream);
int launch_block_gemm_decode(const BlockGemmArgs& L, cudaStream_t stream);
size_t block_gemm_decode_workspace();
int launch_block_gemm_tc(const BlockGemmArgs& L, cudaStream_t stream);
size_t block_gemm_tc_workspace();

}  // namespace cb
