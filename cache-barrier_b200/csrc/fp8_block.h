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

// Bytes that a tile of `width` channels holds of an output row that has `channels` left
// (up to 2^30: times their size more than an int).
__host__ __device__ inline int tile_bytes(int channels, int width, int elem) { return (channels < width ? channels : width) * elem; }

// What joining a tile's parts costs, in k-blocks: `join`, and `each` for every `per`
// parts after the first.
struct JoinCost {
  int join, per, each;
  long long of(long long parts) const { return parts < 2 ? 0 : join + each * ((parts - 1 + per - 1) / per); }
};

// CTAs that share the k-blocks of all tiles, end to end, in equal ranges.
struct SplitPlan {
  int grid;
  long long cost;  // k-blocks of the busiest CTA, with its join
};

// Either x CTAs for every tile, so that ranges end where tiles do, or all `sms`, whose
// ranges cut the tiles anywhere (a part more per tile).
inline SplitPlan plan_split(long long tiles, long long KB, int sms, const JoinCost& c) {
  const long long total = tiles * KB;
  SplitPlan best = {static_cast<int>(total < sms ? total : sms),
                    (total + sms - 1) / sms + c.of((sms + tiles - 1) / tiles + 1)};
  for (long long x = 1; x <= KB && tiles * x <= sms; ++x) {
    const long long cost = (KB + x - 1) / x + c.of(x);
    if (cost <= best.cost) best = {static_cast<int>(tiles * x), cost};
  }
  return best;
}

// 128-element blocks of K that the busiest CTA (pair) works through.
long long block_gemm_pair_blocks(const BlockGemmArgs& L);
long long block_gemm_tc_blocks(const BlockGemmArgs& L);
int launch_block_gemm_pair(const BlockGemmArgs& L, cudaStream_t stream);
int launch_block_gemm_decode(const BlockGemmArgs& L, cudaStream_t stream);
size_t block_gemm_decode_workspace();
int launch_block_gemm_tc(const BlockGemmArgs& L, cudaStream_t stream);
size_t block_gemm_tc_workspace();

}  // namespace cb
