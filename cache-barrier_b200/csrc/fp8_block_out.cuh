// Output of the block-scaled FP8 GEMMs whose epilogue threads each hold one token's row:
// a warp's 32 rows pass through shared memory 64 bytes at a time, so that a store
// instruction writes whole 64-byte runs of 1, 2 or 8 rows, in units of 2, 4 or 16 bytes,
// whichever the output's pointer, strides and N allow. Storing from the threads' own
// rows costs a sector per element where rows are not 16-byte aligned: 1551 x 3294 x
// 1104 took 122 us that way.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "cb_gemm_common.cuh"
#include "cb_ptx.cuh"
#include "fp8_block.h"

namespace cb {

constexpr int kOutPitch = 80;  // bytes of a staged row: 64 and a pad
constexpr int kOutBytes = 32 * kOutPitch;

__device__ __forceinline__ uint32_t pack16(float a, float b, int dtype) {
  if (dtype == CB_DTYPE_BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Bytes of the largest unit that every row of the output is made of.
inline int out_unit(const BlockGemmArgs& L) {
  const int64_t e = L.out_dtype == CB_DTYPE_F32 ? 4 : 2;
  const uint64_t all = reinterpret_cast<uint64_t>(L.out) | static_cast<uint64_t>(L.N * e) | static_cast<uint64_t>(L.o_sm * e) |
                       (L.batch > 1 ? static_cast<uint64_t>(L.o_sb * e) : 0);
  return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 2;
}

// Adds bias[at ..] to every lane's C channels: a lane loads one of 32, all get it from
// there (loads by every lane for itself doubled the time of 1232 x 9920 x 1024).
template <int C>
__device__ __forceinline__ void add_bias(float (&sum)[C], const void* bias, int dtype, long long at, int channels, int lane) {
  float own[C / 32];
#pragma unroll
  for (int c = 0; c < C / 32; ++c) own[c] = c * 32 + lane < channels ? load_elem(bias, dtype, at + c * 32 + lane) : 0.0f;
#pragma unroll
  for (int i = 0; i < C; ++i) sum[i] += __shfl_sync(0xffffffffu, own[i / 32], i % 32);
}

// Staged 64 bytes of 32 rows -> rows [0, rows), bytes [0, bytes) of each.
template <typename U>
__device__ __forceinline__ void flush_rows(const uint8_t* stg, char* out, long long row_bytes, int rows, int bytes, int lane) {
  constexpr int kUnits = 64 / sizeof(U), kRows = 32 / kUnits;  // units of a row, rows at once
  const int at = lane % kUnits * static_cast<int>(sizeof(U)), first = lane / kUnits;
  if (at >= bytes) return;
  char* to = out + first * row_bytes + at;
#pragma unroll 4
  for (int r = first; r < 32; r += kRows, to += kRows * row_bytes)
    if (r < rows) *reinterpret_cast<U*>(to) = *reinterpret_cast<const U*>(stg + r * kOutPitch + at);
}

// sum: this lane's row, C channels from the one that `out` points to in row 0.
template <int C>
__device__ __forceinline__ void store_rows(uint8_t* stg, const float (&sum)[C], char* out, long long row_bytes, int rows, int channels,
                                           int dtype, int unit, int lane) {
  auto flush = [&](int byte0, int elem) {
    __syncwarp();
    const int bytes = tile_bytes(channels, C, elem) - byte0;
    if (unit == 16)
      flush_rows<uint4>(stg, out + byte0, row_bytes, rows, bytes, lane);
    else if (unit == 4)
      flush_rows<uint32_t>(stg, out + byte0, row_bytes, rows, bytes, lane);
    else
      flush_rows<uint16_t>(stg, out + byte0, row_bytes, rows, bytes, lane);
    __syncwarp();
  };
  uint4* const mine = reinterpret_cast<uint4*>(stg + lane * kOutPitch);
  if (dtype == CB_DTYPE_F32) {
#pragma unroll
    for (int c = 0; c < C; c += 16) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        mine[j] = make_uint4(__float_as_uint(sum[c + 4 * j]), __float_as_uint(sum[c + 4 * j + 1]), __float_as_uint(sum[c + 4 * j + 2]),
                             __float_as_uint(sum[c + 4 * j + 3]));
      flush(c * 4, 4);
    }
  } else {
#pragma unroll
    for (int c = 0; c < C; c += 32) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack16(sum[c + j * 8 + 2 * i], sum[c + j * 8 + 2 * i + 1], dtype);
        mine[j] = make_uint4(w[0], w[1], w[2], w[3]);
      }
      flush(c * 2, 2);
    }
  }
}

}  // namespace cb
