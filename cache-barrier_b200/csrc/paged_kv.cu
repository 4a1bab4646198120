// Append of new keys and values to a paged cache:
//   cache[slot / page_size][slot % page_size][head][:] = cvt(row[:] / scale[head])
// for every token's key and value, one launch. 16-bit caches store the row
// unchanged (or converted between bf16 and f16); an e4m3 cache stores it divided
// by the head's scale, saturated, rounded to nearest even.
//
// Bound: HBM for many tokens (each element read and written once; 16384 tokens, eight
// heads of 128, to e4m3: 23.6 to 24.8 us, 4.1 to 4.3 TB/s, with the issue of the 8-bit
// quotients near its limit; to bf16 20.8 us, the copy rate), launch latency for few. One thread moves eight elements at a time (one
// 16-byte load).
//
// The elements of a row are stored by several threads, in no order between tokens: tokens
// that share a slot leave a mixture.
//
// A negative slot skips the token (padding of a captured batch). A slot past the
// cache records CB_DEVERR_BAD_INDEX in *status and is skipped: nothing outside
// the cache is written.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "cb_internal.h"
#include "cb_ptx.cuh"
#include "cb_quant8.cuh"

namespace cb {
namespace {

constexpr int kThreads = 128, kUnroll = 4;

struct AppendParams {
  const void* src[2];  // k, v: [T, heads, D]
  void* dst[2];        // caches
  const float* scale[2];
  const void* slots;
  int slots_i64;
  int heads, D, vecs;  // vecs: ceil(D / 8)
  long long T;
  long long capacity;  // pages * page_size
  int page_size, page_shift;  // page_shift: log2 of the page size, or -1
  long long src_st[2], src_sh[2];              // token and head strides
  long long dst_sp[2], dst_ss[2], dst_sh[2];   // page, slot and head strides
  int* status;
};

__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(__half* o, float v, float) { *o = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* o, float v, float) { *o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(__nv_fp8_storage_t* o, float v, float scale) {
  *o = __nv_cvt_float_to_fp8(__fdiv_rn(v, scale), __NV_SATFINITE, __NV_E4M3);
}

template <typename T>
struct Pair;
template <>
struct Pair<__half> {
  using type = __half2;
};
template <>
struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
};

// Largest magnitude of eight 16-bit values, as pairs (NaN where all of a half are).
template <typename T2>
__device__ __forceinline__ float largest8(const T2* w) {
  const T2 m = __hmax2(__hmax2(__habs2(w[0]), __habs2(w[1])), __hmax2(__habs2(w[2]), __habs2(w[3])));
  return fmaxf(__low2float(m), __high2float(m));
}

// threadIdx.x walks a token's vectors, threadIdx.y and kUnroll its tokens: the slots and
// rows of kUnroll tokens are all requested before the first is used, and the divisions
// (vector to head, slot to page) are per thread or token, not per vector.
template <typename T, typename C, bool VEC>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendParams p) {
  pdl_wait_primary();
  pdl_launch_dependents();
  const int which = blockIdx.y;
  const int row = p.heads * p.vecs;  // vectors of a token
  const long long t0 = (static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y) * kUnroll;
  long long dst_at[kUnroll];  // element offset of the token's slot; -1: none
#pragma unroll
  for (int x = 0; x < kUnroll; ++x) {
    long long slot = -1;
    if (t0 + x < p.T)
      slot = p.slots_i64 ? static_cast<const long long*>(p.slots)[t0 + x] : static_cast<const int*>(p.slots)[t0 + x];
    if (slot >= p.capacity) {
      if (p.status) atomicOr(p.status, CB_DEVERR_BAD_INDEX);
      slot = -1;
    }
    const long long page = p.page_shift >= 0          ? slot >> p.page_shift
                           : slot < (1LL << 31)       ? static_cast<int>(slot) / p.page_size
                                                      : slot / p.page_size;
    dst_at[x] = slot < 0 ? -1 : page * p.dst_sp[which] + (slot - page * p.page_size) * p.dst_ss[which];
  }
  for (int i = threadIdx.x; i < row; i += blockDim.x) {
    const int h = i / p.vecs, at = (i - h * p.vecs) * 8;
    const T* src = static_cast<const T*>(p.src[which]) + t0 * p.src_st[which] + h * p.src_sh[which] + at;
    C* dst = static_cast<C*>(p.dst[which]) + h * p.dst_sh[which] + at;
    const float scale = p.scale[which] ? __ldg(p.scale[which] + h) : 1.0f;
    const float most = 512.0f * scale;  // keys are not bounded by their head's scale
    if constexpr (VEC) {
      uint4 raw[kUnroll];
#pragma unroll
      for (int x = 0; x < kUnroll; ++x)
        raw[x] = dst_at[x] >= 0 ? *reinterpret_cast<const uint4*>(src + x * p.src_st[which]) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int x = 0; x < kUnroll; ++x) {
        if (dst_at[x] < 0) continue;
        const T* e = reinterpret_cast<const T*>(&raw[x]);
        struct alignas(8 * sizeof(C)) Out {
          C v[8];
        } out;
        if constexpr (std::is_same<T, C>::value) {
          out = *reinterpret_cast<const Out*>(&raw[x]);
        } else if constexpr (sizeof(C) == 1) {
          float u[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) u[j] = to_f32(e[j]);
          const uint64_t q = quant8<false>(u, scale, largest8(reinterpret_cast<const typename Pair<T>::type*>(&raw[x])) < most);
          out = *reinterpret_cast<const Out*>(&q);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) put(&out.v[j], to_f32(e[j]), scale);
        }
        *reinterpret_cast<Out*>(dst + dst_at[x]) = out;
      }
    } else {
      const int n = p.D - at < 8 ? p.D - at : 8;
      for (int x = 0; x < kUnroll; ++x) {
        if (dst_at[x] < 0) continue;
        for (int j = 0; j < n; ++j) put(dst + dst_at[x] + j, to_f32(src[x * p.src_st[which] + j]), scale);
      }
    }
  }
}

template <typename T, typename C>
int launch_append(const AppendParams& p, bool vec, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  int tx = 8;  // threads along a token's vectors: a power of two
  while (tx < kThreads && tx < p.heads * p.vecs) tx *= 2;
  const int tokens = kThreads / tx * kUnroll;
  cfg.gridDim = dim3(static_cast<unsigned>((p.T + tokens - 1) / tokens), 2);
  cfg.blockDim = dim3(tx, kThreads / tx);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(vec ? cudaLaunchKernelEx(&cfg, append_kernel<T, C, true>, p)
                         : cudaLaunchKernelEx(&cfg, append_kernel<T, C, false>, p));
}

template <typename T>
int dispatch_cache(const AppendParams& p, int cache_dtype, bool vec, cudaStream_t s) {
  if (cache_dtype == CB_DTYPE_E4M3) return launch_append<T, __nv_fp8_storage_t>(p, vec, s);
  if (cache_dtype == CB_DTYPE_BF16) return launch_append<T, __nv_bfloat16>(p, vec, s);
  return launch_append<T, __half>(p, vec, s);
}

}  // namespace
}  // namespace cb

using namespace cb;

extern "C" CB_API int cb_paged_kv_append(const void* k, const void* v, int dtype, void* k_cache, void* v_cache,
                                         int cache_dtype, const float* k_scale, const float* v_scale,
                                         const void* slots, int slots_i64, int64_t T, int64_t heads, int64_t D,
                                         int64_t num_pages, int64_t page_size, const int64_t* strides, int* status,
                                         cb_stream_t stream) {
  if (T < 0 || heads < 0 || D < 0 || num_pages < 0 || page_size < 1) return CB_ERR_INVALID_ARG;
  if (T == 0 || heads == 0 || D == 0) return CB_OK;
  if (!k || !v || !k_cache || !v_cache || !slots || !strides) return CB_ERR_INVALID_ARG;
  if (dtype != CB_DTYPE_BF16 && dtype != CB_DTYPE_F16) return CB_ERR_DTYPE;
  if (cache_dtype != CB_DTYPE_BF16 && cache_dtype != CB_DTYPE_F16 && cache_dtype != CB_DTYPE_E4M3) return CB_ERR_DTYPE;
  if (cache_dtype != CB_DTYPE_E4M3 && (k_scale || v_scale)) return CB_ERR_INVALID_ARG;
  if (T > 0x7fffffffLL || heads > 65536 || D > 65536 || page_size > 0x7fffffffLL || num_pages > 0x7fffffffLL)
    return CB_ERR_TOO_LARGE;
  AppendParams p = {};
  p.src[0] = k, p.src[1] = v;
  p.dst[0] = k_cache, p.dst[1] = v_cache;
  p.scale[0] = k_scale, p.scale[1] = v_scale;
  p.slots = slots;
  p.slots_i64 = slots_i64;
  p.heads = static_cast<int>(heads);
  p.D = static_cast<int>(D);
  p.vecs = static_cast<int>((D + 7) / 8);
  p.T = T;
  p.capacity = num_pages * page_size;
  p.page_size = static_cast<int>(page_size);
  p.page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (page_size == (1LL << s)) p.page_shift = s;
  const int64_t ce = cache_dtype == CB_DTYPE_E4M3 ? 1 : 2;
  bool vec = D % 8 == 0;
  for (int i = 0; i < 2; ++i) {
    // a dimension of one has no stride: what is given there is not looked at
    const int64_t size[5] = {T, heads, num_pages, page_size, heads};
    int64_t st[5];
    for (int j = 0; j < 5; ++j) {
      st[j] = size[j] == 1 ? 0 : strides[5 * i + j];
      if (st[j] < 0) return CB_ERR_STRIDE;
    }
    p.src_st[i] = st[0], p.src_sh[i] = st[1];
    p.dst_sp[i] = st[2], p.dst_ss[i] = st[3], p.dst_sh[i] = st[4];
    // vectors of eight elements: 16 bytes in, 8 or 16 bytes out
    vec = vec && aligned16(p.src[i]) && st[0] % 8 == 0 && st[1] % 8 == 0 &&
          (reinterpret_cast<uintptr_t>(p.dst[i]) & (8 * ce - 1)) == 0 && st[2] % 8 == 0 && st[3] % 8 == 0 &&
          st[4] % 8 == 0;
  }
  p.status = status;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == CB_DTYPE_BF16) return dispatch_cache<__nv_bfloat16>(p, cache_dtype, vec, s);
  return dispatch_cache<__half>(p, cache_dtype, vec, s);
}
