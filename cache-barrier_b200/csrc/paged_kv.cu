// Append of new keys and values to a paged cache:
//   cache[slot / page_size][slot % page_size][head][:] = cvt(row[:] / scale[head])
// for every token's key and value, one launch. 16-bit caches store the row
// unchanged (or converted between bf16 and f16); an e4m3 cache stores it divided
// by the head's scale, saturated, rounded to nearest even.
//
// Bound: HBM for many tokens (each element read and written once), launch
// latency for few. One thread moves eight elements (one 16-byte load).
//
// A negative slot skips the token (padding of a captured batch). A slot past the
// cache records CB_DEVERR_BAD_INDEX in *status and is skipped: nothing outside
// the cache is written.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "cb_internal.h"
#include "cb_ptx.cuh"

namespace cb {
namespace {

struct AppendParams {
  const void* src[2];  // k, v: [T, heads, D]
  void* dst[2];        // caches
  const float* scale[2];
  const void* slots;
  int slots_i64;
  int heads, D, vecs;  // vecs: ceil(D / 8)
  long long total;     // T * heads * vecs
  long long capacity;  // pages * page_size
  int page_size;
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

template <typename T, typename C, bool VEC>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p) {
  pdl_wait_primary();
  pdl_launch_dependents();
  const int which = blockIdx.y;
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < p.total;
       i += static_cast<long long>(gridDim.x) * blockDim.x) {
    const long long th = i / p.vecs;
    const int at = static_cast<int>(i - th * p.vecs) * 8;
    const long long t = th / p.heads;
    const int h = static_cast<int>(th - t * p.heads);
    const long long slot = p.slots_i64 ? static_cast<const long long*>(p.slots)[t]
                                       : static_cast<long long>(static_cast<const int*>(p.slots)[t]);
    if (slot < 0) continue;
    if (slot >= p.capacity) {
      if (p.status) atomicOr(p.status, CB_DEVERR_BAD_INDEX);
      continue;
    }
    const long long page = slot / p.page_size;
    const T* src = static_cast<const T*>(p.src[which]) + t * p.src_st[which] + h * p.src_sh[which] + at;
    C* dst = static_cast<C*>(p.dst[which]) + page * p.dst_sp[which] + (slot - page * p.page_size) * p.dst_ss[which] +
             h * p.dst_sh[which] + at;
    const float scale = p.scale[which] ? p.scale[which][h] : 1.0f;
    if constexpr (VEC) {
      const uint4 raw = *reinterpret_cast<const uint4*>(src);
      const T* e = reinterpret_cast<const T*>(&raw);
      struct alignas(8 * sizeof(C)) Out {
        C v[8];
      } out;
#pragma unroll
      for (int j = 0; j < 8; ++j) put(&out.v[j], to_f32(e[j]), scale);
      *reinterpret_cast<Out*>(dst) = out;
    } else {
      const int n = p.D - at < 8 ? p.D - at : 8;
      for (int j = 0; j < n; ++j) put(dst + j, to_f32(src[j]), scale);
    }
  }
}

template <typename T, typename C>
int launch_append(const AppendParams& p, bool vec, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  const long long blocks = (p.total + 255) / 256;
  cfg.gridDim = dim3(static_cast<unsigned>(blocks < (1 << 20) ? blocks : (1 << 20)), 2);
  cfg.blockDim = dim3(256);
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
  p.total = T * heads * p.vecs;
  p.capacity = num_pages * page_size;
  p.page_size = static_cast<int>(page_size);
  const int64_t ce = cache_dtype == CB_DTYPE_E4M3 ? 1 : 2;
  bool vec = D % 8 == 0;
  for (int i = 0; i < 2; ++i) {
    const int64_t* st = strides + 5 * i;
    for (int j = 0; j < 5; ++j)
      if (st[j] < 0) return CB_ERR_STRIDE;
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
