// Residual addition + RMSNorm + 8-bit output, one launch, and the e4m3
// activation quantizer with one scale per 128 elements.
//
// Per row of x [rows, H] (f16/bf16), all arithmetic in fp32:
//   h = x + residual                     (stored once, rounded to x's type)
//   r = 1 / sqrt(mean(h^2) + eps),  u = h * weight,  y = u * r
//   step_g = max(amax_g |u| / Q, 2^-100)   (Q = 127 int8, 448 e4m3)
//   q = round(u / step_g),  scale_g = step_g * r        y ~ q * scale_g
// with one group per row (int8, e4m3) or per 128 elements (e4m3). The row factor
// r divides out of y / scale, so q depends on u alone: the sum of squares and the
// group amax come from ONE pass and one joint reduction (quantizing y itself
// needs r first: two dependent reductions), q does not depend on the order of
// the sum, and in the per-128 form q is written before the row's sum is known.
// h enters the norm unrounded; y itself is never formed.
//
// Bound: HBM (7 bytes moved per element with a residual and ~6 flops) for many
// rows, launch + one memory round trip + one reduction for few (5.2 us a call, of which
// the host's part is the most). A row is held in
// registers by one CTA (H > 1024) or one warp; each thread owns vectors of eight
// consecutive elements, so 16 neighbouring lanes hold one 128-element group and
// its amax is four shuffles. Rows longer than the registers hold are read twice.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "cb_internal.h"
#include "cb_ptx.cuh"
#include "cb_quant8.cuh"

namespace cb {
namespace {

constexpr float kNormFloor = 7.888609052210118e-31f;  // 2^-100
constexpr float kQuantFloor = 1.0f / (448.0f * 512.0f);
constexpr int kGroup = 128;
constexpr int kMaxThreads = 1024;

__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ void from_f32(float v, __half& o) { o = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }

// What a group is divided by: zeros (a padded row, or threads past a row's end) stay zeros
// whatever it is, and 1 spares them the division proper that a step of 2^-100 takes
// (8192 rows of 2816, whose last warp is half empty: 46 us with it).
__device__ __forceinline__ float divisor(float amax, float step) { return amax == 0.0f ? 1.0f : step; }

struct NormParams {
  const void* x;
  const void* residual;  // optional
  const void* weight;
  float eps;
  int H;
  long long rows;
  long long x_sm, r_sm, q_sm, h_sm, s_sm;
  void* q;
  float* scale;
  void* h;  // optional
  int int8;  // row-scale form: 1 int8, 0 e4m3
};

// Eight 16-bit elements at p, in the widest pieces that its address allows.
__device__ __forceinline__ uint4 load_raw8(const uint16_t* p) {
  const unsigned a = static_cast<unsigned>(reinterpret_cast<uintptr_t>(p));
  uint4 r;
  if ((a & 15) == 0) return *reinterpret_cast<const uint4*>(p);
  if ((a & 7) == 0) {
    const uint2 x = *reinterpret_cast<const uint2*>(p), y = *reinterpret_cast<const uint2*>(p + 4);
    r = make_uint4(x.x, x.y, y.x, y.y);
  } else if ((a & 3) == 0) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(p);
    r = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(p + 1);
    const uint32_t first = p[0], x = w[0], y = w[1], z = w[2], last = p[7];
    r = make_uint4(first | x << 16, x >> 16 | y << 16, y >> 16 | z << 16, z >> 16 | last << 16);
  }
  return r;
}

__device__ __forceinline__ void store_raw8(uint16_t* p, uint4 r) {
  const unsigned a = static_cast<unsigned>(reinterpret_cast<uintptr_t>(p));
  if ((a & 15) == 0) {
    *reinterpret_cast<uint4*>(p) = r;
  } else if ((a & 7) == 0) {
    *reinterpret_cast<uint2*>(p) = make_uint2(r.x, r.y);
    *reinterpret_cast<uint2*>(p + 4) = make_uint2(r.z, r.w);
  } else if ((a & 3) == 0) {
    uint32_t* w = reinterpret_cast<uint32_t*>(p);
    w[0] = r.x, w[1] = r.y, w[2] = r.z, w[3] = r.w;
  } else {
    uint32_t* w = reinterpret_cast<uint32_t*>(p + 1);
    p[0] = static_cast<uint16_t>(r.x);
    w[0] = r.x >> 16 | r.y << 16, w[1] = r.y >> 16 | r.z << 16, w[2] = r.z >> 16 | r.w << 16;
    p[7] = static_cast<uint16_t>(r.w >> 16);
  }
}

// Eight elements at index `at` of a row as fp32; zeros from `n` on. VEC: rows are whole
// 16-byte vectors; else in pieces (element by element, rows of 8404 took 52 us for 1310).
template <bool VEC, typename T>
__device__ __forceinline__ void load8(const T* row, int at, int n, float (&v)[8]) {
  if (at + 8 <= n || (VEC && at < n)) {
    if constexpr (sizeof(T) == 2) {
      uint4 raw;
      if constexpr (VEC)
        raw = *reinterpret_cast<const uint4*>(row + at);
      else
        raw = load_raw8(reinterpret_cast<const uint16_t*>(row + at));
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = to_f32(e[j]);
    } else if (VEC || (reinterpret_cast<uintptr_t>(row + at) & 15) == 0) {
      const float4 a = *reinterpret_cast<const float4*>(row + at), b = *reinterpret_cast<const float4*>(row + at + 4);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = to_f32(row[at + j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = !VEC && at + j < n ? to_f32(row[at + j]) : 0.0f;
  }
}

template <bool VEC, typename T>
__device__ __forceinline__ void store8(T* row, int at, int n, const float (&v)[8]) {
  if (at + 8 <= n || (VEC && at < n)) {
    uint4 raw;
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int j = 0; j < 8; ++j) from_f32(v[j], e[j]);
    if constexpr (VEC)
      *reinterpret_cast<uint4*>(row + at) = raw;
    else
      store_raw8(reinterpret_cast<uint16_t*>(row + at), raw);
  } else if constexpr (!VEC) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (at + j < n) from_f32(v[j], row[at + j]);
  }
}

template <bool VEC>
__device__ __forceinline__ void store_q8(uint8_t* row, int at, int n, uint64_t q) {
  uint8_t* const p = row + at;
  if constexpr (VEC) {
    if (at < n) *reinterpret_cast<uint64_t*>(p) = q;
  } else if (at + 8 <= n) {
    const unsigned a = static_cast<unsigned>(reinterpret_cast<uintptr_t>(p));
    const uint32_t lo = static_cast<uint32_t>(q), hi = static_cast<uint32_t>(q >> 32);
    if ((a & 7) == 0) {
      *reinterpret_cast<uint64_t*>(p) = q;
    } else if ((a & 3) == 0) {
      uint32_t* w = reinterpret_cast<uint32_t*>(p);
      w[0] = lo, w[1] = hi;
    } else if ((a & 1) == 0) {
      uint16_t* w = reinterpret_cast<uint16_t*>(p);
      w[0] = static_cast<uint16_t>(lo), w[1] = static_cast<uint16_t>(lo >> 16);
      w[2] = static_cast<uint16_t>(hi), w[3] = static_cast<uint16_t>(hi >> 16);
    } else {
      uint16_t* w = reinterpret_cast<uint16_t*>(p + 1);
      p[0] = static_cast<uint8_t>(lo);
      w[0] = static_cast<uint16_t>(lo >> 8), w[1] = static_cast<uint16_t>(q >> 24), w[2] = static_cast<uint16_t>(hi >> 8);
      p[7] = static_cast<uint8_t>(hi >> 24);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (at + j < n) p[j] = static_cast<uint8_t>(q >> (8 * j));
  }
}

__device__ __forceinline__ float amax8(const float (&v)[8]) {
  float m = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(v[j]));
  return m;
}

// Largest of 16 neighbouring lanes (one 128-element group).
__device__ __forceinline__ float group_max(float m) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

__device__ __forceinline__ void warp_sum_max(float& s, float& m) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  }
}

// (sum, max) over the threads of one row: a warp, or the whole CTA.
__device__ __forceinline__ void row_sum_max(float& s, float& m, float2* red) {
  warp_sum_max(s, m);
  if (blockDim.x == 32) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0) red[warp] = make_float2(s, m);
  __syncthreads();
  const float2 v = lane < warps ? red[lane] : make_float2(0.0f, 0.0f);
  s = v.x;
  m = v.y;
  warp_sum_max(s, m);
}

__device__ __forceinline__ float row_factor(float ss, int H, float eps) {
  return __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, static_cast<float>(H)), eps)));
}

// One row per blockDim.x threads, NV vectors of eight elements per thread.
template <typename T, typename W, bool BLOCK, int NV, bool VEC>
__global__ void __launch_bounds__(kMaxThreads) norm_kernel(const NormParams p) {
  pdl_wait_primary();
  pdl_launch_dependents();
  __shared__ float2 red[32];
  const long long row = static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (row >= p.rows) return;  // whole warps: blockDim.x is 32 where blockDim.y is not 1
  const T* x = static_cast<const T*>(p.x) + row * p.x_sm;
  const T* res = p.residual ? static_cast<const T*>(p.residual) + row * p.r_sm : nullptr;
  const W* w = static_cast<const W*>(p.weight);
  T* h = p.h ? static_cast<T*>(p.h) + row * p.h_sm : nullptr;
  uint8_t* q = static_cast<uint8_t*>(p.q) + row * p.q_sm;

  float u[NV][8];
#pragma unroll
  for (int v = 0; v < NV; ++v) load8<VEC>(x, (v * blockDim.x + threadIdx.x) * 8, p.H, u[v]);
  if (res) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float t[8];
      const int at = (v * blockDim.x + threadIdx.x) * 8;
      load8<VEC>(res, at, p.H, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) u[v][j] = __fadd_rn(u[v][j], t[j]);
      if (h) store8<VEC>(h, at, p.H, u[v]);
    }
  }
  float ss = 0.0f, amax = 0.0f;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    float t[8];
    load8<VEC>(w, (v * blockDim.x + threadIdx.x) * 8, p.H, t);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ss = __fmaf_rn(u[v][j], u[v][j], ss);
      u[v][j] = __fmul_rn(u[v][j], t[j]);
    }
  }
  if constexpr (BLOCK) {
    float step[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      amax = group_max(amax8(u[v]));
      step[v] = fmaxf(__fdiv_rn(amax, 448.0f), kNormFloor);
      store_q8<VEC>(q, (v * blockDim.x + threadIdx.x) * 8, p.H, quant8<false>(u[v], divisor(amax, step[v])));
    }
    row_sum_max(ss, amax, red);
    const float r = row_factor(ss, p.H, p.eps);
    if ((threadIdx.x & 15) == 0) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int at = (v * blockDim.x + threadIdx.x) * 8;
        if (at < p.H) p.scale[row * p.s_sm + at / kGroup] = __fmul_rn(step[v], r);
      }
    }
  } else {
#pragma unroll
    for (int v = 0; v < NV; ++v) amax = fmaxf(amax, amax8(u[v]));
    row_sum_max(ss, amax, red);
    const float step = fmaxf(__fdiv_rn(amax, p.int8 ? 127.0f : 448.0f), kNormFloor), div = divisor(amax, step);
#pragma unroll
    for (int v = 0; v < NV; ++v)
      store_q8<VEC>(q, (v * blockDim.x + threadIdx.x) * 8, p.H,
                    p.int8 ? quant8<true>(u[v], div) : quant8<false>(u[v], div));
    if (threadIdx.x == 0) p.scale[row * p.s_sm] = __fmul_rn(step, row_factor(ss, p.H, p.eps));
  }
}

// Many rows: CTAs that walk the rows, with the next AHEAD rows' loads always in flight.
// Every thread copies into shared memory just what it will read itself (cp.async), so a
// row needs no barrier but its reduction's. One CTA per row instead leaves HBM idle
// while the resident CTAs reduce and store (16384 x 8192 with a residual: 199 us; this
// form 144 to 164, 0.87 to 1.0 of the copy rate, by the device).
// The weight stays in registers.
__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

template <typename T, typename W, bool BLOCK, int NV, int AHEAD>
__global__ void __launch_bounds__(512, NV == 4 ? 1 : 2) norm_rows_kernel(const NormParams p) {
  extern __shared__ uint4 sh_rows[];  // [AHEAD + 1][x, residual][NV][thread]
  __shared__ float2 red[2][32];
  pdl_wait_primary();
  pdl_launch_dependents();
  const int tid = threadIdx.x, n = blockDim.x;
  constexpr int kWv = sizeof(W) * 8 / 16;  // 16-byte pieces of eight weights
  uint4 wraw[NV][kWv];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int i = 0; i < kWv; ++i) {
      const int at = (v * n + tid) * 8;
      wraw[v][i] = at < p.H ? reinterpret_cast<const uint4*>(static_cast<const W*>(p.weight) + at)[i] : make_uint4(0, 0, 0, 0);
    }
  auto place = [&](int stage, int which, int v) { return sh_rows + ((stage * 2 + which) * NV + v) * n + tid; };
  auto request = [&](long long row, int stage) {
    if (row < p.rows) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int at = (v * n + tid) * 8;
        if (at >= p.H) continue;
        cp_async16(place(stage, 0, v), static_cast<const T*>(p.x) + row * p.x_sm + at);
        if (p.residual) cp_async16(place(stage, 1, v), static_cast<const T*>(p.residual) + row * p.r_sm + at);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int a = 0; a < AHEAD; ++a) request(blockIdx.x + static_cast<long long>(a) * gridDim.x, a);
  int stage = 0, parity = 0;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x, parity ^= 1) {
    const int last = stage > 0 ? stage - 1 : AHEAD;  // the stage before this one: free
    request(row + static_cast<long long>(AHEAD) * gridDim.x, last);
    asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD) : "memory");
    T* h = p.h ? static_cast<T*>(p.h) + row * p.h_sm : nullptr;
    uint8_t* q = static_cast<uint8_t*>(p.q) + row * p.q_sm;
    float u[NV][8];
    float ss = 0.0f, amax = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int at = (v * n + tid) * 8;
      const int left = at < p.H ? 8 : 0;  // rows are whole vectors
      load8<true>(reinterpret_cast<const T*>(place(stage, 0, v)), 0, left, u[v]);
      if (p.residual) {
        float t[8];
        load8<true>(reinterpret_cast<const T*>(place(stage, 1, v)), 0, left, t);
#pragma unroll
        for (int j = 0; j < 8; ++j) u[v][j] = __fadd_rn(u[v][j], t[j]);
        if (h) store8<true>(h, at, p.H, u[v]);
      }
      float t[8];
      const W* w = reinterpret_cast<const W*>(wraw[v]);
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = to_f32(w[j]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        ss = __fmaf_rn(u[v][j], u[v][j], ss);
        u[v][j] = __fmul_rn(u[v][j], t[j]);
      }
    }
    if constexpr (BLOCK) {
      float step[NV];
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        amax = group_max(amax8(u[v]));
        step[v] = fmaxf(__fdiv_rn(amax, 448.0f), kNormFloor);
        store_q8<true>(q, (v * n + tid) * 8, p.H, quant8<false>(u[v], divisor(amax, step[v])));
      }
      row_sum_max(ss, amax, red[parity]);
      const float r = row_factor(ss, p.H, p.eps);
      if ((tid & 15) == 0) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const int at = (v * n + tid) * 8;
          if (at < p.H) p.scale[row * p.s_sm + at / kGroup] = __fmul_rn(step[v], r);
        }
      }
    } else {
#pragma unroll
      for (int v = 0; v < NV; ++v) amax = fmaxf(amax, amax8(u[v]));
      row_sum_max(ss, amax, red[parity]);
      const float step = fmaxf(__fdiv_rn(amax, p.int8 ? 127.0f : 448.0f), kNormFloor), div = divisor(amax, step);
#pragma unroll
      for (int v = 0; v < NV; ++v)
        store_q8<true>(q, (v * n + tid) * 8, p.H, p.int8 ? quant8<true>(u[v], div) : quant8<false>(u[v], div));
      if (tid == 0) p.scale[row * p.s_sm] = __fmul_rn(step, row_factor(ss, p.H, p.eps));
    }
    stage = stage == AHEAD ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Rows longer than 32768 elements: one CTA per row that reads the row twice (the
// second time from L2). h may be the residual's own buffer, so it is stored in
// the last read of each element.
template <typename T, typename W, bool BLOCK>
__global__ void __launch_bounds__(kMaxThreads) norm_long_kernel(const NormParams p) {
  pdl_wait_primary();
  pdl_launch_dependents();
  __shared__ float2 red[32];
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.x_sm;
  const T* res = p.residual ? static_cast<const T*>(p.residual) + row * p.r_sm : nullptr;
  const W* w = static_cast<const W*>(p.weight);
  T* h = p.h ? static_cast<T*>(p.h) + row * p.h_sm : nullptr;
  uint8_t* q = static_cast<uint8_t*>(p.q) + row * p.q_sm;
  float ss = 0.0f, amax = 0.0f;
  auto weighted = [&](int at, float (&u)[8], float* sum) {
    float t[8];
    load8<false>(x, at, p.H, u);
    if (res) {
      load8<false>(res, at, p.H, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = __fadd_rn(u[j], t[j]);
    }
    if (h && (BLOCK || !sum)) store8<false>(h, at, p.H, u);
    load8<false>(w, at, p.H, t);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (sum) *sum = __fmaf_rn(u[j], u[j], *sum);
      u[j] = __fmul_rn(u[j], t[j]);
    }
  };
  // every thread runs the same number of passes: the group maximum is warp-wide
  const int span = static_cast<int>(blockDim.x) * 8;
  float u[8];
  for (long long base = 0; base < p.H; base += span) {
    const long long at64 = base + threadIdx.x * 8;
    const int at = at64 < p.H ? static_cast<int>(at64) : p.H;
    weighted(at, u, &ss);
    if constexpr (BLOCK) {
      amax = group_max(amax8(u));
      const float step = fmaxf(__fdiv_rn(amax, 448.0f), kNormFloor);
      store_q8<false>(q, at, p.H, quant8<false>(u, divisor(amax, step)));
      if ((threadIdx.x & 15) == 0 && at < p.H) p.scale[row * p.s_sm + at / kGroup] = step;  // times r below
    } else {
      amax = fmaxf(amax, amax8(u));
    }
  }
  row_sum_max(ss, amax, red);
  const float r = row_factor(ss, p.H, p.eps);
  if constexpr (BLOCK) {
    for (long long base = 0; base < p.H; base += span) {
      const long long at = base + threadIdx.x * 8;  // the thread that wrote the step
      if ((threadIdx.x & 15) == 0 && at < p.H) p.scale[row * p.s_sm + at / kGroup] *= r;
    }
  } else {
    const float step = fmaxf(__fdiv_rn(amax, p.int8 ? 127.0f : 448.0f), kNormFloor), div = divisor(amax, step);
    for (long long base = 0; base < p.H; base += span) {
      const long long at = base + threadIdx.x * 8;
      if (at >= p.H) break;
      weighted(static_cast<int>(at), u, nullptr);
      store_q8<false>(q, static_cast<int>(at), p.H, p.int8 ? quant8<true>(u, div) : quant8<false>(u, div));
    }
    if (threadIdx.x == 0) p.scale[row * p.s_sm] = __fmul_rn(step, r);
  }
}

template <typename K, typename P>
int launch(K kernel, dim3 grid, dim3 block, cudaStream_t stream, const P& p, size_t smem = 0) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, p));
}

// Rows per CTA from which the walking kernel is used.
constexpr int kRowsPerCta = 4;

template <typename T, typename W, bool BLOCK, int NV, int AHEAD>
int launch_rows(const NormParams& p, cudaStream_t stream) {
  const int threads = ((p.H / 8 + NV - 1) / NV + 31) / 32 * 32;
  const size_t smem = static_cast<size_t>(AHEAD + 1) * 2 * NV * threads * sizeof(uint4);
  static thread_local int configured_dev = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (configured_dev != dev) {
    if (cudaFuncSetAttribute(norm_rows_kernel<T, W, BLOCK, NV, AHEAD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             200 * 1024) != cudaSuccess)
      return CB_ERR_CUDA;
    configured_dev = dev;
  }
  int per_sm = 1;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, norm_rows_kernel<T, W, BLOCK, NV, AHEAD>, threads, smem) !=
          cudaSuccess || per_sm < 1)
    return CB_ERR_CUDA;
  long long grid = static_cast<long long>(sm_count()) * per_sm;
  if (grid > p.rows) grid = p.rows;
  return launch(norm_rows_kernel<T, W, BLOCK, NV, AHEAD>, dim3(static_cast<unsigned>(grid)), dim3(threads), stream, p, smem);
}

template <typename T, typename W, bool BLOCK>
int launch_norm(const NormParams& p, bool vec, cudaStream_t stream) {
  const int vecs = (p.H + 7) / 8;
  if (vecs > 4 * kMaxThreads)
    return launch(norm_long_kernel<T, W, BLOCK>, dim3(static_cast<unsigned>(p.rows)), dim3(kMaxThreads), stream, p);
  // Up to 512 threads of one, two or four vectors. Short rows keep two more in flight,
  // longer ones one more (8192 elements: 144 us with one, 173 us with three: the more
  // CTAs then fit an SM).
  if (vec && vecs > 128 && vecs <= 2048 && p.rows >= static_cast<long long>(sm_count()) * kRowsPerCta * (vecs > 1024 ? 1 : 2)) {
    if (vecs <= 256) return launch_rows<T, W, BLOCK, 1, 2>(p, stream);
    if (vecs <= 1024) return launch_rows<T, W, BLOCK, 2, 1>(p, stream);
    return launch_rows<T, W, BLOCK, 4, 1>(p, stream);
  }
  // A warp per row up to 1024 elements; else a CTA per row.
  const bool warp_rows = vecs <= 32 * 4;
  int nv = 4;
  if (vec) {
    if (warp_rows)
      nv = vecs <= 32 ? 1 : vecs <= 64 ? 2 : 4;
    else if (p.rows <= 2LL * sm_count())
      nv = vecs <= kMaxThreads ? 1 : vecs <= 2 * kMaxThreads ? 2 : 4;
  }
  const int per = (vecs + nv - 1) / nv;
  const dim3 block(warp_rows ? 32 : (per + 31) / 32 * 32, warp_rows ? 4 : 1);
  const dim3 grid(static_cast<unsigned>((p.rows + block.y - 1) / block.y));
  if (!vec) return launch(norm_kernel<T, W, BLOCK, 4, false>, grid, block, stream, p);
  if (nv == 1) return launch(norm_kernel<T, W, BLOCK, 1, true>, grid, block, stream, p);
  if (nv == 2) return launch(norm_kernel<T, W, BLOCK, 2, true>, grid, block, stream, p);
  return launch(norm_kernel<T, W, BLOCK, 4, true>, grid, block, stream, p);
}

template <typename T>
int dispatch_norm(const NormParams& p, int w_dtype, bool block, bool vec, cudaStream_t s) {
  if (w_dtype == CB_DTYPE_F32)
    return block ? launch_norm<T, float, true>(p, vec, s) : launch_norm<T, float, false>(p, vec, s);
  if (w_dtype == CB_DTYPE_F16)
    return block ? launch_norm<T, __half, true>(p, vec, s) : launch_norm<T, __half, false>(p, vec, s);
  return block ? launch_norm<T, __nv_bfloat16, true>(p, vec, s) : launch_norm<T, __nv_bfloat16, false>(p, vec, s);
}

// ---- e4m3 quantizer, one scale per 128 elements of a row --------------------
//   scale = max(amax / 448, 1 / (448 * 512)),  q = e4m3(a / scale)
// (the scale rule of the library's other e4m3 quantizer). Sixteen lanes per group.
struct QuantParams {
  const void* a;
  uint8_t* q;
  float* scale;
  int M, K, groups;
  long long total;  // batch * M * groups
  long long a_sb, a_sm, q_sb, q_sm, s_sb, s_sm;
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quant_block_kernel(const QuantParams p) {
  pdl_wait_primary();
  pdl_launch_dependents();
  const int lane16 = threadIdx.x & 15;
  const long long first = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 4;
  const long long step_g = (static_cast<long long>(gridDim.x) * blockDim.x) >> 4;
  // the 32 lanes of a warp leave the loop together (group_max is warp-wide)
  for (long long g = first; (g & ~1LL) < p.total; g += step_g) {
    const bool live = g < p.total;
    const long long row = live ? g / p.groups : 0;
    const int kb = live ? static_cast<int>(g - row * p.groups) : 0;
    const long long b = row / p.M, m = row - b * p.M;
    const int n = live ? p.K : 0;
    const int at = kb * kGroup + lane16 * 8;
    float v[8];
    load8<VEC>(static_cast<const T*>(p.a) + b * p.a_sb + m * p.a_sm, at, n, v);
    const float s = fmaxf(__fdiv_rn(group_max(amax8(v)), 448.0f), kQuantFloor);
    store_q8<VEC>(p.q + b * p.q_sb + m * p.q_sm, at, n, quant8<false>(v, s));
    if (live && lane16 == 0) p.scale[b * p.s_sb + m * p.s_sm + kb] = s;
  }
}

bool vec_rows(const void* p, int64_t stride_elems, int elem) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (stride_elems * elem) % 16 == 0;
}

}  // namespace

int launch_quant_fp8_block(const void* a, int a_dtype, int64_t batch, int64_t M, int64_t K, int64_t a_sb, int64_t a_sm,
                           uint8_t* q, int64_t q_sb, int64_t q_sm, float* scale, int64_t s_sb, int64_t s_sm,
                           cudaStream_t stream) {
  QuantParams p = {};
  p.a = a;
  p.q = q;
  p.scale = scale;
  p.M = static_cast<int>(M);
  p.K = static_cast<int>(K);
  p.groups = static_cast<int>((K + kGroup - 1) / kGroup);
  p.total = batch * M * p.groups;
  // a dimension of one has no stride
  if (M == 1) a_sm = q_sm = s_sm = 0;
  if (batch == 1) a_sb = q_sb = s_sb = 0;
  p.a_sb = a_sb, p.a_sm = a_sm, p.q_sb = q_sb, p.q_sm = q_sm, p.s_sb = s_sb, p.s_sm = s_sm;
  const bool vec = K % 8 == 0 && vec_rows(a, a_sm, 2) && a_sb % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 7u) == 0 &&
                   q_sm % 8 == 0 && q_sb % 8 == 0;
  const long long blocks = (p.total + 15) / 16;
  const dim3 grid(static_cast<unsigned>(blocks < (1 << 20) ? blocks : (1 << 20))), block(256);
  if (a_dtype == CB_DTYPE_BF16)
    return vec ? launch(quant_block_kernel<__nv_bfloat16, true>, grid, block, stream, p)
               : launch(quant_block_kernel<__nv_bfloat16, false>, grid, block, stream, p);
  return vec ? launch(quant_block_kernel<__half, true>, grid, block, stream, p)
             : launch(quant_block_kernel<__half, false>, grid, block, stream, p);
}

}  // namespace cb

using namespace cb;

extern "C" CB_API int cb_add_rmsnorm_quant(const void* x, const void* residual, int x_dtype, const void* weight,
                                           int w_dtype, float eps, int64_t rows, int64_t H, int64_t x_sm, int64_t r_sm,
                                           int mode, void* q, int64_t q_sm, float* scale, int64_t s_sm, void* h_out,
                                           int64_t h_sm, cb_stream_t stream) {
  if (rows < 0 || H < 0) return CB_ERR_INVALID_ARG;
  if (mode != CB_NORM_INT8 && mode != CB_NORM_FP8 && mode != CB_NORM_FP8_BLOCK) return CB_ERR_INVALID_ARG;
  if (rows == 0 || H == 0) return CB_OK;
  if (!x || !weight || !q || !scale || (h_out && !residual)) return CB_ERR_INVALID_ARG;
  if (x_dtype != CB_DTYPE_BF16 && x_dtype != CB_DTYPE_F16) return CB_ERR_DTYPE;
  if (w_dtype != CB_DTYPE_BF16 && w_dtype != CB_DTYPE_F16 && w_dtype != CB_DTYPE_F32) return CB_ERR_DTYPE;
  if (rows > 0x7fffffffLL || H > (1LL << 30)) return CB_ERR_TOO_LARGE;
  const bool block = mode == CB_NORM_FP8_BLOCK;
  const int64_t scales = block ? (H + kGroup - 1) / kGroup : 1;
  if (rows > 1 && (x_sm < H || q_sm < H || s_sm < scales || (residual && r_sm < H) || (h_out && h_sm < H)))
    return CB_ERR_STRIDE;
  if (!(eps >= 0.0f)) return CB_ERR_INVALID_ARG;
  NormParams p = {};
  p.x = x;
  p.residual = residual;
  p.weight = weight;
  p.eps = eps;
  p.H = static_cast<int>(H);
  p.rows = rows;
  p.x_sm = x_sm, p.r_sm = r_sm, p.q_sm = q_sm, p.h_sm = h_sm, p.s_sm = s_sm;
  p.q = q;
  p.scale = scale;
  p.h = h_out;
  p.int8 = mode == CB_NORM_INT8;
  // 16-byte vectors: every row of every tensor starts on a vector boundary
  const bool one = rows == 1;
  const bool vec = H % 8 == 0 && vec_rows(x, one ? 0 : x_sm, 2) && vec_rows(weight, 0, 2) &&
                   (!residual || vec_rows(residual, one ? 0 : r_sm, 2)) && (!h_out || vec_rows(h_out, one ? 0 : h_sm, 2)) &&
                   (reinterpret_cast<uintptr_t>(q) & 7u) == 0 && (one || q_sm % 8 == 0);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (x_dtype == CB_DTYPE_BF16) return dispatch_norm<__nv_bfloat16>(p, w_dtype, block, vec, s);
  return dispatch_norm<__half>(p, w_dtype, block, vec, s);
}

extern "C" CB_API int cb_quant_act_fp8_block(const void* a, int a_dtype, int64_t batch, int64_t M, int64_t K,
                                             int64_t a_sb, int64_t a_sm, uint8_t* q, int64_t q_sb, int64_t q_sm,
                                             float* scale, int64_t s_sb, int64_t s_sm, cb_stream_t stream) {
  if (batch < 0 || M < 0 || K < 0) return CB_ERR_INVALID_ARG;
  if (batch == 0 || M == 0 || K == 0) return CB_OK;
  if (!a || !q || !scale) return CB_ERR_INVALID_ARG;
  if (a_dtype != CB_DTYPE_F16 && a_dtype != CB_DTYPE_BF16) return CB_ERR_DTYPE;
  if (batch > 0x7fffffffLL || M > 0x7fffffffLL || K > (1LL << 30)) return CB_ERR_TOO_LARGE;
  if (M > 1 && (a_sm < K || q_sm < K || s_sm < (K + kGroup - 1) / kGroup)) return CB_ERR_STRIDE;
  return launch_quant_fp8_block(a, a_dtype, batch, M, K, a_sb, a_sm, q, q_sb, q_sm, scale, s_sb, s_sm,
                                reinterpret_cast<cudaStream_t>(stream));
}
