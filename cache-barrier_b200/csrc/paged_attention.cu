// Attention of one new token per sequence over a paged key-value cache:
//   z_l = scale * (q . k_l),  out = sum_l softmax(z)_l v_l,  lse = log sum_l exp(z_l)
// over the seq_lens[b] tokens that block_table[b] maps to cache pages; query heads
// share key-value heads in groups of G. bf16 / f16 queries; the cache has the
// queries' type or is e4m3 with one scale per head.
//
// Bound: HBM on the cache (2 * L * heads * D elements read once; 2G flops per
// byte of a 16-bit cache) while sequences are long: eight of 65536 tokens over eight
// heads of 128 take 286 to 306 us by the device, 6.1 to 6.5 TB/s in bf16. An e4m3 cache
// gives a step of 16 tokens half the bytes for the same instructions and latencies: 64
// sequences of 4096 tokens 117 us, 4.0 TB/s (bf16 149 us, 6.3 TB/s). Short sequences are
// bound by an item's chain (page index, keys, scores, values, join): 256 of up to 1000
// tokens 45 us.
//
// One pass with a running maximum and sum. All (sequence, kv head, head block)
// items are cut into tiles of kTile tokens, laid end to end, and the tiles are
// dealt to the CTAs in equal contiguous ranges, so ragged lengths load every SM
// alike; an item's set-up counts as kItemCost tiles, and an item of at most
// kWholeTiles stays whole with the CTA that holds its first unit (64 mixed lengths,
// e4m3: 92 us before these rules and the early requests below, 46 with them). An item
// inside one CTA's range is finished there; a cut item's parts (max, sum, unnormalised output per head) go to the workspace
// and the CTA whose atomic completes the item's count joins them in CTA order: no CTA
// waits, and the bits do not depend on who joins. Where an item has kPartsApart parts
// or more, a launch of its own joins them, one CTA per head (one sequence of 65536
// tokens over one head: 120 us joined by the last CTA, 31 us apart).
//
// Giving each short item to one warp alone (four items' chains at once, no barriers)
// was slower: 52 us against 44 for the 256 sequences, at four times the steps per chain.
//
// A CTA is four warps, and each warp is a worker of its own: it takes 16 of a
// tile's tokens and keeps its own running maximum, sum and output, so the loop
// has no barrier; the warps are joined at the item's end. Keys and values go from
// global memory straight into matrix-instruction fragments:
//   S^T[token, head] = K Q^T   m16n8k16, rows = tokens, columns = up to 8 heads
//   O^T[d, head]    += V^T P^T m16n8k16, rows = d, k = tokens
// The order of d inside a k-step and of the output rows is free, so a lane's
// 16-byte loads of K (token g, d 8t..8t+7) and V (tokens 2t, 2t+1, 2t+8, 2t+9,
// d 8g..8g+7) are the fragments after byte permutes, with no shared memory.
// P^T is the transpose of the S^T accumulator: one movmatrix per 8 tokens and term. P is
// the sum of two values of the products' 16-bit type, the one next below it and what that
// leaves, so that 2^-16 (bf16) or 2^-21 (f16) of a probability is lost, not 2^-9 or 2^-12:
// the output's error against 64 bits is the plain fp32 form's (8 sequences of 65536 tokens,
// bf16, rms 3.00e-4 of the largest output with one term, 2.44e-4 with two). The second
// product costs 0 to 1 % of the time in bf16, 2 to 4 % over e4m3, 5 % with 16 queries per
// head. The remainder of a positive probability is positive, so an infinite value of V
// stays infinite, and that of zero is zero. Heads
// are the narrow side (n = 8): a group of 5 to 8 wastes little and one wasted
// column costs no bandwidth. mma.sync is enough here: at 8 heads the products
// need a few percent of its rate at full cache bandwidth, and tcgen05 would need
// the tiles staged in shared memory first.
//
// e4m3 caches run in f16 (every e4m3 value is an f16 value): the query row is
// scaled by a power of two into f16's range, and that factor and the head's key
// scale return in the fp32 score.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "cb_internal.h"
#include "cb_ptx.cuh"

namespace cb {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 16 * kWarps;  // tokens per tile
constexpr int kCtasPerSm = 4;       // at most; a kernel's registers may allow fewer
// Units that an item's set-up (query fragments, joining the warps) counts for when
// the tiles are dealt out: with mixed lengths some CTAs hold many short items.
constexpr int kItemCost = 2;
constexpr int kWholeTiles = 4;     // items up to this are not cut
constexpr int kJoinThreads = 256;  // of join_kernel
constexpr int kPartsApart = 20;    // parts per item from which they are joined in a launch of their own
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct AttnParams {
  const void* q;
  const void* k;
  const void* v;
  const int* table;
  const int* lens;
  const float* k_scale;  // optional, per kv head
  const float* v_scale;
  void* out;
  float* lse;  // optional
  float scale;
  int B, heads, G, blocks;  // kv heads, queries per kv head, head blocks (of 8 * NT queries) per kv head
  int q_vec;  // query rows are 8-byte aligned
  int num_pages, page, page_shift, max_pages;  // page_shift: log2(page) or -1
  long long q_sb, q_sh, o_sb, o_sh, lse_sb, table_sb;
  long long k_sp, k_ss, k_sh, v_sp, v_ss, v_sh;  // in bytes
  int grid;        // CTAs launched
  int join_apart;  // cut items are joined by join_kernel
  int* status;
  int* counters;
  float* partials;
};

__device__ __forceinline__ uint4 ldg16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ldg8(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// The fp32 value next below v > 0 (v (1 - 2^-24) lies half a unit to one below it); 0 for 0.
__device__ __forceinline__ float below(float v) { return __fmul_rn(v, 0.999999940395355224609375f); }

// 16-bit arithmetic type of the products: bf16, or f16 (f16 queries, e4m3 caches).
template <bool BF16>
struct Math;
template <>
struct Math<true> {
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  // Two values >= 0: the 16-bit values next below them, and what those leave.
  static __device__ __forceinline__ uint32_t split(float lo, float hi, uint32_t& rest) {
    const uint32_t head = __byte_perm(__float_as_uint(below(lo)), __float_as_uint(below(hi)), 0x7632);
    rest = pack(lo - __uint_as_float(head << 16), hi - __uint_as_float(head & 0xffff0000u));
    return head;
  }
};
template <>
struct Math<false> {
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ uint32_t split(float lo, float hi, uint32_t& rest) {
    uint32_t head;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(head) : "f"(below(hi)), "f"(below(lo)));
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&head));
    rest = pack(lo - v.x, hi - v.y);
    return head;
  }
};

// Two e4m3 values (exact) as f16x2.
__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint32_t two) {
  uint32_t d;
  asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(d) : "r"(two));
  return d;
}

__device__ __forceinline__ float q_val(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float q_val(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void put(__half* o, float v) { *o = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* o, float v) { *o = __float2bfloat16_rn(v); }

// The T units of all items dealt to `grid` CTAs: CTA c holds units [start(c), start(c + 1)),
// start(c) = floor(c * T / grid). 32-bit divisions where T allows.
struct Deal {
  long long T, q;
  int grid;
  unsigned r;
  __device__ __forceinline__ Deal(long long units, int max_grid) : T(units) {
    // no more CTAs than units take part, so every one between an item's first and last
    // tile holds a part of it
    grid = T < max_grid ? static_cast<int>(T) : max_grid;
    if (T < (1LL << 31)) {
      const unsigned t = static_cast<unsigned>(T), n = grid > 0 ? static_cast<unsigned>(grid) : 1u;
      q = t / n;
      r = t - static_cast<unsigned>(q) * n;
    } else {
      q = T / grid;
      r = static_cast<unsigned>(T - q * grid);
    }
  }
  __device__ __forceinline__ long long start(int c) const {
    return c * q + static_cast<unsigned>(c) * r / static_cast<unsigned>(grid);  // c * r < 2^20
  }
  // CTA that holds unit u: a guess in floating point, then exact.
  __device__ __forceinline__ int owner(long long u) const {
    int c = static_cast<int>((static_cast<float>(u) + 0.5f) * static_cast<float>(grid) / static_cast<float>(T));
    if (c >= grid) c = grid - 1;
    while (start(c) > u) --c;
    while (start(c + 1) <= u) ++c;
    return c;
  }
};

// Inclusive sum over the CTA's threads; *total receives the whole sum.
__device__ __forceinline__ long long block_scan(long long v, long long* sh, long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) sh[warp] = v;
  __syncthreads();
  long long sum = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) v += sum;
    sum += sh[w];
  }
  *total = sum;
  return v;
}

template <typename QT, bool FP8, int D, int NT>
struct Shape {
  static constexpr bool kBf16 = std::is_same<QT, __nv_bfloat16>::value && !FP8;
  // Probabilities relative to the running maximum carry a factor 2^kShift, which
  // the division by their sum takes out: f16 then keeps them normal down to 2^-29
  // instead of 2^-14 (a long context's typical weight). bf16 has fp32's range.
  static constexpr float kShift = kBf16 ? 0.0f : 15.0f;
  // bf16 queries over an e4m3 cache: rows are scaled into f16's range
  static constexpr bool kScaleQ = FP8 && std::is_same<QT, __nv_bfloat16>::value;
  static constexpr int kElem = FP8 ? 1 : 2;
  static constexpr int kHeads = 8 * NT;          // query heads of a head block
  static constexpr int kKC = D * kElem / 64;     // 16-byte chunks of K per lane and token (four lanes share a row)
  static constexpr int kVLane = D * kElem / 8;   // bytes of V per lane and token (eight lanes share a row)
  static constexpr int kVV = kVLane >= 16 ? 16 : 8;  // bytes of one load
  static constexpr int kVC = kVLane / kVV;
  static constexpr int kKSteps = D / 16;
  // CTAs per SM that the registers are to leave room for. Heads of 128 over e4m3 run four
  // (180 sequences of 5825 tokens, one query per head, with one term per probability:
  // 204 us, with three 219); bf16 needs its registers for 16-byte loads in flight.
  static constexpr int kMinCtas = D == 64 || (FP8 && D == 128 && NT == 1) ? 4 : NT == 1 && (D == 128 || FP8) ? 3 : 2;
  // part of a cut item: max and sum per head, output per head and d
  static constexpr int kPart = kHeads * 2 + kHeads * D;
  // a warp's part in shared memory: rows padded so that the fragments' stores spread over the banks
  static constexpr int kPitch = D + 1;
  static constexpr int kPartSh = kHeads * 2 + kHeads * kPitch;
  static constexpr size_t kSmem = sizeof(float) * kWarps * kPartSh + sizeof(uint2) * kKSteps * NT * 32;
};

template <typename QT, bool FP8, int D, int NT, bool PAGE16>
__global__ void __launch_bounds__(kThreads, Shape<QT, FP8, D, NT>::kMinCtas) attn_kernel(const AttnParams p) {
  using S = Shape<QT, FP8, D, NT>;
  using M = Math<S::kBf16>;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  float* const sh_part = reinterpret_cast<float*>(smem_raw);  // [warp][kPartSh]
  uint2* const sh_q = reinterpret_cast<uint2*>(sh_part + kWarps * S::kPartSh);  // query fragments [k-step][NT][lane]
  __shared__ long long sh_scan[kWarps];
  __shared__ long long sh_found[3];
  __shared__ float sh_qexp[S::kHeads], sh_qmax[kWarps][8];
  __shared__ int sh_last;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  pdl_wait_primary();
  pdl_launch_dependents();

  const long long cap = static_cast<long long>(p.max_pages) * p.page;
  bool bad = false;
  auto length = [&](int b) {
    const int n = p.lens[b];
    if (n < 0 || n > cap) bad = true;
    return n < 0 ? 0 : n > cap ? static_cast<int>(cap) : n;
  };
  const int per_b = p.heads * p.blocks;  // items per sequence
  // Sequences without tokens: zeros and a log sum of -inf.
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    if (length(b) > 0) continue;
    for (int i = tid; i < p.heads * p.G * D; i += kThreads) {
      const int h = i / D;
      put(static_cast<QT*>(p.out) + b * p.o_sb + h * p.o_sh + (i - h * D), 0.0f);
    }
    if (p.lse)
      for (int h = tid; h < p.heads * p.G; h += kThreads) p.lse[b * p.lse_sb + h] = -INFINITY;
  }
  // This CTA's units [t0, t1) of the T units (an item is kItemCost units of set-up,
  // then its tiles), and the sequence that holds t0. Up to kThreads sequences one scan
  // gives both.
  auto tiles_of = [&](int b) {
    const int n = b < p.B ? length(b) : 0;
    return n > 0 ? static_cast<long long>((n + kTile - 1) / kTile + kItemCost) * per_b : 0LL;
  };
  long long n = tiles_of(tid), chunk, T;
  long long incl = block_scan(n, sh_scan, &chunk);
  T = chunk;
  for (int base = kThreads; base < p.B; base += kThreads) {
    long long sum;
    block_scan(tiles_of(base + tid), sh_scan, &sum);
    T += sum;
  }
  if (bad && p.status) atomicOr(p.status, CB_DEVERR_BAD_INDEX);
  const Deal deal(T, static_cast<int>(gridDim.x));
  const int cta = static_cast<int>(blockIdx.x);
  if (cta >= deal.grid) return;
  const long long t0 = deal.start(cta), t1 = deal.start(cta + 1);
  for (long long base = 0, before = 0;;) {
    if (t0 >= incl - n && t0 < incl) {
      sh_found[0] = base + tid;
      sh_found[1] = incl - n;
      sh_found[2] = length(static_cast<int>(base) + tid);
    }
    before += chunk;
    if (t0 < before) break;  // uniform
    base += kThreads;
    n = tiles_of(static_cast<int>(base) + tid);
    incl = block_scan(n, sh_scan, &chunk) + before;
  }
  __syncthreads();
  int b = static_cast<int>(sh_found[0]);
  int len = static_cast<int>(sh_found[2]);
  int tiles = (len + kTile - 1) / kTile;
  const long long in_b = t0 - sh_found[1];
  int item = in_b < (1LL << 31) ? static_cast<int>(static_cast<unsigned>(in_b) / static_cast<unsigned>(tiles + kItemCost))
                                : static_cast<int>(in_b / (tiles + kItemCost));  // item within the sequence
  long long item_at = sh_found[1] + static_cast<long long>(item) * (tiles + kItemCost);  // first unit of the item
  auto next_item = [&] {
    item_at += tiles + kItemCost;
    if (++item == per_b) {
      item = 0;
      if (item_at < t1) {
        do {
          ++b;
          len = length(b);
        } while (len == 0);
        tiles = (len + kTile - 1) / kTile;
      }
    }
  };
  // A short item belongs as a whole to the CTA that holds its first unit.
  if (tiles <= kWholeTiles && t0 > item_at) next_item();
  // this CTA's first tile in the item (0 if the range begins in the set-up units)
  int tile = t0 - item_at > kItemCost ? static_cast<int>(t0 - item_at) - kItemCost : 0;

  for (; item_at + (tiles <= kWholeTiles ? 0 : kItemCost) < t1; next_item(), tile = 0) {
    const long long item_first = item_at + kItemCost;  // unit of the item's first tile
    const int head = item / p.blocks, blk = item - head * p.blocks;
    const int q0 = blk * S::kHeads;                                   // first query of the block, within its group
    const int nq = p.G - q0 < S::kHeads ? p.G - q0 : S::kHeads;       // queries of the block
    const int tile_end =
        tiles <= kWholeTiles || tiles < t1 - item_first ? tiles : static_cast<int>(t1 - item_first);
    const QT* qrow = static_cast<const QT*>(p.q) + b * p.q_sb + static_cast<long long>(head * p.G + q0) * p.q_sh;

    const int* trow = p.table + b * p.table_sb;
    const uint8_t* kbase = static_cast<const uint8_t*>(p.k) + head * p.k_sh;
    const uint8_t* vbase = static_cast<const uint8_t*>(p.v) + head * p.v_sh;
    auto page_of = [&](int tok) { return p.page_shift >= 0 ? tok >> p.page_shift : tok / p.page; };
    // Cache page of a token; -1 past the length or where the table is wrong.
    auto lookup = [&](int tok) {
      if (tok >= len) return -1;
      const int pg = trow[page_of(tok)];
      if (static_cast<unsigned>(pg) >= static_cast<unsigned>(p.num_pages)) {
        if (p.status) atomicOr(p.status, CB_DEVERR_BAD_INDEX);
        return -1;
      }
      return pg;
    };

    // K and V of tile tl for this warp: 16 tokens, rows past the length zero
    uint4 kr[2][S::kKC];
    uint4 vr[4][S::kVC];
    bool k_ok[2];
    int my_pg = -1;  // page of this lane's token (lane & 15); with PAGE16 all 16 share one page
    auto find_page = [&](int tl) {
      const int tok0 = tl * kTile + warp * 16;
      my_pg = lookup(PAGE16 ? tok0 : tok0 + (lane & 15));
    };
    auto load_k = [&](int tl) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int rel = g + 8 * r, tok = tl * kTile + warp * 16 + rel;
        const int pg = PAGE16 ? my_pg : __shfl_sync(0xffffffffu, my_pg, rel);
        k_ok[r] = tok < len && pg >= 0;
        const uint8_t* row = kbase + pg * p.k_sp + static_cast<long long>(tok - page_of(tok) * p.page) * p.k_ss + t * 16;
#pragma unroll
        for (int c = 0; c < S::kKC; ++c) kr[r][c] = k_ok[r] ? ldg16(row + c * 64) : make_uint4(0, 0, 0, 0);
      }
    };
    auto load_v = [&](int tl) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int rel = 2 * t + (r & 1) + 8 * (r >> 1), tok = tl * kTile + warp * 16 + rel;
        const int pg = PAGE16 ? my_pg : __shfl_sync(0xffffffffu, my_pg, rel);
        const bool ok = tok < len && pg >= 0;
        const uint8_t* row =
            vbase + pg * p.v_sp + static_cast<long long>(tok - page_of(tok) * p.page) * p.v_ss + g * S::kVV;
#pragma unroll
        for (int c = 0; c < S::kVC; ++c) {
          if constexpr (S::kVV == 16) {
            vr[r][c] = ok ? ldg16(row + c * 128) : make_uint4(0, 0, 0, 0);
          } else {
            const uint2 two = ok ? ldg8(row + c * 64) : make_uint2(0, 0);
            vr[r][c] = make_uint4(two.x, two.y, 0, 0);
          }
        }
      }
    };
    // this warp's tiles: its 16 tokens of the item's last tile may lie past the length
    const int w_end = (tile_end - 1) * kTile + warp * 16 < len ? tile_end : tile_end - 1;
    // Query fragments: four consecutive elements for each of this thread's k-steps, all
    // of one row; requested before the first tile's keys and values.
    constexpr int kQ = S::kKSteps * NT / kWarps;
    const int q_row = warp % NT * 8 + g;
    auto q_step = [&](int x) { return (x * kWarps + warp) / NT; };
    uint2 qraw[kQ];
#pragma unroll
    for (int x = 0; x < kQ; ++x) {
      // d of the k-step's four elements in lane t: the order of K's 16-byte chunks
      const int ks = q_step(x);
      const int d = FP8 ? (ks >> 2) * 64 + t * 16 + (ks & 3) * 4 : (ks >> 1) * 32 + t * 8 + (ks & 1) * 4;
      const QT* src = qrow + q_row * p.q_sh + d;
      qraw[x] = make_uint2(0, 0);
      if (q_row < nq) {
        if (p.q_vec) {
          qraw[x] = *reinterpret_cast<const uint2*>(src);
        } else {
          QT* e = reinterpret_cast<QT*>(&qraw[x]);
#pragma unroll
          for (int j = 0; j < 4; ++j) e[j] = src[j];
        }
      }
    }
    if (tile < w_end) {
      find_page(tile);
      load_k(tile);
      load_v(tile);
    }
    __syncthreads();  // the previous item is done with the shared memory
    if constexpr (S::kScaleQ) {
      // power of two that brings each query row's largest value to [2^14, 2^15): f16 then
      // holds values down to 2^-28 of it with all of bf16's bits
      float m = 0.0f;
#pragma unroll
      for (int x = 0; x < kQ; ++x) {
        const QT* e = reinterpret_cast<const QT*>(&qraw[x]);
#pragma unroll
        for (int j = 0; j < 4; ++j) m = fmaxf(m, fabsf(q_val(e + j)));
      }
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      if (t == 0) sh_qmax[warp][g] = m;
      __syncthreads();
      if (tid < S::kHeads) {
        float top = 0.0f;
#pragma unroll
        for (int w = tid / 8; w < kWarps; w += NT) top = fmaxf(top, sh_qmax[w][tid % 8]);
        int e = 14;  // an infinite row stays as it is
        if (top > 0.0f && top < INFINITY) e = ilogbf(top);
        if (e < -86) e = -86;  // rows below 2^-86 keep a factor that fp32 holds
        sh_qexp[tid] = ldexpf(1.0f, e - 14);
      }
      __syncthreads();
    }
#pragma unroll
    for (int x = 0; x < kQ; ++x) {
      uint2 frag = qraw[x];
      if constexpr (FP8) {
        const QT* e = reinterpret_cast<const QT*>(&qraw[x]);
        const float f = S::kScaleQ ? 1.0f / sh_qexp[q_row] : 1.0f;
        frag = make_uint2(M::pack(q_val(e) * f, q_val(e + 1) * f), M::pack(q_val(e + 2) * f, q_val(e + 3) * f));
      }
      sh_q[(q_step(x) * NT + warp % NT) * 32 + lane] = frag;
    }
    __syncthreads();
    float zs[NT][2];  // score factor of this lane's two heads
    const float ks_head = FP8 && p.k_scale ? p.k_scale[head] : 1.0f;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        zs[n][j] = p.scale * kLog2e;
        if constexpr (FP8) zs[n][j] = p.scale * ks_head * kLog2e * (S::kScaleQ ? sh_qexp[n * 8 + 2 * t + j] : 1.0f);
      }

    float o[S::kKSteps][NT][4];
    float m_run[NT][2], l_run[NT][2];
#pragma unroll
    for (int i = 0; i < S::kKSteps; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][n][j] = 0.0f;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) m_run[n][j] = -INFINITY, l_run[n][j] = 0.0f;

    for (int tl = tile; tl < w_end; ++tl) {
      // ---- scores ----
      float s[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][j] = 0.0f;
#pragma unroll
      for (int c = 0; c < S::kKC; ++c) {
        const uint32_t* w0 = reinterpret_cast<const uint32_t*>(&kr[0][c]);
        const uint32_t* w1 = reinterpret_cast<const uint32_t*>(&kr[1][c]);
#pragma unroll
        for (int i = 0; i < (FP8 ? 4 : 2); ++i) {
          uint32_t a0, a1, a2, a3;
          if constexpr (FP8) {
            a0 = e4m3x2_f16x2(w0[i]), a1 = e4m3x2_f16x2(w1[i]);
            a2 = e4m3x2_f16x2(w0[i] >> 16), a3 = e4m3x2_f16x2(w1[i] >> 16);
          } else {
            a0 = w0[2 * i], a1 = w1[2 * i], a2 = w0[2 * i + 1], a3 = w1[2 * i + 1];
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint2 bq = sh_q[((c * (FP8 ? 4 : 2) + i) * NT + n) * 32 + lane];
            M::mma(s[n], a0, a1, a2, a3, bq.x, bq.y);
          }
        }
      }
      const bool ok[2] = {k_ok[0], k_ok[1]};
      if (tl + 1 < w_end) {
        find_page(tl + 1);
        load_k(tl + 1);
      }
      // ---- running maximum and sum ----
      uint32_t pb[NT][2], pr[NT][2];  // the probabilities' leading and remaining terms
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float x[4], mx[2];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = ok[j >> 1] ? s[n][j] * zs[n][j & 1] : -INFINITY;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          mx[j] = fmaxf(x[j], x[2 + j]);
#pragma unroll
          for (int sft = 4; sft < 32; sft <<= 1) mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], sft));
          mx[j] = fmaxf(mx[j], m_run[n][j]);
        }
        float al[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float ref = mx[j] == -INFINITY ? 0.0f : mx[j];
          al[j] = exp2_approx(m_run[n][j] - ref);
          m_run[n][j] = mx[j];
          x[j] = exp2_approx(x[j] - ref + S::kShift);
          x[2 + j] = exp2_approx(x[2 + j] - ref + S::kShift);
          l_run[n][j] = l_run[n][j] * al[j] + (x[j] + x[2 + j]);
        }
        if (__any_sync(0xffffffffu, al[0] != 1.0f || al[1] != 1.0f)) {
#pragma unroll
          for (int i = 0; i < S::kKSteps; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][n][j] *= al[j & 1];
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          uint32_t rest;
          pb[n][r] = movmatrix_trans(M::split(x[2 * r], x[2 * r + 1], rest));
          pr[n][r] = movmatrix_trans(rest);
        }
      }
      // ---- output ----
#pragma unroll
      for (int c = 0; c < S::kVC; ++c) {
        const uint32_t* v0 = reinterpret_cast<const uint32_t*>(&vr[0][c]);
        const uint32_t* v1 = reinterpret_cast<const uint32_t*>(&vr[1][c]);
        const uint32_t* v2 = reinterpret_cast<const uint32_t*>(&vr[2][c]);
        const uint32_t* v3 = reinterpret_cast<const uint32_t*>(&vr[3][c]);
#pragma unroll
        for (int w = 0; w < S::kVV / 4; ++w) {
          if constexpr (FP8) {
#pragma unroll
            for (int hl = 0; hl < 2; ++hl) {
              const uint32_t lo = __byte_perm(v0[w], v1[w], hl ? 0x7362 : 0x5140);
              const uint32_t hi = __byte_perm(v2[w], v3[w], hl ? 0x7362 : 0x5140);
              const uint32_t a0 = e4m3x2_f16x2(lo), a1 = e4m3x2_f16x2(lo >> 16);
              const uint32_t a2 = e4m3x2_f16x2(hi), a3 = e4m3x2_f16x2(hi >> 16);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                M::mma(o[(c * (S::kVV / 4) + w) * 2 + hl][n], a0, a1, a2, a3, pb[n][0], pb[n][1]);
                M::mma(o[(c * (S::kVV / 4) + w) * 2 + hl][n], a0, a1, a2, a3, pr[n][0], pr[n][1]);
              }
            }
          } else {
            const uint32_t a0 = __byte_perm(v0[w], v1[w], 0x5410), a1 = __byte_perm(v0[w], v1[w], 0x7632);
            const uint32_t a2 = __byte_perm(v2[w], v3[w], 0x5410), a3 = __byte_perm(v2[w], v3[w], 0x7632);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              M::mma(o[c * (S::kVV / 4) + w][n], a0, a1, a2, a3, pb[n][0], pb[n][1]);
              M::mma(o[c * (S::kVV / 4) + w][n], a0, a1, a2, a3, pr[n][0], pr[n][1]);
            }
          }
        }
      }
      if (tl + 1 < w_end) load_v(tl + 1);
    }

    // ---- join the warps ----
    float* mine = sh_part + warp * S::kPartSh;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int sft = 4; sft < 32; sft <<= 1) l_run[n][j] += __shfl_xor_sync(0xffffffffu, l_run[n][j], sft);
        const int r = n * 8 + 2 * t + j;
        if (g == 0) {
          mine[r] = m_run[n][j];
          mine[S::kHeads + r] = l_run[n][j];
        }
#pragma unroll
        for (int i = 0; i < S::kKSteps; ++i) {
          // the two d of m-tile i in lane g: elements 2i and 2i + 1 of the lane's V bytes
          constexpr int per = S::kVV / S::kElem;  // elements of one load
          const int e = 2 * i, c = e / per;
          const int d = c * per * 8 + g * per + e % per;
          mine[2 * S::kHeads + r * S::kPitch + d] = o[i][n][j];
          mine[2 * S::kHeads + r * S::kPitch + d + 1] = o[i][n][2 + j];
        }
      }
    __syncthreads();
    const bool whole = tile == 0 && tile_end == tiles;
    QT* orow = static_cast<QT*>(p.out) + b * p.o_sb + static_cast<long long>(head * p.G + q0) * p.o_sh;
    float* lrow = p.lse ? p.lse + b * p.lse_sb + head * p.G + q0 : nullptr;
    const float vs = FP8 && p.v_scale ? p.v_scale[head] : 1.0f;
    auto join_warps = [&](bool finish, float* dst) {
      for (int i = tid; i < nq * D; i += kThreads) {
        const int r = i / D, d = i - r * D;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sh_part[w * S::kPartSh + r]);
        const float ref = mx == -INFINITY ? 0.0f : mx;
        float sum = 0.0f, acc = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float* pt = sh_part + w * S::kPartSh;
          const float f = exp2_approx(pt[r] - ref);
          sum = fmaf(f, pt[S::kHeads + r], sum);
          acc = fmaf(f, pt[2 * S::kHeads + r * S::kPitch + d], acc);
        }
        if (finish) {
          put(orow + r * p.o_sh + d, sum == 0.0f ? 0.0f : acc / sum * vs);
          if (lrow && d == 0) lrow[r] = sum == 0.0f ? -INFINITY : (mx + log2f(sum) - S::kShift) * kLn2;
        } else {
          dst[2 * S::kHeads + r * D + d] = acc;
          if (d == 0) dst[r] = mx, dst[S::kHeads + r] = sum;
        }
      }
    };
    // A cut item's parts, joined in CTA order, kJoin at a time: their maxima and sums
    // go to shared memory in one round trip; each thread adds its float4s of the output
    // with the loads of several parts in flight, against a running maximum per head.
    auto join_parts = [&](auto&& part_of, int n_parts) {
      constexpr int kJoin = 32;
      float* const sh_m = sh_part;                          // [kJoin][kHeads]
      float* const sh_l = sh_part + kJoin * S::kHeads;      // [kJoin][kHeads]
      static_assert(2 * kJoin * S::kHeads <= kWarps * S::kPartSh, "maxima and sums must fit");
      constexpr int kF4 = (S::kHeads * D / 4 + kThreads - 1) / kThreads;  // float4s of a thread
      constexpr int kAhead = kF4 > 2 ? 4 : 8;                                  // parts whose loads are in flight
      float4 acc[kF4];
      float mx[kF4], sum[kF4];
#pragma unroll
      for (int x = 0; x < kF4; ++x) acc[x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f), mx[x] = -INFINITY, sum[x] = 0.0f;
      for (int w0 = 0; w0 < n_parts; w0 += kJoin) {
        const int here = n_parts - w0 < kJoin ? n_parts - w0 : kJoin;
        __syncthreads();
        for (int i = tid; i < here * S::kHeads; i += kThreads) {
          const float* pt = part_of(w0 + i / S::kHeads) + i % S::kHeads;
          sh_m[i] = __ldcg(pt);
          sh_l[i] = __ldcg(pt + S::kHeads);
        }
        __syncthreads();
        float ref[kF4];
#pragma unroll
        for (int x = 0; x < kF4; ++x) {
          const int r = (x * kThreads + tid) * 4 / D;
          float top = mx[x];
          for (int w = 0; w < here; ++w) top = fmaxf(top, sh_m[w * S::kHeads + r]);
          ref[x] = top == -INFINITY ? 0.0f : top;
          const float f0 = exp2_approx(mx[x] - ref[x]);
          acc[x].x *= f0, acc[x].y *= f0, acc[x].z *= f0, acc[x].w *= f0, sum[x] *= f0;
          mx[x] = top;
        }
        for (int w = 0; w < here; w += kAhead) {
          float4 v[kAhead][kF4];
#pragma unroll
          for (int y = 0; y < kAhead; ++y)
#pragma unroll
            for (int x = 0; x < kF4; ++x) {
              const int e = (x * kThreads + tid) * 4;
              v[y][x] = w + y < here && e < nq * D
                            ? __ldcg(reinterpret_cast<const float4*>(part_of(w0 + w + y) + 2 * S::kHeads + e))
                            : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
#pragma unroll
          for (int y = 0; y < kAhead; ++y) {
            if (w + y >= here) break;
#pragma unroll
            for (int x = 0; x < kF4; ++x) {
              const int r = (x * kThreads + tid) * 4 / D;
              const float f = exp2_approx(sh_m[(w + y) * S::kHeads + r] - ref[x]);
              sum[x] = fmaf(f, sh_l[(w + y) * S::kHeads + r], sum[x]);
              acc[x].x = fmaf(f, v[y][x].x, acc[x].x), acc[x].y = fmaf(f, v[y][x].y, acc[x].y);
              acc[x].z = fmaf(f, v[y][x].z, acc[x].z), acc[x].w = fmaf(f, v[y][x].w, acc[x].w);
            }
          }
        }
      }
#pragma unroll
      for (int x = 0; x < kF4; ++x) {
        const int e = (x * kThreads + tid) * 4, r = e / D, d = e % D;
        if (r >= nq) break;
        const float f = sum[x] == 0.0f ? 0.0f : vs / sum[x];
        const float v[4] = {acc[x].x, acc[x].y, acc[x].z, acc[x].w};
#pragma unroll
        for (int y = 0; y < 4; ++y) put(orow + r * p.o_sh + d + y, sum[x] == 0.0f ? 0.0f : v[y] * f);
        if (lrow && d == 0) lrow[r] = sum[x] == 0.0f ? -INFINITY : (mx[x] + log2f(sum[x]) - S::kShift) * kLn2;
      }
    };
    if (whole) {
      join_warps(true, nullptr);
    } else {
      // CTAs that hold the item's first and last tile
      const long long last_tile = item_first + tiles - 1;
      const int c_first = deal.owner(item_first), c_last = deal.owner(last_tile);
      // slot 0: the item began in an earlier CTA (this CTA's first segment); 1: it begins here
      auto slot = [&](int c) { return p.partials + (static_cast<long long>(c) * 2 + (c == c_first ? 1 : 0)) * S::kPart; };
      join_warps(false, slot(cta));
      if (p.join_apart) continue;  // join_kernel follows
      __syncthreads();
      if (tid == 0) {
        __threadfence();  // covers the CTA's stores before the barrier
        sh_last = atomicAdd(&p.counters[c_first], 1) == c_last - c_first;
      }
      __syncthreads();
      if (sh_last) {
        __threadfence();
        join_parts([&](int w) { return slot(c_first + w); }, c_last - c_first + 1);
        if (tid == 0) p.counters[c_first] = 0;  // the next launch starts from zero
      }
    }
  }
}

// Joins the parts of cut items in a launch of its own, where few items have many parts
// each (one CTA would read them all): a CTA per item and head, D / 4 threads per part.
template <typename QT, bool FP8, int D, int NT>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const AttnParams p) {
  using S = Shape<QT, FP8, D, NT>;
  constexpr int kLanes = D / 4, kGroups = kJoinThreads / kLanes, kAhead = 8;
  __shared__ float sh_m[kGroups], sh_l[kGroups];
  __shared__ float4 sh_v[kGroups][kLanes];
  const int tid = threadIdx.x, lane = tid & 31;
  const int per_b = p.heads * p.blocks;
  const int b = blockIdx.x / per_b, item = blockIdx.x - b * per_b;
  const int head = item / p.blocks, q0 = (item - head * p.blocks) * S::kHeads, r = blockIdx.y;
  pdl_wait_primary();
  pdl_launch_dependents();
  if (q0 + r >= p.G) return;
  // the same dealing out as the kernel before (B <= 32: every lane one sequence)
  const long long cap = static_cast<long long>(p.max_pages) * p.page;
  long long units = 0, mine = 0;
  int tiles = 0;
  if (lane < p.B) {
    const int n = p.lens[lane];
    const long long len = n < 0 ? 0 : n > cap ? cap : n;
    tiles = static_cast<int>((len + kTile - 1) / kTile);
    units = tiles > 0 ? static_cast<long long>(tiles + kItemCost) * per_b : 0;
    mine = lane < b ? units : 0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    units += __shfl_xor_sync(0xffffffffu, units, o);
    mine += __shfl_xor_sync(0xffffffffu, mine, o);
  }
  tiles = __shfl_sync(0xffffffffu, tiles, b);
  if (tiles <= kWholeTiles) return;
  const Deal deal(units, p.grid);
  const long long first = mine + static_cast<long long>(item) * (tiles + kItemCost) + kItemCost;
  const int c_first = deal.owner(first);
  const int n_parts = deal.owner(first + tiles - 1) - c_first + 1;
  if (n_parts == 1) return;  // stored by its CTA
  auto part_of = [&](int w) { return p.partials + (static_cast<long long>(c_first + w) * 2 + (w == 0 ? 1 : 0)) * S::kPart; };

  const int group = tid / kLanes, e = tid % kLanes;
  float mx = -INFINITY, sum = 0.0f;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int w0 = group; w0 < n_parts; w0 += kGroups * kAhead) {
    float m[kAhead], l[kAhead];
    float4 v[kAhead];
#pragma unroll
    for (int y = 0; y < kAhead; ++y) {
      const bool in = w0 + y * kGroups < n_parts;
      const float* pt = part_of(in ? w0 + y * kGroups : w0);
      m[y] = in ? __ldcg(pt + r) : -INFINITY;
      l[y] = in ? __ldcg(pt + S::kHeads + r) : 0.0f;
      v[y] = __ldcg(reinterpret_cast<const float4*>(pt + 2 * S::kHeads + r * D) + e);
    }
    float top = mx;
#pragma unroll
    for (int y = 0; y < kAhead; ++y) top = fmaxf(top, m[y]);
    const float ref = top == -INFINITY ? 0.0f : top;
    const float f0 = exp2_approx(mx - ref);
    mx = top;
    acc.x *= f0, acc.y *= f0, acc.z *= f0, acc.w *= f0, sum *= f0;
#pragma unroll
    for (int y = 0; y < kAhead; ++y) {
      if (w0 + y * kGroups >= n_parts) break;
      const float f = exp2_approx(m[y] - ref);
      sum = fmaf(f, l[y], sum);
      acc.x = fmaf(f, v[y].x, acc.x), acc.y = fmaf(f, v[y].y, acc.y);
      acc.z = fmaf(f, v[y].z, acc.z), acc.w = fmaf(f, v[y].w, acc.w);
    }
  }
  sh_v[group][e] = acc;
  if (e == 0) sh_m[group] = mx, sh_l[group] = sum;
  __syncthreads();
  if (group != 0) return;
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < kGroups; ++w) top = fmaxf(top, sh_m[w]);
  const float ref = top == -INFINITY ? 0.0f : top;
  acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  sum = 0.0f;
#pragma unroll
  for (int w = 0; w < kGroups; ++w) {
    const float f = exp2_approx(sh_m[w] - ref);
    const float4 u = sh_v[w][e];
    sum = fmaf(f, sh_l[w], sum);
    acc.x = fmaf(f, u.x, acc.x), acc.y = fmaf(f, u.y, acc.y), acc.z = fmaf(f, u.z, acc.z), acc.w = fmaf(f, u.w, acc.w);
  }
  const int hq = head * p.G + q0 + r;
  const float vs = FP8 && p.v_scale ? p.v_scale[head] : 1.0f;
  const float f = sum == 0.0f ? 0.0f : vs / sum;
  const float o[4] = {acc.x, acc.y, acc.z, acc.w};
  QT* out = static_cast<QT*>(p.out) + b * p.o_sb + static_cast<long long>(hq) * p.o_sh + e * 4;
#pragma unroll
  for (int y = 0; y < 4; ++y) put(out + y, sum == 0.0f ? 0.0f : o[y] * f);
  if (p.lse && e == 0) p.lse[b * p.lse_sb + hq] = sum == 0.0f ? -INFINITY : (top + log2f(sum) - S::kShift) * kLn2;
}

template <typename QT, bool FP8, int D, int NT, bool PAGE16>
int launch_kernel(AttnParams p, long long most, cudaStream_t stream) {
  using S = Shape<QT, FP8, D, NT>;
  auto kernel = attn_kernel<QT, FP8, D, NT, PAGE16>;
  static thread_local int configured_dev = -1, per_sm = 1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (configured_dev != dev) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(S::kSmem)) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kThreads, S::kSmem) != cudaSuccess)
      return CB_ERR_CUDA;
    if (per_sm < 1) per_sm = 1;
    if (per_sm > kCtasPerSm) per_sm = kCtasPerSm;
    configured_dev = dev;
  }
  // every SM's share of CTAs, but no more than there can be units of work
  long long grid = static_cast<long long>(sm_count()) * per_sm;
  if (grid > kMaxGrid) grid = kMaxGrid;
  if (grid > most) grid = most < 1 ? 1 : most;
  const long long items = static_cast<long long>(p.B) * p.heads * p.blocks;
  p.grid = static_cast<int>(grid);
  p.join_apart = p.B <= 32 && grid >= items * kPartsApart;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e != cudaSuccess || !p.join_apart) return cuda_status(e);
  cfg.gridDim = dim3(static_cast<unsigned>(items), p.G < S::kHeads ? p.G : S::kHeads);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.dynamicSmemBytes = 0;
  return cuda_status(cudaLaunchKernelEx(&cfg, join_kernel<QT, FP8, D, NT>, p));
}


int attn_grid_limit() {
  int sms = sm_count();
  if (sms <= 0) sms = 148;
  const int g = sms * kCtasPerSm;
  return g < kMaxGrid ? g : kMaxGrid;
}

// Head blocks of 16 queries where a group has more than 8 and the output of 16
// fits the registers (D <= 128), else of 8.
int head_tiles(int G, int D) { return G > 8 && D <= 128 ? 2 : 1; }

template <typename QT, bool FP8, int D>
int dispatch_nt(const AttnParams& p, int nt, bool page16, long long most, cudaStream_t s) {
  if constexpr (D <= 128) {
    if (nt == 2)
      return page16 ? launch_kernel<QT, FP8, D, 2, true>(p, most, s) : launch_kernel<QT, FP8, D, 2, false>(p, most, s);
  }
  return page16 ? launch_kernel<QT, FP8, D, 1, true>(p, most, s) : launch_kernel<QT, FP8, D, 1, false>(p, most, s);
}

template <typename QT, bool FP8>
int dispatch_d(const AttnParams& p, int D, int nt, bool page16, long long most, cudaStream_t s) {
  if (D == 64) return dispatch_nt<QT, FP8, 64>(p, nt, page16, most, s);
  if (D == 128) return dispatch_nt<QT, FP8, 128>(p, nt, page16, most, s);
  return dispatch_nt<QT, FP8, 256>(p, nt, page16, most, s);
}

size_t part_bytes(int G, int D) {
  const size_t heads = 8 * static_cast<size_t>(head_tiles(G, D));
  return sizeof(float) * (heads * 2 + heads * D);
}

}  // namespace

size_t paged_attention_workspace_bytes(int64_t Hq, int64_t Hkv, int64_t D) {
  if (Hkv < 1 || Hq < Hkv || D < 1 || D > 256) return 0;
  return workspace_need(attn_grid_limit(), part_bytes(static_cast<int>(Hq / Hkv), static_cast<int>(D)));
}

}  // namespace cb

using namespace cb;

extern "C" CB_API int cb_paged_decode_attention(const void* q, int q_dtype, const void* k_cache, const void* v_cache,
                                                int cache_dtype, const float* k_scale, const float* v_scale,
                                                const int* block_table, const int* seq_lens, float scale, void* out,
                                                float* lse, int64_t B, int64_t Hq, int64_t Hkv, int64_t D,
                                                int64_t num_pages, int64_t page_size, int64_t max_pages,
                                                const int64_t* strides, void* workspace, size_t workspace_bytes,
                                                cb_stream_t stream) {
  if (B < 0 || Hq < 0 || Hkv < 0 || num_pages < 0 || page_size < 1 || max_pages < 0) return CB_ERR_INVALID_ARG;
  if (B == 0 || Hq == 0) return CB_OK;
  if (!q || !seq_lens || !out || !strides) return CB_ERR_INVALID_ARG;
  if (max_pages > 0 && !block_table) return CB_ERR_INVALID_ARG;
  if (num_pages > 0 && (!k_cache || !v_cache)) return CB_ERR_INVALID_ARG;
  if (q_dtype != CB_DTYPE_BF16 && q_dtype != CB_DTYPE_F16) return CB_ERR_DTYPE;
  if (cache_dtype != q_dtype && cache_dtype != CB_DTYPE_E4M3) return CB_ERR_DTYPE;
  const bool fp8 = cache_dtype == CB_DTYPE_E4M3;
  if (!fp8 && (k_scale || v_scale)) return CB_ERR_INVALID_ARG;
  if ((D != 64 && D != 128 && D != 256) || Hkv < 1 || Hq % Hkv != 0) return CB_ERR_SHAPE;
  if (B > (1 << 24) || Hq > 65536 || num_pages > 0x7fffffffLL || page_size > 0x7fffffffLL ||
      max_pages > 0x7fffffffLL || max_pages * page_size > 0x7fffff00LL)
    return CB_ERR_TOO_LARGE;
  const int64_t e = fp8 ? 1 : 2;
  // a dimension of one has no stride: what is given there is not looked at
  const int64_t size[12] = {B, Hq, B, Hq, B, B, num_pages, page_size, Hkv, num_pages, page_size, Hkv};
  int64_t st[12];
  for (int i = 0; i < 12; ++i) {
    st[i] = size[i] == 1 ? 0 : strides[i];
    if (st[i] < 0) return CB_ERR_STRIDE;
  }
  // cache rows are read in 16-byte vectors
  if (!aligned16(k_cache) || !aligned16(v_cache)) return CB_ERR_ALIGNMENT;
  for (int i = 6; i < 12; ++i)
    if ((st[i] * e) % 16 != 0) return CB_ERR_ALIGNMENT;
  const int G = static_cast<int>(Hq / Hkv);
  const int nt = head_tiles(G, static_cast<int>(D));
  AttnParams p = {};
  p.q = q, p.k = k_cache, p.v = v_cache, p.table = block_table, p.lens = seq_lens;
  p.k_scale = k_scale, p.v_scale = v_scale, p.out = out, p.lse = lse, p.scale = scale;
  p.B = static_cast<int>(B), p.heads = static_cast<int>(Hkv), p.G = G;
  p.blocks = (G + 8 * nt - 1) / (8 * nt);
  p.num_pages = static_cast<int>(num_pages), p.page = static_cast<int>(page_size);
  p.max_pages = static_cast<int>(max_pages);
  p.q_vec = (reinterpret_cast<uintptr_t>(q) & 7u) == 0 && st[0] % 4 == 0 && st[1] % 4 == 0;
  p.page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (page_size == (1LL << s)) p.page_shift = s;
  p.q_sb = st[0], p.q_sh = st[1], p.o_sb = st[2], p.o_sh = st[3];
  p.lse_sb = st[4], p.table_sb = st[5];
  p.k_sp = st[6] * e, p.k_ss = st[7] * e, p.k_sh = st[8] * e;
  p.v_sp = st[9] * e, p.v_ss = st[10] * e, p.v_sh = st[11] * e;
  const long long cap = max_pages * page_size;
  const long long most = B * Hkv * p.blocks * ((cap + kTile - 1) / kTile + kItemCost);
  const size_t need = workspace_need(attn_grid_limit(), part_bytes(G, static_cast<int>(D)));
  if (!workspace || workspace_bytes < need) return CB_ERR_WORKSPACE;
  Workspace ws = carve_workspace(workspace, attn_grid_limit());
  p.status = ws.status, p.counters = ws.counters, p.partials = static_cast<float*>(ws.partials);
  const bool page16 = page_size % 16 == 0;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (q_dtype == CB_DTYPE_BF16)
    return fp8 ? dispatch_d<__nv_bfloat16, true>(p, static_cast<int>(D), nt, page16, most, s)
               : dispatch_d<__nv_bfloat16, false>(p, static_cast<int>(D), nt, page16, most, s);
  return fp8 ? dispatch_d<__half, true>(p, static_cast<int>(D), nt, page16, most, s)
             : dispatch_d<__half, false>(p, static_cast<int>(D), nt, page16, most, s);
}
