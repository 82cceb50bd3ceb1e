// The 4-bit caches (gct_fp4.h): rows read back, rows appended to the camera head's caches, and attention of a few query rows over
// either cache.
#include <math.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "gct_fp4.h"
#include "gct_sm100.h"

namespace gct {
namespace {

// ---- rows read back -------------------------------------------------------------------------------------------

// One thread per (token, head, block of 16, K or V): 8 bytes of values and a scale in, 16 numbers and a scale out.  Neighbouring threads
// take neighbouring blocks of a row, then heads: writes are coalesced, reads are whole 32-byte rows.
template <int D, bool kProducts>
__global__ void __launch_bounds__(256) gct_fp4_read_kernel(const Fp4ReadLaunch p) {
  pdl_wait();
  constexpr int kGroups = D / kFp4Group;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, each = static_cast<int64_t>(p.tokens) * p.heads * kGroups;
  if (i >= 2 * each) return;
  const int kv = i >= each;
  const int64_t at = kv ? i - each : i;
  const int group = static_cast<int>(at % kGroups), h = static_cast<int>(at / kGroups % p.heads), token = static_cast<int>(at / kGroups / p.heads);
  int page, slot;
  if (token >= p.num_special) {
    page = p.at.patch_page;
    slot = p.first + token - p.num_special;
  } else if (token < p.at.sp_n0) {
    page = p.at.sp_page0;
    slot = p.at.sp_off0 + token;
  } else {
    page = p.at.sp_page1;
    slot = token - p.at.sp_n0;
  }
  if (page < 0 || page >= p.num_pages || slot < 0 || slot >= p.page_rows) {
    if (p.status != nullptr) atomicCAS(p.status, 0, kStatusBadIndex);
    return;
  }
  const uint8_t* base = p.v_pool != nullptr ? (kv ? p.v_pool : p.pool) + h * p.layout.bytes
                                            : p.pool + ((static_cast<int64_t>(page) * 2 + kv) * p.heads + h) * p.layout.bytes;
  const Fp4At from = fp4_at<D>(slot, p.layout.full_blocks, p.layout.tail_rows);
  const uint2 w = *reinterpret_cast<const uint2*>(base + from.values + 8 * group);
  const uint32_t scale = static_cast<uint32_t>(base[from.scales + group]) << 7;
  uint32_t c[8];
  fp4_unpack8(w.x, *reinterpret_cast<uint32_t(*)[4]>(&c[0]));
  fp4_unpack8(w.y, *reinterpret_cast<uint32_t(*)[4]>(&c[4]));
  uint32_t o[8];
  if constexpr (kProducts) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t product = half2_mul(c[e], scale | scale << 16);         // exact in half precision, and in bf16
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&product));
      o[e] = pack_bf16x2(f.x, f.y);
    }
    uint4* dst = reinterpret_cast<uint4*>(p.products[kv] + at * kFp4Group);
    dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
    dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {                                            // e4m3 holds every value
      uint32_t r;
      asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f16x2 lo, %1;\n\tcvt.rn.satfinite.e4m3x2.f16x2 hi, %2;\n\tmov.b32 %0, {lo, hi};\n\t}"
          : "=r"(r) : "r"(c[2 * e]), "r"(c[2 * e + 1]));
      o[e] = r;
    }
    *reinterpret_cast<uint4*>(p.values[kv] + at * kFp4Group) = make_uint4(o[0], o[1], o[2], o[3]);
    p.scales[kv][at] = __ushort_as_half(static_cast<unsigned short>(scale));
  }
}

// ---- rows appended to the camera head's caches ------------------------------------------------------------------

// Sixteen values of a row, fp32 at `src` (16-byte aligned): their two words and their scale byte.
struct Fp4Group16 {
  uint32_t w[2], scale;
  __device__ __forceinline__ void quantise(const float* src) {
    float x[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 f = *reinterpret_cast<const float4*>(src + 4 * i);
      x[4 * i] = f.x;
      x[4 * i + 1] = f.y;
      x[4 * i + 2] = f.z;
      x[4 * i + 3] = f.w;
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, fp4_abs_bits(x[i]));
    scale = fp4_scale_byte(top);
    const float s = fp4_scale(scale), r = fp4_reciprocal(s);
    w[0] = fp4_pack8(x, s, r);
    w[1] = fp4_pack8(x + 8, s, r);
  }
  __device__ __forceinline__ void store(uint8_t* values, uint8_t* scale_at) const {
    *reinterpret_cast<uint2*>(values) = make_uint2(w[0], w[1]);
    *scale_at = static_cast<uint8_t>(scale);
  }
};

template <int D>
__global__ void __launch_bounds__(128) gct_fp4_rows_append_kernel(const float* __restrict__ k, const float* __restrict__ v, int rows, uint8_t* cache_k,
                                                                  uint8_t* cache_v, int full_blocks, int64_t head_bytes, int first, int heads) {
  pdl_wait();
  constexpr int kGroups = D / kFp4Group;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x, each = static_cast<int64_t>(rows) * heads * kGroups;
  if (i >= 2 * each) return;
  const bool is_v = i >= each;
  const int64_t at = is_v ? i - each : i;
  const int group = static_cast<int>(at % kGroups), h = static_cast<int>(at / kGroups % heads);
  const int64_t row = at / kGroups / heads;
  Fp4Group16 q;
  q.quantise((is_v ? v : k) + at * kFp4Group);
  uint8_t* base = (is_v ? cache_v : cache_k) + h * head_bytes;
  const Fp4At to = fp4_at<D>(first + row, full_blocks, 0);
  q.store(base + to.values + 8 * group, base + to.scales + group);
}

// ---- attention of a few query rows --------------------------------------------------------------------------------
//
// softmax(q k^T / sqrt(D)) v for eight query rows of a head at a time, over the pages of the paged cache or over a camera head's
// cache and the call's own new rows.  There is almost nothing to compute: a call reads every row of the cache once (4.5 bits a value), so
// what counts is how few instructions a value costs between its arrival and the sum.
//
//  * Four warps compute; a fifth fetches blocks (one bulk copy for K, one for V) into a ring of stages.
//  * Products on mma.sync m16n8k16 in half precision, fp32 sums.  q k^T has the queries as its sixteen rows: the upper eight hold q rounded
//    to half precision, the lower eight what the rounding left, so the sum of both halves is a product with 22 bits of q (q is brought to
//    [2^14, 2^15) by a power of two per row) at the price of one.  (p v)^T has d as its rows and the queries as its eight columns, once with
//    the weights exp2(x - max + 15) and once with their rests.  Results agree with fp32 arithmetic to about 2^-21.  With the queries as rows
//    of p v its sums took twice the registers.  The paged cache's calls take bf16 queries, which leave no rest, and give bf16 results, for
//    which a weight's eleven bits are enough (at most 2^-11 of sum p |v|, an eighth of the result's own rounding): no rests there.
//  * Any order of d is right for q k^T and any order of keys and of d for p v, as long as both operands agree.  A lane takes a
//    quarter row of K as one 8- or 16-byte load (the d that it multiplies are its own), and of V an eighth of a row of the keys t, t+4,
//    t+8, t+12: keys are numbered so that the logits of a lane's query are, without an exchange, the right operand of (p v)^T.
//  * V's operand pairs two keys at one d.  Two words of two keys are woven into words whose bytes hold (key a, key b) with two logical
//    operations and a shift each, before a single conversion makes the pair; a weave after the conversion costs twice that.
//
// One query over 131,928 tokens of 16 heads (152 MB) 39.7 us, 3.8 TB/s, 0.59 of a copy's rate; eight 44.4; one over 10,000 cached rows of
// 16 heads with D = 128 (23 MB, from L2) 12.0 us.  Issue slots bound the first (61 % busy; the copies alone take 29.5 us); the second is a start,
// five blocks or fewer per CTA, and the join of the ranges (9.8 us without computing anything).
constexpr int kRowsWarps = 4;
// Keys of a block that a warp takes per turn.  64: two pairs of warps take blocks by turns, which halves what a warp does once per turn (the
// wait, maximum, vote and shift: some seventy instructions beside five a key); when it was chosen, one query over 131,928 tokens 60.5 us with 32,
// 47.8 with 64.
// 32: all four warps share a block; right for the camera head's short ranges of a few blocks per CTA (1,000 cached tokens 9.2 us, with 64 11.9).
template <bool kPaged>
constexpr int kTurnKeys = kPaged ? 64 : 32;
constexpr int kRowsThreads = 32 * (kRowsWarps + 1);
constexpr float kWeightShift = 15.f;       // weights are at most 2^15

// CTAs that share an SM: five warps of 96 (128) registers each, and 41 (74) KB.  Five CTAs at D = 64 (72 registers, 32 bytes spilled): one query
// over 131,928 tokens 50.6 us, with four 46.4 (before the last steps on either).
template <int D>
constexpr int kRowsCtas = D == 64 ? 4 : 3;

template <int D, bool kPaged>
struct RowsSmem {
  static constexpr int kStages = D == 64 ? 4 : 3;
  static constexpr int kBlock = kFp4BlockBytes<D>;
  static constexpr int new_off = kStages * 2 * kBlock;            // the call's own rows, a block of K and one of V
  static constexpr int new_bytes = kPaged ? 0 : 2 * kBlock;
  static constexpr int stat_off = new_off + new_bytes;            // [warps][8] maximum and sum
  static constexpr int bar_off = stat_off + kRowsWarps * 8 * 2 * 4;
  static constexpr int misc_off = bar_off + 2 * kStages * 8;
  static constexpr int total = misc_off + 16;
  static constexpr int out_off = 0;                               // [warps][8][D] partial outputs, over the ring when it has been read
  static_assert(kRowsWarps * 8 * D * 4 <= new_off, "partial outputs do not fit the ring");
  // the merge of the key ranges: sums of at most 256 lanes over the ring
  static_assert(8 * D / 4 * 32 <= new_off && 128 * 32 <= new_off, "lane sums do not fit the ring");
};

// Floats of a key range's partial result of a query: sums, maximum, sum of weights, and two that make it a multiple of sixteen bytes.
template <int D>
constexpr int kRowsRecord = D + 4;

struct RowsArgs {
  const void* q;
  int q_f32, q_round_bf16, n_q, heads, groups, splits;
  const uint8_t* pool;
  const int32_t* page_table;
  int n_pages, num_pages, page_rows, last_page_rows, blocks_per_page;
  uint8_t *cache_k, *cache_v;
  int cached, blocks, full_blocks, tail_rows;
  int64_t head_bytes;
  const float *k_new, *v_new;
  int n_new, store;
  float scale_log2;
  __nv_bfloat16* out_bf16;
  float *out_f32, *lse, *part;
  int* counters;
  int* status;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// (hi, rest) of a pair
__device__ __forceinline__ void split_f16(float x, float y, uint32_t& hi, uint32_t& rest) {
  hi = pack_f16x2(x, y);
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  rest = pack_f16x2(x - f.x, y - f.y);
}

// Ranges in flight where they are joined: with five, eight queries at D = 128 took 4 us longer, with 13 up to 1.5 us.
constexpr int kJoinAhead = 9;

template <int D, bool kPaged>
__global__ void __launch_bounds__(kRowsThreads, kRowsCtas<D>) gct_fp4_rows_kernel(const RowsArgs a, const __grid_constant__ Fp4Pages pages) {
  using L = RowsSmem<D, kPaged>;
  constexpr bool kRest = !kPaged;                // the second half-precision part of queries and weights
  constexpr int kKeys = kTurnKeys<kPaged>, kStages = L::kStages, kBlock = L::kBlock, kSteps = D / 16, kTiles = D / 16, kWords = D / 32;      // words: of a quarter row
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t bars = smem_u32(smem + L::bar_off);
  auto bar_full = [&](int s) { return bars + 8u * s; };
  auto bar_empty = [&](int s) { return bars + 8u * (kStages + s); };
  volatile int* cta_abort = reinterpret_cast<volatile int*>(smem + L::misc_off);
  int* is_last = reinterpret_cast<int*>(smem + L::misc_off + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  int idx = blockIdx.x;
  const int group = idx % a.groups;
  idx /= a.groups;
  const int split = idx % a.splits, h = idx / a.splits;
  const int g0 = static_cast<int>(static_cast<long long>(split) * a.blocks / a.splits);
  const int g1 = static_cast<int>(static_cast<long long>(split + 1) * a.blocks / a.splits);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar_full(s), 1);
      mbar_init(bar_empty(s), kKeys / 32 == 2 ? 2 : kRowsWarps);
    }
    *cta_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  // Under the end of the kernel before, which leaves the memory idle: the first blocks of the range on their way to L2.  A hint that reads
  // nothing, so it may be given for rows that kernel is still writing.
  if constexpr (!kPaged) {
    if (threadIdx.x < 2 * kStages && static_cast<int>(threadIdx.x >> 1) < g1 - g0) {
      const uint8_t* from = (threadIdx.x & 1 ? a.cache_v : a.cache_k) + h * a.head_bytes + static_cast<int64_t>(g0 + (threadIdx.x >> 1)) * kBlock;
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(from), "r"(kBlock) : "memory");
    }
  }
  pdl_wait();

  if (warp == kRowsWarps) {
    // =========================== producer ===========================
    if (lane == 0) {
      int pi = 0, block = g0;
      if constexpr (kPaged) {
        pi = block / a.blocks_per_page;
        block -= pi * a.blocks_per_page;
      }
      const uint8_t* k = a.cache_k + h * a.head_bytes;
      const uint8_t* v = a.cache_v + h * a.head_bytes;
      for (int j = 0; j < g1 - g0; ++j) {
        const int s = j % kStages;
        if constexpr (kPaged) {
          if (j == 0 || block == 0) {
            const int page = a.page_table == nullptr ? pages.id[pi] : __ldg(a.page_table + pi);
            if (page < 0 || page >= a.num_pages) {
              atomicCAS(a.status, 0, kStatusBadIndex);
              *cta_abort = 1;
              break;
            }
            k = a.pool + (static_cast<int64_t>(page) * 2 * a.heads + h) * a.head_bytes;
            v = k + a.heads * a.head_bytes;
          }
        }
        // naps between looks: spinning, the four fetching warps of an SM took one issue slot in eight
        if (j >= kStages) {
          for (int naps = 0; naps < 64 && !mbar_try_wait(bar_empty(s), ((j / kStages) & 1) ^ 1u); ++naps) __nanosleep(64);
          if (!mbar_wait(bar_empty(s), ((j / kStages) & 1) ^ 1u, cta_abort, a.status)) break;
        }
        const uint32_t bytes = (block < a.full_blocks ? kFp4Rows : a.tail_rows) * kFp4RowBytes<D>;
        const int64_t off = static_cast<int64_t>(block) * kBlock;
        mbar_arrive_expect_tx(bar_full(s), 2 * bytes);
        bulk_load(smem_u32(smem + s * 2 * kBlock), k + off, bytes, bar_full(s));
        bulk_load(smem_u32(smem + s * 2 * kBlock + kBlock), v + off, bytes, bar_full(s));
        ++block;
        if (kPaged && block == a.blocks_per_page) {
          block = 0;
          ++pi;
        }
      }
    }
  } else {
    // =========================== computing warps ===========================
    const int g = lane >> 2, t = lane & 3;
    const int row_q = group * 8 + g;
    // the quarter t of query row g, as the left operand: rows g (rounded) and g + 8 (the rest)
    uint32_t qf[kSteps][4];
    float c;
    {
      float x[D / 4];
      const size_t at = (static_cast<size_t>(row_q) * a.heads + h) * D + t * (D / 4);
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < D / 4; i += 8) {
        if (row_q >= a.n_q) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[i + e] = 0.f;
        } else if (a.q_f32) {
          const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + at + i);
          const float4 u = src[0], w = src[1];
          x[i] = u.x; x[i + 1] = u.y; x[i + 2] = u.z; x[i + 3] = u.w;
          x[i + 4] = w.x; x[i + 5] = w.y; x[i + 6] = w.z; x[i + 7] = w.w;
          if (a.q_round_bf16) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[i + e] = __bfloat162float(__float2bfloat16_rn(x[i + e]));
          }
        } else {
          const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.q) + at + i);
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[i + 2 * e] = __uint_as_float(w[e] << 16);
            x[i + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, fp4_abs_bits(x[i + e]));
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // the power of two that brings the row's largest value to [2^14, 2^15); at most 2^126; 1 for a row of zeros or with a value that
      // is not finite
      const int up = top == 0 || top >= 0x7f800000u ? 0 : min(14 + 127 - static_cast<int>(top >> 23), 126);
      const float f = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
      c = a.scale_log2 / f;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        if constexpr (kRest) {
          split_f16(x[4 * i] * f, x[4 * i + 1] * f, qf[i][0], qf[i][1]);
          split_f16(x[4 * i + 2] * f, x[4 * i + 3] * f, qf[i][2], qf[i][3]);
        } else {                                           // bf16 queries are half-precision numbers as they are
          qf[i][0] = pack_f16x2(x[4 * i] * f, x[4 * i + 1] * f);
          qf[i][2] = pack_f16x2(x[4 * i + 2] * f, x[4 * i + 3] * f);
          qf[i][1] = qf[i][3] = 0u;
        }
      }
    }
    // tile j of (p v)^T: d = (D / 8) g + 2 j and the one behind it, queries 2t and 2t + 1
    float acc[kTiles][4];
#pragma unroll
    for (int j = 0; j < kTiles; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    float m = -INFINITY, l = 0.f;          // of query row g: maximum of the base-2 exponents, sum of this lane's weights

    // kKeys keys from key0 on of a block with `rows` rows of K at kb and of V at vb, the first `valid` of which count
    auto use_block = [&](const uint8_t* kb, const uint8_t* vb, int rows, int valid, int key0, auto whole) {
      constexpr bool kWhole = decltype(whole)::value;        // valid == 128
      if (!kWhole && key0 >= valid) return;
      float x[kKeys / 8][2];
      {
        // column c of tile n is key 16 (n / 2) + 4 (c % 2 + 2 (n % 2)) + c / 2: those of a lane's weights are t, t + 4, t + 8, t + 12
        const int key = key0 + 4 * (g & 1) + (g >> 1);
        const uint8_t* src = kb + key * (D / 2) + t * (D / 8);
        const uint8_t* ss = kb + rows * (D / 2) + key * (D / 16) + t * (D / 64);
#pragma unroll
        for (int n = 0; n < kKeys / 8; n += 2) {           // two tiles by turns: a product depends on the last but one
          uint32_t w[2][kWords], sc[2][kWords / 2];
          float d[2][4] = {};
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            if constexpr (D == 64) {
              const uint2 v = *reinterpret_cast<const uint2*>(src + 8 * (n + u) * (D / 2));
              w[u][0] = v.x; w[u][1] = v.y;
              sc[u][0] = static_cast<uint32_t>(ss[8 * (n + u) * (D / 16)]) * 0x00800080u;
            } else {
              const uint4 v = *reinterpret_cast<const uint4*>(src + 8 * (n + u) * (D / 2));
              w[u][0] = v.x; w[u][1] = v.y; w[u][2] = v.z; w[u][3] = v.w;
              const uint32_t both = *reinterpret_cast<const uint16_t*>(ss + 8 * (n + u) * (D / 16));
              sc[u][0] = (both & 0xffu) * 0x00800080u;
              sc[u][1] = (both >> 8) * 0x00800080u;
            }
          }
#pragma unroll
          for (int i = 0; i < kWords; ++i) {
            uint32_t b[2][4];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              fp4_unpack8(w[u][i], b[u]);
#pragma unroll
              for (int e = 0; e < 4; ++e) b[u][e] = half2_mul(b[u][e], sc[u][i / 2]);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) mma_f16(d[u], qf[2 * i], b[u][0], b[u][1]);
#pragma unroll
            for (int u = 0; u < 2; ++u) mma_f16(d[u], qf[2 * i + 1], b[u][2], b[u][3]);
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            x[n + u][0] = (kRest ? d[u][0] + d[u][2] : d[u][0]) * c;
            x[n + u][1] = (kRest ? d[u][1] + d[u][3] : d[u][1]) * c;
            if constexpr (!kWhole) {
              const int mine = key0 + 8 * (n + u) + t;
              if (mine >= valid) x[n + u][0] = -INFINITY;
              if (mine + 4 >= valid) x[n + u][1] = -INFINITY;
            }
          }
        }
      }
      float mx = fmaxf(x[0][0], x[0][1]);
#pragma unroll
      for (int n = 1; n < kKeys / 8; ++n) mx = max3(mx, x[n][0], x[n][1]);
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      if (__any_sync(0xffffffffu, mx > m)) {
        const float next = fmaxf(m, mx), alpha = next == -INFINITY ? 1.f : fast_exp2(m - next);
        m = next;
        l *= alpha;
        const float a0 = __shfl_sync(0xffffffffu, alpha, 8 * t), a1 = __shfl_sync(0xffffffffu, alpha, 8 * t + 4);      // of queries 2t and 2t + 1
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
          acc[j][0] *= a0;
          acc[j][1] *= a1;
          acc[j][2] *= a0;
          acc[j][3] *= a1;
        }
      }
      const float from = kWeightShift - (m == -INFINITY ? 0.f : m);
      const int key = key0 + t;
      const uint8_t* src = vb + key * (D / 2) + g * (D / 16);
      const uint8_t* ss = vb + rows * (D / 2) + key * (D / 16) + (D == 64 ? g >> 1 : g);
#pragma unroll
      for (int step = 0; step < kKeys / 16; ++step) {
        uint32_t w[4][kWords / 2], sc[4], p[2], rest[2];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int r = 16 * step + 4 * u;
          sc[u] = ss[r * (D / 16)];
          if (!kWhole && key + r >= valid) sc[u] = 0;      // rows past the end count nothing, whatever they hold
          if constexpr (D == 64) {
            w[u][0] = *reinterpret_cast<const uint32_t*>(src + r * (D / 2));
          } else {
            const uint2 both = *reinterpret_cast<const uint2*>(src + r * (D / 2));
            w[u][0] = both.x;
            w[u][1] = both.y;
          }
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float e0 = fast_exp2(x[2 * step + n][0] + from), e1 = fast_exp2(x[2 * step + n][1] + from);
          l += e0 + e1;
          if constexpr (kRest)
            split_f16(e0, e1, p[n], rest[n]);
          else
            p[n] = pack_f16x2(e0, e1);
        }
        const uint32_t s01 = sc[0] << 7 | sc[1] << 23, s23 = sc[2] << 7 | sc[3] << 23;
#pragma unroll
        for (int i = 0; i < kWords / 2; ++i) {
          constexpr uint32_t kLow = 0x0f0f0f0fu;
          uint32_t lo01[4], hi01[4], lo23[4], hi23[4];
          fp4_unpack8((w[0][i] & kLow) | ((w[1][i] << 4) & ~kLow), lo01);
          fp4_unpack8(((w[0][i] >> 4) & kLow) | (w[1][i] & ~kLow), hi01);
          fp4_unpack8((w[2][i] & kLow) | ((w[3][i] << 4) & ~kLow), lo23);
          fp4_unpack8(((w[2][i] >> 4) & kLow) | (w[3][i] & ~kLow), hi23);
          uint32_t v[4][4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e][0] = half2_mul(lo01[e], s01);
            v[e][1] = half2_mul(hi01[e], s01);
            v[e][2] = half2_mul(lo23[e], s23);
            v[e][3] = half2_mul(hi23[e], s23);
            mma_f16(acc[4 * i + e], v[e], p[0], p[1]);
          }
#pragma unroll
          for (int e = 0; kRest && e < 4; ++e) {
            mma_f16(acc[4 * i + e], v[e], rest[0], rest[1]);
          }
        }
      }
    };

    if constexpr (!kPaged) {
      // the call's own rows, 128 at a time: the CTAs of the last key range quantise them, those of the first queries store them
      if (split == a.splits - 1) {
        for (int base = 0; base < a.n_new; base += kFp4Rows) {
          const int rows = min(a.n_new - base, kFp4Rows);
          if (base > 0) asm volatile("bar.sync 1, %0;" ::"n"(32 * kRowsWarps) : "memory");
          for (int i = threadIdx.x; i < 2 * rows * kSteps; i += 32 * kRowsWarps) {
            const bool is_v = i >= rows * kSteps;
            const int r = (is_v ? i - rows * kSteps : i) / kSteps, part = i % kSteps;
            Fp4Group16 q;
            q.quantise((is_v ? a.v_new : a.k_new) + (static_cast<size_t>(base + r) * a.heads + h) * D + part * kFp4Group);
            uint8_t* to = smem + L::new_off + (is_v ? kBlock : 0);
            q.store(to + r * (D / 2) + 8 * part, to + kFp4Rows * (D / 2) + r * kSteps + part);
            if (a.store && group == 0) {
              uint8_t* cache = (is_v ? a.cache_v : a.cache_k) + h * a.head_bytes;
              const Fp4At at = fp4_at<D>(static_cast<int64_t>(a.cached) + base + r, a.full_blocks, a.tail_rows);
              q.store(cache + at.values + 8 * part, cache + at.scales + part);
            }
          }
          asm volatile("bar.sync 1, %0;" ::"n"(32 * kRowsWarps) : "memory");
          // the last warp takes the first rows: the first has those of a short cache
          use_block(smem + L::new_off, smem + L::new_off + kBlock, kFp4Rows, rows, 32 * (kRowsWarps - 1 - warp), std::false_type());
        }
      }
    }
    constexpr int kStep = kKeys == 64 ? 2 : 1;             // 64: a pair of warps takes every other block
    const int pair = kKeys == 64 ? warp >> 1 : 0, key0 = kKeys == 64 ? 64 * (warp & 1) : 32 * warp;
    int page = 0, block = g0 + pair;                       // place of the next block
    if constexpr (kPaged) {
      page = block / a.blocks_per_page;
      block -= page * a.blocks_per_page;
    }
    for (int j = pair; j < g1 - g0; j += kStep) {
      const int s = j % kStages;
      int rows = kFp4Rows, valid;
      if constexpr (kPaged) {
        if (block >= a.full_blocks) rows = a.tail_rows;
        valid = (page == a.n_pages - 1 ? a.last_page_rows : a.page_rows) - block * kFp4Rows;
        block += kStep;
        while (block >= a.blocks_per_page) {
          block -= a.blocks_per_page;
          ++page;
        }
      } else {
        valid = a.cached - block * kFp4Rows;
        block += kStep;
      }
      if (!__all_sync(0xffffffffu, mbar_wait(bar_full(s), (j / kStages) & 1, cta_abort, a.status))) break;
      const uint8_t* at = smem + s * 2 * kBlock;
      if (valid >= kFp4Rows)
        use_block(at, at + kBlock, kFp4Rows, kFp4Rows, key0, std::true_type());
      else
        use_block(at, at + kBlock, rows, valid, key0, std::false_type());
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_empty(s));
    }
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    asm volatile("bar.sync 1, %0;" ::"n"(32 * kRowsWarps) : "memory");      // every warp has read its last stage
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      if (group * 8 + 2 * t + b < a.n_q) {
        float* so = reinterpret_cast<float*>(smem + L::out_off) + (warp * 8 + 2 * t + b) * D + (D / 8) * g;
#pragma unroll
        for (int j = 0; j < kTiles; j += 2) *reinterpret_cast<float4*>(so + 2 * j) = make_float4(acc[j][b], acc[j][2 + b], acc[j + 1][b], acc[j + 1][2 + b]);
      }
    }
    if (t == 0) *reinterpret_cast<float2*>(smem + L::stat_off + (warp * 8 + g) * 8) = make_float2(m, l);
  }
  if (*cta_abort) {
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);      // copies in flight land before the shared memory is given up
  }
  __syncthreads();

  // ---- the four warps, then the key ranges, in order ----
  const float* so = reinterpret_cast<const float*>(smem + L::out_off);
  const float* stat = reinterpret_cast<const float*>(smem + L::stat_off);
  const int rows_here = min(8, a.n_q - group * 8);
  auto finish = [&](int i, int d, float mx, float num, float den) {
    const size_t row = static_cast<size_t>(group * 8 + i) * a.heads + h;
    const float o = num / den;
    if (a.out_bf16 != nullptr) a.out_bf16[row * D + d] = __float2bfloat16_rn(o);
    if (a.out_f32 != nullptr) a.out_f32[row * D + d] = o;
    if (a.lse != nullptr && d == 0) a.lse[row] = (mx + log2f(den) - kWeightShift) * 0.6931471805599453f;
  };
  const size_t item = static_cast<size_t>(h) * a.groups + group;
  constexpr int kRecord = kRowsRecord<D>;
  for (int e = threadIdx.x; e < rows_here * D; e += kRowsThreads) {
    const int i = e / D, d = e % D;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) mx = fmaxf(mx, stat[(w * 8 + i) * 2]);
    float num = 0.f, den = 0.f;
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) {
      const float ms = stat[(w * 8 + i) * 2];
      const float f = ms == mx ? 1.f : fast_exp2(ms - mx);      // 0 for a warp without keys
      num = fmaf(f, so[(w * 8 + i) * D + d], num);
      den = fmaf(f, stat[(w * 8 + i) * 2 + 1], den);
    }
    if (a.splits == 1) {
      finish(i, d, mx, num, den);
    } else {
      float* rec = a.part + ((item * a.splits + split) * 8 + i) * kRecord;
      rec[d] = num;
      if (d == 0) {
        rec[D] = mx;
        rec[D + 1] = den;
      }
    }
  }
  if (a.splits == 1) return;
  // one fence behind the barrier covers the stores of the whole CTA; a fence in every thread took 0.1 to 0.7 us more
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    const int before = atomicAdd(a.counters + item, 1);
    *is_last = before == a.splits - 1;
    if (*is_last) {
      a.counters[item] = 0;
      __threadfence();
    }
  }
  __syncthreads();
  if (!*is_last) return;
  // As many lanes per four columns as there are threads for (a power of two): each adds up every so many-th range against the largest
  // maximum among them, then they are joined in order.  Maxima and sums come in one trip.
  float4* lane_sum = reinterpret_cast<float4*>(smem);
  const float* recs = a.part + item * a.splits * 8 * kRecord;
  constexpr int kCols = D / 4, kAhead = kJoinAhead;
  const int items = rows_here * kCols;
  int lanes = 1;
  while (2 * lanes * items <= 128) lanes *= 2;
  for (int e = threadIdx.x; e < items * lanes; e += kRowsThreads) {
    const int it = e % items, ln = e / items, i = it / kCols, col = it % kCols;
    float mx = -INFINITY, den = 0.f;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int r0 = ln; r0 < a.splits; r0 += kAhead * lanes) {
      float4 o[kAhead];
      float2 ml[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int r = r0 + u * lanes;
        const float* rec = recs + (r * 8 + i) * kRecord;
        ml[u] = r < a.splits ? __ldcg(reinterpret_cast<const float2*>(rec + D)) : make_float2(-INFINITY, 0.f);
        o[u] = r < a.splits ? __ldcg(reinterpret_cast<const float4*>(rec + 4 * col)) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float next = mx;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) next = fmaxf(next, ml[u].x);
      const float old = mx == next ? 1.f : fast_exp2(mx - next);
      mx = next;
      den *= old;
      sum.x *= old;
      sum.y *= old;
      sum.z *= old;
      sum.w *= old;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const float f = ml[u].x == mx ? 1.f : fast_exp2(ml[u].x - mx);
        den = fmaf(f, ml[u].y, den);
        sum.x = fmaf(f, o[u].x, sum.x);
        sum.y = fmaf(f, o[u].y, sum.y);
        sum.z = fmaf(f, o[u].z, sum.z);
        sum.w = fmaf(f, o[u].w, sum.w);
      }
    }
    lane_sum[2 * e] = sum;
    lane_sum[2 * e + 1] = make_float4(mx, den, 0.f, 0.f);
  }
  __syncthreads();
  for (int it = threadIdx.x; it < items; it += kRowsThreads) {
    float mx = -INFINITY, den = 0.f;
    for (int ln = 0; ln < lanes; ++ln) mx = fmaxf(mx, lane_sum[2 * (it + ln * items) + 1].x);
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int ln = 0; ln < lanes; ++ln) {
      const float4 o = lane_sum[2 * (it + ln * items)], md = lane_sum[2 * (it + ln * items) + 1];
      const float f = md.x == mx ? 1.f : fast_exp2(md.x - mx);
      sum.x = fmaf(f, o.x, sum.x);
      sum.y = fmaf(f, o.y, sum.y);
      sum.z = fmaf(f, o.z, sum.z);
      sum.w = fmaf(f, o.w, sum.w);
      den = fmaf(f, md.y, den);
    }
    const int i = it / kCols, d = 4 * (it % kCols);
    finish(i, d, mx, sum.x, den);
    finish(i, d + 1, mx, sum.y, den);
    finish(i, d + 2, mx, sum.z, den);
    finish(i, d + 3, mx, sum.w, den);
  }
}

template <int D, bool kPaged>
int launch_rows_kernel(const RowsArgs& k, const Fp4Pages& pages, dim3 grid, cudaStream_t stream) {
  constexpr int kMaxDevices = 64;
  static std::mutex mu;
  static bool done[kMaxDevices] = {false};
  int dev = -1;
  GCT_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= kMaxDevices) return fail(GCT_ERR_INVALID, "fp4 attention: device ordinal out of range");
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!done[dev]) {
      GCT_CUDA_CHECK(cudaFuncSetAttribute(gct_fp4_rows_kernel<D, kPaged>, cudaFuncAttributeMaxDynamicSharedMemorySize, RowsSmem<D, kPaged>::total));
      done[dev] = true;
    }
  }
  GCT_CUDA_CHECK(launch_pdl(gct_fp4_rows_kernel<D, kPaged>, grid, dim3(kRowsThreads), RowsSmem<D, kPaged>::total, stream, k, pages));
  return GCT_OK;
}

bool misaligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

}  // namespace

// More ranges share the keys among more CTAs of an SM, and make the join longer, which one CTA per (head, eight queries) does in trips to L2.  As
// many as fill one, two, ... CTAs per SM are compared, in hundredths of a us as measured: a trip, and a block at so many CTAs per SM.  us with
// 9 / 18 / 37 ranges (one, two, four CTAs), 16 heads of 64: eight queries over 33 blocks 8.6 / 9.1 / 10.2, 81 blocks 10.6 / 10.3 / 11.6, 161 blocks
// 14.9 / 13.4 / 15.1; six over 181 blocks 16.4 / 14.3 / 14.7, 625 blocks 40.8 / 31.1 / 29.8; one over 81 blocks 10.0 / 9.0 / 8.1.  With 9 / 18 / 27 ranges of
// 16 heads of 128: eight over 24 blocks 11.9 / 15.1 / 14.9, 79 blocks 17.8 / 20.7 / 18.7; one over 79 blocks 14.9 / 14.9 / 12.0.
int fp4_rows_splits(int n_q, int heads, int blocks, int head_dim, int sms, size_t part_floats, int num_counters) {
  constexpr int kTrip = 80, kBlock64[kRowsCtas<64>] = {50, 68, 110, 105}, kBlock128[kRowsCtas<128>] = {98, 180, 200};
  const int64_t items = static_cast<int64_t>((n_q + 7) / 8) * heads;
  if (blocks <= 1 || items > num_counters) return 1;
  const int most_ctas = head_dim == 64 ? kRowsCtas<64> : kRowsCtas<128>, record = head_dim == 64 ? kRowsRecord<64> : kRowsRecord<128>;
  const int64_t most = std::min<int64_t>(blocks, static_cast<int64_t>(part_floats / (static_cast<size_t>(items) * 8 * record)));
  const int columns = std::min(n_q, 8) * (head_dim / 4);
  int lanes = 1;                                           // that share the ranges of four columns of a row, as in the kernel
  while (2 * lanes * columns <= 128) lanes *= 2;
  const int passes = (columns * lanes + kRowsThreads - 1) / kRowsThreads;
  int64_t best = 1, best_cost = -1;
  for (int ctas = most_ctas; ctas >= 1; --ctas) {
    const int64_t splits = std::max<int64_t>(1, std::min(most, static_cast<int64_t>(sms) * ctas / items));
    const int64_t per_sm = std::min<int64_t>(most_ctas, (splits * items + sms - 1) / sms);
    const int64_t trips = passes * ((splits + kJoinAhead * lanes - 1) / (kJoinAhead * lanes));
    const int64_t cost = kTrip * trips + (blocks + splits - 1) / splits * (head_dim == 64 ? kBlock64 : kBlock128)[per_sm - 1];
    if (best_cost < 0 || cost < best_cost) {
      best = splits;
      best_cost = cost;
    }
  }
  return static_cast<int>(best);
}

int launch_fp4_rows(const Fp4RowsLaunch& p, cudaStream_t stream) {
  if (p.q == nullptr || p.n_q <= 0 || p.heads <= 0 || p.status == nullptr || (p.head_dim != 64 && p.head_dim != 128))
    return fail(GCT_ERR_INVALID, "fp4 attention: bad argument");
  const bool paged = p.pool != nullptr;
  if (paged ? (p.page_table == nullptr && p.page_ids == nullptr) || p.head_dim != 64 || p.n_pages <= 0 || p.page_rows <= 0 || p.last_page_rows <= 0 || p.last_page_rows > p.page_rows ||
                  p.n_new != 0
            : p.cache_k == nullptr || p.cache_v == nullptr || p.cached < 0 || p.n_new < 0 || p.cached + p.n_new <= 0 || p.layout.tail_rows != 0)
    return fail(GCT_ERR_INVALID, "fp4 attention: bad cache");
  if (p.n_new > 0 && (p.k_new == nullptr || p.v_new == nullptr)) return fail(GCT_ERR_INVALID, "fp4 attention: bad argument");
  if (!paged && static_cast<int64_t>(p.cached) + (p.store ? p.n_new : 0) > static_cast<int64_t>(p.layout.full_blocks) * kFp4Rows)
    return fail(GCT_ERR_CAPACITY, "fp4 attention: the cache is full");
  for (const void* x : {p.q, static_cast<const void*>(p.pool), static_cast<const void*>(p.cache_k), static_cast<const void*>(p.cache_v),
                        static_cast<const void*>(p.k_new), static_cast<const void*>(p.v_new)})
    if (misaligned16(x)) return fail(GCT_ERR_INVALID, "fp4 attention: tensors must be 16-byte aligned");
  RowsArgs k = {};
  k.q = p.q;
  k.q_f32 = p.q_dtype == GCT_F32;
  k.q_round_bf16 = p.q_round_bf16;
  k.n_q = p.n_q;
  k.heads = p.heads;
  k.groups = (p.n_q + 7) / 8;
  k.pool = p.pool;
  k.page_table = p.page_table;
  k.n_pages = p.n_pages;
  k.num_pages = p.num_pages;
  k.page_rows = p.page_rows;
  k.last_page_rows = p.last_page_rows;
  k.full_blocks = p.layout.full_blocks;
  k.tail_rows = p.layout.tail_rows;
  k.head_bytes = p.layout.bytes;
  k.cache_k = p.cache_k;
  k.cache_v = p.cache_v;
  k.cached = p.cached;
  k.k_new = p.k_new;
  k.v_new = p.v_new;
  k.n_new = p.n_new;
  k.store = p.store;
  if (paged) {
    k.blocks_per_page = (p.page_rows + kFp4Rows - 1) / kFp4Rows;
    k.blocks = (p.n_pages - 1) * k.blocks_per_page + (p.last_page_rows + kFp4Rows - 1) / kFp4Rows;
  } else {
    k.blocks = (p.cached + kFp4Rows - 1) / kFp4Rows;
  }
  int sms = 148;
  const int rc = device_sm_count(&sms);
  if (rc != GCT_OK) return rc;
  k.splits = p.counters == nullptr || p.part == nullptr ? 1 : fp4_rows_splits(p.n_q, p.heads, k.blocks, p.head_dim, sms, p.part_floats, p.num_counters);
  k.scale_log2 = 1.4426950408889634f / sqrtf(static_cast<float>(p.head_dim));
  k.out_bf16 = p.out_bf16;
  k.out_f32 = p.out_f32;
  k.lse = p.lse;
  k.part = p.part;
  k.counters = p.counters;
  k.status = p.status;
  const int64_t ctas = static_cast<int64_t>(k.groups) * k.splits * p.heads;
  if (ctas > 0x7fffffff) return fail(GCT_ERR_INVALID, "fp4 attention: too many rows");
  const dim3 grid(static_cast<unsigned>(ctas));
  Fp4Pages pages = {};
  if (paged && p.page_ids != nullptr) {
    if (p.n_pages > kFp4ArgPages) return fail(GCT_ERR_INVALID, "fp4 attention: too many pages for an argument");
    std::copy(p.page_ids, p.page_ids + p.n_pages, pages.id);
    k.page_table = nullptr;
  }
  if (paged) return launch_rows_kernel<64, true>(k, pages, grid, stream);
  return p.head_dim == 64 ? launch_rows_kernel<64, false>(k, pages, grid, stream) : launch_rows_kernel<128, false>(k, pages, grid, stream);
}

int launch_fp4_read(const Fp4ReadLaunch& p, cudaStream_t stream) {
  if (p.pool == nullptr || p.heads <= 0 || p.tokens < 0 || (p.head_dim != 64 && p.head_dim != 128)) return fail(GCT_ERR_INVALID, "fp4 read: bad argument");
  if (p.tokens == 0) return GCT_OK;
  const bool products = p.products[0] != nullptr;
  for (int i = 0; i < 2; ++i)
    if (products ? p.products[i] == nullptr || misaligned16(p.products[i]) : p.values[i] == nullptr || p.scales[i] == nullptr || misaligned16(p.values[i]))
      return fail(GCT_ERR_INVALID, "fp4 read: outputs must be given and 16-byte aligned");
  const int64_t threads = 2ll * p.tokens * p.heads * (p.head_dim / kFp4Group), ctas = (threads + 255) / 256;
  if (ctas > 0x7fffffff) return fail(GCT_ERR_INVALID, "fp4 read: too many rows");
  auto kernel = p.head_dim == 64 ? (products ? gct_fp4_read_kernel<64, true> : gct_fp4_read_kernel<64, false>)
                                 : (products ? gct_fp4_read_kernel<128, true> : gct_fp4_read_kernel<128, false>);
  GCT_CUDA_CHECK(launch_pdl(kernel, dim3(static_cast<unsigned>(ctas)), dim3(256), 0, stream, p));
  return GCT_OK;
}

int launch_fp4_rows_append(const float* k, const float* v, int rows, uint8_t* cache_k, uint8_t* cache_v, const Fp4Layout& layout, int first, int heads,
                           int head_dim, cudaStream_t stream) {
  if ((rows > 0 && (k == nullptr || v == nullptr)) || cache_k == nullptr || cache_v == nullptr || rows < 0 || first < 0 || heads <= 0 ||
      layout.tail_rows != 0 || (head_dim != 64 && head_dim != 128))
    return fail(GCT_ERR_INVALID, "fp4 append: bad argument");
  if (misaligned16(k) || misaligned16(v) || misaligned16(cache_k) || misaligned16(cache_v)) return fail(GCT_ERR_INVALID, "fp4 append: tensors must be 16-byte aligned");
  if (static_cast<int64_t>(first) + rows > static_cast<int64_t>(layout.full_blocks) * kFp4Rows) return fail(GCT_ERR_CAPACITY, "fp4 append: the cache is full");
  if (rows == 0) return GCT_OK;
  const int64_t ctas = (2ll * rows * heads * (head_dim / kFp4Group) + 127) / 128;
  if (ctas > 0x7fffffff) return fail(GCT_ERR_INVALID, "fp4 append: too many rows");
  auto kernel = head_dim == 64 ? gct_fp4_rows_append_kernel<64> : gct_fp4_rows_append_kernel<128>;
  GCT_CUDA_CHECK(launch_pdl(kernel, dim3(static_cast<unsigned>(ctas)), dim3(128), 0, stream, k, v, rows, cache_k, cache_v, layout.full_blocks, layout.bytes, first,
                            heads));
  return GCT_OK;
}

}  // namespace gct

namespace {

constexpr size_t kDecodeStatusBytes = 256;
constexpr int kDecodeCounters = 2048;
// Counters and partial results of one wave of CTAs; calls with more (head, eight queries) items than counters take one key range.
size_t decode_fp4_workspace(int head_dim) {
  return kDecodeStatusBytes + kDecodeCounters * sizeof(int) + static_cast<size_t>(148 * (head_dim == 64 ? gct::kRowsCtas<64> : gct::kRowsCtas<128>)) * 8 * (head_dim == 64 ? gct::kRowsRecord<64> : gct::kRowsRecord<128>) * sizeof(float);
}

int check_decode_cache(const char* who, int heads, int head_dim, int capacity) {
  if (heads < 1 || (head_dim != 64 && head_dim != 128) || capacity < 1 || capacity % gct::kFp4Rows != 0)
    return gct::fail(GCT_ERR_INVALID, std::string(who) + ": head_dim must be 64 or 128, the capacity a positive multiple of 128");
  return GCT_OK;
}

}  // namespace

extern "C" {

int gct_decode_fp4_sizes(int heads, int head_dim, int capacity, size_t* cache_bytes_out, size_t* workspace_bytes_out) {
  const int rc = check_decode_cache("gct_decode_fp4_sizes", heads, head_dim, capacity);
  if (rc != GCT_OK) return rc;
  if (cache_bytes_out != nullptr) *cache_bytes_out = static_cast<size_t>(heads) * gct::fp4_layout(capacity, head_dim).bytes;
  if (workspace_bytes_out != nullptr) *workspace_bytes_out = decode_fp4_workspace(head_dim);
  return GCT_OK;
}

int gct_decode_attention_fp4(const float* q_dev, const float* k_new_dev, const float* v_new_dev, int n_new, uint8_t* cache_k_dev, uint8_t* cache_v_dev,
                             int cached, int capacity, int store, int heads, int head_dim, float* out_dev, void* workspace_dev, size_t workspace_bytes,
                             void* stream) {
  const int rc = check_decode_cache("gct_decode_attention_fp4", heads, head_dim, capacity);
  if (rc != GCT_OK) return rc;
  if (out_dev == nullptr || workspace_dev == nullptr || n_new < 1) return gct::fail(GCT_ERR_INVALID, "gct_decode_attention_fp4: bad argument");
  if ((reinterpret_cast<uintptr_t>(workspace_dev) & 255) != 0) return gct::fail(GCT_ERR_INVALID, "gct_decode_attention_fp4: the workspace must be 256-byte aligned");
  if (workspace_bytes < decode_fp4_workspace(head_dim)) return gct::fail(GCT_ERR_CAPACITY, "gct_decode_attention_fp4: workspace too small");
  gct::Fp4RowsLaunch p;
  p.q = q_dev;
  p.q_dtype = GCT_F32;
  p.n_q = n_new;
  p.heads = heads;
  p.head_dim = head_dim;
  p.cache_k = cache_k_dev;
  p.cache_v = cache_v_dev;
  p.cached = cached;
  p.layout = gct::fp4_layout(capacity, head_dim);
  p.k_new = k_new_dev;
  p.v_new = v_new_dev;
  p.n_new = n_new;
  p.store = store;
  p.out_f32 = out_dev;
  p.status = static_cast<int*>(workspace_dev);
  p.counters = reinterpret_cast<int*>(static_cast<uint8_t*>(workspace_dev) + kDecodeStatusBytes);
  p.num_counters = kDecodeCounters;
  p.part = reinterpret_cast<float*>(p.counters + kDecodeCounters);
  p.part_floats = (workspace_bytes - kDecodeStatusBytes - kDecodeCounters * sizeof(int)) / sizeof(float);
  return gct::launch_fp4_rows(p, static_cast<cudaStream_t>(stream));
}

int gct_decode_append_fp4(const float* k_dev, const float* v_dev, int rows, uint8_t* cache_k_dev, uint8_t* cache_v_dev, int first, int capacity, int heads,
                          int head_dim, void* stream) {
  const int rc = check_decode_cache("gct_decode_append_fp4", heads, head_dim, capacity);
  if (rc != GCT_OK) return rc;
  return gct::launch_fp4_rows_append(k_dev, v_dev, rows, cache_k_dev, cache_v_dev, gct::fp4_layout(capacity, head_dim), first, heads, head_dim,
                                     static_cast<cudaStream_t>(stream));
}

int gct_decode_read_fp4(const uint8_t* cache_k_dev, const uint8_t* cache_v_dev, int first, int rows, int capacity, int heads, int head_dim,
                        uint8_t* k_values_dev, void* k_scales_dev, uint8_t* v_values_dev, void* v_scales_dev, void* stream) {
  const int rc = check_decode_cache("gct_decode_read_fp4", heads, head_dim, capacity);
  if (rc != GCT_OK) return rc;
  if (cache_k_dev == nullptr || cache_v_dev == nullptr || first < 0 || rows < 0 || rows > capacity - first)
    return gct::fail(GCT_ERR_INVALID, "gct_decode_read_fp4: rows out of range");
  gct::Fp4ReadLaunch p;
  p.pool = cache_k_dev;
  p.v_pool = cache_v_dev;
  p.layout = gct::fp4_layout(capacity, head_dim);
  p.heads = heads;
  p.head_dim = head_dim;
  p.tokens = rows;
  p.first = first;
  p.num_pages = 1;
  p.page_rows = capacity;
  p.at.patch_page = 0;
  p.values[0] = k_values_dev;
  p.values[1] = v_values_dev;
  p.scales[0] = static_cast<__half*>(k_scales_dev);
  p.scales[1] = static_cast<__half*>(v_scales_dev);
  return gct::launch_fp4_read(p, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
