// The 4-bit cache format: how rows are laid out, and how values get in and out.
//
// A row of D values (D = 64 or 128) is cut into blocks of 16.  A block is a scale s and sixteen values c, and stands for s * c.
//   s  a byte of five exponent and three mantissa bits, no sign: shifted left by seven it is the half-precision number s.
//      s = max|x| / 6 rounded to the nearest, ties to even, at most 10240 (so that 6 s is a half-precision number).  0xff (a NaN) marks
//      a block with a value that is not finite: it stays visible, as it does in a cache that holds the values themselves.
//   c  e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives: x / s rounded to the nearest, ties to even, at most 6.
// s has four significant bits and c two: s * c is exact in half precision (down to 2^-18) and in bf16, so the attention kernels compute
// with exactly the values the cache stands for.  x / 6 and x / s are rounded divisions; that a quotient rounds onto a border between two
// results without lying on it cannot happen: a border times 6 or times s has at most seven significant bits, so the nearest other x is far
// enough away (at least 8/15 of a step of the quotient) for its quotient to round to another number.  The result is therefore
// that of exact arithmetic.
//
// Memory.  Rows of one head lie together, in blocks of 128: first the packed values of the block's rows (D / 2 bytes each, the lower four
// bits of a byte first), then their scales (D / 16 bytes each).  The last block of a page holds its rows rounded up to a multiple of four,
// which keeps every block a multiple of 16 bytes, so that one bulk copy fetches it.  A head of a 999-row page takes 36,000 bytes where
// bf16 takes 127,872.
#pragma once

#include <cuda_fp16.h>

#include "gct_common.h"

namespace gct {

constexpr int kFp4Rows = 128;             // rows of a block
constexpr int kFp4Group = 16;             // values of a scale
template <int D>
constexpr int kFp4RowBytes = D / 2 + D / kFp4Group;
template <int D>
constexpr int kFp4BlockBytes = kFp4Rows * kFp4RowBytes<D>;

// `rows` rows of one head.
struct Fp4Layout {
  int full_blocks = 0, tail_rows = 0;     // blocks of 128 rows, and rows of one more block (a multiple of four; 0: there is none)
  int64_t bytes = 0;
};
inline Fp4Layout fp4_layout(int64_t rows, int head_dim) {
  Fp4Layout l;
  l.full_blocks = static_cast<int>(rows / kFp4Rows);
  l.tail_rows = static_cast<int>((rows % kFp4Rows + 3) / 4 * 4);
  l.bytes = (static_cast<int64_t>(l.full_blocks) * kFp4Rows + l.tail_rows) * (head_dim == 64 ? kFp4RowBytes<64> : kFp4RowBytes<128>);
  return l;
}

#ifdef __CUDACC__
// Offsets of row `row` inside its head's region.
struct Fp4At {
  int64_t values, scales;
};
template <int D>
__device__ __forceinline__ Fp4At fp4_at(int64_t row, int full_blocks, int tail_rows) {
  const int64_t block = row / kFp4Rows;
  const int in = static_cast<int>(row % kFp4Rows), rows = block < full_blocks ? kFp4Rows : tail_rows;
  const int64_t base = block * kFp4BlockBytes<D>;
  return {base + in * (D / 2), base + rows * (D / 2) + in * (D / kFp4Group)};
}

__device__ __forceinline__ uint32_t fp4_abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// Scale byte from the largest absolute value of a block, given as its bit pattern (patterns order like the numbers, NaN above all).
__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t largest) {
  if (largest >= 0x7f800000u) return 0xffu;
  const float f = fminf(__fdiv_rn(__uint_as_float(largest), 6.f), 10240.f);
  if (f < 6.103515625e-5f) return static_cast<uint32_t>(__float2int_rn(f * 131072.f));      // below 2^-14: steps of 2^-17
  const uint32_t u = __float_as_uint(f);
  return ((u + 0x7ffffu + ((u >> 20) & 1u)) >> 20) - 8u * (127u - 15u);
}
__device__ __forceinline__ float fp4_scale(uint32_t byte) { return __half2float(__ushort_as_half(static_cast<unsigned short>(byte << 7))); }
// x / s rounded to the nearest, given r = 1 / s rounded to the nearest: a product and one correction by its residual (P. Markstein,
// "Computation of elementary functions on the IBM RISC System/6000 processor", 1990: with a correctly rounded reciprocal the corrected
// quotient is correctly rounded, as long as the residual does not underflow; where it does here, x is far below s / 4 and becomes 0).  s = 0 or
// NaN has r = 0, and every quotient is 0.
__device__ __forceinline__ float fp4_reciprocal(float s) { return s > 0.f ? __frcp_rn(s) : 0.f; }
__device__ __forceinline__ float fp4_quotient(float x, float s, float r) {
  const float q = x * r;
  return r > 0.f ? fmaf(fmaf(-q, s, x), r, q) : 0.f;
}
// Two quotients as two values of a byte, `lo` in its lower four bits.
__device__ __forceinline__ uint32_t fp4_pack2(float lo, float hi) {
  uint32_t r;
  asm("{\n\t.reg .b8 b;\n\t.reg .b16 h;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %1, %2;\n\tmov.b16 h, {b, 0};\n\tcvt.u32.u16 %0, h;\n\t}" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Eight values x with scale s and its reciprocal r (a NaN or zero scale: zeros).
__device__ __forceinline__ uint32_t fp4_pack8(const float* x, float s, float r) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) w |= fp4_pack2(fp4_quotient(x[2 * i], s, r), fp4_quotient(x[2 * i + 1], s, r)) << (8 * i);
  return w;
}
// The eight values of a word as four pairs of half-precision numbers, in order.
__device__ __forceinline__ void fp4_unpack8(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\tcvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}
__device__ __forceinline__ uint32_t half2_mul(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
#endif  // __CUDACC__

// ---- launches (gct_fp4.cu, gct_attn_fp4_sm100.cu) -----------------------------------------------------------

// Rows of a cache read back: `tokens` rows per head; token t lies at slot(t) of a page as the prologue's PageSlots say
// (num_special == 0: row `first` + t of page patch_page).
struct Fp4ReadLaunch {
  const uint8_t* pool = nullptr;         // [pages][2][heads][layout.bytes], or with v_pool: [heads][layout.bytes] each
  const uint8_t* v_pool = nullptr;
  Fp4Layout layout;
  int heads = 0, head_dim = kHeadDim, tokens = 0, num_special = 0, num_pages = 0, page_rows = 0, first = 0;
  PageSlots at;
  uint8_t* values[2] = {nullptr, nullptr};        // K, V: [tokens, heads, D] as e4m3 bytes, with
  __half* scales[2] = {nullptr, nullptr};         // [tokens, heads, D / 16]; or
  __nv_bfloat16* products[2] = {nullptr, nullptr};      // [tokens, heads, D]: s * c
  int* status = nullptr;
};
int launch_fp4_read(const Fp4ReadLaunch& p, cudaStream_t stream);

// key_norm_max[head] = the largest 2-norm of a K row of the pool [pages][2][heads][layout.bytes]
int launch_scan_keys_fp4(const uint8_t* pool, int num_pages, int page_size, int heads, float* key_norm_max, cudaStream_t stream);

// K and V rows [rows, heads, D] fp32 appended at row `first` of the camera head's caches ([heads][layout.bytes] each).
int launch_fp4_rows_append(const float* k, const float* v, int rows, uint8_t* cache_k, uint8_t* cache_v, const Fp4Layout& layout, int first,
                           int heads, int head_dim, cudaStream_t stream);

// The pages of a plan as a kernel argument: it spares the copy of a table to the device ahead of each frame's first call (4 us of the
// stream's time).  Longer plans use the table.
constexpr int kFp4ArgPages = 256;
struct Fp4Pages {
  int32_t id[kFp4ArgPages];
};

// Attention of a few query rows (any number: eight at a time) over a 4-bit cache.
struct Fp4RowsLaunch {
  const void* q = nullptr;               // [n_q, heads, D]
  int q_dtype = GCT_BF16;
  bool q_round_bf16 = false;             // an fp32 q is rounded to bf16 first
  int n_q = 0, heads = 0, head_dim = kHeadDim;
  // paged: pool [pages][2][heads][layout.bytes], page_table; else cache_k / cache_v [heads][layout.bytes] with `cached` rows
  const uint8_t* pool = nullptr;
  const int32_t* page_table = nullptr;
  const int32_t* page_ids = nullptr;     // the same on the host (at most kFp4ArgPages), used instead when given
  int n_pages = 0, num_pages = 0, page_rows = 0, last_page_rows = 0;
  uint8_t* cache_k = nullptr;
  uint8_t* cache_v = nullptr;
  int cached = 0;
  Fp4Layout layout;
  const float* k_new = nullptr;          // [n_new, heads, D]: rows that the queries see too; stored at row `cached` with `store`
  const float* v_new = nullptr;
  int n_new = 0, store = 0;
  __nv_bfloat16* out_bf16 = nullptr;     // [n_q, heads, D]
  float* out_f32 = nullptr;
  float* lse = nullptr;                  // [n_q, heads], natural logarithm
  // partial results of a call in several key ranges, and a counter per (head, eight queries), zero before and after every call
  float* part = nullptr;
  size_t part_floats = 0;
  int* counters = nullptr;
  int num_counters = 0;
  int* status = nullptr;
};
int launch_fp4_rows(const Fp4RowsLaunch& p, cudaStream_t stream);
// Attention of query tiles over a 4-bit pool; `a` as for launch_attention (tm_k, tm_v, key_norm_max and ctas_per_sm are not used).
// page_ids: as for Fp4RowsLaunch; exact_logits: for callers who want the log-sum-exp.
int launch_attention_fp4(const AttnLaunch& a, const uint8_t* pool, const Fp4Layout& layout, int num_pages, const int32_t* page_ids, bool exact_logits,
                         cudaStream_t stream);
// Key ranges that a call of n_q query rows of `heads` heads over `blocks` blocks of 128 rows is cut into.
int fp4_rows_splits(int n_q, int heads, int blocks, int head_dim, int sms, size_t part_floats, int num_counters);

}  // namespace gct
