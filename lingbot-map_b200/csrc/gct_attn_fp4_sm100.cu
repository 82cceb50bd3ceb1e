// Attention of whole query tiles over a 4-bit paged cache: softmax(Q K^T / 8) V with head_dim 64 on tcgen05, half-precision operands, fp32
// accumulation.  The sibling of gct_attn_kernel (gct_attn_sm100.cu): the same tiles of 128 query rows, the same softmax with two threads per
// row, the same split of the KV range over CTAs.  What differs is how K and V reach the tensor core.
//
//   producer warp      fetches blocks of 128 rows, packed (K and V, two bulk copies, 9.2 KB), into a ring
//   unpacking warps    (four for K, four for V) turn a packed block into 128 x 64 half-precision tiles in the 128B-swizzled layout the
//                      products want: a thread takes 32 values at a time, a conversion and a product with the scale per pair.  c * s is
//                      exact; rows past the valid ones get scale zero, so nothing that they hold counts.
//   MMA warps          S = Q K^T and O += P V, as there
//   softmax warps      as there, 32 columns of S at a time, so that 88 registers do (64 at a time spilled: 10 % slower)
//
// A value costs its unpacking once per CTA, for the 256 query rows of two tiles: 16,384 values a block, about 800 of the block's 6,100 warp
// instructions.  1005 queries over 131,928 tokens, kernel and merge back to back: 621 us in a burst (874 TFLOP/s, 0.51 of a library product's rate;
// the bf16 cache 559), 656 under the power cap; with the running maximum 932.  As the steps were made, nine equal ranges: 650 us; with four unpacking
// warps 692, without the fifth K16 step (below) 688, unpacking by the softmax warps between their blocks 742, without any unpacking (wrong
// results) 647 when the whole took 692.  What bounds it: as in gct_attn_kernel issue slots (packed f32x2 operations take two each) and the
// chain S -> registers -> P -> P V; issue 64 % busy, tensor pipe 48 %.
//
// Weights are half-precision numbers of up to 2^15: eleven bits where bf16 has eight.  Q is brought to half precision once per CTA.
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "gct_fp4.h"
#include "gct_sm100.h"

namespace gct {
namespace {

constexpr int kPackedStages = 4, kTileStages = 2;          // blocks (K and V) in flight packed, and unpacked
constexpr uint32_t kPackedBytes = kFp4BlockBytes<64>;
constexpr float kFp4Shift = 7.f;                           // running maximum: weights are at most 2^(kRescaleThreshold + kFp4Shift)
constexpr float kFixedShift = 15.f;                        // fixed reference: weights are at most 2^15
// One pair of logits in so many takes the FMA pipe for its exponentials.  1005 queries over 131,928 tokens, fixed reference / running maximum: three 626 / 951
// us, four 621 / 935, five 647 / 948, six 654 / 960.
constexpr int kPolyDen = 4;
// half-precision operands: formats 0; K-major A and B for S, MN-major B for P V
constexpr uint32_t kIdescS16 = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
constexpr uint32_t kIdescPV16 = (1u << 4) | (1u << 16) | ((64u >> 3) << 17) | ((128u >> 4) << 24);

// Warpgroups: two softmax per query tile, one of producer and MMA warps, two that unpack.
template <int QT>
constexpr int kFp4Threads = 256 * QT + 384;
// Two tiles: 896 threads start with 72 registers each, 64512 in all.  With 88 / 40 / 56 the control warpgroup spilled (28 bytes): 131,928 tokens 629 us, now 621;
// 96 / 40 / 40 627, 88 / 56 / 48 641.
constexpr int kFp4SoftmaxRegs = 88, kFp4ControlRegs = 48, kFp4UnpackRegs = 48;
static_assert(512 * kFp4SoftmaxRegs + 128 * kFp4ControlRegs + 256 * kFp4UnpackRegs <= 896 * 72, "register pool of the CTA exceeded");

template <int QT>
struct Fp4Smem {
  static constexpr uint32_t q_off = 0;
  static constexpr uint32_t tile_off = q_off + QT * kTileBytes;
  static constexpr uint32_t packed_off = tile_off + kTileStages * 2 * kTileBytes;
  static constexpr uint32_t pair_off = packed_off + kPackedStages * 2 * kPackedBytes;      // [2][QT][2][128] floats, as in gct_attn_kernel
  static constexpr uint32_t factor_off = pair_off + 2 * QT * 2 * 128 * 4;              // [QT][128] floats: a row's multiplier in front of exp2
  static constexpr uint32_t ref_off = factor_off + QT * 128 * 4;                       // [QT][128] floats: a row's fixed reference
  // operands of the fifth K16 step of S: columns [16 t, +16) Qx of tile t (column 0 = 15 - reference), [32, 48) Kx (column 0 = 1)
  static constexpr uint32_t x_off = (ref_off + QT * 128 * 4 + 1023) / 1024 * 1024;
  static constexpr uint32_t bar_off = x_off + kTileBytes;
  // q_full, q_ready, verdict, packed_full/empty[], K and V tile_full/empty[], per query tile s_full, s_empty, p_full[2], pv_full[2]
  static constexpr int n_bars = 3 + 2 * kPackedStages + 4 * kTileStages + 6 * QT;
  static constexpr uint32_t misc_off = bar_off + n_bars * 8;
  // [2 kTileStages] valid rows of an unpacked block.  K of block j is freed when S_j is done, which may be before the softmax has looked here;
  // K of block j + 2 kTileStages is unpacked after S_{j + kTileStages}, which began after the softmax had left block j.
  static constexpr uint32_t valid_off = misc_off + 16;
  static constexpr uint32_t total = valid_off + 2 * kTileStages * 4;
};

struct Fp4Args {
  const uint8_t* pool;
  const int32_t* page_table;
  int64_t head_bytes;
  int n_pages, num_pages, page_len, last_page_len, blocks_per_page, total_blocks, full_blocks, tail_rows;
  int n_q, heads, q_groups, splits, split_len, final_bf16;
  float scale_log2;
  __nv_bfloat16* out;
  float *part_o, *part_lse;
  int* status;
  const float* key_norm_max;      // [heads]: bounds the 2-norm of every key of a head (null: unknown)
  float fixed_limit;              // largest bound of a row's exponents that the fixed reference is tried with
};

// kFold: S arrives as the finished base-2 exponent, less the row's reference (bf16 results: q is rounded once more
// with its scale, to at most 2^-11 of each product, eight times finer than the bf16 that q comes in; the error against 64 bits stays 1.7e-3, that
// of the results' own rounding); otherwise scale and reference enter by a multiply-add in fp32, for callers who want the log-sum-exp.
template <int QT, bool kFold>
__global__ void __launch_bounds__(kFp4Threads<QT>, 1) gct_attn_fp4_kernel(const __grid_constant__ CUtensorMap tm_q, const Fp4Args a,
                                                                              const __grid_constant__ Fp4Pages pages) {
  using L = Fp4Smem<QT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bars = sbase + L::bar_off;
  auto bar_q_full = [&]() { return bars; };
  auto bar_q_ready = [&]() { return bars + 8u; };
  auto bar_verdict = [&]() { return bars + 16u; };
  auto bar_packed_full = [&](int s) { return bars + 8u * (3 + s); };
  auto bar_packed_empty = [&](int s) { return bars + 8u * (3 + kPackedStages + s); };
  auto bar_tile_full = [&](int s, int v) { return bars + 8u * (3 + 2 * kPackedStages + 2 * s + v); };      // v: 0 K, 1 V
  auto bar_tile_empty = [&](int s, int v) { return bars + 8u * (3 + 2 * kPackedStages + 2 * kTileStages + 2 * s + v); };
  constexpr int kFirst = 3 + 2 * kPackedStages + 4 * kTileStages;
  auto bar_s_full = [&](int t) { return bars + 8u * (kFirst + 6 * t + 0); };
  auto bar_s_empty = [&](int t) { return bars + 8u * (kFirst + 6 * t + 1); };
  auto bar_p_full = [&](int t, int half) { return bars + 8u * (kFirst + 6 * t + 2 + half); };
  auto bar_pv_full = [&](int t, int half) { return bars + 8u * (kFirst + 6 * t + 4 + half); };
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + L::misc_off);
  volatile int* cta_abort = reinterpret_cast<volatile int*>(smem + L::misc_off + 4);
  volatile int* cta_exact = reinterpret_cast<volatile int*>(smem + L::misc_off + 8);      // running maximum from the start
  volatile int* cta_redo = reinterpret_cast<volatile int*>(smem + L::misc_off + 12);      // the fixed reference has not held

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kProducerWarp = 8 * QT, kFirstMmaWarp = 8 * QT + 1, kFirstUnpackWarp = 8 * QT + 4;
  constexpr uint32_t kTmemCols = QT == 2 ? 512u : 256u;
  constexpr uint32_t kOCol = 128u * QT, kPCol = 192u * QT;

  // ---- work coordinates, as in gct_attn_kernel ----
  int idx = blockIdx.x;
  const int qg = idx % a.q_groups;
  idx /= a.q_groups;
  int split, h, g0, g1;
  if (a.split_len == 0) {
    split = idx % a.splits;
    h = idx / a.splits;
    g0 = static_cast<int>(static_cast<long long>(split) * a.total_blocks / a.splits);
    g1 = static_cast<int>(static_cast<long long>(split + 1) * a.total_blocks / a.splits);
  } else {
    h = idx % a.heads;
    split = idx / a.heads;
    g0 = split * a.split_len;
    g1 = split == a.splits - 1 ? a.total_blocks : g0 + a.split_len;
  }
  const int nblk = g1 - g0;

  // ---- set-up ----
  if (threadIdx.x == 0) {
    mbar_init(bar_q_full(), 1);
    mbar_init(bar_q_ready(), 4 * QT);
    mbar_init(bar_verdict(), 8 * QT);
    for (int s = 0; s < kPackedStages; ++s) {
      mbar_init(bar_packed_full(s), 1);
      mbar_init(bar_packed_empty(s), 8);
    }
    for (int s = 0; s < kTileStages; ++s) {
      for (int v = 0; v < 2; ++v) {
        mbar_init(bar_tile_full(s, v), 4);
        mbar_init(bar_tile_empty(s, v), QT);
      }
    }
    for (int t = 0; t < QT; ++t) {
      mbar_init(bar_s_full(t), 1);
      mbar_init(bar_s_empty(t), 8);
      mbar_init(bar_p_full(t, 0), 4);
      mbar_init(bar_p_full(t, 1), 4);
      mbar_init(bar_pv_full(t, 0), 1);
      mbar_init(bar_pv_full(t, 1), 1);
    }
    *cta_abort = 0;
    *cta_exact = a.key_norm_max == nullptr;
    *cta_redo = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kFirstMmaWarp) tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), kTmemCols);
  if (warp == kProducerWarp && lane == 0) tma_prefetch_desc(&tm_q);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();

  // A CTA goes through its KV range a second time when the fixed reference has not held; every role but the softmax waits here for
  // the verdict: behind the first pass, or as soon as the running maximum is chosen from the start (a short range may be unpacked before that).
  auto again = [&]() -> bool { return mbar_wait(bar_verdict(), 0, cta_abort, a.status) && *cta_redo != 0; };

  // Where a role is in its range: the page, how many of its blocks are left, this one included, the rows that this block holds in memory and
  // those of them that are valid.
  struct Place {
    int page, left, rows, valid;
  };
  auto blocks_of = [&](int page) { return page == a.n_pages - 1 ? a.total_blocks - page * a.blocks_per_page : a.blocks_per_page; };
  auto end_of_page = [&](Place& p) {                       // at the last block of a page
    const int block = blocks_of(p.page) - 1;
    p.rows = block < a.full_blocks ? kFp4Rows : a.tail_rows;
    p.valid = (p.page == a.n_pages - 1 ? a.last_page_len : a.page_len) - block * kFp4Rows;
  };
  auto first_place = [&]() -> Place {
    Place p = {g0 / a.blocks_per_page, 0, kFp4Rows, kFp4Rows};
    p.left = blocks_of(p.page) - (g0 - p.page * a.blocks_per_page);
    if (p.left == 1) end_of_page(p);
    return p;
  };
  auto advance = [&](Place& p) {
    if (--p.left > 1) return;
    if (p.left == 0) {
      p = {p.page + 1, blocks_of(p.page + 1), kFp4Rows, kFp4Rows};
      if (p.left > 1) return;
    }
    end_of_page(p);
  };
  // keys of the range: whole blocks, less what the last block of each page that ends in it lacks
  auto keys_of_range = [&]() -> int {
    const int first = g0 / a.blocks_per_page, last = (g1 - 1) / a.blocks_per_page;
    const bool whole = g1 == a.total_blocks || g1 % a.blocks_per_page == 0;      // the range's last page ends in it
    const int lack = a.blocks_per_page * kFp4Rows - a.page_len;
    int keys = nblk * kFp4Rows - (last - first) * lack;
    if (whole) keys -= last == a.n_pages - 1 ? (a.total_blocks - last * a.blocks_per_page) * kFp4Rows - a.last_page_len : lack;
    return keys;
  };

  if (warp >= kFirstUnpackWarp) {
    // =========================== unpacking warps: four take K, four V ===========================
    if constexpr (QT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFp4UnpackRegs));
    // A thread takes half rows (sixteen bytes, 32 values) of rows tid / 2 and 64 further on: loads are consecutive, and eight threads
    // store to four rows and both their halves, which the swizzle puts into eight different 16-byte columns.
    const int v = (warp - kFirstUnpackWarp) >> 2, tid = (threadIdx.x - 32 * kFirstUnpackWarp) & 127, row = tid >> 1;
    const uint32_t to0 = sbase + L::tile_off + v * kTileBytes + row * 128 + ((((tid & 1) * 4) ^ (row & 7)) << 4);
    auto wait = [&](uint32_t bar, uint32_t parity) -> bool { return __all_sync(0xffffffffu, mbar_wait(bar, parity, cta_abort, a.status)); };
    Place at = first_place();
    for (int j = 0, end = nblk; j < end; ++j) {
      const int ps = j % kPackedStages, ts = j % kTileStages, rows = at.rows, valid = at.valid;
      if (!wait(bar_packed_full(ps), (j / kPackedStages) & 1) || !wait(bar_tile_empty(ts, v), ((j / kTileStages) & 1) ^ 1u)) break;
      const uint8_t* from = smem + L::packed_off + (ps * 2 + v) * kPackedBytes;
      uint4 w[2];
      uint32_t scales[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        w[u] = *reinterpret_cast<const uint4*>(from + tid * 16 + u * 2048);
        scales[u] = *reinterpret_cast<const uint16_t*>(from + rows * 32 + tid * 2 + u * 256);
      }
      if (valid < kFp4Rows) {
        if (row >= valid) scales[0] = 0;
        if (row + 64 >= valid) scales[1] = 0;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t s0 = (scales[u] & 0xffu) * 0x00800080u, s1 = (scales[u] >> 8) * 0x00800080u;
        const uint32_t words[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t p[4];
          fp4_unpack8(words[e], p);
          const uint32_t s = e < 2 ? s0 : s1;
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(((to0 + ts * 2 * kTileBytes) ^ (e << 4)) + u * 8192), "r"(half2_mul(p[0], s)),
                       "r"(half2_mul(p[1], s)), "r"(half2_mul(p[2], s)), "r"(half2_mul(p[3], s))
                       : "memory");
        }
      }
      if (v == 0 && tid == 0) *reinterpret_cast<volatile int*>(smem + L::valid_off + 4 * (j % (2 * kTileStages))) = valid;
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar_tile_full(ts, v));
        mbar_arrive(bar_packed_empty(ps));
      }
      advance(at);
      if (j + 1 == nblk && __all_sync(0xffffffffu, again())) {
        end = 2 * nblk;
        at = first_place();
      }
    }
  } else if (warp == kProducerWarp) {
    // =========================== producer ===========================
    if constexpr (QT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFp4ControlRegs));
    if (lane == 0) {
      mbar_arrive_expect_tx(bar_q_full(), QT * kTileBytes);
      for (int t = 0; t < QT; ++t) tma_load_4d(sbase + L::q_off + t * kTileBytes, &tm_q, bar_q_full(), 0, h, (qg * QT + t) * kTileM, 0);
      int cur = -1;
      const uint8_t* from = nullptr;
      Place at = first_place();
      for (int j = 0, end = nblk; j < end; ++j) {
        if (at.page != cur) {
          cur = at.page;
          const int page = a.page_table == nullptr ? pages.id[cur] : __ldg(a.page_table + cur);
          if (page < 0 || page >= a.num_pages) {
            atomicCAS(a.status, 0, kStatusBadIndex);
            *cta_abort = 1;
            break;
          }
          from = a.pool + (static_cast<int64_t>(page) * 2 * a.heads + h) * a.head_bytes + static_cast<int64_t>(blocks_of(cur) - at.left) * kPackedBytes;
        }
        const int ps = j % kPackedStages;
        if (!mbar_wait(bar_packed_empty(ps), ((j / kPackedStages) & 1) ^ 1u, cta_abort, a.status)) break;
        const uint32_t bytes = at.rows * kFp4RowBytes<64>, to = sbase + L::packed_off + ps * 2 * kPackedBytes;
        mbar_arrive_expect_tx(bar_packed_full(ps), 2 * bytes);
        bulk_load(to, from, bytes, bar_packed_full(ps));
        bulk_load(to + kPackedBytes, from + a.heads * a.head_bytes, bytes, bar_packed_full(ps));
        from += kPackedBytes;
        advance(at);
        if (j + 1 == nblk && again()) {
          end = 2 * nblk;
          at = first_place();
          cur = -1;
        }
      }
    }
  } else if (warp > kProducerWarp) {
    // =========================== MMA issuer of tile t ===========================
    if constexpr (QT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFp4ControlRegs));
    const int t = warp - kFirstMmaWarp;
    if (t < QT) {
      const uint32_t lead = elect_one();
      auto tile_parity = [](int j) -> uint32_t { return (j / kTileStages) & 1; };
      auto issue_s = [&](int s) {
        const uint64_t ad = smem_desc(sbase + L::q_off + t * kTileBytes, 16, 1024);
        const uint64_t bd = smem_desc(sbase + L::tile_off + s * 2 * kTileBytes, 16, 1024);
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_ss(lead, tmem_base + t * 128, ad + 2 * k, bd + 2 * k, kIdescS16, k > 0);
        if constexpr (kFold) {
          const uint64_t xd = smem_desc(sbase + L::x_off, 16, 1024);
          umma_ss(lead, tmem_base + t * 128, xd + 2 * t, xd + 4, kIdescS16, 1u);
        }
      };
      auto issue_pv = [&](int s, int half, uint32_t accumulate) {
        const uint64_t bd = smem_desc(sbase + L::tile_off + (2 * s + 1) * kTileBytes, 16, 1024);
#pragma unroll
        for (int k = 4 * half; k < 4 * half + 4; ++k)
          umma_ts(lead, tmem_base + kOCol + t * 64, tmem_base + kPCol + t * 64 + k * 8, bd + k * 128, kIdescPV16, k > 0 ? 1u : accumulate);
      };
      auto wait = [&](uint32_t bar, uint32_t parity) -> bool { return __all_sync(0xffffffffu, mbar_wait(bar, parity, cta_abort, a.status)); };
      // block j of all passes; S_j may overwrite S_{j-1} once that is in registers
      auto start_s = [&](int j) -> bool {
        const int s = j % kTileStages;
        if (j > 0 && !wait(bar_s_empty(t), (j - 1) & 1)) return false;
        if (!wait(bar_tile_full(s, 0), tile_parity(j))) return false;
        tc_fence_after();
        issue_s(s);
        tc_commit_elected(lead, bar_s_full(t));
        tc_commit_elected(lead, bar_tile_empty(s, 0));
        return true;
      };
      bool ok = wait(bar_q_ready(), 0);
      bool both = *cta_exact != 0;            // a running maximum: either half's threads may have rescaled O before
      for (int first = 0; ok;) {
        ok = start_s(first);
        for (int j = first; ok && j < first + nblk; ++j) {
          if (j + 1 < first + nblk && !(ok = start_s(j + 1))) break;
          const int s = j % kTileStages;
          if (!(ok = wait(bar_p_full(t, 0), j & 1))) break;
          if (both && !(ok = wait(bar_p_full(t, 1), j & 1))) break;
          if (!(ok = wait(bar_tile_full(s, 1), tile_parity(j)))) break;
          tc_fence_after();
          issue_pv(s, 0, j > first ? 1u : 0u);
          tc_commit_elected(lead, bar_pv_full(t, 0));
          if (!both) {
            if (!(ok = wait(bar_p_full(t, 1), j & 1))) break;
            tc_fence_after();
          }
          issue_pv(s, 1, 1u);
          tc_commit_elected(lead, bar_pv_full(t, 1));
          tc_commit_elected(lead, bar_tile_empty(s, 1));
        }
        if (!ok || both || first > 0 || !__all_sync(0xffffffffu, again())) break;
        first = nblk;
        both = true;
      }
    }
  } else {
    // =========================== softmax ===========================
    if constexpr (QT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kFp4SoftmaxRegs));
    const int t = warp >> 3, half = (warp >> 2) & 1;
    const int row = ((warp & 3) << 5) | lane;
    const uint32_t lane_addr = static_cast<uint32_t>((warp & 3) << 5) << 16;
    const uint32_t s_addr = tmem_base + lane_addr + t * 128 + half * 64;
    const uint32_t o_addr = tmem_base + lane_addr + kOCol + t * 64 + half * 32;
    const uint32_t p_addr = tmem_base + lane_addr + kPCol + t * 64 + half * 32;
    const uint32_t pair_mine = sbase + L::pair_off + (2 * t + half) * 512 + row * 4;
    const uint32_t pair_other = sbase + L::pair_off + (2 * t + (half ^ 1)) * 512 + row * 4;
    const int pair_bar = 1 + 4 * t + (warp & 3);
    const uint32_t lead = lane == 0 ? 1u : 0u;
    bool ok = true;
    auto wait_v = [&](uint32_t bar, uint32_t parity) -> bool { return __all_sync(0xffffffffu, mbar_wait(bar, parity, cta_abort, a.status)); };
    auto wait_u = [&](uint32_t bar, uint32_t parity) -> bool { return mbar_wait(bar, parity, cta_abort, a.status); };
    auto pair_sync = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory"); };
    auto pair_exchange = [&](float x, uint32_t slot) -> float {
      asm volatile("st.shared.f32 [%0], %1;" ::"r"(pair_mine + slot), "f"(x) : "memory");
      pair_sync();
      float y;
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(y) : "r"(pair_other + slot) : "memory");
      return y;
    };
    constexpr uint32_t kPairSlot = QT * 2 * 128 * 4;

    // ---- once per CTA: the Q row in half precision, its factor and its fixed reference ----
    // Normalised: times the power of two that puts its largest value into [2^14, 2^15): bf16 queries lose nothing that an fp32 sum would keep, and
    // the row's factor in front of the exponential undoes it.  Folded: times scale * log2(e), where the reference holds and the row's values
    // lie well inside the range of half precision.
    float* factor = reinterpret_cast<float*>(smem + L::factor_off) + t * 128 + row;
    float* reference = reinterpret_cast<float*>(smem + L::ref_off) + t * 128 + row;
    auto softmax_sync = [&]() { asm volatile("bar.sync 15, %0;" ::"n"(256 * QT) : "memory"); };      // all softmax threads, also after a failed wait
    {
      const uint32_t q_row = sbase + L::q_off + t * kTileBytes + row * 128;
      auto chunk = [&](int j) { return q_row + ((static_cast<uint32_t>(j) ^ (row & 7)) << 4); };
      uint32_t top = 0;
      if (half == 0) {
        ok = wait_v(bar_q_full(), 0);
        if (ok) {
          float sq = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            uint32_t w[4];
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(chunk(j)));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float lo = __uint_as_float(w[i] << 16), hi = __uint_as_float(w[i] & 0xffff0000u);
              top = max(top, max(fp4_abs_bits(lo), fp4_abs_bits(hi)));
              sq = fmaf(lo, lo, fmaf(hi, hi, sq));
            }
          }
          if (a.key_norm_max != nullptr) {
            // rounded up: to an eighth, which half precision holds, and by more than what rounding adds to the row (2^-11 relative)
            const float ref = ceilf(8.008f * sqrtf(sq) * __ldg(a.key_norm_max + h) * a.scale_log2) * 0.125f, largest = __uint_as_float(top) * a.scale_log2;
            *reference = ref;
            if (!(ref <= a.fixed_limit) || (kFold && top != 0 && !(largest >= 0x1p-8f && largest <= 0x1p15f))) *cta_exact = 1;     // NaN too
          }
        }
      }
      softmax_sync();
      if (half == 0 && ok) {
        const bool folded = kFold && *cta_exact == 0;
        // at most 2^64; 1 for a row of zeros or with a value that is not finite
        const int up = top == 0 || top >= 0x7f800000u ? 0 : min(14 + 127 - static_cast<int>(top >> 23), 64);
        const float f = folded ? a.scale_log2 : __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
        *factor = folded ? 1.f : a.scale_log2 / f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t w[4];
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(chunk(j)));
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = pack_f16x2(__uint_as_float(w[i] << 16) * f, __uint_as_float(w[i] & 0xffff0000u) * f);
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(chunk(j)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
        }
        if constexpr (kFold) {
          const uint32_t x_row = sbase + L::x_off + row * 128;
          auto st_chunk = [&](int j, uint32_t first) {
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %2, %2};" ::"r"(x_row + ((static_cast<uint32_t>(j) ^ (row & 7)) << 4)), "r"(first), "r"(0u) : "memory");
          };
          st_chunk(2 * t, folded ? pack_f16x2(kFixedShift - *reference, 0.f) : 0u);
          st_chunk(2 * t + 1, 0u);
          if (t == 0) {
            st_chunk(4, 0x3c00u);
            st_chunk(5, 0u);
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_q_ready());
      }
    }
    const bool fixed = *cta_exact == 0;
    if (!fixed && lane == 0) mbar_arrive(bar_verdict());
    pair_sync();                                           // the factor of the row
    const float c = *factor;
    float m = -INFINITY, l = 0.f;                          // m: reference maximum (units of S); l: sum over this half

    // P = exp2(S c + shift) of some logits as half-precision pairs, and their sum, software-pipelined over pairs as in gct_attn_kernel.
    // kBelow: exponents may lie below -126.
    auto sweep = [&](auto& s, auto& pk, float shift, auto below) -> float {
      constexpr int kPairs = sizeof(pk) / sizeof(pk[0]);
      constexpr bool kBelow = decltype(below)::value;
      const float2 c2 = make_float2(c, c), shift2 = make_float2(shift, shift);
      float2 acc0 = make_float2(0.f, 0.f), acc1 = make_float2(0.f, 0.f);
      auto pair_ffma = [&](int q) {
        if constexpr (!kBelow && kFold) return;            // S is the exponent
        const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[2 * q]), __uint_as_float(s[2 * q + 1])), c2, shift2);
        s[2 * q] = __float_as_uint(x.x);
        s[2 * q + 1] = __float_as_uint(x.y);
      };
      auto pair_exp = [&](int q) {
        if ((q + 1) / kPolyDen != q / kPolyDen) {
          const float2 x = make_float2(__uint_as_float(s[2 * q]), __uint_as_float(s[2 * q + 1]));
          const float2 e = kBelow ? exp2_poly2(x) : exp2_poly2_inrange(x);
          s[2 * q] = __float_as_uint(e.x);
          s[2 * q + 1] = __float_as_uint(e.y);
        } else {
          s[2 * q] = __float_as_uint(fast_exp2(__uint_as_float(s[2 * q])));
          s[2 * q + 1] = __float_as_uint(fast_exp2(__uint_as_float(s[2 * q + 1])));
        }
      };
      auto pair_sum = [&](int q) {
        const float2 e = make_float2(__uint_as_float(s[2 * q]), __uint_as_float(s[2 * q + 1]));
        if (q & 1) acc1 = __fadd2_rn(acc1, e); else acc0 = __fadd2_rn(acc0, e);
        pk[q] = pack_f16x2(e.x, e.y);
      };
#pragma unroll
      for (int q = 0; q < kFfmaAhead; ++q) pair_ffma(q);
#pragma unroll
      for (int q = 0; q < kPairs; ++q) {
        if (q + kFfmaAhead < kPairs) pair_ffma(q + kFfmaAhead);
        pair_exp(q);
        if (q >= kSumLag) pair_sum(q - kSumLag);
      }
#pragma unroll
      for (int q = kPairs - kSumLag; q < kPairs; ++q) pair_sum(q);
      return (acc0.x + acc0.y) + (acc1.x + acc1.y);
    };
    using Yes = std::true_type;
    using No = std::false_type;
    auto load_s = [&](int ch, int valid, uint32_t hidden, uint32_t (&s)[32]) {       // 32 columns of this thread's half; `valid` of the 64 count
      tmem_ld32(s_addr + 32 * ch, s);
      tmem_wait_ld();
      if (valid < 64) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (32 * ch + i >= valid) s[i] = hidden;
      }
    };
    auto s_taken = [&]() {                                 // the tensor core may overwrite S with the next block
      tc_fence_before();
      __syncwarp();
      mbar_arrive_elected(lead, bar_s_empty(t));
    };
    auto p_stored = [&]() {
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      mbar_arrive_elected(lead, bar_p_full(t, half));
    };
    auto valid_rows = [&](int j) { return *reinterpret_cast<volatile int*>(smem + L::valid_off + 4 * (j % (2 * kTileStages))); };
    // ---- fixed reference: |q| max|k| bounds every exponent of the row (Cauchy-Schwarz); no maximum, no exchange, no rescaling ----
    // Weights are exp2(x - ref + 15), at most 2^15.  Half precision holds them to 2^-25 at least, so over n keys at most n 2^-25 of the sum is lost
    // to rounding small ones; a row whose sum is at least n 2^-15 has lost less than 2^-10 of it.  A CTA with a row below that goes through its
    // range again with the running maximum.
    bool held = false;
    if (fixed) {
      const float shift = kFold ? 0.f : kFixedShift - *reference;
      const uint32_t hidden = __float_as_uint(kFold ? -100.f : (-100.f - shift) / c);      // weighs 2^-100
      for (int j = 0; ok && j < nblk; ++j) {
        if (!(ok = wait_u(bar_s_full(t), j & 1))) break;
        tc_fence_after();
        const int valid = valid_rows(j) - 64 * half;
#pragma unroll
        for (int ch = 0; ch < 2; ++ch) {
          uint32_t s[32], pk[16];
          tmem_ld32(s_addr + 32 * ch, s);
          tmem_wait_ld();
          if (ch == 1) s_taken();
          if (valid < 64) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (32 * ch + i >= valid) s[i] = hidden;
          }
          l += sweep(s, pk, shift, No());
          if (ch == 0 && j > 0) {                          // P is free once the product of the block before has read it
            if (!(ok = wait_u(bar_pv_full(t, half), (j - 1) & 1))) break;
            tc_fence_after();
          }
          tmem_st16(p_addr + 16 * ch, pk);
        }
        if (!ok) break;
        p_stored();
      }
      __syncwarp();
      if (ok && nblk > 0) ok = wait_v(bar_pv_full(t, 1), (nblk - 1) & 1);
      const float other = pair_exchange(l, 0);
      l = half == 0 ? l + other : other + l;
      if (ok && !(l >= static_cast<float>(keys_of_range()) * 0x1p-15f)) *cta_redo = 1;
      softmax_sync();
      held = *cta_redo == 0;
      if (lane == 0) mbar_arrive(bar_verdict());
      if (held) {
        m = *reference;
      } else {
        l = 0.f;
      }
    }
    // ---- running maximum ----
    if (!held) {
      const int first = fixed ? nblk : 0;
      int met = 0;
      for (int j = first; ok && j < first + nblk; ++j) {
        if (!(ok = wait_u(bar_s_full(t), j & 1))) break;
        tc_fence_after();
        const int valid = valid_rows(j) - 64 * half;
        // S is read twice: the maximum, then the weights
        uint32_t s[32], pk[16];
        float mx = -INFINITY;
#pragma unroll
        for (int ch = 0; ch < 2; ++ch) {
          load_s(ch, valid, 0xff800000u, s);
          float mxc[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) mxc[i] = __uint_as_float(s[i]);
#pragma unroll
          for (int i = 4; i < 32; i += 2) mxc[(i >> 1) & 3] = max3(mxc[(i >> 1) & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
          mx = fmaxf(mx, fmaxf(fmaxf(mxc[0], mxc[1]), fmaxf(mxc[2], mxc[3])));
        }
        mx = fmaxf(mx, pair_exchange(mx, ((met + 1) & 1) * kPairSlot));
        ++met;
        float alpha = 1.f;
        if ((mx - m) * c > kRescaleThreshold) {            // always true on the first block (m = -inf)
          alpha = fast_exp2((m - mx) * c);
          m = mx;
        }
        // exponents so large that rounding m * c would move them: the maximum is taken off first
        const float base = m * c;
        const bool huge = __any_sync(0xffffffffu, fabsf(base) > 65536.f);
        l *= alpha;
#pragma unroll
        for (int ch = 0; ch < 2; ++ch) {
          load_s(ch, valid, 0xff800000u, s);
          if (ch == 1) s_taken();
          if (huge) {
#pragma unroll
            for (int i = 0; i < 32; ++i) s[i] = __float_as_uint(__uint_as_float(s[i]) - m);
          }
          l += sweep(s, pk, kFp4Shift - (huge ? 0.f : base), Yes());
          if (ch == 0 && j > first) {
            if (!(ok = wait_u(bar_pv_full(t, 1), (j - 1) & 1))) break;
            tc_fence_after();
            if (__any_sync(0xffffffffu, alpha != 1.f)) {
              uint32_t ob[32];
              tmem_ld32(o_addr, ob);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) ob[i] = __float_as_uint(__uint_as_float(ob[i]) * alpha);
              tmem_st32(o_addr, ob);
            }
          }
          tmem_st16(p_addr + 16 * ch, pk);
        }
        if (!ok) break;
        p_stored();
      }
      __syncwarp();
      for (; met < nblk; ++met) pair_sync();
      if (ok && nblk > 0) ok = wait_v(bar_pv_full(t, 1), (first + nblk - 1) & 1);
      const float other = pair_exchange(l, ((nblk + 1) & 1) * kPairSlot);
      l = half == 0 ? l + other : other + l;
      // as above: the exponent that weighs 2^kFixedShift; a first pass has left its reference folded into S
      m = m * c + (kFixedShift - kFp4Shift) - (kFold && fixed ? kFixedShift - *reference : 0.f);
    }

    // ---- epilogue: O / l ----
    const int qrow = (qg * QT + t) * kTileM + row;
    if (ok && nblk > 0) {
      tc_fence_after();
      uint32_t ob[32];
      tmem_ld32(o_addr, ob);
      tmem_wait_ld();
      const float inv = 1.f / l;
      const size_t rowidx = static_cast<size_t>(qrow < a.n_q ? qrow : 0) * a.heads + h;
      const size_t prow = static_cast<size_t>(split) * a.n_q * a.heads + rowidx;
      if (qrow < a.n_q) {
        if (a.final_bf16) {
          uint4* dst = reinterpret_cast<uint4*>(a.out + rowidx * kHeadDim + half * 32);
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4) {
            uint4 w;
            w.x = pack_bf16x2(__uint_as_float(ob[q4 * 8 + 0]) * inv, __uint_as_float(ob[q4 * 8 + 1]) * inv);
            w.y = pack_bf16x2(__uint_as_float(ob[q4 * 8 + 2]) * inv, __uint_as_float(ob[q4 * 8 + 3]) * inv);
            w.z = pack_bf16x2(__uint_as_float(ob[q4 * 8 + 4]) * inv, __uint_as_float(ob[q4 * 8 + 5]) * inv);
            w.w = pack_bf16x2(__uint_as_float(ob[q4 * 8 + 6]) * inv, __uint_as_float(ob[q4 * 8 + 7]) * inv);
            dst[q4] = w;
          }
        } else {
          float4* dst = reinterpret_cast<float4*>(a.part_o + prow * kHeadDim + half * 32);
#pragma unroll
          for (int q4 = 0; q4 < 8; ++q4)
            dst[q4] = make_float4(__uint_as_float(ob[q4 * 4 + 0]) * inv, __uint_as_float(ob[q4 * 4 + 1]) * inv, __uint_as_float(ob[q4 * 4 + 2]) * inv,
                                  __uint_as_float(ob[q4 * 4 + 3]) * inv);
          if (half == 0) a.part_lse[prow] = (m + log2f(l) - kFixedShift) * 0.6931471805599453f;
        }
      }
    }
  }

  // ---- teardown: every thread arrives here, also after an abort ----
  if (*cta_abort) {
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kFirstMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

std::mutex g_fp4_mutex;
bool g_fp4_ready[64] = {false};

int prepare_device() {
  int dev = -1;
  GCT_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return fail(GCT_ERR_INVALID, "attention: device ordinal out of range");
  std::lock_guard<std::mutex> lock(g_fp4_mutex);
  if (g_fp4_ready[dev]) return GCT_OK;
  // setmaxnreg hands out no more registers than the CTA was launched with and waits for ever for the rest: never launch such a build
  auto prepare = [](auto kernel, int smem, int pool) -> int {
    GCT_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    cudaFuncAttributes attr;
    GCT_CUDA_CHECK(cudaFuncGetAttributes(&attr, kernel));
    return attr.numRegs < pool ? fail(GCT_ERR_INVALID, "attention: the kernel was built with fewer registers than its warpgroups share") : GCT_OK;
  };
  constexpr int kPool = (512 * kFp4SoftmaxRegs + 128 * kFp4ControlRegs + 256 * kFp4UnpackRegs) / kFp4Threads<2>;
  int rc = prepare(gct_attn_fp4_kernel<2, true>, Fp4Smem<2>::total + 1024, kPool);
  if (rc == GCT_OK) rc = prepare(gct_attn_fp4_kernel<2, false>, Fp4Smem<2>::total + 1024, kPool);
  if (rc == GCT_OK) rc = prepare(gct_attn_fp4_kernel<1, true>, Fp4Smem<1>::total + 1024, 0);
  if (rc == GCT_OK) rc = prepare(gct_attn_fp4_kernel<1, false>, Fp4Smem<1>::total + 1024, 0);
  if (rc != GCT_OK) return rc;
  g_fp4_ready[dev] = true;
  return GCT_OK;
}

}  // namespace

int launch_attention_fp4(const AttnLaunch& a, const uint8_t* pool, const Fp4Layout& layout, int num_pages, const int32_t* page_ids, bool exact_logits,
                         cudaStream_t stream) {
  if (a.n_q <= 0 || a.heads <= 0 || a.batch != 1 || a.n_pages <= 0 || a.page_len <= 0 || a.last_page_len <= 0 || a.last_page_len > a.page_len ||
      pool == nullptr || (a.page_table == nullptr && page_ids == nullptr) || a.status == nullptr || (a.q_tiles_per_cta != 1 && a.q_tiles_per_cta != 2))
    return fail(GCT_ERR_INVALID, "attention: bad shape");
  Fp4Args k = {};
  k.pool = pool;
  k.page_table = a.page_table;
  k.head_bytes = layout.bytes;
  k.n_pages = a.n_pages;
  k.num_pages = num_pages;
  k.page_len = a.page_len;
  k.last_page_len = a.last_page_len;
  k.blocks_per_page = (a.page_len + kBlockN - 1) / kBlockN;
  k.total_blocks = (a.n_pages - 1) * k.blocks_per_page + (a.last_page_len + kBlockN - 1) / kBlockN;
  k.full_blocks = layout.full_blocks;
  k.tail_rows = layout.tail_rows;
  k.n_q = a.n_q;
  k.heads = a.heads;
  const int rows_per_cta = kTileM * a.q_tiles_per_cta;
  k.q_groups = (a.n_q + rows_per_cta - 1) / rows_per_cta;
  k.splits = a.splits;
  k.split_len = a.split_len;
  k.final_bf16 = a.final_bf16 ? 1 : 0;
  k.scale_log2 = 0.125f * 1.4426950408889634f;
  k.out = a.out;
  k.part_o = a.part_o;
  k.part_lse = a.part_lse;
  k.status = a.status;
  k.key_norm_max = a.key_norm_max;
  k.fixed_limit = a.bounded_limit;
  if (a.splits < 1 || a.splits > k.total_blocks) return fail(GCT_ERR_INVALID, "attention: splits out of range");
  if (a.split_len != 0) {
    const long long rest = static_cast<long long>(k.total_blocks) - static_cast<long long>(a.splits - 1) * a.split_len;
    if (a.split_len < 0 || a.splits < 2 || rest < 1 || rest > a.split_len) return fail(GCT_ERR_INVALID, "attention: split_len does not cover the KV blocks");
  }
  if (a.final_bf16 ? a.splits != 1 || a.out == nullptr : a.part_o == nullptr || a.part_lse == nullptr)
    return fail(GCT_ERR_INVALID, "attention: output buffers missing");
  const long long grid = static_cast<long long>(k.q_groups) * a.splits * a.heads;
  if (grid > 0x7fffffffLL) return fail(GCT_ERR_INVALID, "attention: grid too large");
  const int rc = prepare_device();
  if (rc != GCT_OK) return rc;
  const dim3 g(static_cast<unsigned>(grid));
  Fp4Pages pages = {};
  if (page_ids != nullptr) {
    if (a.n_pages > kFp4ArgPages) return fail(GCT_ERR_INVALID, "attention: too many pages for an argument");
    std::copy(page_ids, page_ids + a.n_pages, pages.id);
    k.page_table = nullptr;
  }
  auto launch = [&](auto kernel, int threads, int smem) { return launch_pdl(kernel, g, dim3(threads), smem, stream, a.tm_q, k, pages); };
  if (a.q_tiles_per_cta == 2)
    GCT_CUDA_CHECK(launch(exact_logits ? gct_attn_fp4_kernel<2, false> : gct_attn_fp4_kernel<2, true>, kFp4Threads<2>, Fp4Smem<2>::total + 1024));
  else
    GCT_CUDA_CHECK(launch(exact_logits ? gct_attn_fp4_kernel<1, false> : gct_attn_fp4_kernel<1, true>, kFp4Threads<1>, Fp4Smem<1>::total + 1024));
  return GCT_OK;
}

}  // namespace gct
