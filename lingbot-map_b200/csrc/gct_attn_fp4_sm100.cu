// Attention of whole query tiles over a 4-bit paged cache: softmax(Q K^T / 8) V with head_dim 64 on tcgen05, half-precision operands, fp32
// accumulation.  The sibling of gct_attn_kernel (gct_attn_sm100.cu): the same tiles of 128 query rows, the same softmax with two threads per
// row, the same split of the KV range over CTAs.  What differs is how K and V reach the tensor core.
//
//   producer warp      fetches blocks of 128 rows of K and V by turns, packed, one bulk copy each (4.6 KB), into a ring
//   dequantising warps (four) turn a packed block into a 128 x 64 half-precision tile in the 128B-swizzled layout the products want: a
//                      thread takes 32 values at a time, a conversion and a product with the scale per pair.  c * s is exact, rows past the
//                      valid ones get scale zero, so nothing that they hold counts.
//   MMA warps          S = Q K^T and O += P V, as there
//
// A value costs its unpacking once per CTA, for the 256 query rows of two tiles: 16,384 values a block, about 170 of the block's 2,000
// clocks of issue.  Q is brought to half precision once per CTA: each row times the power of two that puts its largest value into
// [2^14, 2^15) - bf16 queries lose nothing that an fp32 sum would keep - and the row's factor goes back into the multiply-add in front
// of its exponential.  Weights are half-precision numbers of up to 2^15: eleven bits where bf16 has eight.
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
// half-precision operands: formats 0; K-major A and B for S, MN-major B for P V
constexpr uint32_t kIdescS16 = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
constexpr uint32_t kIdescPV16 = (1u << 4) | (1u << 16) | ((64u >> 3) << 17) | ((128u >> 4) << 24);

// Warpgroups: two softmax per query tile, one of producer and MMA warps, one dequantising.
template <int QT>
constexpr int kFp4Threads = 256 * QT + 256;
// Two tiles: 768 threads start with 80 registers each; 512 * 96 + 128 * 40 + 128 * 56 = 61440 = 768 * 80.
constexpr int kFp4SoftmaxRegs = 96, kFp4ControlRegs = 40, kFp4UnpackRegs = 56;
static_assert(512 * kFp4SoftmaxRegs + 128 * kFp4ControlRegs + 128 * kFp4UnpackRegs <= 768 * 80, "register pool of the CTA exceeded");

template <int QT>
struct Fp4Smem {
  static constexpr uint32_t q_off = 0;
  static constexpr uint32_t tile_off = q_off + QT * kTileBytes;
  static constexpr uint32_t packed_off = tile_off + kTileStages * 2 * kTileBytes;
  static constexpr uint32_t pair_off = packed_off + kPackedStages * 2 * kPackedBytes;      // [2][QT][2][128] floats, as in gct_attn_kernel
  static constexpr uint32_t factor_off = pair_off + 2 * QT * 2 * 128 * 4;              // [QT][128] floats: a row's multiplier in front of exp2
  static constexpr uint32_t ref_off = factor_off + QT * 128 * 4;                       // [QT][128] floats: a row's fixed reference
  static constexpr uint32_t bar_off = ref_off + QT * 128 * 4;
  // q_full, q_ready, verdict, packed_full/empty[], K and V tile_full/empty[], per query tile s_full, s_empty, p_full[2], pv_full[2]
  static constexpr int n_bars = 3 + 2 * kPackedStages + 4 * kTileStages + 6 * QT;
  static constexpr uint32_t misc_off = bar_off + n_bars * 8;
  static constexpr uint32_t total = misc_off + 16;
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

template <int QT>
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
      mbar_init(bar_packed_empty(s), 4);
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

  // Where a role is in its range: the page, the block in it and how many blocks of the page are left, this one included.
  struct Place {
    int page, block, left;
  };
  auto blocks_of = [&](int page) { return page == a.n_pages - 1 ? a.total_blocks - page * a.blocks_per_page : a.blocks_per_page; };
  auto first_place = [&]() -> Place {
    const int page = g0 / a.blocks_per_page, block = g0 - page * a.blocks_per_page;
    return {page, block, blocks_of(page) - block};
  };
  auto advance = [&](Place& p) {
    ++p.block;
    if (--p.left == 0) p = {p.page + 1, 0, blocks_of(p.page + 1)};
  };
  // rows that block `block` of a page holds in memory, and those of it that are valid
  auto rows_of = [&](const Place& p) { return p.block < a.full_blocks ? kFp4Rows : a.tail_rows; };
  auto valid_of = [&](const Place& p) { return p.left > 1 ? kFp4Rows : (p.page == a.n_pages - 1 ? a.last_page_len : a.page_len) - p.block * kFp4Rows; };

  if (warp >= kFirstUnpackWarp) {
    // =========================== dequantising warps ===========================
    if constexpr (QT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFp4UnpackRegs));
    // A thread takes half rows (sixteen bytes, 32 values) of rows tid / 2 and 64 further on: loads are consecutive, and eight threads
    // store to four rows and both their halves, which the swizzle puts into eight different 16-byte columns.
    const int tid = threadIdx.x - 32 * kFirstUnpackWarp, row = tid >> 1;
    const uint32_t to0 = sbase + L::tile_off + row * 128 + ((((tid & 1) * 4) ^ (row & 7)) << 4);
    auto unpack = [&](const uint8_t* from, uint32_t to, int rows, int valid) {
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
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"((to ^ (e << 4)) + u * 8192), "r"(half2_mul(p[0], s)), "r"(half2_mul(p[1], s)),
                       "r"(half2_mul(p[2], s)), "r"(half2_mul(p[3], s))
                       : "memory");
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
    };
    auto wait = [&](uint32_t bar, uint32_t parity) -> bool { return __all_sync(0xffffffffu, mbar_wait(bar, parity, cta_abort, a.status)); };
    Place at = first_place();
    for (int j = 0, end = nblk; j < end; ++j) {
      const int ps = j % kPackedStages, ts = j % kTileStages, rows = rows_of(at), valid = valid_of(at);
      const uint8_t* from = smem + L::packed_off + ps * 2 * kPackedBytes;
      const uint32_t to = to0 + ts * 2 * kTileBytes, empty = ((j / kTileStages) & 1) ^ 1u;
      if (!wait(bar_packed_full(ps), (j / kPackedStages) & 1) || !wait(bar_tile_empty(ts, 0), empty)) break;
      unpack(from, to, rows, valid);
      if (lane == 0) mbar_arrive(bar_tile_full(ts, 0));
      if (!wait(bar_tile_empty(ts, 1), empty)) break;
      unpack(from + kPackedBytes, to + kTileBytes, rows, valid);
      if (lane == 0) {
        mbar_arrive(bar_tile_full(ts, 1));
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
      const uint8_t* base = nullptr;
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
          base = a.pool + (static_cast<int64_t>(page) * 2 * a.heads + h) * a.head_bytes;
        }
        const int ps = j % kPackedStages;
        if (!mbar_wait(bar_packed_empty(ps), ((j / kPackedStages) & 1) ^ 1u, cta_abort, a.status)) break;
        const uint32_t bytes = rows_of(at) * kFp4RowBytes<64>, to = sbase + L::packed_off + ps * 2 * kPackedBytes;
        const uint8_t* from = base + static_cast<int64_t>(at.block) * kPackedBytes;
        mbar_arrive_expect_tx(bar_packed_full(ps), 2 * bytes);
        bulk_load(to, from, bytes, bar_packed_full(ps));
        bulk_load(to + kPackedBytes, from + a.heads * a.head_bytes, bytes, bar_packed_full(ps));
        advance(at);
        if (j + 1 == nblk && again()) {
          end = 2 * nblk;
          at = first_place();
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
    float* factor = reinterpret_cast<float*>(smem + L::factor_off) + t * 128 + row;
    float* reference = reinterpret_cast<float*>(smem + L::ref_off) + t * 128 + row;
    if (half == 0) {
      ok = wait_v(bar_q_full(), 0);
      if (ok) {
        const uint32_t q_row = sbase + L::q_off + t * kTileBytes + row * 128;
        uint32_t w[32], top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[4 * j]), "=r"(w[4 * j + 1]), "=r"(w[4 * j + 2]), "=r"(w[4 * j + 3])
                       : "r"(q_row + ((static_cast<uint32_t>(j) ^ (row & 7)) << 4)));
#pragma unroll
          for (int i = 0; i < 4; ++i) top = max(top, max(w[4 * j + i] & 0x7fff0000u, (w[4 * j + i] & 0x7fffu) << 16));
        }
        // at most 2^126; 1 for a row of zeros or with a value that is not finite
        const int up = top == 0 || top >= 0x7f800000u ? 0 : min(14 + 127 - static_cast<int>(top >> 23), 126);
        const float f = __uint_as_float(static_cast<uint32_t>(127 + up) << 23), c = a.scale_log2 / f;
        *factor = c;
        float sq = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            w[4 * j + i] = pack_f16x2(__uint_as_float(w[4 * j + i] << 16) * f, __uint_as_float(w[4 * j + i] & 0xffff0000u) * f);
            const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w[4 * j + i]));
            sq = fmaf(x.x, x.x, fmaf(x.y, x.y, sq));
          }
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(q_row + ((static_cast<uint32_t>(j) ^ (row & 7)) << 4)), "r"(w[4 * j]),
                       "r"(w[4 * j + 1]), "r"(w[4 * j + 2]), "r"(w[4 * j + 3])
                       : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        if (a.key_norm_max != nullptr) {
          const float ref = sqrtf(sq) * __ldg(a.key_norm_max + h) * c;
          *reference = ref;
          if (!(ref <= a.fixed_limit)) *cta_exact = 1;     // too loose, infinite or NaN
        }
      }
    }
    auto softmax_sync = [&]() { asm volatile("bar.sync 15, %0;" ::"n"(256 * QT) : "memory"); };      // all softmax threads, also after a failed wait
    softmax_sync();
    const bool fixed = *cta_exact == 0;
    if (lane == 0) {
      if (half == 0 && ok) mbar_arrive(bar_q_ready());
      if (!fixed) mbar_arrive(bar_verdict());
    }
    const float c = *factor;
    float m = -INFINITY, l = 0.f;                          // m: reference maximum (units of S); l: sum over this half

    int pi, left;
    auto rewind = [&]() {
      pi = g0 / a.blocks_per_page;
      left = blocks_of(pi) - (g0 - pi * a.blocks_per_page);
    };
    auto tail_valid = [&]() -> int {
      const int valid = (pi == a.n_pages - 1 ? a.last_page_len : a.page_len) - (blocks_of(pi) - 1) * kBlockN - 64 * half;
      left = blocks_of(++pi);
      return valid;
    };
    // P = exp2(S c + shift) of 64 logits as half-precision pairs, and their sum, software-pipelined over pairs as in gct_attn_kernel.  kNum of
    // kDen pairs take the FMA pipe; kBelow: exponents may lie below -126.
    auto sweep = [&](uint32_t (&s)[64], uint32_t (&pk)[32], float shift, auto below, auto num, auto den) -> float {
      constexpr bool kBelow = decltype(below)::value;
      constexpr int kNum = decltype(num)::value, kDen = decltype(den)::value;
      const float2 c2 = make_float2(c, c), shift2 = make_float2(shift, shift);
      float2 acc0 = make_float2(0.f, 0.f), acc1 = make_float2(0.f, 0.f);
      auto pair_ffma = [&](int q) {
        const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[2 * q]), __uint_as_float(s[2 * q + 1])), c2, shift2);
        s[2 * q] = __float_as_uint(x.x);
        s[2 * q + 1] = __float_as_uint(x.y);
      };
      auto pair_exp = [&](int q) {
        if (((q + 1) * kNum) / kDen != (q * kNum) / kDen) {
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
      for (int q = 0; q < 32; ++q) {
        if (q + kFfmaAhead < 32) pair_ffma(q + kFfmaAhead);
        pair_exp(q);
        if (q >= kSumLag) pair_sum(q - kSumLag);
      }
#pragma unroll
      for (int q = 32 - kSumLag; q < 32; ++q) pair_sum(q);
      return (acc0.x + acc0.y) + (acc1.x + acc1.y);
    };
    using std::integral_constant;
    using Yes = std::true_type;
    using No = std::false_type;
    // S of block j in registers, the tile free for the next
    auto load_s = [&](int j, uint32_t (&s)[64]) -> bool {
      if (!wait_u(bar_s_full(t), j & 1)) return false;
      tc_fence_after();
      tmem_ld32(s_addr, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
      tmem_ld32(s_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(&s[32]));
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      mbar_arrive_elected(lead, bar_s_empty(t));
      return true;
    };
    auto store_p = [&](const uint32_t (&pk)[32]) {
      tmem_st32(p_addr, pk);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      mbar_arrive_elected(lead, bar_p_full(t, half));
    };
    auto mask = [&](uint32_t (&s)[64], int valid) {
#pragma unroll
      for (int i = 0; i < 64; ++i)
        if (i >= valid) s[i] = 0xff800000u;
    };

    // ---- fixed reference: |q| max|k| bounds every exponent of the row (Cauchy-Schwarz); no maximum, no exchange, no rescaling ----
    // Weights are exp2(x - ref + 15), at most 2^15.  Half precision holds them to 2^-25 at least, so over n keys at most n 2^-25 of the sum is lost
    // to rounding small ones; a row whose sum is at least n 2^-15 has lost less than 2^-10 of it.  A CTA with a row below that goes through its
    // range again with the running maximum.
    bool held = false;
    rewind();
    if (fixed) {
      const float shift = kFixedShift - *reference;
      int keys = nblk * kBlockN;
      for (int j = 0; ok && j < nblk; ++j) {
        uint32_t s[64], pk[32];
        if (!(ok = load_s(j, s))) break;
        int valid = 64;
        if (--left == 0) {
          valid = tail_valid();
          keys -= kBlockN - min(valid + 64 * half, kBlockN);
        }
        if (valid < 64) {
          mask(s, valid);
          l += sweep(s, pk, shift, Yes(), integral_constant<int, 0>(), integral_constant<int, 1>());
        } else {
          l += sweep(s, pk, shift, No(), integral_constant<int, 1>(), integral_constant<int, 4>());
        }
        if (j > 0) {
          if (!(ok = wait_u(bar_pv_full(t, half), (j - 1) & 1))) break;
          tc_fence_after();
        }
        store_p(pk);
      }
      __syncwarp();
      if (ok && nblk > 0) ok = wait_v(bar_pv_full(t, 1), (nblk - 1) & 1);
      const float other = pair_exchange(l, 0);
      l = half == 0 ? l + other : other + l;
      if (ok && !(l >= static_cast<float>(keys) * 0x1p-15f)) *cta_redo = 1;
      softmax_sync();
      held = *cta_redo == 0;
      if (lane == 0) mbar_arrive(bar_verdict());
      if (held) {
        m = *reference;
      } else {
        l = 0.f;
        rewind();
      }
    }
    // ---- running maximum ----
    if (!held) {
      const int first = fixed ? nblk : 0;
      int met = 0;
      for (int j = first; ok && j < first + nblk; ++j) {
        uint32_t s[64], pk[32];
        if (!(ok = load_s(j, s))) break;
        if (--left == 0) {
          const int valid = tail_valid();
          if (valid < 64) mask(s, valid);
        }
        float mxc[4];
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) mxc[ch] = __uint_as_float(s[ch]);
#pragma unroll
        for (int i = 4; i < 64; i += 2) mxc[(i >> 1) & 3] = max3(mxc[(i >> 1) & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
        float mx = fmaxf(fmaxf(mxc[0], mxc[1]), fmaxf(mxc[2], mxc[3]));
        mx = fmaxf(mx, pair_exchange(mx, ((met + 1) & 1) * kPairSlot));
        ++met;
        float alpha = 1.f;
        if ((mx - m) * c > kRescaleThreshold) {            // always true on the first block (m = -inf)
          alpha = fast_exp2((m - mx) * c);
          m = mx;
        }
        const float sum = sweep(s, pk, kFp4Shift - m * c, Yes(), integral_constant<int, QT == 2 ? 2 : 1>(), integral_constant<int, QT == 2 ? 7 : 3>());
        l = fmaf(l, alpha, sum);
        if (j > first) {
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
        store_p(pk);
      }
      __syncwarp();
      for (; met < nblk; ++met) pair_sync();
      if (ok && nblk > 0) ok = wait_v(bar_pv_full(t, 1), (first + nblk - 1) & 1);
      const float other = pair_exchange(l, ((nblk + 1) & 1) * kPairSlot);
      l = half == 0 ? l + other : other + l;
      m = m * c + (kFixedShift - kFp4Shift);               // as below: the exponent that weighs 2^kFixedShift
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
  GCT_CUDA_CHECK(cudaFuncSetAttribute(gct_attn_fp4_kernel<1>, cudaFuncAttributeMaxDynamicSharedMemorySize, Fp4Smem<1>::total + 1024));
  GCT_CUDA_CHECK(cudaFuncSetAttribute(gct_attn_fp4_kernel<2>, cudaFuncAttributeMaxDynamicSharedMemorySize, Fp4Smem<2>::total + 1024));
  // setmaxnreg hands out no more registers than the CTA was launched with and waits for ever for the rest: never launch such a build
  cudaFuncAttributes attr;
  GCT_CUDA_CHECK(cudaFuncGetAttributes(&attr, gct_attn_fp4_kernel<2>));
  if (attr.numRegs * kFp4Threads<2> < 512 * kFp4SoftmaxRegs + 128 * kFp4ControlRegs + 128 * kFp4UnpackRegs)
    return fail(GCT_ERR_INVALID, "attention: the kernel was built with fewer registers than its warpgroups share");
  g_fp4_ready[dev] = true;
  return GCT_OK;
}

}  // namespace

int launch_attention_fp4(const AttnLaunch& a, const uint8_t* pool, const Fp4Layout& layout, int num_pages, const int32_t* page_ids, cudaStream_t stream) {
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
  if (a.q_tiles_per_cta == 2)
    GCT_CUDA_CHECK(launch_pdl(gct_attn_fp4_kernel<2>, g, dim3(kFp4Threads<2>), Fp4Smem<2>::total + 1024, stream, a.tm_q, k, pages));
  else
    GCT_CUDA_CHECK(launch_pdl(gct_attn_fp4_kernel<1>, g, dim3(kFp4Threads<1>), Fp4Smem<1>::total + 1024, stream, a.tm_q, k, pages));
  return GCT_OK;
}

}  // namespace gct
