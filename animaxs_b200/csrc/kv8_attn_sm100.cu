// kv8_attn_sm100.cu -- attention of many query rows over the 8-bit K/V cache:
// cross attention of an image's tokens to a cached context, prompt chunks.
//
// The mathematics is that of kv8_rows_sm100.cu (the blocks' scales folded into
// the exponent); the products run on the tensor cores with 128-row tcgen05
// tiles.  Those take fp16 operands from shared memory, so four warps turn each
// 64-key block from codes into the fp16 layout the MMAs read, exactly, as it
// arrives; two 128-row query tiles share every converted block.
//
// Rows: with a power-of-two group the rows of a kv head are its query tokens x
// the group's heads (row = token * group + head), so that short chunks fill a
// tile; otherwise every query head is on its own (24 heads x 512 queries on 4096
// keys, batch 2: 66.3 to 66.9 us with groups of 1, 2, 3 and 4).
//
// A work item is a pair of query tiles (A, B) of one (sequence, head line), dealt
// round-robin to one persistent CTA per SM; where the pairs alone would leave
// SMs idle, the keys are split over the CTAs (kv8_attn_plan) and kv8_join_kernel
// joins the parts in order.  Sixteen warps:
//   0-3, 4-7   softmax of tile A / B: thread t owns row t (= TMEM lane t)
//   8-11       conversion of each K and V block
//   12, 15     MMA issuers of tile A / B (12 owns TMEM); one warp for both spent
//              2300 cycles a block on its waits, commits and issues
//   13         TMA producer: Q tiles; code blocks K_0, V_0, K_1, V_1, ... into a 2-slot ring
//   14         scheduler: works out the CTA's next items ahead of the other roles
//              (divisions and the length's load, 2000 cycles when every role did it)
// TMEM (512 columns): scores of tile A in two buffers of 64 columns, [0,64) and
// [64,128), of tile B in [128,192) and [192,256), O_A [256,..), O_B.  P (fp16)
// overlays the first half of the scores it came from.  With two buffers the
// scores of block b + 1 are there when the softmax of block b ends; with one
// buffer of 128 keys each softmax waited 1200 of its 4300 cycles for
// PV(j) and QK(j + 1).  O is rescaled only when a row's maximum grows by more
// than 2^8.
//
// Measured (GPU time of a call in a graph): 4096 queries x 16 heads on up to 512
// keys, batch 8 (int8) 104 us; 512 queries x 16 heads on 8704 keys, batch 2 (e4m3,
// causal) 76.6 us = 923 TFLOP/s, 0.55 of the measured bf16 peak.  No unit is full:
// tensor pipe 34 % of active cycles, exp2 35 %, ALU 37 %, shared memory 26 %, DRAM
// 24 %; half the QK MMAs gained 4 %, no exp2 5 %, no conversion stores 1 %.  Of 2060
// cycles a block (clocks in the kernel) a softmax warp works 1840 (maximum 430,
// exponentials and P 1130: two tiles share the exp2 unit, 1024), an MMA warp 1425
// (QK at N = 64 reads 6 KB of shared memory per 32 cycles of MMA).
// Slower, each measured: 128-key blocks (128 us for the first), a maximum taken a
// block ahead (141), exponentials before the maximum is known (115), an epilogue
// warpgroup of its own (111), e4m3 conversion on the ALU (95 against 83 then).
//
// Every wait is bounded; a timeout raises the CTA's abort flag and the status
// bit, and the CTA drains and exits.
#include <atomic>

#include "api_internal.h"
#include "flash_common.cuh"
#include "kernels.h"
#include "kv8_common.cuh"

namespace ax {
namespace {

constexpr int kThreads = 512;
constexpr int kRaw = 2;     // code slots
constexpr uint32_t kBarBytes = 768;
constexpr int kKStages = 4, kVStages = 3;  // fp16 blocks
constexpr int kBlk = kKv8Block;
constexpr int kItems = 2;  // items worked out ahead
constexpr int kItemReaders = 15;
template <int HD>
struct Smem {
  static constexpr uint32_t kTile = kTileM * HD * 2;  // fp16 query tile
  static constexpr uint32_t kKv = kBlk * HD * 2;      // fp16 K or V block
  static constexpr uint32_t kCodes = kBlk * HD;       // its codes
  static constexpr uint32_t kQ = 0;                      // Q_A, Q_B
  static constexpr uint32_t kK = kQ + 2 * kTile;
  static constexpr uint32_t kV = kK + kKStages * kKv;
  static constexpr uint32_t kRing = kV + kVStages * kKv;
  // Output stage: per softmax warp, 32 rows x 64 columns fp16.
  static constexpr uint32_t kStage = kRing + kRaw * kCodes;
  static constexpr uint32_t kBar = kStage + 8 * 4096;
  static constexpr uint32_t kBytes = kBar + kBarBytes + 1024;  // + alignment slack
};
static_assert(Smem<128>::kBytes <= 227 * 1024, "shared memory exceeds the 227 KiB opt-in");

enum : int {
  kBarQ = 0,
  kBarRawFull,                             // +slot
  kBarRawEmpty = kBarRawFull + kRaw,       // +slot (4 warp arrivals)
  kBarKFull = kBarRawEmpty + kRaw,         // +stage (4 warp arrivals)
  kBarVFull = kBarKFull + kKStages,        // +stage (4 warp arrivals)
  kBarVEmpty = kBarVFull + kVStages,       // +stage (2: tile A, tile B): the block's PVs have retired
  kBarSFull = kBarVEmpty + kVStages,       // +2*tile + buffer
  kBarPFull = kBarSFull + 4,               // +2*tile + buffer (4 warp arrivals)
  kBarODone = kBarPFull + 4,               // +tile
  kBarQFree = kBarODone + 2,               // (2: tile A, tile B)
  kBarItemFull,                            // +entry
  kBarItemEmpty = kBarItemFull + kItems,   // +entry (15 arrivals: every consuming warp)
  kBarDone = kBarItemEmpty + kItems,       // +tile
  kNumBars = kBarDone + 2
};
constexpr uint32_t kSlotTmem = kNumBars * 8;
constexpr uint32_t kSlotAbort = kSlotTmem + 4;
// Per key block: factor of the scores, log2 scale_v, 1 / scale_v (float4, eight
// blocks deep: K block g is converted after PV(g - 4) retired, which follows
// the softmax's use of block g - 4).
constexpr int kScales = 8;
constexpr uint32_t kSlotScale = 320;
constexpr uint32_t kSlotItem = kSlotScale + kScales * 16;  // Item [kItems]
static_assert(kSlotAbort + 4 <= kSlotScale && kSlotItem + kItems * 48 <= kBarBytes, "barrier block overflows");
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColO = 256;

// Register split (setmaxnreg) of the 512 x 128 registers of the launch: softmax
// 2 x 128 threads, conversion 128, MMA / TMA 128 (build.py checks the sum).
#define AX_KV8_SOFTMAX_REGS 176
#define AX_KV8_CONVERT_REGS 80
#define AX_KV8_OTHER_REGS 80

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const void* tmap, uint32_t bar, int c0, int c1, int c2,
                                            int c3, int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
      "l"(tmap), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
      : "memory");
}

// K-major operand of 64-column SW128 panels of `rows` rows; k-step kk = 16 columns.
template <int ROWS>
__device__ __forceinline__ uint64_t panel_off(int kk) {
  return static_cast<uint64_t>(((kk >> 2) * ROWS * 128 + (kk & 3) * 32) >> 4);
}
constexpr uint32_t kIdescQK = idesc_f16_f32(kTileM, kBlk, false);  // B = K block, K-major
template <int HD>
constexpr uint32_t kIdescPV = idesc_f16_f32(kTileM, HD, true);     // B = V block, MN-major

template <int HD>
__device__ __forceinline__ void issue_qk64(uint32_t d_tmem, uint32_t q_tile, uint32_t k_block) {
  const uint64_t a = sw128_desc(q_tile, 16, 1024), b = sw128_desc(k_block, 16, 1024);
#pragma unroll
  for (int kk = 0; kk < HD / 16; ++kk)
    umma_f16_ss_warp(d_tmem, a + panel_off<kTileM>(kk), b + panel_off<kBlk>(kk), kIdescQK, kk > 0 ? 1u : 0u);
}
// O (+)= P V over the block's 64 keys: k-step kk covers keys [16kk, 16kk+16) =
// 2 groups of 8 rows (1024 B apart); the 64-wide head_dim panels are 8 KiB apart.
template <int HD>
__device__ __forceinline__ void issue_pv64(uint32_t d_tmem, uint32_t p_tmem, uint32_t v_block, bool accumulate) {
  const uint64_t b = sw128_desc(v_block, kBlk * 128, 1024);
#pragma unroll
  for (int kk = 0; kk < kBlk / 16; ++kk)
    umma_f16_ts_warp(d_tmem, p_tmem + kk * 8, b + static_cast<uint64_t>((kk * 2048) >> 4), kIdescPV<HD>,
                     accumulate || kk > 0 ? 1u : 0u);
}

// Place in a ring: stage, and parity of the phase its use completes.
template <int N>
struct Ring {
  uint32_t stage = 0, phase = 0;
  __device__ __forceinline__ void next() {
    if (++stage == N) {
      stage = 0;
      phase ^= 1u;
    }
  }
};

__device__ __forceinline__ void tma_store_5d(const void* tmap, uint32_t src, int c0, int c1, int c2, int c3, int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5, %6}], [%1];" ::"l"(tmap),
      "r"(src), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
      : "memory");
}

struct alignas(16) Item {
  int q0, h, b, kvh;
  int len;
  int j0;          // first key block
  int nA, nB, n;   // key blocks of A, of B, of the item
  int w;           // its number, -1 past the last one
  int pad[2];
};
static_assert(sizeof(Item) == 48, "items are read as three 16-byte words");

// Split keys, by parts: p.parts CTAs to each unit (pair of tiles).  By shares
// (parts 0): the blocks of all units, p.blocks each as if none were shorter, in a
// row; CTA c takes [share_begin(c), share_begin(c + 1)), which is less than a
// unit and so touches at most two.
__device__ __forceinline__ int share_begin(const Kv8AttnParams& p, int c) { return c * p.each + min(c, p.more); }
__device__ __forceinline__ int share_owner(const Kv8AttnParams& p, int v) {
  const int big = p.more * (p.each + 1);
  return v < big ? v / (p.each + 1) : p.more + (v - big) / p.each;
}

// The part [lo, hi) of p.blocks of unit w; `part` is where its partial result goes.
__device__ __forceinline__ Item kv8_item(const Kv8AttnParams& p, int w, int lo, int hi, int part) {
  Item it;
  it.w = part;
  const int pair = p.causal ? p.pairs - 1 - w % p.pairs : w % p.pairs;  // the longest first
  w /= p.pairs;
  it.h = w % p.lines;
  it.b = w / p.lines;
  it.kvh = p.pack == p.group ? it.h : it.h / p.group;
  it.q0 = pair * 2 * kTileM;
  it.len = kv8_len(p.lens, p.kv_valid, p.kv_len, it.b);
  auto blocks = [&](int r0) {
    if (r0 >= p.rows) return 0;
    int e = it.len;
    if (p.causal) e = min(e, max(it.len - p.q_len + min(r0 + kTileM - 1, p.rows - 1) / p.pack + 1, 0));
    return (e + kBlk - 1) / kBlk;
  };
  const int a = blocks(it.q0), b = blocks(it.q0 + kTileM);
  const int n = max(a, b);
  // A shorter unit is cut in the same proportions.
  const bool all = n == p.blocks || (lo == 0 && hi == p.blocks);
  it.j0 = all ? lo : static_cast<int>(static_cast<long long>(n) * lo / p.blocks);
  const int j1 = all ? min(hi, n) : static_cast<int>(static_cast<long long>(n) * hi / p.blocks);
  it.nA = max(min(a, j1) - it.j0, 0);
  it.nB = max(min(b, j1) - it.j0, 0);
  it.n = j1 - it.j0;
  return it;
}


template <int FMT, int HD>
__global__ void __launch_bounds__(kThreads, 1)
    kv8_attn_sm100_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                          const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o,
                          const Kv8AttnParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  using L = Smem<HD>;
  const uint32_t sQ = base + L::kQ, sK = base + L::kK, sV = base + L::kV, sR = base + L::kRing;
  const uint32_t bar0 = base + L::kBar;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gbase + L::kBar + kSlotTmem);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + L::kBar + kSlotAbort);
#define BAR(i) (bar0 + 8u * static_cast<uint32_t>(i))
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int w0 = static_cast<int>(blockIdx.x);
  const int wstep = static_cast<int>(gridDim.x);

  if (threadIdx.x == 0) {
    for (int i = 0; i < kNumBars; ++i) {
      uint32_t count = 1;
      if (i >= kBarRawEmpty && i < kBarRawEmpty + kRaw) count = 4;
      if (i >= kBarKFull && i < kBarKFull + kKStages) count = 4;
      if (i >= kBarVFull && i < kBarVFull + kVStages) count = 4;
      if (i >= kBarVEmpty && i < kBarVEmpty + kVStages) count = 2;
      if (i == kBarQFree) count = 2;
      if (i >= kBarPFull && i < kBarPFull + 4) count = 4;
      if (i >= kBarItemEmpty && i < kBarItemEmpty + kItems) count = kItemReaders;
      mbar_init(BAR(i), count);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 12) {
    tmem_alloc(bar0 + kSlotTmem, kTmemCols);
    tmem_relinquish();
  }
  if (warp == 13 && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    tma_prefetch_desc(&tm_o);
  }
  pdl_wait();  // (its successor is not started early: that cost 4 % of a full launch)
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // The CTA's next item (every consuming warp calls it once per item, converged
  // or, for the producer, from its one active lane); w is -1 past the last one.
  uint32_t items_read = 0;
  auto next_item = [&](bool one_lane, bool& ok) {
    const uint32_t e = items_read % kItems, ph = (items_read / kItems) & 1u;
    ++items_read;
    Item I;
    I.w = -1;
    ok = one_lane ? mbar_wait(BAR(kBarItemFull + e), ph, abort_flag, p.status)
                  : mbar_wait_warp(BAR(kBarItemFull + e), ph, abort_flag, p.status);
    if (!ok) return I;
    const uint32_t at = base + L::kBar + kSlotItem + e * sizeof(Item);
    const uint4 a = ld_shared_v4u(at), b = ld_shared_v4u(at + 16), c = ld_shared_v4u(at + 32);
    I.q0 = a.x, I.h = a.y, I.b = a.z, I.kvh = a.w;
    I.len = b.x, I.j0 = b.y, I.nA = b.z, I.nB = b.w;
    I.n = c.x, I.w = c.y;
    if (!one_lane) __syncwarp();
    if (one_lane || lane == 0) mbar_arrive(BAR(kBarItemEmpty + e));
    return I;
  };

  if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(AX_KV8_OTHER_REGS));
    if (warp == 13) {
      // ---------------------------------------------------------- producer --
      if (lane == 0) {
        int armed_q = 0, armed[kRaw] = {};
        uint32_t g = 0;  // code blocks loaded so far
        auto load = [&](const CUtensorMap* tm, int row0, int head) -> bool {
          const uint32_t slot = g % kRaw;
          if (!mbar_wait(BAR(kBarRawEmpty + slot), ((g / kRaw) & 1u) ^ 1u, abort_flag, p.status)) return false;
          mbar_arrive_expect_tx(BAR(kBarRawFull + slot), L::kCodes);
          tma_load_3d(sR + slot * L::kCodes, tm, BAR(kBarRawFull + slot), 0, row0, head);
          ++armed[slot];
          ++g;
          return true;
        };
        bool ok = true;
        int it = 0;
        while (true) {
          const Item I = next_item(true, ok);
          if (!ok || I.w < 0) break;
          if (I.n == 0) continue;
          const int head = I.b * p.kv_heads + I.kvh;
          // The first K and V block before Q, whose buffer is still in use: they
          // are converted while the previous item drains.
          if (!(ok = load(&tm_k, I.j0 * kBlk, head))) break;
          if (!(ok = load(&tm_v, I.j0 * kBlk, head))) break;
          if (it > 0 && !(ok = mbar_wait(BAR(kBarQFree), static_cast<uint32_t>((it - 1) & 1), abort_flag, p.status)))
            break;
          const int first = I.nA > 0 ? 0 : 1, last = I.nB > 0 ? 1 : 0;
          mbar_arrive_expect_tx(BAR(kBarQ), (last - first + 1) * L::kTile);
          for (int x = first; x <= last; ++x)
#pragma unroll
            for (int c = 0; c < HD / 64; ++c)
              tma_load_5d(sQ + x * L::kTile + c * kPanelBytes, &tm_q, BAR(kBarQ), 64 * c, 0,
                          (I.q0 + x * kTileM) / p.pack, I.h, p.q_batch != 0 ? I.b : 0);
          ++armed_q;
          ++it;
          for (int j = 1; ok && j < I.n; ++j) {
            if (!(ok = load(&tm_k, (I.j0 + j) * kBlk, head))) break;
            ok = load(&tm_v, (I.j0 + j) * kBlk, head);
          }
          if (!ok) break;
        }
        // Never leave the CTA with a tensor copy still landing in shared memory.
        if (armed_q) mbar_wait_drain(BAR(kBarQ), (armed_q - 1) & 1);
        for (int s = 0; s < kRaw; ++s)
          if (armed[s]) mbar_wait_drain(BAR(kBarRawFull + s), (armed[s] - 1) & 1);
      }
    } else if (warp == 12 || warp == 15) {
      // --------------------------------------------------------------- MMA --
      // One warp per query tile; both count every block of an item in and out,
      // so that a stage is free when both are past it.
      const int X = warp == 12 ? 0 : 1;
      const uint32_t tS = tmem + X * 128, tO = tmem + kColO + X * HD, q_tile = sQ + X * L::kTile;
      Ring<kKStages> gk;  // the next K block
      Ring<kVStages> gv;  // the next V block
      uint32_t tX = 0;    // blocks of this tile in earlier items
      bool ok = true;
      uint32_t it = 0;
      // QK of the tile's block number t (a running count) into score buffer t % 2.
      auto qk = [&](uint32_t t) -> bool {
        if (!mbar_wait_warp(BAR(kBarKFull + gk.stage), gk.phase, abort_flag, p.status)) return false;
        tc_fence_after();
        issue_qk64<HD>(tS + (t & 1u) * 64, q_tile, sK + gk.stage * L::kKv);
        tc_commit_warp(BAR(kBarSFull + 2 * X + (t & 1u)));
        gk.next();
        return true;
      };
      while (true) {
        const Item I = next_item(false, ok);
        if (!ok || I.w < 0) break;
        const int n = I.n, nX = X ? I.nB : I.nA;
        if (n == 0) continue;
        if (!(ok = mbar_wait_warp(BAR(kBarQ), it & 1u, abort_flag, p.status))) break;
        ++it;
        for (int j = 0; ok && j < 2 && j < nX; ++j) ok = qk(tX + j);
        if (!ok) break;
        if (nX > 0 && nX <= 2) tc_commit_warp(BAR(kBarQFree));  // the tile's last QK
        for (int j = 0; j < nX; ++j) {
          // V block j was converted before K block j + 1, which this warp has
          // waited for already, unless j is the last.
          if (j == nX - 1 && !(ok = mbar_wait_warp(BAR(kBarVFull + gv.stage), gv.phase, abort_flag, p.status))) break;
          const uint32_t t = tX + j;
          // An item's first P is published after the previous epilogue has read O.
          if (!(ok = mbar_wait_warp(BAR(kBarPFull + 2 * X + (t & 1u)), (t >> 1) & 1u, abort_flag, p.status))) break;
          tc_fence_after();
          issue_pv64<HD>(tO, tS + (t & 1u) * 64, sV + gv.stage * L::kKv, j > 0);
          if (j == nX - 1) tc_commit_warp(BAR(kBarODone + X));
          tc_commit_warp(BAR(kBarVEmpty + gv.stage));
          gv.next();
          // A buffer's next scores follow the PV that reads its P (same thread, issue order).
          if (j + 2 < nX) {
            if (!(ok = qk(t + 2))) break;
            if (j + 2 == nX - 1) tc_commit_warp(BAR(kBarQFree));
          }
        }
        if (!ok) break;
        tX += nX;
        if (nX == 0 && lane == 0) mbar_arrive(BAR(kBarQFree));
        // Blocks that only the other tile reads: past them once they are there
        // (an earlier arrival could count for the stage's previous use).
        for (int j = nX; j < n; ++j) {
          if (!(ok = mbar_wait_warp(BAR(kBarVFull + gv.stage), gv.phase, abort_flag, p.status))) break;
          if (lane == 0) mbar_arrive(BAR(kBarVEmpty + gv.stage));
          gk.next();
          gv.next();
        }
        if (!ok) break;
      }
      // All MMAs this warp issued must retire before TMEM is released.
      tc_commit_warp(BAR(kBarDone + X));
      mbar_wait_drain(BAR(kBarDone + X), 0);
      __syncwarp();
    } else if (warp == 14) {
      // --------------------------------------------------------- scheduler --
      if (lane == 0) {
        // Whole units round-robin, or a part of one, or a share's parts of one or two.
        int v = 0, end = 0, w = w0;
        if (p.split && p.parts > 0) {
          w = w0 / p.parts;
          const int k = w0 - w * p.parts;
          v = w * p.blocks + p.blocks * k / p.parts;
          end = w * p.blocks + p.blocks * (k + 1) / p.parts;
        } else if (p.split) {
          v = share_begin(p, w0);
          end = share_begin(p, w0 + 1);
          w = v / p.blocks;
        }
        for (uint32_t i = 0;; ++i) {
          const bool last = p.split ? v >= end : w >= p.n_items;
          Item I;
          if (!last) {
            const int lo = p.split ? v - w * p.blocks : 0, hi = p.split ? min(lo + end - v, p.blocks) : p.blocks;
            I = kv8_item(p, w, lo, hi, 2 * w0 + static_cast<int>(i));
            v += hi - lo;
            w += p.split ? 1 : wstep;
          } else
            I.q0 = I.h = I.b = I.kvh = I.len = I.j0 = I.nA = I.nB = I.n = 0, I.w = -1;
          const uint32_t e = i % kItems;
          if (!mbar_wait(BAR(kBarItemEmpty + e), ((i / kItems) & 1u) ^ 1u, abort_flag, p.status)) break;
          const uint32_t at = base + L::kBar + kSlotItem + e * sizeof(Item);
          st_shared_v4(at, I.q0, I.h, I.b, I.kvh);
          st_shared_v4(at + 16, I.len, I.j0, I.nA, I.nB);
          st_shared_v4(at + 32, I.n, I.w, 0, 0);
          mbar_arrive(BAR(kBarItemFull + e));
          if (last) break;
        }
      }
    }
  } else if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(AX_KV8_CONVERT_REGS));
    // ---------------------------------------------------------- conversion --
    // Thread t turns half a row (key t % 64, its half t / 64) of each block:
    // 16-byte runs of 16 codes become two 16-byte units of the 64-column SW128
    // panels.  Eight lanes that share a phase hold eight consecutive rows, so
    // loads and stores meet no bank twice.
    const int t = threadIdx.x - 256;
    const int key = t & 63, part = t >> 6;
    uint32_t g = 0;  // code blocks taken so far: K and V alternate
    Ring<kKStages> rk;
    Ring<kVStages> rv;
    bool ok = true;
    float nk = 0.f, nv = 0.f;  // scales of the next K block
    float sv = 0.f;            // scale of the next V block
    auto scales = [&](const Item& I, int j) {
      const long long at = (static_cast<long long>(I.b) * p.kv_heads + I.kvh) * p.n_blocks + I.j0 + j;
      nk = p.k_scale[at];
      nv = p.v_scale[at];
    };
    while (true) {
      const Item I = next_item(false, ok);
      if (!ok || I.w < 0) break;
      if (I.n > 0) scales(I, 0);
      for (int jj = 0; ok && jj < 2 * I.n; ++jj, ++g) {
        const bool is_v = (g & 1u) != 0;
        const uint32_t slot = g % kRaw;
        ok = mbar_wait_warp(BAR(kBarRawFull + slot), (g / kRaw) & 1u, abort_flag, p.status);
        if (!ok) break;
        const uint32_t src = sR + slot * L::kCodes + key * HD;
        uint4 c[HD / 32];
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) {
          const int run = part * (HD / 32) + i;
          c[i] = ld_shared_v4u(src + (HD == 128 ? run ^ (key & 7) : run ^ ((key >> 1) & 3)) * 16);
        }
        // The slot's next tensor copy must not overtake these reads.
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(BAR(kBarRawEmpty + slot));
        // What lies past the length may decode to NaN: such keys become zeros.  So do
        // the codes of a block whose factor is 0 (a scale of 0, or one whose product
        // with the softmax scale underflows): its scores, or values, are 0.
        const float factor = is_v ? (sv > kKv8NoValue ? sv : 0.f) : nk * p.scale_log2;
        if ((I.j0 + (jj >> 1)) * kBlk + key >= I.len || !(factor > 0.f)) {
#pragma unroll
          for (int i = 0; i < HD / 32; ++i) c[i] = make_uint4(0u, 0u, 0u, 0u);
        }
        // K block g takes the stage of K block g - 4, whose QKs retired before the
        // PVs of block g - 4, which V block g - 1 has waited for.
        if (is_v) ok = mbar_wait_warp(BAR(kBarVEmpty + rv.stage), rv.phase ^ 1u, abort_flag, p.status);
        if (!ok) break;
        const uint32_t dst = (is_v ? sV + rv.stage * L::kKv : sK + rk.stage * L::kKv) + key * 128;
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) {
          uint32_t h[8];
          kv8_to_half2<FMT>(c[i].x, h[0], h[1]);
          kv8_to_half2<FMT>(c[i].y, h[2], h[3]);
          kv8_to_half2<FMT>(c[i].z, h[4], h[5]);
          kv8_to_half2<FMT>(c[i].w, h[6], h[7]);
          const int run = part * (HD / 32) + i;
          const uint32_t at = dst + (run >> 2) * (kBlk * 128);
          const int u = (run & 3) * 2;
          st_shared_v4(at + ((u ^ (key & 7)) << 4), h[0], h[1], h[2], h[3]);
          st_shared_v4(at + (((u + 1) ^ (key & 7)) << 4), h[4], h[5], h[6], h[7]);
        }
        if (!is_v) {
          // With 1 in place of a factor of 0 a masked -inf does not meet 0.
          if (t == 0)
            st_shared_v4(base + L::kBar + kSlotScale + ((g >> 1) % kScales) * 16,
                         __float_as_uint(factor > 0.f ? factor : 1.f),
                         __float_as_uint(nv > kKv8NoValue ? __log2f(nv) : kKv8NoScale),
                         __float_as_uint(nv > kKv8NoValue ? __fdividef(1.f, nv) : kKv8NoScaleInverse), 0u);
          sv = nv;
          if (jj + 2 < 2 * I.n) scales(I, (jj >> 1) + 1);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (is_v) {
          if (lane == 0) mbar_arrive(BAR(kBarVFull + rv.stage));
          rv.next();
        } else {
          if (lane == 0) mbar_arrive(BAR(kBarKFull + rk.stage));
          rk.next();
        }
      }
      if (!ok) break;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(AX_KV8_SOFTMAX_REGS));
    // ------------------------------------------------------------- softmax --
    const int X = warp >> 2;          // 0: tile A, 1: tile B
    const int t = threadIdx.x & 127;  // row within the tile == TMEM lane
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t o_addr = tmem + lane_base + kColO + X * HD;
    bool ok = true;
    uint32_t tX = 0;  // blocks of this query tile in earlier items
    uint32_t gt = 0;  // key blocks of earlier items
    uint32_t eX = 0;  // epilogues done in earlier items
    while (true) {
      const Item I = next_item(false, ok);
      if (!ok || I.w < 0) break;
      const int row = I.q0 + X * kTileM + t;
      const int nX = X ? I.nB : I.nA;
      const int tok = row >> p.pack_log2;
      const int lim = p.causal ? min(I.len, I.len - p.q_len + tok + 1) : I.len;  // keys visible to this row
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < nX; ++j) {
        const int key0 = (I.j0 + j) * kBlk;
        const uint32_t tt = tX + j, buf = tt & 1u;
        const uint32_t s_addr = tmem + lane_base + X * 128 + buf * 64;
        ok = mbar_wait(BAR(kBarSFull + 2 * X + buf), (tt >> 1) & 1u, abort_flag, p.status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        uint32_t s[2][32];
        tmem_ld32(s_addr, s[0]);
        tmem_ld32(s_addr + 32, s[1]);
        // Factor, log2 scale_v, 1 / scale_v of the block.
        const float4 fac = ld_shared_v4f(base + L::kBar + kSlotScale + ((gt + j) % kScales) * 16);
        tmem_ld_wait(s[0]);
        asm volatile("" : AX_RW32(s[1])::"memory");
        if (key0 + kBlk > lim) {
#pragma unroll
          for (int c = 0; c < kBlk; ++c)
            if (key0 + c >= lim) s[c >> 5][c & 31] = __float_as_uint(-INFINITY);
        }
        // Row maximum of s + log2 scale_v.
#define SV(c) __uint_as_float(s[(c) >> 5][(c) & 31])
        float mx[4];
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          mx[a] = fmax3(SV(a), SV(a + 4), SV(a + 8));
#pragma unroll
          for (int c = 12; c < 60; c += 8) mx[a] = fmax3(mx[a], SV(a + c), SV(a + c + 4));
          mx[a] = fmaxf(mx[a], SV(a + 60));
        }
#undef SV
        const float m_new = fmaxf(m, fmaf(fmaxf(fmax3(mx[0], mx[1], mx[2]), mx[3]), fac.x, fac.y));
        const bool grow = m_new > m + kRescaleThreshold;  // also true at the first block with a visible key
        const float alpha = grow ? ex2_approx(m - m_new) : 1.f;
        if (grow) {
          l *= alpha;
          m = m_new;
        }
        if (j > 0 && __any_sync(0xffffffffu, grow)) {
          // O must hold PV(0..j-1) and nothing more: V block j - 1 is released
          // when its PVs have retired, and PV_X(j) starts only after this warp's
          // arrival below, so the phase waited for cannot be passed.
          const uint32_t v = gt + j - 1;
          ok = mbar_wait(BAR(kBarVEmpty + v % kVStages), (v / kVStages) & 1u, abort_flag, p.status);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1  // unrolled, it spills
          for (int c4 = 0; c4 < HD / 32; ++c4) {
            uint32_t o[32];
            tmem_ld32(o_addr + c4 * 32, o);
            tmem_ld_wait(o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st32(o_addr + c4 * 32, o);
          }
        }
        const float off = fac.y - ((m == -INFINITY) ? 0.f : m);
        const float2 mulv = make_float2(fac.x, fac.x), offv = make_float2(off, off);
        float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        uint32_t pk[32];
#pragma unroll
        for (int c = 0; c < kBlk; c += 2) {
          const float2 x = fma2(make_float2(__uint_as_float(s[c >> 5][c & 31]),
                                            __uint_as_float(s[c >> 5][(c + 1) & 31])),
                                mulv, offv);
          const float2 pr = make_float2(ex2_approx(x.x), ex2_approx(x.y));
          acc[(c >> 1) & 1] = add2(acc[(c >> 1) & 1], pr);
          pk[c >> 1] = pack_half2(pr.x, pr.y);
        }
        tmem_st32(s_addr, pk);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(BAR(kBarPFull + 2 * X + buf));
        const float2 a = add2(acc[0], acc[1]);
        l = fmaf(a.x + a.y, fac.z, l);
      }
      if (!ok) break;
      if (nX > 0) {
        ok = mbar_wait(BAR(kBarODone + X), eX & 1u, abort_flag, p.status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        ++eX;
      }
      tX += nX;
      gt += I.n;
      // A row without a visible key has m = -inf and l = 0; one with NaN scores has l = NaN.
      const bool none = nX == 0 || (m == -INFINITY && l == l);
      if (p.split) {
        // [part][tile][HD / 4][128 rows] float4, then m and l of the rows.
        float* part = p.part + (2LL * I.w + X) * (kTileM * (HD + 2));
        const bool live = row < p.rows;
        if (live) {
          part[kTileM * HD + t] = none ? -INFINITY : m;
          part[kTileM * HD + kTileM + t] = none ? 0.f : l;
        }
        if (nX > 0) {
#pragma unroll 1
          for (int c4 = 0; c4 < HD / 32; ++c4) {
            uint32_t o[32];
            tmem_ld32(o_addr + c4 * 32, o);
            tmem_ld_wait(o);
            if (live) {
#pragma unroll
              for (int i = 0; i < 32; i += 4)
                reinterpret_cast<uint4*>(part)[(c4 * 8 + i / 4) * kTileM + t] =
                    make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
            }
          }
        }
      } else {
        // Each warp stages its 32 rows, 64 columns at a time, in the tensor-store
        // layout (16-byte unit u of row r at unit u ^ (r % 8)) and its lane 0
        // writes them with one TMA store; rows past the last are clipped.  (Plain
        // stores, even four lanes to a row, kept the load/store unit busy for
        // 2000 cycles an item.)
        const float inv_l = none ? 0.f : 1.f / l;
        const uint32_t wstage = base + L::kStage + static_cast<uint32_t>(warp) * 4096u;
        const uint32_t stage = wstage + lane * 128u;
        const int row0 = I.q0 + X * kTileM + (warp & 3) * 32;
#pragma unroll 1
        for (int rd = 0; rd < HD / 64; ++rd) {
          uint32_t o[2][32];
          tmem_ld32(o_addr + rd * 64, o[0]);  // stale where the item has no keys: replaced by zeros below
          tmem_ld32(o_addr + rd * 64 + 32, o[1]);
          tmem_ld_wait(o[0]);
          asm volatile("" : AX_RW32(o[1])::"memory");
          // The stage's previous store (last round or item) has been read.
          if (lane == 0) tma_store_wait_read();
          __syncwarp();
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const uint32_t* v = &o[u >> 2][(u & 3) * 8];
            uint32_t h[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              h[i] = pack_half2(__uint_as_float(v[2 * i]) * inv_l, __uint_as_float(v[2 * i + 1]) * inv_l);
              if (none) h[i] = 0u;
            }
            st_shared_v4(stage + ((u ^ (lane & 7)) << 4), h[0], h[1], h[2], h[3]);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && row0 < p.rows) {
            tma_store_5d(&tm_o, wstage, 64 * rd, row0 & (p.pack - 1), row0 >> p.pack_log2, I.h, I.b);
            tma_store_commit();
          }
        }
      }
      tc_fence_before();  // O has been read before the next item's first P is published
    }
  }

  if (warp < 8 && lane == 0) tma_store_wait_all();  // the output stores have completed
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
#undef BAR
}

// Joins the parts of every row in order: O = sum O'_s 2^(m_s - m) / sum l_s 2^(m_s - m).
// A thread takes 8 output values of a row; consecutive threads take consecutive rows.
template <int HD>
__global__ void __launch_bounds__(128) kv8_join_kernel(const Kv8AttnParams p) {
  pdl_start();
  pdl_wait();
  const int t = threadIdx.x;
  const int d8 = blockIdx.x % (HD / 8);
  int w = blockIdx.x / (HD / 8);  // (sequence, line, pair, tile)
  const int X = w & 1;
  w >>= 1;
  const int pair = w % p.pairs;
  const int row = pair * 2 * kTileM + X * kTileM + t;
  if (row >= p.rows) return;
  const int unit = w - pair + (p.causal ? p.pairs - 1 - pair : pair);  // as kv8_item numbers it
  const int h = w / p.pairs % p.lines, b = w / p.pairs / p.lines;
  float m = -INFINITY, l = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f), c = a;
  int first = unit * p.parts, n = p.parts;
  bool second = false;  // of its CTA's parts, as a unit's first may be
  if (n == 0) {
    first = share_owner(p, unit * p.blocks);
    n = share_owner(p, (unit + 1) * p.blocks - 1) - first + 1;
    second = share_begin(p, first) < unit * p.blocks;
  }
  constexpr int kJoin = 4;
  const float* part0 = p.part + (4LL * first + X) * (kTileM * (HD + 2));
#pragma unroll 1
  for (int s0 = 0; s0 < n; s0 += kJoin) {  // the loads of kJoin parts in flight
    float pm[kJoin], pl[kJoin];
    float4 x[kJoin], y[kJoin];
#pragma unroll
    for (int i = 0; i < kJoin; ++i) {
      const int s = s0 + i;
      pm[i] = -INFINITY;
      pl[i] = 0.f;
      if (s >= n) continue;
      const float* part = part0 + (4LL * s + (s == 0 && second ? 2 : 0)) * (kTileM * (HD + 2));
      pm[i] = part[kTileM * HD + t];
      pl[i] = part[kTileM * HD + kTileM + t];
      x[i] = reinterpret_cast<const float4*>(part)[(2 * d8) * kTileM + t];
      y[i] = reinterpret_cast<const float4*>(part)[(2 * d8 + 1) * kTileM + t];
    }
#pragma unroll
    for (int i = 0; i < kJoin; ++i) {
      const float mn = fmaxf(m, pm[i]);
      const float fo = m == mn ? 1.f : ex2_approx(m - mn);
      const float fn = pm[i] == mn ? 1.f : ex2_approx(pm[i] - mn);
      m = mn;
      l = l * fo + pl[i] * fn;
      if (pm[i] == -INFINITY && pl[i] == 0.f) continue;  // nothing stored (the first live part makes fo 0)
      a = make_float4(a.x * fo + x[i].x * fn, a.y * fo + x[i].y * fn, a.z * fo + x[i].z * fn, a.w * fo + x[i].w * fn);
      c = make_float4(c.x * fo + y[i].x * fn, c.y * fo + y[i].y * fn, c.z * fo + y[i].z * fn, c.w * fo + y[i].w * fn);
    }
  }
  const float inv = m == -INFINITY && l == l ? 0.f : 1.f / l;
  const int head = h * p.pack + row % p.pack;
  *reinterpret_cast<uint4*>(p.o + b * p.o_batch + static_cast<long long>(row / p.pack) * p.o_tok + head * p.o_head +
                            d8 * 8) =
      make_uint4(pack_half2(a.x * inv, a.y * inv), pack_half2(a.z * inv, a.w * inv),
                 pack_half2(c.x * inv, c.y * inv), pack_half2(c.z * inv, c.w * inv));
}

template <int FMT, int HD>
cudaError_t launch_hd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& to,
                      const Kv8AttnParams& p, int grid, int dev, cudaStream_t stream) {
  static std::atomic<uint64_t> configured{0};
  const uint64_t bit = 1ull << (dev & 63);
  auto kernel = kv8_attn_sm100_kernel<FMT, HD>;
  if ((configured.load(std::memory_order_acquire) & bit) == 0) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<HD>::kBytes);
    if (e != cudaSuccess) return e;
    configured.fetch_or(bit, std::memory_order_acq_rel);
  }
  cudaError_t e = launch_pdl(kernel, grid, kThreads, Smem<HD>::kBytes, stream, tq, tk, tv, to, p);
  if (e == cudaSuccess && p.split)
    e = launch_pdl(kv8_join_kernel<HD>, p.batch * p.lines * p.pairs * 2 * (HD / 8), 128, 0, stream, p);
  return e;
}

}  // namespace

// Fills in the rows, pairs and shares of a launch.  A pair of tiles over all its
// keys is one item when the pairs fill the SMs; otherwise the keys are cut into
// shares, whichever leaves the busiest SM the least to do: a whole number of
// CTAs to each pair, or equal shares over all SMs.  Each item's start and end
// counts as four key blocks' time.
bool kv8_attn_plan(Kv8AttnParams* p, int sms) {
  p->pack = kTileM % p->group == 0 ? p->group : 1;
  p->pack_log2 = 0;
  while ((1 << p->pack_log2) < p->pack) ++p->pack_log2;
  p->lines = p->kv_heads * p->group / p->pack;
  p->rows = p->q_len * p->pack;
  p->pairs = (p->rows + 2 * kTileM - 1) / (2 * kTileM);
  const long long pairs = static_cast<long long>(p->batch) * p->lines * p->pairs;
  const long long blocks = (p->kv_len + kBlk - 1) / kBlk;
  p->blocks = static_cast<int>(blocks);
  long long ctas = 0;  // 0: not split
  p->parts = 0;
  if (pairs < sms && blocks * sms <= 0x7fffffffLL) {
    long long best = blocks + 4;
    for (long long n = 2; n <= blocks && pairs * n <= sms; ++n) {
      const long long cost = (blocks + n - 1) / n + 4;
      if (cost < best) best = cost, ctas = pairs * n, p->parts = static_cast<int>(n);
    }
    if (pairs * blocks >= sms && (pairs * blocks + sms - 1) / sms + 8 < best) {
      ctas = sms;
      p->parts = 0;
    }
  }
  p->split = ctas != 0;
  p->each = p->split ? static_cast<int>(pairs * blocks / ctas) : 0;
  p->more = p->split ? static_cast<int>(pairs * blocks % ctas) : 0;
  if (pairs > 0x7fffffffLL / (2 * 16)) return false;
  p->n_items = static_cast<int>(pairs);
  p->grid = static_cast<int>(p->split ? ctas : pairs < sms ? pairs : sms);
  return true;
}
size_t kv8_attn_part_floats(int head_dim, int grid) {
  return 4 * static_cast<size_t>(grid) * kTileM * (head_dim + 2);
}

cudaError_t launch_kv8_attn(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                            const CUtensorMap& to, const Kv8AttnParams& p, int dev, cudaStream_t stream) {
  const int grid = p.grid;
  if (p.format == kKv8Int8)
    return p.head_dim == 128 ? launch_hd<kKv8Int8, 128>(tq, tk, tv, to, p, grid, dev, stream)
                             : launch_hd<kKv8Int8, 64>(tq, tk, tv, to, p, grid, dev, stream);
  return p.head_dim == 128 ? launch_hd<kKv8E4m3, 128>(tq, tk, tv, to, p, grid, dev, stream)
                           : launch_hd<kKv8E4m3, 64>(tq, tk, tv, to, p, grid, dev, stream);
}

}  // namespace ax
