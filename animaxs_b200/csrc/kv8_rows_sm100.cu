// kv8_rows_sm100.cu -- attention of a few query rows over the 8-bit K/V cache.
//
// A kv head's query rows (its query heads x the call's query tokens, up to 16)
// are taken together, so that each code is read and converted once for all of
// them.  With r rows the kernel does 4 r flops a code byte: HBM bounds it, and
// everything here serves to keep loads in flight and the conversion cheap.
//
// Mathematics, per 64-key block c (the tokens that share a scale): with
// acc = q . code_k,
//   s  = acc * (scale_k[c] * softmax scale * log2 e)
//   p' = 2^(s + log2 scale_v[c] - m'),  m' = running maximum of s + log2 scale_v
//   O' = sum p' code_v,   l = sum_c (1 / scale_v[c]) sum p',   O = O' / l,
// so the scales cost one multiply-add per score, which the softmax needs
// anyway, p' never exceeds 2^8 (see the lazy rescale below) whatever the
// scales, and the codes enter both products unscaled, exact as fp16.
//
// Work: every (sequence, kv head) is a line of 32-key tiles.  A warp takes a
// contiguous share of them and runs by itself: its lane 0 keeps a ring of tiles
// in flight by TMA, all lanes take a tile into registers, and no other warp is
// waited for until the share is done.  Shares are cut in one of two ways:
//  * a cluster of 1 to 8 CTAs to each line, where that leaves a warp few tiles.
//    The warps of a CTA join their parts in shared memory, the CTAs of the
//    cluster theirs in distributed shared memory;
//  * equal shares of all lines together, so that ragged lengths and single long
//    sequences load the SMs alike.  What crosses a CTA's share goes through a
//    workspace: each CTA stores its part (m', l, O') and counts itself in, and
//    the last one to arrive joins the parts.
// Parts are joined in warp and CTA order, so the result does not depend on the
// order of arrival.
//
// Measured (int8, group 2, head_dim 128; GPU time of a call in a graph): batch
// 1 x 8 kv heads, one query token on 300 keys 5.1 us (equal shares 8.0, of which
// 3 are the join through global memory), on 2048 keys 5.5 (8.5); a tile costs a
// warp 1.4 us when nothing is in flight before it, hence the bound on a
// cluster's shares.  One token on 131071 keys (e4m3) 52.2 us = 5.15 TB/s, 0.79 of the
// copy rate; the loop alone 0.91.  HBM bounds the loop; around it are 1 us of
// start, the SMs' spread (+-13 % with equal shares) and 3 us of join.
//
// Products: m16n8k16 mma.sync with the cache as the 16-wide operand and the
// query rows as the 8-wide one (one or two column tiles):
//   S^T [16 keys x 8 rows] = K Q^T,   O^T [16 d x 8 rows] += V^T P^T.
// A 128-row tcgen05 tile would be mostly empty at these row counts, and codes
// would have to pass through shared memory a second time.  Which codes of a
// row form an MMA's k index (K) or m index (V) is free as long as Q, or the
// stored O, follows: a lane takes 16-byte runs (32 codes of each of two K
// rows, 16 of each of four V rows), which TMA's swizzle spreads over the banks.
#include <atomic>

#include "api_internal.h"
#include "kernels.h"
#include "kv8_common.cuh"
#include "sm100_ptx.cuh"

namespace ax {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kTileKeys = 32;
constexpr int kAlone = 3;          // tiles of a warp up to which a line has a cluster of its own (kv8_rows_plan)
constexpr float kRescale = 8.f;    // log2 units by which the maximum may lag

// What a slot holds: the line's first tile (-1: nothing), sequence, kv head and tiles.
struct alignas(16) SlotInfo {
  int line, b, h, tiles;
};

// NT: column tiles of 8 query rows (1 or 2).
template <int HD, int NT>
struct RowsSmem {
  static constexpr int kRows = 8 * NT;
  static constexpr int kStages = NT == 1 ? 3 : 2;
  static constexpr uint32_t kCodes = kTileKeys * HD;              // codes of K (or V) of a tile
  static constexpr uint32_t kRing = kWarps * kStages * 2 * kCodes;
  static constexpr uint32_t kSlot = kRows * (HD + 2) * 4;         // O' [rows][HD], m' [rows], l [rows]
  static constexpr uint32_t kHead = kRing;                        // [warp] part of the share's first line
  static constexpr uint32_t kPrefix = kHead + kWarps * kSlot;     // int32 [kThreads + 1]
  static constexpr uint32_t kBar = (kPrefix + (kThreads + 1) * 4 + 15) / 16 * 16;
  static constexpr uint32_t kInfo = (kBar + kWarps * kStages * 8 + 15) / 16 * 16;  // SlotInfo [2 * warp]
  static constexpr uint32_t kBytes = kInfo + 2 * kWarps * 16 + 16 + 1024;  // + alignment slack
  // The part of a share's last line goes to the warp's own ring, which is idle by then.
  static_assert(kStages * 2 * kCodes >= kSlot, "a slot must fit a warp's ring");
  static_assert(kBytes <= 227 * 1024, "shared memory exceeds the 227 KiB opt-in");
};

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transpose of an 8 x 8 matrix of 16-bit values held one row per four lanes.
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ uint2 ld_shared_v2u(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_v4f(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster_v2f(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

// A place among the tiles: tile `tile` of `tiles` of kv head h of sequence b.
struct Place {
  int b, h, tile, tiles;
};

template <int FMT, int HD, int NT>
__global__ void __launch_bounds__(kThreads, 1)
    kv8_rows_sm100_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                          const Kv8AttnParams p) {
  extern __shared__ uint8_t smem_raw[];
  using L = RowsSmem<HD, NT>;
  constexpr int kStages = L::kStages;
  constexpr int kF4 = HD / 4;  // float4 units of a row
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  int* prefix = reinterpret_cast<int*>(gbase + L::kPrefix);
  SlotInfo* info = reinterpret_cast<SlotInfo*>(gbase + L::kInfo);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + L::kInfo + 2 * kWarps * 16);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t ring = base + warp * kStages * 2 * L::kCodes;
  const uint32_t bar = base + L::kBar + warp * kStages * 8;

  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(bar + 8 * i, 1);
    info[2 * warp].line = info[2 * warp + 1].line = -1;
    mbar_fence_init();
  }
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    prefix[0] = 0;
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  pdl_start();
  pdl_wait();
  const int lines = p.batch * p.kv_heads;
  int c0 = 0, c1 = 0;  // the CTA's tiles
  bool alone = p.alone;  // a cluster to each line, known before the lengths are
  const int rank = static_cast<int>(blockIdx.x) & ((1 << p.cluster_log2) - 1);  // in the cluster
  // prefix[t]: tiles of one line of the sequences before group t (kThreads
  // groups of `per` sequences).
  const int per = (p.batch + kThreads - 1) / kThreads;
  auto tiles_in = [&](int b) { return (kv8_len(p.lens, p.kv_valid, p.kv_len, b) + kTileKeys - 1) / kTileKeys; };
  int all = 0, longest = 0;
  if (!alone) {
    int scan = 0;
    for (int b = threadIdx.x * per; b < min((static_cast<int>(threadIdx.x) + 1) * per, p.batch); ++b) {
      const int n = tiles_in(b);
      scan += n;
      longest = max(longest, n);
    }
    longest = __reduce_max_sync(0xffffffffu, longest);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += u;
    }
    int* warp_sum = reinterpret_cast<int*>(gbase + L::kHead);  // free until a share ends
    if (lane == 31) {
      warp_sum[warp] = scan;
      warp_sum[kWarps + warp] = longest;
    }
    __syncthreads();
    int before = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const int v = warp_sum[i];
      if (i < warp) before += v;
      all += v;
      longest = max(longest, warp_sum[kWarps + i]);
    }
    prefix[threadIdx.x + 1] = scan + before;
  }
  __syncthreads();
  // Up to kThreads sequences their tiles are in shared memory.
  auto tiles_of = [&](int b) { return per == 1 ? prefix[b + 1] - prefix[b] : tiles_in(b); };
  // Shares: no more CTAs than tiles, so that every CTA has one and arrives
  // where it is counted.  The first `more` CTAs take one tile more.
  int grid = 1, each = 0, more = 0;
  if (!alone) {
    const int total = all * p.kv_heads;  // a cache of 2^46 codes has fewer than 2^31 tiles on any GPU
    grid = max(min(static_cast<int>(gridDim.x), total), 1);
    each = total / grid;
    more = total - each * grid;
    // Or known only now: a CTA to each line when no line is long.
    alone = lines <= static_cast<int>(gridDim.x) && longest <= kWarps * kAlone + each;
  }
  auto cta_begin = [&](int i) { return i * each + min(i, more); };
  Place mine{0, 0, 0, 0};
  if (alone) {
    const int line = static_cast<int>(blockIdx.x) >> p.cluster_log2;
    mine.b = line / p.kv_heads;
    mine.h = line - mine.b * p.kv_heads;
    if (mine.b < p.batch) mine.tiles = tiles_in(mine.b);
    c0 = (mine.tiles * rank) >> p.cluster_log2;
    c1 = (mine.tiles * (rank + 1)) >> p.cluster_log2;
  } else if (static_cast<int>(blockIdx.x) < grid) {
    c0 = cta_begin(blockIdx.x);
    c1 = cta_begin(blockIdx.x + 1);
  }
  const int u0 = c0 + (c1 - c0) * warp / kWarps, u1 = c0 + (c1 - c0) * (warp + 1) / kWarps;
  static_assert(kThreads == 256, "locate() searches 32 x 8 groups");
  auto locate = [&](int u) {  // by a converged warp
    // The last group with prefix * kv_heads <= u: by eights, then one by one.
    int s = 8 * __popc(__ballot_sync(0xffffffffu, prefix[8 * (lane + 1)] * p.kv_heads <= u));
    s += __popc(__ballot_sync(0xffffffffu, lane < 8 && prefix[s + (lane & 7) + 1] * p.kv_heads <= u));
    Place at;
    at.b = s * per;
    int r = u - prefix[s] * p.kv_heads;
    at.tiles = tiles_of(at.b);
    while (r >= at.tiles * p.kv_heads) {
      r -= at.tiles * p.kv_heads;
      at.tiles = tiles_of(++at.b);
    }
    at.h = r / at.tiles;
    at.tile = r - at.h * at.tiles;
    return at;
  };
  // To the next tile; called only when there is one.
  auto advance = [&](Place& at) {
    if (++at.tile < at.tiles) return;
    at.tile = 0;
    if (++at.h < p.kv_heads) return;
    at.h = 0;
    do {
      at.tiles = tiles_of(++at.b);
    } while (at.tiles == 0);
  };
  auto row_token = [&](int r) { return (r * p.group_inv) >> 16; };  // r / group
  auto store8 = [&](int b, int h, int row, int d, const float (&v)[8], float inv) {  // 8 outputs of a row
    const int tok = row_token(row);
    const int head = h * p.group + row - tok * p.group;
    *reinterpret_cast<uint4*>(p.o + b * p.o_batch + tok * p.o_tok + head * p.o_head + d) =
        make_uint4(pack_half2(v[0] * inv, v[1] * inv), pack_half2(v[2] * inv, v[3] * inv),
                   pack_half2(v[4] * inv, v[5] * inv), pack_half2(v[6] * inv, v[7] * inv));
  };
  // A row without keys has m' = -inf and l = 0 and becomes 0; one with NaN scores has l = NaN.
  auto inverse = [](float m, float l) { return m == -INFINITY && l == l ? 0.f : 1.f / l; };
  // Rows of sequences without keys.
  const float zero[8] = {};
  if (alone) {
    if (mine.tiles == 0 && mine.b < p.batch && rank == 0)
      for (int i = threadIdx.x; i < p.rows * (HD / 8); i += kThreads)
        store8(mine.b, mine.h, i / (HD / 8), i % (HD / 8) * 8, zero, 0.f);
  } else {
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
      if (tiles_of(b) > 0) continue;
      for (int i = threadIdx.x; i < p.rows * p.kv_heads * (HD / 8); i += kThreads) {
        const int r = i / (HD / 8);
        store8(b, r / p.rows, r % p.rows, i % (HD / 8) * 8, zero, 0.f);
      }
    }
  }

  const int g = lane >> 2, c = lane & 3;  // MMA group and position in it
  bool ok = true;
  if (u0 < u1) {
    // ------------------------------------------------------- the warp's share --
    Place at = mine;
    if (alone)
      at.tile = u0;
    else
      at = locate(u0);
    Place ahead = at;  // the next tile to load (lane 0)
    int ua = u0;
    auto load = [&](uint32_t st) {
      if (ua > u0) advance(ahead);
      ++ua;
      const uint32_t dst = ring + st * 2 * L::kCodes;
      const int head = ahead.b * p.kv_heads + ahead.h;
      mbar_arrive_expect_tx(bar + 8 * st, 2 * L::kCodes);
      tma_load_3d(dst, &tm_k, bar + 8 * st, 0, ahead.tile * kTileKeys, head);
      tma_load_3d(dst + L::kCodes, &tm_v, bar + 8 * st, 0, ahead.tile * kTileKeys, head);
    };
    if (lane == 0)
      for (int i = 0; i < kStages && ua < u1; ++i) load(i);
    auto scales = [&](const Place& s, float& k, float& v) {
      const long long idx =
          (static_cast<long long>(s.b) * p.kv_heads + s.h) * p.n_blocks + s.tile / (kKv8Block / kTileKeys);
      k = p.k_scale[idx];
      v = p.v_scale[idx];
    };
    Place nx = at;  // the next tile's place, whose scales are loaded ahead
    float sk_next, sv_next;
    scales(at, sk_next, sv_next);
    uint32_t st = 0, ph = 0;
    for (int u = u0; u < u1;) {
      // One line's tiles [at.tile, at.tile + count).
      const Place seg = at;
      const int count = min(seg.tiles - seg.tile, u1 - u);
      const int len = kv8_len(p.lens, p.kv_valid, p.kv_len, seg.b);
      const int line0 = u - seg.tile;
      uint32_t qf[NT][HD / 16][2];
      int lim[NT][2];  // keys visible to rows 8 nt + 2c and the next
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int r = 8 * nt + 2 * c + x;
          lim[nt][x] = p.causal && r < p.rows ? min(len, len - p.q_len + row_token(r) + 1) : len;
        }
        const int r = 8 * nt + g;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) qf[nt][k][0] = qf[nt][k][1] = 0u;
        if (r < p.rows) {
          const int tok = row_token(r);
          const int head = seg.h * p.group + r - tok * p.group;
          // This lane's k indexes: HD / 4 consecutive values of the row, four of them in each MMA step.
          const uint4* src = reinterpret_cast<const uint4*>(p.q + seg.b * p.q_batch + tok * p.q_tok + head * p.q_head +
                                                            c * (HD / 4));
#pragma unroll
          for (int k = 0; k < HD / 32; ++k) {
            const uint4 v = src[k];
            qf[nt][2 * k][0] = v.x;
            qf[nt][2 * k][1] = v.y;
            qf[nt][2 * k + 1][0] = v.z;
            qf[nt][2 * k + 1][1] = v.w;
          }
        }
      }
      float acc[NT][HD / 16][4];
      float m[NT][2], l[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int j = 0; j < HD / 16; ++j) acc[nt][j][0] = acc[nt][j][1] = acc[nt][j][2] = acc[nt][j][3] = 0.f;
      }
      // Keys from here on are hidden from some row.
      const int edge = min(len, p.causal ? len - p.q_len + 1 : len);
      for (int t = 0; t < count; ++t, ++u) {
        const float sk = sk_next, sv = sv_next;
        const int key0 = nx.tile * kTileKeys;
        if (u + 1 < u1) {
          advance(nx);
          scales(nx, sk_next, sv_next);
        }
        if (ok) ok = mbar_wait_warp(bar + 8 * st, ph, abort_flag, p.status);
        if (!ok) continue;
        const uint32_t kt = ring + st * 2 * L::kCodes, vt = kt + L::kCodes;
        // K: the lane's runs of rows 16 i + g and 16 i + g + 8.
        uint32_t kw[2][2][HD / 16];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int key = 16 * i + 8 * x + g;
#pragma unroll
            for (int k = 0; k < HD / 64; ++k) {
              const int run = c * (HD / 64) + k;
              const int at16 = HD == 128 ? run ^ (key & 7) : run ^ ((key >> 1) & 3);
              const uint4 v = ld_shared_v4u(kt + key * HD + at16 * 16);
              kw[i][x][4 * k] = v.x;
              kw[i][x][4 * k + 1] = v.y;
              kw[i][x][4 * k + 2] = v.z;
              kw[i][x][4 * k + 3] = v.w;
            }
          }
        // V: HD / 8 codes of each of the lane's keys 16 i + 2c, + 1, + 8, + 9.
        uint32_t vw[2][4][HD / 32];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int key = 16 * i + 2 * c + (x & 1) + (x >> 1) * 8;
            if constexpr (HD == 128) {
              const uint4 v = ld_shared_v4u(vt + key * HD + ((g ^ (key & 7)) << 4));
              vw[i][x][0] = v.x;
              vw[i][x][1] = v.y;
              vw[i][x][2] = v.z;
              vw[i][x][3] = v.w;
            } else {
              const uint2 v = ld_shared_v2u(vt + key * HD + (((g >> 1) ^ ((key >> 1) & 3)) << 4) + (g & 1) * 8);
              vw[i][x][0] = v.x;
              vw[i][x][1] = v.y;
            }
          }
        float s[NT][2][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) s[nt][i][0] = s[nt][i][1] = s[nt][i][2] = s[nt][i][3] = 0.f;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t a0, a1, a2, a3;
            kv8_to_half2<FMT>(kw[i][0][k], a0, a2);
            kv8_to_half2<FMT>(kw[i][1][k], a1, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_16816(s[nt][i], a0, a1, a2, a3, qf[nt][k][0], qf[nt][k][1]);
          }
        // A factor of 0 (a scale of 0, or one whose product with the softmax scale
        // underflows) makes scores of 0, whatever the codes; with 1 in its place a
        // masked -inf does not meet 0.  A V scale of 0 makes values of 0.
        const float factor = sk * p.scale_log2;
        const float mul = factor > 0.f ? factor : 1.f;
        const bool valued = sv > kKv8NoValue;
        const float lsv = valued ? __log2f(sv) : kKv8NoScale;
        const float isv = valued ? __fdividef(1.f, sv) : kKv8NoScaleInverse;
        if (key0 + kTileKeys > edge || !(factor > 0.f) || !valued) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (!(factor > 0.f)) s[nt][i][e] *= 0.f;
                if (key0 + 16 * i + 8 * (e >> 1) + g >= lim[nt][e & 1]) s[nt][i][e] = -INFINITY;
              }
          if (FMT == kKv8E4m3 || !valued) {
            // What lies past the length may decode to NaN (e4m3), and 0 * NaN is NaN.
            const int live = valued ? len : 0;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int x = 0; x < 4; ++x)
                if (key0 + 16 * i + 2 * c + (x & 1) + (x >> 1) * 8 >= live) {
#pragma unroll
                  for (int k = 0; k < HD / 32; ++k) vw[i][x][k] = 0u;
                }
          }
        }
        bool grow = false;
        float top[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float mx = fmaxf(fmaxf(s[nt][0][x], s[nt][0][2 + x]), fmaxf(s[nt][1][x], s[nt][1][2 + x]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            top[nt][x] = fmaf(mx, mul, lsv);
            grow |= top[nt][x] > m[nt][x] + kRescale;
          }
        if (__any_sync(0xffffffffu, grow)) {
          // The maximum moves, and what is summed so far with it, only when it
          // would otherwise lag by more than 2^8 (fp16 holds p' up to 2^16).
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float mn = fmaxf(m[nt][x], top[nt][x]);
              const float f = mn == m[nt][x] ? 1.f : ex2_approx(m[nt][x] - mn);
              m[nt][x] = mn;
              l[nt][x] *= f;
#pragma unroll
              for (int j = 0; j < HD / 16; ++j) {
                acc[nt][j][x] *= f;
                acc[nt][j][2 + x] *= f;
              }
            }
        }
        // The tile is in registers: its stage takes the next load.  Here rather than
        // right behind the loads from it, which the fence would wait for (3 % of
        // batch 8 x 16 heads on 4096 keys).
        if (u + kStages < u1) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) load(st);
        }
        if (++st == kStages) {
          st = 0;
          ph ^= 1u;
        }
        uint32_t pf[NT][2][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float off[2], sum[2] = {0.f, 0.f};
#pragma unroll
          for (int x = 0; x < 2; ++x) off[x] = lsv - (m[nt][x] == -INFINITY ? 0.f : m[nt][x]);
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const float a = ex2_approx(fmaf(s[nt][i][2 * y], mul, off[0]));
              const float b = ex2_approx(fmaf(s[nt][i][2 * y + 1], mul, off[1]));
              sum[0] += a;
              sum[1] += b;
              pf[nt][i][y] = transpose8(pack_half2(a, b));
            }
          l[nt][0] = fmaf(sum[0], isv, l[nt][0]);
          l[nt][1] = fmaf(sum[1], isv, l[nt][1]);
        }
        // O'^T += V^T P^T: MMA j takes codes 2j and 2j + 1 of every lane's run.
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int k = 0; k < HD / 32; ++k)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const uint32_t sel = y == 0 ? 0x5140u : 0x7362u;  // codes 0, 1 / 2, 3 of two keys, interleaved
              uint32_t a0, a1, a2, a3;
              kv8_to_half2<FMT>(prmt(vw[i][0][k], vw[i][1][k], sel), a0, a1);
              kv8_to_half2<FMT>(prmt(vw[i][2][k], vw[i][3][k], sel), a2, a3);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma_16816(acc[nt][2 * k + y], a0, a1, a2, a3, pf[nt][i][0], pf[nt][i][1]);
            }
      }
      at = nx;
      // The line's sums over the lanes of a column; then out, or into a slot.
      const bool whole = seg.tile == 0 && count == seg.tiles;
      const bool first = line0 + seg.tile == u0;  // the share's first line
      float* slot = reinterpret_cast<float*>(gbase + (first ? L::kHead + warp * L::kSlot : ring - base));
      if (!whole && !first) __syncwarp();  // the ring's last tile has been read by all lanes
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float sum = l[nt][x];
          sum += __shfl_xor_sync(0xffffffffu, sum, 4);
          sum += __shfl_xor_sync(0xffffffffu, sum, 8);
          sum += __shfl_xor_sync(0xffffffffu, sum, 16);
          const int row = 8 * nt + 2 * c + x;
          if (row < p.rows) {
            if (whole) {
              const float inv = inverse(m[nt][x], sum);
#pragma unroll
              for (int j = 0; j < HD / 16; j += 4) {
                const float v[8] = {acc[nt][j][x],     acc[nt][j][2 + x],     acc[nt][j + 1][x], acc[nt][j + 1][2 + x],
                                    acc[nt][j + 2][x], acc[nt][j + 2][2 + x], acc[nt][j + 3][x], acc[nt][j + 3][2 + x]};
                if (ok) store8(seg.b, seg.h, row, g * (HD / 8) + 2 * j, v, inv);
              }
            } else {
#pragma unroll
              for (int j = 0; j < HD / 16; j += 2)
                reinterpret_cast<float4*>(slot)[row * kF4 + g * (HD / 32) + j / 2] =
                    make_float4(acc[nt][j][x], acc[nt][j][2 + x], acc[nt][j + 1][x], acc[nt][j + 1][2 + x]);
              if (g == 0) {
                slot[L::kRows * HD + row] = m[nt][x];
                slot[L::kRows * HD + L::kRows + row] = sum;
              }
            }
          }
        }
      if (!whole && lane == 0 && ok) info[2 * warp + (first ? 0 : 1)] = SlotInfo{line0, seg.b, seg.h, seg.tiles};
    }
    // On a timeout, loads of this warp may still be landing.
    if (!ok && lane == 0)
      for (int i = 0; i < kStages; ++i) mbar_wait_drain(bar + 8 * i, ph ^ (i < static_cast<int>(st) ? 1u : 0u));
  }
  __syncthreads();
  const int units = p.rows * kF4;
  if (alone) {
    // --------------------------------------- the line's parts in this cluster --
    if (mine.tiles < 2) return;  // no keys, or one warp had them all
    const bool joint = p.cluster_log2 != 0;
    if (!joint && (*abort_flag != 0 || info[2 * (kWarps - 1)].line < 0)) return;
    auto put = [&](int e, const float4& v, float m, float l) {
      const float inv = inverse(m, l);
      const int r = e / kF4;
      const int tok = row_token(r);
      const int head = mine.h * p.group + r - tok * p.group;
      *reinterpret_cast<uint2*>(p.o + mine.b * p.o_batch + tok * p.o_tok + head * p.o_head + e % kF4 * 4) =
          make_uint2(pack_half2(v.x * inv, v.y * inv), pack_half2(v.z * inv, v.w * inv));
    };
    // Sum of eight parts whose loads are all in flight; get(i, v, m, l) says whether there is an i-th.
    auto join = [&](auto get, float4& v, float& m, float& l) {
      float pm[8], pl[8];
      float4 o[8];
      m = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        pm[i] = -INFINITY;
        pl[i] = 0.f;
        o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        get(i, o[i], pm[i], pl[i]);
        m = fmaxf(m, pm[i]);
      }
      v = make_float4(0.f, 0.f, 0.f, 0.f);
      l = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float f = pm[i] == m ? 1.f : ex2_approx(pm[i] - m);
        l = fmaf(pl[i], f, l);
        v = make_float4(fmaf(o[i].x, f, v.x), fmaf(o[i].y, f, v.y), fmaf(o[i].z, f, v.z), fmaf(o[i].w, f, v.w));
      }
    };
    float4 v;
    float m, l;
    float4* part_v = reinterpret_cast<float4*>(gbase);                      // the CTA's part: the rings are idle
    float* part_ml = reinterpret_cast<float*>(gbase) + L::kRows * HD;       // (m', l) per row
#pragma unroll 1
    for (int e = threadIdx.x; e < units; e += kThreads) {
      static_assert(kWarps == 8, "join() takes eight parts");
      join([&](int i, float4& ov, float& om, float& ol) {
        const float* part = reinterpret_cast<const float*>(gbase + L::kHead + i * L::kSlot);
        if (info[2 * i].line >= 0) {
          ov = reinterpret_cast<const float4*>(part)[e];
          om = part[L::kRows * HD + e / kF4];
          ol = part[L::kRows * HD + L::kRows + e / kF4];
        }
      }, v, m, l);
      if (!joint) {
        put(e, v, m, l);
      } else {
        part_v[e] = v;
        if (e % kF4 == 0) reinterpret_cast<float2*>(part_ml)[e / kF4] = make_float2(m, l);
      }
    }
    if (!joint) return;
    __syncwarp();
    cluster_sync();
    // Each CTA of the cluster joins a share of the outputs, in CTA order.
    const int n = 1 << p.cluster_log2;
#pragma unroll 1
    for (int e = rank + n * static_cast<int>(threadIdx.x); e < units; e += n * kThreads) {
      const uint32_t at_v = base + e * 16u, at_ml = base + L::kRows * HD * 4u + e / kF4 * 8u;
      join([&](int i, float4& ov, float& om, float& ol) {
        if (i < n) {
          ov = ld_cluster_v4f(mapa_shared(at_v, i));
          const float2 ml = ld_cluster_v2f(mapa_shared(at_ml, i));
          om = ml.x;
          ol = ml.y;
        }
      }, v, m, l);
      put(e, v, m, l);
    }
    __syncwarp();
    cluster_sync();  // the parts have been read
    return;
  }
  if (*abort_flag != 0 || c0 >= c1) return;

  // ------------------------------------------- lines that cross warps or CTAs --
  // Slots in order (first and last line of warp 0, of warp 1, ...); the slots of
  // one line are a run.  Warp 0 lists the runs: mask of the slots, and in
  // ends[0] / ends[1] the line that goes on before / behind the CTA's share.
  // All code from here on runs once, out of a cold instruction cache, so it is
  // kept small rather than unrolled.
  uint32_t* runs = reinterpret_cast<uint32_t*>(prefix);          // [kWarps + 1]
  int* ends = prefix + kWarps + 2;                               // slot index of the line, -1: none
  volatile int* n_runs = prefix + kWarps + 4;
  constexpr int kPart = L::kSlot / 4;
  auto put = [&](const SlotInfo& at, int e, const float4& v, float m, float l) {
    const float inv = inverse(m, l);
    const int r = e / kF4;
    const int tok = row_token(r);
    const int head = at.h * p.group + r - tok * p.group;
    *reinterpret_cast<uint2*>(p.o + at.b * p.o_batch + tok * p.o_tok + head * p.o_head + e % kF4 * 4) =
        make_uint2(pack_half2(v.x * inv, v.y * inv), pack_half2(v.z * inv, v.w * inv));
  };
  auto add_part = [](float4& v, float& m, float& l, const float4& o, float pm, float pl) {
    const float mn = fmaxf(m, pm);
    const float fo = m == mn ? 1.f : ex2_approx(m - mn);
    const float fn = pm == mn ? 1.f : ex2_approx(pm - mn);
    m = mn;
    l = l * fo + pl * fn;
    v = make_float4(v.x * fo + o.x * fn, v.y * fo + o.y * fn, v.z * fo + o.z * fn, v.w * fo + o.w * fn);
  };
  if (warp == 0) {
    SlotInfo at{-1, 0, 0, 0};
    if (lane < 2 * kWarps) at = info[lane];
    const uint32_t valid = __ballot_sync(0xffffffffu, at.line >= 0);
    const uint32_t below = valid & ((1u << lane) - 1u);
    const int prev = __shfl_sync(0xffffffffu, at.line, below != 0u ? 31 - __clz(below) : 0);
    const bool start = at.line >= 0 && (below == 0u || prev != at.line);
    const uint32_t starts = __ballot_sync(0xffffffffu, start);
    const uint32_t later = starts & ~((2u << lane) - 1u);
    if (lane < 2) ends[lane] = -1;
    __syncwarp();
    if (start) {
      runs[__popc(starts & ((1u << lane) - 1u))] =
          valid & ~((1u << lane) - 1u) & (later != 0u ? (later & -later) - 1u : ~0u);
      if (at.line < c0 || at.line + at.tiles > c1) ends[at.line <= c0 ? 0 : 1] = lane;
    }
    if (lane == 0) *n_runs = __popc(starts);
  }
  __syncthreads();
  const int work = *n_runs * units;
#pragma unroll 1
  for (int i = threadIdx.x; i < work; i += kThreads) {
    const int run = i / units, e = i - run * units;
    uint32_t mask = runs[run];
    const SlotInfo at = info[__ffs(mask) - 1];
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, l = 0.f;
#pragma unroll 1
    for (; mask != 0u; mask &= mask - 1u) {
      const int k = __ffs(mask) - 1;
      const float* part = reinterpret_cast<const float*>(
          gbase + ((k & 1) ? static_cast<uint32_t>(k >> 1) * kStages * 2 * L::kCodes : L::kHead + (k >> 1) * L::kSlot));
      add_part(v, m, l, reinterpret_cast<const float4*>(part)[e], part[L::kRows * HD + e / kF4],
               part[L::kRows * HD + L::kRows + e / kF4]);
    }
    if (at.line >= c0 && at.line + at.tiles <= c1) {
      put(at, e, v, m, l);
    } else {
      float* mine = p.part + (2LL * blockIdx.x + (at.line <= c0 ? 0 : 1)) * kPart;  // a part per end of the share
      reinterpret_cast<float4*>(mine)[e] = v;
      if (e % kF4 == 0) {
        mine[L::kRows * HD + e / kF4] = m;
        mine[L::kRows * HD + L::kRows + e / kF4] = l;
      }
    }
  }
  if (ends[0] < 0 && ends[1] < 0) return;
  // Count in; the CTA of a line's last part joins them all, in CTA order.
  auto owner = [&](int u) {  // the CTA whose share holds tile u
    const int big = more * (each + 1);
    return u < big ? u / (each + 1) : more + (u - big) / each;
  };
  __syncthreads();  // the counting threads' releases cover the CTA's stores
  if (threadIdx.x < 2) {
    int parts = 0;  // of the line, if this CTA has to join them
    if (ends[threadIdx.x] >= 0) {
      const SlotInfo at = info[ends[threadIdx.x]];
      // Of the lines that start in a CTA only its last one can go on behind it.
      const int first = owner(at.line);
      const int n = owner(at.line + at.tiles - 1) - first + 1;
      unsigned* count = p.count + first;
      unsigned was;
      asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(was) : "l"(count) : "memory");
      if (static_cast<int>(was) == n - 1) {
        *count = 0u;  // ready for the next launch
        parts = n;
      }
    }
    runs[threadIdx.x] = static_cast<uint32_t>(parts);
  }
  __syncthreads();
  float4* sums = reinterpret_cast<float4*>(gbase);  // [kThreads] O', then (m', l); the rings are idle
#pragma unroll 1
  for (int end = 0; end < 2; ++end) {
    const int parts = static_cast<int>(runs[end]);
    if (parts == 0) continue;
    const SlotInfo at = info[ends[end]];
    const int first = owner(at.line);
    const float* part0 = p.part + 2LL * first * kPart;
    // Only the first part may lie behind its CTA's first tile.
    const int skip = at.line <= cta_begin(first) ? 0 : kPart;
    // More than eight parts: groups of threads take a range of them each (one
    // token on 131071 keys 55.6 -> 53.8 us); up to eight are one round of loads.
    const int groups = parts > 8 ? max(kThreads / units, 1) : 1;
    const int group = static_cast<int>(threadIdx.x) / units;
    if (groups > 1) __syncthreads();  // sums is free
#pragma unroll 1
    for (int e = threadIdx.x - group * units; group < groups && e < units; e += kThreads) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      float m = -INFINITY, l = 0.f;
      const int k1 = parts * (group + 1) / groups;
#pragma unroll 1
      for (int k = parts * group / groups; k < k1; k += 8) {
        float4 o[8];
        float pm[8], pl[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int x = min(k + i, k1 - 1);
          const float* s = part0 + 2LL * x * kPart + (x == 0 ? skip : 0);
          pm[i] = __ldcg(s + L::kRows * HD + e / kF4);
          pl[i] = __ldcg(s + L::kRows * HD + L::kRows + e / kF4);
          o[i] = __ldcg(reinterpret_cast<const float4*>(s) + e);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (k + i < k1) add_part(v, m, l, o[i], pm[i], pl[i]);
      }
      if (groups == 1) {
        put(at, e, v, m, l);
      } else {
        sums[threadIdx.x] = v;
        reinterpret_cast<float2*>(sums + kThreads)[threadIdx.x] = make_float2(m, l);
      }
    }
    if (groups == 1) continue;
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < units) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      float m = -INFINITY, l = 0.f;
#pragma unroll 1
      for (int i = 0; i < groups; ++i) {
        const float2 ml = reinterpret_cast<const float2*>(sums + kThreads)[i * units + threadIdx.x];
        add_part(v, m, l, sums[i * units + threadIdx.x], ml.x, ml.y);
      }
      put(at, threadIdx.x, v, m, l);
    }
  }
}

template <int FMT, int HD, int NT>
cudaError_t launch_nt(const CUtensorMap& tk, const CUtensorMap& tv, const Kv8AttnParams& p, int grid, int dev,
                      cudaStream_t stream) {
  static std::atomic<uint64_t> configured{0};
  const uint64_t bit = 1ull << (dev & 63);
  auto kernel = kv8_rows_sm100_kernel<FMT, HD, NT>;
  if ((configured.load(std::memory_order_acquire) & bit) == 0) {
    const cudaError_t e =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, RowsSmem<HD, NT>::kBytes);
    if (e != cudaSuccess) return e;
    configured.fetch_or(bit, std::memory_order_acq_rel);
  }
  return launch_pdl_cluster(kernel, grid, 1u << p.cluster_log2, kThreads, RowsSmem<HD, NT>::kBytes, stream, tk, tv, p);
}
template <int FMT, int HD>
cudaError_t launch_hd(const CUtensorMap& tk, const CUtensorMap& tv, const Kv8AttnParams& p, int grid, int dev,
                      cudaStream_t stream) {
  return p.rows <= 8 ? launch_nt<FMT, HD, 1>(tk, tv, p, grid, dev, stream)
                     : launch_nt<FMT, HD, 2>(tk, tv, p, grid, dev, stream);
}

}  // namespace

// One CTA per SM, but none without a tile when every sequence is as long as it can be.
int kv8_rows_plan(Kv8AttnParams* p, int sms) {
  const long long lines = static_cast<long long>(p->batch) * p->kv_heads;
  const long long longest = (p->kv_len + kTileKeys - 1) / kTileKeys;
  const long long tiles = lines * longest;
  p->group_inv = 65536 / p->group + 1;
  p->cluster_log2 = 0;
  // Twice the CTAs while a warp has more than one tile and they fit in one wave:
  // clusters of eight do not fill every GPC (16 of them took a second wave).
  while (p->cluster_log2 < 3 && longest > kWarps << p->cluster_log2 &&
         (lines << (p->cluster_log2 + 1)) * 8 <= sms * (p->cluster_log2 < 2 ? 7 : 6))
    ++p->cluster_log2;
  p->alone = lines <= sms &&
             longest <= (kWarps * kAlone + (p->lens == nullptr ? tiles / sms : 0)) << p->cluster_log2;
  if (p->alone) return static_cast<int>(lines << p->cluster_log2);
  p->cluster_log2 = 0;
  return static_cast<int>(tiles < sms ? (tiles > 0 ? tiles : 1) : sms);
}
int kv8_rows_tile() { return kTileKeys; }
size_t kv8_rows_part_floats(int head_dim, int grid) { return 2 * static_cast<size_t>(grid) * 16 * (head_dim + 2); }

cudaError_t launch_kv8_rows(const CUtensorMap& tk, const CUtensorMap& tv, const Kv8AttnParams& p, int grid, int dev,
                            cudaStream_t stream) {
  if (p.format == kKv8Int8)
    return p.head_dim == 128 ? launch_hd<kKv8Int8, 128>(tk, tv, p, grid, dev, stream)
                             : launch_hd<kKv8Int8, 64>(tk, tv, p, grid, dev, stream);
  return p.head_dim == 128 ? launch_hd<kKv8E4m3, 128>(tk, tv, p, grid, dev, stream)
                           : launch_hd<kKv8E4m3, 64>(tk, tv, p, grid, dev, stream);
}

}  // namespace ax
