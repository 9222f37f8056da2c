// kv8_rows_sm100.cu -- attention of a few query rows over the 8-bit K/V cache.
//
// A kv head's query rows (its query heads x the call's query tokens) are taken
// 16 at a time, so that each code is read and converted once for all of them.
// With r rows the kernel does 4 r flops a code byte: at a few rows HBM bounds
// it, and everything here serves to keep loads in flight.
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
// Work: every (sequence, kv head, row tile) is a row of key tiles of 64; all
// of them together form one line of tiles that is cut into equal contiguous
// shares, one per CTA (two CTAs per SM), so ragged lengths and single long
// sequences load the SMs alike.  A CTA that covers only part of a sequence's
// keys stores (m', l, O') in its workspace slot and counts itself in; the last
// one to arrive joins the parts in CTA order, so the result does not depend on
// the order of arrival.
//
// A CTA: warp 4 loads tiles (16 KiB: 64 K rows, 64 V rows) by TMA into a ring;
// warps 0-3 take 16 keys of each tile each, with their own m', l, O' and no
// synchronisation among them until the CTA leaves the sequence.  The products
// are m16n8k16 mma.sync: with at most 16 rows a 128-row tcgen05 tile would be
// mostly empty, and reading codes from shared memory into fragments and
// converting them there avoids a second pass through shared memory.  Which of
// a row's codes form an MMA's k (for K) or n (for V) index is free as long as Q,
// or the stored O, follows: a lane takes 16-byte runs of a row (32 codes
// of one K row, 16 of each of its four V rows), which TMA's swizzle spreads over all banks.
#include <atomic>

#include "api_internal.h"
#include "kernels.h"
#include "kv8_common.cuh"
#include "sm100_ptx.cuh"

namespace ax {
namespace {

constexpr int kStages = 4;
constexpr int kConsumers = 128;
constexpr int kThreads = kConsumers + 32;
constexpr int kCtasPerSm = 2;
constexpr float kRescale = 8.f;  // log2 units by which the maximum may lag
constexpr float kNoScale = -33.f;  // stands for log2 of the scale of an all-zero V block (below any real one)

template <int HD>
struct RowsSmem {
  static constexpr uint32_t kTile = kKv8Block * HD;             // codes of K (or V) of a tile
  static constexpr uint32_t kRing = 0;
  static constexpr uint32_t kMerge = kRing + kStages * 2 * kTile;  // [4 warps][16 rows][HD] fp32
  static constexpr uint32_t kStat = kMerge + 4 * 16 * HD * 4;      // [4 warps][16 rows] m', l
  static constexpr uint32_t kPrefix = kStat + 4 * 16 * 8;          // tiles of the sequences before each share
  static constexpr uint32_t kBar = kPrefix + (kConsumers + 1) * 8 + 8;
  static constexpr uint32_t kBytes = kBar + 2 * kStages * 8 + 16 + 1024;  // + alignment slack
};
static_assert(2 * (RowsSmem<128>::kBytes + 1024) <= 228 * 1024, "two CTAs must fit on an SM");

__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint2 ld_shared_v2u(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void* tmap, uint32_t bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(tmap), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// A place in the line of tiles: tile `tile` of `tiles` of (sequence b, row line
// hr = kv head * row_tiles + row tile).
struct Place {
  int b, hr, tile, tiles;
};

template <int FMT, int HD>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
    kv8_rows_sm100_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                          const Kv8AttnParams p) {
  extern __shared__ uint8_t smem_raw[];
  using L = RowsSmem<HD>;
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  float* stat = reinterpret_cast<float*>(gbase + L::kStat);
  long long* prefix = reinterpret_cast<long long*>(gbase + L::kPrefix);
  const uint32_t bar_full = base + L::kBar, bar_empty = bar_full + 8 * kStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + L::kBar + 16 * kStages);
  volatile unsigned* last_flag = reinterpret_cast<volatile unsigned*>(gbase + L::kBar + 16 * kStages + 4);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(bar_full + 8 * i, 1);
      mbar_init(bar_empty + 8 * i, kConsumers / 32);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 4 && lane == 0) {
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  // prefix[t] = tiles of one row line of the sequences before share t (128
  // shares of `per` sequences each).
  auto tiles_of = [&](int b) { return (kv8_len(p.lens, p.kv_valid, p.kv_len, b) + kKv8Block - 1) / kKv8Block; };
  const int per = (p.batch + kConsumers - 1) / kConsumers;
  if (warp < 4) {
    long long sum = 0;
    for (int b = threadIdx.x * per; b < min((static_cast<int>(threadIdx.x) + 1) * per, p.batch); ++b) sum += tiles_of(b);
    prefix[threadIdx.x + 1] = sum;
    if (threadIdx.x == 0) prefix[0] = 0;
  }
  __syncthreads();
  if (warp == 0) {
    long long run = 0;
    for (int i = 0; i < kConsumers / 32; ++i) {
      long long v = prefix[1 + i * 32 + lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      prefix[1 + i * 32 + lane] = v + run;
      run += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  __syncthreads();
  const int lines = p.kv_heads * p.row_tiles;  // row lines per sequence
  const long long total = prefix[kConsumers] * lines;
  // No more shares than tiles, so that every share has one and arrives where it is counted.
  const long long grid = max(min(static_cast<long long>(gridDim.x), total), 1LL);
  auto share_begin = [&](long long i) { return total * i / grid; };
  const bool idle = blockIdx.x >= grid;
  const long long u0 = idle ? total : share_begin(blockIdx.x), u1 = idle ? total : share_begin(blockIdx.x + 1LL);
  // The CTA whose share holds tile u.
  auto owner = [&](long long u) {
    long long i = min((u * grid) / total, grid - 1);
    while (share_begin(i + 1) <= u) ++i;
    while (share_begin(i) > u) --i;
    return i;
  };
  auto locate = [&](long long u) {
    int s = 0;  // share of sequences: the last one with prefix * lines <= u
    for (int step = kConsumers / 2; step > 0; step >>= 1)
      if (prefix[s + step] * lines <= u) s += step;
    Place at;
    at.b = s * per;
    u -= prefix[s] * lines;
    at.tiles = tiles_of(at.b);
    while (u >= static_cast<long long>(at.tiles) * lines) {
      u -= static_cast<long long>(at.tiles) * lines;
      at.tiles = tiles_of(++at.b);
    }
    at.hr = static_cast<int>(u / at.tiles);
    at.tile = static_cast<int>(u % at.tiles);
    return at;
  };
  // To the next tile; called only when there is one.
  auto advance = [&](Place& at) {
    if (++at.tile < at.tiles) return;
    at.tile = 0;
    if (++at.hr < lines) return;
    at.hr = 0;
    do {
      at.tiles = tiles_of(++at.b);
    } while (at.tiles == 0);
  };

  if (warp == 4) {
    // ------------------------------------------------------------ producer --
    if (lane == 0 && u0 < u1) {
      Place at = locate(u0);
      uint32_t i = 0;
      for (long long u = u0; u < u1; ++u, ++i) {
        if (u > u0) advance(at);
        const uint32_t st = i % kStages;
        if (!mbar_wait(bar_empty + 8 * st, ((i / kStages) & 1u) ^ 1u, abort_flag, p.status)) break;
        const uint32_t dst = base + L::kRing + st * 2 * L::kTile;
        const int head = at.b * p.kv_heads + at.hr / p.row_tiles;
        mbar_arrive_expect_tx(bar_full + 8 * st, 2 * L::kTile);
        tma_load_3d(dst, &tm_k, bar_full + 8 * st, 0, at.tile * kKv8Block, head);
        tma_load_3d(dst + L::kTile, &tm_v, bar_full + 8 * st, 0, at.tile * kKv8Block, head);
      }
      // Every copy has landed before the CTA can end: wait for the last use of each stage.
      for (uint32_t k = i > kStages ? i - kStages : 0; k < i; ++k)
        mbar_wait_drain(bar_full + 8 * (k % kStages), (k / kStages) & 1u);
    }
    return;
  }

  // ------------------------------------------------------------- consumers --
  const int g = lane >> 2, c = lane & 3;  // MMA group (row / key / column) and position in it
  auto sync = [&] { named_bar_sync(1, kConsumers); };
  // Rows of sequences without keys.
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
    if (tiles_of(b) > 0) continue;
    const long long n = static_cast<long long>(p.rows) * p.kv_heads * (HD / 8);
    for (long long i = threadIdx.x; i < n; i += kConsumers) {
      const int d8 = static_cast<int>(i % (HD / 8));
      const long long r = i / (HD / 8);
      const int head = static_cast<int>(r % (static_cast<long long>(p.kv_heads) * p.group));
      const long long tok = r / (static_cast<long long>(p.kv_heads) * p.group);
      *reinterpret_cast<uint4*>(p.o + b * p.o_batch + tok * p.o_tok + head * p.o_head + d8 * 8) = make_uint4(0, 0, 0, 0);
    }
  }
  if (u0 >= u1) return;

  bool ok = true;
  uint32_t i = 0;
  Place at = locate(u0);
  Place nx = at;  // the next tile's place, whose scales are loaded ahead
  auto scales = [&](const Place& s, float& k, float& v) {
    const long long idx =
        (static_cast<long long>(s.b) * p.kv_heads + s.hr / p.row_tiles) * p.n_blocks + s.tile;
    k = __ldg(p.k_scale + idx);
    v = __ldg(p.v_scale + idx);
  };
  float sk_next, sv_next;
  scales(at, sk_next, sv_next);
  for (long long u = u0; u < u1;) {
    // One sequence's row line: tiles [at.tile, at.tile + count).
    const int count = static_cast<int>(min(static_cast<long long>(at.tiles - at.tile), u1 - u));
    const Place seg = at;
    const int kvh = seg.hr / p.row_tiles;
    const int r0 = (seg.hr % p.row_tiles) * 16;
    const int len = kv8_len(p.lens, p.kv_valid, p.kv_len, seg.b);
    uint32_t qf[HD / 16][4];
    int lim[2];  // keys visible to rows g and g + 8
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = r0 + g + 8 * x;
      lim[x] = 0;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) qf[k][x] = qf[k][x + 2] = 0u;
      if (r < p.rows) {
        const int tok = r / p.group;
        const int head = kvh * p.group + r % p.group;
        lim[x] = p.causal ? min(len, len - p.q_len + tok + 1) : len;
        // This lane's k indexes: HD / 4 consecutive values of the row; MMA step k takes four of them.
        const uint4* src = reinterpret_cast<const uint4*>(p.q + seg.b * p.q_batch + tok * p.q_tok + head * p.q_head +
                                                          c * (HD / 4));
#pragma unroll
        for (int k = 0; k < HD / 32; ++k) {
          const uint4 v = __ldg(src + k);
          qf[2 * k][x] = v.x;
          qf[2 * k][x + 2] = v.y;
          qf[2 * k + 1][x] = v.z;
          qf[2 * k + 1][x + 2] = v.w;
        }
      }
    }
    float acc[HD / 8][4];
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    for (int t = 0; t < count; ++t, ++u, ++i) {
      const float sk = sk_next, sv = sv_next;
      at = nx;
      if (u + 1 < u1) {
        advance(nx);
        scales(nx, sk_next, sv_next);
      }
      const uint32_t st = i % kStages;
      if (ok) ok = mbar_wait_warp(bar_full + 8 * st, (i / kStages) & 1u, abort_flag, p.status);
      if (!ok) continue;
      const uint32_t kt = base + L::kRing + st * 2 * L::kTile, vt = kt + L::kTile;
      // K rows of the warp's 16 keys (8 per MMA column tile).
      uint32_t kw[2][HD / 16];
#pragma unroll
      for (int n8 = 0; n8 < 2; ++n8) {
        const int key = warp * 16 + n8 * 8 + g;
#pragma unroll
        for (int k = 0; k < HD / 64; ++k) {
          // 16-byte run c * (HD / 64) + k of the row, at its swizzled place.
          const int run = c * (HD / 64) + k;
          const int at16 = HD == 128 ? run ^ (key & 7) : run ^ ((key >> 1) & 3);
          const uint4 v = ld_shared_v4u(kt + key * HD + at16 * 16);
          kw[n8][4 * k] = v.x;
          kw[n8][4 * k + 1] = v.y;
          kw[n8][4 * k + 2] = v.z;
          kw[n8][4 * k + 3] = v.w;
        }
      }
      // V: HD / 8 codes of each of the lane's four keys 2c, 2c + 1, 2c + 8, 2c + 9.
      uint32_t vw[4][HD / 32];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int key = warp * 16 + 2 * c + (x & 1) + (x >> 1) * 8;
        if constexpr (HD == 128) {
          const uint4 v = ld_shared_v4u(vt + key * HD + ((g ^ (key & 7)) << 4));
          vw[x][0] = v.x;
          vw[x][1] = v.y;
          vw[x][2] = v.z;
          vw[x][3] = v.w;
        } else {
          const uint2 v = ld_shared_v2u(vt + key * HD + (((g >> 1) ^ ((key >> 1) & 3)) << 4) + (g & 1) * 8);
          vw[x][0] = v.x;
          vw[x][1] = v.y;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_empty + 8 * st);  // the stage is in registers
      float s[2][4];
#pragma unroll
      for (int n8 = 0; n8 < 2; ++n8) {
        s[n8][0] = s[n8][1] = s[n8][2] = s[n8][3] = 0.f;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          uint32_t b0, b1;
          kv8_to_half2<FMT>(kw[n8][k], b0, b1);
          mma_16816(s[n8], qf[k], b0, b1);
        }
      }
      // A block whose K scale is 0 has only zero codes: any factor gives its
      // scores, 0; 1 keeps a masked -inf from meeting 0.
      const float mul = sk > 0.f ? sk * p.scale_log2 : 1.f;
      const float lsv = sv > 0.f ? __log2f(sv) : kNoScale;
      const float isv = sv > 0.f ? __fdividef(1.f, sv) : 8589934592.f;  // 2^33
      const int key0 = at.tile * kKv8Block + warp * 16 + 2 * c;
      const bool edge = at.tile * kKv8Block + kKv8Block > min(len, p.causal ? len - p.q_len + 1 : len);
      if (edge) {
#pragma unroll
        for (int n8 = 0; n8 < 2; ++n8)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (key0 + n8 * 8 + (e & 1) >= lim[e >> 1]) s[n8][e] = -INFINITY;
        if constexpr (FMT == kKv8E4m3) {
          // What lies past the length may decode to NaN, and 0 * NaN is NaN.
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (key0 + (x & 1) + (x >> 1) * 8 >= len) {
#pragma unroll
              for (int k = 0; k < HD / 32; ++k) vw[x][k] = 0u;
            }
        }
      }
      bool grow = false;
      float top[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float mx = fmaxf(fmaxf(s[0][2 * x], s[0][2 * x + 1]), fmaxf(s[1][2 * x], s[1][2 * x + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        top[x] = fmaf(mx, mul, lsv);
        grow |= top[x] > m[x] + kRescale;
      }
      if (__any_sync(0xffffffffu, grow)) {
        // The maximum moves, and what is summed so far with it, only when it
        // would otherwise lag by more than 2^8 (fp16 holds p' up to 2^16).
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float mn = fmaxf(m[x], top[x]);
          const float f = mn == m[x] ? 1.f : ex2_approx(m[x] - mn);
          m[x] = mn;
          l[x] *= f;
#pragma unroll
          for (int j = 0; j < HD / 8; ++j) {
            acc[j][2 * x] *= f;
            acc[j][2 * x + 1] *= f;
          }
        }
      }
      uint32_t pf[4];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float off = lsv - (m[x] == -INFINITY ? 0.f : m[x]);
        float sum = 0.f;
#pragma unroll
        for (int n8 = 0; n8 < 2; ++n8) {
          const float a = ex2_approx(fmaf(s[n8][2 * x], mul, off));
          const float b = ex2_approx(fmaf(s[n8][2 * x + 1], mul, off));
          sum += a + b;
          pf[2 * n8 + x] = pack_half2(a, b);
        }
        l[x] = fmaf(sum, isv, l[x]);
      }
      // O' += P V: MMA j takes code j of every lane's run, so its columns are d = (HD / 8) n + j.
#pragma unroll
      for (int k = 0; k < HD / 32; ++k) {
        const uint32_t a0 = prmt(vw[0][k], vw[1][k], 0x5140u), a1 = prmt(vw[0][k], vw[1][k], 0x7362u);
        const uint32_t c0 = prmt(vw[2][k], vw[3][k], 0x5140u), c1 = prmt(vw[2][k], vw[3][k], 0x7362u);
        uint32_t lo0, lo1, lo2, lo3, hi0, hi1, hi2, hi3;
        kv8_to_half2<FMT>(a0, lo0, lo1);
        kv8_to_half2<FMT>(a1, lo2, lo3);
        kv8_to_half2<FMT>(c0, hi0, hi1);
        kv8_to_half2<FMT>(c1, hi2, hi3);
        mma_16816(acc[4 * k], pf, lo0, hi0);
        mma_16816(acc[4 * k + 1], pf, lo1, hi1);
        mma_16816(acc[4 * k + 2], pf, lo2, hi2);
        mma_16816(acc[4 * k + 3], pf, lo3, hi3);
      }
    }
    at = nx;

    // Join the four warps' parts: rows' maxima and sums first, then O'.
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
      if (c == 0) {
        stat[(warp * 16 + g + 8 * x) * 2] = m[x];
        stat[(warp * 16 + g + 8 * x) * 2 + 1] = l[x];
      }
    }
    sync();
    float* merge = reinterpret_cast<float*>(gbase + L::kMerge);
    // 16-byte unit f of row r is kept at unit f ^ mix(f, r), which spreads a
    // quarter warp's stores over the banks.
    auto unit = [](int r, int f) {
      const int mix = HD == 128 ? ((f >> 3) & 3) | ((r & 1) << 2) : ((f >> 3) & 1) | ((r & 1) << 1);
      return r * (HD / 4) + (f ^ mix);
    };
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = g + 8 * x;
      float mm = m[x];
#pragma unroll
      for (int w = 0; w < 4; ++w) mm = fmaxf(mm, stat[(w * 16 + r) * 2]);
      const float f = m[x] == mm ? 1.f : ex2_approx(m[x] - mm);
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int j = 0; j < HD / 8; j += 4) {
          const float4 v = make_float4(acc[j][2 * x + half] * f, acc[j + 1][2 * x + half] * f,
                                       acc[j + 2][2 * x + half] * f, acc[j + 3][2 * x + half] * f);
          const int f4 = ((2 * c + half) * (HD / 8) + j) / 4;
          reinterpret_cast<float4*>(merge)[warp * 16 * (HD / 4) + unit(r, f4)] = v;
        }
    }
    sync();
    const bool whole = count == seg.tiles;
    const long long line0 = u - count - seg.tile;  // the line's first tile
    float* slot = p.part + (2LL * blockIdx.x + (u - count == u0 ? 0 : 1)) * (16 * HD + 32);
    const int rows_here = min(16, p.rows - r0);
    auto store = [&](int r, int f4, float4 v, float inv) {
      const int row = r0 + r;
      const int tok = row / p.group;
      const int head = kvh * p.group + row % p.group;
      *reinterpret_cast<uint2*>(p.o + seg.b * p.o_batch + tok * p.o_tok + head * p.o_head + f4 * 4) =
          make_uint2(pack_half2(v.x * inv, v.y * inv), pack_half2(v.z * inv, v.w * inv));
    };
    // A row without keys has m' = -inf and l = 0 and becomes 0; one with NaN scores has l = NaN.
    auto inverse = [](float mm, float ll) { return mm == -INFINITY && ll == ll ? 0.f : 1.f / ll; };
    if (ok) {
      for (int e = threadIdx.x; e < rows_here * (HD / 4); e += kConsumers) {
        const int r = e / (HD / 4), f4 = e % (HD / 4);
        float mm = -INFINITY, ll = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) mm = fmaxf(mm, stat[(w * 16 + r) * 2]);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float mw = stat[(w * 16 + r) * 2];
          ll += stat[(w * 16 + r) * 2 + 1] * (mw == mm ? 1.f : ex2_approx(mw - mm));
          const float4 o = reinterpret_cast<const float4*>(merge)[w * 16 * (HD / 4) + unit(r, f4)];
          v = make_float4(v.x + o.x, v.y + o.y, v.z + o.z, v.w + o.w);
        }
        if (whole) {
          store(r, f4, v, inverse(mm, ll));
        } else {
          reinterpret_cast<float4*>(slot + 32)[r * (HD / 4) + f4] = v;
          if (f4 == 0) {
            slot[r] = mm;
            slot[16 + r] = ll;
          }
        }
      }
    }
    if (!whole) {
      // Count in; the last part of the line joins them all, in CTA order.
      __threadfence();
      sync();
      const long long first = owner(line0), last = owner(line0 + seg.tiles - 1);
      unsigned* count_at = p.count + static_cast<long long>(seg.b) * lines + seg.hr;
      if (threadIdx.x == 0) {
        const unsigned n = static_cast<unsigned>(last - first + 1);
        const unsigned before = ok ? atomicAdd(count_at, 1u) : 0u;
        *last_flag = ok && before == n - 1 ? 1u : 0u;
        if (ok && before == n - 1) *count_at = 0u;  // ready for the next launch
      }
      sync();
      if (*last_flag != 0u) {
        __threadfence();
        for (int e = threadIdx.x; e < rows_here * (HD / 4); e += kConsumers) {
          const int r = e / (HD / 4), f4 = e % (HD / 4);
          float mm = -INFINITY, ll = 0.f;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
          for (long long k = first; k <= last; ++k) {
            // A part that does not start its CTA's share can only be the first.
            const float* part = p.part + (2 * k + (k == first && share_begin(k) != line0 ? 1 : 0)) * (16 * HD + 32);
            const float pm = __ldcg(part + r), pl = __ldcg(part + 16 + r);
            const float4 o = __ldcg(reinterpret_cast<const float4*>(part + 32) + r * (HD / 4) + f4);
            const float mn = fmaxf(mm, pm);
            const float fo = mm == mn ? 1.f : ex2_approx(mm - mn);
            const float fn = pm == mn ? 1.f : ex2_approx(pm - mn);
            mm = mn;
            ll = ll * fo + pl * fn;
            v = make_float4(v.x * fo + o.x * fn, v.y * fo + o.y * fn, v.z * fo + o.z * fn, v.w * fo + o.w * fn);
          }
          store(r, f4, v, inverse(mm, ll));
        }
      }
    }
    sync();  // merge and stat are free again
  }
}

template <int FMT, int HD>
cudaError_t launch_hd(const CUtensorMap& tk, const CUtensorMap& tv, const Kv8AttnParams& p, int grid, int dev,
                      cudaStream_t stream) {
  static std::atomic<uint64_t> configured{0};
  const uint64_t bit = 1ull << (dev & 63);
  auto kernel = kv8_rows_sm100_kernel<FMT, HD>;
  if ((configured.load(std::memory_order_acquire) & bit) == 0) {
    const cudaError_t e =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, RowsSmem<HD>::kBytes);
    if (e != cudaSuccess) return e;
    configured.fetch_or(bit, std::memory_order_acq_rel);
  }
  kernel<<<grid, kThreads, RowsSmem<HD>::kBytes, stream>>>(tk, tv, p);
  return cudaGetLastError();
}

}  // namespace

// Two CTAs per SM, but none without a tile when every sequence is as long as it can be.
int kv8_rows_grid(const Kv8AttnParams& p, int sms) {
  const long long tiles = static_cast<long long>(p.batch) * p.kv_heads * p.row_tiles *
                          ((p.kv_len + kKv8Block - 1) / kKv8Block);
  const long long most = static_cast<long long>(kCtasPerSm) * sms;
  return static_cast<int>(tiles < most ? (tiles > 0 ? tiles : 1) : most);
}
size_t kv8_rows_part_floats(int head_dim, int grid) { return 2 * static_cast<size_t>(grid) * (16 * head_dim + 32); }

cudaError_t launch_kv8_rows(const CUtensorMap& tk, const CUtensorMap& tv, const Kv8AttnParams& p, int grid, int dev,
                            cudaStream_t stream) {
  if (p.format == kKv8Int8)
    return p.head_dim == 128 ? launch_hd<kKv8Int8, 128>(tk, tv, p, grid, dev, stream)
                             : launch_hd<kKv8Int8, 64>(tk, tv, p, grid, dev, stream);
  return p.head_dim == 128 ? launch_hd<kKv8E4m3, 128>(tk, tv, p, grid, dev, stream)
                           : launch_hd<kKv8E4m3, 64>(tk, tv, p, grid, dev, stream);
}

}  // namespace ax
