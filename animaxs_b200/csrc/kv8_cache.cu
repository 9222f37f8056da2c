// kv8_cache.cu -- writing the 8-bit K/V cache and reading it back
// (animaxs_kv8_write, animaxs_kv8_read in include/animaxs_attn.h).
//
// Both are streams: 2 bytes in and 1 out per value (write), 1 in and 2 out
// (read), so HBM bounds them when there is enough to move and the latency of
// one dependent chain (positions -> rows -> maximum -> codes) when there is not.
//
// Measured (GPU time of a call in a graph, bytes moved over it; a copy reaches
// 6.54 TB/s): write of 1 token x 8 heads x 8 sequences 2.4 us, of 8 x 512 tokens
// x 16 heads 10.1 us = 4.98 TB/s, of 2 x up to 16385 tokens x 8 heads 20.1 us =
// 5.98 TB/s; read of 32741 tokens x 8 heads 32.8 us = 6.13 TB/s.  The middle
// sizes are a few waves of short CTAs, whose start and end are not hidden.
// Threads a CTA: 64 and 256 wrote the second in 12.6 and 10.7 us, 128 and 512 read
// the last in 33.7 and 38.7.
#include "kernels.h"
#include "kv8_common.cuh"
#include "sm100_ptx.cuh"

namespace ax {
namespace {

constexpr int kWriteThreads = 128;

__device__ __forceinline__ __half2 as_half2(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }

// The magnitudes of a pair, 0 in place of what is not finite.
__device__ __forceinline__ __half2 finite_abs(uint32_t w) {
  const __half2 a = __habs2(as_half2(w));
  const __half2 inf = __halves2half2(__ushort_as_half(0x7C00), __ushort_as_half(0x7C00));
  return as_half2(__hlt2_mask(a, inf) & as_u32(a));  // NaN compares false
}
// A pair with 0 in place of NaN.
__device__ __forceinline__ uint32_t nan_to_zero(uint32_t w) { return __heq2_mask(as_half2(w), as_half2(w)) & w; }

// Four values to codes.  kFinite: all of them are finite, so that none is
// beyond +-M after the scaling (a * (1 / (a / M)) rounds to M) and none is NaN.
template <int FMT, bool kFinite>
__device__ __forceinline__ uint32_t quantise4(uint32_t a, uint32_t b, float inv) {
  if constexpr (!kFinite) {
    a = nan_to_zero(a);
    b = nan_to_zero(b);
  }
  float2 x = __half22float2(as_half2(a)), y = __half22float2(as_half2(b));
  // The product is rounded before it is rounded to an integer: a packed
  // multiply would be contracted with the packed addition below, .rn or not.
  x = make_float2(__fmul_rn(x.x, inv), __fmul_rn(x.y, inv));
  y = make_float2(__fmul_rn(y.x, inv), __fmul_rn(y.y, inv));
  if constexpr (FMT == kKv8Int8 && kFinite) {
    constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: the sum's low mantissa bits are the rounded integer
    const float2 k2 = make_float2(kMagic, kMagic), p = add2(x, k2), q = add2(y, k2);
    return prmt(prmt(__float_as_uint(p.x), __float_as_uint(p.y), 0x0040u),
                prmt(__float_as_uint(q.x), __float_as_uint(q.y), 0x0040u), 0x5410u);
  } else {
    return kv8_pack4<FMT>(x.x, x.y, y.x, y.y);
  }
}

// One CTA per (64-token block, head, sequence, K or V): it alone reads and
// writes that block's codes and scale.  A thread keeps its 8-value shares of
// all the block's rows in registers between the maximum and the rounding, so
// the source is read once.
template <int FMT, int HD>
__global__ void __launch_bounds__(kWriteThreads) kv8_write_kernel(const Kv8WriteParams p, int window) {
  constexpr int kLanes = HD / 8;                       // threads per row
  constexpr int kRowsPerPass = kWriteThreads / kLanes;
  constexpr int kPasses = kKv8Block / kRowsPerPass;
  __shared__ float warp_max[kWriteThreads / 32];
  pdl_start();
  int w = blockIdx.x;
  const int kv = w & 1;
  w >>= 1;
  const int h = w % p.kv_heads;
  w /= p.kv_heads;
  const int b = w / window;
  const int wi = w % window;
  pdl_wait();
  const long long start = p.starts != nullptr ? p.starts[b] : p.start;
  const int n = p.counts != nullptr ? min(max(p.counts[b], 0), p.tokens) : p.tokens;
  const long long first = start > 0 ? start : 0;                               // first written position
  const long long end = start + n < p.capacity ? start + n : p.capacity;       // one past the last
  const long long blk0 = (first / kKv8Block + wi) * kKv8Block;                 // this block's first position
  const int lo = static_cast<int>(max(first - blk0, 0LL));                     // rows [lo, hi) are new
  const int hi = static_cast<int>(min(end - blk0, static_cast<long long>(kKv8Block)));
  if (lo >= hi) return;
  const int lane = threadIdx.x % kLanes;
  const int row0 = threadIdx.x / kLanes;
  const long long bh = static_cast<long long>(b) * p.kv_heads + h;
  const int n_blocks = (p.capacity + kKv8Block - 1) / kKv8Block;
  float* scale = p.scale[kv] + bh * n_blocks + blk0 / kKv8Block;
  uint8_t* codes = p.codes[kv] + (bh * p.capacity + blk0) * HD + lane * 8;
  const __half* src = p.src[kv] + b * p.bat[kv] + h * p.head[kv] + (blk0 - start) * p.tok[kv] + lane * 8;
  const float before = lo > 0 ? *scale : 0.f;
  uint4 x[kPasses];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int r = row0 + i * kRowsPerPass;
    if (r >= lo && r < hi) x[i] = *reinterpret_cast<const uint4*>(src + r * p.tok[kv]);
  }
  // Largest magnitude; NaN and infinity show in it and send the thread to the
  // slower form (most of the kernel's instructions are per value, and it is
  // bound by them: 512 tokens x 16 heads x 8 prompts 13.0 us with the checks
  // on every value).
  const __half2 none = __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
  __half2 mx = none;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int r = row0 + i * kRowsPerPass;
    if (r >= lo && r < hi)
      mx = __hmax2_nan(mx, __hmax2_nan(__hmax2_nan(__habs2(as_half2(x[i].x)), __habs2(as_half2(x[i].y))),
                                       __hmax2_nan(__habs2(as_half2(x[i].z)), __habs2(as_half2(x[i].w)))));
  }
  const bool finite = __hlt(__low2half(mx), __ushort_as_half(0x7C00)) && __hlt(__high2half(mx), __ushort_as_half(0x7C00));
  if (!finite) {
    mx = none;
#pragma unroll 1
    for (int i = 0; i < kPasses; ++i) {
      const int r = row0 + i * kRowsPerPass;
      if (r >= lo && r < hi) {
        const uint4 v = *reinterpret_cast<const uint4*>(src + r * p.tok[kv]);
        mx = __hmax2(mx, __hmax2(__hmax2(finite_abs(v.x), finite_abs(v.y)), __hmax2(finite_abs(v.z), finite_abs(v.w))));
      }
    }
  }
  float a = fmaxf(__low2float(mx), __high2float(mx));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
  if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = a;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWriteThreads / 32; ++i) a = fmaxf(a, warp_max[i]);
  const float s = fmaxf(__fmul_rn(a, 1.f / kKv8Top<FMT>), before);
  // A scale that a caller put there may be so small that 1 / s overflows; only values of
  // 0 meet it, whose codes are 0.
  const float inv = s > 0.f ? fminf(__fdiv_rn(1.f, s), 3.402823466e38f) : 0.f;
  if (finite) {
    // With a scale of 0 every finite value is 0, and 0 * 0 rounds to code 0.
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int r = row0 + i * kRowsPerPass;
      if (r >= lo && r < hi)
        *reinterpret_cast<uint2*>(codes + static_cast<long long>(r) * HD) =
            make_uint2(quantise4<FMT, true>(x[i].x, x[i].y, inv), quantise4<FMT, true>(x[i].z, x[i].w, inv));
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < kPasses; ++i) {
      const int r = row0 + i * kRowsPerPass;
      if (r >= lo && r < hi) {
        const uint4 v = *reinterpret_cast<const uint4*>(src + r * p.tok[kv]);
        uint2 c = make_uint2(0u, 0u);
        if (inv > 0.f) c = make_uint2(quantise4<FMT, false>(v.x, v.y, inv), quantise4<FMT, false>(v.z, v.w, inv));
        *reinterpret_cast<uint2*>(codes + static_cast<long long>(r) * HD) = c;
      }
    }
  }
  if (threadIdx.x == 0) *scale = s;
  if (lo > 0 && s > before) {
    // Older tokens of the block under the larger scale.
    const float f = __fmul_rn(before, inv);
    for (int r = row0; r < lo; r += kRowsPerPass) {
      uint2* at = reinterpret_cast<uint2*>(codes + static_cast<long long>(r) * HD);
      uint2 c = *at;
      uint32_t* word[2] = {&c.x, &c.y};
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t l, u;
        kv8_to_half2<FMT>(*word[k], l, u);
        const float2 fl = __half22float2(*reinterpret_cast<const __half2*>(&l));
        const float2 fu = __half22float2(*reinterpret_cast<const __half2*>(&u));
        *word[k] = kv8_pack4<FMT>(__fmul_rn(fl.x, f), __fmul_rn(fl.y, f), __fmul_rn(fu.x, f), __fmul_rn(fu.y, f));
      }
      *at = c;
    }
  }
}

constexpr int kReadThreads = 256;

// One CTA per (64 positions, head, sequence, K or V); a thread turns 8 codes
// into 16 bytes, several rows in flight.
template <int FMT, int HD>
__global__ void __launch_bounds__(kReadThreads) kv8_read_kernel(const Kv8ReadParams p, int chunks) {
  constexpr int kLanes = HD / 8;
  constexpr int kRowsPerPass = kReadThreads / kLanes;
  constexpr int kPasses = kKv8Block / kRowsPerPass;
  pdl_start();
  int w = blockIdx.x;
  const int kv = w & 1;
  w >>= 1;
  const int h = w % p.kv_heads;
  w /= p.kv_heads;
  const int b = w / chunks;
  const int t0 = w % chunks * kKv8Block;
  pdl_wait();
  const int len = p.lens != nullptr ? p.lens[b] : p.capacity;
  const int lane = threadIdx.x % kLanes;
  const long long bh = static_cast<long long>(b) * p.kv_heads + h;
  const int n_blocks = (p.capacity + kKv8Block - 1) / kKv8Block;
  const float* scale = (kv ? p.scale[1] : p.scale[0]) + bh * n_blocks;
  const uint8_t* codes = (kv ? p.codes[1] : p.codes[0]) + bh * p.capacity * HD + lane * 8;
  __half* out = (kv ? p.out[1] : p.out[0]) + b * p.bat + h * p.head + lane * 8;
  uint2 c[kPasses];
  float s[kPasses];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int t = t0 + threadIdx.x / kLanes + i * kRowsPerPass;
    const int pos = p.start + t;
    c[i] = make_uint2(0u, 0u);
    s[i] = 0.f;
    if (t < p.tokens && pos < len) {
      c[i] = *reinterpret_cast<const uint2*>(codes + static_cast<long long>(pos) * HD);
      s[i] = scale[pos / kKv8Block];
    }
  }
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int t = t0 + threadIdx.x / kLanes + i * kRowsPerPass;
    if (t < p.tokens) {
      uint32_t r[4];
      const uint32_t word[2] = {c[i].x, c[i].y};
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t l, u;
        kv8_to_half2<FMT>(word[k], l, u);
        const float2 fl = __half22float2(*reinterpret_cast<const __half2*>(&l));
        const float2 fu = __half22float2(*reinterpret_cast<const __half2*>(&u));
        const __half2 hl = __floats2half2_rn(fl.x * s[i], fl.y * s[i]);
        const __half2 hu = __floats2half2_rn(fu.x * s[i], fu.y * s[i]);
        r[2 * k] = *reinterpret_cast<const uint32_t*>(&hl);
        r[2 * k + 1] = *reinterpret_cast<const uint32_t*>(&hu);
      }
      *reinterpret_cast<uint4*>(out + static_cast<long long>(t) * p.tok) = make_uint4(r[0], r[1], r[2], r[3]);
    }
  }
}

}  // namespace

cudaError_t launch_kv8_write(const Kv8WriteParams& p, cudaStream_t stream) {
  const int window = static_cast<int>(kv8_write_window(p.tokens, p.capacity));
  const long long ctas = 2LL * window * p.batch * p.kv_heads;
  if (ctas > 0x7fffffffLL) return cudaErrorInvalidValue;
  auto kernel = p.format == kKv8Int8
                    ? (p.head_dim == 128 ? kv8_write_kernel<kKv8Int8, 128> : kv8_write_kernel<kKv8Int8, 64>)
                    : (p.head_dim == 128 ? kv8_write_kernel<kKv8E4m3, 128> : kv8_write_kernel<kKv8E4m3, 64>);
  return launch_pdl(kernel, static_cast<unsigned>(ctas), kWriteThreads, 0, stream, p, window);
}

cudaError_t launch_kv8_read(const Kv8ReadParams& p, cudaStream_t stream) {
  const int chunks = static_cast<int>((p.tokens + kKv8Block - 1LL) / kKv8Block);
  const long long ctas = 2LL * chunks * p.batch * p.kv_heads;
  if (ctas > 0x7fffffffLL) return cudaErrorInvalidValue;
  auto kernel = p.format == kKv8Int8
                    ? (p.head_dim == 128 ? kv8_read_kernel<kKv8Int8, 128> : kv8_read_kernel<kKv8Int8, 64>)
                    : (p.head_dim == 128 ? kv8_read_kernel<kKv8E4m3, 128> : kv8_read_kernel<kKv8E4m3, 64>);
  return launch_pdl(kernel, static_cast<unsigned>(ctas), kReadThreads, 0, stream, p, chunks);
}

}  // namespace ax
