// kv8_common.cuh -- codes of the 8-bit K/V cache: quantising, and conversion to
// fp16 pairs (exact for both formats: int8 has 7 bits, e4m3 has 4, fp16 has 11).
#pragma once

#include <cuda_fp16.h>

#include <cstdint>
#include <utility>

#include "../../include/animaxs_attn.h"

namespace ax {

constexpr int kKv8Int8 = ANIMAXS_KV8_INT8;
constexpr int kKv8E4m3 = ANIMAXS_KV8_E4M3;
template <int FMT>
constexpr float kKv8Top = FMT == kKv8Int8 ? 127.f : 448.f;

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  return __byte_perm(a, b, sel);
}

// A V scale up to this stands for 0: its values vanish in an fp16 output, while the
// weights of its keys have to count, and 1 / scale and the probabilities scaled by
// it would leave the range of fp32.
constexpr float kKv8NoValue = 8.27180613e-25f;  // 2^-80
// Stands for log2 of such a scale (below that of any written block, 2^-33).
constexpr float kKv8NoScale = -33.f;
constexpr float kKv8NoScaleInverse = 8589934592.f;  // 2^33

// Four codes (one per byte of w) -> half2 of bytes 0, 1 and half2 of bytes 2, 3.
// int8: code + 128 is placed under the exponent of 1024 (0x64xx = 1024 + xx)
// and 1152 is subtracted, all exact: 1.25 instructions a value.
// e4m3: the hardware conversion of two codes.
template <int FMT>
__device__ __forceinline__ void kv8_to_half2(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (FMT == kKv8Int8) {
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
    uint32_t a = prmt(u, 0x64646464u, 0x4140u), b = prmt(u, 0x64646464u, 0x4342u);
    const __half2 ha = __hsub2(*reinterpret_cast<__half2*>(&a), off);
    const __half2 hb = __hsub2(*reinterpret_cast<__half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&ha);
    hi = *reinterpret_cast<const uint32_t*>(&hb);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\t"
        "mov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
}

// Four fp32 values -> four codes.  Values are already x * (1 / scale).
template <int FMT>
__device__ __forceinline__ uint32_t kv8_pack4(float a, float b, float c, float d) {
  if constexpr (FMT == kKv8Int8) {
    // Clamp, then round to nearest even: adding 1.5 * 2^23 leaves the integer in
    // the low mantissa bits.
    constexpr float kMagic = 12582912.0f;
    const uint32_t ia = __float_as_uint(__fadd_rn(fminf(fmaxf(a, -127.f), 127.f), kMagic));
    const uint32_t ib = __float_as_uint(__fadd_rn(fminf(fmaxf(b, -127.f), 127.f), kMagic));
    const uint32_t ic = __float_as_uint(__fadd_rn(fminf(fmaxf(c, -127.f), 127.f), kMagic));
    const uint32_t id = __float_as_uint(__fadd_rn(fminf(fmaxf(d, -127.f), 127.f), kMagic));
    return prmt(prmt(ia, ib, 0x0040u), prmt(ic, id, 0x0040u), 0x5410u);
  } else {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
        "mov.b32 %0, {l, h};\n\t}"
        : "=r"(r)
        : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
  }
}

// Programmatic dependent launch: the kernels of the cache follow one another
// (a step writes, then attends), so each may be set up while the one before it
// ends.  pdl_wait() returns when that one has completed and its writes are
// visible; nothing of global memory is touched before it.  What a predecessor may
// have written (lengths, scales, codes, q, k, v, partial results) is read by
// ordinary loads: the non-coherent ones (__ldg) are for data that nobody writes
// while the kernel is resident, and may be moved across the wait.
__device__ __forceinline__ void pdl_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... Params, typename... Args>
cudaError_t launch_pdl_cluster(void (*kernel)(Params...), unsigned grid, unsigned cluster, unsigned threads,
                               size_t smem, cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}
template <typename... Params, typename... Args>
cudaError_t launch_pdl(void (*kernel)(Params...), unsigned grid, unsigned threads, size_t smem, cudaStream_t stream,
                       Args&&... args) {
  return launch_pdl_cluster(kernel, grid, 1, threads, smem, stream, std::forward<Args>(args)...);
}

// A sequence's length, within [0, kv_len].
__device__ __forceinline__ int kv8_len(const int* lens, int kv_valid, int kv_len, int b) {
  const int n = lens != nullptr ? lens[b] : kv_valid;
  return min(max(n, 0), kv_len);
}

}  // namespace ax
