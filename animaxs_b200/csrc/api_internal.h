// api_internal.h -- context layout and helpers shared by the C-ABI translation units.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <string>
#include <vector>

#include "../../include/animaxs_attn.h"
#include <nvtx3/nvToolsExt.h>

// NVTX range around a C ABI call (header-only NVTX v3: a no-op unless a
// profiler injects itself), so a capture can attribute kernels to the call.
struct AxRange {
  explicit AxRange(const char* name) { nvtxRangePushA(name); }
  ~AxRange() { nvtxRangePop(); }
  AxRange(const AxRange&) = delete;
  AxRange& operator=(const AxRange&) = delete;
};

// A device buffer of the context that grows on demand (ax_grow_buffer).
struct AxBuffer {
  void* ptr = nullptr;
  size_t bytes = 0;
  bool captured = false;  // a call in stream capture used it: a graph may hold its address
};

struct animaxs_attn_ctx {
  int device = 0;
  int num_sms = 0;
  AxBuffer scratch;               // normalised q/k copies, decoded weights, re-laid RoPE tables
  AxBuffer staging;               // head-sharded path: per-rank slice + gather buffer
  std::vector<void*> retired;     // outgrown buffers that captured graphs may point at
  // Workspaces of split 8-bit-cache attention, each made at its first use as large
  // as any call on this device needs and never moved: captured graphs point at them.
  float* kv8_rows_part = nullptr;      // few rows: partial results
  unsigned int* kv8_count = nullptr;   // few rows: arrivals [num_sms], zero between calls
  float* kv8_tile_part = nullptr;      // many rows: partial results
  unsigned int* d_status = nullptr;  // device status word written by kernels
  int64_t query_tiles = 0;
  bool timing = false;                        // bracket each attention kernel with events
  unsigned int* score_probe = nullptr;        // device uint32[4] probe slot, or nullptr
  std::vector<cudaEvent_t> events;            // pool: pairs (start, stop)
  size_t events_used = 0;                     // events recorded since the last read
  std::string last_error;
};

// Output redirection for the head-sharded path: query head h is written at
// ptr + (h - head_base) * head.
struct AxOutView {
  void* ptr;
  int64_t tok, head, batch;
  int head_base;
};

int ax_set_error(animaxs_attn_ctx* ctx, int code, const char* fmt, ...);
int ax_cuda_fail(animaxs_attn_ctx* ctx, cudaError_t e, const char* what);
// At least `bytes` in `buffer` for a call on `stream`; an outgrown buffer that a graph may
// hold lives until the context is destroyed.
int ax_grow_buffer(animaxs_attn_ctx* ctx, AxBuffer* buffer, size_t bytes, cudaStream_t stream, const char* what);
int ax_ensure_scratch(animaxs_attn_ctx* ctx, size_t bytes, cudaStream_t stream);
// While kernel timing is on: records the start of a launch on `stream` and gives the event
// that ax_timing_end records behind it (nullptr while it is off).
int ax_timing_begin(animaxs_attn_ctx* ctx, cudaStream_t stream, cudaEvent_t* stop);
void ax_timing_end(animaxs_attn_ctx* ctx, cudaStream_t stream, cudaEvent_t stop);
int ax_validate(animaxs_attn_ctx* ctx, const animaxs_attn_desc* d, const void* q, const void* k,
                const void* v, const void* o);
int ax_make_tmap(animaxs_attn_ctx* ctx, CUtensorMap* map, const void* base, int64_t dim, int64_t rows,
                 int64_t heads, int64_t batch, int64_t st, int64_t sh, int64_t sb, int box_rows = 128);
// [heads][rows][dim] bytes, packed (dim 64 or 128); box = dim bytes x box_rows rows,
// swizzled by the row length (64 or 128 bytes).
int ax_make_tmap_codes(animaxs_attn_ctx* ctx, CUtensorMap* map, const void* base, int64_t dim, int64_t rows,
                       int64_t heads, int box_rows);
// fp16 q or o as [batch][lines][tokens][pack][dim], pack a power of two <= 128;
// box = 64 columns x box_rows rows (of up to box_rows heads), 128B swizzle.
int ax_make_tmap_rows(animaxs_attn_ctx* ctx, CUtensorMap* map, const void* base, int64_t dim, int64_t pack,
                      int64_t tokens, int64_t lines, int64_t batch, int64_t st, int64_t sh, int64_t sb, int box_rows);
// Peers of a fused head-sharded call: the epilogue stores every output tile
// also at o + delta[i] and the CTAs count their items on arrive[i].
struct AxPeers {
  int n;
  long long delta[7];
  unsigned int* arrive[7];
  const unsigned int* go;  // the stores and arrivals happen only if *go == go_value
  unsigned int go_value;
};
int ax_forward_range(animaxs_attn_ctx* ctx, const animaxs_attn_desc* d, const void* q,
                     const void* k, const void* v, void* o, int heads_begin, int heads_count,
                     const AxOutView* o_view, cudaStream_t stream, const AxPeers* peers = nullptr);
