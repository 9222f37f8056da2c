// kernels.h -- host-side launch interface of the CUDA kernels (internal to the library).
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace ax {

// Parameters of the flash-attention kernels (attn_fwd_sm100.cu, attn_wide_sm100.cu).  q/k/v arrive
// through TMA tensor maps over [batch][head][token][head_dim] fp16 views (any
// strides); the output leaves through TMA tensor stores from a shared-memory
// stage (the launchers build its tensor map from `o` and the strides below).
struct AttnFwdParams {
  int head_dim;          // 64 or 128 (attn_fwd_sm100.cu), 256 or 384 (attn_wide_sm100.cu)
  int q_len;
  int kv_len;
  int heads_per_kv;      // heads / kv_heads (GQA group size)
  int kv_valid;          // keys >= kv_valid masked (already clamped to [1, kv_len])
  const int* kv_valid_dev;  // optional per-batch override (device)
  int causal;
  int n_q_tiles;         // query tiles per head: pairs or single 128-row tiles (head dims 64 / 128,
                         // chosen by launch_attn_fwd), 128-row tiles (wide)
  int single_tiles;      // set by launch_attn_fwd (head dims 64 / 128): items are single 128-row tiles
  int head_offset;       // first query head handled by this launch
  int heads_in_launch;   // set by launch_attn_fwd: query heads of this launch
  int n_items;           // set by launch_attn_fwd: n_q_tiles * heads_in_launch * batch
  int n_split;           // set by the wide launcher: CTAs (one cluster) sharing a query tile's keys
  int o_head_base;       // output head index = h - o_head_base
  float scale_log2;      // softmax scale * log2(e)
  __half* o;
  long long o_tok, o_head, o_batch;  // output strides (elements)
  unsigned int* status;  // device status word (bit 0: a bounded wait timed out)
  unsigned int* probe;   // score-health slot uint32[4] (animaxs_attn_set_score_probe) or nullptr
  int fp32_p;            // FP32_SCORES_AND_SOFTMAX: P x V from fp32 P (hi + lo fp16 terms)
  // Fused head-sharded gather (head dims 64 / 128; n_peers = 0 otherwise): the
  // epilogue also stores every output tile at the same offset in each peer's
  // output (peer GPU memory mapped into this process), and each CTA that
  // finished without a timeout adds its item count to every peer's arrival
  // word for this rank.
  int n_peers;
  long long peer_delta[7];           // bytes from `o` to the peer's copy of it
  unsigned int* peer_arrive[7];      // the peer's arrival word for this rank
  // The peer stores and arrivals happen only if *peer_go == peer_go_value:
  // the handshake before the call writes it when every peer was ready.
  const unsigned int* peer_go;
  unsigned int peer_go_value;
};

constexpr int kMaxPeers = 7;  // 8 GPUs per node

constexpr unsigned int kStatusTimeoutBit = 1u;  // a bounded device wait expired

constexpr int kTileM = 128;   // query rows per CTA
constexpr int kTileN = 128;   // keys per K/V tile
constexpr int kHeadDim = 128;   // DiT / Qwen; the LLM adapter runs 64

// One normalisation job: a [batch][tokens][heads][head_dim] fp16 tensor with strides.
struct NormJob {
  const __half* in;
  __half* out;
  long long in_tok, in_head, in_batch;
  long long out_tok, out_head, out_batch;
  int tokens, heads, batch;
  const __half* weight;  // shared [128] weight or nullptr (ones)
  long long rows;        // batch * tokens * heads
};

struct NormParams {
  NormJob job[2];
  int njobs;
  int head_dim;          // 64 or 128
  float eps;
  const float* rope;     // [tokens][head_dim/2][2][2] or nullptr (no rotation)
  unsigned int* status;  // device status word (nullable)

};

cudaError_t launch_attn_fwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                            const AttnFwdParams& p, int heads_in_launch, int batch,
                            cudaStream_t stream);

// Head dim 64 / 128, one query tile per item with three score buffers in TMEM
// (attn_s3_sm100.cu; called by launch_attn_fwd).
cudaError_t launch_attn_s3(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                           const AttnFwdParams& p, int heads_in_launch, int batch, int dev, int sms,
                           cudaStream_t stream);

// Head dims 256 / 384 (called by launch_attn_fwd).
cudaError_t launch_attn_wide(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                             const AttnFwdParams& p, int heads_in_launch, int batch, int dev,
                             cudaStream_t stream);

int attn_fwd_rows_per_cta();  // query rows of a paired work item (head dims 64 / 128)
// Work items launch_attn_fwd deals for head dims 64 / 128 (pairs of query
// tiles, or single tiles when pairs would leave more than half of `sms` idle,
// or, for a launch with peer stores, any of them idle).
long long attn_fwd_work_items(int q_len, int heads_in_launch, int batch, int sms, bool peers);

cudaError_t launch_qk_norm(NormParams p, cudaStream_t stream);

// Peer handshake of the fused head-sharded path (peer_sync.cu): one block adds
// `add` to each peer's word `signal[i]` (release, system scope), then waits
// until every own word `wait[i]` (i != rank) has reached `target` (acquire,
// system scope; bounded by timeout_ns, after which kStatusTimeoutBit is set)
// and, if no wait gave up, writes `go_value` to `go`.
struct PeerSyncParams {
  unsigned int* signal[8];   // peers' words for this rank (mapped here); nullptr: no signal
  unsigned int add;
  const unsigned int* wait;  // this rank's [world] words
  unsigned int target;
  int world, rank;
  unsigned long long timeout_ns;
  unsigned int* status;
  unsigned int* go;          // set to go_value when every wait succeeded (nullptr: not written)
  unsigned int go_value;
};
cudaError_t launch_peer_sync(const PeerSyncParams& p, cudaStream_t stream);

// Fused attention projections (proj_sm100.cu): out = x w^T over fp16 operands
// with fp32 accumulation, then one of three epilogues.
enum ProjMode : int {
  kProjStore = 0,    // out fp16 = fp16(acc)
  kProjQkvNorm = 1,  // q / k column ranges: per-128-column-head RMSNorm (+ split-half RoPE)
  kProjGateAdd = 2,  // residual fp32 += float(fp16(acc)) * gate[row / tokens][col]
};
struct ProjParams {
  int m, n, k;
  int tokens;               // rows per image (RoPE row = row % tokens, gate row = row / tokens)
  int mode;                 // ProjMode
  int q_cols, k_cols;       // kProjQkvNorm: [0, q_cols) q heads, [q_cols, q_cols + k_cols) k heads
  const __half* q_w;        // kProjQkvNorm: shared [128] norm weights, or nullptr (ones)
  const __half* k_w;
  const float* rope;        // pair-major [64][tokens] (cos, sin) float2 (launch_rope_pairs), or nullptr
  float eps;
  const float* gate;        // kProjGateAdd: [images][gate_stride] fp32
  long long gate_stride;
  int tiles_n;              // ceil(n / 256)
  int tiles;                // ceil(m / 256) * tiles_n (256 x 256 tiles, one per CTA pair)
  unsigned int* status;
};
cudaError_t launch_proj(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tout,
                        const ProjParams& p, cudaStream_t stream);
int proj_kernel_attributes(int* regs, int* max_threads, int* smem_static, int* smem_dynamic_max);
// [rows][64][2][2] table blocks -> [64][rows] (cos, sin) pairs in `out` (rows*512 bytes).
cudaError_t launch_rope_pairs(const float* table, void* out, int rows, cudaStream_t stream);

// ---- 8-bit K/V cache (kv8_cache.cu, kv8_rows_sm100.cu) ----
constexpr int kKv8Block = 64;  // tokens that share a scale

struct Kv8WriteParams {
  int format, head_dim, batch, kv_heads, capacity, tokens, start;
  const int* starts;  // per sequence, or nullptr
  const int* counts;
  const __half* src[2];  // k, v
  long long tok[2], head[2], bat[2];
  uint8_t* codes[2];
  float* scale[2];
};
// 64-token blocks of a head that `tokens` tokens from any start can touch.
inline long long kv8_write_window(long long tokens, long long capacity) {
  const long long window = (tokens + kKv8Block - 2) / kKv8Block + 1, all = (capacity + kKv8Block - 1) / kKv8Block;
  return window < all ? window : all;
}
cudaError_t launch_kv8_write(const Kv8WriteParams& p, cudaStream_t stream);

struct Kv8ReadParams {
  int format, head_dim, batch, kv_heads, capacity, start, tokens;
  const int* lens;  // per sequence, or nullptr
  const uint8_t* codes[2];
  const float* scale[2];
  __half* out[2];
  long long tok, head, bat;
};
cudaError_t launch_kv8_read(const Kv8ReadParams& p, cudaStream_t stream);

struct Kv8AttnParams {
  int format, head_dim, batch, kv_heads, group;  // group = query heads per kv head
  int q_len, kv_len, capacity, n_blocks;         // n_blocks = scales per head
  int kv_valid;                                  // length of every sequence without lens
  const int* lens;                               // DEVICE per-sequence lengths, or nullptr
  int causal;
  float scale_log2;
  const __half* q;
  long long q_tok, q_head, q_batch;
  __half* o;
  long long o_tok, o_head, o_batch;
  const float* k_scale;
  const float* v_scale;
  int rows;             // group * q_len: query rows of a kv head
  // Few rows (kv8_rows_plan): each line to a cluster of its own, of 2^cluster_log2
  // CTAs; floor(65536 / group) + 1, which divides the row numbers.
  bool alone;
  int cluster_log2, group_inv;
  float* part;          // workspace: partial results (kv8_rows_part_floats, kv8_attn_part_floats)
  unsigned int* count;  // arrivals at a line that crosses CTAs, by the CTA it starts in; zero between launches
  unsigned int* status;
  // Many rows (kv8_attn_plan): heads of a row line, row lines per sequence,
  // pairs of query tiles per line, pairs in all, key blocks of kv_len, CTAs.  Keys
  // split over the CTAs: `parts` to a pair, or (parts 0) equal shares of `each`
  // blocks, one more for the first `more` CTAs.
  // `rows` is then the rows of a line.
  int pack, pack_log2, lines, pairs, n_items, blocks, grid;
  bool split;
  int parts, each, more;
};
// Attention of up to 16 query rows over the cache (kv8_rows_sm100.cu); tk/tv are
// ax_make_tmap_codes maps with boxes of kv8_rows_tile() rows.
int kv8_rows_tile();
int kv8_rows_plan(Kv8AttnParams* p, int sms);
size_t kv8_rows_part_floats(int head_dim, int grid);
cudaError_t launch_kv8_rows(const CUtensorMap& tk, const CUtensorMap& tv, const Kv8AttnParams& p, int grid,
                            int dev, cudaStream_t stream);

// Attention over the cache in pairs of 128-row query tiles (kv8_attn_sm100.cu);
// tk/tv have 64-row boxes, tq and to are ax_make_tmap_rows maps of 128 and 32 rows.
bool kv8_attn_plan(Kv8AttnParams* p, int sms);  // false: too many items
size_t kv8_attn_part_floats(int head_dim, int grid);
cudaError_t launch_kv8_attn(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                            const CUtensorMap& to, const Kv8AttnParams& p, int dev, cudaStream_t stream);

// W8 (bits 8) / W4 (bits 4) codes + fp16 scale/zero per row and 64 columns ->
// fp16 [rows][out_stride] (dequant_sm100.cu).
cudaError_t launch_dequant(int bits, const void* packed, const void* scale, const void* zero, void* out,
                           int rows, int k, int64_t packed_stride, int64_t out_stride, int sms,
                           cudaStream_t stream);

}  // namespace ax
