// Argument bundles and launcher declarations shared by the attention entry points.
#pragma once

#include "common.h"

namespace xlite {

struct AttentionArgs {
    const void *qkv;
    const void *k_cache;
    const void *v_cache;
    void *output;
    const int32_t *query_start_loc;
    const int32_t *lens;
    const int32_t *cached_lens;
    const int32_t *block_tables;
    uint32_t total_tokens, n_heads, n_kv_heads, head_dim, block_size, batch, max_num_block;
    int dtype, kv_dtype;
    const float *k_scale;
    const float *v_scale;
    void *workspace;
    size_t workspace_bytes;
    // a batch served by two kernels: kOnlySingle = only the sequences with exactly one query row (the decode
    // kernels), kSkipSingle = all the others (the prefill kernel, the dequantising copy)
    int rows_mode;
    // a bf16 model over the fp16 copy of a quantised cache, on a kernel that converts at its edges: dtype says
    // FP16 (the products), qkv and output are bf16
    bool io_bf16;
    // a drafted tree per sequence: row r sees every cached position, and of the step's own positions those whose bit is
    // set in its mask_words words (nullptr: causal)
    const uint32_t *tree_mask;
    uint32_t mask_words;
};
enum { kAllRows = 0, kOnlySingle = 1, kSkipSingle = 2 };

inline bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// the low n bits (none below 0, all from 32 on)
__device__ __forceinline__ uint32_t ones(int32_t n)
{
    return static_cast<uint32_t>((1ull << min(max(n, 0), 32)) - 1);
}
// Which of the positions j0 .. j0 + 31 a tree row sees, as bits. `words`: the row's mask, bit n = drafted node n, which sits
// at position `cached` + n; every position below `cached` is seen, none at or beyond `cached` + `nodes`.
__device__ __forceinline__ uint32_t tree_seen(const uint32_t *words, uint32_t n_words, uint32_t j0, uint32_t cached, uint32_t nodes)
{
    const int32_t off = static_cast<int32_t>(j0 - cached);   // the node of position j0; negative: cached positions
    const int32_t i = off >> 5;
    const uint32_t sh = static_cast<uint32_t>(off) & 31u;
    // (loads from clamped indexes, selected afterwards: a load under a condition is awaited on its own)
    const int32_t last = static_cast<int32_t>(n_words) - 1;
    const uint32_t a = words[min(max(i, 0), last)], b = words[min(max(i + 1, 0), last)];
    const uint64_t both = (i >= 0 && i <= last ? a : 0u) | (static_cast<uint64_t>(i + 1 >= 0 && i + 1 <= last ? b : 0u) << 32);
    uint32_t seen = static_cast<uint32_t>(both >> sh);
    seen |= ones(-off);
    return seen & ones(static_cast<int32_t>(nodes) - off);   // (nodes - off: positions of the sequence from j0 on)
}

// 16-bit pairs with an infinity or a NaN in either half
template <typename T>
__device__ __forceinline__ bool not_finite2(uint32_t w)
{
    constexpr uint32_t e = T::kCode == XLITE_HIP_BF16 ? 0x7f80u : 0x7c00u;
    return static_cast<uint32_t>((w & e) == e) | static_cast<uint32_t>((w & (e << 16)) == (e << 16));
}

// the pair with its infinities and NaNs as zeros
template <typename T>
__device__ __forceinline__ uint32_t finite_only(uint32_t w)
{
    constexpr uint32_t e = T::kCode == XLITE_HIP_BF16 ? 0x7f80u : 0x7c00u;
    return ((w & e) == e ? 0u : w & 0xffffu) | ((w & (e << 16)) == (e << 16) ? 0u : w & 0xffff0000u);
}
// eight 16-bit values as indicators (1 or 0) of +infinity (what = 0), -infinity (1) or NaN (2)
template <typename T>
__device__ __forceinline__ uint4 odd_values(const uint2 &lo, const uint2 &hi, int what)
{
    constexpr uint32_t e = T::kCode == XLITE_HIP_BF16 ? 0x7f80u : 0x7c00u, one = T::kCode == XLITE_HIP_BF16 ? 0x3f80u : 0x3c00u;
    auto is = [&](uint32_t h) {
        return what == 0 ? h == e : what == 1 ? h == (e | 0x8000u) : (h & 0x7fffu) > e;
    };
    auto pair = [&](uint32_t w) { return (is(w & 0xffffu) ? one : 0u) | (is(w >> 16) ? one << 16 : 0u); };
    return make_uint4(pair(lo.x), pair(lo.y), pair(hi.x), pair(hi.y));
}

struct MlaArgs {
    const void *q_absorb;
    const void *qr;
    const void *k_cache;     // paged [blocks, block_size, kv_lora_rank] or dense [batch, index_topk, ...]
    const void *pe_cache;
    void *o_absorb;
    const int32_t *query_start_loc;
    const int32_t *lens;
    const int32_t *cached_lens;
    const int32_t *block_tables;   // nullptr: dense per-sequence cache (mla_v3)
    uint32_t total_tokens, n_heads, rope_head_dim, kv_lora_rank, block_size, batch, max_num_blocks;
    uint32_t dense_len;            // mla_v3: entries per sequence, attention is not causal
    float scale;
    const int32_t *topk_indices;
    uint32_t top_k;
    int dtype;
    void *workspace;
    size_t workspace_bytes;
};

// merge.hip: scratch for split-KV partial results and their merge.
// Layout of the workspace: cnt[rows * n_heads] int32 (number of partials of a (row, head); 0 = the
// producer stored the final value itself), then acc[rows * n_heads][max_slots][dv] and
// ml[rows * n_heads][max_slots][2] (running maximum in the log2 domain, sum) in fp32.
struct PartialBuffers {
    int32_t *cnt;
    float *acc;
    float *ml;
};
size_t partial_bytes(uint32_t rows, uint32_t n_heads, uint32_t dv, uint32_t max_slots);
PartialBuffers carve_partials(void *workspace, uint32_t rows, uint32_t n_heads, uint32_t dv, uint32_t max_slots);
int launch_merge(hipStream_t stream, int dtype, void *out, const PartialBuffers &b, uint32_t rows,
                 uint32_t n_heads, uint32_t dv, uint32_t max_slots);
int launch_clear_counts(hipStream_t stream, const PartialBuffers &b, uint32_t rows, uint32_t n_heads);
// Partials of the MLA decode kernel: a row's s-th segment sits in slot 2 c0 + (1 - first flag) for s = 0 and
// 2 (c0 + s) after that (meta = segments, c0, first flag per row); acc holds O / l in the 16-bit activation type.
int launch_merge_mla(hipStream_t stream, int dtype, void *out, const uint16_t *acc, const float *ml, const int32_t *meta,
                     uint32_t rows, uint32_t n_heads, uint32_t dv);
// The same slot scheme with fp32 partials (O, maximum in the log2 domain, normaliser), [slot][head][dv].
int launch_merge_meta(hipStream_t stream, int dtype, void *out, const float *acc, const float *ml, const int32_t *meta,
                      uint32_t rows, uint32_t n_heads, uint32_t dv);

// decode_attention.hip
bool decode_supported(uint32_t head_dim);
void decode_geometry(uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, uint32_t *g_kernel,
                     uint32_t *head_chunks, uint32_t *nkv_wg, uint32_t *zdim);
uint32_t decode_pick_tile(uint32_t batch, uint32_t n_kv_heads, uint32_t block_size,
                          uint32_t max_num_block, uint32_t zdim);
size_t decode_workspace_bytes(uint32_t total_tokens, uint32_t n_heads, uint32_t head_dim,
                              uint32_t max_tiles);
int launch_decode(hipStream_t stream, const AttentionArgs &a, uint32_t tile_tokens);

// decode_mfma.hip
bool decode_dma256_supported(uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, uint32_t block_size, int kv_dtype);
bool decode_mfma_supported(uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, uint32_t block_size,
                           uint32_t total_tokens);
struct DecodeSplitPlan {
    uint32_t max_chunks;   // bound on the number of chunks, hence of partial slots (two per chunk)
    size_t meta_bytes, ml_bytes, acc_bytes;
};
size_t decode_mfma_workspace_bytes(uint32_t batch, uint32_t n_heads, uint32_t head_dim, uint32_t block_size,
                                   uint32_t max_num_block);
// `rope`: the batch's rope_and_cache arguments, for a batch that decode_mfma_whole_rows accepts: the kernel then
// rotates and stores the rows itself
struct RopeArgs;
bool decode_mfma_whole_rows(const AttentionArgs &a);
int launch_decode_mfma(hipStream_t stream, const AttentionArgs &a, const RopeArgs *rope = nullptr);
uint32_t decode_mfma_slice_units();   // units (rows, sequences) one launch of the decode kernels can split

// mla_decode.hip
struct MlaDecodeParams {
    const uint16_t *q_absorb;
    const uint16_t *qr;
    const uint16_t *k_cache;
    const uint16_t *pe_cache;
    uint16_t *out;
    const int32_t *query_start_loc;
    const int32_t *lens;
    const int32_t *cached_lens;
    const int32_t *block_tables;   // nullptr: dense cache, dense_len rows per sequence, no causality
    int32_t *part_meta;   // [total_rows][4]: segments of the row (0: stored directly), first chunk, first-in-chunk flag
    float *part_acc;      // [2 * chunks][n_heads][512] 16-bit, O / l of a partial slot
    float *part_ml;       // [2 * chunks][n_heads][2]: running maximum (log2 domain), sum
    uint32_t n_heads;
    uint32_t batch;
    uint32_t total_rows;
    uint32_t block_size;
    uint32_t max_num_blocks;
    uint32_t dense_len;
    uint32_t chunk_min_steps;
    float scale_log2e;
    const int32_t *topk_indices;   // [total_rows][top_k] position lists (top_k == 0: none)
    uint32_t top_k;
    unsigned long long *clock_probe;   // nullptr, or where workgroup 0 leaves its shader-clock and wall-clock stamps
    uint32_t by_pos;      // 1: block sizes that are not a multiple of 32 - every row walks a list of positions, its own
                          // (0, 1, 2, ...) unless topk_indices gives it one
};
bool mla_decode_supported(const MlaArgs &a);
size_t mla_decode_workspace_bytes(const MlaArgs &a);
int launch_mla_decode(hipStream_t stream, const MlaArgs &a);

// prefill_mfma.hip
bool prefill_mfma_supported(const AttentionArgs &a);
bool prefill_kv8_supported(const AttentionArgs &a);
int launch_prefill_mfma(hipStream_t stream, const AttentionArgs &a);
size_t prefill_mfma_workspace_bytes(uint32_t total_tokens, uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim,
                                    uint32_t batch, uint32_t max_ctx);

// tree_stream.hip
bool tree_stream_supported(uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, uint32_t block_size, uint32_t batch,
                           uint32_t max_num_block, int kv_dtype);
size_t tree_stream_workspace_bytes(uint32_t total_tokens, uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, uint32_t batch,
                                   uint32_t block_size, uint32_t max_num_block);
int launch_tree_stream(hipStream_t stream, const AttentionArgs &a);

// kv_dequant.hip: the 16-bit copy of a quantised cache's visible blocks, at the front of the workspace
size_t kv_dequant_bytes(uint32_t n_kv_heads, uint32_t head_dim, uint32_t block_size, uint32_t batch, uint32_t max_num_block);
int launch_kv_dequant(hipStream_t stream, AttentionArgs *a);
// bf16 models run over the fp16 copy in fp16: converted queries and an fp16 result buffer in the workspace
size_t kv_dequant_f16_io_bytes(uint32_t total_tokens, uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim);
int launch_kv_dequant_f16_begin(hipStream_t stream, AttentionArgs *a, void **real_out);
int launch_kv_dequant_f16_finish(hipStream_t stream, const AttentionArgs &a, void *real_out);

// mla_topk.hip
size_t mla_topk_scratch_bytes(uint32_t total_tokens, uint32_t kv_lora_rank, uint32_t rope_head_dim, uint32_t top_k);
int launch_mla_topk(hipStream_t stream, const MlaArgs &a);

// mfma_attention.hip
bool mfma_gqa_supported(uint32_t head_dim);
size_t mfma_workspace_bytes(uint32_t total_tokens, uint32_t n_heads, uint32_t dv, uint32_t splits);
uint32_t mfma_pick_splits(uint32_t total_tokens, uint32_t rows_per_token, uint32_t batch,
                          uint32_t parallel_heads, uint32_t max_ctx, uint32_t tile);
int launch_mfma_gqa(hipStream_t stream, const AttentionArgs &a);
int launch_mfma_mla(hipStream_t stream, const MlaArgs &a);
// mla_generic.hip: any latent / rotary size, no matrix instructions
int launch_mla_generic(hipStream_t stream, const MlaArgs &a);

}  // namespace xlite
