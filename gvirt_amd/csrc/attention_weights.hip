// What every cached position was attended to: for each sequence, kv head g and position j
//     weights[j][g] (+)= sum over the counted rows r and the heads h of g of  exp(q_rh . k_j) / sum_{j' <= c + r} exp(q_rh . k_j')
// (c cached positions; row r sees positions 0 .. c + r; j <= c + r). Positions of the step itself start at zero, older ones
// keep what earlier steps left. No value of V is involved.
//
// Two kernels over the scores, which are formed twice instead of stored (a chunk of 2048 rows behind 6144 positions has
// 0.9 G of them, 3.7 GB in fp32):
//   row statistics: log2 of every row's normaliser. A wave owns 32 M rows (an M row: a counted row and one query head of the
//     kv head) as the columns of S^T = K Q^T, so a row's running maximum and sum live in one lane pair.
//   column sums: a wave owns 32 positions as the columns of S = Q K^T and walks the M rows, so a position's sum lives in
//     one lane pair: no atomics, one owner per weight, the same order of additions in every run.
// Both are bound by the exponentials (one per score in each) and the vector instructions around them.
#include <algorithm>
#include <type_traits>

#include "attention_common.h"
#include "kv8.h"

namespace xlite {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr uint32_t kRowTile = kWaves * 32;    // M rows of a workgroup of the first kernel
constexpr uint32_t kPosTile = kWaves * 32;    // positions of a workgroup of the second one
constexpr uint32_t kMinSplit = 256;           // positions a split of the first kernel walks at least

template <typename T>
__device__ __forceinline__ f32x16_t mfma32(const uint4 &a, const uint4 &b, f32x16_t c)
{
    if constexpr (T::kCode == XLITE_HIP_BF16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    }
}

struct WeightsParams {
    const uint16_t *q;
    const unsigned char *k_cache;
    const float *k_scale;          // 8-bit caches: [slot][kv head]
    float *weights;                // [slot][kv head]
    const int32_t *query_start_loc;
    const int32_t *lens;
    const int32_t *cached_lens;
    const int32_t *block_tables;
    float *stats;                  // [split][kv head][token * G + head of the group][2]: maximum (log2 domain), sum
    float *norm;                   // [kv head][token * G + head of the group]: -log2 of the row's normaliser
    uint32_t q_tok_stride;
    uint32_t group, n_kv_heads, batch, block_size, max_num_block;
    uint32_t window;               // counted rows: the last `window` of every sequence (0: all)
    uint32_t tiles_per_seq;        // row tiles of a sequence when a window bounds them (0: ids from the prefix sums)
    uint32_t m_total;              // total_tokens * G
    uint32_t splits, split_len;
};

// what a workgroup knows about its sequence
struct Sequence {
    uint32_t nodes, cached, start, first;   // rows of the step, cached positions, first token, first counted row
    uint32_t m_rows;                        // counted rows x G
};
__device__ __forceinline__ Sequence sequence_of(const WeightsParams &p, uint32_t seq)
{
    const int32_t n = p.lens[seq], c = p.cached_lens[seq], s = p.query_start_loc[seq];
    Sequence q;
    q.nodes = static_cast<uint32_t>(max(n, 0));
    q.cached = static_cast<uint32_t>(c);
    q.start = static_cast<uint32_t>(s);
    q.first = p.window != 0 && q.nodes > p.window ? q.nodes - p.window : 0u;
    q.m_rows = (q.nodes - q.first) * p.group;
    return q;
}

__device__ __forceinline__ uint64_t slot_of(const WeightsParams &p, const int32_t *table, uint32_t pos)
{
    const uint32_t b = pos / p.block_size;
    return static_cast<uint64_t>(static_cast<uint32_t>(table[b])) * p.block_size + (pos - b * p.block_size);
}

// chunk c (eight elements) of a cache row as T; a byte cache's values exactly, without their scale
template <typename T, int KVF>
__device__ __forceinline__ uint4 cache_chunk(const unsigned char *row, uint32_t c)
{
    if constexpr (KVF == XLITE_HIP_KV_SAME) {
        return *reinterpret_cast<const uint4 *>(row + c * 16);
    } else {
        return dequant8<T, KVF>(*reinterpret_cast<const uint2 *>(row + c * 8), 1.0f);
    }
}

template <typename T, int D, int KVF>
__global__ void __launch_bounds__(kThreads)
row_stats_kernel(const WeightsParams p)
{
    constexpr int KS = D / 16;
    constexpr uint32_t ROWB = D * (KVF == XLITE_HIP_KV_SAME ? 2 : 1);
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, half = lane >> 5;
    const uint32_t kvh = blockIdx.z, split = blockIdx.y, G = p.group;

    // ---- which rows: the tiles of a sequence are numbered from floor(start * G / tile) + i (a formula of the prefix sums,
    // at least as many ids as it has tiles), or evenly when a window bounds the counted rows
    uint32_t seq = 0, mt;
    if (p.tiles_per_seq != 0) {
        seq = blockIdx.x / p.tiles_per_seq;
        mt = blockIdx.x % p.tiles_per_seq;
    } else {
        auto first_id = [&](uint32_t i) {
            return static_cast<uint32_t>(static_cast<uint64_t>(p.query_start_loc[i]) * G / kRowTile) + i;
        };
        uint32_t hi = p.batch;
        while (hi - seq > 1) {
            const uint32_t mid = (seq + hi) >> 1;
            if (first_id(mid) <= blockIdx.x) {
                seq = mid;
            } else {
                hi = mid;
            }
        }
        mt = blockIdx.x - first_id(seq);
    }
    const Sequence s = sequence_of(p, seq);
    const uint32_t m_wave = mt * kRowTile + wave * 32;
    if (m_wave >= s.m_rows) {
        return;
    }
    const uint32_t m = min(m_wave + col, s.m_rows - 1);
    const uint32_t r = s.first + m / G;
    const uint32_t vis = s.cached + r + 1;                                       // of this lane's row
    const uint32_t vis_first = s.cached + s.first + m_wave / G + 1;              // of the wave's first row, the least
    const uint32_t vis_last = s.cached + s.first + min(m_wave + 31, s.m_rows - 1) / G + 1;
    const uint32_t begin = split * p.split_len, end = min(vis_last, begin + p.split_len);
    const int32_t *table = p.block_tables + static_cast<uint64_t>(seq) * p.max_num_block;

    float m_run = -INFINITY, l_run = 0.f;
    if (begin < end) {
        uint4 qreg[KS];
        const uint16_t *src = p.q + static_cast<uint64_t>(s.start + r) * p.q_tok_stride + static_cast<uint64_t>(kvh * G + m % G) * D;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            qreg[ks] = *reinterpret_cast<const uint4 *>(src + ks * 16 + half * 8);
        }
        for (uint32_t t0 = begin; t0 < end; t0 += 32) {
            // (positions past the end repeat the last one; their scores are masked)
            const uint64_t at = slot_of(p, table, min(t0 + col, end - 1)) * p.n_kv_heads + kvh;
            const unsigned char *row = p.k_cache + at * ROWB;
            f32x16_t S;
#pragma unroll
            for (int k = 0; k < 16; k++) {
                S[k] = 0.f;
            }
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                S = mfma32<T>(cache_chunk<T, KVF>(row, 2 * ks + half), qreg[ks], S);
            }
            if constexpr (KVF != XLITE_HIP_KV_SAME) {
                const float scale = p.k_scale[at];   // of position t0 + col; register k holds another one
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    S[k] *= __shfl(scale, static_cast<int>((k / 4) * 8 + half * 4 + (k % 4)));
                }
            }
            const uint32_t lim = min(vis, end);
            if (t0 + 32 > min(vis_first, end)) {
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    S[k] = t0 + (k / 4) * 8 + half * 4 + (k % 4) < lim ? S[k] : -INFINITY;
                }
            }
            float mx = m_run;
#pragma unroll
            for (int k = 0; k < 16; k++) {
                mx = fmaxf(mx, S[k]);
            }
            const float m_safe = mx == -INFINITY ? 0.f : mx;
            const float neg = -m_safe * kLog2e;
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < 16; k++) {
                sum += fast_exp2(__builtin_fmaf(S[k], kLog2e, neg));
            }
            l_run = l_run * fast_exp2((m_run - m_safe) * kLog2e) + sum;
            m_run = mx;
        }
    }
    // the two halves of a row's positions
    const float m_other = __shfl_xor(m_run, 32), l_other = __shfl_xor(l_run, 32);
    const float m_all = fmaxf(m_run, m_other);
    const float m_safe = m_all == -INFINITY ? 0.f : m_all;
    const float l_all = l_run * fast_exp2((m_run - m_safe) * kLog2e) + l_other * fast_exp2((m_other - m_safe) * kLog2e);
    if (half == 0 && m_wave + col < s.m_rows) {
        const uint64_t i = static_cast<uint64_t>(kvh) * p.m_total + static_cast<uint64_t>(s.start + s.first) * G + m_wave + col;
        if (p.splits == 1) {
            p.norm[i] = -(m_all * kLog2e + __log2f(l_all));
        } else {
            *reinterpret_cast<float2 *>(p.stats + (static_cast<uint64_t>(split) * p.n_kv_heads * p.m_total + i) * 2) =
                make_float2(m_all * kLog2e, l_all);
        }
    }
}

// joins the splits of every row (rows that nobody counted hold whatever the workspace held; nobody reads them)
__global__ void __launch_bounds__(256)
join_stats_kernel(const float *__restrict__ stats, float *__restrict__ norm, uint32_t rows, uint32_t splits)
{
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= rows) {
        return;
    }
    float m = -INFINITY, l = 0.f;
    for (uint32_t s = 0; s < splits; s++) {
        const float2 x = *reinterpret_cast<const float2 *>(stats + (static_cast<uint64_t>(s) * rows + i) * 2);
        const float mx = fmaxf(m, x.x), safe = mx == -INFINITY ? 0.f : mx;
        l = l * fast_exp2(m - safe) + x.y * fast_exp2(x.x - safe);
        m = mx;
    }
    norm[i] = -(m + __log2f(l));
}

template <typename T, int D, int KVF>
__global__ void __launch_bounds__(kThreads)
column_sums_kernel(const WeightsParams p)
{
    constexpr int KS = D / 16;
    constexpr uint32_t ROWB = D * (KVF == XLITE_HIP_KV_SAME ? 2 : 1);
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, half = lane >> 5;
    const uint32_t kvh = blockIdx.z, seq = blockIdx.y, G = p.group;
    const Sequence s = sequence_of(p, seq);
    const uint32_t total = s.cached + s.nodes;
    const uint32_t p0 = blockIdx.x * kPosTile + wave * 32;   // the wave's first position
    if (s.nodes == 0 || p0 >= total) {
        return;
    }
    const int32_t *table = p.block_tables + static_cast<uint64_t>(seq) * p.max_num_block;
    const uint32_t t = p0 + col;
    const uint64_t at = slot_of(p, table, min(t, total - 1)) * p.n_kv_heads + kvh;
    const unsigned char *row = p.k_cache + at * ROWB;
    uint4 kreg[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
        kreg[ks] = cache_chunk<T, KVF>(row, 2 * ks + half);
    }
    float mul = kLog2e;
    if constexpr (KVF != XLITE_HIP_KV_SAME) {
        mul *= p.k_scale[at];
    }
    // the first row that sees the wave's first position (rows before it see none of its positions)
    const uint32_t first_seen = p0 > s.cached + s.first ? (p0 - s.cached - s.first) * G : 0u;
    const uint64_t tok0 = s.start + s.first;
    const float *norm = p.norm + static_cast<uint64_t>(kvh) * p.m_total + tok0 * G;
    float acc = 0.f;
    for (uint32_t m0 = first_seen & ~31u; m0 < s.m_rows; m0 += 32) {
        const uint32_t m = min(m0 + col, s.m_rows - 1);
        const uint16_t *src = p.q + (tok0 + m / G) * p.q_tok_stride + static_cast<uint64_t>(kvh * G + m % G) * D;
        uint4 qop[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            qop[ks] = *reinterpret_cast<const uint4 *>(src + ks * 16 + half * 8);
        }
        float n[16];
#pragma unroll
        for (int k = 0; k < 16; k++) {
            n[k] = norm[min(m0 + (k / 4) * 8 + half * 4 + (k % 4), s.m_rows - 1)];
        }
        f32x16_t S;
#pragma unroll
        for (int k = 0; k < 16; k++) {
            S[k] = 0.f;
        }
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            S = mfma32<T>(qop[ks], kreg[ks], S);
        }
        float sum = 0.f;
        if (m0 + 32 > s.m_rows || p0 + 31 > s.cached + s.first + m0 / G) {
#pragma unroll
            for (int k = 0; k < 16; k++) {
                const uint32_t mk = m0 + (k / 4) * 8 + half * 4 + (k % 4);
                const float e = fast_exp2(__builtin_fmaf(S[k], mul, n[k]));
                sum += mk < s.m_rows && t <= s.cached + s.first + mk / G ? e : 0.f;
            }
        } else {
#pragma unroll
            for (int k = 0; k < 16; k++) {
                sum += fast_exp2(__builtin_fmaf(S[k], mul, n[k]));
            }
        }
        acc += sum;   // (a tile's sum first: 16 additions, then one per tile, instead of one chain over every row)
    }
    acc += __shfl_xor(acc, 32);
    if (half == 0 && t < total) {
        p.weights[at] = t < s.cached ? p.weights[at] + acc : acc;
    }
}

// KV splits of the row statistics: enough workgroups for four per compute unit
uint32_t stat_tiles(uint32_t total_tokens, uint32_t group, uint32_t batch, uint32_t window, uint32_t *per_seq)
{
    const uint64_t bounded = window == 0 ? 0 : static_cast<uint64_t>(std::min(window, total_tokens)) * group;
    *per_seq = static_cast<uint32_t>((bounded + kRowTile - 1) / kRowTile);
    const uint32_t by_prefix = ceil_div(total_tokens * group, kRowTile) + batch;
    if (*per_seq != 0 && static_cast<uint64_t>(*per_seq) * batch <= by_prefix) {
        return *per_seq * batch;
    }
    *per_seq = 0;
    return by_prefix;
}
uint32_t stat_splits(uint32_t tiles, uint32_t n_kv_heads, uint32_t max_ctx)
{
    const uint32_t want = ceil_div(1024u, std::max(1u, tiles * n_kv_heads));
    return std::max(1u, std::min(want, max_ctx / kMinSplit));
}

}  // namespace

}  // namespace xlite

using namespace xlite;

extern "C" size_t xlite_hip_attention_weights_workspace_bytes(uint32_t total_tokens, uint32_t n_heads, uint32_t n_kv_heads,
                                                              uint32_t block_size, uint32_t batch, uint32_t max_num_block,
                                                              uint32_t window)
{
    if (total_tokens == 0 || batch == 0 || n_kv_heads == 0 || n_heads % n_kv_heads != 0) {
        return 0;
    }
    uint32_t per_seq;
    const uint32_t tiles = stat_tiles(total_tokens, n_heads / n_kv_heads, batch, window, &per_seq);
    const uint64_t splits = stat_splits(tiles, n_kv_heads, max_num_block * block_size);
    const uint64_t rows = static_cast<uint64_t>(total_tokens) * n_heads;
    return static_cast<size_t>((rows + (splits > 1 ? 2 * splits * rows : 0)) * sizeof(float));
}

extern "C" int xlite_hip_attention_weights(void *stream, const void *qkv, const void *k_cache, float *weights,
                                           const int32_t *query_start_loc, const int32_t *lens, const int32_t *cached_lens,
                                           const int32_t *block_tables, uint32_t total_tokens, uint32_t n_heads,
                                           uint32_t n_kv_heads, uint32_t head_dim, uint32_t block_size, uint32_t batch,
                                           uint32_t max_num_block, uint32_t window, int dtype, int kv_dtype,
                                           const float *k_scale, void *workspace, size_t workspace_bytes)
{
    XL_REQUIRE(dtype == XLITE_HIP_FP16 || dtype == XLITE_HIP_BF16, "qkv/kCache dtype unsupported!");
    XL_REQUIRE(kv_dtype == XLITE_HIP_KV_SAME || kv_dtype == XLITE_HIP_KV_INT8 || kv_dtype == XLITE_HIP_KV_FP8,
               "kv cache dtype unsupported!");
    if (batch == 0 || total_tokens == 0) {
        return XLITE_HIP_OK;
    }
    XL_REQUIRE(qkv && k_cache && weights && query_start_loc && lens && cached_lens && block_tables, "null tensor");
    XL_REQUIRE(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0, "n_heads must be a positive multiple of n_kv_heads");
    XL_REQUIRE(block_size > 0 && max_num_block > 0, "block_size and max_num_block must be positive");
    XL_REQUIRE(static_cast<uint64_t>(max_num_block) * block_size < (1ull << 31), "block tables reach beyond 2^31 positions");
    XL_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "head_dim must be 64, 128 or 256");
    XL_REQUIRE(kv_dtype == XLITE_HIP_KV_SAME || k_scale, "a quantised K cache needs k_scale");
    XL_REQUIRE(kv_dtype == XLITE_HIP_KV_SAME || head_dim != 256, "quantised KV caches: head_dim must be 64 or 128");
    XL_REQUIRE(static_cast<uint64_t>(total_tokens) * n_heads < (1ull << 31) && batch <= 65535 && n_kv_heads <= 65535,
               "more rows than one launch takes");
    const size_t need = xlite_hip_attention_weights_workspace_bytes(total_tokens, n_heads, n_kv_heads, block_size, batch,
                                                                    max_num_block, window);
    if (workspace == nullptr || workspace_bytes < need) {
        return fail(XLITE_HIP_ENOSPC, __func__, "workspace too small: need " + std::to_string(need) + " bytes, have " +
                                                    std::to_string(workspace == nullptr ? 0 : workspace_bytes));
    }
    hipStream_t s = as_stream(stream);
    const uint32_t G = n_heads / n_kv_heads, max_ctx = max_num_block * block_size;
    WeightsParams p{};
    p.q = static_cast<const uint16_t *>(qkv);
    p.k_cache = static_cast<const unsigned char *>(k_cache);
    p.k_scale = k_scale;
    p.weights = weights;
    p.query_start_loc = query_start_loc;
    p.lens = lens;
    p.cached_lens = cached_lens;
    p.block_tables = block_tables;
    p.q_tok_stride = (n_heads + 2 * n_kv_heads) * head_dim;
    p.group = G;
    p.n_kv_heads = n_kv_heads;
    p.batch = batch;
    p.block_size = block_size;
    p.max_num_block = max_num_block;
    p.window = window;
    p.m_total = total_tokens * G;
    const uint32_t tiles = stat_tiles(total_tokens, G, batch, window, &p.tiles_per_seq);
    p.splits = stat_splits(tiles, n_kv_heads, max_ctx);
    p.split_len = ceil_div(ceil_div(max_ctx, p.splits), 32u) * 32u;
    const uint32_t rows = total_tokens * n_heads;
    p.norm = static_cast<float *>(workspace);
    p.stats = p.norm + rows;
    auto launch = [&](auto t, auto d, auto kvf) -> int {
        using T = decltype(t);
        constexpr int D = decltype(d)::value, KVF = decltype(kvf)::value;
        row_stats_kernel<T, D, KVF><<<dim3(tiles, p.splits, n_kv_heads), kThreads, 0, s>>>(p);
        XL_LAUNCH_CHECK();
        if (p.splits > 1) {
            join_stats_kernel<<<ceil_div(rows, 256u), 256, 0, s>>>(p.stats, p.norm, rows, p.splits);
            XL_LAUNCH_CHECK();
        }
        column_sums_kernel<T, D, KVF><<<dim3(ceil_div(max_ctx, kPosTile), batch, n_kv_heads), kThreads, 0, s>>>(p);
        XL_LAUNCH_CHECK();
        return XLITE_HIP_OK;
    };
    auto with_dim = [&](auto t, auto kvf) -> int {
        using D64 = std::integral_constant<int, 64>;
        using D128 = std::integral_constant<int, 128>;
        if constexpr (decltype(kvf)::value == XLITE_HIP_KV_SAME) {
            if (head_dim == 256) {
                return launch(t, std::integral_constant<int, 256>{}, kvf);
            }
        }
        return head_dim == 128 ? launch(t, D128{}, kvf) : launch(t, D64{}, kvf);
    };
    auto with_cache = [&](auto t) -> int {
        switch (kv_dtype) {
        case XLITE_HIP_KV_INT8: return with_dim(t, std::integral_constant<int, XLITE_HIP_KV_INT8>{});
        case XLITE_HIP_KV_FP8: return with_dim(t, std::integral_constant<int, XLITE_HIP_KV_FP8>{});
        default: return with_dim(t, std::integral_constant<int, XLITE_HIP_KV_SAME>{});
        }
    };
    return dtype == XLITE_HIP_BF16 ? with_cache(BF16{}) : with_cache(FP16{});
}
